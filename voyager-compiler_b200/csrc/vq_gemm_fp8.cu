// E4M3 x E4M3 linear with float32 scales per block of 128 on the
// 5th-generation tensor cores (tcgen05.mma.kind::f8f6f4):
//
//   out[m, n] = bf16( bias[n] + sum_kb sa[m, kb] * sw[n / 128, kb]
//                     * sum_{k in block kb} a[m, k] * w[n, k] )
//
// The scales are any float32 values, so they cannot ride in the MMA: each
// 128-column block of K is one tensor-core product (exact products, float32
// sums) into its own TMEM buffer, and the promotion warps read it back
// (tcgen05.ld) and add it, times its scale, to float32 sums in registers.
// The MMAs of the next blocks run meanwhile: one multiply-add per output and
// block on the CUDA cores against 128 on the tensor cores.
//
// k_fp8_wide  many tokens: tiles of 128 tokens (TMEM lanes) x BN weight rows
//             (columns), persistent; a thread's scale is one scalar per block.
// k_fp8_few   few tokens: tiles of 128 weight rows (lanes) x BN tokens, so
//             that no lane is idle when the weight is all there is to read;
//             K is split over a cluster of CTAs, whose float32 sums are added
//             in rank order through distributed shared memory.
//
// TMA zero-fills rows and columns past the operands' ends.  Waits are
// bounded.  No TMA multicast is used.
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <algorithm>

#include "voyager_b200.h"
#include "vq_e4m3.cuh"
#include "vq_tc.cuh"

namespace vq {
namespace f8 {

using namespace vq::e4;
using namespace vq::tc;

enum { ERR_FULL = 321, ERR_EMPTY = 322, ERR_ACC = 323, ERR_DRAIN = 324 };

constexpr int BK = 128;  // K columns per stage = one scale block

struct Args {
  const float *sa, *sw;
  const uint16_t* bias;
  uint16_t* out;
  int64_t ldo;
  int M, N, nk;        // nk = ceil(K / 128)
  int mt, nt, tiles;   // tiles of this kernel's shape
  int splits;          // k_fp8_few: CTAs of a cluster
  int vec;             // out rows take 16-byte stores
};

// Instruction descriptor, kind::f8f6f4: E4M3 x E4M3, float32 sums, K-major
// operands, M x N.
__host__ __device__ constexpr uint32_t idesc(uint32_t M, uint32_t N) {
  return (1u << 4) | ((N >> 3) << 17) | ((M >> 4) << 24);
}
__device__ __forceinline__ void mma_f8(uint32_t d, uint64_t da, uint64_t db, uint32_t id, uint32_t acc) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
      "l"(da), "l"(db), "r"(id), "r"(acc));
}
__device__ __forceinline__ void tmem_ld16(uint32_t taddr, uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,"
      "%14,%15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]),
        "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]),
        "=r"(r[14]), "=r"(r[15])
      : "r"(taddr));
}

// The four K = 32 MMAs of one stage (SWIZZLE_128B operands) into TMEM columns d.
__device__ __forceinline__ void mma_stage(uint32_t d, uint64_t da, uint64_t db, uint32_t id) {
#pragma unroll
  for (uint32_t j = 0; j < 4; ++j) mma_f8(d, desc_at(da, 2 * j), desc_at(db, 2 * j), id, j > 0);
}

// Before the CTA frees its TMEM and leaves: the loads of the last round of
// stages that the producer armed have landed (a stage never armed reads as
// complete at parity 1).
template <int STAGES>
__device__ __forceinline__ void drain_loads(uint32_t full0, int stage, uint32_t phase) {
#pragma unroll 1
  for (int s = 0; s < STAGES; ++s)
    mbar_wait(full0 + 8 * s, s < stage ? phase : phase ^ 1, nullptr, ERR_DRAIN);
}

// ---------------------------------------------------------------------------
template <int BN>
struct Wide {
  static constexpr int STAGES = BN == 256 ? 4 : 6;
  static constexpr int A_BYTES = 128 * BK, B_BYTES = BN * BK, STAGE = A_BYTES + B_BYTES;
  static constexpr int BUFS = 512 / BN;
  static constexpr int THREADS = 320;
  static constexpr int SMEM = STAGES * STAGE + 1024 + 256;
  static constexpr int COLS = BN / 2;  // columns per promotion warp
};

// Tile -> (token tile, weight tile): token tiles fastest within groups of 8,
// so that the CTAs of a wave share few rows of both operands.
__device__ __forceinline__ void tile_of(const Args& a, int t, int& tm, int& tn) {
  const int per = 8 * a.nt, gr = t / per, in = t - gr * per;
  const int rows = min(8, a.mt - gr * 8);
  tn = in / rows;
  tm = gr * 8 + in - tn * rows;
}

template <int BN>
__global__ void __launch_bounds__(Wide<BN>::THREADS, 1)
    k_fp8_wide(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_w,
               const __grid_constant__ Args a) {
  using C = Wide<BN>;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                             ~(uintptr_t)1023);
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + C::STAGES * C::STAGE);
  const uint32_t full0 = smem_u32(bars), empty0 = full0 + 8 * C::STAGES;
  const uint32_t acc_full0 = empty0 + 8 * C::STAGES, acc_empty0 = acc_full0 + 8 * C::BUFS;
  const uint32_t drain = acc_empty0 + 8 * C::BUFS;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 2 * C::STAGES + 2 * C::BUFS + 1);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int s = 0; s < C::STAGES; ++s) mbar_init(full0 + 8 * s, 1), mbar_init(empty0 + 8 * s, 1);
    for (int s = 0; s < C::BUFS; ++s) mbar_init(acc_full0 + 8 * s, 1), mbar_init(acc_empty0 + 8 * s, 8);
    mbar_init(drain, 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(
                     smem_u32(tmem_slot)), "r"(512));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;

  if (warp == 0) {
    if (lane == 0) {
      int stage = 0;
      uint32_t phase = 0;
      bool ok = true;
      for (int t = blockIdx.x; t < a.tiles && ok; t += gridDim.x) {
        int tm, tn;
        tile_of(a, t, tm, tn);
        for (int kt = 0; kt < a.nk; ++kt) {
          if (!mbar_wait(empty0 + 8 * stage, phase ^ 1, nullptr, ERR_EMPTY)) {
            ok = false;
            break;
          }
          const uint32_t dst = smem_u32(smem) + stage * C::STAGE;
          mbar_expect_tx(full0 + 8 * stage, C::STAGE);
          tma_load_2d(dst, &map_a, kt * BK, tm * 128, full0 + 8 * stage);
          tma_load_2d(dst + C::A_BYTES, &map_w, kt * BK, tn * BN, full0 + 8 * stage);
          if (++stage == C::STAGES) stage = 0, phase ^= 1;
        }
      }
      drain_loads<C::STAGES>(full0, stage, phase);
    }
  } else if (warp == 1) {
    if (lane == 0) {
      int stage = 0, buf = 0;
      uint32_t phase = 0, bphase = 0;
      bool ok = true;
      for (int t = blockIdx.x; t < a.tiles && ok; t += gridDim.x) {
        for (int kt = 0; kt < a.nk; ++kt) {
          if (!mbar_wait(acc_empty0 + 8 * buf, bphase ^ 1, nullptr, ERR_ACC) ||
              !mbar_wait(full0 + 8 * stage, phase, nullptr, ERR_FULL)) {
            ok = false;
            break;
          }
          tc_fence_after();
          const uint32_t s0 = smem_u32(smem) + stage * C::STAGE;
          mma_stage(tmem + buf * BN, sw128_desc(s0), sw128_desc(s0 + C::A_BYTES), idesc(128, BN));
          tc_commit(empty0 + 8 * stage);
          tc_commit(acc_full0 + 8 * buf);
          if (++stage == C::STAGES) stage = 0, phase ^= 1;
          if (++buf == C::BUFS) buf = 0, bphase ^= 1;
        }
      }
      tc_commit(drain);
      mbar_wait(drain, 0, nullptr, ERR_DRAIN);
    }
  } else {
    // promotion: warps 2..9, two per TMEM lane quarter, COLS columns each
    const int q = warp & 3, half = (warp - 2) >> 2;
    int buf = 0;
    uint32_t bphase = 0;
    bool ok = true;
    for (int t = blockIdx.x; t < a.tiles && ok; t += gridDim.x) {
      int tm, tn;
      tile_of(a, t, tm, tn);
      const int row = tm * 128 + q * 32 + lane;
      const int col0 = tn * BN + half * C::COLS;
      const float* sa = a.sa + (int64_t)min(row, a.M - 1) * a.nk;
      const float* sw = a.sw + (int64_t)min(col0 / 128, (a.N - 1) / 128) * a.nk;
      float acc[C::COLS];
#pragma unroll
      for (int i = 0; i < C::COLS; ++i) acc[i] = 0.0f;
      float na = __ldg(sa), nw = __ldg(sw);
      for (int kt = 0; kt < a.nk; ++kt) {
        const float s = na * nw;
        const int kn = min(kt + 1, a.nk - 1);
        na = __ldg(sa + kn), nw = __ldg(sw + kn);
        if (!mbar_wait_warp(acc_full0 + 8 * buf, bphase, nullptr, ERR_ACC)) {
          ok = false;
          break;
        }
        tc_fence_after();
        const uint32_t taddr = tmem + ((uint32_t)(q * 32) << 16) + buf * BN + half * C::COLS;
#pragma unroll
        for (int c = 0; c < C::COLS / 32; ++c) {
          uint32_t r[32];
          tmem_ld32(taddr + c * 32, r);
          tmem_ld_wait();
#pragma unroll
          for (int i = 0; i < 32; ++i)
            acc[c * 32 + i] = fmaf(__uint_as_float(r[i]), s, acc[c * 32 + i]);
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(acc_empty0 + 8 * buf);
        if (++buf == C::BUFS) buf = 0, bphase ^= 1;
      }
      if (row < a.M && ok) {
        uint16_t* o = a.out + (int64_t)row * a.ldo + col0;
#pragma unroll
        for (int c = 0; c < C::COLS; c += 8) {
          if (a.vec && col0 + c + 8 <= a.N) {
            float v[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = acc[c + i];
            if (a.bias) {
              float bb[8];
              BF16::load8(a.bias + col0 + c, bb);
#pragma unroll
              for (int i = 0; i < 8; ++i) v[i] += bb[i];
            }
            BF16::store8(o + c, v);
          } else {
#pragma unroll
            for (int i = 0; i < 8; ++i)
              if (col0 + c + i < a.N)
                BF16::store(o + c + i, acc[c + i] + (a.bias ? BF16::load(a.bias + col0 + c + i) : 0.0f));
          }
        }
      }
    }
  }
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512));
  }
}

// ---------------------------------------------------------------------------
template <int BN>
struct Few {
  static constexpr int W_BYTES = 128 * BK, X_BYTES = BN * BK, STAGE = W_BYTES + X_BYTES;
  static constexpr int STAGES = BN == 16 ? 5 : BN == 32 ? 4 : BN == 64 ? 4 : 3;
  static constexpr int BUFS = BN == 128 ? 2 : 4;
  static constexpr int TMEM = BUFS * BN < 32 ? 32 : BUFS * BN;
  static constexpr int THREADS = 192;
  static constexpr int KC = 16;  // K blocks per refill of the scales
  static constexpr int LD = 132; // floats per token of the sums in shared memory
  static constexpr int RING = STAGES * STAGE > BN * LD * 4 ? STAGES * STAGE : BN * LD * 4;
  static constexpr int SMEM = RING + KC * BN * 4 + 1024 + 256;
  static_assert(2 * SMEM + 2048 <= 227 * 1024, "two CTAs per SM");
};

template <int BN>
__global__ void __launch_bounds__(Few<BN>::THREADS, 2)
    k_fp8_few(const __grid_constant__ CUtensorMap map_x, const __grid_constant__ CUtensorMap map_w,
              const __grid_constant__ Args a) {
  using C = Few<BN>;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                             ~(uintptr_t)1023);
  float* s_scale = reinterpret_cast<float*>(smem + C::RING);  // [KC][BN]
  uint64_t* bars = reinterpret_cast<uint64_t*>(s_scale + C::KC * BN);
  const uint32_t full0 = smem_u32(bars), empty0 = full0 + 8 * C::STAGES;
  const uint32_t acc_full0 = empty0 + 8 * C::STAGES, acc_empty0 = acc_full0 + 8 * C::BUFS;
  const uint32_t drain = acc_empty0 + 8 * C::BUFS;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 2 * C::STAGES + 2 * C::BUFS + 1);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rank = a.splits > 1 ? (int)cluster_ctarank() : 0;
  const int tile = blockIdx.x / a.splits, tm = tile / a.nt, tn = tile - tm * a.nt;
  const int kb0 = (int)((int64_t)a.nk * rank / a.splits);
  const int kb1 = (int)((int64_t)a.nk * (rank + 1) / a.splits);
  if (threadIdx.x == 0) {
    for (int s = 0; s < C::STAGES; ++s) mbar_init(full0 + 8 * s, 1), mbar_init(empty0 + 8 * s, 1);
    for (int s = 0; s < C::BUFS; ++s) mbar_init(acc_full0 + 8 * s, 1), mbar_init(acc_empty0 + 8 * s, 4);
    mbar_init(drain, 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(
                     smem_u32(tmem_slot)), "r"(C::TMEM));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;

  if (warp == 0) {
    if (lane == 0) {
      int stage = 0;
      uint32_t phase = 0;
      for (int kt = kb0; kt < kb1; ++kt) {
        if (!mbar_wait(empty0 + 8 * stage, phase ^ 1, nullptr, ERR_EMPTY)) break;
        const uint32_t dst = smem_u32(smem) + stage * C::STAGE;
        mbar_expect_tx(full0 + 8 * stage, C::STAGE);
        tma_load_2d(dst, &map_w, kt * BK, tn * 128, full0 + 8 * stage);
        tma_load_2d(dst + C::W_BYTES, &map_x, kt * BK, tm * BN, full0 + 8 * stage);
        if (++stage == C::STAGES) stage = 0, phase ^= 1;
      }
      drain_loads<C::STAGES>(full0, stage, phase);
    }
  } else if (warp == 1) {
    if (lane == 0) {
      int stage = 0, buf = 0;
      uint32_t phase = 0, bphase = 0;
      for (int kt = kb0; kt < kb1; ++kt) {
        if (!mbar_wait(acc_empty0 + 8 * buf, bphase ^ 1, nullptr, ERR_ACC) ||
            !mbar_wait(full0 + 8 * stage, phase, nullptr, ERR_FULL))
          break;
        tc_fence_after();
        const uint32_t s0 = smem_u32(smem) + stage * C::STAGE;
        mma_stage(tmem + buf * BN, sw128_desc(s0), sw128_desc(s0 + C::W_BYTES), idesc(128, BN));
        tc_commit(empty0 + 8 * stage);
        tc_commit(acc_full0 + 8 * buf);
        if (++stage == C::STAGES) stage = 0, phase ^= 1;
        if (++buf == C::BUFS) buf = 0, bphase ^= 1;
      }
      tc_commit(drain);
      mbar_wait(drain, 0, nullptr, ERR_DRAIN);
    }
  }
  float acc[BN];
  const int q = warp & 3;  // TMEM lane quarter of warps 2..5
  if (warp >= 2) {
    int buf = 0;
    uint32_t bphase = 0;
    const int pt = threadIdx.x - 64;
    const float* sw = a.sw + (int64_t)tn * a.nk;
#pragma unroll
    for (int i = 0; i < BN; ++i) acc[i] = 0.0f;
    bool ok = true;
    for (int kc = kb0; kc < kb1; kc += C::KC) {
      // the scales of the next KC blocks, sa * sw per block and token
      asm volatile("bar.sync 1, 128;" ::: "memory");
      const int n = min(C::KC, kb1 - kc);
      for (int i = pt; i < C::KC * BN; i += 128) {
        const int j = i / C::KC, k = i % C::KC;  // consecutive threads: consecutive blocks of a token
        const int m = min(tm * BN + j, a.M - 1);
        if (k < n) s_scale[k * BN + j] = __ldg(a.sa + (int64_t)m * a.nk + kc + k) * __ldg(sw + kc + k);
      }
      asm volatile("bar.sync 1, 128;" ::: "memory");
      for (int k = 0; k < n && ok; ++k) {
        if (!mbar_wait_warp(acc_full0 + 8 * buf, bphase, nullptr, ERR_ACC)) {
          ok = false;
          break;
        }
        tc_fence_after();
        const uint32_t taddr = tmem + ((uint32_t)(q * 32) << 16) + buf * BN;
#pragma unroll
        for (int c = 0; c < BN; c += 16) {
          uint32_t r[16];
          tmem_ld16(taddr + c, r);
          tmem_ld_wait();
#pragma unroll
          for (int i = 0; i < 16; i += 4) {
            const float4 s = *reinterpret_cast<const float4*>(s_scale + k * BN + c + i);
            acc[c + i] = fmaf(__uint_as_float(r[i]), s.x, acc[c + i]);
            acc[c + i + 1] = fmaf(__uint_as_float(r[i + 1]), s.y, acc[c + i + 1]);
            acc[c + i + 2] = fmaf(__uint_as_float(r[i + 2]), s.z, acc[c + i + 2]);
            acc[c + i + 3] = fmaf(__uint_as_float(r[i + 3]), s.w, acc[c + i + 3]);
          }
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(acc_empty0 + 8 * buf);
        if (++buf == C::BUFS) buf = 0, bphase ^= 1;
      }
    }
  }
  // Every MMA has read its stage and every load has landed (the producer and
  // the MMA thread waited for theirs), so the ring holds the sums from here
  // on: [BN tokens][128 rows].
  __syncthreads();
  float* red = reinterpret_cast<float*>(smem);
  if (warp >= 2) {
#pragma unroll
    for (int i = 0; i < BN; ++i) red[i * C::LD + q * 32 + lane] = acc[i];
  }
  if (a.splits > 1)
    cluster_sync();
  else
    __syncthreads();
  // tokens rank, rank + splits, ..; a thread takes 4 weight rows of a token
  const int ntok = min(BN, a.M - tm * BN);
  const uint32_t red_addr = smem_u32(red);
  for (int i = threadIdx.x; i < BN * 32; i += C::THREADS) {
    const int j = (i >> 5) * a.splits + rank, f = (i & 31) * 4, n = tn * 128 + f;
    if (j >= ntok) break;
    float v[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    for (int r = 0; r < a.splits; ++r) {
      float x[4];
      const uint32_t p = red_addr + (j * C::LD + f) * 4;
      const uint32_t src = a.splits > 1 ? mapa_shared(p, r) : p;
      asm volatile("ld.shared::cluster.v4.f32 {%0,%1,%2,%3}, [%4];"
                   : "=f"(x[0]), "=f"(x[1]), "=f"(x[2]), "=f"(x[3]) : "r"(src) : "memory");
#pragma unroll
      for (int k = 0; k < 4; ++k) v[k] += x[k];
    }
    uint16_t* o = a.out + (int64_t)(tm * BN + j) * a.ldo + n;
    if (a.bias) {
#pragma unroll
      for (int k = 0; k < 4; ++k)
        if (n + k < a.N) v[k] += BF16::load(a.bias + n + k);
    }
    if (a.vec && n + 4 <= a.N) {
      *reinterpret_cast<uint2*>(o) = make_uint2(bf_pack(v[0], v[1]), bf_pack(v[2], v[3]));
    } else {
#pragma unroll
      for (int k = 0; k < 4; ++k)
        if (n + k < a.N) BF16::store(o + k, v[k]);
    }
  }
  if (warp == 1) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(C::TMEM));
  }
  if (a.splits > 1) cluster_sync();  // the peers have read this CTA's sums
}

// ---------------------------------------------------------------------------
template <int BN>
int launch_wide(const void* x, const void* w, int64_t K, Args a, cudaStream_t st) {
  using C = Wide<BN>;
  static_assert((2 * C::STAGES + 2 * C::BUFS + 2) * 8 <= 256, "barrier area");
  CUtensorMap ma, mw;
  if (!vq::mx::make_map(&ma, x, a.M, K, 128) || !vq::mx::make_map(&mw, w, a.N, K, BN)) return VQ_ERR_CUDA;
  if (cudaFuncSetAttribute(k_fp8_wide<BN>, cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM) !=
      cudaSuccess)
    return VQ_ERR_CUDA;
  a.mt = (a.M + 127) / 128;
  a.nt = (a.N + BN - 1) / BN;
  a.tiles = a.mt * a.nt;
  k_fp8_wide<BN><<<std::min(a.tiles, vq::mx::sm_count()), C::THREADS, C::SMEM, st>>>(ma, mw, a);
  return cudaGetLastError() == cudaSuccess ? VQ_OK : VQ_ERR_CUDA;
}

template <int BN>
int launch_few(const void* x, const void* w, int64_t K, Args a, cudaStream_t st) {
  using C = Few<BN>;
  static_assert((2 * C::STAGES + 2 * C::BUFS + 2) * 8 <= 256, "barrier area");
  CUtensorMap mx_, mw;
  if (!vq::mx::make_map(&mx_, x, a.M, K, BN) || !vq::mx::make_map(&mw, w, a.N, K, 128)) return VQ_ERR_CUDA;
  if (cudaFuncSetAttribute(k_fp8_few<BN>, cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM) !=
      cudaSuccess)
    return VQ_ERR_CUDA;
  a.mt = (a.M + BN - 1) / BN;
  a.nt = (a.N + 127) / 128;
  a.tiles = a.mt * a.nt;
  // K split so that the waves of two CTAs per SM take least: blocks per CTA,
  // plus a constant 6 for a CTA's start and the join
  const int slots = 2 * vq::mx::sm_count();
  int best = 1;
  int64_t cost = 1ll << 60;
  for (int s = 1; s <= 8 && s <= a.nk; ++s) {
    const int64_t c = ((int64_t)a.tiles * s + slots - 1) / slots * ((a.nk + s - 1) / s + 6);
    if (c < cost) cost = c, best = s;
  }
  a.splits = best;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(a.tiles * best));
  cfg.blockDim = dim3(C::THREADS);
  cfg.dynamicSmemBytes = C::SMEM;
  cfg.stream = st;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = best, at[0].val.clusterDim.y = 1, at[0].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, k_fp8_few<BN>, mx_, mw, a) == cudaSuccess ? VQ_OK : VQ_ERR_CUDA;
}

int sticky_f8(int* out, int clear, cudaStream_t st) { return vq::tc::sticky_read(out, clear, st); }

}  // namespace f8
}  // namespace vq

using namespace vq::f8;

extern "C" int vq_linear_fp8_block(const void* x, const float* x_scale, const void* w,
                                   const float* w_scale, const void* bias, int64_t M, int64_t N,
                                   int64_t K, void* out, int64_t ldo, void* stream) {
  if (M < 0 || N <= 0 || K <= 0 || M >= (1ll << 30) || N >= (1ll << 30) || K >= (1ll << 30))
    return VQ_ERR_INVALID;
  if (K % 16) return VQ_ERR_UNSUPPORTED;  // TMA rows
  if (ldo < N) return VQ_ERR_SHAPE;
  if (M == 0) return VQ_OK;
  if (!x || !x_scale || !w || !w_scale || !out) return VQ_ERR_NULL;
  if ((reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(w)) & 15) return VQ_ERR_ALIGNMENT;
  if ((reinterpret_cast<uintptr_t>(x_scale) | reinterpret_cast<uintptr_t>(w_scale)) & 3)
    return VQ_ERR_ALIGNMENT;
  if ((reinterpret_cast<uintptr_t>(bias) | reinterpret_cast<uintptr_t>(out)) & 1) return VQ_ERR_ALIGNMENT;
  if ((M + 15) / 16 * ((N + 127) / 128) >= (1ll << 27)) return VQ_ERR_INVALID;
  Args a = {};
  a.sa = x_scale, a.sw = w_scale;
  a.bias = (const uint16_t*)bias;
  a.out = (uint16_t*)out;
  a.ldo = ldo;
  a.M = (int)M, a.N = (int)N, a.nk = (int)((K + 127) / 128);
  a.vec = ldo % 8 == 0 && !(reinterpret_cast<uintptr_t>(out) & 15) && !(reinterpret_cast<uintptr_t>(bias) & 15);
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  if (M <= 16) return launch_few<16>(x, w, K, a, st);
  if (M <= 32) return launch_few<32>(x, w, K, a, st);
  if (M <= 64) return launch_few<64>(x, w, K, a, st);
  if (M <= 128) return launch_few<128>(x, w, K, a, st);
  const int64_t big = ((M + 127) / 128) * ((N + 255) / 256);
  return big >= vq::mx::sm_count() ? launch_wide<256>(x, w, K, a, st) : launch_wide<128>(x, w, K, a, st);
}
