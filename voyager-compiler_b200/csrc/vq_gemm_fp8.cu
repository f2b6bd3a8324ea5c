// E4M3 x E4M3 linear with float32 scales per block of 128 on the
// 5th-generation tensor cores (tcgen05.mma.kind::f8f6f4):
//
//   out[m, n] = bf16( bias[n] + sum_kb sa[m, kb] * sw[n / 128, kb]
//                     * sum_{k in block kb} a[m, k] * w[n, k] )
//
// The scales are float32 values of any mantissa, so they cannot ride in the MMA
// (their product sa * sw is formed first, in float32: below 2^-126 it loses
// bits, beyond the range it is an infinity): each 128-column block of K is one tensor-core product (exact products, float32
// sums) into its own TMEM buffer, and the promotion warps read it back
// (tcgen05.ld) and add it, times its scale, to float32 sums in registers.
// The MMAs of the next blocks run meanwhile: one multiply-add per output and
// block on the CUDA cores against 128 on the tensor cores.
//
// k_fp8_pair  many tokens: tiles of 256 tokens (TMEM lanes) x 256 weight rows
//             (columns) on CTA pairs, persistent; k_fp8_one the same with
//             128 x 128 tiles on single CTAs.  A thread's scale is one scalar
//             per block.
// k_fp8_few   few tokens: tiles of 128 weight rows (lanes) x BN tokens, so
//             that no lane is idle when the weight is all there is to read;
//             K is split over a cluster of CTAs, whose float32 sums are added
//             in rank order through distributed shared memory.
//
// A kernel lets the next one start (programmatic dependent launch) only when
// all its CTAs hold their TMEM: the next one's CTAs could otherwise take it
// first and wait for a kernel that waits for them.
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
#include "vq_pdl.cuh"
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
  int splits;          // CTAs of a cluster that share a tile's K (k_fp8_few, k_fp8_one)
  int vec, vec4;       // out rows take 4-byte, 8-byte stores
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
// The loads so far have landed; r is named so that no use of it moves above.
__device__ __forceinline__ void tmem_wait(uint32_t (&r)[16]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]),
                 "+r"(r[7]), "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]),
                 "+r"(r[13]), "+r"(r[14]), "+r"(r[15])
               :
               : "memory");
}
__device__ __forceinline__ void tmem_wait(uint32_t (&r)[32]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]),
                 "+r"(r[7]), "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]),
                 "+r"(r[13]), "+r"(r[14]), "+r"(r[15]), "+r"(r[16]), "+r"(r[17]), "+r"(r[18]),
                 "+r"(r[19]), "+r"(r[20]), "+r"(r[21]), "+r"(r[22]), "+r"(r[23]), "+r"(r[24]),
                 "+r"(r[25]), "+r"(r[26]), "+r"(r[27]), "+r"(r[28]), "+r"(r[29])
               :
               : "memory");
  asm volatile("" : "+r"(r[30]), "+r"(r[31]));
}

// acc += r * s for two neighbouring columns in one instruction (each lane's
// product and sum rounded as fmaf rounds them).
__device__ __forceinline__ void fma2(uint64_t& acc, uint32_t r0, uint32_t r1, uint64_t s) {
  asm("{\n\t.reg .b64 t;\n\tmov.b64 t, {%1, %2};\n\tfma.rn.f32x2 %0, t, %3, %0;\n\t}"
      : "+l"(acc) : "r"(r0), "r"(r1), "l"(s));
}
__device__ __forceinline__ uint64_t pair(float lo, float hi) {
  uint64_t v;
  asm("mov.b64 %0, {%1, %2};" : "=l"(v) : "f"(lo), "f"(hi));
  return v;
}
__device__ __forceinline__ float2 unpair(uint64_t v) {
  float2 f;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(f.x), "=f"(f.y) : "l"(v));
  return f;
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
// Promotion, shared by the two kernels for many tokens: one warp takes 32
// token rows (a TMEM lane quarter) x COLS columns of each tile.
constexpr int OUT_BYTES = 33 * 32 * 4;  // its staging: 32 rows x 64 columns of bf16, padded by a word

// Adds the tile's nk blocks: the TMEM loads run one 32-column chunk ahead of
// the multiply-adds, across the blocks too, so that the wait for a block's
// MMAs hides behind the last chunk of the block before.  full(buf) waits for
// a buffer (false: gave up), done(buf) gives it back; buffers are `bstep`
// TMEM columns apart.
template <int COLS, int BUFS, typename Full, typename Done>
__device__ __forceinline__ bool promote(uint64_t (&acc)[COLS / 2], const float* sa, const float* sw, int nk,
                                        uint32_t tbase, uint32_t bstep, int& buf, uint32_t& phase, Full full,
                                        Done done) {
  constexpr int CH = COLS / 32;
  static_assert(CH % 2 == 0, "the chunk buffers alternate");
  uint32_t r[2][32];
  bool ok = full(buf, phase);
  if (!ok) return false;
  float s = __ldg(sa) * __ldg(sw);
  tc_fence_after();
  tmem_ld32(tbase + buf * bstep, r[0]);
  for (int kt = 0; kt < nk; ++kt) {
    const int kn = min(kt + 1, nk - 1);
    const float na = __ldg(sa + kn), nw = __ldg(sw + kn);
    const uint64_t s2 = pair(s, s);
#pragma unroll
    for (int c = 0; c < CH; ++c) {
      tmem_wait(r[c & 1]);
      if (c + 1 < CH) {
        tmem_ld32(tbase + buf * bstep + (c + 1) * 32, r[(c + 1) & 1]);
      } else {
        tc_fence_before();
        done(buf);
        if (++buf == BUFS) buf = 0, phase ^= 1;
        if (kt + 1 < nk) {
          if (ok) ok = full(buf, phase);
          tc_fence_after();
          tmem_ld32(tbase + buf * bstep, r[0]);
        }
      }
#pragma unroll
      for (int i = 0; i < 16; ++i) fma2(acc[c * 16 + i], r[c & 1][2 * i], r[c & 1][2 * i + 1], s2);
    }
    s = na * nw;
    if (!ok) {
      tmem_wait(r[0]);
      return false;
    }
  }
  return true;
}

// This warp's columns of the bias into its staging, ahead of the tile.
template <int COLS>
__device__ __forceinline__ void fetch_bias(const Args& a, uint32_t* stage, int col0, int lane) {
  if (!a.bias) return;
  float* sb = reinterpret_cast<float*>(stage);
  __syncwarp();
#pragma unroll
  for (int c = 0; c < COLS; c += 32)
    sb[c + lane] = col0 + c + lane < a.N ? BF16::load(a.bias + col0 + c + lane) : 0.0f;
}

// Sums (+ bias) to bf16 rows through the staging, so that a warp's stores run
// along the rows.
template <int COLS>
__device__ __forceinline__ void store_rows(const Args& a, uint64_t (&acc)[COLS / 2], uint32_t* stage, int r0,
                                           int col0, int lane) {
  if (a.bias) {
    __syncwarp();
    const float4* sb = reinterpret_cast<const float4*>(stage);
#pragma unroll
    for (int c = 0; c < COLS / 4; ++c) {
      const float4 v = sb[c];
      const float2 x = unpair(acc[2 * c]), y = unpair(acc[2 * c + 1]);
      acc[2 * c] = pair(x.x + v.x, x.y + v.y);
      acc[2 * c + 1] = pair(y.x + v.z, y.y + v.w);
    }
  }
  const int rows = min(32, a.M - r0);
#pragma unroll
  for (int c = 0; c < COLS; c += 64) {
    __syncwarp();
#pragma unroll
    for (int j = 0; j < 32; ++j) {
      const float2 v = unpair(acc[c / 2 + j]);
      stage[lane * 33 + j] = bf_pack(v.x, v.y);
    }
    __syncwarp();
    const int col = col0 + c + 2 * lane;
    uint16_t* o = a.out + (int64_t)r0 * a.ldo + col;
    if (a.vec && col + 2 <= a.N) {
#pragma unroll 8
      for (int i = 0; i < rows; ++i) *reinterpret_cast<uint32_t*>(o + (int64_t)i * a.ldo) = stage[i * 33 + lane];
    } else {
#pragma unroll 4
      for (int i = 0; i < rows; ++i) {
        const uint32_t w = stage[i * 33 + lane];
        if (col < a.N) o[(int64_t)i * a.ldo] = (uint16_t)w;
        if (col + 1 < a.N) o[(int64_t)i * a.ldo + 1] = (uint16_t)(w >> 16);
      }
    }
  }
}

// Tile -> (token tile, weight tile): token tiles fastest within groups of 8,
// so that the CTAs of a wave share few rows of both operands.
__device__ __forceinline__ void tile_of(const Args& a, int t, int& tm, int& tn) {
  const int per = 8 * a.nt, gr = t / per, in = t - gr * per;
  const int rows = min(8, a.mt - gr * 8);
  tn = in / rows;
  tm = gr * 8 + in - tn * rows;
}

// The scales of a row and of a 128-row weight block, clamped to what exists.
__device__ __forceinline__ const float* sa_of(const Args& a, int row) {
  return a.sa + (int64_t)min(row, a.M - 1) * a.nk;
}
__device__ __forceinline__ const float* sw_of(const Args& a, int block) {
  return a.sw + (int64_t)min(block, (a.N - 1) / 128) * a.nk;
}

// One lane of a converged warp.  The warp that issues the MMAs runs its loop
// whole, with the instructions under this predicate: the operands then stay
// in uniform registers (a loop run by lane 0 alone took twice the time per
// MMA, moving them there: 535 against 230 cycles per block of 4 MMAs and
// their commits).
__device__ __forceinline__ bool elect_one() {
  uint32_t p;
  asm volatile("{\n\t.reg .pred P;\n\telect.sync _|P, 0xFFFFFFFF;\n\tselp.u32 %0, 1, 0, P;\n\t}" : "=r"(p));
  return p != 0;
}

// Four neighbouring float32 sums at `p` (this CTA's shared address) of the
// cluster's CTAs, added in rank order; all loads in flight together.
__device__ __forceinline__ void cluster_sum4(uint32_t p, int splits, float (&v)[4]) {
  float x[8][4];
#pragma unroll
  for (int r = 0; r < 8; ++r)
    if (r < splits) {
      const uint32_t src = splits > 1 ? mapa_shared(p, r) : p;
      asm volatile("ld.shared::cluster.v4.f32 {%0,%1,%2,%3}, [%4];"
                   : "=f"(x[r][0]), "=f"(x[r][1]), "=f"(x[r][2]), "=f"(x[r][3]) : "r"(src) : "memory");
    }
  v[0] = v[1] = v[2] = v[3] = 0.0f;
#pragma unroll
  for (int r = 0; r < 8; ++r)
    if (r < splits) {
#pragma unroll
      for (int k = 0; k < 4; ++k) v[k] += x[r][k];
    }
}
// Four neighbouring outputs (+ bias) of a row, from column n on.
__device__ __forceinline__ void store4(const Args& a, int row, int n, float (&v)[4]) {
  uint16_t* o = a.out + (int64_t)row * a.ldo + n;
  if (a.bias) {
#pragma unroll
    for (int k = 0; k < 4; ++k)
      if (n + k < a.N) v[k] += BF16::load(a.bias + n + k);
  }
  if (a.vec4 && n + 4 <= a.N) {
    *reinterpret_cast<uint2*>(o) = make_uint2(bf_pack(v[0], v[1]), bf_pack(v[2], v[3]));
  } else {
#pragma unroll
    for (int k = 0; k < 4; ++k)
      if (n + k < a.N) BF16::store(o + k, v[k]);
  }
}

// ---------------------------------------------------------------------------
// 128 x 128 tiles: four TMEM buffers of 128 columns.  Persistent, one CTA per
// tile; where there are tiles for half of the SMs or less, a cluster of
// a.splits CTAs per tile, each with a part of K, whose float32 sums meet in
// shared memory (the grid then has every tile's CTAs).  Bound by the hand-over
// of the buffers, about 0.4 us a block of K, and by start and end: 333 tokens,
// 5003 x 2000, 120 tiles of 16 blocks: 11.1 us.
struct One {
  static constexpr int STAGES = 6, STAGE = 2 * 128 * BK, BUFS = 4, THREADS = 384, COLS = 64;
  static constexpr int LD = 132;  // floats per row of the sums in shared memory
  static_assert(128 * LD * 4 <= STAGES * STAGE, "the sums fit the ring");
  static constexpr int SMEM = STAGES * STAGE + 8 * OUT_BYTES + 1024 + 256;
};

__global__ void __launch_bounds__(One::THREADS, 1)
    k_fp8_one(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_w,
              const __grid_constant__ Args a) {
  using C = One;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                             ~(uintptr_t)1023);
  uint32_t* out_stage = reinterpret_cast<uint32_t*>(smem + C::STAGES * C::STAGE);
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + C::STAGES * C::STAGE + 8 * OUT_BYTES);
  const uint32_t full0 = smem_u32(bars), empty0 = full0 + 8 * C::STAGES;
  const uint32_t acc_full0 = empty0 + 8 * C::STAGES, acc_empty0 = acc_full0 + 8 * C::BUFS;
  const uint32_t drain = acc_empty0 + 8 * C::BUFS;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 2 * C::STAGES + 2 * C::BUFS + 1);
  const int warp = __shfl_sync(FULL, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  const int rank = a.splits > 1 ? (int)cluster_ctarank() : 0;
  const int first = blockIdx.x / a.splits, step = gridDim.x / a.splits;
  const int kb0 = (int)((int64_t)a.nk * rank / a.splits), kb1 = (int)((int64_t)a.nk * (rank + 1) / a.splits);
  auto load = [&](int tm, int tn, int kt, int stage) {
    const uint32_t dst = smem_u32(smem) + stage * C::STAGE;
    mbar_expect_tx(full0 + 8 * stage, C::STAGE);
    tma_load_2d(dst, &map_a, kt * BK, tm * 128, full0 + 8 * stage);
    tma_load_2d(dst + 128 * BK, &map_w, kt * BK, tn * 128, full0 + 8 * stage);
  };
  const int pre = min(C::STAGES, kb1 - kb0);  // loads that need no one's leave
  if (threadIdx.x == 0) {
    for (int s = 0; s < C::STAGES; ++s) mbar_init(full0 + 8 * s, 1), mbar_init(empty0 + 8 * s, 1);
    for (int s = 0; s < C::BUFS; ++s) mbar_init(acc_full0 + 8 * s, 1), mbar_init(acc_empty0 + 8 * s, 8);
    mbar_init(drain, 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    prefetch_map(&map_a);
    prefetch_map(&map_w);
    pdl::wait();
    int tm, tn;
    tile_of(a, first, tm, tn);
    for (int i = 0; i < pre; ++i) load(tm, tn, kb0 + i, i);
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
  pdl::trigger();  // after the allocation
  pdl::wait();

  if (warp == 0 && lane == 0) {
    int stage = pre == C::STAGES ? 0 : pre;
    uint32_t phase = pre == C::STAGES ? 1 : 0;
    bool ok = true;
    for (int t = first; t < a.tiles && ok; t += step) {
      int tm, tn;
      tile_of(a, t, tm, tn);
      for (int kt = t == first ? kb0 + pre : kb0; kt < kb1; ++kt) {
        if (!mbar_wait(empty0 + 8 * stage, phase ^ 1, nullptr, ERR_EMPTY)) {
          ok = false;
          break;
        }
        load(tm, tn, kt, stage);
        if (++stage == C::STAGES) stage = 0, phase ^= 1;
      }
    }
    drain_loads<C::STAGES>(full0, stage, phase);
  } else if (warp == 1) {
    const uint64_t da0 = sw128_desc(smem_u32(smem)), dw0 = sw128_desc(smem_u32(smem) + 128 * BK);
    int stage = 0, buf = 0;
    uint32_t phase = 0, bphase = 0;
    bool ok = true;
    for (int t = first; t < a.tiles && ok; t += step) {
      for (int kt = kb0; kt < kb1; ++kt) {
        if (!mbar_wait_warp(acc_empty0 + 8 * buf, bphase ^ 1, nullptr, ERR_ACC) ||
            !mbar_wait_warp(full0 + 8 * stage, phase, nullptr, ERR_FULL)) {
          ok = false;
          break;
        }
        tc_fence_after();
        if (elect_one()) {
          const uint32_t so = stage * (C::STAGE / 16);
          mma_stage(tmem + buf * 128, desc_at(da0, so), desc_at(dw0, so), idesc(128, 128));
          tc_commit(acc_full0 + 8 * buf);
          tc_commit(empty0 + 8 * stage);
        }
        __syncwarp();
        if (++stage == C::STAGES) stage = 0, phase ^= 1;
        if (++buf == C::BUFS) buf = 0, bphase ^= 1;
      }
    }
    if (elect_one()) {
      tc_commit(drain);
      mbar_wait(drain, 0, nullptr, ERR_DRAIN);
    }
    __syncwarp();
  } else if (warp >= 4) {
    // warps 4..11: two per TMEM lane quarter, 64 columns each
    const int q = warp & 3, half = (warp - 4) >> 2;
    uint32_t* stage_out = out_stage + (warp - 4) * (OUT_BYTES / 4);
    int buf = 0;
    uint32_t bphase = 0;
    for (int t = first; t < a.tiles; t += step) {
      int tm, tn;
      tile_of(a, t, tm, tn);
      const int r0 = tm * 128 + q * 32, col0 = tn * 128 + half * C::COLS;
      fetch_bias<C::COLS>(a, stage_out, col0, lane);
      uint64_t acc[C::COLS / 2];
#pragma unroll
      for (int i = 0; i < C::COLS / 2; ++i) acc[i] = 0;
      if (!promote<C::COLS, C::BUFS>(
              acc, sa_of(a, r0 + lane) + kb0, sw_of(a, tn) + kb0, kb1 - kb0,
              tmem + ((uint32_t)(q * 32) << 16) + half * C::COLS, 128, buf, bphase,
              [&](int b, uint32_t ph) { return mbar_wait_warp(acc_full0 + 8 * b, ph, nullptr, ERR_ACC); },
              [&](int b) {
                __syncwarp();
                if (lane == 0) mbar_arrive(acc_empty0 + 8 * b);
              }))
        break;
      if (a.splits == 1) {
        store_rows<C::COLS>(a, acc, stage_out, r0, col0, lane);
      } else {
        // every MMA is done, so the ring is free: [128 rows][128 sums]
        float* red = reinterpret_cast<float*>(smem) + (q * 32 + lane) * C::LD + half * C::COLS;
#pragma unroll
        for (int i = 0; i < C::COLS / 4; ++i) {
          const float2 x = unpair(acc[2 * i]), y = unpair(acc[2 * i + 1]);
          reinterpret_cast<float4*>(red)[i] = make_float4(x.x, x.y, y.x, y.y);
        }
      }
    }
  }
  __syncthreads();
  if (a.splits > 1) {
    cluster_sync();
    int tm, tn;
    tile_of(a, first, tm, tn);
    // rows rank, rank + splits, ..; a warp takes a row
    for (int r = rank + warp * a.splits; r < min(128, a.M - tm * 128); r += C::THREADS / 32 * a.splits) {
      float v[4];
      cluster_sum4(smem_u32(smem) + (r * C::LD + lane * 4) * 4, a.splits, v);
      store4(a, tm * 128 + r, tn * 128 + lane * 4, v);
    }
  }
  if (warp == 1) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512));
  }
  if (a.splits > 1) cluster_sync();  // the peers have read this CTA's sums
}

// ---------------------------------------------------------------------------
// 256 x 256 tiles on CTA pairs (cta_group::2): each CTA holds 128 token rows
// in its TMEM and loads those and half of the weight rows, 32 KB per block
// instead of the 48 KB that a CTA of its own needs for 128 x 256.  The even
// CTA issues the MMAs.  4096 tokens, 22016 x 4096: 362 us, 2.04 PFLOP/s (429
// where the power cap sets the clock); the tensor pipe is 51 % active, the
// promotion's readback and multiply-adds of 256 columns a block set the pace.
struct Pair {
  static constexpr int BN = 256, COLS = BN / 2, A_BYTES = 128 * BK, STAGE = A_BYTES + BN / 2 * BK, STAGES = 6;
  // 3 warpgroups per CTA: TMA and MMA issue, then two of promotion.  The
  // launch gives every thread 168 registers; setmaxnreg moves them to the
  // promotion (128 * 40 + 256 * 232 = 384 * 168), which needs about 215.
  static constexpr int THREADS = 384, ISSUE_REGS = 40, PROMOTE_REGS = 232;
  static constexpr int SMEM = STAGES * STAGE + 8 * OUT_BYTES + 1024 + 256;
  static_assert(SMEM <= 227 * 1024 && STAGE % 1024 == 0, "shared memory");
};

__device__ __forceinline__ void mma_f8_pair(uint32_t d, uint64_t da, uint64_t db, uint32_t id, uint32_t acc) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::2.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
      "l"(da), "l"(db), "r"(id), "r"(acc));
}

__global__ void __launch_bounds__(Pair::THREADS, 1)
    k_fp8_pair(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_w,
               const __grid_constant__ Args a) {
  using C = Pair;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                             ~(uintptr_t)1023);
  uint32_t* out_stage = reinterpret_cast<uint32_t*>(smem + C::STAGES * C::STAGE);
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + C::STAGES * C::STAGE + 8 * OUT_BYTES);
  const uint32_t full0 = smem_u32(bars), empty0 = full0 + 8 * C::STAGES;
  const uint32_t acc_full0 = empty0 + 8 * C::STAGES, acc_empty0 = acc_full0 + 8 * 2;
  const uint32_t drain = acc_empty0 + 8 * 2;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 2 * C::STAGES + 5);
  const uint32_t rank = cluster_ctarank();  // 0: issues the pair's MMAs
  const int warp = __shfl_sync(FULL, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  const int pair_id = blockIdx.x >> 1, npairs = gridDim.x >> 1;
  if (threadIdx.x == 0) {
    for (int s = 0; s < C::STAGES; ++s) mbar_init(full0 + 8 * s, 1), mbar_init(empty0 + 8 * s, 1);
    for (int s = 0; s < 2; ++s) mbar_init(acc_full0 + 8 * s, 1), mbar_init(acc_empty0 + 8 * s, 16);
    mbar_init(drain, 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(
                     smem_u32(tmem_slot)), "r"(512));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;");
  }
  tc_fence_before();
  cluster_sync();  // both CTAs' barriers exist before any use across them
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  pdl::trigger();  // after the allocation
  pdl::wait();

  if (warp < 4) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(C::ISSUE_REGS));
    if (warp == 0 && lane == 0) {
      int stage = 0;
      uint32_t phase = 0;
      bool ok = true;
      const uint32_t fb0 = mapa_shared(full0, 0);  // both CTAs' loads count on the even CTA
      for (int t = pair_id; t < a.tiles && ok; t += npairs) {
        int tm, tn;
        tile_of(a, t, tm, tn);
        const int ya = tm * 256 + (int)rank * 128, yw = tn * C::BN + (int)rank * (C::BN / 2);
        for (int kt = 0; kt < a.nk; ++kt) {
          if (!mbar_wait(empty0 + 8 * stage, phase ^ 1, nullptr, ERR_EMPTY)) {
            ok = false;
            break;
          }
          const uint32_t dst = smem_u32(smem) + stage * C::STAGE, fb = fb0 + 8 * stage;
          if (rank == 0) mbar_expect_tx(full0 + 8 * stage, 2 * C::STAGE);
          tma_load_2d_pair(dst, &map_a, kt * BK, ya, fb);
          tma_load_2d_pair(dst + C::A_BYTES, &map_w, kt * BK, yw, fb);
          if (++stage == C::STAGES) stage = 0, phase ^= 1;
        }
      }
      if (rank == 0) drain_loads<C::STAGES>(full0, stage, phase);
    } else if (warp == 1 && rank == 0) {
      int stage = 0, buf = 0;
      uint32_t phase = 0, bphase = 0;
      bool ok = true;
      const uint32_t s0 = smem_u32(smem);
      const uint64_t da0 = sw128_desc(s0), dw0 = sw128_desc(s0 + C::A_BYTES);
      for (int t = pair_id; t < a.tiles && ok; t += npairs) {
        for (int kt = 0; kt < a.nk; ++kt) {
          if (!mbar_wait_warp(acc_empty0 + 8 * buf, bphase ^ 1, nullptr, ERR_ACC) ||
              !mbar_wait_warp(full0 + 8 * stage, phase, nullptr, ERR_FULL)) {
            ok = false;
            break;
          }
          tc_fence_after();
          if (elect_one()) {
            const uint32_t so = stage * (C::STAGE / 16);
#pragma unroll
            for (uint32_t j = 0; j < 4; ++j)
              mma_f8_pair(tmem + buf * C::BN, desc_at(da0, so + 2 * j), desc_at(dw0, so + 2 * j),
                          idesc(256, C::BN), j > 0);
            tc_commit_pair(acc_full0 + 8 * buf, 0x3);
            tc_commit_pair(empty0 + 8 * stage, 0x3);
          }
          __syncwarp();
          if (++stage == C::STAGES) stage = 0, phase ^= 1;
          if (++buf == 2) buf = 0, bphase ^= 1;
        }
      }
      if (elect_one()) {
        tc_commit_pair(drain, 0x1);
        mbar_wait(drain, 0, nullptr, ERR_DRAIN);
      }
      __syncwarp();
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(C::PROMOTE_REGS));
    const int q = warp & 3, half = (warp - 4) >> 2;
    uint32_t* stage_out = out_stage + (warp - 4) * (OUT_BYTES / 4);
    const uint32_t give0 = mapa_shared(acc_empty0, 0);
    int buf = 0;
    uint32_t bphase = 0;
    for (int t = pair_id; t < a.tiles; t += npairs) {
      int tm, tn;
      tile_of(a, t, tm, tn);
      const int r0 = tm * 256 + (int)rank * 128 + q * 32, col0 = tn * C::BN + half * C::COLS;
      fetch_bias<C::COLS>(a, stage_out, col0, lane);
      uint64_t acc[C::COLS / 2];
#pragma unroll
      for (int i = 0; i < C::COLS / 2; ++i) acc[i] = 0;
      if (!promote<C::COLS, 2>(
              acc, sa_of(a, r0 + lane), sw_of(a, col0 / 128), a.nk, tmem + ((uint32_t)(q * 32) << 16) + half * C::COLS, C::BN, buf, bphase,
              [&](int b, uint32_t ph) { return mbar_wait_warp(acc_full0 + 8 * b, ph, nullptr, ERR_ACC); },
              [&](int b) {
                __syncwarp();
                if (lane == 0) mbar_arrive_cluster(give0 + 8 * b);
              }))
        break;
      store_rows<C::COLS>(a, acc, stage_out, r0, col0, lane);
    }
  }
  __syncwarp();
  tc_fence_before();
  cluster_sync();  // both CTAs are done with the pair's TMEM and barriers
  if (warp == 1) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512));
  }
}

// ---------------------------------------------------------------------------
// Bound by HBM, one token 12288 x 4096: 11.9 us, 4.2 TB/s, of which start, first
// loads and the end take 4.  PER_SM: CTAs on an SM.  One with a deep ring and
// registers for a whole buffer's readback while the tiles are no more than the
// SMs (64 tokens, 12288 x 4096: 16.5 us, with two 23.2; one CTA a SM also
// spreads the clusters), two where they are more (one token, 22016 x 4096, 172
// tiles: 19.1 us, with one 26.6).
template <int BN, int PER_SM>
struct Few {
  static constexpr int W_BYTES = 128 * BK, X_BYTES = BN * BK, STAGE = W_BYTES + X_BYTES;
  static constexpr int STAGES = PER_SM == 1 ? (BN == 16 ? 10 : BN == 32 ? 9 : 7) : BN == 16 ? 6 : BN == 32 ? 5 : 4;
  static constexpr int BUFS = 4;
  static constexpr int TMEM = BUFS * BN < 32 ? 32 : BUFS * BN;
  static constexpr int THREADS = 192;
  static constexpr int KC = 32;  // K blocks per refill of the scales
  static constexpr int LS = BN + 4;  // floats per block of them in shared memory
  static constexpr int LD = 132; // floats per token of the sums in shared memory
  static constexpr int RING = STAGES * STAGE > BN * LD * 4 ? STAGES * STAGE : BN * LD * 4;
  static constexpr int SMEM = RING + KC * LS * 4 + 1024 + 256;
  static_assert(PER_SM * (SMEM + 1024) <= 228 * 1024, "CTAs per SM");
};

template <int BN, int PER_SM>
__global__ void __launch_bounds__(Few<BN, PER_SM>::THREADS, PER_SM)
    k_fp8_few(const __grid_constant__ CUtensorMap map_x, const __grid_constant__ CUtensorMap map_w,
              const __grid_constant__ Args a) {
  using C = Few<BN, PER_SM>;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                             ~(uintptr_t)1023);
  float* s_scale = reinterpret_cast<float*>(smem + C::RING);  // [KC][LS]
  uint64_t* bars = reinterpret_cast<uint64_t*>(s_scale + C::KC * C::LS);
  const uint32_t full0 = smem_u32(bars), empty0 = full0 + 8 * C::STAGES;
  const uint32_t acc_full0 = empty0 + 8 * C::STAGES, acc_empty0 = acc_full0 + 8 * C::BUFS;
  const uint32_t drain = acc_empty0 + 8 * C::BUFS;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 2 * C::STAGES + 2 * C::BUFS + 1);
  const int warp = __shfl_sync(FULL, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  const int rank = a.splits > 1 ? (int)cluster_ctarank() : 0;
  const int tile = blockIdx.x / a.splits, tm = tile / a.nt, tn = tile - tm * a.nt;
  const int kb0 = (int)((int64_t)a.nk * rank / a.splits);
  const int kb1 = (int)((int64_t)a.nk * (rank + 1) / a.splits);
  auto load = [&](int kt, int stage) {
    const uint32_t dst = smem_u32(smem) + stage * C::STAGE;
    mbar_expect_tx(full0 + 8 * stage, C::STAGE);
    tma_load_2d(dst, &map_w, kt * BK, tn * 128, full0 + 8 * stage);
    tma_load_2d(dst + C::W_BYTES, &map_x, kt * BK, tm * BN, full0 + 8 * stage);
  };
  if (threadIdx.x == 0) {
    for (int s = 0; s < C::STAGES; ++s) mbar_init(full0 + 8 * s, 1), mbar_init(empty0 + 8 * s, 1);
    for (int s = 0; s < C::BUFS; ++s) mbar_init(acc_full0 + 8 * s, 1), mbar_init(acc_empty0 + 8 * s, 4);
    mbar_init(drain, 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    prefetch_map(&map_x);
    prefetch_map(&map_w);
    pdl::wait();
    // the ring's first round needs no one's leave
    for (int i = 0; i < min(C::STAGES, kb1 - kb0); ++i) load(kb0 + i, i);
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
  pdl::trigger();  // after the allocation
  pdl::wait();

  if (warp == 0) {
    if (lane == 0) {
      const int first = min(C::STAGES, kb1 - kb0);
      int stage = first == C::STAGES ? 0 : first;
      uint32_t phase = first == C::STAGES ? 1 : 0;
      for (int kt = kb0 + first; kt < kb1; ++kt) {
        if (!mbar_wait(empty0 + 8 * stage, phase ^ 1, nullptr, ERR_EMPTY)) break;
        load(kt, stage);
        if (++stage == C::STAGES) stage = 0, phase ^= 1;
      }
      drain_loads<C::STAGES>(full0, stage, phase);
    }
  } else if (warp == 1) {
    int stage = 0, buf = 0;
    uint32_t phase = 0, bphase = 0;
    const uint64_t dw0 = sw128_desc(smem_u32(smem)), dx0 = sw128_desc(smem_u32(smem) + C::W_BYTES);
    for (int kt = kb0; kt < kb1; ++kt) {
      if (!mbar_wait_warp(acc_empty0 + 8 * buf, bphase ^ 1, nullptr, ERR_ACC) ||
          !mbar_wait_warp(full0 + 8 * stage, phase, nullptr, ERR_FULL))
        break;
      tc_fence_after();
      if (elect_one()) {
        const uint32_t so = stage * (C::STAGE / 16);
        mma_stage(tmem + buf * BN, desc_at(dw0, so), desc_at(dx0, so), idesc(128, BN));
        tc_commit(acc_full0 + 8 * buf);
        tc_commit(empty0 + 8 * stage);
      }
      __syncwarp();
      if (++stage == C::STAGES) stage = 0, phase ^= 1;
      if (++buf == C::BUFS) buf = 0, bphase ^= 1;
    }
    if (elect_one()) {
      tc_commit(drain);
      mbar_wait(drain, 0, nullptr, ERR_DRAIN);
    }
    __syncwarp();
  }
  uint64_t acc[BN / 2];  // two tokens each
  const int q = warp & 3;  // TMEM lane quarter of warps 2..5
  if (warp >= 2) {
    int buf = 0;
    uint32_t bphase = 0;
    const int pt = threadIdx.x - 64;
    const float* sw = a.sw + (int64_t)tn * a.nk;
#pragma unroll
    for (int i = 0; i < BN / 2; ++i) acc[i] = 0;
    bool ok = true;
    for (int kc = kb0; kc < kb1; kc += C::KC) {
      // the scales of the next KC blocks, sa * sw per block and token, all
      // loads in flight together (one at a time they cost 10 us at 128 tokens)
      const int n = min(C::KC, kb1 - kc);
      constexpr int PER = C::KC * BN / 128;
      float sv[PER];
#pragma unroll
      for (int u = 0; u < PER; ++u) {
        const int i = pt + u * 128, j = i / C::KC, k = min(i % C::KC, n - 1);
        const int m = min(tm * BN + j, a.M - 1);
        sv[u] = __ldg(a.sa + (int64_t)m * a.nk + kc + k) * __ldg(sw + kc + k);
      }
      asm volatile("bar.sync 1, 128;" ::: "memory");
#pragma unroll
      for (int u = 0; u < PER; ++u) {
        const int i = pt + u * 128;
        s_scale[i % C::KC * C::LS + i / C::KC] = sv[u];
      }
      asm volatile("bar.sync 1, 128;" ::: "memory");
      for (int k = 0; k < n && ok; ++k) {
        if (!mbar_wait_warp(acc_full0 + 8 * buf, bphase, nullptr, ERR_ACC)) {
          ok = false;
          break;
        }
        tc_fence_after();
        const uint32_t taddr = tmem + ((uint32_t)(q * 32) << 16) + buf * BN;
        uint32_t r[BN / 16][16];
#pragma unroll
        for (int c = 0; c < BN / 16; ++c) tmem_ld16(taddr + 16 * c, r[c]);
#pragma unroll
        for (int c = 0; c < BN / 16; ++c) {
          tmem_wait(r[c]);
#pragma unroll
          for (int i = 0; i < 16; i += 4) {
            const ulonglong2 s = *reinterpret_cast<const ulonglong2*>(s_scale + k * C::LS + 16 * c + i);
            fma2(acc[8 * c + i / 2], r[c][i], r[c][i + 1], s.x);
            fma2(acc[8 * c + i / 2 + 1], r[c][i + 2], r[c][i + 3], s.y);
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
    for (int i = 0; i < BN; ++i)
      red[i * C::LD + q * 32 + lane] = i % 2 ? unpair(acc[i / 2]).y : unpair(acc[i / 2]).x;
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
    float v[4];
    cluster_sum4(red_addr + (j * C::LD + f) * 4, a.splits, v);
    store4(a, tm * BN + j, n, v);
  }
  if (warp == 1) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(C::TMEM));
  }
  if (a.splits > 1) cluster_sync();  // the peers have read this CTA's sums
}

// ---------------------------------------------------------------------------
// Clusters of s CTAs of kernel F that the device holds at once (asked once per
// device and size; one CTA an SM): clusters of 3, for one, reach 135 SMs.
template <auto F>
int resident_clusters(int s, int threads, int smem) {
  static int known[64][9] = {};
  int dev = 0;
  cudaGetDevice(&dev);
  dev = dev < 0 || dev > 63 ? 0 : dev;
  if (known[dev][s] == 0) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(s);
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = s, at[0].val.clusterDim.y = 1, at[0].val.clusterDim.z = 1;
    cfg.attrs = at;
    cfg.numAttrs = 1;
    int n = 0;
    if (cudaOccupancyMaxActiveClusters(&n, F, &cfg) != cudaSuccess || n <= 0) {
      (void)cudaGetLastError();
      n = 1;
    }
    known[dev][s] = n;
  }
  return known[dev][s];
}

// K split so that the waves of resident clusters take least: blocks per CTA,
// plus 6 for a CTA's start and, split, the join.
template <auto F>
int best_split(int tiles, int nk, int threads, int smem) {
  int best = 1;
  int64_t cost = 1ll << 60;
  for (int s = 1; s <= 8 && s <= nk; ++s) {
    const int64_t res = resident_clusters<F>(s, threads, smem);
    const int64_t c = (tiles + res - 1) / res * ((nk + s - 1) / s + 6);
    if (c < cost) cost = c, best = s;
  }
  return best;
}

int launch_many(const void* x, const void* w, int64_t K, Args a, cudaStream_t st) {
  static_assert((2 * One::STAGES + 2 * One::BUFS + 2) * 8 <= 256 && (2 * Pair::STAGES + 6) * 8 <= 256,
                "barrier areas");
  CUtensorMap ma, mw;
  const int sms = vq::mx::sm_count();
  // pairs once their 256 x 256 tiles fill the SMs; below that, four times as
  // many tiles of 128 x 128
  const int64_t pair_tiles = (int64_t)((a.M + 255) / 256) * ((a.N + Pair::BN - 1) / Pair::BN);
  if (pair_tiles * 2 >= sms) {
    if (!vq::mx::make_map(&ma, x, a.M, K, 128) || !vq::mx::make_map(&mw, w, a.N, K, Pair::BN / 2))
      return VQ_ERR_CUDA;
    if (!allow_smem<k_fp8_pair>(Pair::SMEM)) return VQ_ERR_CUDA;
    a.mt = (a.M + 255) / 256;
    a.nt = (a.N + Pair::BN - 1) / Pair::BN;
    a.tiles = a.mt * a.nt;
    return pdl::launch<k_fp8_pair>(2 * std::min(a.tiles, sms / 2), Pair::THREADS, Pair::SMEM, st, 2, ma, mw, a)
               ? VQ_OK : VQ_ERR_CUDA;
  }
  if (!vq::mx::make_map(&ma, x, a.M, K, 128) || !vq::mx::make_map(&mw, w, a.N, K, 128)) return VQ_ERR_CUDA;
  if (!allow_smem<k_fp8_one>(One::SMEM)) return VQ_ERR_CUDA;
  a.mt = (a.M + 127) / 128;
  a.nt = (a.N + 127) / 128;
  a.tiles = a.mt * a.nt;
  a.splits = 2 * a.tiles <= sms ? best_split<k_fp8_one>(a.tiles, a.nk, One::THREADS, One::SMEM) : 1;
  const int grid = a.splits > 1 ? a.tiles * a.splits : std::min(a.tiles, sms);
  return pdl::launch<k_fp8_one>(grid, One::THREADS, One::SMEM, st, a.splits, ma, mw, a) ? VQ_OK : VQ_ERR_CUDA;
}

template <int BN, int PER_SM>
int launch_few(const void* x, const void* w, int64_t K, Args a, cudaStream_t st) {
  using C = Few<BN, PER_SM>;
  static_assert((2 * C::STAGES + 2 * C::BUFS + 2) * 8 <= 256, "barrier area");
  CUtensorMap mx_, mw;
  if (!vq::mx::make_map(&mx_, x, a.M, K, BN) || !vq::mx::make_map(&mw, w, a.N, K, 128)) return VQ_ERR_CUDA;
  if (!allow_smem<k_fp8_few<BN, PER_SM>>(C::SMEM)) return VQ_ERR_CUDA;
  a.splits = PER_SM == 1 ? best_split<k_fp8_few<BN, PER_SM>>(a.tiles, a.nk, C::THREADS, C::SMEM) : 1;
  return pdl::launch<k_fp8_few<BN, PER_SM>>(a.tiles * a.splits, C::THREADS, C::SMEM, st, a.splits, mx_, mw, a)
             ? VQ_OK : VQ_ERR_CUDA;
}
template <int BN>
int launch_few(const void* x, const void* w, int64_t K, Args a, cudaStream_t st) {
  a.mt = (a.M + BN - 1) / BN;
  a.nt = (a.N + 127) / 128;
  a.tiles = a.mt * a.nt;
  return a.tiles <= vq::mx::sm_count() ? launch_few<BN, 1>(x, w, K, a, st) : launch_few<BN, 2>(x, w, K, a, st);
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
  a.vec = ldo % 2 == 0 && !(reinterpret_cast<uintptr_t>(out) & 3);
  a.vec4 = ldo % 4 == 0 && !(reinterpret_cast<uintptr_t>(out) & 7);
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  if (M <= 16) return launch_few<16>(x, w, K, a, st);
  if (M <= 32) return launch_few<32>(x, w, K, a, st);
  if (M <= 64) return launch_few<64>(x, w, K, a, st);
  return launch_many(x, w, K, a, st);
}
