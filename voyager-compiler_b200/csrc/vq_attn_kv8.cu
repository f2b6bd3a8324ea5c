// Attention of the newest tokens over a paged E4M3 key / value cache.
//
//   o[b, t, h] = sum_j softmax_j(q . k_j * sm_scale) v_j,  j <= held[b] + t,
//   k_j = code * k_scale[page of j, head], v_j likewise
//
// for the T newest tokens (t < counts[b]) of each sequence, whose keys and
// values the cache already holds.  The query heads that share a kv head and
// the T tokens are the rows of one product: row r = t * G + g, in groups of
// 8 * NT rows.
//
// Mathematics: flash decoding.  A warp takes 32-key tiles and computes
// S^T = K Q^T with mma.m16n8k16 in f16: E4M3 converts to f16 exactly, and q is
// scaled per row by a power of two to a largest value of 2^14 .. 2^15, so that
// f16 holds every bf16 down to 2^-31 of it exactly.  With the page's k_scale
// the scores are s (base-2 exponents, float32); m = max s and l = sum 2^(s - m)
// run in float32.  The weights of O^T += V^T P^T take the page's v_scale in:
// P = 2^(15 + s + log2 v_scale - w), w = max(s + log2 v_scale), as f16: relative
// error 2^-11 down to 2^-29 of the largest term, whatever the scales of the
// pages are (with weights relative to m alone, a page of large values and small
// weights lost all its bits).  The output is O 2^(w - 15 - m) / l.  S^T leaves
// the tensor cores with keys along the lanes; movmatrix turns the f16 pairs
// into the operand of the second product.
//
// Work: one CTA of 4 warps per (sequence, kv head, row group, chunk of
// keys); its warps take the chunk's tiles in turn, each with a ring of its
// own that TMA fills (K and V, 32 x D bytes each, SWIZZLE_128B /
// SWIZZLE_64B: the fragment loads then meet no bank conflict for D = 128).
// Chunks of one row group are joined by the CTA that finishes last, in chunk
// order, so the result does not depend on the order of arrival.
//
// Bound by HBM: 2 D bytes per key and kv head.
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <algorithm>

#include "voyager_b200.h"
#include "vq_e4m3.cuh"
#include "vq_tc.cuh"

namespace vq {
namespace kva {

using namespace vq::e4;
using namespace vq::tc;

enum { ERR_WAIT = 311, ERR_PAGE = 312, ERR_CAPACITY = 313, ERR_COUNT = 314 };

constexpr int WARPS = 4, THREADS = WARPS * 32, TILE = 32;
constexpr float NEG_INF = -__builtin_huge_valf();
constexpr float P_EXP = 15.0f;  // the largest weight is 2^15 in f16

struct Args {
  const uint16_t* q;  // bf16, strides in elements
  int64_t qb, qt, qh;
  uint16_t* out;  // bf16 [B, T, H, D]
  const float *k_scale, *v_scale;
  const int32_t *block_table, *lengths, *counts;
  float* part;        // [pairs * groups][chunks][ROWS * (D + 3)]
  int32_t* done;      // [pairs * groups] zero before, zero after
  int B, T, H, Hkv, G, page_log2, width, pages;
  int groups, chunks, chunk;  // row groups per (b, kv head); keys per chunk, a multiple of TILE
  float sm_log2;              // sm_scale * log2(e)
};

template <int D, int NT>
struct Cfg {
  static constexpr int ROWS = 8 * NT;
  static constexpr int TILE_BYTES = TILE * D;
  static constexpr int STAGES = D == 128 ? 3 : 5;
  static constexpr int RING = STAGES * 2 * TILE_BYTES;  // per warp
  static constexpr int SMEM_RING = WARPS * RING;
  static constexpr int PAGES_MAX = 512;                 // pages of one chunk
  static constexpr int MERGE = WARPS * ROWS * (D + 3) * 4;
  static_assert(MERGE <= SMEM_RING, "the join reuses the ring");
  static constexpr int SMEM = SMEM_RING + 1024 + PAGES_MAX * 12 + 256;
};

__device__ __forceinline__ void mma(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                    uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
      "{%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t transpose8x8(uint32_t v) {
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}
__device__ __forceinline__ float ex2(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
__device__ __forceinline__ uint4 lds128(uint32_t a) {
  uint4 v;
  asm volatile("ld.shared.v4.b32 {%0,%1,%2,%3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(a));
  return v;
}
__device__ __forceinline__ uint2 lds64(uint32_t a) {
  uint2 v;
  asm volatile("ld.shared.v2.b32 {%0,%1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(a));
  return v;
}
__device__ __forceinline__ uint32_t f16x2(float lo, float hi) {
  __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<uint32_t*>(&h);
}
// A word has an E4M3 NaN byte (0x7F or 0xFF).
__device__ __forceinline__ uint32_t has_nan(uint32_t w) {
  return __vcmpeq4(w & 0x7F7F7F7Fu, 0x7F7F7F7Fu);
}

// Byte offset of 16-byte chunk c of row r in a TMA-swizzled tile of D-byte rows.
template <int D>
__device__ __forceinline__ uint32_t swz(int r, int c) {
  return D == 128 ? (uint32_t)(r * 128 + ((c ^ (r & 7)) << 4))
                  : (uint32_t)(r * 64 + ((c ^ ((r >> 1) & 3)) << 4));
}

// A running softmax and one output value: m, l, w and O as above.
struct State {
  float m = NEG_INF, l = 0.0f, w = NEG_INF, x = 0.0f;
  __device__ __forceinline__ void add(float m2, float l2, float w2, float x2) {
    const float mn = fmaxf(m, m2), wn = fmaxf(w, w2);
    const float mr = mn == NEG_INF ? 0.0f : mn, wr = wn == NEG_INF ? 0.0f : wn;
    l = l * ex2(m - mr) + l2 * ex2(m2 - mr);
    x = x * ex2(w - wr) + x2 * ex2(w2 - wr);
    m = mn, w = wn;
  }
  __device__ __forceinline__ float value() const {
    return l == 0.0f || w == NEG_INF ? 0.0f * x : __fdiv_rn(x * ex2(w - P_EXP - m), l);
  }
};

template <int D, int NT>
__global__ void __launch_bounds__(THREADS)
    k_attn_kv8(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v,
               const __grid_constant__ Args a) {
  using C = Cfg<D, NT>;
  constexpr int KS = D / 16;   // k steps of the scores, and m tiles of the output
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                             ~(uintptr_t)1023);
  int32_t* s_row = reinterpret_cast<int32_t*>(smem + C::SMEM_RING);      // cache row of each page
  float* s_ks = reinterpret_cast<float*>(s_row + C::PAGES_MAX);
  float* s_lv = s_ks + C::PAGES_MAX;  // log2 of v_scale
  uint64_t* bars = reinterpret_cast<uint64_t*>(s_lv + C::PAGES_MAX);     // [WARPS][STAGES]
  __shared__ int s_last;

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int chunk = blockIdx.x;
  const int grp = blockIdx.y % a.groups, kvh = blockIdx.y / a.groups, b = blockIdx.z;
  const int pair = ((b * a.Hkv) + kvh) * a.groups + grp;

  // the plan of this sequence
  int held = a.lengths[b], cnt = a.counts ? a.counts[b] : a.T;
  if (held < 0 || cnt < 0 || cnt > a.T) {
    note_err(nullptr, ERR_COUNT);
    cnt = held < 0 ? 0 : min(max(cnt, 0), a.T);
    held = max(held, 0);
  }
  const int64_t cap = (int64_t)a.width << a.page_log2;
  if (held + (int64_t)cnt > cap) {
    note_err(nullptr, ERR_CAPACITY);
    cnt = held >= cap ? 0 : (int)(cap - held);
  }
  const int row0 = grp * C::ROWS;
  const int nrows = min(C::ROWS, cnt * a.G - row0);  // rows of this group with a query
  // keys that some row of this group sees
  const int end = nrows > 0 ? held + (row0 + nrows - 1) / a.G + 1 : 0;
  const int nchunks = max(1, (end + a.chunk - 1) / a.chunk);
  if (chunk >= nchunks) return;
  const int k0 = chunk * a.chunk, k1 = min(end, k0 + a.chunk);
  const int ntiles = k1 > k0 ? (k1 - k0 + TILE - 1) / TILE : 0;

  if (lane == 0) {
    for (int s = 0; s < C::STAGES; ++s) mbar_init(smem_u32(bars + warp * C::STAGES + s), 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  // the chunk's pages (a chunk starts on a page: it is a multiple of the page size or within one)
  const int p0 = k0 >> a.page_log2;
  const int np = ntiles ? ((k1 - 1) >> a.page_log2) - p0 + 1 : 0;
  for (int i = threadIdx.x; i < np; i += THREADS) {
    int pid = a.block_table[(int64_t)b * a.width + p0 + i];
    if (pid < 0 || pid >= a.pages) {
      note_err(nullptr, ERR_PAGE);
      pid = 0;
    }
    const int blk = pid * a.Hkv + kvh;
    s_row[i] = blk << a.page_log2;
    s_ks[i] = a.k_scale[blk];
    s_lv[i] = log2f(a.v_scale[blk]);
  }
  __syncthreads();

  const uint32_t ring = smem_u32(smem) + warp * C::RING;
  const uint32_t bar0 = smem_u32(bars + warp * C::STAGES);
  auto issue = [&](int tile, int stage) {  // lane 0
    const int key = k0 + tile * TILE;
    const int y = s_row[(key >> a.page_log2) - p0] + (key & ((1 << a.page_log2) - 1));
    const uint32_t bar = bar0 + 8 * stage, dst = ring + stage * 2 * C::TILE_BYTES;
    mbar_expect_tx(bar, 2 * C::TILE_BYTES);
    tma_load_2d(dst, &map_k, 0, y, bar);
    tma_load_2d(dst + C::TILE_BYTES, &map_v, 0, y, bar);
  };
  const int mine = ntiles > warp ? (ntiles - warp + WARPS - 1) / WARPS : 0;  // tiles warp, warp + 4, ..
  int issued = 0;
  if (lane == 0)
    for (; issued < min(mine, C::STAGES); ++issued) issue(warp + issued * WARPS, issued);

  // Q as the second operand of S^T = K Q^T.  Lane (g, t) holds row g's
  // columns D/4 * t ..: k step w takes its 4 columns D/4 * t + 4 w ...
  uint32_t qf[NT][KS][2];
  float qs[NT];  // the power of two taken out of row g's query
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    const int r = row0 + n * 8 + g;
    uint32_t w[D / 8];
#pragma unroll
    for (int i = 0; i < D / 8; ++i) w[i] = 0;
    if (r < row0 + nrows) {
      const uint16_t* p = a.q + (int64_t)b * a.qb + (int64_t)(r / a.G) * a.qt +
                          (int64_t)(kvh * a.G + r % a.G) * a.qh + t * (D / 4);
#pragma unroll
      for (int i = 0; i < D / 32; ++i) {
        const uint4 v = __ldg(reinterpret_cast<const uint4*>(p) + i);
        w[4 * i] = v.x, w[4 * i + 1] = v.y, w[4 * i + 2] = v.z, w[4 * i + 3] = v.w;
      }
    }
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < D / 8; ++i) {
      const uint32_t v = w[i] & 0x7FFF7FFFu;
      m = max(m, max(v & 0xFFFFu, v >> 16));
    }
    m = max(m, __shfl_xor_sync(FULL, m, 1));
    m = max(m, __shfl_xor_sync(FULL, m, 2));
    const int e = min(max((int)(m >> 7), 15), 253);  // the largest value's exponent field
    const float up = __uint_as_float((uint32_t)(254 + 14 - e) << 23);
    qs[n] = __uint_as_float((uint32_t)(e - 14) << 23);
#pragma unroll
    for (int i = 0; i < D / 8; ++i)
      qf[n][i >> 1][i & 1] = f16x2(bf_lo(w[i]) * up, bf_hi(w[i]) * up);
  }
  // for the scores' columns 2t, 2t + 1 of each row tile: the query's factor
  // and the last key the row sees (rows without a query are not written)
  float cs[NT][2];
  int lim[NT][2];
#pragma unroll
  for (int n = 0; n < NT; ++n)
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      cs[n][c] = __shfl_sync(FULL, qs[n], (2 * t + c) * 4) * a.sm_log2;
      const int r = n * 8 + 2 * t + c;
      lim[n][c] = held + (row0 + r) / a.G;
    }
  const int free_end = held + row0 / a.G + 1;  // keys below: every row sees them

  float o[NT][KS][4];
  float mx[NT][2], sum[NT][2], wx[NT][2];  // m, l, w of columns 2t, 2t + 1
#pragma unroll
  for (int n = 0; n < NT; ++n) {
#pragma unroll
    for (int j = 0; j < KS; ++j) o[n][j][0] = o[n][j][1] = o[n][j][2] = o[n][j][3] = 0.0f;
    mx[n][0] = mx[n][1] = wx[n][0] = wx[n][1] = NEG_INF;
    sum[n][0] = sum[n][1] = 0.0f;
  }

  int stage = 0;
  uint32_t phase = 0;
  for (int i = 0; i < mine; ++i) {
    const int key0 = k0 + (warp + i * WARPS) * TILE;
    const int pg = (key0 >> a.page_log2) - p0;
    const float ks = s_ks[pg], lv = s_lv[pg];
    if (!mbar_wait_warp(bar0 + 8 * stage, phase, nullptr, ERR_WAIT)) break;
    const uint32_t kb = ring + stage * 2 * C::TILE_BYTES, vb = kb + C::TILE_BYTES;
    const bool tail = key0 + TILE > free_end;

    // scores: two m tiles of 16 keys
    float s[NT][2][4];
#pragma unroll
    for (int mt = 0; mt < 2; ++mt) {
#pragma unroll
      for (int n = 0; n < NT; ++n) s[n][mt][0] = s[n][mt][1] = s[n][mt][2] = s[n][mt][3] = 0.0f;
      uint32_t ka[D / 16], kc[D / 16];  // rows g and g + 8 of the tile, D / 4 columns
      const int r = mt * 16 + g;
#pragma unroll
      for (int c = 0; c < D / 64; ++c) {
        const uint4 x = lds128(kb + swz<D>(r, t * (D / 64) + c));
        const uint4 y = lds128(kb + swz<D>(r + 8, t * (D / 64) + c));
        ka[4 * c] = x.x, ka[4 * c + 1] = x.y, ka[4 * c + 2] = x.z, ka[4 * c + 3] = x.w;
        kc[4 * c] = y.x, kc[4 * c + 1] = y.y, kc[4 * c + 2] = y.z, kc[4 * c + 3] = y.w;
      }
#pragma unroll
      for (int w = 0; w < KS; ++w) {
        const uint32_t a0 = unpack2(ka[w]), a2 = unpack2_hi(ka[w]);
        const uint32_t a1 = unpack2(kc[w]), a3 = unpack2_hi(kc[w]);
#pragma unroll
        for (int n = 0; n < NT; ++n) mma(s[n][mt], a0, a1, a2, a3, qf[n][w][0], qf[n][w][1]);
      }
    }

    // running maxima and sum; P^T as the second operand of the output
    uint32_t pf[NT][2][2];
    float corr[NT][2];
    bool grew = false;
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      const float f0 = cs[n][0] * ks, f1 = cs[n][1] * ks;
#pragma unroll
      for (int mt = 0; mt < 2; ++mt) {
        s[n][mt][0] *= f0, s[n][mt][2] *= f0;
        s[n][mt][1] *= f1, s[n][mt][3] *= f1;
        if (tail) {
          const int key = key0 + mt * 16 + g;
          if (key > lim[n][0]) s[n][mt][0] = NEG_INF;
          if (key > lim[n][1]) s[n][mt][1] = NEG_INF;
          if (key + 8 > lim[n][0]) s[n][mt][2] = NEG_INF;
          if (key + 8 > lim[n][1]) s[n][mt][3] = NEG_INF;
        }
      }
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        float m = fmaxf(fmaxf(s[n][0][c], s[n][0][c + 2]), fmaxf(s[n][1][c], s[n][1][c + 2]));
        m = fmaxf(m, __shfl_xor_sync(FULL, m, 4));
        m = fmaxf(m, __shfl_xor_sync(FULL, m, 8));
        m = fmaxf(m, __shfl_xor_sync(FULL, m, 16));
        const float w = fmaxf(m + lv, wx[n][c]);
        m = fmaxf(m, mx[n][c]);
        // nothing seen yet (or every v_scale 0): every weight is 0
        const float ref = m == NEG_INF ? 0.0f : m, wref = w == NEG_INF ? 0.0f : w;
        const float lower = ex2(mx[n][c] - ref);
        corr[n][c] = ex2(wx[n][c] - wref);
        grew |= w != wx[n][c];
        mx[n][c] = m;
        wx[n][c] = w;
        const float pref = wref - lv - P_EXP;
        float add = 0.0f;
#pragma unroll
        for (int mt = 0; mt < 2; ++mt) {
          add += ex2(s[n][mt][c] - ref) + ex2(s[n][mt][c + 2] - ref);
          s[n][mt][c] = ex2(s[n][mt][c] - pref);
          s[n][mt][c + 2] = ex2(s[n][mt][c + 2] - pref);
        }
        sum[n][c] = fmaf(sum[n][c], lower, add);
      }
#pragma unroll
      for (int mt = 0; mt < 2; ++mt) {
        pf[n][mt][0] = transpose8x8(f16x2(s[n][mt][0], s[n][mt][1]));
        pf[n][mt][1] = transpose8x8(f16x2(s[n][mt][2], s[n][mt][3]));
      }
    }
    if (__any_sync(FULL, grew)) {
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int j = 0; j < KS; ++j) {
          o[n][j][0] *= corr[n][0], o[n][j][2] *= corr[n][0];
          o[n][j][1] *= corr[n][1], o[n][j][3] *= corr[n][1];
        }
    }

    // output: lane (g, t) holds columns D/8 * g .. of keys 2t, 2t+1, 2t+8, 2t+9
    // of each half tile
    constexpr int VW = D / 32;  // words of D / 8 columns
    uint32_t v[2][4][VW];
#pragma unroll
    for (int mt = 0; mt < 2; ++mt)
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const int r = mt * 16 + 2 * t + (k & 1) + (k >> 1) * 8;
        if (D == 128) {
          const uint4 x = lds128(vb + swz<D>(r, g));
          v[mt][k][0] = x.x, v[mt][k][1] = x.y, v[mt][k][VW - 2] = x.z, v[mt][k][VW - 1] = x.w;
        } else {
          const uint2 x = lds64(vb + swz<D>(r, g >> 1) + (g & 1) * 8);
          v[mt][k][0] = x.x, v[mt][k][1] = x.y;
        }
      }
    // O^T tile by tile; rows g and g + 8 of m tile j are columns 2j and 2j + 1
    auto product = [&](int n, int j, const uint32_t (&x)[2][4][VW], float (&acc)[4]) {
#pragma unroll
      for (int mt = 0; mt < 2; ++mt) {
        const uint32_t sel = (j & 1) ? 0x7362u : 0x5140u;
        const uint32_t lo = __byte_perm(x[mt][0][j >> 1], x[mt][1][j >> 1], sel);
        const uint32_t hi = __byte_perm(x[mt][2][j >> 1], x[mt][3][j >> 1], sel);
        mma(acc, unpack2(lo), unpack2_hi(lo), unpack2(hi), unpack2_hi(hi), pf[n][mt][0], pf[n][mt][1]);
      }
    };
    uint32_t odd = 0;  // a NaN value where some row sees it and another does not, or past the end
    if (tail) {
#pragma unroll
      for (int mt = 0; mt < 2; ++mt)
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const int key = key0 + mt * 16 + 2 * t + (k & 1) + (k >> 1) * 8;
#pragma unroll
          for (int w = 0; w < VW; ++w) {
            if (key >= end) v[mt][k][w] = 0;  // slots that hold no token of this sequence
            odd |= has_nan(v[mt][k][w]);
          }
        }
      odd = __any_sync(FULL, odd != 0);
    }
    if (!odd) {
#pragma unroll
      for (int j = 0; j < KS; ++j)
#pragma unroll
        for (int n = 0; n < NT; ++n) product(n, j, v, o[n][j]);
    } else {
      // 0 * NaN is NaN, also for a row that may not see the value: each row
      // gets a product of its own with the values it does not see taken as 0
#pragma unroll 1
      for (int n8 = 0; n8 < C::ROWS; ++n8) {
        const int last = held + (row0 + n8) / a.G;
        uint32_t x[2][4][VW];
#pragma unroll
        for (int mt = 0; mt < 2; ++mt)
#pragma unroll
          for (int k = 0; k < 4; ++k)
#pragma unroll
            for (int w = 0; w < VW; ++w)
              x[mt][k][w] =
                  key0 + mt * 16 + 2 * t + (k & 1) + (k >> 1) * 8 > last ? 0u : v[mt][k][w];
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          if (n != n8 >> 3) continue;
          const bool c0 = (n8 & 7) == 2 * t, c1 = (n8 & 7) == 2 * t + 1;
#pragma unroll
          for (int j = 0; j < KS; ++j) {
            float acc[4] = {0.0f, 0.0f, 0.0f, 0.0f};
            product(n, j, x, acc);
            if (c0) o[n][j][0] += acc[0], o[n][j][2] += acc[2];
            if (c1) o[n][j][1] += acc[1], o[n][j][3] += acc[3];
          }
        }
      }
    }
    __syncwarp();  // every lane has read the stage
    if (lane == 0 && issued < mine) {
      issue(warp + issued * WARPS, stage);
      ++issued;
    }
    if (++stage == C::STAGES) stage = 0, phase ^= 1;
  }
  // after a wait that gave up: this warp's loads land before the ring is reused
  {
    const int n = __shfl_sync(FULL, issued, 0);
    for (int i = max(0, n - C::STAGES); i < n; ++i)
      mbar_wait(bar0 + 8 * (i % C::STAGES), (i / C::STAGES) & 1, nullptr, ERR_WAIT);
  }

  // ---- join the warps: the ring becomes [WARPS][ROWS][D] O, then maxima and sums ----
  __syncthreads();
  float* so = reinterpret_cast<float*>(smem);
  float* sm = so + WARPS * C::ROWS * D;
  float* sl = sm + WARPS * C::ROWS;
  float* sw = sl + WARPS * C::ROWS;
#pragma unroll
  for (int n = 0; n < NT; ++n)
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      float l = sum[n][c];
      l += __shfl_xor_sync(FULL, l, 4);
      l += __shfl_xor_sync(FULL, l, 8);
      l += __shfl_xor_sync(FULL, l, 16);
      const int r = n * 8 + 2 * t + c;
      if (g == 0) {
        sm[warp * C::ROWS + r] = mx[n][c];
        sl[warp * C::ROWS + r] = l;
        sw[warp * C::ROWS + r] = wx[n][c];
      }
      float* p = so + (warp * C::ROWS + r) * D + g * (D / 8);
#pragma unroll
      for (int j = 0; j < KS; ++j)
        *reinterpret_cast<float2*>(p + 2 * j) = make_float2(o[n][j][c], o[n][j][c + 2]);
    }
  __syncthreads();
  constexpr int PART = C::ROWS * (D + 3);  // O, then m, l and w of each row
  float* mine_part = a.part + ((int64_t)pair * a.chunks + chunk) * PART;
  for (int i = threadIdx.x; i < C::ROWS * D; i += THREADS) {
    const int r = i / D, d = i % D;
    State st;
#pragma unroll
    for (int w = 0; w < WARPS; ++w)
      st.add(sm[w * C::ROWS + r], sl[w * C::ROWS + r], sw[w * C::ROWS + r], so[(w * C::ROWS + r) * D + d]);
    if (nchunks == 1) {
      const int row = row0 + r;
      if (row < a.T * a.G)
        BF16::store(a.out + (((int64_t)b * a.T + row / a.G) * a.H + kvh * a.G + row % a.G) * D + d,
                    r < nrows ? st.value() : 0.0f);
    } else {
      mine_part[r * D + d] = st.x;
      if (d == 0) {
        mine_part[C::ROWS * D + r] = st.m;
        mine_part[C::ROWS * (D + 1) + r] = st.l;
        mine_part[C::ROWS * (D + 2) + r] = st.w;
      }
    }
  }
  if (nchunks == 1) return;

  // ---- join the chunks: the last CTA of the pair reads them in order ----
  __threadfence();
  __syncthreads();
  if (threadIdx.x == 0) s_last = atomicAdd(a.done + pair, 1) == nchunks - 1;
  __syncthreads();
  if (!s_last) return;
  __threadfence();
  const float* all = a.part + (int64_t)pair * a.chunks * PART;
  for (int i = threadIdx.x; i < C::ROWS * D; i += THREADS) {
    const int r = i / D, d = i % D, row = row0 + r;
    if (row >= a.T * a.G) continue;
    State st;
    for (int c = 0; c < nchunks; ++c) {
      const float* p = all + (int64_t)c * PART;
      st.add(__ldcg(p + C::ROWS * D + r), __ldcg(p + C::ROWS * (D + 1) + r),
             __ldcg(p + C::ROWS * (D + 2) + r), __ldcg(p + r * D + d));
    }
    BF16::store(a.out + (((int64_t)b * a.T + row / a.G) * a.H + kvh * a.G + row % a.G) * D + d,
                r < nrows ? st.value() : 0.0f);
  }
  if (threadIdx.x == 0) a.done[pair] = 0;
}

// How a call's work is cut: keys per chunk (a multiple of 128, at most
// PAGES_MAX pages), chunks of the longest sequence, row tiles.
struct Cut {
  int nt, groups, chunk, chunks;
};
Cut cut_of(int64_t batch, int64_t tokens, int heads, int kv_heads, int page, int64_t capacity) {
  Cut c;
  const int64_t rows = tokens * (heads / kv_heads);
  c.nt = rows > 8 ? 2 : 1;
  c.groups = (int)((rows + 8 * c.nt - 1) / (8 * c.nt));
  const int64_t pairs = batch * kv_heads * c.groups;
  // about four waves of two CTAs per SM at the longest length, 512 keys or more
  const int64_t want = std::max<int64_t>(1, (8 * vq::mx::sm_count() + pairs - 1) / pairs);
  int64_t chunk = std::max<int64_t>(512, (capacity + want - 1) / want);
  chunk = (chunk + 127) / 128 * 128;
  chunk = std::min<int64_t>(chunk, 512ll * page);
  c.chunk = (int)chunk;
  c.chunks = (int)std::max<int64_t>(1, (capacity + chunk - 1) / chunk);
  return c;
}

template <int D, int NT>
int launch(const CUtensorMap& mk, const CUtensorMap& mv, const Args& a, cudaStream_t st) {
  using C = Cfg<D, NT>;
  static_assert(WARPS * C::STAGES * 8 <= 256, "barrier area");
  if (!allow_smem<k_attn_kv8<D, NT>>(C::SMEM))
    return VQ_ERR_CUDA;
  k_attn_kv8<D, NT><<<dim3(a.chunks, a.Hkv * a.groups, a.B), THREADS, C::SMEM, st>>>(mk, mv, a);
  return cudaGetLastError() == cudaSuccess ? VQ_OK : VQ_ERR_CUDA;
}

int sticky_kva(int* out, int clear, cudaStream_t st) { return vq::tc::sticky_read(out, clear, st); }

}  // namespace kva
}  // namespace vq

using namespace vq::kva;

extern "C" {

int vq_attn_kv8_workspace(int64_t batch, int64_t tokens, int32_t heads, int32_t kv_heads,
                          int32_t head_dim, int32_t page, int64_t table_width, int64_t* floats,
                          int64_t* counters) {
  if (!floats || !counters) return VQ_ERR_NULL;
  if (batch < 0 || tokens < 0 || kv_heads <= 0 || heads <= 0 || heads % kv_heads || head_dim <= 0 ||
      page <= 0 || table_width < 0)
    return VQ_ERR_INVALID;
  const Cut c = cut_of(std::max<int64_t>(batch, 1), std::max<int64_t>(tokens, 1), heads, kv_heads, page,
                       table_width * page);
  *counters = batch * kv_heads * c.groups;
  *floats = c.chunks == 1 ? 0 : *counters * c.chunks * 8 * c.nt * (head_dim + 3);
  return VQ_OK;
}

int vq_attn_kv8(const void* q, const int64_t* q_strides, int64_t batch, int64_t tokens, int32_t heads,
                int32_t kv_heads, int32_t head_dim, const void* k_codes, const void* v_codes,
                const float* k_scale, const float* v_scale, int64_t pages, int32_t page,
                const void* block_table, int64_t table_width, const void* lengths, const void* counts,
                float sm_scale, float* workspace, int64_t workspace_floats, int32_t* counters,
                int64_t counters_len, void* out, void* stream) {
  if (head_dim != 64 && head_dim != 128) return VQ_ERR_UNSUPPORTED;
  if (page != 32 && page != 64 && page != 128) return VQ_ERR_UNSUPPORTED;
  if (batch < 0 || tokens < 0 || heads <= 0 || kv_heads <= 0 || heads % kv_heads || table_width < 0 ||
      pages < 0 || pages * kv_heads * page >= (1ll << 31) || table_width * page >= (1ll << 31) ||
      tokens >= (1 << 20) || batch > 65535 || batch * tokens * heads >= (1ll << 31))
    return VQ_ERR_INVALID;
  if (batch == 0 || tokens == 0) return VQ_OK;
  if (!q || !q_strides || !k_codes || !v_codes || !k_scale || !v_scale || !block_table || !lengths ||
      !counters || !out)
    return VQ_ERR_NULL;
  const void* p16[5] = {q, k_codes, v_codes, out, workspace};
  for (const void* p : p16)
    if (reinterpret_cast<uintptr_t>(p) & 15) return VQ_ERR_ALIGNMENT;
  for (int i = 0; i < 3; ++i)
    if (q_strides[i] % 8) return VQ_ERR_ALIGNMENT;
  const Cut c = cut_of(batch, tokens, heads, kv_heads, page, table_width * page);
  const int64_t pairs = batch * kv_heads * c.groups;
  if (c.groups * (int64_t)kv_heads > 65535) return VQ_ERR_INVALID;
  if (counters_len < pairs) return VQ_ERR_INVALID;
  if (c.chunks > 1 && (!workspace || workspace_floats < pairs * c.chunks * 8 * c.nt * (head_dim + 3)))
    return VQ_ERR_INVALID;
  if (pages == 0 || table_width == 0) {  // an empty cache: no row sees a key
    if (table_width) return VQ_ERR_INVALID;
    return cudaMemsetAsync(out, 0, (size_t)(batch * tokens * heads * head_dim * 2),
                           reinterpret_cast<cudaStream_t>(stream)) == cudaSuccess ? VQ_OK : VQ_ERR_CUDA;
  }
  CUtensorMap mk, mv;
  const uint64_t rows = (uint64_t)pages * kv_heads * page;
  if (!vq::mx::make_map_box(&mk, k_codes, rows, head_dim, head_dim, TILE, head_dim) ||
      !vq::mx::make_map_box(&mv, v_codes, rows, head_dim, head_dim, TILE, head_dim))
    return VQ_ERR_CUDA;
  Args a;
  a.q = (const uint16_t*)q;
  a.qb = q_strides[0], a.qt = q_strides[1], a.qh = q_strides[2];
  a.out = (uint16_t*)out;
  a.k_scale = k_scale, a.v_scale = v_scale;
  a.block_table = (const int32_t*)block_table;
  a.lengths = (const int32_t*)lengths;
  a.counts = (const int32_t*)counts;
  a.part = workspace;
  a.done = counters;
  a.B = (int)batch, a.T = (int)tokens, a.H = heads, a.Hkv = kv_heads, a.G = heads / kv_heads;
  a.page_log2 = page == 32 ? 5 : page == 64 ? 6 : 7;
  a.width = (int)table_width, a.pages = (int)pages;
  a.groups = c.groups, a.chunks = c.chunks, a.chunk = c.chunk;
  a.sm_log2 = sm_scale * 1.4426950408889634f;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  if (head_dim == 128) return c.nt == 1 ? launch<128, 1>(mk, mv, a, st) : launch<128, 2>(mk, mv, a, st);
  return c.nt == 1 ? launch<64, 1>(mk, mv, a, st) : launch<64, 2>(mk, mv, a, st);
}

}  // extern "C"
