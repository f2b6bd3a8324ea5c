// Attention of the newest tokens over a paged key / value cache, in E4M3 or in 4 bits.
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
// Work: the keys of every (sequence, row group, kv head) in units of 128,
// laid end to end and cut into equal runs, one per CTA (two or three per SM), so
// that unequal lengths leave no SM idle; a run may span several heads or
// sequences.  Each of a CTA's 4 warps takes one 32-key tile of every unit and
// has a ring of its own that TMA fills (K and V, 32 x D bytes each,
// SWIZZLE_128B / SWIZZLE_64B: the fragment loads then meet no bank conflict
// for D = 128).  The pieces of a head that was cut are joined by the CTA that
// finishes last, in the CTAs' order, so the result does not depend on the
// order of arrival.
//
// Bound by HBM: 2 D bytes per key and kv head (4 sequences of 131000 keys, 8 x 8
// heads of 128: 168 us, 6.4 TB/s); one short sequence by a chain of latencies
// (99 keys: 7 us); several row tiles by the products (5 tokens x 7 heads of 64:
// 24 us where the bytes take 2.5).
//
// FP4: the cache of vq_rope_append_kv4 (E2M1 codes, an E4M3 scale per 16 columns of
// a token, a float32 factor per head), for calls with few rows a kv head; the others
// are vq_attn_kv4.cu's.  The same work with these differences:
//  - a tile's codes and scales lie side by side, so that four untiled copies fetch
//    it; the fragment loads' bank conflicts are avoided by the order of the keys
//    within the product (key4), which no sum depends on.
//  - code * scale is exact in f16 (6 significant bits): four conversions of E2M1 pairs
//    and four products with the scale's pair make a word's operands.  A key pair's codes
//    lie in one word, so that V needs no shuffle.
//  - no page has a factor of its own, so the weights are relative to m alone, and m
//    and O move only where some score of the tile passes m (a vote): 2^(15 + s - m).
//  - a NaN scale makes K's scores NaN as it is.  V's is looked for only in tiles whose
//    keys some row does not see (0 * NaN); its key is noted, and the rows that see
//    it get NaN at the end.
// Bound by the latency of a warp's chain at 12 warps an SM (161 registers): 676
// instructions a warp and tile of 32 keys and 8 rows, of which the loads, conversions
// and products of 4.5 KB are most, in half of the issue slots; HBM has 9/16 of E4M3's
// bytes.  4 sequences of 131000 keys, 8 x 8 heads of 128: 144 us over and over, where the
// power cap takes the clock to 1.82 GHz (4.2 TB/s), 133 in short runs; 32 sequences to
// 8192, 8 x 4 heads: 45 us where E4M3 takes 53; 99 keys: 7.4 us.
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <algorithm>
#include <type_traits>

#include "voyager_b200.h"
#include "vq_e4m3.cuh"
#include "vq_pdl.cuh"
#include "vq_tc.cuh"

namespace vq {
namespace kv4 {  // vq_attn_kv4.cu
int64_t workspace(int64_t batch, int64_t tokens, int heads, int kv_heads, int head_dim, int64_t capacity);
int attend(const void* q, const int64_t* q_strides, int64_t batch, int64_t tokens, int heads, int kv_heads, int head_dim,
           const void* k_codes, const void* v_codes, const void* k_scale, const void* v_scale, const float* k_factor,
           const float* v_factor, int64_t pages, int page, const void* block_table, int64_t table_width,
           const void* lengths, const void* counts, float sm_scale, float* workspace, int64_t workspace_floats,
           void* out, cudaStream_t st);
}  // namespace kv4
namespace kva {

using namespace vq::e4;
using namespace vq::tc;

enum { ERR_WAIT = 311, ERR_PAGE = 312, ERR_CAPACITY = 313, ERR_COUNT = 314 };

constexpr int WARPS = 4, THREADS = WARPS * 32, TILE = 32, UNIT = WARPS * TILE;
constexpr int PLANS = 256;
constexpr float NEG_INF = -__builtin_huge_valf();
constexpr float P_EXP = 15.0f;  // the largest weight is 2^15 in f16

struct Args {
  const uint16_t* q;  // bf16, strides in elements
  int64_t qb, qt, qh;
  uint16_t* out;  // bf16 [B, T, H, D]
  const float *k_scale, *v_scale;  // per page and head; in 4 bits per head: the factors
  const uint8_t *k_codes, *v_codes, *k_bscale, *v_bscale;  // in 4 bits: the codes, E4M3 [pages, Hkv, page, D / 16]
  const int32_t *block_table, *lengths, *counts;
  float* part;        // [CTAs][2][ROWS * (D + 3)]: pieces of heads that were cut
  int32_t* done;      // [B * groups * Hkv] zero before, zero after
  int B, T, H, Hkv, G, page_log2, width, pages;
  int groups;         // row groups per sequence
  uint32_t by_g;      // ceil(2^31 / G)
  float sm_log2;              // sm_scale * log2(e)
};

// CTAs per SM.  Three with heads of 64 and one row tile (24 sequences of 28631
// keys: 130 us against 149 with two, in deeper rings than now); otherwise the third CTA costs more in
// joins and shallower rings than its warps give (heads of 128, 32 sequences:
// 66 us against 55).  In 4 bits, where a warp's chain is longer, three with one row tile.
constexpr int ctas_per_sm(int head_dim, int nt, bool fp4) {
  return (head_dim == 64 || fp4) && nt == 1 ? 3 : 2;
}

template <int D, int NT, bool FP4>
struct Cfg {
  static constexpr int ROWS = 8 * NT;
  // a stage holds codes of K, codes of V; in 4 bits then their scales
  static constexpr int TILE_BYTES = FP4 ? TILE * D / 2 : TILE * D, SCALE_BYTES = FP4 ? TILE * D / 16 : 0;
  static constexpr int STAGE = 2 * (TILE_BYTES + SCALE_BYTES);
  // Two stages a warp: 128 KB in flight an SM (96 KB at heads of 64) fill HBM, and
  // more only lengthens the queue that every other access waits in (4 sequences
  // of 131000 keys: 168 us, with three 178; heads of 64, 24 sequences of 28631:
  // 118, with four 126).  In 4 bits a stage is 9/16 as large: two of them at heads of
  // 128 and three CTAs an SM (108 KB), three at heads of 64 (81 KB).
  static constexpr int PER_SM = ctas_per_sm(D, NT, FP4);
  static constexpr int STAGES = FP4 ? (D == 128 ? 2 : 3) : D == 128 || PER_SM == 3 ? 2 : 3;
  static constexpr int RING = STAGES * STAGE;  // per warp
  static constexpr int SMEM_RING = WARPS * RING;
  // the warps' O meet in SUMS buffers, rows LD floats apart
  static constexpr int SUMS = NT == 1 ? 2 : 1, LD = D + 4;
  static constexpr int JOIN = (SUMS * ROWS * LD + 3 * WARPS * ROWS + 4 * ROWS) * 4;
  static constexpr int SMEM = SMEM_RING + JOIN + 1024 + 256;
  static_assert(JOIN % 16 == 0 && WARPS * STAGES * 8 <= 256, "barriers after the join's area");
  static_assert(SUMS * ROWS * LD >= 8 * THREADS, "a join's groups meet there");
  static_assert(3 * ROWS <= THREADS, "a thread for each of a row's m, l and w");
  static_assert(PER_SM * (SMEM + 3200 + 1024) <= 227 * 1024, "CTAs per SM");
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
// Bits 0x80 of it: the word's bytes that are an E4M3 NaN (0x7F or 0xFF).
__device__ __forceinline__ uint32_t nan_bits(uint32_t w) { return (w & 0x7F7F7F7Fu) + 0x01010101u; }

__device__ __forceinline__ uint32_t lds32(uint32_t a) {
  uint32_t v;
  asm volatile("ld.shared.b32 %0, [%1];" : "=r"(v) : "r"(a));
  return v;
}
__device__ __forceinline__ uint32_t lds16(uint32_t a) {
  uint16_t v;
  asm volatile("ld.shared.b16 %0, [%1];" : "=h"(v) : "r"(a));
  return v;
}
__device__ __forceinline__ uint32_t lds8(uint32_t a) {
  uint32_t v;
  asm volatile("ld.shared.u8 %0, [%1];" : "=r"(v) : "r"(a));
  return v;
}
// In 4 bits: the key, of each 8, that index i of the products stands for.  The
// keys 2t of lanes t, and those of two neighbouring g, then lie in different
// banks.
__device__ __forceinline__ int key4(int i) { return (i & 12) | (0x9C >> ((i & 3) * 2) & 3); }
// One lane of a converged warp: the copies' operands stay in uniform registers.
__device__ __forceinline__ bool elect_one() {
  uint32_t p;
  asm volatile("{\n\t.reg .pred P;\n\telect.sync _|P, 0xFFFFFFFF;\n\tselp.u32 %0, 1, 0, P;\n\t}" : "=r"(p));
  return p != 0;
}

// Byte offset of 16-byte chunk c of row r in a TMA-swizzled tile of D-byte rows.
template <int D>
__device__ __forceinline__ uint32_t swz(int r, int c) {
  return D == 128 ? (uint32_t)(r * 128 + ((c ^ (r & 7)) << 4))
                  : (uint32_t)(r * 64 + ((c ^ ((r >> 1) & 3)) << 4));
}

// The output's factor of O from a row's m, l and w (0 for a row without keys).
__device__ __forceinline__ float out_scale(float m, float l, float w) {
  return l == 0.0f || w == NEG_INF ? 0.0f : __fdiv_rn(ex2(w - P_EXP - m), l);
}

// A sequence's tokens held and new tokens, brought to what fits.
__device__ __forceinline__ int2 plan_of(const Args& a, int b, int& err) {
  int held = a.lengths[b], cnt = a.counts ? a.counts[b] : a.T;
  if (held < 0 || cnt < 0 || cnt > a.T) {
    err = ERR_COUNT;
    cnt = held < 0 ? 0 : min(max(cnt, 0), a.T);
    held = max(held, 0);
  }
  const int64_t cap = (int64_t)a.width << a.page_log2;
  if (held + (int64_t)cnt > cap) {
    err = ERR_CAPACITY;
    cnt = held >= cap ? 0 : (int)(cap - held);
  }
  return make_int2(held, cnt);
}
// Entry e = (sequence, row group): the rows of it that have a query, the
// tokens held, and the keys that some of its rows sees.
struct Entry {
  int b, row0, nrows, held, end;
};
template <int ROWS>
__device__ __forceinline__ Entry entry_of(const Args& a, int e, const int2* plans) {
  Entry x;
  x.b = a.groups == 1 ? e : e / a.groups;
  x.row0 = (e - x.b * a.groups) * ROWS;
  int err;
  const int2 plan = x.b < PLANS ? plans[x.b] : plan_of(a, x.b, err);
  x.held = plan.x;
  x.nrows = min(ROWS, plan.y * a.G - x.row0);
  x.end = 0;
  if (x.nrows > 0) x.end = x.held + (a.groups == 1 ? plan.y : (x.row0 + x.nrows - 1) / a.G + 1);
  return x;
}
__device__ __forceinline__ int units_of(const Entry& x) { return (x.end + UNIT - 1) / UNIT; }

template <int D, int NT, bool FP4>
__global__ void __launch_bounds__(THREADS, ctas_per_sm(D, NT, FP4))
    k_attn_kv(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v,
               const __grid_constant__ Args a) {
  using C = Cfg<D, NT, FP4>;
  constexpr int KS = D / 16;   // k steps of the scores, and m tiles of the output
  constexpr int PART = C::ROWS * (D + 3);  // O, then m, l and w of each row
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                             ~(uintptr_t)1023);
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + C::SMEM_RING + C::JOIN);  // [WARPS][STAGES]
  __shared__ int s_last, s_entry, s_before, s_run[2];
  __shared__ long long s_sum[WARPS];
  __shared__ int s_top[WARPS];
  __shared__ int2 s_plan[PLANS];  // the first sequences' plans

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  pdl::trigger();
  if (lane == 0) {
    for (int s = 0; s < C::STAGES; ++s) mbar_init(smem_u32(bars + warp * C::STAGES + s), 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }

  if (!FP4 && threadIdx.x == 0) {
    prefetch_map(&map_k);
    prefetch_map(&map_v);
  }
  pdl::wait();

  // ---- this CTA's run of units: a scan of the entries' unit counts (and, in
  // the upper 32 bits, of the entries that have any) ----
  for (int b = threadIdx.x; b < (blockIdx.x == 0 ? a.B : min(a.B, PLANS)); b += THREADS) {
    int err = 0;
    const int2 plan = plan_of(a, b, err);
    if (b < PLANS) s_plan[b] = plan;
    if (err && blockIdx.x == 0) note_err(nullptr, err);
  }
  __syncthreads();
  auto entry = [&](int e) { return entry_of<C::ROWS>(a, e, s_plan); };
  const int entries = a.B * a.groups, per = (entries + THREADS - 1) / THREADS;
  const int e0 = min(entries, (int)threadIdx.x * per), e1 = min(entries, e0 + per);
  long long own = 0;
  int top = 0;  // units of the longest head
#pragma unroll 1
  for (int e = e0; e < e1; ++e) {
    const int u = units_of(entry(e));
    own += u ? u + (1ll << 32) : 0;
    top = max(top, u);
  }
  long long scan = own;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const long long y = __shfl_up_sync(FULL, scan, d);
    if (lane >= d) scan += y;
  }
  top = __reduce_max_sync(FULL, top);
  if (lane == 31) s_sum[warp] = scan, s_top[warp] = top;
  __syncthreads();
  long long total = 0, before = scan - own;
#pragma unroll
  for (int w = 0; w < WARPS; ++w) {
    if (w < warp) before += s_sum[w];
    total += s_sum[w];
    top = max(top, s_top[w]);
  }
  // CTAs with work.  A piece more of a head costs its join about an eighth of
  // a unit's time, so a run is at least sqrt(units / 8) of an average head.
  // Where heads are not few a head counts HEAD units more than it has: opening,
  // joining and closing one takes that long.  A cut in those moves to the
  // head's begin, and where a run about holds the longest head one within HEAD
  // of a head's end moves there (256 heads of 609 keys on 296 CTAs: 15 us
  // against 20; longer heads only give unequal runs).
  const int heads = (int)(total >> 32) * a.Hkv, real = (int)total * a.Hkv;
  const float least = heads ? fmaxf(1.0f, sqrtf(0.125f * (float)real / (float)heads)) : 1.0f;
  const int runs = min((int)gridDim.x, (int)ceilf((float)real / least));
  // (In 4 bits, whose units take half as long to read but not to multiply: 3; 32
  // sequences to 8192 keys 46.3 us, with 5 47.7, with 1 47.5.)
  const int HEAD = 6 * heads >= runs ? (FP4 ? 3 : 5) : 0;
  const int all = real + HEAD * heads;
  const int base = runs ? all / runs : 0, near_end = 4 * (top + HEAD) <= 5 * base ? HEAD : 0;
  const int rest = all - base * runs;  // the first `rest` runs have one more
  auto run_of = [&](int at) {  // the run that holds this unit, by the cuts as they were before they moved
    const int far = at - rest * (base + 1);
    return (far < 0 ? 0 : rest) + (far < 0 ? at : far) / (far < 0 ? base + 1 : base);
  };
  auto run_begin = [&](int c) { return c * base + min(c, rest); };
  if ((int)blockIdx.x < runs) {
    const int cut0 = run_begin(blockIdx.x), cut1 = run_begin(blockIdx.x + 1);
    int at = ((int)before + HEAD * (int)(before >> 32)) * a.Hkv;
    const int to = at + ((int)own + HEAD * (int)(own >> 32)) * a.Hkv;
    if ((at <= cut0 && cut0 < to) || (at <= cut1 && cut1 < to)) {
#pragma unroll 1
      for (int e = e0; e < e1; ++e) {
        const int w = units_of(entry(e)) + HEAD;
        if (w == HEAD) continue;
        auto moved = [&](int cut) {
          const int ps = at + (cut - at) / w * w;
          return ps + w - cut <= near_end ? ps + w : cut - ps <= HEAD ? ps : cut;
        };
        const int next = at + w * a.Hkv;
        if (at <= cut0 && cut0 < next) {
          s_entry = e;
          s_before = at;
          s_run[0] = moved(cut0);
        }
        if (at <= cut1 && cut1 < next) s_run[1] = moved(cut1);
        at = next;
      }
    }
    if (threadIdx.x == 0 && cut1 == all) s_run[1] = all;
  } else if (threadIdx.x == 0) {
    s_run[0] = s_run[1] = 0;
  }
  __syncthreads();
  const int lo = s_run[0], hi = s_run[1];

  const uint32_t ring = smem_u32(smem) + warp * C::RING;
  const uint32_t bar0 = smem_u32(bars + warp * C::STAGES);
  int stage = 0;      // of the next tile to read; the ring runs on from segment to segment
  uint32_t phase = 0;
  bool ok = true;
  int pos = lo, ebase = s_before, e = s_entry - 1, units = 0;
  Entry x = {};

  // In 4 bits: where this lane's parts of a stage's first 8 keys lie: rows of K by
  // g and of V by t, and their scales.
  const uint32_t at_k = key4(g) * (D / 2) + t * (D / 8);
  const uint32_t at_ks = 2 * C::TILE_BYTES + key4(g) * (D / 16) + (D == 128 ? 2 * t : t);
  const uint32_t at_v0 = C::TILE_BYTES + key4(2 * t) * (D / 2) + g * (D / 16);
  const uint32_t at_v1 = C::TILE_BYTES + key4(2 * t + 1) * (D / 2) + g * (D / 16);
  const uint32_t at_vs0 = 2 * C::TILE_BYTES + C::SCALE_BYTES + key4(2 * t) * (D / 16) + (D == 128 ? g : g >> 1);
  const uint32_t at_vs1 = 2 * C::TILE_BYTES + C::SCALE_BYTES + key4(2 * t + 1) * (D / 16) + (D == 128 ? g : g >> 1);

  // A segment: the part of one head (entry, kv head) in this run.
  struct Seg {
    int b, row0, nrows, held, end, kvh, k0, k1, units, slot, pair;
    int tok0, head0;  // of row 0
    int ps;  // where the head begins
    bool whole;
  } sg = {};
  // A lane knows the page of tile 32 m + lane of the warp's tiles: its row in
  // the cache and its scales, n_ for the batch m that is being issued, c_ for
  // the one being read; the block table is read a batch ahead.  A page outside
  // the cache has n_v = -1, so that its logarithm is NaN: its tiles load page 0
  // and are passed over.
  int n_row = 0, pid_next = 0, mine = 0, issued = 0, wstage = 0;
  float n_ks = 0.0f, n_v = 0.0f, c_ks = 0.0f, c_lv = 0.0f;
  uint32_t skip = 0;  // in 4 bits: the stages whose tile is in no page
  auto key_of = [&](int tile) { return min(sg.k0 + (warp + tile * WARPS) * TILE, sg.k1 - 1); };
  auto pid_of = [&](int tile) { return a.block_table[(int64_t)sg.b * a.width + (key_of(tile) >> a.page_log2)]; };
  auto issue = [&]() {
    if ((issued & 31) == 0) {
      const bool outside = pid_next < 0 || pid_next >= a.pages;
      if (outside) note_err(nullptr, ERR_PAGE);
      const int blk = (outside ? 0 : pid_next) * a.Hkv + sg.kvh;
      n_row = (blk << a.page_log2) + (key_of(issued + lane) & ((1 << a.page_log2) - 1) & ~(TILE - 1));
      if constexpr (FP4) {
        n_v = 1.0f;
      } else {
        n_ks = a.k_scale[blk];
        n_v = a.v_scale[blk];
      }
      n_v = outside ? -1.0f : n_v >= 0.0f ? n_v : -NEG_INF;  // no logarithm: the output is NaN
      if (FP4 && outside) n_row = -1;
      pid_next = pid_of(issued + lane + 32);
    }
    int y = __shfl_sync(FULL, n_row, issued & 31);
    if (FP4 && y < 0) skip |= 1u << wstage, y = 0;
    if (FP4 ? elect_one() : lane == 0) {
      const uint32_t bar = bar0 + 8 * wstage, dst = ring + wstage * C::STAGE;
      mbar_expect_tx(bar, C::STAGE);
      if constexpr (!FP4) {
        tma_load_2d(dst, &map_k, 0, y, bar);
        tma_load_2d(dst + C::TILE_BYTES, &map_v, 0, y, bar);
      } else {  // 32 keys lie side by side
        bulk_load(dst, a.k_codes + (int64_t)y * (D / 2), C::TILE_BYTES, bar);
        bulk_load(dst + C::TILE_BYTES, a.v_codes + (int64_t)y * (D / 2), C::TILE_BYTES, bar);
        bulk_load(dst + 2 * C::TILE_BYTES, a.k_bscale + (int64_t)y * (D / 16), C::SCALE_BYTES, bar);
        bulk_load(dst + 2 * C::TILE_BYTES + C::SCALE_BYTES, a.v_bscale + (int64_t)y * (D / 16), C::SCALE_BYTES, bar);
      }
    }
    ++issued;
    if (++wstage == C::STAGES) wstage = 0;
  };
  // The next segment; start() puts its first loads on their way.
  auto open = [&]() {
#pragma unroll 1
    while (units == 0 || pos >= ebase + (units + HEAD) * a.Hkv) {  // the next entry with keys
      if (units) ebase += (units + HEAD) * a.Hkv;
      x = entry(++e);
      units = units_of(x);
    }
    sg.b = x.b, sg.row0 = x.row0, sg.nrows = x.nrows, sg.held = x.held, sg.end = x.end, sg.units = units;
    sg.tok0 = a.groups == 1 ? 0 : x.row0 / a.G;
    sg.head0 = x.row0 - sg.tok0 * a.G;
    sg.kvh = (pos - ebase) / (units + HEAD);
    sg.pair = e * a.Hkv + sg.kvh;
    sg.ps = ebase + sg.kvh * (units + HEAD);
    const int u0 = max(0, pos - sg.ps - HEAD), u1 = min(units, hi - sg.ps - HEAD);
    sg.whole = u0 == 0 && u1 == units;
    sg.slot = pos == lo ? 0 : 1;
    pos = min(hi, sg.ps + HEAD + units);
    sg.k0 = u0 * UNIT, sg.k1 = min(x.end, u1 * UNIT);
    const int ntiles = (sg.k1 - sg.k0 + TILE - 1) / TILE;
    // tiles warp, warp + 4, ..; none after a wait that gave up
    mine = ok && ntiles > warp ? (ntiles - warp + WARPS - 1) / WARPS : 0;
    issued = 0;
    wstage = stage;
    if (mine > 0) pid_next = pid_of(lane);
  };
  auto start = [&]() {
#pragma unroll 1
    for (int i = 0; i < min(mine, C::STAGES); ++i) issue();
  };
  // Row r of a segment: its token and its head in the group.
  auto row_of = [&](const Seg& sg, int r) {
    const int at = sg.head0 + r, n = (int)__umulhi(2u * at, a.by_g);
    return make_int2(sg.tok0 + n, at - n * a.G);
  };
  // The queries of the segment as they lie in memory: lane (g, t) takes row
  // g's columns D/4 * t ...
  uint32_t qw[NT][D / 8];
  auto load_q = [&]() {
#pragma unroll
    for (int n = 0; n < NT; ++n) {
#pragma unroll
      for (int i = 0; i < D / 8; ++i) qw[n][i] = 0;
      if (n * 8 + g < sg.nrows) {
        const int2 row = row_of(sg, n * 8 + g);
        const uint16_t* p = a.q + (int64_t)sg.b * a.qb + (int64_t)row.x * a.qt +
                            (int64_t)(sg.kvh * a.G + row.y) * a.qh + t * (D / 4);
#pragma unroll
        for (int i = 0; i < D / 32; ++i) {
          const uint4 v = __ldg(reinterpret_cast<const uint4*>(p) + i);
          qw[n][4 * i] = v.x, qw[n][4 * i + 1] = v.y, qw[n][4 * i + 2] = v.z, qw[n][4 * i + 3] = v.w;
        }
      }
    }
  };
  float o[NT][KS][4] = {};
  float mx[NT][2] = {}, sum[NT][2] = {}, wx[NT][2] = {};  // m, l, w of columns 2t, 2t + 1
  auto join = [&](const Seg& cur) {
  // ---- join the warps ----
  float* sums = reinterpret_cast<float*>(smem + C::SMEM_RING);  // [SUMS][ROWS][LD]
  float* sm = sums + C::SUMS * C::ROWS * C::LD;                 // [WARPS][ROWS] m, l, w
  float* sl = sm + WARPS * C::ROWS;
  float* sw = sl + WARPS * C::ROWS;
  float* fin = sw + WARPS * C::ROWS;                            // [ROWS] m, l, w, the output's factor
  const float factor = FP4 ? __ldg(a.v_scale + cur.kvh) : 1.0f;
  __syncthreads();  // the last join's readers are done
#pragma unroll
  for (int n = 0; n < NT; ++n)
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      float l = sum[n][c];
      l += __shfl_xor_sync(FULL, l, 4);
      l += __shfl_xor_sync(FULL, l, 8);
      l += __shfl_xor_sync(FULL, l, 16);
      if (FP4) l *= 1.0f / 32768.0f;  // sums of weights, which are 2^15 times the probabilities
      if (g == 0) {
        const int r = warp * C::ROWS + n * 8 + 2 * t + c;
        sm[r] = mx[n][c], sl[r] = l, sw[r] = wx[n][c];
      }
    }
  __syncthreads();
  if (threadIdx.x < C::ROWS) {
    float m = NEG_INF, w = NEG_INF, l = 0.0f;
#pragma unroll
    for (int k = 0; k < WARPS; ++k) {
      m = fmaxf(m, sm[k * C::ROWS + threadIdx.x]);
      w = fmaxf(w, sw[k * C::ROWS + threadIdx.x]);
    }
    const float ref = m == NEG_INF ? 0.0f : m;
#pragma unroll
    for (int k = 0; k < WARPS; ++k)
      l = fmaf(sl[k * C::ROWS + threadIdx.x], ex2(sm[k * C::ROWS + threadIdx.x] - ref), l);
    fin[threadIdx.x] = m, fin[C::ROWS + threadIdx.x] = l, fin[2 * C::ROWS + threadIdx.x] = w;
    fin[3 * C::ROWS + threadIdx.x] = (int)threadIdx.x < cur.nrows ? out_scale(m, l, w) * factor : 0.0f;
  }
  // every warp's O relative to the CTA's w, added in the warps' order.  Column
  // d = D/8 g + 2j + i of a row lies at place 16 j + 2 g + i of it: the lanes of
  // a store then meet no bank twice.
#pragma unroll
  for (int k = 0; k < WARPS / C::SUMS; ++k) {
    if (warp / C::SUMS == k) {
      float* dst = sums + (warp % C::SUMS) * C::ROWS * C::LD;
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          const int r = n * 8 + 2 * t + c;
          float w = sw[r];
#pragma unroll
          for (int q = 1; q < WARPS; ++q) w = fmaxf(w, sw[q * C::ROWS + r]);
          const float f = ex2(wx[n][c] - (w == NEG_INF ? 0.0f : w));
#pragma unroll
          for (int j = 0; j < KS; ++j) {
            float2* p = reinterpret_cast<float2*>(dst + r * C::LD + 16 * j + 2 * g);
            float2 v = k ? *p : make_float2(0.0f, 0.0f);
            v.x = fmaf(o[n][j][c], f, v.x);
            v.y = fmaf(o[n][j][c + 2], f, v.y);
            *p = v;
          }
        }
    }
    __syncthreads();
  }
  auto out_row = [&](int r) {
    const int2 row = row_of(cur, r);
    return a.out + (((int64_t)cur.b * a.T + row.x) * a.H + cur.kvh * a.G + row.y) * D;
  };
  if (cur.whole) {
    const int rows = min(C::ROWS, a.T * a.G - cur.row0);
    for (int i = threadIdx.x; i < rows * (D / 2); i += THREADS) {
      const int r = i / (D / 2), d = i % (D / 2) * 2;
      const float2* p = reinterpret_cast<const float2*>(sums + r * C::LD + d % (D / 8) * 8 + d / (D / 8) * 2);
      float2 v = *p;
      if (C::SUMS == 2) {
        const float2 u = p[C::ROWS * C::LD / 2];
        v.x += u.x, v.y += u.y;
      }
      const float f = fin[3 * C::ROWS + r];
      // a row without a query is 0 even where its sums are not finite
      *reinterpret_cast<uint32_t*>(out_row(r) + d) = r < cur.nrows ? bf_pack(v.x * f, v.y * f) : 0u;
    }
    return;
  }

  // ---- a piece of a head: [ROWS][D] of O in place order, then m, l and w ----
  float* piece_out = a.part + ((int64_t)blockIdx.x * 2 + cur.slot) * PART;
  for (int i = threadIdx.x; i < cur.nrows * (D / 4); i += THREADS) {
    const int r = i / (D / 4), d = i % (D / 4) * 4;
    const float4* p = reinterpret_cast<const float4*>(sums + r * C::LD + d);
    float4 v = *p;
    if (C::SUMS == 2) {
      const float4 u = p[C::ROWS * C::LD / 4];
      v.x += u.x, v.y += u.y, v.z += u.z, v.w += u.w;
    }
    reinterpret_cast<float4*>(piece_out)[i] = v;
  }
  if (threadIdx.x < 3 * C::ROWS) piece_out[C::ROWS * D + threadIdx.x] = fin[threadIdx.x];
  // the CTA that finishes last reads the head's pieces in the CTAs' order
  const int still = cur.units + HEAD - near_end - 1;  // the last place where a cut stays in the head
  const int c0 = run_of(cur.ps + min(HEAD, still)), c1 = run_of(cur.ps + still);
  const int pieces = c1 - c0 + 1;
  __syncthreads();
  if (threadIdx.x == 0) {
    int n;  // releases every thread's stores, which the barrier has ordered before it
    asm volatile("atom.add.acq_rel.gpu.global.s32 %0, [%1], 1;" : "=r"(n) : "l"(a.done + cur.pair) : "memory");
    s_last = n == pieces - 1;
  }
  __syncthreads();
  if (!s_last) return;
  const int slot0 = run_begin(c0) + near_end >= cur.ps ? 0 : 1;  // the first CTA's run may begin before the head
  auto piece = [&](int c) { return a.part + ((int64_t)(c0 + c) * 2 + (c == 0 ? slot0 : 0)) * PART; };
  // A group of D / 8 lanes takes a row, eight places a lane; where there are
  // groups enough, `split` of them share a row and take every split-th piece.
  // All loads of PRE pieces a group travel together.
  constexpr int LPR = D / 8, GROUPS = THREADS / LPR, PRE = C::PER_SM == 3 ? 4 : 8;
  const int gl = lane % LPR, grp = threadIdx.x / LPR;
  int log_split = 0;
  while ((cur.nrows << (log_split + 1)) <= GROUPS) ++log_split;
  const int split = 1 << log_split, sub = grp & (split - 1);
#pragma unroll 1
  for (int k = grp >> log_split; k - (grp >> log_split) < cur.nrows; k += GROUPS >> log_split) {
    const int r = min(k, cur.nrows - 1);  // beyond the last: that one again
    float4 pre[PRE][2];
    float pw[PRE];
    auto fetch = [&](int cb) {
#pragma unroll
      for (int q = 0; q < PRE; ++q) {
        const float* p = piece(min(cb + q * split, pieces - 1));
        const float4* o4 = reinterpret_cast<const float4*>(p + r * D) + gl;
        pre[q][0] = __ldcg(o4), pre[q][1] = __ldcg(o4 + LPR);
        pw[q] = __ldcg(p + C::ROWS * (D + 2) + r);
      }
    };
    fetch(sub);
    float m = NEG_INF, w = NEG_INF, l = 0.0f;
#pragma unroll 1
    for (int cb = gl; cb < pieces; cb += 4 * LPR) {
      float mc[4], lc[4];
      float mn = m;
#pragma unroll
      for (int q = 0; q < 4; ++q) {  // beyond the last: that one's maxima again, no sum
        const int c = cb + q * LPR;
        const float* p = piece(min(c, pieces - 1)) + C::ROWS * D + r;
        mc[q] = __ldcg(p), lc[q] = c < pieces ? __ldcg(p + C::ROWS) : 0.0f;
        w = fmaxf(w, __ldcg(p + 2 * C::ROWS));
      }
#pragma unroll
      for (int q = 0; q < 4; ++q) mn = fmaxf(mn, mc[q]);
      const float ref = mn == NEG_INF ? 0.0f : mn;
      l *= ex2(m - ref);
#pragma unroll
      for (int q = 0; q < 4; ++q) l = fmaf(lc[q], ex2(mc[q] - ref), l);
      m = mn;
    }
#pragma unroll
    for (int d = LPR / 2; d; d >>= 1) {
      const float m2 = __shfl_xor_sync(FULL, m, d), l2 = __shfl_xor_sync(FULL, l, d);
      const float mn = fmaxf(m, m2), ref = mn == NEG_INF ? 0.0f : mn;
      l = l * ex2(m - ref) + l2 * ex2(m2 - ref);
      m = mn;
      w = fmaxf(w, __shfl_xor_sync(FULL, w, d));
    }
    const float wr = w == NEG_INF ? 0.0f : w;
    float v[8] = {};
#pragma unroll 1
    for (int cb = sub; cb < pieces; cb += PRE * split) {
      if (cb != sub) fetch(cb);
#pragma unroll
      for (int q = 0; q < PRE; ++q)
        if (cb + q * split < pieces) {
          const float f = ex2(pw[q] - wr);
          const float4 x = pre[q][0], y = pre[q][1];
          v[0] = fmaf(x.x, f, v[0]), v[1] = fmaf(x.y, f, v[1]), v[2] = fmaf(x.z, f, v[2]);
          v[3] = fmaf(x.w, f, v[3]), v[4] = fmaf(y.x, f, v[4]), v[5] = fmaf(y.y, f, v[5]);
          v[6] = fmaf(y.z, f, v[6]), v[7] = fmaf(y.w, f, v[7]);
        }
    }
    if (split > 1) {  // one round; the sums' readers are past the barriers above
      float4* mine = reinterpret_cast<float4*>(sums) + threadIdx.x;
      mine[0] = make_float4(v[0], v[1], v[2], v[3]);
      mine[THREADS] = make_float4(v[4], v[5], v[6], v[7]);
      __syncthreads();
      if (sub == 0) {
#pragma unroll 1
        for (int q = 1; q < split; ++q) {
          const float4 x = mine[q * LPR], y = mine[THREADS + q * LPR];
          v[0] += x.x, v[1] += x.y, v[2] += x.z, v[3] += x.w;
          v[4] += y.x, v[5] += y.y, v[6] += y.z, v[7] += y.w;
        }
      }
    }
    if (sub == 0) {
      const float f = out_scale(m, l, w) * factor;
      // places 4 gl .. and D/2 + 4 gl ..: columns D/8 g2 + 2j of g2 = 2 gl % 8
      // and the next, j = gl / 4 and D/32 more
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int j = gl / 4 + h * (D / 32), g2 = 2 * gl % 8;
        uint16_t* p = out_row(r) + g2 * (D / 8) + 2 * j;
        *reinterpret_cast<uint32_t*>(p) = bf_pack(v[4 * h] * f, v[4 * h + 1] * f);
        *reinterpret_cast<uint32_t*>(p + D / 8) = bf_pack(v[4 * h + 2] * f, v[4 * h + 3] * f);
      }
    }
  }
  // rows of the group that have no query
  const int blank = min(C::ROWS, a.T * a.G - cur.row0) - cur.nrows;
  for (int i = threadIdx.x; i < blank * (D / 2); i += THREADS)
    reinterpret_cast<uint32_t*>(out_row(cur.nrows + i / (D / 2)))[i % (D / 2)] = 0u;
  if (threadIdx.x == 0) a.done[cur.pair] = 0;
  };
  for (bool done = false;; done = true) {
  const Seg cur = sg;
  const bool more = pos < hi;
  if (more) {  // its loads run under the join
    open();
    start();
    load_q();
  }
  if (done) {
    join(cur);
  } else {
    // row groups without a query are written here: no unit belongs to them
#pragma unroll 1
    for (int e = blockIdx.x; e < entries; e += gridDim.x) {
      const Entry x = entry(e);
      if (x.nrows > 0) continue;
      const int rows = min(C::ROWS, a.T * a.G - x.row0);
      for (int i = threadIdx.x; i < rows * a.Hkv * (D / 8); i += THREADS) {
        const int row = x.row0 + i / (D / 8) % rows, h = i / (D / 8) / rows;
        reinterpret_cast<uint4*>(a.out + (((int64_t)x.b * a.T + row / a.G) * a.H + h * a.G + row % a.G) * D)
            [i % (D / 8)] = make_uint4(0, 0, 0, 0);
      }
    }
  }
  if (!more) break;
  const int held = sg.held, end = sg.end, k0 = sg.k0;

  const float sm_head = FP4 ? a.sm_log2 * __ldg(a.k_scale + sg.kvh) : a.sm_log2;
  // Q as the second operand of S^T = K Q^T: k step w takes the lane's 4
  // columns D/4 * t + 4 w ...
  uint32_t qf[NT][KS][2];
  float qs[NT];  // the power of two taken out of row g's query
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < D / 8; ++i) {
      const uint32_t v = qw[n][i] & 0x7FFF7FFFu;
      m = max(m, max(v & 0xFFFFu, v >> 16));
    }
    m = max(m, __shfl_xor_sync(FULL, m, 1));
    m = max(m, __shfl_xor_sync(FULL, m, 2));
    const int e = min(max((int)(m >> 7), 15), 253);  // the largest value's exponent field
    float up = __uint_as_float((uint32_t)(254 + 14 - e) << 23);
    if (FP4) up = copysignf(up, sm_head);  // a negative scale turns the query
    qs[n] = __uint_as_float((uint32_t)(e - 14) << 23);
#pragma unroll
    for (int i = 0; i < D / 8; ++i)
      qf[n][i >> 1][i & 1] = f16x2(bf_lo(qw[n][i]) * up, bf_hi(qw[n][i]) * up);
  }
  // for the scores' columns 2t, 2t + 1 of each row tile: the query's factor
  // and the last key the row sees (rows without a query are not written)
  float cs[NT][2];
  int lim[NT][2];
#pragma unroll
  for (int n = 0; n < NT; ++n)
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      cs[n][c] = __shfl_sync(FULL, qs[n], (2 * t + c) * 4) * (FP4 ? fabsf(sm_head) : sm_head);
      // never 0, so that a masked score stays -infinity; NaN stays
      if (FP4 && cs[n][c] < 1.17549435e-38f) cs[n][c] = 1.17549435e-38f;
      lim[n][c] = held + row_of(sg, n * 8 + 2 * t + c).x;
    }
  const int free_end = held + sg.tok0 + 1;  // keys below: every row sees them

#pragma unroll
  for (int n = 0; n < NT; ++n) {
#pragma unroll
    for (int j = 0; j < KS; ++j) o[n][j][0] = o[n][j][1] = o[n][j][2] = o[n][j][3] = 0.0f;
    mx[n][0] = mx[n][1] = wx[n][0] = wx[n][1] = NEG_INF;
    sum[n][0] = sum[n][1] = 0.0f;
  }

  int i = 0;
  int nan_key = 0x7FFFFFFF;  // in 4 bits: the first key whose values in this lane's block are NaN
  auto advance = [&]() {
    __syncwarp();  // every lane has read the stage
    if (issued < mine) issue();
    if (++stage == C::STAGES) stage = 0, phase ^= 1;
  };
  for (; i < mine; ++i, advance()) {
    const int key0 = k0 + (warp + i * WARPS) * TILE;
    if (!FP4 && (i & 31) == 0) c_ks = n_ks, c_lv = log2f(n_v);
    const float ks = FP4 ? 1.0f : __shfl_sync(FULL, c_ks, i & 31), lv = FP4 ? 0.0f : __shfl_sync(FULL, c_lv, i & 31);
    ok = mbar_wait_warp(bar0 + 8 * stage, phase, nullptr, ERR_WAIT);
    if (!ok) break;
    if (FP4 ? skip >> stage & 1u : lv != lv) {  // a page outside the cache
      skip &= ~(1u << stage);
      continue;
    }
    const uint32_t kb = ring + stage * C::STAGE, vb = kb + C::TILE_BYTES;
    // the key that index r of the products stands for
    auto place = [](int r) { return FP4 ? key4(r) : r; };
    const bool tail = key0 + TILE > free_end;

    // scores: two m tiles of 16 keys
    float s[NT][2][4];
#pragma unroll
    for (int mt = 0; mt < 2; ++mt) {
#pragma unroll
      for (int n = 0; n < NT; ++n) s[n][mt][0] = s[n][mt][1] = s[n][mt][2] = s[n][mt][3] = 0.0f;
      const int r = mt * 16 + place(g);
      if constexpr (FP4) {
        // rows r and r + 8 of the tile, D / 4 columns, in D / 64 blocks of 16
        uint32_t x[D / 32], y[D / 32], sx[D / 64], sy[D / 64];
        const uint32_t ka = kb + at_k + mt * (16 * D / 2), kc = kb + at_ks + mt * D;  // 8 rows on: half of that
        if constexpr (D == 128) {
          const uint4 p = lds128(ka), q = lds128(ka + 512);
          x[0] = p.x, x[1] = p.y, x[D / 32 - 2] = p.z, x[D / 32 - 1] = p.w;
          y[0] = q.x, y[1] = q.y, y[D / 32 - 2] = q.z, y[D / 32 - 1] = q.w;
          const uint32_t u = unpack2(lds16(kc)), w = unpack2(lds16(kc + 64));
          sx[0] = __byte_perm(u, u, 0x1010), sx[D / 64 - 1] = __byte_perm(u, u, 0x3232);
          sy[0] = __byte_perm(w, w, 0x1010), sy[D / 64 - 1] = __byte_perm(w, w, 0x3232);
        } else {
          const uint2 p = lds64(ka), q = lds64(ka + 256);
          x[0] = p.x, x[1] = p.y, y[0] = q.x, y[1] = q.y;
          sx[0] = unpack2(lds8(kc) * 0x0101u), sy[0] = unpack2(lds8(kc + 32) * 0x0101u);
        }
#pragma unroll
        for (int w = 0; w < D / 32; ++w) {
          uint32_t hx[4], hy[4];
          e2m1_f16(x[w], hx);
          e2m1_f16(y[w], hy);
#pragma unroll
          for (int j = 0; j < 4; ++j) hx[j] = mul_f16x2(hx[j], sx[w >> 1]), hy[j] = mul_f16x2(hy[j], sy[w >> 1]);
#pragma unroll
          for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int n = 0; n < NT; ++n)
              mma(s[n][mt], hx[2 * j], hy[2 * j], hx[2 * j + 1], hy[2 * j + 1], qf[n][2 * w + j][0], qf[n][2 * w + j][1]);
        }
      } else {
        uint32_t ka[D / 16], kc[D / 16];  // rows g and g + 8 of the tile, D / 4 columns
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
    }

    // running maxima and sum; P^T as the second operand of the output
    uint32_t pf[NT][2][2];
    float corr[NT][2];
    bool grew = false;
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      if constexpr (FP4) {
        // One page's values weigh as another's: w is m, the weights are their sum's terms.
        // The lanes of a column meet only where one of them has found a larger score.
        if (tail) {
#pragma unroll
          for (int mt = 0; mt < 2; ++mt) {
            const int key = key0 + mt * 16 + place(g);
            if (key > lim[n][0]) s[n][mt][0] = NEG_INF;
            if (key > lim[n][1]) s[n][mt][1] = NEG_INF;
            if (key + 8 > lim[n][0]) s[n][mt][2] = NEG_INF;
            if (key + 8 > lim[n][1]) s[n][mt][3] = NEG_INF;
          }
        }
        float top[2];
#pragma unroll
        for (int c = 0; c < 2; ++c)  // cs > 0: -infinity stays
          top[c] = fmaxf(fmaxf(s[n][0][c], s[n][0][c + 2]), fmaxf(s[n][1][c], s[n][1][c + 2])) * cs[n][c];
        corr[n][0] = corr[n][1] = 1.0f;
        if (__any_sync(FULL, top[0] > mx[n][0] || top[1] > mx[n][1])) {
          grew = true;
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            float m = fmaxf(top[c], __shfl_xor_sync(FULL, top[c], 4));
            m = fmaxf(m, __shfl_xor_sync(FULL, m, 8));
            m = fmaxf(fmaxf(m, __shfl_xor_sync(FULL, m, 16)), mx[n][c]);
            corr[n][c] = m == NEG_INF ? 1.0f : ex2(mx[n][c] - m);
            mx[n][c] = wx[n][c] = m;
            sum[n][c] *= corr[n][c];
          }
        }
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          const float bias = P_EXP - (mx[n][c] == NEG_INF ? 0.0f : mx[n][c]);
#pragma unroll
          for (int mt = 0; mt < 2; ++mt) {
            s[n][mt][c] = ex2(fmaf(s[n][mt][c], cs[n][c], bias));
            s[n][mt][c + 2] = ex2(fmaf(s[n][mt][c + 2], cs[n][c], bias));
          }
          sum[n][c] += (s[n][0][c] + s[n][0][c + 2]) + (s[n][1][c] + s[n][1][c + 2]);
        }
      } else {
        const float f0 = cs[n][0] * ks, f1 = cs[n][1] * ks;
#pragma unroll
        for (int mt = 0; mt < 2; ++mt) {
          s[n][mt][0] *= f0, s[n][mt][2] *= f0;
          s[n][mt][1] *= f1, s[n][mt][3] *= f1;
          if (tail) {
            const int key = key0 + mt * 16 + place(g);
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
      }
#pragma unroll
      for (int mt = 0; mt < 2; ++mt) {
        pf[n][mt][0] = transpose8x8(f16x2(s[n][mt][0], s[n][mt][1]));
        pf[n][mt][1] = transpose8x8(f16x2(s[n][mt][2], s[n][mt][3]));
      }
    }
    if (FP4 ? grew : __any_sync(FULL, grew)) {
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
    if constexpr (FP4) {
      constexpr int VW = D / 64;  // words of D / 8 columns
      // the pairs of keys (2t, 2t+1) and (2t+8, 2t+9): words whose bytes are one
      // column's two codes, even columns and odd, and the two scales
      uint32_t ev[2][2][VW], od[2][2][VW], sp[2][2];
      uint32_t odd = 0;
#pragma unroll
      for (int mt = 0; mt < 2; ++mt)
#pragma unroll
        for (int p = 0; p < 2; ++p) {
          const int r0 = mt * 16 + p * 8 + key4(2 * t), r1 = mt * 16 + p * 8 + key4(2 * t + 1);
          uint32_t x[VW], y[VW], e0, e1;
          const uint32_t on = (mt * 16 + p * 8) * (D / 2), ons = on / 8;
          if constexpr (D == 128) {
            const uint2 u = lds64(kb + at_v0 + on), w = lds64(kb + at_v1 + on);
            x[0] = u.x, x[VW - 1] = u.y, y[0] = w.x, y[VW - 1] = w.y;
          } else {
            x[0] = lds32(kb + at_v0 + on), y[0] = lds32(kb + at_v1 + on);
          }
          e0 = lds8(kb + at_vs0 + ons), e1 = lds8(kb + at_vs1 + ons);
          if (tail) {
            if (key0 + r0 >= end) e0 = 0;  // slots that hold no token of this sequence
            if (key0 + r1 >= end) e1 = 0;
          }
          sp[mt][p] = e0 | e1 << 8;
          if (tail) odd |= nan_bits(sp[mt][p]);
#pragma unroll
          for (int w = 0; w < VW; ++w) {
            ev[mt][p][w] = (x[w] & 0x0F0F0F0Fu) | (y[w] << 4 & 0xF0F0F0F0u);
            od[mt][p][w] = (x[w] >> 4 & 0x0F0F0F0Fu) | (y[w] & 0xF0F0F0F0u);
          }
        }
      // 0 * NaN is NaN, also for a row that may not see the value: where rows differ in
      // what they see a NaN enters as 0, its key is noted, and the rows that see it get
      // NaN at the segment's end
      if (tail && (odd & 0x8080u)) {
#pragma unroll
        for (int q = 0; q < 8; ++q)
          if ((sp[q >> 2][q >> 1 & 1] >> (8 * (q & 1)) & 0x7Fu) == 0x7Fu) {
            nan_key = min(nan_key, key0 + (q >> 2) * 16 + (q >> 1 & 1) * 8 + key4(2 * t + (q & 1)));
            sp[q >> 2][q >> 1 & 1] &= ~(0xFFu << (8 * (q & 1)));
          }
      }
#pragma unroll
      for (int mt = 0; mt < 2; ++mt) {
        const uint32_t s0 = unpack2(sp[mt][0]), s1 = unpack2(sp[mt][1]);
#pragma unroll
        for (int w = 0; w < VW; ++w) {
          uint32_t a0[4], a1[4], a2[4], a3[4];
          e2m1_f16(ev[mt][0][w], a0), e2m1_f16(od[mt][0][w], a1), e2m1_f16(ev[mt][1][w], a2), e2m1_f16(od[mt][1][w], a3);
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            a0[j] = mul_f16x2(a0[j], s0), a1[j] = mul_f16x2(a1[j], s0);
            a2[j] = mul_f16x2(a2[j], s1), a3[j] = mul_f16x2(a3[j], s1);
#pragma unroll
            for (int n = 0; n < NT; ++n) mma(o[n][4 * w + j], a0[j], a1[j], a2[j], a3[j], pf[n][mt][0], pf[n][mt][1]);
          }
        }
      }
      continue;
    }
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
            odd |= nan_bits(v[mt][k][w]);
          }
        }
      odd = __any_sync(FULL, (odd & 0x80808080u) != 0);
    }
    if (!odd) {
#pragma unroll
      for (int j = 0; j < KS; ++j)
#pragma unroll
        for (int n = 0; n < NT; ++n) product(n, j, v, o[n][j]);
    } else {
      // 0 * NaN is NaN, also for a row that may not see the value: each row
      // gets a product of its own with the values it does not see taken as 0
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll 1
        for (int r = 0; r < 8; ++r) {
          const int last = held + row_of(sg, n * 8 + r).x;
          uint32_t x[2][4][VW];
#pragma unroll
          for (int mt = 0; mt < 2; ++mt)
#pragma unroll
            for (int k = 0; k < 4; ++k)
#pragma unroll
              for (int w = 0; w < VW; ++w)
                x[mt][k][w] =
                    key0 + mt * 16 + 2 * t + (k & 1) + (k >> 1) * 8 > last ? 0u : v[mt][k][w];
          const bool c0 = r == 2 * t, c1 = r == 2 * t + 1;
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
  if (FP4) {
    nan_key = min(nan_key, __shfl_xor_sync(FULL, nan_key, 1));
    nan_key = min(nan_key, __shfl_xor_sync(FULL, nan_key, 2));
    if (nan_key != 0x7FFFFFFF) {
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int c = 0; c < 2; ++c)
          if (nan_key <= lim[n][c])
#pragma unroll
            for (int j = 0; j < KS; ++j) o[n][j][c] = o[n][j][c + 2] = __uint_as_float(0x7FC00000u);
    }
  }
  // after a wait that gave up: the loads in flight land before the ring is reused
  for (; i < issued; ++i) {
    mbar_wait(bar0 + 8 * stage, phase, nullptr, ERR_WAIT);
    if (++stage == C::STAGES) stage = 0, phase ^= 1;
  }

  }
}

// A cache of no pages or a block table of no columns: no row sees a key.  The
// output is 0 and the plan is checked as ever.
__global__ void __launch_bounds__(THREADS) k_attn_none(const __grid_constant__ Args a, int64_t chunks) {
  pdl::trigger();
  pdl::wait();
  const int64_t first = (int64_t)blockIdx.x * THREADS + threadIdx.x, step = (int64_t)gridDim.x * THREADS;
  for (int64_t i = first; i < chunks; i += step) reinterpret_cast<uint4*>(a.out)[i] = make_uint4(0, 0, 0, 0);
  for (int64_t b = first; b < a.B; b += step) {
    int err = 0;
    const int2 plan = plan_of(a, (int)b, err);
    if (!err && plan.y > 0) err = ERR_PAGE;  // tokens, but no page to hold them
    if (err) note_err(nullptr, err);
  }
}

// The longest block table: its keys, and the 2^14 beyond them that the batches
// read ahead may name before they are brought back to the last, fit 31 bits.
constexpr int64_t max_width(int32_t page) { return ((1ll << 31) - (1 << 14)) / page; }

// How a call's work is cut: row tiles of 8, row groups, and CTAs: as many as
// fit at once, or one per unit where the longest lengths give fewer.
struct Cut {
  int nt, groups, ctas;
};
Cut cut_of(int64_t batch, int64_t tokens, int heads, int kv_heads, int head_dim, int64_t capacity, bool fp4) {
  Cut c;
  // Row tiles per group: two.  Three, which fit the registers at heads of 64,
  // where the tiles come out even (96 rows: 120 us against 129, 24 rows 48
  // against 55; 35 rows would take 32 against 26).
  const int64_t tiles = (tokens * (heads / kv_heads) + 7) / 8;
  const int64_t most = head_dim == 64 && tiles % 3 == 0 ? 3 : 2;
  c.groups = (int)((tiles + most - 1) / most);
  c.nt = (int)((tiles + c.groups - 1) / c.groups);
  const int64_t units = std::max<int64_t>(1, (capacity + UNIT - 1) / UNIT);
  c.ctas = (int)std::min<int64_t>(ctas_per_sm(head_dim, c.nt, fp4) * vq::mx::sm_count(), batch * c.groups * kv_heads * units);
  return c;
}

template <int D, int NT, bool FP4>
int launch(const CUtensorMap& mk, const CUtensorMap& mv, const Args& a, int ctas, cudaStream_t st) {
  using C = Cfg<D, NT, FP4>;
  static_assert(WARPS * C::STAGES * 8 <= 256, "barrier area");
  if (!allow_smem<k_attn_kv<D, NT, FP4>>(C::SMEM))
    return VQ_ERR_CUDA;
  return pdl::launch<k_attn_kv<D, NT, FP4>>(ctas, THREADS, C::SMEM, st, 1, mk, mv, a) ? VQ_OK : VQ_ERR_CUDA;
}

int sticky_kva(int* out, int clear, cudaStream_t st) { return vq::tc::sticky_read(out, clear, st); }

}  // namespace kva
}  // namespace vq

using namespace vq::kva;

// Whether a call on the 4-bit cache is this file's, or vq_attn_kv4.cu's.  There a
// tile of 128 keys costs the same for 1 to 128 rows a kv head, here once for every
// group of 16; the start there costs about 10 us more, and heads cost more.  The host
// knows the table's width only, so that t is the tiles of sequences that fill it; where
// lengths lie evenly below that, about half of them are there.  With h heads (sequences
// x kv heads), g groups of 16 rows, here / there in us:
//                                        equal lengths   unequal
//   D = 128  48 rows,  h 128, t 2048        54 / 44       33 / 36
//                      h 32,  t 4032        80 / 61       40 / 44
//                      h 512, t 4096       107 / 84       57 / 86
//            128 rows, h 32,  t 256         30 / 31       20 / 29
//                      h 32,  t 1024        61 / 40       32 / 37
//                      h 512, t 4096       259 / 90       98 / 82
//   D = 64   35 rows,  h 24,  t 3768        56 / 50       25 / 40
//            48 rows,  h 32,  t 4032        54 / 50       32 / 37
//            128 rows, h 32,  t 1024        45 / 30       25 / 27
// Over 400 such points the choice costs 4 % on average, and half at the worst, where lengths
// are unlike what the width says.  Up to 32 rows always run here, more than 128 never.
static bool few_rows(int64_t batch, int64_t rows, int kv_heads, int head_dim, int64_t capacity) {
  const int64_t g = (rows + 15) / 16, h = batch * kv_heads, t = h * ((capacity + 127) / 128);
  return g <= 8 && (head_dim == 64 ? t * (4 * g - 11) <= 6000 : t * (4 * g - 10) <= 6400 + 4 * h);
}

static int workspace(int64_t batch, int64_t tokens, int32_t heads, int32_t kv_heads, int32_t head_dim, int32_t page,
                     int64_t table_width, int64_t* floats, int64_t* counters, bool fp4) {
  if (!floats || !counters) return VQ_ERR_NULL;
  if (batch < 0 || tokens < 0 || kv_heads <= 0 || heads <= 0 || heads % kv_heads || head_dim <= 0 ||
      page <= 0 || table_width < 0 || table_width > max_width(page))
    return VQ_ERR_INVALID;
  if (fp4 && !few_rows(batch, tokens * (heads / kv_heads), kv_heads, head_dim, table_width * page)) {
    *floats = vq::kv4::workspace(batch, tokens, heads, kv_heads, head_dim, table_width * page);
    *counters = 0;
    return VQ_OK;
  }
  const Cut c = cut_of(std::max<int64_t>(batch, 1), std::max<int64_t>(tokens, 1), heads, kv_heads,
                       head_dim, table_width * page, fp4);
  *counters = batch * kv_heads * c.groups;
  *floats = (int64_t)c.ctas * 2 * 8 * c.nt * (head_dim + 3);
  return VQ_OK;
}

// In E4M3 k_scale and v_scale are float32 per page and head; in 4 bits the
// bytes of a block each, and k_factor and v_factor float32 per head.
static int attention(const void* q, const int64_t* q_strides, int64_t batch, int64_t tokens, int32_t heads,
                     int32_t kv_heads, int32_t head_dim, const void* k_codes, const void* v_codes,
                     const void* k_scale, const void* v_scale, const float* k_factor, const float* v_factor,
                     int64_t pages, int32_t page, const void* block_table, int64_t table_width, const void* lengths,
                     const void* counts, float sm_scale, float* workspace, int64_t workspace_floats,
                     int32_t* counters, int64_t counters_len, void* out, void* stream, bool fp4) {
  if (head_dim != 64 && head_dim != 128) return VQ_ERR_UNSUPPORTED;
  if (page != 32 && page != 64 && page != 128) return VQ_ERR_UNSUPPORTED;
  if (batch < 0 || tokens < 0 || heads <= 0 || kv_heads <= 0 || heads % kv_heads || table_width < 0 ||
      pages < 0 || pages * kv_heads * page >= (1ll << 31) || table_width > max_width(page) ||
      tokens >= (1 << 20) || batch > (1 << 24) || batch * tokens * heads >= (1ll << 31) || heads / kv_heads > (1 << 15))
    return VQ_ERR_INVALID;
  if (batch == 0 || tokens == 0) return VQ_OK;
  Args a;
  a.out = (uint16_t*)out;
  a.lengths = (const int32_t*)lengths;
  a.counts = (const int32_t*)counts;
  a.B = (int)batch, a.T = (int)tokens, a.H = heads, a.Hkv = kv_heads, a.G = heads / kv_heads;
  a.page_log2 = page == 32 ? 5 : page == 64 ? 6 : 7;
  a.width = (int)table_width, a.pages = (int)pages;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  if (pages == 0 || table_width == 0) {  // nothing to read: their pointers may be null
    if (!lengths || !out) return VQ_ERR_NULL;
    if (reinterpret_cast<uintptr_t>(out) & 15) return VQ_ERR_ALIGNMENT;
    const int64_t chunks = batch * tokens * heads * (head_dim / 8);
    const int64_t ctas = std::min<int64_t>((chunks + THREADS - 1) / THREADS, 8 * vq::mx::sm_count());
    return vq::pdl::launch<k_attn_none>((unsigned)ctas, THREADS, 0, st, 1, a, chunks) ? VQ_OK : VQ_ERR_CUDA;
  }
  const bool few = !fp4 || few_rows(batch, tokens * a.G, kv_heads, head_dim, table_width * page);
  if (!q || !q_strides || !k_codes || !v_codes || !k_scale || !v_scale || !block_table || !lengths ||
      (few && !counters) || !out || (fp4 && (!k_factor || !v_factor)))
    return VQ_ERR_NULL;
  const void* p16[7] = {q, k_codes, v_codes, out, workspace, fp4 ? k_scale : nullptr, fp4 ? v_scale : nullptr};
  for (const void* p : p16)
    if (reinterpret_cast<uintptr_t>(p) & 15) return VQ_ERR_ALIGNMENT;
  if (fp4 && (reinterpret_cast<uintptr_t>(out) & 31)) return VQ_ERR_ALIGNMENT;
  for (int i = 0; i < 3; ++i)
    if (q_strides[i] % 8) return VQ_ERR_ALIGNMENT;
  if (!few)
    return vq::kv4::attend(q, q_strides, batch, tokens, heads, kv_heads, head_dim, k_codes, v_codes, k_scale, v_scale,
                           k_factor, v_factor, pages, page, block_table, table_width, lengths, counts, sm_scale,
                           workspace, workspace_floats, out, st);
  const Cut c = cut_of(batch, tokens, heads, kv_heads, head_dim, table_width * page, fp4);
  const int64_t pairs = batch * kv_heads * c.groups;
  // the units of all heads, counted in 32 bits
  if (pairs * ((table_width * page + UNIT - 1) / UNIT + 8) >= (1ll << 31) || counters_len < pairs)
    return VQ_ERR_INVALID;
  if (!workspace || workspace_floats < (int64_t)c.ctas * 2 * 8 * c.nt * (head_dim + 3)) return VQ_ERR_INVALID;
  CUtensorMap mk, mv;
  const uint64_t rows = (uint64_t)pages * kv_heads * page;
  if (fp4)
    mk = mv = {};  // not used
  else if (!vq::mx::make_map_box(&mk, k_codes, rows, head_dim, head_dim, TILE, head_dim) ||
           !vq::mx::make_map_box(&mv, v_codes, rows, head_dim, head_dim, TILE, head_dim))
    return VQ_ERR_CUDA;
  a.k_codes = fp4 ? (const uint8_t*)k_codes : nullptr, a.v_codes = fp4 ? (const uint8_t*)v_codes : nullptr;
  a.q = (const uint16_t*)q;
  a.qb = q_strides[0], a.qt = q_strides[1], a.qh = q_strides[2];
  a.k_scale = fp4 ? k_factor : (const float*)k_scale, a.v_scale = fp4 ? v_factor : (const float*)v_scale;
  a.k_bscale = fp4 ? (const uint8_t*)k_scale : nullptr, a.v_bscale = fp4 ? (const uint8_t*)v_scale : nullptr;
  a.block_table = (const int32_t*)block_table;
  a.part = workspace;
  a.done = counters;
  a.groups = c.groups;
  a.by_g = (uint32_t)(((1ll << 31) + a.G - 1) / a.G);
  a.sm_log2 = sm_scale * 1.4426950408889634f;
  auto run = [&](auto four) {
    constexpr bool F = decltype(four)::value;
    if (head_dim == 128)
      return c.nt == 1 ? launch<128, 1, F>(mk, mv, a, c.ctas, st) : launch<128, 2, F>(mk, mv, a, c.ctas, st);
    return c.nt == 1   ? launch<64, 1, F>(mk, mv, a, c.ctas, st)
           : c.nt == 2 ? launch<64, 2, F>(mk, mv, a, c.ctas, st)
                       : launch<64, 3, F>(mk, mv, a, c.ctas, st);
  };
  return fp4 ? run(std::true_type()) : run(std::false_type());
}

extern "C" {

int vq_attn_kv8_workspace(int64_t batch, int64_t tokens, int32_t heads, int32_t kv_heads,
                          int32_t head_dim, int32_t page, int64_t table_width, int64_t* floats,
                          int64_t* counters) {
  return workspace(batch, tokens, heads, kv_heads, head_dim, page, table_width, floats, counters, false);
}
int vq_attn_kv4_workspace(int64_t batch, int64_t tokens, int32_t heads, int32_t kv_heads,
                          int32_t head_dim, int32_t page, int64_t table_width, int64_t* floats,
                          int64_t* counters) {
  return workspace(batch, tokens, heads, kv_heads, head_dim, page, table_width, floats, counters, true);
}

int vq_attn_kv8(const void* q, const int64_t* q_strides, int64_t batch, int64_t tokens, int32_t heads,
                int32_t kv_heads, int32_t head_dim, const void* k_codes, const void* v_codes,
                const float* k_scale, const float* v_scale, int64_t pages, int32_t page,
                const void* block_table, int64_t table_width, const void* lengths, const void* counts,
                float sm_scale, float* workspace, int64_t workspace_floats, int32_t* counters,
                int64_t counters_len, void* out, void* stream) {
  return attention(q, q_strides, batch, tokens, heads, kv_heads, head_dim, k_codes, v_codes, k_scale, v_scale, nullptr,
                   nullptr, pages, page, block_table, table_width, lengths, counts, sm_scale, workspace,
                   workspace_floats, counters, counters_len, out, stream, false);
}

int vq_attn_kv4(const void* q, const int64_t* q_strides, int64_t batch, int64_t tokens, int32_t heads,
                int32_t kv_heads, int32_t head_dim, const void* k_codes, const void* v_codes,
                const void* k_scale, const void* v_scale, const float* k_factor, const float* v_factor,
                int64_t pages, int32_t page, const void* block_table, int64_t table_width, const void* lengths,
                const void* counts, float sm_scale, float* workspace, int64_t workspace_floats,
                int32_t* counters, int64_t counters_len, void* out, void* stream) {
  return attention(q, q_strides, batch, tokens, heads, kv_heads, head_dim, k_codes, v_codes, k_scale, v_scale,
                   k_factor, v_factor, pages, page, block_table, table_width, lengths, counts, sm_scale, workspace,
                   workspace_floats, counters, counters_len, out, stream, true);
}

}  // extern "C"
