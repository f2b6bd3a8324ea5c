// Attention of many query rows over the paged 4-bit key / value cache: prompts,
// pieces of prompts, and drafts of many rows a kv head (vq_attn_kv.cu's
// few_rows() says from where on).
//
//   o[b, t, h] = sum_j softmax_j(q . k_j * sm_scale) v_j,  j <= held[b] + t,
//   k_j = code * scale * factor, v_j likewise (vq_rope_append_kv4's cache)
//
// The T tokens and the G query heads that share a kv head are the rows of one
// product: row r = t * G + g.
//
// Mathematics: S = Q K^T and O += P V on tcgen05 in f16, float32 accumulators in
// tensor memory.  code * scale has at most 6 significant bits within 2^-10 ..
// 2688, so a cache tile is exact in f16; q is scaled per row by a power of two to
// a largest value of 2^14 .. 2^15, so that f16 holds every bf16 down to 2^-31 of
// it exactly.  Scores are base-2 exponents s (float32); P = 2^(s - m + 11) in f16,
// m a running reference that is at most 4 below the row's maximum: P <= 2^15, and
// O is scaled anew only where the maximum has left m by more than that.  A weight's
// relative error is 2^-11 down to 2^-25 of the largest, below it is off by at most
// 2^-36 of the largest (vq_attn_kv.cu's: 2^-29 and 2^-40).
// l = sum of the unrounded P in float32; the output is O / l * factor of V.
//
// A value whose scale is NaN enters the product as 0, and the smallest key of each
// block of 16 columns that has one is noted: the rows that see it get NaN there at
// the end, the others nothing (0 * NaN would reach every row of the tile).
//
// Work: two streams of 128 rows, each with a warpgroup for its softmax (a thread
// is a row) and its own S and O in tensor memory.  PAIR: the streams are 256 rows
// of a head and share the keys.  Otherwise a head has at most 128 rows: both
// streams have them and take every other tile of keys; their sums meet in shared
// memory.  A tile of 128 keys goes in two halves of 64: S of a half is asked for
// as soon as the weights in its place have been used, so that while one half is in
// the softmax the tensor cores have the stream's other half and the other stream.
// P lies in place of its half of S and is the second product's first operand.
//
// Warps: eight of softmax; four turn K and four V from codes to f16 in shared
// memory, in the SWIZZLE_128B layout that serves K as K-major and V as MN-major
// operand (a tile's codes travel to registers while its buffer is still in use);
// one a stream issues its MMAs, so that neither stream waits for the other's weights;
// one looks up where the tiles lie, some ahead, and asks for their lines in L2.  The
// softmax needs 144 registers, the conversion 56.
//
// The tiles of every (sequence, row tile, kv head) lie end to end and are cut into
// equal runs, one per CTA, one CTA per SM; the pieces of a head that was cut are
// joined by the CTA that finishes last, in the CTAs' order.  With many heads of
// PAIR rows, where the CTAs idle for less than a cut costs, they are not cut: a CTA
// takes the next one off a counter, the long ones first.
//
// Bound by the softmax warps' own chain, 2100 cycles a half tile: 200 to find the scores
// there, 420 to read them and their maximum, 1250 for the weights (the exponentials'
// unit is shared by the streams' warps, 1024 at its rate), 250 to store and hand over;
// the tensor pipe has 1024 of work in that time (S at N = 64 reads the queries anew for
// every half, 6 KB an MMA).  Slower were, on forms that took 187 to 193 us for the 500
// tokens below: sixteen warps of softmax at 88 registers (208), the next half's scores
// read under this one's weights (212: spills), weights of the two streams in turn (193
// against 187), whole tiles.  Pairs of CTAs (cta_group::2) would share the conversion of a
// tile; not built.  500 tokens x 5 heads on 16011 held, 8 kv heads of 128: 184 us in short
// runs, 905 TFLOP/s (193 over and over); 4 prompts of 2048 tokens, 8 x 4 heads: 192 us, 716;
// 25 tokens x 4 heads on 8 x 16000 (two streams of one row tile): 96 us, 545.  Few tiles:
// start, ends and joins, about 22 us.
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <algorithm>

#include "voyager_b200.h"
#include "vq_e4m3.cuh"
#include "vq_pdl.cuh"
#include "vq_tc.cuh"

namespace vq {
namespace kv4 {

using namespace vq::e4;
using namespace vq::tc;

enum { ERR_WAIT = 331, ERR_PAGE = 332, ERR_CAPACITY = 333, ERR_COUNT = 334 };

constexpr int TILE = 128;  // keys
constexpr int PLANS = 128;
// warps: 0-7 softmax (a stream's four each), 8-11 K and 12-15 V from codes to f16, 16 and 18 the streams' MMAs, 17
// where the tiles lie, 19 none (a warpgroup's registers are split together)
constexpr int SM_WARPS = 8, W_DQ = 8, W_MMA = 16, W_SCOUT = 17, WARPS = 20, THREADS = WARPS * 32;
// registers a thread: launched with 96; a warpgroup of 4 warps gives some up or takes them
constexpr int R_LAUNCH = 96, R_SOFT = 144, R_DQ = 56, R_REST = 80;
static_assert(2 * R_SOFT + 2 * R_DQ + R_REST <= 5 * R_LAUNCH, "a register taken was given up before");
constexpr int SOFT = SM_WARPS * 32;
constexpr float NEG_INF = -__builtin_huge_valf();
// The largest weight is 2^P_EXP .. 2^(P_EXP + LAG) in f16.  A smaller LAG keeps more of the
// small weights but moves the reference, and O with it, more often: 4 x 2048 tokens, 8 x 4
// heads of 128, take 187 us with 8, 192 with 4, 209 with 2, 225 with 1.
constexpr float P_EXP = 11.0f, LAG = 4.0f;
constexpr int NAN_SETS = 3;  // a segment's, of which the epilogue of one and the loads of two more can be under way

// S and P: two of each stream, for the halves of a tile
enum { B_KFULL = 0, B_KEMPTY = 2, B_VFULL = 4, B_VEMPTY = 6, B_QFULL = 8, B_ODONE = 10, B_SFULL = 12, B_PFULL = 36,
       B_SOFT = 16, B_DRAIN = 18, B_TFULL = 20, B_TEMPTY = 24, B_GFULL = 28, B_GEMPTY = 32, B_OFULL = 40, NBARS = 42 };
static_assert(NBARS * 8 <= 512, "barrier area");
// tiles whose places are known, and words of pages outside the cache (of a tile until its softmax has begun: the two in
// the buffers and those known)
constexpr int TURNS = 4, BAD_TURNS = 16, SEGS = 4;
constexpr uint32_t NO_TILE = 0xFFFFFFFFu;

constexpr uint32_t TMEM_COLS = 512, COL_S = 0, COL_O = 256;  // stream i: S at 128 i, O at 256 + 128 i

template <int D>
struct Lay {
  static constexpr int TILE_BYTES = TILE * D * 2, HALF = TILE * 128;
  static constexpr int OFF_Q = 0, OFF_K = 2 * TILE_BYTES, OFF_V = 4 * TILE_BYTES, OFF_BAR = 6 * TILE_BYTES;
  static constexpr int SMEM = OFF_BAR + 512 + 1024;
};

struct Args {
  const uint16_t* q;
  int64_t qb, qt, qh;
  uint16_t* out;
  const uint8_t *k_codes, *v_codes, *k_scale, *v_scale;
  const float *k_factor, *v_factor;
  const int32_t *block_table, *lengths, *counts;
  float* part;    // [CTAs][2][streams with rows of their own][D + 2][128]: pieces of heads that were cut
  int32_t* done;  // [B * groups * Hkv][streams ..] pieces that are there: k_zero's zeros at the start
  int32_t* next;  // heads taken whole so far, likewise
  int B, T, H, Hkv, G, page_log2, width, pages, groups;
  float sm_log2;
};

__device__ __forceinline__ float ex2(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
__device__ __forceinline__ uint32_t f16x2(float lo, float hi) {
  __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<uint32_t*>(&h);
}
__device__ __forceinline__ void sts128(uint32_t a, uint32_t x, uint32_t y, uint32_t z, uint32_t w) {
  asm volatile("st.shared.v4.b32 [%0], {%1,%2,%3,%4};" ::"r"(a), "r"(x), "r"(y), "r"(z), "r"(w) : "memory");
}
// 16 words of this warp's 32 TMEM lanes (lane = thread) to columns taddr ..
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(
          taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
      "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}
__device__ __forceinline__ void tmem_ld16(uint32_t taddr, uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(taddr));
}
__device__ __forceinline__ void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// f16 x f16 -> float32; b_mn: the second operand is MN-major.
__host__ __device__ constexpr uint32_t idesc_f16(uint32_t n, bool b_mn) {
  return (1u << 4) | (b_mn ? 1u << 16 : 0u) | ((n >> 3) << 17) | ((128u >> 4) << 24);
}
// MN-major SWIZZLE_128B: 64 columns (128 bytes) a row, 8 rows of K 1024 bytes
// apart, the next 64 columns `half` bytes on.
__device__ __forceinline__ uint64_t mn_desc(uint32_t saddr, uint32_t half) {
  return (sw128_desc(saddr) & ~((uint64_t)0x3FFF << 16)) | ((uint64_t)(half >> 4) << 16);
}
__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accum) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(accum));
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t accum) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d), "r"(a), "l"(b), "r"(idesc), "r"(accum));
}

// One lane of a converged warp, the same each time.
__device__ __forceinline__ bool elect_one() {
  uint32_t p;
  asm volatile("{\n\t.reg .pred P;\n\telect.sync _|P, 0xFFFFFFFF;\n\tselp.u32 %0, 1, 0, P;\n\t}" : "=r"(p));
  return p != 0;
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
// Entry e = (sequence, row tile): its rows that have a query, the tokens held,
// and the keys that some of its rows sees.
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
  x.end = x.nrows > 0 ? x.held + (x.row0 + x.nrows - 1) / a.G + 1 : 0;
  return x;
}
__device__ __forceinline__ int tiles_of(const Entry& x) { return (x.end + TILE - 1) / TILE; }

// The fewest tiles of a run: a piece more of a head costs its join about as much
// time as a tile, and pieces' joins run one after the other.
__device__ __forceinline__ float run_least(int tiles, int heads) {
  return heads ? fmaxf(1.0f, sqrtf((float)tiles / (float)heads)) : 1.0f;
}

// What opening and ending a head costs, in tiles: the cuts count it.
template <bool PAIR>
struct Cost {
  static constexpr int HEAD = PAIR ? 2 : 1;
};
constexpr float CUT = 5.0f;

// This CTA's run lies from lo to hi; its first head is of `entry`, which begins
// at `before`.  Heads lie end to end, HEAD + tiles each; a cut within the first
// HEAD of one moves to its begin.
struct Run {
  int lo, hi, entry, before, base, rest;  // the first `rest` runs are base + 1 long
  int uncut;                              // no cuts: heads are taken whole, one after the other
};
__device__ __forceinline__ int run_of(const Run& r, int at);
// Segments, one after the other: the part of one head (entry, kv head) in the run.
struct Seg {
  int b, row0, nrows, held, end, kvh, t0, t1, tiles, slot, pair, ps;
  bool whole;
  __device__ __forceinline__ void set(const Entry& x, int e, int kv_heads, int h, int n) {
    b = x.b, row0 = x.row0, nrows = x.nrows, held = x.held, end = x.end, tiles = n;
    kvh = h, pair = e * kv_heads + h;
  }
};
template <int ROWS, int HEAD>
struct Segments {
  const Args& a;
  const int2* plans;
  Run r;
  int pos, ebase, e, tiles;
  Entry x;
  __device__ __forceinline__ Segments(const Args& a_, const int2* p, const Run& run)
      : a(a_), plans(p), r(run), pos(run.lo), ebase(run.before), e(run.entry - 1), tiles(0), x() {}
  __device__ __forceinline__ bool next(Seg& s) {
    if (pos >= r.hi) return false;
#pragma unroll 1
    while (tiles == 0 || pos >= ebase + (tiles + HEAD) * a.Hkv) {
      if (tiles) ebase += (tiles + HEAD) * a.Hkv;
      x = entry_of<ROWS>(a, ++e, plans);
      tiles = tiles_of(x);
    }
    s.set(x, e, a.Hkv, (pos - ebase) / (tiles + HEAD), tiles);
    s.ps = ebase + s.kvh * (tiles + HEAD);
    s.t0 = max(0, pos - s.ps - HEAD);
    s.t1 = min(tiles, r.hi - s.ps - HEAD);
    s.whole = s.t0 == 0 && s.t1 == tiles;
    s.slot = pos == r.lo ? 0 : 1;
    pos = min(r.hi, s.ps + HEAD + tiles);
    return true;
  }
};
// The run that holds this place, by the cuts as they were before they moved.
__device__ __forceinline__ int run_of(const Run& r, int at) {
  const int far = at - r.rest * (r.base + 1);
  return (far < 0 ? 0 : r.rest) + (far < 0 ? at : far) / (far < 0 ? r.base + 1 : r.base);
}

// The weights of 32 scores and their sum; masked scores are -infinity.
__device__ __forceinline__ void weights32(uint32_t (&v)[32], float f, float bias, float2& sum, uint32_t (&p)[16]) {
  const float2 ff = make_float2(f, f), bb = make_float2(bias, bias);
  float2 e[16];
#pragma unroll
  for (int q = 0; q < 16; ++q) {
    e[q] = __ffma2_rn(make_float2(__uint_as_float(v[2 * q]), __uint_as_float(v[2 * q + 1])), ff, bb);
    asm volatile("ex2.approx.ftz.f32 %0, %0;" : "+f"(e[q].x));
    asm volatile("ex2.approx.ftz.f32 %0, %0;" : "+f"(e[q].y));
  }
#pragma unroll
  for (int q = 0; q < 16; ++q) {
    sum = __fadd2_rn(sum, e[q]);
    p[q] = f16x2(e[q].x, e[q].y);
  }
}
__device__ __forceinline__ float max32(const uint32_t (&v)[32], float m) {
#pragma unroll
  for (int q = 0; q < 32; q += 2) m = fmaxf(fmaxf(__uint_as_float(v[q]), __uint_as_float(v[q + 1])), m);
  return m;
}
// 32 bytes, a whole sector.
__device__ __forceinline__ void stg256(void* p, const uint32_t (&w)[8]) {
  asm volatile("st.global.v8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"l"(p), "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3]),
               "r"(w[4]), "r"(w[5]), "r"(w[6]), "r"(w[7]) : "memory");
}
__device__ __forceinline__ uint4 lds128(uint32_t a) {
  uint4 v;
  asm volatile("ld.shared.v4.b32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(a) : "memory");
  return v;
}

template <int D, bool PAIR>
__global__ void __launch_bounds__(THREADS, 1) k_attn_kv4(const __grid_constant__ Args a) {
  using L = Lay<D>;
  constexpr int ROWS = PAIR ? 256 : 128, KS = D / 16, HEAD = Cost<PAIR>::HEAD;
  constexpr int PIECE = 128 * (D + 2);  // of a stream
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* smem =
      reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + L::OFF_BAR);
  __shared__ uint32_t s_tmem;
  __shared__ int s_last[2], s_nan[SM_WARPS][NAN_SETS][D / 16];
  __shared__ long long s_sum[WARPS];
  __shared__ int2 s_plan[PLANS];
  __shared__ Run s_run;
  __shared__ int s_top;
  __shared__ uint32_t s_bad[BAD_TURNS];        // of a tile: a byte per 32 keys, not 0: outside the cache
  __shared__ uint4 s_tile[TURNS][4];
  __shared__ Seg s_seg[SEGS];                   // the segments under way; no tiles: the end
  __shared__ float s_ml[2 * 128];     // not PAIR: the second stream's m and l
  const uint32_t sbase = smem_u32(smem);
  auto bar = [&](int i) { return smem_u32(bars + i); };
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  if (threadIdx.x == 0) {
    for (int i = 0; i < 2; ++i) {
      // one arrival a warp, or a commit
      mbar_init(bar(B_KFULL + i), 4), mbar_init(bar(B_KEMPTY + i), PAIR ? 2 : 1);
      mbar_init(bar(B_VFULL + i), 4), mbar_init(bar(B_VEMPTY + i), PAIR ? 2 : 1);
      mbar_init(bar(B_QFULL + i), 4), mbar_init(bar(B_ODONE + i), 1), mbar_init(bar(B_OFULL + i), 1);
      mbar_init(bar(B_SFULL + i), 1), mbar_init(bar(B_SFULL + 2 + i), 1);
      mbar_init(bar(B_PFULL + i), 4), mbar_init(bar(B_PFULL + 2 + i), 4);
      mbar_init(bar(B_SOFT + i), PAIR ? 4 : 8), mbar_init(bar(B_DRAIN + i), 1);
    }
    for (int i = 0; i < TURNS; ++i) mbar_init(bar(B_TFULL + i), 1), mbar_init(bar(B_TEMPTY + i), 8);
    for (int i = 0; i < SEGS; ++i) mbar_init(bar(B_GFULL + i), 1), mbar_init(bar(B_GEMPTY + i), SM_WARPS + 2);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == W_MMA) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&s_tmem)),
                 "r"(TMEM_COLS));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
  }
  for (int i = threadIdx.x; i < SM_WARPS * NAN_SETS * (D / 16); i += THREADS) (&s_nan[0][0][0])[i] = 0x7FFFFFFF;
  if (threadIdx.x == 0) s_run.lo = s_run.hi = s_top = 0;
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = s_tmem;
  pdl::trigger();  // every CTA holds its tensor memory before the next kernel's can ask for it
  pdl::wait();

  // ---- this CTA's run of tiles ----
  for (int b = threadIdx.x; b < (blockIdx.x == 0 ? a.B : min(a.B, PLANS)); b += THREADS) {
    int err = 0;
    const int2 plan = plan_of(a, b, err);
    if (b < PLANS) s_plan[b] = plan;
    if (err && blockIdx.x == 0) note_err(nullptr, err);
  }
  __syncthreads();
  const int entries = a.B * a.groups, per = (entries + THREADS - 1) / THREADS;
  const int e0 = min(entries, (int)threadIdx.x * per), e1 = min(entries, e0 + per);
  long long own = 0;  // tiles, and in the upper half entries that have any
  int top = 0;
#pragma unroll 1
  for (int e = e0; e < e1; ++e) {
    const int u = tiles_of(entry_of<ROWS>(a, e, s_plan));
    own += u ? u + (1ll << 32) : 0;
    top = max(top, u);
  }
  long long scan = own;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const long long y = __shfl_up_sync(FULL, scan, d);
    if (lane >= d) scan += y;
  }
  if (lane == 31) s_sum[warp] = scan;
  __syncthreads();
  long long total = 0, before = scan - own;
#pragma unroll
  for (int w = 0; w < WARPS; ++w) {
    if (w < warp) before += s_sum[w];
    total += s_sum[w];
  }
  // The longest head, for the choice between cut and uncut heads.
  top = __reduce_max_sync(FULL, top);
  if (lane == 0) atomicMax(&s_top, top);
  __syncthreads();
  top = s_top;
  {
    const int heads = (int)(total >> 32) * a.Hkv, real = (int)total * a.Hkv, all = real + HEAD * heads;
    // Uncut, CTAs idle at the end for about a quarter of an average head where
    // lengths differ (the long ones come first), and for what a whole number of equal
    // heads leaves where they do not; a cut costs its pieces' way through memory and
    // their join, about CUT tiles a CTA.
    const int ctas = (int)gridDim.x;
    const float mean = heads ? (float)all / (float)heads : 0.0f;
    const float idle = 2.0f * (top + HEAD) <= 3.0f * mean
                           ? (float)((heads + ctas - 1) / ctas) * mean - (float)all / (float)ctas : 0.25f * mean;
    const bool uncut = PAIR && heads >= 2 * ctas && idle <= CUT;
    if (threadIdx.x == 0) s_run.uncut = uncut;
    const int runs = uncut ? 0 : min(ctas, (int)ceilf((float)real / run_least(real, heads)));
    const int base = runs ? all / runs : 0, rest = all - base * runs;
    const int cut0 = blockIdx.x * base + min((int)blockIdx.x, rest), cut1 = cut0 + base + ((int)blockIdx.x < rest);
    int at = ((int)before + HEAD * (int)(before >> 32)) * a.Hkv;
    const int to = at + ((int)own + HEAD * (int)(own >> 32)) * a.Hkv;
    if ((int)blockIdx.x < runs) {
      if ((at <= cut0 && cut0 < to) || (at <= cut1 && cut1 < to)) {
#pragma unroll 1
        for (int e = e0; e < e1; ++e) {
          const int w = tiles_of(entry_of<ROWS>(a, e, s_plan)) + HEAD;
          if (w == HEAD) continue;
          auto moved = [&](int cut) {
            const int ps = at + (cut - at) / w * w;
            return cut - ps <= HEAD ? ps : cut;
          };
          const int next = at + w * a.Hkv;
          if (at <= cut0 && cut0 < next)
            s_run.entry = e, s_run.before = at, s_run.base = base, s_run.rest = rest, s_run.lo = moved(cut0);
          if (at <= cut1 && cut1 < next) s_run.hi = moved(cut1);
          at = next;
        }
      }
      if (threadIdx.x == 0 && cut1 == all) s_run.hi = all;
    }
  }
  __syncthreads();
  // a warp's arrival, its threads' writes before it
  auto arrive = [&](int b) {
    __syncwarp();
    if (lane == 0) mbar_arrive(bar(b));
  };

  if (warp >= W_DQ && warp < W_MMA) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(R_DQ));
    // ---------------- codes to f16: a warp takes 32 keys of a tile ----------------
    constexpr int LPR = D / 32, PASS = LPR, KPP = 32 / LPR;  // lanes a key, passes, keys a pass
    const bool is_v = warp >= W_DQ + 4;
    const int wq = warp & 3, c = lane % LPR, kr = lane / LPR;
    const int64_t at = (int64_t)kr * (D / 2) + 16 * c;  // of this lane in 32 keys' codes; an eighth of it in the scales
    const uint8_t *codes = (is_v ? a.v_codes : a.k_codes) + at, *scales = (is_v ? a.v_scale : a.k_scale) + at / 8;
    const int b_full = is_v ? B_VFULL : B_KFULL, b_empty = is_v ? B_VEMPTY : B_KEMPTY;
    const uint32_t buf0 = sbase + (is_v ? L::OFF_V : L::OFF_K);
    uint4 raw[PASS];
    uint32_t sc[PASS];
    auto load = [&](int row) {
      const uint8_t *x = codes + (int64_t)row * (D / 2), *y = scales + (int64_t)row * (D / 16);
#pragma unroll
      for (int p = 0; p < PASS; ++p) {
        // volatile: issued here, before the wait for the buffer
        asm volatile("ld.global.nc.L1::no_allocate.v4.b32 {%0,%1,%2,%3}, [%4];"
                     : "=r"(raw[p].x), "=r"(raw[p].y), "=r"(raw[p].z), "=r"(raw[p].w)
                     : "l"(x + p * KPP * (D / 2)));
        uint16_t e;
        asm volatile("ld.global.nc.L1::no_allocate.b16 %0, [%1];" : "=h"(e) : "l"(y + p * KPP * (D / 16)));
        sc[p] = e;
      }
    };
    // lanes of the row's second half go through their chunks in another order: the
    // eight lanes that store together then meet eight different groups of banks
    const int turn = D == 128 ? c & 2 : 0;
    auto convert = [&](uint32_t dst, const uint4& v, uint32_t s2, int k) {
      const int r = wq * 32 + k;
      uint32_t w[4] = {v.x, v.y, v.z, v.w};
      const uint32_t ss = unpack2(s2);
      uint32_t s0 = __byte_perm(ss, ss, 0x1010), s1 = __byte_perm(ss, ss, 0x3232);
      if (turn) {
        uint32_t x = w[0];
        w[0] = w[2], w[2] = x;
        x = w[1], w[1] = w[3], w[3] = x;
        x = s0, s0 = s1, s1 = x;
      }
      const uint32_t rowp = dst + (D == 128 ? (c >> 1) * L::HALF : 0) + r * 128;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        uint32_t h[4];
        e2m1_f16(w[i], h);
#pragma unroll
        for (int j = 0; j < 4; ++j) h[j] = mul_f16x2(h[j], i < 2 ? s0 : s1);
        const int chunk = (c & 1) * 4 + (i ^ turn);
        sts128(rowp + ((chunk ^ (r & 7)) << 4), h[0], h[1], h[2], h[3]);
      }
    };
    int slot = 0;
    uint32_t sphase = 0;
    uint4 now = {};  // row, key, keys that hold a token, set
    auto next_tile = [&]() {
      const bool ok = mbar_wait_warp(bar(B_TFULL + slot), sphase, nullptr, ERR_WAIT);
      now = s_tile[slot][wq];
      arrive(B_TEMPTY + slot);
      if (++slot == TURNS) slot = 0, sphase ^= 1;
      return ok && now.x != NO_TILE;
    };
    int buf = 0;
    uint32_t phase = 1;
    while (next_tile()) {
      load(now.x);
      if (!mbar_wait_warp(bar(b_empty + buf), phase, nullptr, ERR_WAIT)) break;
      if (is_v) {
        uint32_t odd = 0;
#pragma unroll
        for (int p = 0; p < PASS; ++p) {
          if (p * KPP + kr >= (int)now.z) sc[p] = 0;  // no token of this sequence
          odd |= (sc[p] & 0x7F7Fu) + 0x0101u;
        }
        if (odd & 0x8080u) {  // a NaN: its key noted, its values 0
#pragma unroll
          for (int p = 0; p < PASS; ++p)
#pragma unroll 1
            for (int h = 0; h < 16; h += 8)
              if ((sc[p] >> h & 0x7Fu) == 0x7Fu) {
#pragma unroll 1
                for (int w = 0; w < SM_WARPS; ++w)
                  atomicMin(&s_nan[w][now.w][2 * c + (h >> 3)], (int)now.y + p * KPP + kr);
                sc[p] &= ~(0xFFu << h);
              }
        }
      }
#pragma unroll
      for (int p = 0; p < PASS; ++p) convert(buf0 + buf * L::TILE_BYTES, raw[p], sc[p], p * KPP + kr);
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      arrive(b_full + buf);
      if (++buf == 2) buf = 0, phase ^= 1;
    }
  } else if (warp >= W_MMA) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(R_REST));
    if (warp == W_SCOUT) {
      // ---------------- where the tiles lie, some ahead: lane g < 4 for 32 keys each ----------------
      int slot = 0, set = 0, turn = 0;
      uint32_t phase = 1, bturn = 0, gphase = 1;
      bool ok = true;
      Segments<ROWS, HEAD> segs(a, s_plan, s_run);
      Seg sg;
      auto publish = [&]() {
        ok = mbar_wait_warp(bar(B_GEMPTY + turn), gphase, nullptr, ERR_WAIT);
        if (ok && lane == 0) s_seg[turn] = sg;
        if (ok) arrive(B_GFULL + turn);
        if (++turn == SEGS) turn = 0, gphase ^= 1;
        return ok;
      };
      const int heads = a.B * a.groups * a.Hkv;
      auto next = [&]() {
        if (!s_run.uncut) return segs.next(sg);
        // the next head that no CTA has taken, sequences' last row tiles (the longest) first
        while (true) {
          int k = 0;
          if (lane == 0) k = atomicAdd(a.next, 1);
          k = __shfl_sync(FULL, k, 0);
          if (k >= heads) return false;
          const int kvh = k % a.Hkv, b = k / a.Hkv % a.B, e = b * a.groups + a.groups - 1 - k / a.Hkv / a.B;
          const Entry x = entry_of<ROWS>(a, e, s_plan);
          const int n = tiles_of(x);
          if (n == 0) continue;
          sg.set(x, e, a.Hkv, kvh, n);
          sg.ps = sg.slot = sg.t0 = 0, sg.t1 = n, sg.whole = true;
          return true;
        }
      };
      while (ok && next()) {
        if (!publish()) break;
        for (int t = sg.t0; t < sg.t1; ++t) {
          const int key0 = t * TILE + (lane & 3) * 32, left = sg.end - key0;
          const int key = min(key0, sg.end - 1);
          const int pid = __ldg(a.block_table + (int64_t)sg.b * a.width + (key >> a.page_log2));
          const bool out = pid < 0 || pid >= a.pages, bad = out && left > 0;
          const int row = (((out ? 0 : pid) * a.Hkv + sg.kvh) << a.page_log2) + (key0 & ((1 << a.page_log2) - 1));
          if (bad && lane < 4) note_err(nullptr, ERR_PAGE);
          if (!(ok = mbar_wait_warp(bar(B_TEMPTY + slot), phase, nullptr, ERR_WAIT))) break;
          if (lane < 4) {
            s_tile[slot][lane] = make_uint4(row, key0, bad ? 0 : max(0, min(32, left)), set);
            reinterpret_cast<uint8_t*>(s_bad + bturn)[lane] = bad;
          }
          arrive(B_TFULL + slot);
          // its lines to L2: a lane a line of 128 bytes
          constexpr int LINES = 32 * D / 2 / 128;  // of 32 keys' codes
#pragma unroll
          for (int g = 0; g < 4; ++g) {
            const int64_t r = __shfl_sync(FULL, row, g);
            const int i = lane % LINES;
            const uint8_t* p = (lane < LINES ? a.k_codes : a.v_codes) + r * (D / 2) + i * 128;
            if (lane < 2 * LINES) asm volatile("prefetch.global.L2 [%0];" ::"l"(p));
            if (lane < 4) {
              p = (lane < 2 ? a.k_scale : a.v_scale) + r * (D / 16) + (lane & 1) * 128;
              if (D == 128 || !(lane & 1)) asm volatile("prefetch.global.L2 [%0];" ::"l"(p));
            }
          }
          if (++slot == TURNS) slot = 0, phase ^= 1;
          bturn = (bturn + 1) & (BAD_TURNS - 1);
        }
        set = set == NAN_SETS - 1 ? 0 : set + 1;
      }
      sg.t0 = sg.t1 = 0;
      if (ok && publish() && mbar_wait_warp(bar(B_TEMPTY + slot), phase, nullptr, ERR_WAIT)) {
        if (lane < 4) s_tile[slot][lane] = make_uint4(NO_TILE, 0, 0, 0);
        arrive(B_TFULL + slot);
      }
    } else if (warp != W_MMA + 3) {
      // ---------------- MMA issuers, one a stream ----------------
      // The whole warp runs the loop and one lane issues: the operands then stay in
      // uniform registers.
      constexpr uint32_t ID_S = idesc_f16(64, false), ID_O = idesc_f16(D, true);
      constexpr uint32_t TILE16 = L::TILE_BYTES / 16;
      const int i = warp == W_MMA ? 0 : 1;
      const uint64_t dq = sw128_desc(sbase + L::OFF_Q + i * L::TILE_BYTES), dk = sw128_desc(sbase + L::OFF_K),
                     dv = mn_desc(sbase + L::OFF_V, L::HALF);
      const uint32_t ts = tmem + COL_S + i * 128, to = tmem + COL_O + i * 128;
      uint32_t qph = 0, pph = 0;  // pph: bits of the halves
      bool ok = true;
      // S of a half (64 keys) of tile g; `release`: the stream's last use of its keys
      auto scores = [&](int half, int g, bool release) {
        if (elect_one()) {
          const uint64_t k = desc_at(dk, (g & 1) * TILE16 + half * (64 * 128 / 16));
#pragma unroll
          for (int s = 0; s < KS; ++s) {
            const uint32_t off = ((s >> 2) * L::HALF + (s & 3) * 32) / 16;
            mma_ss(ts + half * 64, desc_at(dq, off), desc_at(k, off), ID_S, s > 0);
          }
          tc_commit(bar(B_SFULL + 2 * i + half));
          if (release) tc_commit(bar(B_KEMPTY + (g & 1)));
        }
        __syncwarp();
      };
      // O and that half's values
      auto values = [&](int half, int g, bool first, bool last) {
        if (elect_one()) {
          const uint64_t v = desc_at(dv, (g & 1) * TILE16 + half * (64 * 128 / 16));
          const uint32_t p = ts + half * 64;
#pragma unroll
          for (int s = 0; s < 4; ++s) mma_ts(to, p + s * 8, desc_at(v, s * 128), ID_O, !first || s > 0);
          tc_commit(bar(B_ODONE + i));
          if (last) tc_commit(bar(B_OFULL + i));
          if (half) tc_commit(bar(B_VEMPTY + (g & 1)));
        }
        __syncwarp();
      };
      auto take = [&](int b, uint32_t parity) {
        ok = ok && mbar_wait_warp(bar(b), parity, nullptr, ERR_WAIT);
        tc_fence_after();
        return ok;
      };
      // PAIR: every tile is both streams'; otherwise tile t of a segment is stream t % 2's
      constexpr int STEP = PAIR ? 1 : 2;
      int turn = 0, g0 = 0;  // g0: tiles before the segment
      uint32_t gphase = 0;
      while (true) {
        ok = mbar_wait_warp(bar(B_GFULL + turn), gphase, nullptr, ERR_WAIT);
        if (!ok) break;
        const int n = s_seg[turn].t1 - s_seg[turn].t0;
        arrive(B_GEMPTY + turn);
        if (n == 0) break;
        if (++turn == SEGS) turn = 0, gphase ^= 1;
        // a half's scores are asked for when the weights in their place have been
        // used, two halves ahead of the softmax
        const int j0 = PAIR ? 0 : i;
        if (!take(B_QFULL + i, qph)) break;
        qph ^= 1;
        if (j0 < n) {
          if (!take(B_KFULL + ((g0 + j0) & 1), (g0 + j0) >> 1 & 1)) break;
          scores(0, g0 + j0, false);
          scores(1, g0 + j0, true);
        }
        for (int j = j0; j < n && ok; j += STEP) {
          const int g = g0 + j;
          const bool again = j + STEP < n;
          if (!take(B_VFULL + (g & 1), g >> 1 & 1)) break;
          if (again && !take(B_KFULL + ((g + STEP) & 1), (g + STEP) >> 1 & 1)) break;
#pragma unroll 1
          for (int half = 0; half < 2; ++half) {
            if (!take(B_PFULL + 2 * i + half, pph >> half & 1)) break;
            pph ^= 1u << half;
            values(half, g, j == j0 && half == 0, half && !again);
            if (again) scores(half, g + STEP, half);
          }
        }
        if (!ok) break;
        g0 += n;
      }
      // every MMA issued has completed before the TMEM is released
      if (elect_one()) {
        tc_commit(bar(B_DRAIN + i));
        mbar_wait(bar(B_DRAIN + i), 0, nullptr, ERR_WAIT);
      }
      __syncwarp();
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(R_SOFT));
    // ---------------- softmax, and the ends of segments ----------------
    const int i = warp >> 2, wq = warp & 3, r = wq * 32 + lane;  // stream, its row
    const int first = PAIR ? i * 128 : 0;                        // of the stream's rows in the tile
    const uint32_t tq = tmem + ((uint32_t)(wq * 32) << 16);
    const uint32_t ts = tq + COL_S + i * 128, to = tq + COL_O + i * 128;
    const uint32_t sq = sbase + L::OFF_Q + i * L::TILE_BYTES;
    uint32_t sph = 0, oph = 0, softph = 0, given = 0;  // sph: bits of the halves; given: weights so far, in halves
    int set = 0, bturn = 0;  // of s_nan; of s_bad, at the segment's first tile
    bool ok = true;
    // the threads that end a segment together: a stream's, or both streams'; bounded, as every wait
    auto soft_sync = [&]() {
      arrive(B_SOFT + (PAIR ? i : 0));
      ok = mbar_wait_warp(bar(B_SOFT + (PAIR ? i : 0)), softph, nullptr, ERR_WAIT);
      softph ^= 1;
      return ok;
    };
    // A segment's rows: this thread's token and head, and whether they are there.
    struct Row {
      int tok, head;
      bool live, exists;
    };
    auto row_of = [&](const Seg& s) {
      Row x;
      const int at = s.row0 + first + r;
      x.tok = at / a.G, x.head = s.kvh * a.G + at - x.tok * a.G;
      x.live = first + r < s.nrows, x.exists = at < a.T * a.G;
      return x;
    };
    // The queries as they lie, to their place in shared memory: a warp's 32 rows,
    // some at a time, 16 bytes a lane.
    auto fetch_q = [&](const Seg& s, const Row& x) {
      const int64_t off = (int64_t)s.b * a.qb + (int64_t)x.tok * a.qt + (int64_t)x.head * a.qh;
      constexpr int CH = D / 8, PER = 32 / CH;  // chunks a row, rows a step
      const int ch = lane % CH;
      const uint32_t there = __ballot_sync(FULL, x.live);
#pragma unroll
      for (int k = 0; k < 32 / PER; ++k) {
        const int rr = k * PER + lane / CH;
        const int64_t o = __shfl_sync(FULL, off, rr);
        const uint32_t dst = sq + (ch >> 3) * L::HALF + (wq * 32 + rr) * 128 + (((ch & 7) ^ (rr & 7)) << 4);
        if (there >> rr & 1u)
          asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(a.q + o + ch * 8) : "memory");
        else
          sts128(dst, 0, 0, 0, 0);
      }
    };
    // ... and in f16, scaled by the row's power of two; a negative scale turns them.
    // Returns the scores' factor: that power of two, the scale and the keys' factor;
    // never 0, so that a masked score stays -infinity.
    auto finish_q = [&](float scale) {
      asm volatile("cp.async.wait_all;" ::: "memory");
      __syncwarp();
      uint32_t m = 0;
#pragma unroll
      for (int q = 0; q < D / 8; ++q) {
        const uint4 v = lds128(sq + (q >> 3) * L::HALF + r * 128 + (((q & 7) ^ (r & 7)) << 4));
        m = __vmaxu2(m, __vmaxu2(__vmaxu2(v.x & 0x7FFF7FFFu, v.y & 0x7FFF7FFFu),
                                 __vmaxu2(v.z & 0x7FFF7FFFu, v.w & 0x7FFF7FFFu)));
      }
      m = max(m & 0xFFFFu, m >> 16);
      const int e = min(max((int)(m >> 7), 15), 253);  // the largest value's exponent field
      const float up = copysignf(__uint_as_float((uint32_t)(254 + 14 - e) << 23), scale);
#pragma unroll
      for (int q = 0; q < D / 8; ++q) {
        const uint32_t at = sq + (q >> 3) * L::HALF + r * 128 + (((q & 7) ^ (r & 7)) << 4);
        const uint4 v = lds128(at);
        sts128(at, f16x2(bf_lo(v.x) * up, bf_hi(v.x) * up), f16x2(bf_lo(v.y) * up, bf_hi(v.y) * up),
               f16x2(bf_lo(v.z) * up, bf_hi(v.z) * up), f16x2(bf_lo(v.w) * up, bf_hi(v.w) * up));
      }
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      arrive(B_QFULL + i);
      const float f = fmaxf(__uint_as_float((uint32_t)(e - 14) << 23) * fabsf(scale), 1.17549435e-38f);
      return scale != scale ? scale : f;
    };

    // row tiles without a query are written here: no tile of keys belongs to them
#pragma unroll 1
    for (int e = blockIdx.x; e < entries; e += gridDim.x) {
      const Entry x = entry_of<ROWS>(a, e, s_plan);
      if (x.nrows > 0) continue;
      const int rows = min(ROWS, a.T * a.G - x.row0);
      for (int64_t n = threadIdx.x; n < (int64_t)rows * a.Hkv * (D / 8); n += SOFT) {
        const int q = (int)(n / (D / 8)), rr = x.row0 + q % rows, h = q / rows;
        reinterpret_cast<uint4*>(a.out + (((int64_t)x.b * a.T + rr / a.G) * a.H + h * a.G + rr % a.G) * D)[n % (D / 8)] =
            make_uint4(0, 0, 0, 0);
      }
    }

    int turn = 0;
    uint32_t gphase = 0;
    // the segment of this turn: whether there is one
    auto segment = [&]() {
      ok = mbar_wait_warp(bar(B_GFULL + turn), gphase, nullptr, ERR_WAIT);
      return ok && s_seg[turn].t1 > 0;
    };
    auto scale_of = [&](const Seg& g) { return a.sm_log2 * __ldg(a.k_factor + g.kvh); };
    bool more = segment();
    float f = 0.0f;
    if (more) {
      fetch_q(s_seg[turn], row_of(s_seg[turn]));
      f = finish_q(scale_of(s_seg[turn]));
    }
    while (more) {
      const Seg& cur = s_seg[turn];  // stays until this warp has let it go
      const int mine = turn;
      if (++turn == SEGS) turn = 0, gphase ^= 1;
      int limit;  // the last key that the row sees
      {
        const Row x = row_of(cur);
        limit = x.live ? cur.held + x.tok : -1;
      }
      // keys below: every row of the warp sees them (rows without a query do not count)
      const int free_end = min(__reduce_min_sync(FULL, limit >= 0 ? limit : 0x7FFFFFFE), 0x7FFFFFFE) + 1;
      const bool any_live = __any_sync(FULL, limit >= 0);
      const float vf = __ldg(a.v_factor + cur.kvh);
      float m = NEG_INF, l = 0.0f;
      const int n = cur.t1 - cur.t0, key00 = cur.t0 * TILE;
      bool any = false;  // this stream has had a tile
      // The products of all weights given so far are done.  The scores that were just
      // read were asked for after the product before the last, so that only the last
      // can be under way and the parity is of its phase.
      auto products = [&]() { return mbar_wait_warp(bar(B_ODONE + i), (given - 1) & 1, nullptr, ERR_WAIT); };
      for (int j = PAIR ? 0 : i; j < n && ok; j += PAIR ? 1 : 2)
#pragma unroll 1
        for (int half = 0; half < 2; ++half) {
          if (!(ok = mbar_wait_warp(bar(B_SFULL + 2 * i + half), sph >> half & 1, nullptr, ERR_WAIT))) break;
          sph ^= 1u << half;
          tc_fence_after();
          // the last scores are there, so the queries' place is free: the next ones travel under this tile
          if (PAIR && half && j + 1 == n && (more = segment())) fetch_q(s_seg[turn], row_of(s_seg[turn]));
          if (any_live) {
            const int key0 = key00 + j * TILE + half * 64;
            const uint32_t th = ts + half * 64, bad = s_bad[(bturn + j) & (BAD_TURNS - 1)] >> (16 * half) & 0xFFFFu;
            uint32_t va[32], vb[32], p[16];
            float2 sum = make_float2(0.0f, 0.0f);
            tmem_ld32(th, va);
            tmem_ld32(th + 32, vb);
            tmem_ld_wait();
            if (key0 + 64 > free_end || bad) {
              // -infinity where the key lies past the row's last, or in no page
              const int stay = limit + 1 - key0, na = bad & 0xFFu ? 0 : stay, nb = bad >> 8 ? 0 : stay - 32;
#pragma unroll
              for (int q = 0; q < 32; ++q) va[q] = q < na ? va[q] : 0xFF800000u, vb[q] = q < nb ? vb[q] : 0xFF800000u;
            }
            const float mx = fmaxf(max32(va, NEG_INF), max32(vb, NEG_INF)), top = mx == NEG_INF ? NEG_INF : mx * f;
            if (__any_sync(FULL, top > m + LAG)) {  // the reference moves, O and l with it
              const float mn = fmaxf(m, top), corr = mn == NEG_INF ? 1.0f : ex2(m - mn);
              m = mn;
              l *= corr;
              if (any) {
                if (!(ok = products())) break;
                tc_fence_after();
#pragma unroll 1
                for (int c = 0; c < D / 16; ++c) {
                  uint32_t o[16];
                  tmem_ld16(to + 16 * c, o);
                  tmem_ld_wait();
#pragma unroll
                  for (int q = 0; q < 16; ++q) o[q] = __float_as_uint(__uint_as_float(o[q]) * corr);
                  tmem_st16(to + 16 * c, o);
                }
              }
            }
            const float bias = m == NEG_INF ? P_EXP : P_EXP - m;
            weights32(va, f, bias, sum, p);
            tmem_st16(th, p);
            weights32(vb, f, bias, sum, p);
            tmem_st16(th + 16, p);
            l += sum.x + sum.y;
            tmem_st_wait();
            any = true;
          }
          tc_fence_before();
          arrive(B_PFULL + 2 * i + half);
          ++given;
        }
      if (!ok) break;
      if (PAIR && more) f = finish_q(scale_of(s_seg[turn]));  // while the last product runs
      bturn = (bturn + n) & (BAD_TURNS - 1);
      const bool had = PAIR || i < n;  // this stream's O has been written
      if (had) {
        if (!(ok = mbar_wait_warp(bar(B_OFULL + i), oph, nullptr, ERR_WAIT))) break;
        oph ^= 1;
        tc_fence_after();
      }
      // ---- the end of a segment ----
      const Row now = row_of(cur);
      uint16_t* orow = a.out + (((int64_t)cur.b * a.T + now.tok) * a.H + now.head) * D;
      const bool writer = PAIR || i == 0;
      float ow = 1.0f, xw = 0.0f;  // weights of this stream's O and of the other's
      const float4* other = reinterpret_cast<const float4*>(smem + L::OFF_Q);
      if (!PAIR) {  // the second stream's sums to the first, through the queries' place
        if (!soft_sync()) break;  // whose last reader may be the other stream: its last scores are there
        if (i == 1) {
          s_ml[r] = m, s_ml[128 + r] = l;
          if (had && any_live)
#pragma unroll
            for (int c = 0; c < D / 32; ++c) {
              uint32_t v[32];
              tmem_ld32(to + 32 * c, v);
              tmem_ld_wait();
#pragma unroll
              for (int q = 0; q < 8; ++q)
                sts128(smem_u32(other + r * (D / 4) + ((8 * c + q) ^ (r & 7))), v[4 * q], v[4 * q + 1], v[4 * q + 2],
                       v[4 * q + 3]);
            }
        }
        if (!soft_sync()) break;
        if (i == 0 && n > 1) {
          const float m1 = s_ml[r], mn = fmaxf(m, m1), ref = mn == NEG_INF ? 0.0f : mn;
          ow = ex2(m - ref), xw = ex2(m1 - ref);
          l = l * ow + s_ml[128 + r] * xw;
          m = mn;
        }
      }
      const float of = l == 0.0f ? 0.0f : __fdiv_rn(vf, l);
      float* piece = a.part + (((int64_t)blockIdx.x * 2 + cur.slot) * (PAIR ? 2 : 1) + (PAIR ? i : 0)) * PIECE;
      if (writer && any_live) {
#pragma unroll
        for (int c = 0; c < D / 32; ++c) {
          uint32_t v[32];
          tmem_ld32(to + 32 * c, v);
          tmem_ld_wait();
          if (!PAIR && n > 1) {
#pragma unroll
            for (int q = 0; q < 8; ++q) {
              const float4 y = other[r * (D / 4) + ((8 * c + q) ^ (r & 7))];
              v[4 * q] = __float_as_uint(__uint_as_float(v[4 * q]) * ow + y.x * xw);
              v[4 * q + 1] = __float_as_uint(__uint_as_float(v[4 * q + 1]) * ow + y.y * xw);
              v[4 * q + 2] = __float_as_uint(__uint_as_float(v[4 * q + 2]) * ow + y.z * xw);
              v[4 * q + 3] = __float_as_uint(__uint_as_float(v[4 * q + 3]) * ow + y.w * xw);
            }
          }
#pragma unroll
          for (int h = 0; h < 2; ++h)
            if (s_nan[warp][set][2 * c + h] <= limit)
#pragma unroll
              for (int q = 0; q < 16; ++q) v[16 * h + q] = 0x7FC00000u;
          if (now.live) {
            if (cur.whole) {
#pragma unroll
              for (int q = 0; q < 2; ++q) {
                uint32_t w[8];
#pragma unroll
                for (int k = 0; k < 8; ++k)
                  w[k] = bf_pack(__uint_as_float(v[16 * q + 2 * k]) * of, __uint_as_float(v[16 * q + 2 * k + 1]) * of);
                stg256(orow + 32 * c + 16 * q, w);
              }
            } else {
#pragma unroll
              for (int q = 0; q < 8; ++q)
                reinterpret_cast<uint4*>(piece)[(8 * c + q) * 128 + r] =
                    make_uint4(v[4 * q], v[4 * q + 1], v[4 * q + 2], v[4 * q + 3]);
            }
          }
        }
      }
      auto blank = [&]() {  // a row without a query
#pragma unroll
        for (int q = 0; q < D / 8; ++q) reinterpret_cast<uint4*>(orow)[q] = make_uint4(0, 0, 0, 0);
      };
      if (cur.whole) {
        if (writer && !now.live && now.exists) blank();
      } else {
        if (writer && now.live) piece[128 * D + r] = m, piece[128 * (D + 1) + r] = l;
        // the stream that finishes last reads the head's pieces in the CTAs' order
        const int c0 = run_of(s_run, cur.ps + HEAD), pieces = run_of(s_run, cur.ps + HEAD + cur.tiles - 1) - c0 + 1;
        // which of its first run's pieces is the head's
        const int slot0 = c0 * s_run.base + min(c0, s_run.rest) >= cur.ps ? 0 : 1, me = PAIR ? i : 0;
        int* done = a.done + (PAIR ? 2 * cur.pair + i : cur.pair);
        if (!soft_sync()) break;
        if (threadIdx.x == (PAIR ? 128 * i : 0)) {
          int k;  // releases every thread's stores, which the barrier has ordered before it
          asm volatile("atom.add.acq_rel.gpu.global.s32 %0, [%1], 1;" : "=r"(k) : "l"(done) : "memory");
          s_last[me] = k == pieces - 1;
        }
        if (!soft_sync()) break;
        if (s_last[me]) {
          auto at_piece = [&](int p) {
            return a.part + (((int64_t)(c0 + p) * 2 + (p == 0 ? slot0 : 0)) * (PAIR ? 2 : 1) + me) * PIECE;
          };
          // A warp takes 32 rows and every wpb-th 16 columns of them, two at a time.
          const int rows = min(128, cur.nrows - first), blocks = max(1, (rows + 31) / 32);
          constexpr int W = PAIR ? 4 : 8;
          const int w = PAIR ? wq : warp, wpb = W / (blocks == 3 ? 4 : blocks), blk = w / wpb;
          const int rr = blk * 32 + lane, at = cur.row0 + first + rr;
          const bool there = rr < rows;
          const int tok = at / a.G, head = cur.kvh * a.G + at - tok * a.G;
          uint16_t* dst = a.out + (((int64_t)cur.b * a.T + tok) * a.H + head) * D;
          if (there) {
            float mm = NEG_INF, ll = 0.0f;
            for (int p0 = 0; p0 < pieces; p0 += 4) {
              float pm[4], pl[4], mn = mm;
#pragma unroll
              for (int q = 0; q < 4; ++q) {  // beyond the last: that one's maximum again, no sum
                const float* src = at_piece(min(p0 + q, pieces - 1)) + 128 * D + rr;
                pm[q] = __ldcg(src), pl[q] = p0 + q < pieces ? __ldcg(src + 128) : 0.0f;
              }
#pragma unroll
              for (int q = 0; q < 4; ++q) mn = fmaxf(mn, pm[q]);
              const float ref = mn == NEG_INF ? 0.0f : mn;
              ll *= ex2(mm - ref);
#pragma unroll
              for (int q = 0; q < 4; ++q) ll = fmaf(pl[q], ex2(pm[q] - ref), ll);
              mm = mn;
            }
            const float ref = mm == NEG_INF ? 0.0f : mm, g = ll == 0.0f ? 0.0f : __fdiv_rn(vf, ll);
#pragma unroll 1
            for (int c = w % wpb; c < D / 16; c += 2 * wpb) {
              float4 acc[2][4] = {};
#pragma unroll 1
              for (int p0 = 0; p0 < pieces; p0 += 2) {  // all loads of two pieces in flight together
                float4 y[2][2][4];
                float pm[2];
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                  const float* src = at_piece(min(p0 + k, pieces - 1));
                  pm[k] = __ldcg(src + 128 * D + rr);
#pragma unroll
                  for (int h = 0; h < 2; ++h)
#pragma unroll
                    for (int q = 0; q < 4; ++q)
                      y[k][h][q] = __ldcg(reinterpret_cast<const float4*>(src) +
                                          (4 * min(c + h * wpb, D / 16 - 1) + q) * 128 + rr);
                }
#pragma unroll
                for (int k = 0; k < 2; ++k)
                  if (p0 + k < pieces) {
                    const float e = ex2(pm[k] - ref);
#pragma unroll
                    for (int h = 0; h < 2; ++h)
#pragma unroll
                      for (int q = 0; q < 4; ++q) {
                        float4 &t = acc[h][q], z = y[k][h][q];
                        t.x = fmaf(z.x, e, t.x), t.y = fmaf(z.y, e, t.y), t.z = fmaf(z.z, e, t.z), t.w = fmaf(z.w, e, t.w);
                      }
                  }
              }
#pragma unroll
              for (int h = 0; h < 2; ++h)
                if (c + h * wpb < D / 16) {
                  uint32_t o[8];
#pragma unroll
                  for (int q = 0; q < 4; ++q)
                    o[2 * q] = bf_pack(acc[h][q].x * g, acc[h][q].y * g), o[2 * q + 1] = bf_pack(acc[h][q].z * g, acc[h][q].w * g);
                  stg256(dst + 16 * (c + h * wpb), o);
                }
            }
          }
          if (writer && !now.live && now.exists) blank();
        }
      }
      // the set of NaNs is for another segment
      __syncwarp();
      if (lane < D / 16) s_nan[warp][set][lane] = 0x7FFFFFFF;
      set = set == NAN_SETS - 1 ? 0 : set + 1;
      arrive(B_GEMPTY + mine);
      if (!PAIR) {
        if (!soft_sync()) break;  // the queries' place was read
        more = segment();
        if (more) {
          fetch_q(s_seg[turn], row_of(s_seg[turn]));
          f = finish_q(scale_of(s_seg[turn]));
        }
      }
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
  }
  tc_fence_before();
  __syncthreads();
  if (warp == W_MMA) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(TMEM_COLS));
  }
}

// A launch's counters to 0, in the stream before it.  They are the call's own and lie in
// its workspace: a launch whose waits gave up leaves them anywhere, and kept from call to
// call they would have the next one skip heads.
constexpr int ZERO_THREADS = 256;
__global__ void __launch_bounds__(ZERO_THREADS) k_zero(int32_t* counters, int64_t n) {
  pdl::trigger();
  pdl::wait();
  for (int64_t i = (int64_t)blockIdx.x * ZERO_THREADS + threadIdx.x; i < n; i += (int64_t)gridDim.x * ZERO_THREADS)
    counters[i] = 0;
}

// How a call's work is cut: rows a tile, row tiles of a sequence, and CTAs; floats of
// pieces and, behind them in the workspace, counters.
struct Cut {
  int rows, groups, ctas;
  int64_t floats, counters;
};
static Cut cut_of(int64_t batch, int64_t tokens, int heads, int kv_heads, int head_dim, int64_t capacity) {
  const int64_t rows = tokens * (heads / kv_heads);
  Cut c;
  c.rows = rows > 128 ? 256 : 128;
  c.groups = (int)((rows + c.rows - 1) / c.rows);
  const int64_t tiles = std::max<int64_t>(1, (capacity + TILE - 1) / TILE);
  c.ctas = (int)std::min<int64_t>(vq::mx::sm_count(), std::max<int64_t>(1, batch) * c.groups * kv_heads * tiles);
  c.floats = (int64_t)c.ctas * 2 * c.rows * (head_dim + 2);
  c.counters = batch * kv_heads * c.groups * (c.rows / 128) + 1;
  return c;
}

int64_t workspace(int64_t batch, int64_t tokens, int heads, int kv_heads, int head_dim, int64_t capacity) {
  const Cut c = cut_of(batch, tokens, heads, kv_heads, head_dim, capacity);
  return c.floats + c.counters;
}

template <int D, bool PAIR>
static int launch(const Args& a, int ctas, cudaStream_t st) {
  if (!allow_smem<k_attn_kv4<D, PAIR>>(Lay<D>::SMEM)) return VQ_ERR_CUDA;
  // the registers that the split takes up have to be there at the launch
  static const int regs = [] {
    cudaFuncAttributes at;
    return cudaFuncGetAttributes(&at, k_attn_kv4<D, PAIR>) == cudaSuccess ? at.numRegs : 0;
  }();
  if (regs < R_LAUNCH) return VQ_ERR_CUDA;
  return pdl::launch<k_attn_kv4<D, PAIR>>(ctas, THREADS, Lay<D>::SMEM, st, 1, a) ? VQ_OK : VQ_ERR_CUDA;
}

// Checked arguments (vq_attn_kv4), but for the sizes of the workspaces.
int attend(const void* q, const int64_t* q_strides, int64_t batch, int64_t tokens, int heads, int kv_heads, int head_dim,
           const void* k_codes, const void* v_codes, const void* k_scale, const void* v_scale, const float* k_factor,
           const float* v_factor, int64_t pages, int page, const void* block_table, int64_t table_width,
           const void* lengths, const void* counts, float sm_scale, float* workspace, int64_t workspace_floats,
           void* out, cudaStream_t st) {
  const int64_t capacity = table_width * page;
  const Cut c = cut_of(batch, tokens, heads, kv_heads, head_dim, capacity);
  const int64_t pairs = batch * kv_heads * c.groups;
  // the tiles of all heads, counted in 32 bits
  if (pairs * ((capacity + TILE - 1) / TILE + 3) >= (1ll << 31)) return VQ_ERR_INVALID;
  if (!workspace || workspace_floats < c.floats + c.counters) return VQ_ERR_INVALID;
  Args a;
  a.q = (const uint16_t*)q;
  a.qb = q_strides[0], a.qt = q_strides[1], a.qh = q_strides[2];
  a.out = (uint16_t*)out;
  a.k_codes = (const uint8_t*)k_codes, a.v_codes = (const uint8_t*)v_codes;
  a.k_scale = (const uint8_t*)k_scale, a.v_scale = (const uint8_t*)v_scale;
  a.k_factor = k_factor, a.v_factor = v_factor;
  a.block_table = (const int32_t*)block_table;
  a.lengths = (const int32_t*)lengths;
  a.counts = (const int32_t*)counts;
  a.part = workspace;
  a.next = reinterpret_cast<int32_t*>(workspace + c.floats), a.done = a.next + 1;
  a.B = (int)batch, a.T = (int)tokens, a.H = heads, a.Hkv = kv_heads, a.G = heads / kv_heads;
  a.page_log2 = page == 32 ? 5 : page == 64 ? 6 : 7;
  a.width = (int)table_width, a.pages = (int)pages, a.groups = c.groups;
  a.sm_log2 = sm_scale * 1.4426950408889634f;
  const unsigned zero_ctas = (unsigned)std::min<int64_t>((c.counters + ZERO_THREADS - 1) / ZERO_THREADS, vq::mx::sm_count());
  if (!pdl::launch<k_zero>(zero_ctas, ZERO_THREADS, 0, st, 1, a.next, c.counters)) return VQ_ERR_CUDA;
  if (head_dim == 128) return c.rows == 256 ? launch<128, true>(a, c.ctas, st) : launch<128, false>(a, c.ctas, st);
  return c.rows == 256 ? launch<64, true>(a, c.ctas, st) : launch<64, false>(a, c.ctas, st);
}

// This file's sticky word (vq_device_errors).
int sticky_kv4(int* out, int clear, cudaStream_t st) { return vq::tc::sticky_read(out, clear, st); }

}  // namespace kv4
}  // namespace vq
