// Rotary positions and the append to a paged key / value cache held in E4M3, or in
// 4 bits (further down); the heads of q and k normalised before they turn, or not.
//
// The E4M3 cache: codes [pages, kv_heads, page, D] E4M3 bytes and one float32
// scale per (page, head), for the keys and for the values.  A sequence's
// token p lies in slot p % page of the page block_table[b][p / page].
//
// Rotation: the pair (a, b) of columns at angle theta = position * frequency
// becomes (a cos - b sin, a sin + b cos), cos and sin read from a float32
// table [positions, rot / 2, 2]; pairs are columns (i, i + rot / 2), or
// (2i, 2i + 1) when interleaved; columns past rot stay.  float32 throughout:
// q is rounded once to its type, k goes to its codes unrounded.
//
// Block scale: the least power of two s with max|value| / s <= 448 over the
// block's tokens, in [2^-100, 2^120].  A power of two makes value / s exact,
// and lets a block's scale grow when a later token needs it: the codes it
// holds are then multiplied by old / new, exact but for codes that become
// subnormal.  A NaN gives a NaN code and does not enter the maximum; an
// infinity (a turned value beyond float32's range is one) saturates.
//
// Bound by HBM for prompts (the projections read once, q and the codes
// written once) and by latency for single tokens.  A head's norm is a sum over the
// lanes that hold it, in registers: 8 x 2048 tokens, 8 x 4 heads of 128 in bf16 take
// 76 us with both norms (floor 58; a chain of instructions beside HBM), interleaved 99,
// in float32 198 (floor 109); one token 2.9 us.  At 80 registers the forms with norms
// spill 4 to 16 bytes a thread.
#include <cuda_runtime.h>
#include <stdint.h>

#include <algorithm>

#include "voyager_b200.h"
#include "vq_e4m3.cuh"
#include "vq_pdl.cuh"
#include "vq_tc.cuh"

namespace vq {
namespace kv {

using namespace vq::e4;

// Codes of the sticky device word for plans (lengths, counts, block table)
// that do not fit: the tokens concerned are left out.
enum { ERR_PAGE = 301, ERR_CAPACITY = 302, ERR_COUNT = 303 };

struct Strides {
  int64_t b, t, h;  // elements
};

struct Args {
  const void *q, *k, *v;
  Strides sq, sk, sv;
  const float2* table;  // [positions, rot / 2] (cos, sin)
  void* q_out;          // [B, T, H, D]
  uint8_t *k_codes, *v_codes;
  float *k_scale, *v_scale;
  const int32_t* block_table;  // [B, width]
  const int32_t* lengths;      // [B] tokens held before the call
  const int32_t* counts;       // [B] new tokens, or null: T
  int B, T, H, Hkv, rot, page, width, pages, interleaved;
  int q_blocks, W;  // CTAs of the q part; pages that T tokens can touch
  int hq, hc;       // heads per thread of the q part, per CTA of the cache part
  const void *q_norm, *k_norm;  // [D] in q's type, or null: that part has no norm
  float eps;
  // the 4-bit cache: E4M3 bytes [pages, Hkv, page, D / 16], and a factor for each head
  uint8_t *k_bscale, *v_bscale;
  const float *k_factor, *v_factor;
};

// One thread's 16 columns of a head as 8 pairs: unit u of D / 16 is pairs
// 8u .. 8u + 7 of the rot / 2 rotated pairs, or 16 plain columns past them.
// c0, c1: the first columns of the two groups of 8.
template <bool IL>
__device__ __forceinline__ void unit_cols(int u, int rot, int& c0, int& c1) {
  if (!IL && u * 16 < rot) {
    c0 = u * 8;
    c1 = u * 8 + (rot >> 1);
  } else {
    c0 = u * 16;
    c1 = c0 + 8;
  }
}

// The angles of unit u of one position (ones and zeros past rot).
__device__ __forceinline__ void load_angles(const float2* cs, int u, int rot, float (&c)[8], float (&s)[8]) {
  if (u * 16 < rot) {
    const float4* t = reinterpret_cast<const float4*>(cs + u * 8);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float4 f = __ldg(t + i);
      c[2 * i] = f.x, s[2 * i] = f.y, c[2 * i + 1] = f.z, s[2 * i + 1] = f.w;
    }
  }
}
// x0 / x1: columns c0.. / c1.. of the unit, turned.
template <bool IL>
__device__ __forceinline__ void turn(float (&x0)[8], float (&x1)[8], const float (&c)[8], const float (&s)[8]) {
  if (IL) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float a = x0[2 * i], b = x0[2 * i + 1];
      x0[2 * i] = a * c[i] - b * s[i];
      x0[2 * i + 1] = a * s[i] + b * c[i];
      const float d = x1[2 * i], e = x1[2 * i + 1];
      x1[2 * i] = d * c[4 + i] - e * s[4 + i];
      x1[2 * i + 1] = d * s[4 + i] + e * c[4 + i];
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float a = x0[i], b = x1[i];
      x0[i] = a * c[i] - b * s[i];
      x1[i] = a * s[i] + b * c[i];
    }
  }
}

// A head's RMSNorm: its U lanes, side by side in a warp, hold 16 columns each.
template <typename T, int U>
__device__ __forceinline__ void head_norm(float (&x0)[8], float (&x1)[8], const void* weight, int c0, int c1,
                                          float eps) {
  float w0[8], w1[8];
  T::load8(reinterpret_cast<const typename T::type*>(weight) + c0, w0);
  T::load8(reinterpret_cast<const typename T::type*>(weight) + c1, w1);
  float s = 0.0f;
#pragma unroll
  for (int j = 0; j < 8; ++j) s = fmaf(x0[j], x0[j], fmaf(x1[j], x1[j], s));
  const uint32_t lanes = ((1u << U) - 1) << (threadIdx.x & 31 & ~(U - 1));
#pragma unroll
  for (int d = U / 2; d; d >>= 1) s += __shfl_xor_sync(lanes, s, d);
  const float f = rsqrtf(fmaf(s, 1.0f / (16 * U), eps));
#pragma unroll
  for (int j = 0; j < 8; ++j) x0[j] = x0[j] * f * w0[j], x1[j] = x1[j] * f * w1[j];
}

// New tokens of sequence b that fit the plan, and the tokens it holds.
__device__ __forceinline__ int plan(const Args& a, int b, int& held) {
  held = a.lengths[b];
  int n = a.counts ? a.counts[b] : a.T;
  if (n > a.T || n < 0 || held < 0) {
    tc::note_err(nullptr, ERR_COUNT);
    n = held < 0 ? 0 : min(max(n, 0), a.T);
    held = max(held, 0);
  }
  const int64_t cap = (int64_t)a.width * a.page;
  if (held + (int64_t)n > cap) {
    tc::note_err(nullptr, ERR_CAPACITY);
    n = held >= cap ? 0 : (int)(cap - held);
  }
  return n;
}

// The least power of two s with amax / s <= 448 = 1.75 * 2^8, in
// [2^-100, 2^120]: amax = m * 2^x gives 2^(x - 8), or 2^(x - 7) for m > 1.75.
__device__ __forceinline__ float pow2_scale(float amax) {
  const uint32_t b = __float_as_uint(amax);
  int e = (int)(b >> 23) - 127 - 8 + ((b & 0x7FFFFFu) > 0x600000u ? 1 : 0);
  e = min(max(e, -100), 120);
  return __uint_as_float((uint32_t)(e + 127) << 23);
}

// A unit of a row to memory: in one 32-byte store where its columns lie side
// by side (two of 16 bytes would each fill half of every sector that a warp
// touches: 178 us against 172 for the 8 prompts below, turned by 16 columns).
template <typename T>
__device__ __forceinline__ void store_unit(typename T::type* row, int c0, int c1, const float (&x0)[8],
                                           const float (&x1)[8]) {
  if (sizeof(*row) == 2 && c1 == c0 + 8) {
    asm volatile("st.global.v8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"l"(row + c0), "r"(bf_pack(x0[0], x0[1])),
                 "r"(bf_pack(x0[2], x0[3])), "r"(bf_pack(x0[4], x0[5])), "r"(bf_pack(x0[6], x0[7])),
                 "r"(bf_pack(x1[0], x1[1])), "r"(bf_pack(x1[2], x1[3])), "r"(bf_pack(x1[4], x1[5])),
                 "r"(bf_pack(x1[6], x1[7])) : "memory");
  } else {
    T::store8(row + c0, x0);
    T::store8(row + c1, x1);
  }
}

constexpr int QH = 2;  // heads of a token that a thread of the q part takes at a time

// The q part: thread `i` of it takes its unit of a.hq heads of a token (a
// multiple of QH), so that the token's angles, twice the bytes of a bf16 unit,
// are read once for them.
struct QUnit {
  int u, h0, h1, b, t, c0, c1;
  int64_t row;
  bool any;
};
template <bool IL, int D>
__device__ __forceinline__ QUnit q_unit(const Args& a, int64_t i) {
  constexpr int U = D / 16;
  QUnit x;
  x.u = (int)(i % U);
  int64_t r = i / U;
  const int hg = (a.H + a.hq - 1) / a.hq;
  x.h0 = (int)(r % hg) * a.hq, x.h1 = min(a.H, x.h0 + a.hq);
  r /= hg;
  x.any = r < (int64_t)a.B * a.T;
  x.row = r;
  x.b = (int)(r / a.T), x.t = (int)(r - (int64_t)x.b * a.T);
  unit_cols<IL>(x.u, a.rot, x.c0, x.c1);
  return x;
}
template <typename T, bool IL, int D, bool NORM>
__device__ __forceinline__ void turn_q(const Args& a, int64_t i) {
  using E = typename T::type;
  const QUnit x = q_unit<IL, D>(a, i);
  if (!x.any) return;
  E* out = reinterpret_cast<E*>(a.q_out) + x.row * a.H * D;
  const E* p = reinterpret_cast<const E*>(a.q) + x.b * a.sq.b + x.t * a.sq.t;
  float x0[QH][8], x1[QH][8], c[8], s[8];
#pragma unroll
  for (int q = 0; q < QH; ++q)
    if (x.h0 + q < x.h1) {
      T::load8(p + (x.h0 + q) * a.sq.h + x.c0, x0[q]);
      T::load8(p + (x.h0 + q) * a.sq.h + x.c1, x1[q]);
    }
  int held;
  const bool live = x.t < plan(a, x.b, held), turns = live && x.u * 16 < a.rot;
  if (turns) load_angles(a.table + (int64_t)(held + x.t) * (a.rot >> 1), x.u, a.rot, c, s);
#pragma unroll
  for (int q = 0; q < QH; ++q)
    if (x.h0 + q < x.h1) {
      if (NORM && a.q_norm) head_norm<T, D / 16>(x0[q], x1[q], a.q_norm, x.c0, x.c1, a.eps);
      if (turns) turn<IL>(x0[q], x1[q], c, s);
      if (!live) {
#pragma unroll
        for (int j = 0; j < 8; ++j) x0[q][j] = x1[q][j] = 0.0f;
      }
      store_unit<T>(out + (x.h0 + q) * D, x.c0, x.c1, x0[q], x1[q]);
    }
}

// A thread's own ring in shared memory, filled by cp.async: DEPTH steps of four
// groups of 8 elements.  Only the thread itself reads it, so waiting for its
// own copies is enough; registers for that many loads in flight would halve
// the threads that fit (one step ahead in registers: 159 us for 8 prompts of
// 2048 tokens and 32 heads, against 105 at the HBM copy rate).
template <typename T, int TH>
struct Ring {
  using E = typename T::type;
  static constexpr int DEPTH = 3, CH = sizeof(E) / 2;  // 16-byte chunks per group
  static constexpr int BYTES = DEPTH * 4 * CH * 16 * TH;
  uint32_t base;
  __device__ __forceinline__ explicit Ring(void* smem) : base(tc::smem_u32(smem) + threadIdx.x * 16) {}
  __device__ __forceinline__ uint32_t at(int step, int group) const {
    return base + ((step % DEPTH) * 4 + group) * CH * 16 * TH;
  }
  __device__ __forceinline__ void fetch(int step, int group, const E* p) const {
#pragma unroll
    for (int c = 0; c < CH; ++c)
      asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(at(step, group) + c * 16 * TH),
                   "l"(reinterpret_cast<const char*>(p) + 16 * c) : "memory");
  }
  __device__ __forceinline__ void commit() const { asm volatile("cp.async.commit_group;" ::: "memory"); }
  // every step but the newest DEPTH - 1 has landed
  __device__ __forceinline__ void wait() const {
    asm volatile("cp.async.wait_group %0;" ::"n"(DEPTH - 1) : "memory");
  }
  __device__ __forceinline__ void read(int step, int group, float (&v)[8]) const {
    typename T::Raw r;
    uint4* u = reinterpret_cast<uint4*>(&r);
#pragma unroll
    for (int c = 0; c < CH; ++c)
      asm volatile("ld.shared.v4.b32 {%0,%1,%2,%3}, [%4];"
                   : "=r"(u[c].x), "=r"(u[c].y), "=r"(u[c].z), "=r"(u[c].w)
                   : "r"(at(step, group) + c * 16 * TH) : "memory");
    T::widen8(r, v);
  }
};

// The q part alone, beside k_rope_append.
constexpr int Q_THREADS = 256;
template <typename T, bool IL, int D, bool NORM>
__global__ void __launch_bounds__(Q_THREADS) k_turn_q(const __grid_constant__ Args a) {
  using E = typename T::type;
  extern __shared__ __align__(16) uint8_t smem[];
  const Ring<T, Q_THREADS> ring(smem);
  pdl::wait();
  pdl::trigger();  // k_rope_append waits for nothing else that this one waited for
  const QUnit x = q_unit<IL, D>(a, (int64_t)blockIdx.x * Q_THREADS + threadIdx.x);
  if (!x.any) return;
  E* out = reinterpret_cast<E*>(a.q_out) + x.row * a.H * D;
  const E* p = reinterpret_cast<const E*>(a.q) + x.b * a.sq.b + x.t * a.sq.t;
  const int steps = (x.h1 - x.h0 + QH - 1) / QH;
  auto fetch = [&](int k) {
    if (k < steps) {
#pragma unroll
      for (int q = 0; q < QH; ++q) {
        const E* r = p + min(x.h0 + k * QH + q, x.h1 - 1) * a.sq.h;
        ring.fetch(k, 2 * q, r + x.c0);
        ring.fetch(k, 2 * q + 1, r + x.c1);
      }
    }
    ring.commit();
  };
#pragma unroll
  for (int k = 0; k < Ring<T, Q_THREADS>::DEPTH - 1; ++k) fetch(k);
  int held;
  const bool live = x.t < plan(a, x.b, held), turns = live && x.u * 16 < a.rot;
  float c[8], s[8];
  if (turns) load_angles(a.table + (int64_t)(held + x.t) * (a.rot >> 1), x.u, a.rot, c, s);
  for (int k = 0; k < steps; ++k) {
    fetch(k + Ring<T, Q_THREADS>::DEPTH - 1);
    ring.wait();
#pragma unroll
    for (int q = 0; q < QH; ++q) {
      const int h = x.h0 + k * QH + q;
      float x0[8], x1[8];
      ring.read(k, 2 * q, x0);
      ring.read(k, 2 * q + 1, x1);
      if (NORM && a.q_norm) head_norm<T, D / 16>(x0, x1, a.q_norm, x.c0, x.c1, a.eps);
      if (turns) turn<IL>(x0, x1, c, s);
      if (!live) {
#pragma unroll
        for (int j = 0; j < 8; ++j) x0[j] = x1[j] = 0.0f;
      }
      if (h < x.h1) store_unit<T>(out + h * D, x.c0, x.c1, x0, x1);
    }
  }
  asm volatile("cp.async.wait_all;" ::: "memory");
}

// The block that the w-th touched page of sequence b is for a head: which new
// tokens go into it (t0 .. t0 + tokens - 1, from slot0 on) and where it lies.
struct Block {
  int t0, tokens, slot0, pid;
  int64_t pos;  // of its first new token
};
__device__ __forceinline__ Block block_of(const Args& a, int b, int w) {
  Block k;
  int held;
  const int n = plan(a, b, held);
  const int first = held / a.page + w;  // the sequence's page number
  const int64_t begin = (int64_t)first * a.page;
  k.pos = max((int64_t)held, begin);
  k.tokens = (int)max(min((int64_t)held + n, begin + a.page) - k.pos, (int64_t)0);
  k.t0 = (int)(k.pos - held);
  k.slot0 = (int)(k.pos - begin);
  k.pid = 0;
  if (k.tokens > 0) {
    k.pid = a.block_table[(int64_t)b * a.width + first];
    if (k.pid < 0 || k.pid >= a.pages) {
      tc::note_err(nullptr, ERR_PAGE);
      k.tokens = 0;
    }
  }
  return k;
}

__device__ __forceinline__ float amax16(const float (&x0)[8], const float (&x1)[8], float m) {
#pragma unroll
  for (int j = 0; j < 8; ++j) m = fmaxf(m, fmaxf(fabsf(x0[j]), fabsf(x1[j])));
  return m;
}
// 16 columns as codes, 8 bytes at o + c0 and at o + c1.
__device__ __forceinline__ void store_codes(uint8_t* o, int c0, int c1, const float (&x0)[8],
                                            const float (&x1)[8], float inv) {
  uint2 k0, k1;
  k0.x = pack4(x0[0] * inv, x0[1] * inv, x0[2] * inv, x0[3] * inv);
  k0.y = pack4(x0[4] * inv, x0[5] * inv, x0[6] * inv, x0[7] * inv);
  k1.x = pack4(x1[0] * inv, x1[1] * inv, x1[2] * inv, x1[3] * inv);
  k1.y = pack4(x1[4] * inv, x1[5] * inv, x1[6] * inv, x1[7] * inv);
  if (c1 == c0 + 8) {
    *reinterpret_cast<uint4*>(o + c0) = make_uint4(k0.x, k0.y, k1.x, k1.y);
  } else {
    *reinterpret_cast<uint2*>(o + c0) = k0;
    *reinterpret_cast<uint2*>(o + c1) = k1;
  }
}
// 16 codes brought to the scale was / f.
__device__ __forceinline__ void rescale16(uint4* p, float f) {
  uint4 v = *p;
  uint32_t* w = reinterpret_cast<uint32_t*>(&v);
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const float2 l = half2f(unpack2(w[j])), g = half2f(unpack2_hi(w[j]));
    w[j] = pack4(l.x * f, l.y * f, g.x * f, g.y * f);
  }
  *p = v;
}

// Many new tokens: a CTA takes a.hc blocks (page, head) of the keys or the
// values one after the other, so that the angles of a page's tokens come from
// L1 after the first.  TH = page * D / 32 threads: two units of every thread
// are a whole block, held in registers between its maximum and its codes,
// while the next two blocks' loads are in flight.  768 threads an SM: 8 prompts
// of 2048 tokens, 32 heads of 128, q included: 132 us (5.1 TB/s); with 512, 140,
// with 1024 and spilled registers 162.
template <typename T, bool IL, int D, int TH, bool NORM>
__global__ void __launch_bounds__(TH, TH > 512 ? 1 : 768 / TH) k_rope_append(const __grid_constant__ Args a) {
  using E = typename T::type;
  constexpr int U = D / 16, ROWS = TH / U, IT = 2;  // threads per token, tokens per pass, passes
  __shared__ uint32_t part[2][TH / 32];
  pdl::trigger();
  int i = blockIdx.x;
  const int hg = (a.Hkv + a.hc - 1) / a.hc, h0 = i % hg * a.hc, h1 = min(a.Hkv, h0 + a.hc);
  i /= hg;
  const bool is_v = i & 1;
  i >>= 1;
  const int b = i / a.W;
  const Block k = block_of(a, b, i % a.W);
  // k_turn_q, launched before this kernel, shares nothing with it, so only the
  // end waits: kernels behind this one then come after both
  if (k.tokens <= 0) {
    pdl::wait();
    return;
  }
  const int u = threadIdx.x % U, r0 = threadIdx.x / U;
  const Strides st = is_v ? a.sv : a.sk;
  const E* src = reinterpret_cast<const E*>(is_v ? a.v : a.k) + b * st.b + k.t0 * st.t + r0 * st.t;
  int c0, c1;
  unit_cols<IL>(u, a.rot, c0, c1);
  const bool turns = !is_v && u * 16 < a.rot;
  extern __shared__ __align__(16) uint8_t smem[];
  const Ring<T, TH> ring(smem);
  auto fetch = [&](int h) {
    if (h < h1) {
#pragma unroll
      for (int it = 0; it < IT; ++it)
        if (it * ROWS + r0 < k.tokens) {
          const E* p = src + h * st.h + it * ROWS * st.t;
          ring.fetch(h - h0, 2 * it, p + c0);
          ring.fetch(h - h0, 2 * it + 1, p + c1);
        }
    }
    ring.commit();
  };
#pragma unroll
  for (int d = 0; d < Ring<T, TH>::DEPTH - 1; ++d) fetch(h0 + d);
  for (int h = h0; h < h1; ++h) {
    const int64_t blk = (int64_t)k.pid * a.Hkv + h;
    uint8_t* codes = (is_v ? a.v_codes : a.k_codes) + blk * a.page * D;
    float* scale = (is_v ? a.v_scale : a.k_scale) + blk;
    const float was = k.slot0 ? *scale : 0.0f;  // slot 0 written now: a fresh block
    fetch(h + Ring<T, TH>::DEPTH - 1);
    ring.wait();
    float x0[IT][8], x1[IT][8];
#pragma unroll
    for (int it = 0; it < IT; ++it)
      if (it * ROWS + r0 < k.tokens) {
        ring.read(h - h0, 2 * it, x0[it]);
        ring.read(h - h0, 2 * it + 1, x1[it]);
      }
    float m = 0.0f;
#pragma unroll
    for (int it = 0; it < IT; ++it)
      if (it * ROWS + r0 < k.tokens) {
        if (NORM && !is_v && a.k_norm) head_norm<T, U>(x0[it], x1[it], a.k_norm, c0, c1, a.eps);
        if (turns) {
          float c[8], s[8];
          load_angles(a.table + (k.pos + it * ROWS + r0) * (a.rot >> 1), u, a.rot, c, s);
          turn<IL>(x0[it], x1[it], c, s);
        }
        m = amax16(x0[it], x1[it], m);
      }
    // magnitudes order as their bit patterns do
    uint32_t mb = __reduce_max_sync(FULL, __float_as_uint(m));
    if ((threadIdx.x & 31) == 0) part[h & 1][threadIdx.x >> 5] = mb;
    __syncthreads();  // two buffers: the next head's maxima do not meet this one's readers
#pragma unroll
    for (int j = 0; j < TH / 32; ++j) mb = max(mb, part[h & 1][j]);
    const float s = fmaxf(pow2_scale(__uint_as_float(mb)), was);
    const float inv = __fdiv_rn(1.0f, s);  // exact: s is a power of two
#pragma unroll
    for (int it = 0; it < IT; ++it)
      if (it * ROWS + r0 < k.tokens)
        store_codes(codes + (k.slot0 + it * ROWS + r0) * D, c0, c1, x0[it], x1[it], inv);
    if (k.slot0 && s != was)  // the tokens that the block holds, at the new scale
      for (int c = threadIdx.x; c < k.slot0 * U; c += TH)
        rescale16(reinterpret_cast<uint4*>(codes) + c, was * inv);
    if (threadIdx.x == 0) *scale = s;  // every thread read the old one before the barrier
  }
  asm volatile("cp.async.wait_all;" ::: "memory");
  pdl::wait();
}

// Few new tokens (T <= G of 1, 2 or 4, or 8 at D = 64): G * D / 16 lanes take
// a block, so that a warp holds several and no lane waits at a barrier.  Bound
// by latency (plan, block table, the block's scale): one token 2.3 us, 64
// sequences 2.6, of which the bytes take 0.2.
constexpr int FEW_THREADS = 128;
template <typename T, bool IL, int D, int G, bool NORM>
__global__ void __launch_bounds__(FEW_THREADS) k_rope_append_few(const __grid_constant__ Args a) {
  using E = typename T::type;
  constexpr int U = D / 16, L = G * U;  // lanes per block
  pdl::trigger();
  pdl::wait();
  if ((int)blockIdx.x < a.q_blocks) {
    turn_q<T, IL, D, NORM>(a, (int64_t)blockIdx.x * FEW_THREADS + threadIdx.x);
    return;
  }
  int i = (((int)blockIdx.x - a.q_blocks) * FEW_THREADS + (int)threadIdx.x) / L;
  const bool live = i < a.B * a.W * 2 * a.Hkv;
  i = live ? i : 0;
  const int h = i % a.Hkv;
  i /= a.Hkv;
  const bool is_v = i & 1;
  i >>= 1;
  const int b = i / a.W, l = threadIdx.x % L, u = l % U, r = l / U;
  const Block k = block_of(a, b, i % a.W);
  const bool mine = live && r < k.tokens;
  const Strides st = is_v ? a.sv : a.sk;
  int c0, c1;
  unit_cols<IL>(u, a.rot, c0, c1);
  const int64_t blk = (int64_t)k.pid * a.Hkv + h;
  uint8_t* codes = (is_v ? a.v_codes : a.k_codes) + blk * a.page * D;
  float* scale = (is_v ? a.v_scale : a.k_scale) + blk;
  float x0[8], x1[8], was = 0.0f, m = 0.0f;
  if (mine) {
    const E* p = reinterpret_cast<const E*>(is_v ? a.v : a.k) + b * st.b + (k.t0 + r) * st.t + h * st.h;
    T::load8(p + c0, x0);
    T::load8(p + c1, x1);
    if (NORM && !is_v && a.k_norm) head_norm<T, U>(x0, x1, a.k_norm, c0, c1, a.eps);
    if (!is_v && u * 16 < a.rot) {
      float c[8], s[8];
      load_angles(a.table + (k.pos + r) * (a.rot >> 1), u, a.rot, c, s);
      turn<IL>(x0, x1, c, s);
    }
    m = amax16(x0, x1, 0.0f);
  }
  if (live && k.tokens > 0 && k.slot0) was = *scale;
#pragma unroll
  for (int d = L / 2; d; d >>= 1) m = fmaxf(m, __shfl_xor_sync(FULL, m, d));
  const float s = fmaxf(pow2_scale(m), was), inv = __fdiv_rn(1.0f, s);
  if (mine) store_codes(codes + (k.slot0 + r) * D, c0, c1, x0, x1, inv);
  __syncwarp();  // every lane has read the old scale before one writes the new
  if (live && k.tokens > 0) {
    if (k.slot0 && s != was)
      for (int c = l; c < k.slot0 * U; c += L) rescale16(reinterpret_cast<uint4*>(codes) + c, was * inv);
    if (l == 0) *scale = s;
  }
}

template <typename T, bool IL, int D, int TH, bool NORM>
void launch_cache(const Args& a, unsigned n, int64_t& blocks, cudaStream_t st) {
  if (!tc::allow_smem<k_rope_append<T, IL, D, TH, NORM>>(Ring<T, TH>::BYTES) ||
      !pdl::launch<k_rope_append<T, IL, D, TH, NORM>>(n, TH, Ring<T, TH>::BYTES, st, 1, a))
    blocks = -1;
}
// blocks: of the largest launch (2^31 or more: nothing launched), -1: a CUDA call failed.
template <typename T, bool IL, int D, bool NORM>
void launch_d(Args& a, int64_t& blocks, cudaStream_t st) {
  const int64_t items = (int64_t)a.B * a.W * 2 * a.Hkv;
  auto q_ctas = [&](int th) {
    return ((int64_t)a.B * a.T * ((a.H + a.hq - 1) / a.hq) * (D / 16) + th - 1) / th;
  };
  a.hq = QH;
  const int per_warp = 512 / D;  // tokens a warp holds
  if (a.T <= per_warp) {
    const int g = a.T == 1 ? 1 : a.T == 2 ? 2 : a.T <= 4 ? 4 : 8;
    blocks = q_ctas(FEW_THREADS) + (items * g * (D / 16) + FEW_THREADS - 1) / FEW_THREADS;
    if (blocks >= (1ll << 31)) return;
    a.q_blocks = (int)q_ctas(FEW_THREADS);
    const unsigned n = (unsigned)blocks;
    const bool ok = g == 1   ? pdl::launch<k_rope_append_few<T, IL, D, 1, NORM>>(n, FEW_THREADS, 0, st, 1, a)
                    : g == 2 ? pdl::launch<k_rope_append_few<T, IL, D, 2, NORM>>(n, FEW_THREADS, 0, st, 1, a)
                    : g == 4 ? pdl::launch<k_rope_append_few<T, IL, D, 4, NORM>>(n, FEW_THREADS, 0, st, 1, a)
                             : pdl::launch<k_rope_append_few<T, IL, D, 512 / D, NORM>>(n, FEW_THREADS, 0, st, 1, a);
    if (!ok) blocks = -1;
    return;
  }
  // more heads per thread and per CTA while the SMs are filled all the same:
  // twice over by the q part, in 8 CTAs each by the cache part
  const int sms = vq::mx::sm_count();
  while (a.hq < a.H && q_ctas(Q_THREADS) >= 12 * sms) a.hq *= 2;
  a.hc = 1;
  while (a.hc < 4 && a.hc < a.Hkv && items / (2 * a.hc) >= 8 * sms) a.hc *= 2;
  blocks = std::max(q_ctas(Q_THREADS), (int64_t)a.B * a.W * 2 * ((a.Hkv + a.hc - 1) / a.hc));
  if (blocks >= (1ll << 31)) return;
  if (!tc::allow_smem<k_turn_q<T, IL, D, NORM>>(Ring<T, Q_THREADS>::BYTES) ||
      !pdl::launch<k_turn_q<T, IL, D, NORM>, false>((unsigned)q_ctas(Q_THREADS), Q_THREADS, Ring<T, Q_THREADS>::BYTES, st, 1, a)) {
    blocks = -1;
    return;
  }
  const unsigned n = (unsigned)(a.B * a.W * 2 * ((a.Hkv + a.hc - 1) / a.hc));
  if (a.page == 32)
    launch_cache<T, IL, D, D, NORM>(a, n, blocks, st);
  else if (a.page == 64)
    launch_cache<T, IL, D, 2 * D, NORM>(a, n, blocks, st);
  else
    launch_cache<T, IL, D, 4 * D, NORM>(a, n, blocks, st);
}
template <typename T, bool NORM>
void launch_norm(Args& a, int D, int64_t& blocks, cudaStream_t st) {
  if (D == 128)
    a.interleaved ? launch_d<T, true, 128, NORM>(a, blocks, st) : launch_d<T, false, 128, NORM>(a, blocks, st);
  else
    a.interleaved ? launch_d<T, true, 64, NORM>(a, blocks, st) : launch_d<T, false, 64, NORM>(a, blocks, st);
}
template <typename T>
void launch(Args& a, int D, int64_t& blocks, cudaStream_t st) {
  a.q_norm || a.k_norm ? launch_norm<T, true>(a, D, blocks, st) : launch_norm<T, false>(a, D, blocks, st);
}

// ---- the cache in 4 bits ----------------------------------------------------
//
// Codes [pages, kv_heads, page, D / 2], two E2M1 values a byte (the even column
// in the low half), and one E4M3 scale per 16 columns of a token [pages,
// kv_heads, page, D / 16]; a value is code * scale * the head's float32 factor f.
//
//   scale = E4M3(max|x| / (6 f)), at least 2^-9;  code = E2M1(x / (scale f))
//
// Both round to nearest, ties to even, and saturate; a NaN makes its block's
// scale NaN.  A token's blocks are its own: nothing that the cache holds is read
// or changed, and a thread needs no more than its neighbour's maximum.
//
// A quotient is q = x r with one correction by its remainder, q + (x - q d) r
// (Markstein 1990), r the divisor's reciprocal to about 2^-22: a quotient that
// float32 holds, as ties between two codes are, comes out exactly, since its error
// falls to 2^-44, and bf16 values meet ties often.  Divisors lie within 2^-126 .. 2^126.

__device__ __forceinline__ float reciprocal(float d) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(d));
  return r;
}
// turn() with two columns an instruction.
template <bool IL>
__device__ __forceinline__ void turn4(float (&x0)[8], float (&x1)[8], const float (&c)[8], const float (&s)[8]) {
  if (IL) return turn<IL>(x0, x1, c, s);
#pragma unroll
  for (int i = 0; i < 8; i += 2) {
    const float2 a = make_float2(x0[i], x0[i + 1]), b = make_float2(x1[i], x1[i + 1]);
    const float2 cc = make_float2(c[i], c[i + 1]), ss = make_float2(s[i], s[i + 1]), ns = make_float2(-s[i], -s[i + 1]);
    const float2 p = __ffma2_rn(a, cc, __fmul2_rn(b, ns)), q = __ffma2_rn(a, ss, __fmul2_rn(b, cc));
    x0[i] = p.x, x0[i + 1] = p.y, x1[i] = q.x, x1[i + 1] = q.y;
  }
}
// 8 values, their quotients by d, as codes: 4 bytes.  `finite`: the correction's
// products stay in float32; a block with quotients beyond goes without it, and those
// saturate all the same.
__device__ __forceinline__ uint32_t e2m1_codes(const float (&x)[8], float d, float r, bool finite) {
  float y[8];
  const float2 rr = make_float2(r, r), nd = make_float2(-d, -d);
#pragma unroll
  for (int j = 0; j < 8; j += 2) {
    const float2 v = make_float2(x[j], x[j + 1]);
    float2 q = __fmul2_rn(v, rr);
    if (finite) q = __ffma2_rn(__ffma2_rn(q, nd, v), rr, q);
    y[j] = q.x, y[j + 1] = q.y;
  }
  uint32_t w;
  asm("{\n\t.reg .b8 a, b, c, d;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 a, %2, %1;\n\tcvt.rn.satfinite.e2m1x2.f32 b, %4, %3;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 c, %6, %5;\n\tcvt.rn.satfinite.e2m1x2.f32 d, %8, %7;\n\t"
      "mov.b32 %0, {a, b, c, d};\n\t}"
      : "=r"(w)
      : "f"(y[0]), "f"(y[1]), "f"(y[2]), "f"(y[3]), "f"(y[4]), "f"(y[5]), "f"(y[6]), "f"(y[7]));
  return w;
}
// The largest magnitude; NaN where one is.
__device__ __forceinline__ float amax_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float amax8(const float (&x)[8]) {
  float m = fabsf(x[0]);
#pragma unroll
  for (int j = 1; j < 8; ++j) m = amax_nan(m, fabsf(x[j]));
  return m;
}
// A block's scale byte, what its values are divided by, and that one's reciprocal.
__device__ __forceinline__ uint32_t block_scale4(float amax, float f, float& d, float& r) {
  const float six = 6.0f * f, r6 = reciprocal(six);
  float a;  // from 464 on a quotient saturates, an infinity's too; NaN stays
  asm("min.NaN.f32 %0, %1, %2;" : "=f"(a) : "f"(amax), "f"(1024.0f * six));
  float q = a * r6;
  q = fmaf(fmaf(-q, six, a), r6, q);
  const uint32_t b = max(pack2(q, 0.0f) & 0xFFu, 1u);
  d = half2f(unpack2(b)).x * f;
  r = reciprocal(d);
  return b;
}
// One unit's 16 columns of a key or value head to its token's place.  `split`:
// the unit's two groups of 8 lie in two blocks, whose other halves are the
// units of other lanes of the head (group g of a turned head is the first of
// lane g, or the second of lane g - R).
template <int U>
__device__ __forceinline__ void store4(uint8_t* codes, uint8_t* scale, const float (&x0)[8], const float (&x1)[8],
                                       float f, int u, int rot, bool split, bool store) {
  float m0 = amax8(x0), m1 = amax8(x1);
  const int R = rot >> 4;
  if (split) {
    const int lane = threadIdx.x & 31, first = lane & ~(U - 1);
    const uint32_t lanes = ((1u << U) - 1) << first;
    // every lane of the head asks; those past the turned columns keep their own
    const bool turned = u < R;
    const int p0 = turned ? u ^ 1 : 0, p1 = turned ? (u + R) ^ 1 : 0;
    const int s0 = first + (p0 < R ? p0 : p0 - R), s1 = first + (p1 < R ? p1 : p1 - R);
    const float a0 = __shfl_sync(lanes, m0, s0), a1 = __shfl_sync(lanes, m1, s0);
    const float b0 = __shfl_sync(lanes, m0, s1), b1 = __shfl_sync(lanes, m1, s1);
    const float n0 = amax_nan(m0, p0 < R ? a0 : a1), n1 = amax_nan(m1, p1 < R ? b0 : b1), n = amax_nan(m0, m1);
    m0 = turned ? n0 : n, m1 = turned ? n1 : n;
    split = turned;
  } else {
    m0 = m1 = amax_nan(m0, m1);
  }
  if (!store) return;
  float d0, d1, r0, r1;
  const uint32_t e0 = block_scale4(m0, f, d0, r0);
  uint32_t e1 = e0;
  if (split)
    e1 = block_scale4(m1, f, d1, r1);
  else
    d1 = d0, r1 = r0;
  const uint32_t w0 = e2m1_codes(x0, d0, r0, m0 < 0x1p100f * d0), w1 = e2m1_codes(x1, d1, r1, m1 < 0x1p100f * d1);
  if (split) {
    const int g1 = u + R;
    reinterpret_cast<uint32_t*>(codes)[u] = w0;
    reinterpret_cast<uint32_t*>(codes)[g1] = w1;
    if (!(u & 1)) scale[u >> 1] = (uint8_t)e0;
    if (!(g1 & 1)) scale[g1 >> 1] = (uint8_t)e1;
  } else {
    reinterpret_cast<uint2*>(codes)[u] = make_uint2(w0, w1);
    scale[u] = (uint8_t)e0;
  }
}

// Few heads in all: thread `i` takes its unit of one head of a token, the heads of
// q, k and v counted on.
struct Unit4 {
  int u, h, b, t;
  int64_t row;
};
template <int D>
__device__ __forceinline__ Unit4 unit4(const Args& a, int64_t i) {
  constexpr int U = D / 16;
  Unit4 x;
  x.u = (int)(i % U);
  const int64_t rows = (int64_t)a.B * a.T, r = i / U;
  x.h = (int)min(r / rows, (int64_t)(a.H + 2 * a.Hkv));
  x.row = r - r / rows * rows;
  x.b = (int)(x.row / a.T), x.t = (int)(x.row - (int64_t)x.b * a.T);
  return x;
}
// Where a head's unit lies: its row, and the first columns of its two groups.
// Values do not turn, so their units are 16 columns that lie side by side.
template <typename T, bool IL>
__device__ __forceinline__ const typename T::type* head_row(const Args& a, const Unit4& x, int h, int& c0, int& c1) {
  using E = typename T::type;
  const bool is_v = h >= a.H + a.Hkv, is_k = h >= a.H && !is_v;
  unit_cols<IL>(x.u, is_v ? 0 : a.rot, c0, c1);
  const Strides& s = is_v ? a.sv : is_k ? a.sk : a.sq;
  const E* p = reinterpret_cast<const E*>(is_v ? a.v : is_k ? a.k : a.q);
  return p + x.b * s.b + x.t * s.t + (h - (is_v ? a.H + a.Hkv : is_k ? a.H : 0)) * s.h;
}
// A token's place: live, its slot of the cache (-1: none) and its angles.
struct Token4 {
  bool live, turns;
  int64_t slot;  // (page * Hkv) * page size + place in it
  float c[8], s[8];
};
__device__ __forceinline__ Token4 token4(const Args& a, const Unit4& x) {
  Token4 k;
  int held;
  k.live = x.t < plan(a, x.b, held);
  k.turns = k.live && x.u * 16 < a.rot;
  k.slot = -1;
  if (k.turns) load_angles(a.table + (int64_t)(held + x.t) * (a.rot >> 1), x.u, a.rot, k.c, k.s);
  if (k.live && x.h >= a.H) {
    const int pos = held + x.t, at = pos / a.page;
    const int pid = a.block_table[(int64_t)x.b * a.width + at];
    if (pid < 0 || pid >= a.pages)
      tc::note_err(nullptr, ERR_PAGE);
    else
      k.slot = (int64_t)pid * a.Hkv * a.page + (pos - at * a.page);
  }
  return k;
}
template <typename T, bool IL, int D, bool NORM>
__device__ __forceinline__ void finish4(const Args& a, const Unit4& x, const Token4& k, int h, int c0, int c1,
                                        float (&x0)[8], float (&x1)[8]) {
  constexpr int U = D / 16;
  const bool is_q = h < a.H, is_v = h >= a.H + a.Hkv;
  if (!is_v) {
    const void* w = is_q ? a.q_norm : a.k_norm;
    if (NORM && w) head_norm<T, U>(x0, x1, w, c0, c1, a.eps);
    if (k.turns) turn4<IL>(x0, x1, k.c, k.s);
  }
  if (is_q) {
    if (!k.live) {
#pragma unroll
      for (int j = 0; j < 8; ++j) x0[j] = x1[j] = 0.0f;
    }
    store_unit<T>(reinterpret_cast<typename T::type*>(a.q_out) + (x.row * a.H + h) * D, c0, c1, x0, x1);
  } else {
    const int kvh = h - a.H - (is_v ? a.Hkv : 0);
    const int64_t at = (k.slot < 0 ? 0 : k.slot) + (int64_t)kvh * a.page;
    store4<U>((is_v ? a.v_codes : a.k_codes) + at * (D / 2), (is_v ? a.v_bscale : a.k_bscale) + at * U, x0, x1,
              __ldg((is_v ? a.v_factor : a.k_factor) + kvh), x.u, a.rot, !IL && !is_v, k.slot >= 0);
  }
}

// Bound by latency: the plan, the block table, the heads, the angles.  One token, 8 x 4
// heads of 128: 1.9 us; 96 sequences, normalised: 4.1 us (floor 0.3).
template <typename T, bool IL, int D, bool NORM>
__global__ void __launch_bounds__(FEW_THREADS) k_append4_few(const __grid_constant__ Args a) {
  pdl::trigger();
  pdl::wait();
  const Unit4 x = unit4<D>(a, (int64_t)blockIdx.x * FEW_THREADS + threadIdx.x);
  if (x.h >= a.H + 2 * a.Hkv) return;
  int c0, c1;
  const typename T::type* p = head_row<T, IL>(a, x, x.h, c0, c1);
  float x0[8], x1[8];
  T::load8(p + c0, x0);
  T::load8(p + c1, x1);
  const Token4 k = token4(a, x);
  finish4<T, IL, D, NORM>(a, x, k, x.h, c0, c1, x0, x1);
}

// Many: the keys and values beside k_turn_q, half of the CTAs each; a thread takes
// its unit of a.hc heads of a token, QH at a time, whose loads travel through a ring.
// The tokens of a warp are neighbours, so that their codes and scales fill sectors.
// Bound by latency: 227 instructions a unit of 16 columns (rotation, maxima, quotients
// with their correction), one after the other, a third of an SM's warps, issue slots 50
// to 59 % busy.  8 x 2048 tokens, 32 heads of 128: 126 us with k_turn_q's 39, floor 94, with
// norms 146; 8 x 4 heads: 66, floor 55, with norms 74, interleaved 92, in float32 187 (floor
// 107).  The forms with norms spill 8 to 16 bytes a thread at 80 registers.
template <typename T, bool IL, int D, bool NORM>
__global__ void __launch_bounds__(Q_THREADS, 3) k_append4(const __grid_constant__ Args a) {
  using E = typename T::type;
  constexpr int U = D / 16;
  extern __shared__ __align__(16) uint8_t smem[];
  const Ring<T, Q_THREADS> ring(smem);
  pdl::trigger();
  const bool is_v = blockIdx.x & 1;
  const int64_t i = (int64_t)(blockIdx.x >> 1) * Q_THREADS + threadIdx.x, rows = (int64_t)a.B * a.T, at = i / U;
  const int u = (int)(i % U), h0 = (int)min(at / rows * a.hc, (int64_t)a.Hkv), h1 = min(a.Hkv, h0 + a.hc);
  const int64_t row = at % rows;
  const int b = (int)(row / a.T), t = (int)(row - (int64_t)b * a.T);
  int held, pid = -1, pos = 0;
  if (h0 < h1 && t < plan(a, b, held)) {
    pos = held + t;
    pid = a.block_table[(int64_t)b * a.width + pos / a.page];
    if (pid < 0 || pid >= a.pages) tc::note_err(nullptr, ERR_PAGE), pid = -1;
  }
  // a token's U lanes go together; k_turn_q, launched before this kernel, shares
  // nothing with it, so only the end waits
  if (pid >= 0) {
    const Strides st = is_v ? a.sv : a.sk;
    const E* src = reinterpret_cast<const E*>(is_v ? a.v : a.k) + b * st.b + t * st.t;
    int c0, c1;
    unit_cols<IL>(u, is_v ? 0 : a.rot, c0, c1);
    const int steps = (h1 - h0 + QH - 1) / QH;
    auto fetch = [&](int k) {
      if (k < steps) {
#pragma unroll
        for (int q = 0; q < QH; ++q) {
          const E* p = src + min(h0 + k * QH + q, h1 - 1) * st.h;
          ring.fetch(k, 2 * q, p + c0);
          ring.fetch(k, 2 * q + 1, p + c1);
        }
      }
      ring.commit();
    };
#pragma unroll
    for (int k = 0; k < Ring<T, Q_THREADS>::DEPTH - 1; ++k) fetch(k);
    const bool turns = !is_v && u * 16 < a.rot;
    float c[8], s[8];
    if (turns) load_angles(a.table + (int64_t)pos * (a.rot >> 1), u, a.rot, c, s);
    const int64_t slot = (int64_t)pid * a.Hkv * a.page + pos % a.page;
    uint8_t* codes = (is_v ? a.v_codes : a.k_codes) + slot * (D / 2);
    uint8_t* scale = (is_v ? a.v_bscale : a.k_bscale) + slot * U;
    const float* factor = is_v ? a.v_factor : a.k_factor;
    for (int k = 0; k < steps; ++k) {
      fetch(k + Ring<T, Q_THREADS>::DEPTH - 1);
      ring.wait();
#pragma unroll
      for (int q = 0; q < QH; ++q) {
        const int h = h0 + k * QH + q;
        float x0[8], x1[8];
        ring.read(k, 2 * q, x0);
        ring.read(k, 2 * q + 1, x1);
        if (h < h1) {
          if (NORM && !is_v && a.k_norm) head_norm<T, U>(x0, x1, a.k_norm, c0, c1, a.eps);
          if (turns) turn4<IL>(x0, x1, c, s);
          const int64_t on = (int64_t)h * a.page;
          store4<U>(codes + on * (D / 2), scale + on * U, x0, x1, __ldg(factor + h), u, a.rot, !IL && !is_v, true);
        }
      }
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
  }
  pdl::wait();
}

template <typename T, bool IL, int D, bool NORM>
void launch4_d(Args& a, int64_t& blocks, cudaStream_t st) {
  const int all = a.H + 2 * a.Hkv, sms = vq::mx::sm_count();
  auto ctas = [&](int heads, int each, int th) {
    return ((int64_t)a.B * a.T * ((heads + each - 1) / each) * (D / 16) + th - 1) / th;
  };
  a.hq = 1;
  blocks = ctas(all, 1, FEW_THREADS);
  if (blocks <= 16 * sms) {
    if (!pdl::launch<k_append4_few<T, IL, D, NORM>>((unsigned)blocks, FEW_THREADS, 0, st, 1, a)) blocks = -1;
    return;
  }
  // more heads per thread while the SMs are filled all the same, twice over by each
  // part; beyond 16 keys and values only lengthen the last CTAs (32 heads, 8 x 2048
  // tokens: 133 us with 32 a thread, 128 with 16)
  a.hq = a.hc = QH;
  while (a.hq < a.H && ctas(a.H, a.hq, Q_THREADS) >= 12 * sms) a.hq *= 2;
  while (a.hc < std::min(a.Hkv, 16) && ctas(a.Hkv, a.hc, Q_THREADS) >= 6 * sms) a.hc *= 2;
  const int64_t nq = ctas(a.H, a.hq, Q_THREADS), nc = 2 * ctas(a.Hkv, a.hc, Q_THREADS);
  blocks = std::max(nq, nc);
  if (blocks >= (1ll << 31)) return;
  constexpr int BYTES = Ring<T, Q_THREADS>::BYTES;
  if (!tc::allow_smem<k_turn_q<T, IL, D, NORM>>(BYTES) || !tc::allow_smem<k_append4<T, IL, D, NORM>>(BYTES) ||
      !pdl::launch<k_turn_q<T, IL, D, NORM>, false>((unsigned)nq, Q_THREADS, BYTES, st, 1, a) ||
      !pdl::launch<k_append4<T, IL, D, NORM>>((unsigned)nc, Q_THREADS, BYTES, st, 1, a))
    blocks = -1;
}
template <typename T, bool IL, int D>
void launch4_n(Args& a, int64_t& blocks, cudaStream_t st) {
  a.q_norm || a.k_norm ? launch4_d<T, IL, D, true>(a, blocks, st) : launch4_d<T, IL, D, false>(a, blocks, st);
}
template <typename T>
void launch4(Args& a, int D, int64_t& blocks, cudaStream_t st) {
  if (D == 128)
    a.interleaved ? launch4_n<T, true, 128>(a, blocks, st) : launch4_n<T, false, 128>(a, blocks, st);
  else
    a.interleaved ? launch4_n<T, true, 64>(a, blocks, st) : launch4_n<T, false, 64>(a, blocks, st);
}

// E2M1 codes as E4M3 codes of the same values: the magnitudes from a table of
// eight bytes (0, .5, 1, 1.5, 2, 3, 4, 6), the sign moved.  Bound by HBM, mostly
// writes: 8 x 2048 tokens' pool (8 x 34 pages of 64, 32 heads of 128) 36 us, 6 TB/s.
__device__ __forceinline__ uint32_t e2m1_to_e4m3(uint32_t nib4) {  // four codes, one in each byte's low half
  const uint32_t lo = 0x3C383000u, hi = 0x4C484440u;
  const uint32_t sel = nib4 & 0x07070707u;
  const uint32_t s16 = (sel & 0x7u) | ((sel >> 4) & 0x70u) | ((sel >> 8) & 0x700u) | ((sel >> 12) & 0x7000u);
  return __byte_perm(lo, hi, s16) | ((nib4 & 0x08080808u) << 4);
}
constexpr int UNPACK_THREADS = 256, UNPACK = 4;  // chunks a thread and turn, all loads in flight together
__global__ void __launch_bounds__(UNPACK_THREADS)
    k_unpack4(const uint4* k, const uint4* v, uint4* ko, uint4* vo, int64_t chunks) {
  pdl::trigger();
  pdl::wait();
  const bool second = blockIdx.x & 1;  // the values
  const uint4* in = second ? v : k;
  uint4* out = second ? vo : ko;
  const int64_t step = (int64_t)(gridDim.x >> 1) * (UNPACK_THREADS * UNPACK);
  for (int64_t i = (int64_t)(blockIdx.x >> 1) * (UNPACK_THREADS * UNPACK) + threadIdx.x; i < chunks; i += step) {
    uint4 w[UNPACK];
#pragma unroll
    for (int n = 0; n < UNPACK; ++n)
      w[n] = i + n * UNPACK_THREADS < chunks ? __ldg(in + i + n * UNPACK_THREADS) : make_uint4(0, 0, 0, 0);
#pragma unroll
    for (int n = 0; n < UNPACK; ++n) {
      const uint32_t x[4] = {w[n].x, w[n].y, w[n].z, w[n].w};
      uint32_t o[8];
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const uint32_t even = e2m1_to_e4m3(x[q] & 0x0F0F0F0Fu), odd = e2m1_to_e4m3((x[q] >> 4) & 0x0F0F0F0Fu);
        o[2 * q] = __byte_perm(even, odd, 0x5140), o[2 * q + 1] = __byte_perm(even, odd, 0x7362);
      }
      if (i + n * UNPACK_THREADS < chunks)
        asm volatile("st.global.v8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"l"(out + 2 * (i + n * UNPACK_THREADS)),
                     "r"(o[0]), "r"(o[1]), "r"(o[2]), "r"(o[3]), "r"(o[4]), "r"(o[5]), "r"(o[6]), "r"(o[7]) : "memory");
    }
  }
}

// This file's sticky word (vq_device_errors).
int sticky_kv(int* out, int clear, cudaStream_t st) { return vq::tc::sticky_read(out, clear, st); }

}  // namespace kv
}  // namespace vq

using namespace vq::kv;

// What both caches' entry points check and take alike.  `align_v`: the codes'.
static int arguments(Args& a, const void* q, const void* k, const void* v, const int64_t* strides, int32_t dtype,
                     const float* table, int64_t positions, int32_t rot, int32_t interleaved, int64_t batch,
                     int64_t tokens, int32_t heads, int32_t kv_heads, int32_t head_dim, const void* block_table,
                     int64_t table_width, const void* lengths, const void* counts, int64_t pages, int32_t page,
                     const void* q_norm, const void* k_norm, float eps, void* q_out, void* k_codes, void* v_codes,
                     const void* k_scale, const void* v_scale, bool& none) {
  if (dtype != VQ_BF16 && dtype != VQ_F32) return VQ_ERR_UNSUPPORTED;
  if (head_dim != 64 && head_dim != 128) return VQ_ERR_UNSUPPORTED;
  if (page != 32 && page != 64 && page != 128) return VQ_ERR_UNSUPPORTED;
  if (batch < 0 || tokens < 0 || heads <= 0 || kv_heads <= 0 || heads % kv_heads || rot < 16 ||
      rot > head_dim || rot % 16 || table_width < 0 || pages < 0 || batch > (1 << 24) ||
      tokens > (1 << 24) || table_width > (1 << 24) || pages * kv_heads * page >= (1ll << 31))
    return VQ_ERR_INVALID;
  none = batch == 0 || tokens == 0;
  if (none) return VQ_OK;
  if (!q || !k || !v || !strides || !lengths || !q_out) return VQ_ERR_NULL;
  // a table of no columns and a cache of no pages are not read: may be null
  if (table_width && (!table || !block_table)) return VQ_ERR_NULL;
  if (pages && (!k_codes || !v_codes || !k_scale || !v_scale)) return VQ_ERR_NULL;
  if (positions < table_width * page) return VQ_ERR_SHAPE;  // every position the plan can name
  const int eb = dtype == VQ_BF16 ? 2 : 4;
  const void* p16[9] = {q, k, v, q_out, k_codes, v_codes, table, q_norm, k_norm};
  for (const void* p : p16)
    if (reinterpret_cast<uintptr_t>(p) & 15) return VQ_ERR_ALIGNMENT;
  if (reinterpret_cast<uintptr_t>(q_out) & 31) return VQ_ERR_ALIGNMENT;
  for (int i = 0; i < 9; ++i)
    if (strides[i] * eb % 16) return VQ_ERR_ALIGNMENT;
  a = {};
  a.q = q, a.k = k, a.v = v;
  a.sq = {strides[0], strides[1], strides[2]};
  a.sk = {strides[3], strides[4], strides[5]};
  a.sv = {strides[6], strides[7], strides[8]};
  a.table = reinterpret_cast<const float2*>(table);
  a.q_out = q_out;
  a.k_codes = (uint8_t*)k_codes, a.v_codes = (uint8_t*)v_codes;
  a.block_table = (const int32_t*)block_table;
  a.lengths = (const int32_t*)lengths;
  a.counts = (const int32_t*)counts;
  a.B = (int)batch, a.T = (int)tokens, a.H = heads, a.Hkv = kv_heads;
  a.rot = rot, a.page = page, a.width = (int)table_width, a.pages = (int)pages;
  a.interleaved = interleaved;
  a.q_norm = q_norm, a.k_norm = k_norm, a.eps = eps;
  return VQ_OK;
}

extern "C" {

int vq_rope_append_kv8_norm(const void* q, const void* k, const void* v, const int64_t* strides,
                            int32_t dtype, const float* table, int64_t positions, int32_t rot,
                            int32_t interleaved, int64_t batch, int64_t tokens, int32_t heads,
                            int32_t kv_heads, int32_t head_dim, const void* block_table,
                            int64_t table_width, const void* lengths, const void* counts,
                            int64_t pages, int32_t page, const void* q_norm, const void* k_norm, float eps,
                            void* q_out, void* k_codes, void* v_codes, float* k_scale, float* v_scale,
                            void* stream) {
  Args a;
  bool none;
  const int bad = arguments(a, q, k, v, strides, dtype, table, positions, rot, interleaved, batch, tokens, heads,
                            kv_heads, head_dim, block_table, table_width, lengths, counts, pages, page, q_norm,
                            k_norm, eps, q_out, k_codes, v_codes, k_scale, v_scale, none);
  if (bad || none) return bad;
  a.k_scale = k_scale, a.v_scale = v_scale;
  a.W = (int)((tokens - 1 + page - 1) / page) + 1;
  if (batch * a.W * 2 * kv_heads >= (1ll << 26)) return VQ_ERR_INVALID;  // items times 32 lanes in 31 bits
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  int64_t blocks = 0;
  if (dtype == VQ_BF16)
    launch<BF16>(a, head_dim, blocks, st);
  else
    launch<F32>(a, head_dim, blocks, st);
  if (blocks < 0) return VQ_ERR_CUDA;
  if (blocks >= (1ll << 31)) return VQ_ERR_INVALID;
  return VQ_OK;
}

int vq_rope_append_kv8(const void* q, const void* k, const void* v, const int64_t* strides,
                       int32_t dtype, const float* table, int64_t positions, int32_t rot,
                       int32_t interleaved, int64_t batch, int64_t tokens, int32_t heads,
                       int32_t kv_heads, int32_t head_dim, const void* block_table,
                       int64_t table_width, const void* lengths, const void* counts, int64_t pages,
                       int32_t page, void* q_out, void* k_codes, void* v_codes, float* k_scale,
                       float* v_scale, void* stream) {
  return vq_rope_append_kv8_norm(q, k, v, strides, dtype, table, positions, rot, interleaved, batch, tokens, heads,
                                 kv_heads, head_dim, block_table, table_width, lengths, counts, pages, page, nullptr,
                                 nullptr, 0.0f, q_out, k_codes, v_codes, k_scale, v_scale, stream);
}

int vq_rope_append_kv4(const void* q, const void* k, const void* v, const int64_t* strides,
                       int32_t dtype, const float* table, int64_t positions, int32_t rot,
                       int32_t interleaved, int64_t batch, int64_t tokens, int32_t heads,
                       int32_t kv_heads, int32_t head_dim, const void* block_table,
                       int64_t table_width, const void* lengths, const void* counts, int64_t pages,
                       int32_t page, const void* q_norm, const void* k_norm, float eps, void* q_out,
                       void* k_codes, void* v_codes, void* k_scale, void* v_scale, const float* k_factor,
                       const float* v_factor, void* stream) {
  Args a;
  bool none;
  const int bad = arguments(a, q, k, v, strides, dtype, table, positions, rot, interleaved, batch, tokens, heads,
                            kv_heads, head_dim, block_table, table_width, lengths, counts, pages, page, q_norm,
                            k_norm, eps, q_out, k_codes, v_codes, k_scale, v_scale, none);
  if (bad || none) return bad;
  if (!k_factor || !v_factor) return VQ_ERR_NULL;
  a.k_bscale = (uint8_t*)k_scale, a.v_bscale = (uint8_t*)v_scale;
  a.k_factor = k_factor, a.v_factor = v_factor;
  if (heads > (1 << 20) || batch * tokens >= (1ll << 31)) return VQ_ERR_INVALID;  // heads and tokens in 31 bits
  int64_t blocks = 0;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  if (dtype == VQ_BF16)
    launch4<BF16>(a, head_dim, blocks, st);
  else
    launch4<F32>(a, head_dim, blocks, st);
  if (blocks < 0) return VQ_ERR_CUDA;
  if (blocks >= (1ll << 31)) return VQ_ERR_INVALID;
  return VQ_OK;
}

int vq_kv4_unpack(const void* k_codes, const void* v_codes, int64_t bytes, void* k_out, void* v_out, void* stream) {
  if (bytes < 0 || bytes % 16) return VQ_ERR_INVALID;
  if (bytes == 0) return VQ_OK;
  if (!k_codes || !v_codes || !k_out || !v_out) return VQ_ERR_NULL;
  const void* p16[4] = {k_codes, v_codes, k_out, v_out};
  for (const void* p : p16)
    if (reinterpret_cast<uintptr_t>(p) & 15) return VQ_ERR_ALIGNMENT;
  if ((reinterpret_cast<uintptr_t>(k_out) | reinterpret_cast<uintptr_t>(v_out)) & 31) return VQ_ERR_ALIGNMENT;
  const int64_t chunks = bytes / 16, ctas = (chunks + UNPACK_THREADS * UNPACK - 1) / (UNPACK_THREADS * UNPACK);
  const unsigned n = 2 * (unsigned)std::min<int64_t>(ctas, 4 * vq::mx::sm_count());
  return vq::pdl::launch<k_unpack4>(n, UNPACK_THREADS, 0, reinterpret_cast<cudaStream_t>(stream), 1,
                                    (const uint4*)k_codes, (const uint4*)v_codes, (uint4*)k_out, (uint4*)v_out, chunks)
             ? VQ_OK
             : VQ_ERR_CUDA;
}

}  // extern "C"
