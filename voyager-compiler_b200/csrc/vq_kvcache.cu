// Rotary positions and the append to a paged key / value cache held in E4M3.
//
// The cache: codes [pages, kv_heads, page, D] E4M3 bytes and one float32
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
// written once) and by latency for single tokens.
#include <cuda_runtime.h>
#include <stdint.h>

#include <algorithm>

#include "voyager_b200.h"
#include "vq_e4m3.cuh"
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

// Load and rotate the unit: x0 / x1 hold columns c0.. / c1.. after it.
template <typename T, bool IL>
__device__ __forceinline__ void load_unit(const typename T::type* p, const float2* cs, int u, int rot,
                                          float (&x0)[8], float (&x1)[8], int& c0, int& c1) {
  unit_cols<IL>(u, rot, c0, c1);
  T::load8(p + c0, x0);
  T::load8(p + c1, x1);
  if (cs && u * 16 < rot) {
    const float4* t = reinterpret_cast<const float4*>(cs + u * 8);
    float c[8], s[8];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float4 f = __ldg(t + i);
      c[2 * i] = f.x, s[2 * i] = f.y, c[2 * i + 1] = f.z, s[2 * i + 1] = f.w;
    }
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

constexpr int THREADS = 256;

template <typename T, bool IL, int D, int IT>
__global__ void __launch_bounds__(THREADS) k_rope_append(const Args a) {
  using E = typename T::type;
  constexpr int U = D / 16;            // threads per head row
  constexpr int ROWS = THREADS / U;    // rows per pass
  if ((int)blockIdx.x < a.q_blocks) {
    // ---- q: one unit per thread ----
    const int64_t i = (int64_t)blockIdx.x * THREADS + threadIdx.x;
    const int u = (int)(i % U);
    int64_t r = i / U;
    const int64_t row = r;
    if (row >= (int64_t)a.B * a.T * a.H) return;
    const int h = (int)(r % a.H);
    r /= a.H;
    const int t = (int)(r % a.T), b = (int)(r / a.T);
    int held;
    const int n = plan(a, b, held);
    E* out = reinterpret_cast<E*>(a.q_out) + row * D;
    float x0[8], x1[8];
    int c0, c1;
    if (t < n) {
      const E* p = reinterpret_cast<const E*>(a.q) + b * a.sq.b + t * a.sq.t + h * a.sq.h;
      load_unit<T, IL>(p, a.table + (int64_t)(held + t) * (a.rot >> 1), u, a.rot, x0, x1, c0, c1);
    } else {
      unit_cols<IL>(u, a.rot, c0, c1);
#pragma unroll
      for (int j = 0; j < 8; ++j) x0[j] = x1[j] = 0.0f;
    }
    T::store8(out + c0, x0);
    T::store8(out + c1, x1);
    return;
  }
  // ---- one block (page, head) of the keys or the values per CTA ----
  __shared__ float part[THREADS / 32];
  int64_t i = (int64_t)blockIdx.x - a.q_blocks;
  const int h = (int)(i % a.Hkv);
  i /= a.Hkv;
  const bool is_v = i & 1;
  i >>= 1;
  const int w = (int)(i % a.W), b = (int)(i / a.W);
  int held;
  const int n = plan(a, b, held);
  const int first = held / a.page + w;  // the sequence's page number
  const int64_t lo = max((int64_t)held, (int64_t)first * a.page);
  const int64_t hi = min((int64_t)held + n, (int64_t)(first + 1) * a.page);
  if (lo >= hi) return;
  const int pid = a.block_table[(int64_t)b * a.width + first];
  if (pid < 0 || pid >= a.pages) {
    if (threadIdx.x == 0) tc::note_err(nullptr, ERR_PAGE);
    return;
  }
  const int t0 = (int)(lo - held), tokens = (int)(hi - lo), slot0 = (int)(lo - (int64_t)first * a.page);
  const int u = threadIdx.x % U, r0 = threadIdx.x / U;
  const E* src = is_v ? reinterpret_cast<const E*>(a.v) + b * a.sv.b + h * a.sv.h
                      : reinterpret_cast<const E*>(a.k) + b * a.sk.b + h * a.sk.h;
  const int64_t st = is_v ? a.sv.t : a.sk.t;
  const int64_t blk = (int64_t)pid * a.Hkv + h;
  uint8_t* codes = (is_v ? a.v_codes : a.k_codes) + blk * a.page * D;
  float* scale = (is_v ? a.v_scale : a.k_scale) + blk;
  float x0[IT][8], x1[IT][8];
  int c0, c1;
  unit_cols<IL>(u, a.rot, c0, c1);
  float m = 0.0f;
#pragma unroll
  for (int it = 0; it < IT; ++it) {
    const int r = it * ROWS + r0;
    if (r < tokens) {
      const float2* cs = is_v ? nullptr : a.table + (lo + r) * (a.rot >> 1);
      load_unit<T, IL>(src + (t0 + r) * st, cs, u, a.rot, x0[it], x1[it], c0, c1);
#pragma unroll
      for (int j = 0; j < 8; ++j) m = fmaxf(m, fmaxf(fabsf(x0[it][j]), fabsf(x1[it][j])));
    }
  }
#pragma unroll
  for (int d = 16; d; d >>= 1) m = fmaxf(m, __shfl_xor_sync(FULL, m, d));
  if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = m;
  const float was = slot0 ? *scale : 0.0f;  // slot 0 written now: a fresh block
  __syncthreads();
#pragma unroll
  for (int j = 0; j < THREADS / 32; ++j) m = fmaxf(m, part[j]);
  const float s = fmaxf(pow2_scale(m), was), inv = __fdiv_rn(1.0f, s);  // exact: s is a power of two
#pragma unroll
  for (int it = 0; it < IT; ++it) {
    const int r = it * ROWS + r0;
    if (r < tokens) {
      uint8_t* o = codes + (slot0 + r) * D;
#pragma unroll
      for (int j = 0; j < 8; ++j) x0[it][j] *= inv, x1[it][j] *= inv;
      *reinterpret_cast<uint2*>(o + c0) = make_uint2(pack4(x0[it][0], x0[it][1], x0[it][2], x0[it][3]),
                                                     pack4(x0[it][4], x0[it][5], x0[it][6], x0[it][7]));
      *reinterpret_cast<uint2*>(o + c1) = make_uint2(pack4(x1[it][0], x1[it][1], x1[it][2], x1[it][3]),
                                                     pack4(x1[it][4], x1[it][5], x1[it][6], x1[it][7]));
    }
  }
  if (slot0 && s != was) {  // the tokens that the block holds, at the new scale
    const float f = was * inv;
    for (int c = threadIdx.x; c < slot0 * U; c += THREADS) {
      uint4* p = reinterpret_cast<uint4*>(codes) + c;
      uint4 v = *p;
      uint32_t* wv = reinterpret_cast<uint32_t*>(&v);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float2 l = half2f(unpack2(wv[j])), g = half2f(unpack2_hi(wv[j]));
        wv[j] = pack4(l.x * f, l.y * f, g.x * f, g.y * f);
      }
      *p = v;
    }
  }
  if (threadIdx.x == 0) *scale = s;
}

template <typename T, bool IL, int D>
void launch_it(const Args& a, unsigned grid, cudaStream_t st) {
  const int it = std::max(1, a.page * (D / 16) / THREADS);
  if (it == 1)
    k_rope_append<T, IL, D, 1><<<grid, THREADS, 0, st>>>(a);
  else if (it == 2)
    k_rope_append<T, IL, D, 2><<<grid, THREADS, 0, st>>>(a);
  else
    k_rope_append<T, IL, D, 4><<<grid, THREADS, 0, st>>>(a);
}
template <typename T>
void launch(const Args& a, int D, unsigned grid, cudaStream_t st) {
  if (D == 128)
    a.interleaved ? launch_it<T, true, 128>(a, grid, st) : launch_it<T, false, 128>(a, grid, st);
  else
    a.interleaved ? launch_it<T, true, 64>(a, grid, st) : launch_it<T, false, 64>(a, grid, st);
}

// This file's sticky word (vq_device_errors).
int sticky_kv(int* out, int clear, cudaStream_t st) { return vq::tc::sticky_read(out, clear, st); }

}  // namespace kv
}  // namespace vq

using namespace vq::kv;

extern "C" int vq_rope_append_kv8(const void* q, const void* k, const void* v, const int64_t* strides,
                                  int32_t dtype, const float* table, int64_t positions, int32_t rot,
                                  int32_t interleaved, int64_t batch, int64_t tokens, int32_t heads,
                                  int32_t kv_heads, int32_t head_dim, const void* block_table,
                                  int64_t table_width, const void* lengths, const void* counts,
                                  int64_t pages, int32_t page, void* q_out, void* k_codes,
                                  void* v_codes, float* k_scale, float* v_scale, void* stream) {
  if (dtype != VQ_BF16 && dtype != VQ_F32) return VQ_ERR_UNSUPPORTED;
  if (head_dim != 64 && head_dim != 128) return VQ_ERR_UNSUPPORTED;
  if (page != 32 && page != 64 && page != 128) return VQ_ERR_UNSUPPORTED;
  if (batch < 0 || tokens < 0 || heads <= 0 || kv_heads <= 0 || heads % kv_heads || rot < 16 ||
      rot > head_dim || rot % 16 || table_width < 0 || pages < 0 || batch > (1 << 24) ||
      tokens > (1 << 24) || table_width > (1 << 24) || pages * kv_heads * page >= (1ll << 31))
    return VQ_ERR_INVALID;
  if (batch == 0 || tokens == 0) return VQ_OK;
  if (!q || !k || !v || !strides || !table || !block_table || !lengths || !q_out || !k_codes ||
      !v_codes || !k_scale || !v_scale)
    return VQ_ERR_NULL;
  if (positions < table_width * page) return VQ_ERR_SHAPE;  // every position the plan can name
  const int eb = dtype == VQ_BF16 ? 2 : 4;
  const void* p16[6] = {q, k, v, q_out, k_codes, v_codes};
  for (const void* p : p16)
    if (reinterpret_cast<uintptr_t>(p) & 15) return VQ_ERR_ALIGNMENT;
  if (reinterpret_cast<uintptr_t>(table) & 15) return VQ_ERR_ALIGNMENT;
  for (int i = 0; i < 9; ++i)
    if (strides[i] * eb % 16) return VQ_ERR_ALIGNMENT;
  Args a;
  a.q = q, a.k = k, a.v = v;
  a.sq = {strides[0], strides[1], strides[2]};
  a.sk = {strides[3], strides[4], strides[5]};
  a.sv = {strides[6], strides[7], strides[8]};
  a.table = reinterpret_cast<const float2*>(table);
  a.q_out = q_out;
  a.k_codes = (uint8_t*)k_codes, a.v_codes = (uint8_t*)v_codes;
  a.k_scale = k_scale, a.v_scale = v_scale;
  a.block_table = (const int32_t*)block_table;
  a.lengths = (const int32_t*)lengths;
  a.counts = (const int32_t*)counts;
  a.B = (int)batch, a.T = (int)tokens, a.H = heads, a.Hkv = kv_heads;
  a.rot = rot, a.page = page, a.width = (int)table_width, a.pages = (int)pages;
  a.interleaved = interleaved;
  a.W = (int)((tokens - 1 + page - 1) / page) + 1;
  const int64_t qb = (batch * tokens * heads * (head_dim / 16) + THREADS - 1) / THREADS;
  const int64_t kb = batch * a.W * 2 * kv_heads;
  if (qb + kb >= (1ll << 31)) return VQ_ERR_INVALID;
  a.q_blocks = (int)qb;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  if (dtype == VQ_BF16)
    launch<BF16>(a, head_dim, (unsigned)(qb + kb), st);
  else
    launch<F32>(a, head_dim, (unsigned)(qb + kb), st);
  return cudaGetLastError() == cudaSuccess ? VQ_OK : VQ_ERR_CUDA;
}
