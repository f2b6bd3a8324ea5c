// RMSNorm (with the residual's addition) and E4M3 quantization with one
// float32 scale per 128 columns of a row:
//
//   h = x + r                          (float32; hidden = h in x's type)
//   y = h * rsqrt(mean(h^2) + eps) * w (float32; without w: y = h)
//   s = max|y| / 448 per 128 columns   (1 where that is 0)
//   code = E4M3(y / s)
//
// Everything between the loads and the stores is float32: the norm is that
// of the unrounded sum, and each output is rounded once.  The row's factor
// f cancels in y / s = 448 z / max|z|, z = h w; computed so, a quotient that
// is a tie in the reals (with bf16 inputs many are, both products having few
// bits) comes out as one, where roundings of y and s would move it.  So that
// z has y's range, f = p m with p a power of two and 1 <= m < 2: z = (h p) w,
// the first product exact, and s = max|z| m / 448.  A NaN in a block
// makes its scale and codes NaN (maxima are taken on magnitude bits, where
// NaN sorts above infinity).
//
// Bound by HBM: x, r read once, hidden and codes written once (7 bytes per
// bf16 element with the residual).  A row stays in its threads' registers
// between the sum of squares and the quantization.
#include <cuda_runtime.h>
#include <stdint.h>

#include <algorithm>

#include "voyager_b200.h"
#include "vq_e4m3.cuh"
#include "vq_pdl.cuh"
#include "vq_tc.cuh"

namespace vq {
namespace fp8n {

using namespace vq::e4;

struct Args {
  const void* x;
  const void* r;  // or null
  const void* w;  // or null: no norm
  int64_t ldx, ldr;
  int64_t rows;
  int cols, nblk;  // nblk = ceil(cols / 128)
  int eb;          // bytes of an element
  float eps;
  uint8_t* codes;  // [rows, cols]
  float* scale;    // [rows, nblk]
  void* hidden;    // [rows, cols], with r only
};

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int d = 16; d; d >>= 1) v += __shfl_xor_sync(FULL, v, d);
  return v;
}
__device__ __forceinline__ uint32_t mag(float v) { return __float_as_uint(v) & 0x7FFFFFFFu; }

// Two neighbouring float32 in one register pair, each lane rounded as the
// scalar operation rounds it.
using Two = uint64_t;
__device__ __forceinline__ Two two(float lo, float hi) {
  Two v;
  asm("mov.b64 %0, {%1, %2};" : "=l"(v) : "f"(lo), "f"(hi));
  return v;
}
__device__ __forceinline__ float2 each(Two v) {
  float2 f;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(f.x), "=f"(f.y) : "l"(v));
  return f;
}
__device__ __forceinline__ Two add2(Two a, Two b) {
  Two d;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
__device__ __forceinline__ Two mul2(Two a, Two b) {
  Two d;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
__device__ __forceinline__ Two fma2(Two a, Two b, Two c) {
  Two d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
  return d;
}
// max(|m|, |v.lo|, |v.hi|), NaN if one is.
__device__ __forceinline__ float max_abs(float m, Two v) {
  const float2 f = each(v);
  float d;
  asm("max.NaN.abs.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(m), "f"(f.x), "f"(f.y));
  return d;
}

// The sum of v over the CTA's threads, in every thread; `part` holds one
// float per warp.
__device__ __forceinline__ float block_sum(float v, float* part) {
  v = warp_sum(v);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, n = blockDim.x >> 5;
  if (lane == 0) part[warp] = v;
  __syncthreads();
  return warp_sum(lane < n ? part[lane] : 0.0f);
}

// f = p m.  Zero, infinity and NaN (a row whose squares overflow, or of zeros
// with eps = 0) stay whole.
struct Factor {
  float p = 1.0f, m = 1.0f;
  __device__ __forceinline__ void set(float f) {
    const uint32_t b = __float_as_uint(f), e = b & 0x7F800000u;
    const bool whole = e == 0 || e == 0x7F800000u;
    p = whole ? f : __uint_as_float(e);
    m = whole ? 1.0f : __uint_as_float((b & 0x7FFFFFu) | 0x3F800000u);
  }
};

// A block's scale and its values over that scale, from max|z| as bits.  With
// max|z| = 2^e n and 1 <= n < 2 (less than 1 below 2^-118), 448 z / max|z| =
// t / n, t = (448 2^-e) z: nothing but a z too small for a code leaves
// float32's range, so the product with 1 / n and one correction by its
// remainder (Markstein, IBM J. Res. Dev. 34, 1990) serve every block.
struct Block {
  float c, n, r, s;
  __device__ __forceinline__ Block(uint32_t bits, const Factor& f) {
    const int e = min(max((int)(bits >> 23), 9), 254);  // biased
    c = __uint_as_float((uint32_t)(254 + 8 - e) << 23) * 1.75f;
    n = __uint_as_float(bits) * __uint_as_float(e == 254 ? 0x00400000u : (uint32_t)(254 - e) << 23);
    s = over(n * f.m, QMAX, 1.0f / QMAX) * __uint_as_float((uint32_t)e << 23);
    if (s == 0.0f) s = n = 1.0f, c = 0.0f;
    if (bits >= 0x7F800000u) {  // infinity over infinity is NaN, the rest of its block 0
      s = __uint_as_float(bits);
      c = bits == 0x7F800000u ? 0.0f : s;
      n = 1.0f;
    }
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(n));
  }
  // t / n with r near 1 / n
  static __device__ __forceinline__ float over(float t, float n, float r) {
    const float q = t * r;
    return fmaf(fmaf(-q, n, t), r, q);
  }
  __device__ __forceinline__ float operator()(float z) const { return over(z * c, n, r); }
};

// A CTA takes rows blockIdx.x, + gridDim.x, ..; NV groups of 8 consecutive
// elements per thread; columns a multiple of 8, rows 16-byte aligned.  A block
// of 128 columns is 16 neighbouring lanes.  The next row's loads are in
// flight while this one is summed and quantized (without that the SMs waited
// for them half the time: 16384 x 4096 bf16 with a residual took 111 us, now
// 72, the copy rate), and the weight stays in registers.  Two neighbouring
// elements go through each float32 instruction (one by one: 78 us).
template <typename T, int NV, int MAXT>
__global__ void __launch_bounds__(MAXT) k_norm_vec(const Args a) {
  using E = typename T::type;
  using Raw = typename T::Raw;
  __shared__ float part[2][32];
  const E* x = reinterpret_cast<const E*>(a.x);
  const E* r = reinterpret_cast<const E*>(a.r);
  const E* w = reinterpret_cast<const E*>(a.w);
  pdl::trigger();
  pdl::wait();
  auto col = [&](int i) { return (i * (int)blockDim.x + (int)threadIdx.x) * 8; };
  Raw rx[NV] = {}, rr[NV] = {}, rw[NV] = {};
  auto fetch = [&](int64_t row) {
#pragma unroll
    for (int i = 0; i < NV; ++i)
      if (col(i) < a.cols) {
        rx[i] = T::fetch8(x + row * a.ldx + col(i));
        if (a.r) rr[i] = T::fetch8(r + row * a.ldr + col(i));
      }
  };
  auto widen = [](const Raw& r, Two (&v)[4]) {
    float f[8];
    T::widen8(r, f);
#pragma unroll
    for (int k = 0; k < 4; ++k) v[k] = two(f[2 * k], f[2 * k + 1]);
  };
  fetch(blockIdx.x);
  if (a.w) {
#pragma unroll
    for (int i = 0; i < NV; ++i)
      if (col(i) < a.cols) rw[i] = T::fetch8(w + col(i));
  }
  int flip = 0;
  for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x, flip ^= 1) {
    E* hid = reinterpret_cast<E*>(a.hidden) + row * a.cols;
    Two h[NV][4], sq = 0;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      widen(rx[i], h[i]);
      if (a.r) {
        Two q[4];
        widen(rr[i], q);
#pragma unroll
        for (int k = 0; k < 4; ++k) h[i][k] = add2(h[i][k], q[k]);
      }
#pragma unroll
      for (int k = 0; k < 4; ++k) sq = fma2(h[i][k], h[i][k], sq);
    }
    if (row + gridDim.x < a.rows) fetch(row + gridDim.x);
    if (a.r) {
#pragma unroll
      for (int i = 0; i < NV; ++i)
        if (col(i) < a.cols) {
          float v[8];
#pragma unroll
          for (int k = 0; k < 4; ++k) v[2 * k] = each(h[i][k]).x, v[2 * k + 1] = each(h[i][k]).y;
          T::store8(hid + col(i), v);
        }
    }
    Factor f;
    const float ss = each(sq).x + each(sq).y;
    // two buffers of partial sums: the next row's do not meet this one's readers
    if (a.w) f.set(rsqrtf(__fdiv_rn(block_sum(ss, part[flip]), (float)a.cols) + a.eps));
    const Two p = two(f.p, f.p);
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = col(i);
      if (a.w) {
        Two g[4];
        widen(rw[i], g);
#pragma unroll
        for (int k = 0; k < 4; ++k) h[i][k] = mul2(mul2(h[i][k], p), g[k]);
      }
      float top = 0.0f;
#pragma unroll
      for (int k = 0; k < 4; ++k) top = max_abs(top, h[i][k]);
      uint32_t m = c < a.cols ? mag(top) : 0;  // past the row 0, whatever f is
#pragma unroll
      for (int d = 8; d; d >>= 1) m = max(m, __shfl_xor_sync(FULL, m, d));
      if (c < a.cols) {
        const Block blk(m, f);
        const Two bc = two(blk.c, blk.c), br = two(blk.r, blk.r), bn = two(-blk.n, -blk.n);
        uint32_t q[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {  // Block's operator(), two at a time
          const Two t = mul2(h[i][k], bc), u = mul2(t, br);
          const float2 v = each(fma2(fma2(u, bn, t), br, u));
          q[k] = pack2(v.x, v.y);
        }
        *reinterpret_cast<uint2*>(a.codes + row * a.cols + c) = make_uint2(q[0] | q[1] << 16, q[2] | q[3] << 16);
        if ((threadIdx.x & 15) == 0) a.scale[row * a.nblk + (c >> 7)] = blk.s;
      }
    }
  }
}

// Columns that are no multiple of 8, or rows off 16 bytes: a warp takes NB
// blocks of 128 columns, VEC neighbouring elements a load (2 where rows keep
// the pairs aligned), so that its loads and stores stay dense.  Rows as in
// k_norm_vec; with NB = 4 the registers hold no second row.
// (One CTA per row took 34.6 us for 7158 x 1630 bf16 with a residual, 22.3
// now; instructions bound it: 20 us without the residual.)
template <typename T, int VEC>
struct Few {  // VEC elements as they lie in memory
  using E = typename T::type;
  E v[VEC];
  __device__ __forceinline__ void load(const E* p) {
    if (VEC == 1)
      v[0] = __ldg(p);
    else if (sizeof(E) == 2)
      *reinterpret_cast<uint32_t*>(v) = __ldg(reinterpret_cast<const uint32_t*>(p));
    else
      *reinterpret_cast<float2*>(v) = __ldg(reinterpret_cast<const float2*>(p));
  }
};
template <typename T, int VEC>
__device__ __forceinline__ void store_v(typename T::type* p, const float (&v)[VEC]) {
  if (VEC == 1)
    T::store(p, v[0]);
  else if (sizeof(*p) == 2)
    *reinterpret_cast<uint32_t*>(p) = bf_pack(v[0], v[VEC - 1]);
  else
    *reinterpret_cast<float2*>(p) = make_float2(v[0], v[VEC - 1]);
}
template <typename T, int NB, int VEC, int MAXT>
__global__ void __launch_bounds__(MAXT) k_norm_blocks(const Args a) {
  using E = typename T::type;
  constexpr int PER = 4 / VEC;  // loads of a lane per block
  constexpr int N = NB * PER;
  constexpr bool AHEAD = NB < 4;
  __shared__ float part[2][32];
  const E* x = reinterpret_cast<const E*>(a.x);
  const E* r = reinterpret_cast<const E*>(a.r);
  const E* w = reinterpret_cast<const E*>(a.w);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  auto col = [&](int i) { return warp * NB * 128 + lane * VEC + i * 32 * VEC; };
  pdl::trigger();
  pdl::wait();
  alignas(8) Few<T, VEC> rx[N] = {}, rr[N] = {}, rw[N] = {};
  auto fetch = [&](int64_t row) {
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (col(i) < a.cols) rx[i].load(x + row * a.ldx + col(i));
    if (a.r) {
#pragma unroll
      for (int i = 0; i < N; ++i)
        if (col(i) < a.cols) rr[i].load(r + row * a.ldr + col(i));
    }
  };
  auto fetch_w = [&]() {
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (col(i) < a.cols) rw[i].load(w + col(i));
  };
  if (AHEAD) {
    fetch(blockIdx.x);
    if (a.w) fetch_w();
  }
  int flip = 0;
  for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x, flip ^= 1) {
    E* hid = reinterpret_cast<E*>(a.hidden) + row * a.cols;
    if (!AHEAD) fetch(row);
    float h[N][VEC], ss = 0.0f;
#pragma unroll
    for (int i = 0; i < N; ++i)
#pragma unroll
      for (int k = 0; k < VEC; ++k) {
        h[i][k] = T::load(rx[i].v + k);
        if (a.r) h[i][k] += T::load(rr[i].v + k);
        ss = fmaf(h[i][k], h[i][k], ss);
      }
    if (AHEAD && row + gridDim.x < a.rows) fetch(row + gridDim.x);
    if (a.r) {
#pragma unroll
      for (int i = 0; i < N; ++i)
        if (col(i) < a.cols) store_v<T, VEC>(hid + col(i), h[i]);
    }
    Factor f;
    if (a.w) {
      if (!AHEAD) fetch_w();
      f.set(rsqrtf(__fdiv_rn(block_sum(ss, part[flip]), (float)a.cols) + a.eps));
#pragma unroll
      for (int i = 0; i < N; ++i)
#pragma unroll
        for (int k = 0; k < VEC; ++k)  // past the row 0, whatever f is
          h[i][k] = col(i) < a.cols ? h[i][k] * f.p * T::load(rw[i].v + k) : 0.0f;
    }
#pragma unroll
    for (int b = 0; b < NB; ++b) {
      uint32_t m = 0;
#pragma unroll
      for (int i = 0; i < PER; ++i)
#pragma unroll
        for (int k = 0; k < VEC; ++k) m = max(m, mag(h[b * PER + i][k]));
      m = __reduce_max_sync(FULL, m);
      const Block over(m, f);
#pragma unroll
      for (int i = 0; i < PER; ++i) {
        const int c = col(b * PER + i);
        if (c < a.cols) {
          const uint32_t q = pack2(over(h[b * PER + i][0]), over(h[b * PER + i][VEC - 1]));
          if (VEC == 1)
            a.codes[row * a.cols + c] = (uint8_t)q;
          else
            *reinterpret_cast<uint16_t*>(a.codes + row * a.cols + c) = (uint16_t)q;
        }
      }
      const int blk = warp * NB + b;
      if (lane == 0 && blk < a.nblk) a.scale[row * a.nblk + blk] = over.s;
    }
  }
}

// Rows too long for that: one warp per 128 columns at a time, element loads;
// the row is read again for the quantization.
template <typename T>
__global__ void __launch_bounds__(1024) k_norm_any(const Args a) {
  using E = typename T::type;
  __shared__ float part[32];
  pdl::trigger();
  pdl::wait();
  const int64_t row = blockIdx.x;
  const E* x = reinterpret_cast<const E*>(a.x) + row * a.ldx;
  const E* r = a.r ? reinterpret_cast<const E*>(a.r) + row * a.ldr : nullptr;
  const E* w = reinterpret_cast<const E*>(a.w);
  Factor f;
  if (a.w) {
    float ss = 0.0f;
    for (int c = threadIdx.x; c < a.cols; c += blockDim.x) {
      const float h = T::load(x + c) + (r ? T::load(r + c) : 0.0f);
      ss = fmaf(h, h, ss);
    }
    f.set(rsqrtf(__fdiv_rn(block_sum(ss, part), (float)a.cols) + a.eps));
  }
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, nw = blockDim.x >> 5;
  for (int b = warp; b < a.nblk; b += nw) {
    float z[4];
    uint32_t m = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int c = b * 128 + j * 32 + lane;
      z[j] = 0.0f;
      if (c < a.cols) {
        float h = T::load(x + c);
        if (r) {
          h += T::load(r + c);
          T::store(reinterpret_cast<E*>(a.hidden) + row * a.cols + c, h);
        }
        z[j] = a.w ? h * f.p * T::load(w + c) : h;
      }
      m = max(m, mag(z[j]));
    }
    m = __reduce_max_sync(FULL, m);
    const Block over(m, f);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int c = b * 128 + j * 32 + lane;
      if (c < a.cols) a.codes[row * a.cols + c] = (uint8_t)pack2(over(z[j]), 0.0f);
    }
    if (lane == 0) a.scale[row * a.nblk + b] = over.s;
  }
}

// As many CTAs as fit at once (asked once per device and CTA size), or one per
// row; but no more per SM than have 56 KB of next rows in flight, beyond which
// HBM slows down (16384 x 4096 bf16 with a residual: 72 us with three CTAs of
// 16 KB, 81 with four; 16384 x 3328: 60 with four of 13 KB, 65 with three), and
// three at least (9000 x 5120: 55 us, with two 70).
template <auto F>
bool launch_rows(const Args& a, int threads, cudaStream_t st) {
  static int known[64][33] = {};
  int dev = 0;
  cudaGetDevice(&dev);
  dev = dev < 0 || dev > 63 ? 0 : dev;
  int& per_sm = known[dev][threads / 32];
  if (per_sm == 0) {
    int n = 0;
    if (cudaOccupancyMaxActiveBlocksPerMultiprocessor(&n, F, threads, 0) != cudaSuccess || n < 1) {
      (void)cudaGetLastError();
      n = 1;
    }
    per_sm = n;
  }
  const int64_t ahead = (int64_t)a.cols * a.eb * (a.r ? 2 : 1);
  const int64_t most = std::max<int64_t>(3, (56 << 10) / ahead);
  const int64_t grid = std::min(a.rows, std::min<int64_t>(per_sm, most) * vq::mx::sm_count());
  if (a.rows > grid)  // long enough
    return pdl::launch<F, false>((unsigned)grid, threads, 0, st, 1, a);
  return pdl::launch<F>((unsigned)grid, threads, 0, st, 1, a);
}

template <typename T, int VEC>
bool launch_blocks(const Args& a, cudaStream_t st) {
  // blocks a warp: one while there are few rows (latency), else two (four:
  // 34.6 against 26.9 us for 7158 x 1630) where a CTA holds the row so
  const int nb = (a.rows < 256 && a.nblk <= 32) || a.nblk <= 2 ? 1 : a.nblk <= 64 ? 2 : 4;
  const int threads = (a.nblk + nb - 1) / nb * 32;
  if (nb == 1)
    return threads <= 256 ? launch_rows<k_norm_blocks<T, 1, VEC, 256>>(a, threads, st)
                          : launch_rows<k_norm_blocks<T, 1, VEC, 1024>>(a, threads, st);
  else if (nb == 2)
    return threads <= 256 ? launch_rows<k_norm_blocks<T, 2, VEC, 256>>(a, threads, st)
                          : launch_rows<k_norm_blocks<T, 2, VEC, 1024>>(a, threads, st);
  else
    return launch_rows<k_norm_blocks<T, 4, VEC, 1024>>(a, threads, st);
}

// vec: elements that every row start keeps together (8, 2 or 1).
template <typename T>
bool launch(const Args& a, int vec, cudaStream_t st) {
  const int groups = (a.cols + 7) / 8;
  const unsigned rows = (unsigned)a.rows;
  if (vec == 8 && groups <= 4096) {
    // groups a thread: one while there are few rows (latency), else up to four
    // in threads of at most 256, so that an SM holds several rows
    int nv = 1;
    while (groups > nv * (a.rows < 256 ? 1024 : 256) && nv < 4) nv *= 2;
    const int threads = std::min(1024, ((groups + nv - 1) / nv + 31) / 32 * 32);
    if (nv == 1)
      return threads <= 256 ? launch_rows<k_norm_vec<T, 1, 256>>(a, threads, st) : launch_rows<k_norm_vec<T, 1, 1024>>(a, threads, st);
    else if (nv == 2)
      return threads <= 256 ? launch_rows<k_norm_vec<T, 2, 256>>(a, threads, st) : launch_rows<k_norm_vec<T, 2, 1024>>(a, threads, st);
    else
      return threads <= 256 ? launch_rows<k_norm_vec<T, 4, 256>>(a, threads, st) : launch_rows<k_norm_vec<T, 4, 1024>>(a, threads, st);
  } else if (a.nblk <= 128) {
    return vec >= 2 ? launch_blocks<T, 2>(a, st) : launch_blocks<T, 1>(a, st);
  } else {
    return pdl::launch<k_norm_any<T>>(rows, 1024, 0, st, 1, a);
  }
}

}  // namespace fp8n
}  // namespace vq

using namespace vq::fp8n;

extern "C" int vq_norm_quantize_fp8(const void* x, int64_t ldx, const void* residual, int64_t ldr,
                                    const void* weight, int32_t dtype, int64_t rows, int64_t cols,
                                    float eps, void* codes, float* scale, void* hidden,
                                    void* stream) {
  if (rows < 0 || cols <= 0 || cols > (1 << 24) || rows >= (1ll << 31)) return VQ_ERR_INVALID;
  if (dtype != VQ_BF16 && dtype != VQ_F32) return VQ_ERR_UNSUPPORTED;
  if (rows == 0) return VQ_OK;
  if (!x || !codes || !scale || (residual && !hidden)) return VQ_ERR_NULL;
  if (ldx < cols || (residual && ldr < cols)) return VQ_ERR_SHAPE;
  const int eb = dtype == VQ_BF16 ? 2 : 4;
  auto aligned = [](const void* p, uintptr_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; };
  if (!aligned(x, eb) || !aligned(residual, eb) || !aligned(weight, eb) || !aligned(hidden, eb) ||
      !aligned(scale, 4))
    return VQ_ERR_ALIGNMENT;
  Args a;
  a.x = x;
  a.r = residual;
  a.w = weight;
  a.ldx = ldx;
  a.ldr = residual ? ldr : 0;
  a.rows = rows;
  a.cols = (int)cols;
  a.eb = eb;
  a.nblk = (int)((cols + 127) / 128);
  a.eps = eps;
  a.codes = reinterpret_cast<uint8_t*>(codes);
  a.scale = scale;
  a.hidden = residual ? hidden : nullptr;
  auto keeps = [&](int n) {  // n elements together at the start of every row
    const uintptr_t b = (uintptr_t)n * eb > 16 ? 16 : (uintptr_t)n * eb;
    return cols % n == 0 && aligned(x, b) && aligned(residual, b) && aligned(weight, b) &&
           aligned(a.hidden, b) && aligned(codes, n) && (uintptr_t)(ldx * eb) % b == 0 &&
           (uintptr_t)(a.ldr * eb) % b == 0;
  };
  const int vec = keeps(8) ? 8 : keeps(2) ? 2 : 1;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  const bool ok = dtype == VQ_BF16 ? launch<BF16>(a, vec, st) : launch<F32>(a, vec, st);
  return ok ? VQ_OK : VQ_ERR_CUDA;
}
