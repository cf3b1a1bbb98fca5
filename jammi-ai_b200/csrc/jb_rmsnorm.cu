// RMS norm with the residual's addition, in the rows' type or as per-row int8
// (the format jb_op_linear_s8 reads), and the way back from int8 rows.
//
//   s = x + r,  h = round(s),  y = s * rsqrt(mean(s^2) + eps) * gamma
//   int8: a = max |y| over the row, scale = a / 127, q = rint(y * (127 / a))
//
// s, the statistics and y stay in f32: y is computed and quantised from the
// unrounded sum, so h (the residual stream of the next layer) carries the
// only rounding of the addition and q the only one of the norm.
//
// Memory-bound: x and r are read once and every output is written once, the
// row held in registers between its two reductions (the sum of squares and
// the maximum).  Rows of up to 1024 16-bit columns belong to one warp (no
// barrier; the next row's loads are issued before the current row's
// reductions); wider rows to a CTA of four, eight or sixteen warps with the
// same registers per thread.  Rows whose width or base address rules 16-byte
// loads out, and rows of more than 4096 vectors, are read element by element.
//
// Measured, inputs and outputs out of cache, with residual and sum, bf16 unless
// said (captured calls; a copy runs at 6.54 TB/s):
//   36870 x 768    y 39.3 us, 5.8 TB/s    int8 33.8 us, 5.9 TB/s
//            f32   y 76.2 us, 5.9 TB/s    int8 58.2 us, 6.3 TB/s
//   9001 x 4096    y 52.3 us, 5.6 TB/s    int8 44.5 us, 5.8 TB/s
//            f32   y 91.0 us, 6.5 TB/s
//            f16, no residual             int8 22.0 us, 5.0 TB/s
//   3000 x 20000   y 128 us, 3.8 TB/s     int8 136 us  (the scalar kernel: 213, 240)
//   36870 x 770    y 75 us, 3.0 TB/s      int8 87 us   (single elements)
//   9001 x 4095    y 86 us, 3.4 TB/s      int8 102 us  (single elements)
//   12 x 768       2.3 us, int8 2.7: launch and one row's latency
// What is left to the copy's rate are the reductions between a row's loads
// and its stores, which the next row's loads cover only in part.  Rows of more
// than 2048 vectors have no other CTA on their SM to cover them at all and, with a
// residual, spill 96 to 120 bytes a thread; odd rows issue a load per element.
#include <algorithm>
#include <atomic>

#include "jb_common.cuh"
#include "jb_internal.h"

namespace jb {
namespace {

// 16-byte vectors of T.
template <typename T> struct Row;
template <> struct Row<bf16> {
  static constexpr int N = 8;
  __device__ static void unpack(const uint4& raw, float* v) {
    const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      v[2 * e] = __uint_as_float(w[e] << 16);
      v[2 * e + 1] = __uint_as_float(w[e] & 0xffff0000u);
    }
  }
  __device__ static uint4 pack(const float* v) {
    uint4 raw;
    __nv_bfloat162* h = reinterpret_cast<__nv_bfloat162*>(&raw);
#pragma unroll
    for (int e = 0; e < 4; ++e) h[e] = __floats2bfloat162_rn(v[2 * e], v[2 * e + 1]);
    return raw;
  }
};
template <> struct Row<f16> {
  static constexpr int N = 8;
  __device__ static void unpack(const uint4& raw, float* v) {
    const __half2* h = reinterpret_cast<const __half2*>(&raw);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float2 f = __half22float2(h[e]);
      v[2 * e] = f.x;
      v[2 * e + 1] = f.y;
    }
  }
  __device__ static uint4 pack(const float* v) {
    uint4 raw;
    __half2* h = reinterpret_cast<__half2*>(&raw);
#pragma unroll
    for (int e = 0; e < 4; ++e) h[e] = __floats2half2_rn(v[2 * e], v[2 * e + 1]);
    return raw;
  }
};
template <> struct Row<float> {
  static constexpr int N = 4;
  __device__ static void unpack(const uint4& raw, float* v) {
    v[0] = __uint_as_float(raw.x); v[1] = __uint_as_float(raw.y);
    v[2] = __uint_as_float(raw.z); v[3] = __uint_as_float(raw.w);
  }
  __device__ static uint4 pack(const float* v) {
    return make_uint4(__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]),
                      __float_as_uint(v[3]));
  }
};

// Bits of |v|: they order as the values do, infinities above every finite
// value and NaNs above those, so one integer maximum finds the row's largest
// magnitude and whether the row holds anything that is not finite.
__device__ __forceinline__ unsigned abs_bits(float v) { return __float_as_uint(v) & 0x7fffffffu; }
constexpr unsigned kInfBits = 0x7f800000u;

// mean(s^2) + eps as summed, unless the squares left f32's range (infinite, or
// so small that they lost bits): then a row's sum is taken again of s * c.  The
// test costs ordinary rows nothing up to 1024 columns, 1% at 4096 and 4 to 6% in
// the wider kernels, where it keeps the next pass's loads behind the statistics.
__device__ __forceinline__ bool in_range(float var) { return var >= 0x1p-90f && var < INFINITY; }
// c = 2^-floor(log2(max(|s| of the row, sqrt(eps)))): s * c and eps * c^2 are
// below 4.  0: the row holds a NaN or an infinity, whose statistics stand.
__device__ __forceinline__ float range_scale(unsigned top, float eps) {
  if (top >= kInfBits) return 0.f;
  const int field = static_cast<int>(max(top, __float_as_uint(sqrtf(eps))) >> 23);
  return __uint_as_float(static_cast<uint32_t>(max(254 - field, 1)) << 23);
}

// The row's quantiser from the bits of its largest |y|: q = rint(y * up * inv).
// `up` is 1 except in rows so small that 127 / a would overflow.  A row with a
// NaN or an infinity has scale NaN and q 0.
struct RowQuant {
  float up, inv, scale;
};
__device__ __forceinline__ RowQuant row_quant(unsigned top) {
  if (top >= kInfBits) return {0.f, 0.f, __int_as_float(0x7fffffff)};
  const float a = __uint_as_float(top);
  const float up = a < 0x1p-100f ? 0x1p100f : 1.f;
  return {up, a > 0.f ? 127.0f / (a * up) : 0.f, a / 127.0f};
}
// rint(v) of |v| <= 127 (1 + 2^-22) in the low byte: v + 1.5 * 2^23 rounds to
// the nearest integer, ties to even.  The product is rounded on its own (never
// contracted into the addition), as rint(y * inv) is.
__device__ __forceinline__ uint32_t rint_byte(float v, float inv) {
  return __float_as_uint(__fadd_rn(__fmul_rn(v, inv), 12582912.0f));
}
__device__ __forceinline__ uint32_t rint4(const float* v, float inv) {
  return __byte_perm(__byte_perm(rint_byte(v[0], inv), rint_byte(v[1], inv), 0x0040),
                     __byte_perm(rint_byte(v[2], inv), rint_byte(v[3], inv), 0x0040), 0x5410);
}

// W warps per row (W == 1: eight rows per 256-thread CTA, persistent, the
// next row prefetched; W > 1: a CTA of W warps per row).  MAXV 16-byte
// vectors of the row per lane.  QUANT: int8 rows instead of y.
template <typename T, int MAXV, int W, bool RES, bool QUANT>
__global__ void __launch_bounds__(W == 1 ? 256 : 32 * W) rmsnorm_kernel(RmsArgs a) {
  constexpr int VN = Row<T>::N;
  constexpr int kRows = W == 1 ? 8 : 1;
  constexpr int kLanes = 32 * W;  // lanes of a row
  // x, r of up to four vectors are fetched a row ahead; wider rows lean on
  // the other CTAs of the SM instead of on more registers
  constexpr bool kAhead = MAXV * (RES ? 2 : 1) <= 8;
  __shared__ float red[W == 1 ? 1 : 2 * W];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int at = W == 1 ? lane : threadIdx.x;  // this thread's first vector
  const int nvec = a.cols / VN;
  const int stride = gridDim.x * kRows;
  int row = blockIdx.x * kRows + (W == 1 ? warp : 0);

  auto fetch = [&](int r, uint4 (&xr)[MAXV], uint4 (&rr)[MAXV]) {
    const size_t off = static_cast<size_t>(r) * a.cols;
    const uint4* x = reinterpret_cast<const uint4*>(static_cast<const T*>(a.x) + off);
    const uint4* res = reinterpret_cast<const uint4*>(static_cast<const T*>(a.resid) + (RES ? off : 0));
#pragma unroll
    for (int i = 0; i < MAXV; ++i) {
      if (at + i * kLanes < nvec) {
        xr[i] = x[at + i * kLanes];
        if constexpr (RES) rr[i] = res[at + i * kLanes];
      }
    }
  };
  uint4 xr[MAXV], rr[MAXV];
  if (kAhead && row < a.rows) fetch(row, xr, rr);
  for (; row < a.rows; row += stride) {
    const size_t off = static_cast<size_t>(row) * a.cols;
    if (!kAhead) fetch(row, xr, rr);
    float v[MAXV * VN];
    float2 ss = make_float2(0.f, 0.f);
#pragma unroll
    for (int i = 0; i < MAXV; ++i) {
      if (at + i * kLanes < nvec) {
        Row<T>::unpack(xr[i], v + i * VN);
        if constexpr (RES) {
          float t[VN];
          Row<T>::unpack(rr[i], t);
#pragma unroll
          for (int e = 0; e < VN; ++e) v[i * VN + e] += t[e];
        }
#pragma unroll
        for (int e = 0; e < VN; e += 2) {
          const float2 p = make_float2(v[i * VN + e], v[i * VN + e + 1]);
          ss = __ffma2_rn(p, p, ss);
        }
      }
    }
    if (kAhead && row + stride < a.rows) fetch(row + stride, xr, rr);
    if constexpr (RES) {
      if (a.sum) {
#pragma unroll
        for (int i = 0; i < MAXV; ++i)
          if (at + i * kLanes < nvec)
            reinterpret_cast<uint4*>(static_cast<T*>(a.sum) + off)[at + i * kLanes] = Row<T>::pack(v + i * VN);
      }
    }
    float total = warp_sum(ss.x + ss.y);
    if constexpr (W > 1) {
      if (lane == 0) red[warp] = total;
      __syncthreads();
      total = 0.f;
#pragma unroll
      for (int w = 0; w < W; ++w) total += red[w];
    }
    float var = total / static_cast<float>(a.cols) + a.eps;
    if (!in_range(var)) {  // uniform over the row
      unsigned big = 0;
#pragma unroll
      for (int i = 0; i < MAXV; ++i)
        if (at + i * kLanes < nvec)
#pragma unroll
          for (int e = 0; e < VN; ++e) big = max(big, abs_bits(v[i * VN + e]));
      big = __reduce_max_sync(0xffffffffu, big);
      if constexpr (W > 1) {
        if (lane == 0) red[W + warp] = __uint_as_float(big);
        __syncthreads();  // and the sums of `red`'s first half have been read
#pragma unroll
        for (int w = 0; w < W; ++w) big = max(big, __float_as_uint(red[W + w]));
      }
      const float c = range_scale(big, a.eps);
      if (c != 0.f) {
        float again = 0.f;
#pragma unroll
        for (int i = 0; i < MAXV; ++i)
          if (at + i * kLanes < nvec)
#pragma unroll
            for (int e = 0; e < VN; ++e) {
              v[i * VN + e] *= c;
              again = fmaf(v[i * VN + e], v[i * VN + e], again);
            }
        again = warp_sum(again);
        if constexpr (W > 1) {
          if (lane == 0) red[warp] = again;
          __syncthreads();
          again = 0.f;
#pragma unroll
          for (int w = 0; w < W; ++w) again += red[w];
        }
        var = again / static_cast<float>(a.cols) + a.eps * c * c;
      }
    }
    const float rstd = 1.0f / sqrtf(var);
    unsigned top = 0;
#pragma unroll
    for (int i = 0; i < MAXV; ++i) {
      const int vi = at + i * kLanes;
      if (vi < nvec) {
        const float4* g4 = reinterpret_cast<const float4*>(a.gamma + vi * VN);
#pragma unroll
        for (int q = 0; q < VN / 4; ++q) {
          const float4 g = __ldg(g4 + q);
          float* p = v + i * VN + 4 * q;
          const float2 y01 = __fmul2_rn(__fmul2_rn(make_float2(p[0], p[1]), f2(rstd)), make_float2(g.x, g.y));
          const float2 y23 = __fmul2_rn(__fmul2_rn(make_float2(p[2], p[3]), f2(rstd)), make_float2(g.z, g.w));
          p[0] = y01.x; p[1] = y01.y; p[2] = y23.x; p[3] = y23.y;
          if constexpr (QUANT)
            top = max(max(top, max(abs_bits(p[0]), abs_bits(p[1]))), max(abs_bits(p[2]), abs_bits(p[3])));
        }
        if constexpr (!QUANT)
          reinterpret_cast<uint4*>(static_cast<T*>(a.y) + off)[vi] = Row<T>::pack(v + i * VN);
      }
    }
    if constexpr (QUANT) {
      top = __reduce_max_sync(0xffffffffu, top);
      if constexpr (W > 1) {
        if (lane == 0) red[W + warp] = __uint_as_float(top);
        __syncthreads();
#pragma unroll
        for (int w = 0; w < W; ++w) top = max(top, __float_as_uint(red[W + w]));
      }
      const RowQuant rq = row_quant(top);
      if (rq.up != 1.f) {  // uniform over the row: a tiny or a not finite row
#pragma unroll
        for (int e = 0; e < MAXV * VN; ++e) v[e] = rq.up == 0.f ? 0.f : v[e] * rq.up;
      }
#pragma unroll
      for (int i = 0; i < MAXV; ++i) {
        const int vi = at + i * kLanes;
        if (vi < nvec) {
          if constexpr (VN == 8)
            *reinterpret_cast<uint2*>(a.q + off + vi * 8) =
                make_uint2(rint4(v + i * 8, rq.inv), rint4(v + i * 8 + 4, rq.inv));
          else
            *reinterpret_cast<uint32_t*>(a.q + off + vi * 4) = rint4(v + i * 4, rq.inv);
        }
      }
      if (at == 0) a.scale[row] = rq.scale;
    }
    // W > 1: `red`'s first half is written again only after the second
    // barrier (QUANT) or below
    if constexpr (W > 1 && !QUANT) __syncthreads();
  }
}

// Narrow rows of any width and alignment: a warp per row with single elements,
// E of them per lane (times by calls, launch gaps included).  Up to 1024 columns (36870 x 770 bf16 with residual 80 us,
// int8 94; f32 without residual 64, int8 74; the form below, a CTA per row, takes
// 104, 164, 100, 150), but 256 of f32 with a residual, where the misaligned
// lines of two wide rows do not stay in L1 from one warp access to the next
// (36870 x 770: 215 us, int8 219; below 103 and 152).
template <typename T, int E>
__global__ void __launch_bounds__(256) rmsnorm_ragged_kernel(RmsArgs a) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  for (int row = blockIdx.x * 8 + warp; row < a.rows; row += gridDim.x * 8) {
    const size_t off = static_cast<size_t>(row) * a.cols;
    const T* x = static_cast<const T*>(a.x) + off;
    float v[E];
    float ss = 0.f;
#pragma unroll
    for (int i = 0; i < E; ++i) v[i] = lane + 32 * i < a.cols ? to_f(x[lane + 32 * i]) : 0.f;
    if (a.resid) {
      const T* r = static_cast<const T*>(a.resid) + off;
      T t[E];
#pragma unroll
      for (int i = 0; i < E; ++i)
        if (lane + 32 * i < a.cols) t[i] = r[lane + 32 * i];
#pragma unroll
      for (int i = 0; i < E; ++i)
        if (lane + 32 * i < a.cols) v[i] += to_f(t[i]);
      if (a.sum) {
#pragma unroll
        for (int i = 0; i < E; ++i)
          if (lane + 32 * i < a.cols) static_cast<T*>(a.sum)[off + lane + 32 * i] = from_f<T>(v[i]);
      }
    }
#pragma unroll
    for (int i = 0; i < E; ++i) ss = fmaf(v[i], v[i], ss);
    float var = warp_sum(ss) / static_cast<float>(a.cols) + a.eps;
    if (!in_range(var)) {  // uniform over the row
      unsigned big = 0;
#pragma unroll
      for (int i = 0; i < E; ++i) big = max(big, abs_bits(v[i]));
      const float c = range_scale(__reduce_max_sync(0xffffffffu, big), a.eps);
      if (c != 0.f) {
        ss = 0.f;
#pragma unroll
        for (int i = 0; i < E; ++i) {
          v[i] *= c;
          ss = fmaf(v[i], v[i], ss);
        }
        var = warp_sum(ss) / static_cast<float>(a.cols) + a.eps * c * c;
      }
    }
    const float rstd = 1.0f / sqrtf(var);
    unsigned top = 0;
#pragma unroll
    for (int i = 0; i < E; ++i) {
      const int c = lane + 32 * i;
      if (c < a.cols) {
        v[i] = v[i] * rstd * __ldg(a.gamma + c);
        top = max(top, abs_bits(v[i]));
        if (a.y) static_cast<T*>(a.y)[off + c] = from_f<T>(v[i]);
      }
    }
    if (a.q) {
      const RowQuant rq = row_quant(__reduce_max_sync(0xffffffffu, top));
#pragma unroll
      for (int i = 0; i < E; ++i) {
        const int c = lane + 32 * i;
        if (c < a.cols)
          a.q[off + c] = static_cast<int8_t>(rint_byte(rq.up == 0.f ? 0.f : v[i] * rq.up, rq.inv) & 0xffu);
      }
      if (lane == 0) a.scale[row] = rq.scale;
    }
  }
}

// Wider rows of any width and alignment: a CTA per row, each element read
// again (mostly out of L1) in every pass and every output written in the last
// one (so outputs may replace inputs element for element).  9001 x 4095 bf16
// with residual 90 us, int8 104 us; with the row in registers 96 to 113 us
// (fewer loads in flight).
template <typename T>
__global__ void __launch_bounds__(256) rmsnorm_scalar_kernel(RmsArgs a) {
  __shared__ float red[8];
  __shared__ unsigned redm[8];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  for (int row = blockIdx.x; row < a.rows; row += gridDim.x) {
    const size_t off = static_cast<size_t>(row) * a.cols;
    const T* x = static_cast<const T*>(a.x) + off;
    const T* r = a.resid ? static_cast<const T*>(a.resid) + off : nullptr;
    auto s_at = [&](int c) { return r ? to_f(x[c]) + to_f(r[c]) : to_f(x[c]); };
    float scale = 1.f;  // of s in the statistics and y, see in_range
    auto mean_square = [&] {
      float ss = 0.f;
      for (int c = threadIdx.x; c < a.cols; c += 256) {
        const float s = s_at(c) * scale;
        ss = fmaf(s, s, ss);
      }
      ss = warp_sum(ss);
      if (lane == 0) red[warp] = ss;
      __syncthreads();
      float total = 0.f;
      for (int w = 0; w < 8; ++w) total += red[w];
      return total / static_cast<float>(a.cols);
    };
    float var = mean_square() + a.eps;
    if (!in_range(var)) {  // uniform over the row
      unsigned big = 0;
      for (int c = threadIdx.x; c < a.cols; c += 256) big = max(big, abs_bits(s_at(c)));
      big = __reduce_max_sync(0xffffffffu, big);
      if (lane == 0) redm[warp] = big;
      __syncthreads();  // and `red` has been read
      for (int w = 0; w < 8; ++w) big = max(big, redm[w]);
      const float c = range_scale(big, a.eps);
      if (c != 0.f) {
        scale = c;
        var = mean_square() + a.eps * c * c;
      }
      __syncthreads();  // redm has been read
    }
    const float rstd = 1.0f / sqrtf(var);
    RowQuant rq{1.f, 0.f, 0.f};
    if (a.q) {
      unsigned top = 0;
      for (int c = threadIdx.x; c < a.cols; c += 256) top = max(top, abs_bits(s_at(c) * scale * rstd * __ldg(a.gamma + c)));
      top = __reduce_max_sync(0xffffffffu, top);
      if (lane == 0) redm[warp] = top;
      __syncthreads();
      for (int w = 0; w < 8; ++w) top = max(top, redm[w]);
      rq = row_quant(top);
      if (threadIdx.x == 0) a.scale[row] = rq.scale;
    }
    for (int c = threadIdx.x; c < a.cols; c += 256) {
      const float s = s_at(c);
      const float y = s * scale * rstd * __ldg(a.gamma + c);
      if (a.sum) static_cast<T*>(a.sum)[off + c] = from_f<T>(s);
      if (a.q)
        a.q[off + c] = static_cast<int8_t>(rint_byte(rq.up == 0.f ? 0.f : y * rq.up, rq.inv) & 0xffu);
      else
        static_cast<T*>(a.y)[off + c] = from_f<T>(y);
    }
    __syncthreads();  // red / redm free for the next row
  }
}

bool aligned(const void* p, size_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }

// CTAs of one wave: as many as the kernel's registers let reside.
template <auto Kern>
unsigned wave(int block, long long need) {
  static std::atomic<int> cached{0};
  int per_sm = cached.load(std::memory_order_relaxed);
  if (!per_sm) {
    if (cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per_sm, Kern, block, 0) != cudaSuccess || per_sm < 1)
      per_sm = 1;
    cached.store(per_sm, std::memory_order_relaxed);
  }
  int dev = 0;
  cudaGetDevice(&dev);
  return static_cast<unsigned>(std::min<long long>(need, static_cast<long long>(num_sms(dev)) * per_sm));
}

template <typename T, int MAXV, int W, bool RES, bool QUANT>
void launch_rows(const RmsArgs& a, cudaStream_t s) {
  constexpr auto kern = rmsnorm_kernel<T, MAXV, W, RES, QUANT>;
  constexpr int block = W == 1 ? 256 : 32 * W;
  const unsigned grid = wave<kern>(block, W == 1 ? (a.rows + 7ll) / 8 : a.rows);
  kern<<<grid, block, 0, s>>>(a);
}
template <typename T, int MAXV, int W>
void launch_form(const RmsArgs& a, cudaStream_t s) {
  if (a.q)
    a.resid ? launch_rows<T, MAXV, W, true, true>(a, s) : launch_rows<T, MAXV, W, false, true>(a, s);
  else
    a.resid ? launch_rows<T, MAXV, W, true, false>(a, s) : launch_rows<T, MAXV, W, false, false>(a, s);
}
template <typename T, int E>
void launch_ragged(const RmsArgs& a, cudaStream_t s) {
  constexpr auto kern = rmsnorm_ragged_kernel<T, E>;
  kern<<<wave<kern>(256, (a.rows + 7ll) / 8), 256, 0, s>>>(a);
}
template <typename T>
void launch_width(const RmsArgs& a, cudaStream_t s) {
  constexpr int VN = Row<T>::N;
  const int nvec = a.cols / VN;
  const bool vec = a.cols % VN == 0 && aligned(a.x, 16) && aligned(a.resid, 16) && aligned(a.sum, 16) &&
                   aligned(a.y, 16) && aligned(a.gamma, 16) && aligned(a.q, VN);
  if (!vec || nvec > 512 * 8) {
    if (a.cols <= 256) {
      launch_ragged<T, 8>(a, s);
    } else if (a.cols <= 1024 && (sizeof(T) == 2 || !a.resid)) {
      launch_ragged<T, 32>(a, s);
    } else {
      rmsnorm_scalar_kernel<T><<<wave<rmsnorm_scalar_kernel<T>>(256, a.rows), 256, 0, s>>>(a);
    }
  } else if (nvec <= 32) {
    launch_form<T, 1, 1>(a, s);
  } else if (nvec <= 96) {
    launch_form<T, 3, 1>(a, s);
  } else if (nvec <= 128) {
    launch_form<T, 4, 1>(a, s);
  } else if (nvec <= 256) {
    launch_form<T, 2, 4>(a, s);
  } else if (nvec <= 512) {
    launch_form<T, 4, 4>(a, s);
  } else if (nvec <= 2048) {
    launch_form<T, 8, 8>(a, s);
  } else {
    launch_form<T, 8, 16>(a, s);
  }
}

// y = q * scale, rounded to T.  A warp per row, eight codes per lane and
// load; other widths and alignments element by element.  36870 x 768 to bf16
// 17.3 us out of cache (4.9 TB/s), 9001 x 4096 to f16 20.3 us (5.5 TB/s).  Short of
// the copy's rate for the eight conversions per load (XU pipe 61%) and a
// row's loads that wait for the row before.
template <typename T>
__global__ void __launch_bounds__(256) dequantize_rows_kernel(const int8_t* __restrict__ q,
                                                              const float* __restrict__ scale, T* y, int rows,
                                                              int cols, int vec) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  for (int row = blockIdx.x * 8 + warp; row < rows; row += gridDim.x * 8) {
    const size_t off = static_cast<size_t>(row) * cols;
    const float s = scale[row];
    if (vec) {
#pragma unroll 4
      for (int c = lane * 8; c < cols; c += 256) {
        const uint2 raw = *reinterpret_cast<const uint2*>(q + off + c);
        float v[8];
#pragma unroll
        for (int e = 0; e < 8; ++e)
          v[e] = static_cast<float>(static_cast<int8_t>((e < 4 ? raw.x : raw.y) >> (8 * (e & 3)))) * s;
        if constexpr (sizeof(T) == 2) {
          *reinterpret_cast<uint4*>(y + off + c) = Row<T>::pack(v);
        } else {
          reinterpret_cast<uint4*>(y + off + c)[0] = Row<T>::pack(v);
          reinterpret_cast<uint4*>(y + off + c)[1] = Row<T>::pack(v + 4);
        }
      }
    } else {
      for (int c = lane; c < cols; c += 32) y[off + c] = from_f<T>(static_cast<float>(q[off + c]) * s);
    }
  }
}
template <typename T>
void launch_dequantize(const int8_t* q, const float* scale, void* y, int rows, int cols, cudaStream_t s) {
  const int vec = cols % 8 == 0 && aligned(q, 8) && aligned(y, 16);
  const unsigned grid = wave<dequantize_rows_kernel<T>>(256, (rows + 7ll) / 8);
  dequantize_rows_kernel<T><<<grid, 256, 0, s>>>(q, scale, static_cast<T*>(y), rows, cols, vec);
}

}  // namespace

cudaError_t launch_rmsnorm(const RmsArgs& a, int dtype, cudaStream_t s) {
  if (a.rows == 0) return cudaSuccess;
  switch (dtype) {
    case JB_DT_F32: launch_width<float>(a, s); break;
    case JB_DT_BF16: launch_width<bf16>(a, s); break;
    case JB_DT_F16: launch_width<f16>(a, s); break;
    default: return cudaErrorInvalidValue;
  }
  return cudaGetLastError();
}

cudaError_t launch_dequantize_rows(const int8_t* q, const float* scale, void* y, int dtype, int rows, int cols,
                                   cudaStream_t s) {
  if (rows == 0) return cudaSuccess;
  switch (dtype) {
    case JB_DT_F32: launch_dequantize<float>(q, scale, y, rows, cols, s); break;
    case JB_DT_BF16: launch_dequantize<bf16>(q, scale, y, rows, cols, s); break;
    case JB_DT_F16: launch_dequantize<f16>(q, scale, y, rows, cols, s); break;
    default: return cudaErrorInvalidValue;
  }
  return cudaGetLastError();
}

}  // namespace jb
