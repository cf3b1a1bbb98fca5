// MXFP4 rows (OCP Microscaling Formats v1.0): quantisation and the way back.
//
// Every 32 consecutive elements of a row share a power-of-two scale 2^E,
// E = floor(log2(max |x|)) - 2 (2 = the exponent of e2m1's largest value, 6),
// clamped to [-127, 127] and stored as the byte E + 127 (E8M0); each element
// is e2m1(x 2^-E): nearest, ties to even, saturated at 6.  x 2^-E is exact
// (a power of two times an f32 value, the product normal for every element
// that does not round to zero), so the conversion is the only rounding.  A
// block that holds a NaN or an infinity has scale byte 255 (NaN) and codes 0.
//
// floor(log2 max) is the exponent field of the largest magnitude, so E + 127
// = max(field - 2, 0); a subnormal maximum has field 0.
//
// Two codes share a byte (the even column in the low half).  Scale bytes lie
// in the order the tensor core's scale-factor copy reads them
// (jb_mxfp4_gemm.cu): tiles of 128 rows x 4 blocks (512 bytes, K fastest),
// row r and block b of a tile at (r % 32) * 16 + (r / 32) * 4 + b.  Rows and
// blocks that pad the last tiles have scale byte 0.
#include <algorithm>

#include "jb_common.cuh"
#include "jb_internal.h"

namespace jb {
namespace {

// A CTA takes 32 rows (a quarter of the scale tiles' rows) x up to 1024
// columns: whole runs of 2 KB of a 16-bit row, which DRAM serves better than
// the 256 bytes of one scale tile (see the quantiser).
constexpr int kMxRows = 32;
constexpr int kMxCols = 1024;
constexpr int kMxThreads = 256;

// The CTA's place.  SEGS = 256-column pieces of a row in the band (a template
// parameter of the kernels: a piece's row and column cost no division).
struct MxPlace {
  int row0, col0, nrows, tiles;  // tiles: scale tiles of a row
  __device__ __forceinline__ MxPlace(int rows, int cols) {
    const int bands = (cols + kMxCols - 1) / kMxCols;
    row0 = blockIdx.x / bands * kMxRows;
    col0 = blockIdx.x % bands * kMxCols;
    nrows = max(0, min(kMxRows, rows - row0));
    tiles = (cols + 127) / 128;
  }
};

// Eight consecutive elements as loaded, and widened.
template <typename T>
struct Raw8 {
  uint4 v;
  __device__ __forceinline__ void load(const T* p) { v = __ldg(reinterpret_cast<const uint4*>(p)); }
  __device__ __forceinline__ void zero() { v = make_uint4(0, 0, 0, 0); }
};
template <>
struct Raw8<float> {
  uint4 v, w;
  __device__ __forceinline__ void load(const float* p) {
    v = __ldg(reinterpret_cast<const uint4*>(p));
    w = __ldg(reinterpret_cast<const uint4*>(p) + 1);
  }
  __device__ __forceinline__ void zero() { v = w = make_uint4(0, 0, 0, 0); }
};
__device__ __forceinline__ void widen(const Raw8<float>& r, float (&v)[8]) {
  const uint32_t w[8] = {r.v.x, r.v.y, r.v.z, r.v.w, r.w.x, r.w.y, r.w.z, r.w.w};
#pragma unroll
  for (int e = 0; e < 8; ++e) v[e] = __uint_as_float(w[e]);
}
__device__ __forceinline__ void widen(const Raw8<bf16>& r, float (&v)[8]) {
  const uint32_t w[4] = {r.v.x, r.v.y, r.v.z, r.v.w};
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    v[2 * e] = __uint_as_float(w[e] << 16);
    v[2 * e + 1] = __uint_as_float(w[e] & 0xffff0000u);
  }
}
__device__ __forceinline__ void widen(const Raw8<f16>& r, float (&v)[8]) {
  const __half2* h = reinterpret_cast<const __half2*>(&r.v);
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const float2 f = __half22float2(h[e]);
    v[2 * e] = f.x;
    v[2 * e + 1] = f.y;
  }
}

// Bits of the largest |x| as f32 (bits of magnitudes order as the values do,
// NaN above infinity); 16-bit types two elements at a time.
__device__ __forceinline__ unsigned top_bits(const Raw8<float>& r) {
  const uint32_t w[8] = {r.v.x, r.v.y, r.v.z, r.v.w, r.w.x, r.w.y, r.w.z, r.w.w};
  unsigned top = 0;
#pragma unroll
  for (int e = 0; e < 8; ++e) top = max(top, w[e] & 0x7fffffffu);
  return top;
}
__device__ __forceinline__ unsigned top_half(const uint4& v) {
  const unsigned m = __vmaxu2(__vmaxu2(v.x & 0x7fff7fffu, v.y & 0x7fff7fffu),
                              __vmaxu2(v.z & 0x7fff7fffu, v.w & 0x7fff7fffu));
  return max(m >> 16, m & 0xffffu);
}
__device__ __forceinline__ unsigned top_bits(const Raw8<bf16>& r) { return top_half(r.v) << 16; }
__device__ __forceinline__ unsigned top_bits(const Raw8<f16>& r) {
  return __float_as_uint(__half2float(__ushort_as_half(static_cast<unsigned short>(top_half(r.v)))));
}

// Eight e2m1 codes of v (v[0] in the low nibble).
__device__ __forceinline__ uint32_t e2m1x8(const float (&v)[8]) {
  uint32_t r;
  asm("{\n\t.reg .b8 b0, b1, b2, b3;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b0, %2, %1;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b1, %4, %3;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b2, %6, %5;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b3, %8, %7;\n\t"
      "mov.b32 %0, {b0, b1, b2, b3};\n\t}"
      : "=r"(r)
      : "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]), "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7]));
  return r;
}

// Warp w takes rows w, w + 8, ... of the CTA: a piece is a row's 256 columns
// (32 lanes of eight elements, four lanes to a block, two shuffles for its
// maximum), up to eight pieces in flight.  Scale bytes are gathered in shared
// memory and written as words: [tile][row] four blocks, 16 bytes apart in the
// tile.  Memory-bound: 20479 x 4096 bf16 35.1 us, 6.0 TB/s (a copy: 6.5); 20479 x
// 1024 13.0 us, 4.1 TB/s, whose 640 CTAs are 1.08 waves of four to an SM (64
// registers; the four-segment form spills two of them).  (One CTA per scale tile,
// which reads 256 bytes of a row, took 47.5 us at 20479 x 4096.)
template <typename T, int SEGS>
__global__ void __launch_bounds__(kMxThreads) quantize_mxfp4_kernel(const T* __restrict__ x, uint8_t* __restrict__ q,
                                                                    uint8_t* __restrict__ scale, int rows, int cols) {
  constexpr int kRows = SEGS == 1 ? 4 : 2;  // rows of a warp in flight
  __shared__ __align__(16) uint32_t words[kMxCols / 128 * kMxRows];
  const MxPlace p(rows, cols);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  words[threadIdx.x] = 0;  // padding rows and blocks
  __syncthreads();
  const size_t at = static_cast<size_t>(p.row0) * cols + p.col0 + lane * 8;
  const int left = cols - p.col0 - lane * 8;  // columns from this lane's first one on
  for (int r0 = warp; r0 < p.nrows; r0 += 8 * kRows) {
    Raw8<T> raw[kRows * SEGS];
#pragma unroll
    for (int u = 0; u < kRows * SEGS; ++u) {
      const int row = r0 + 8 * (u / SEGS), c = u % SEGS * 256;
      raw[u].zero();
      if (row < p.nrows && c < left) raw[u].load(x + at + static_cast<size_t>(row) * cols + c);
    }
#pragma unroll
    for (int u = 0; u < kRows * SEGS; ++u) {
      const int row = r0 + 8 * (u / SEGS), c = u % SEGS * 256;
      unsigned top = top_bits(raw[u]);
      top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
      top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
      const int field = static_cast<int>(top >> 23);
      const int e8 = field == 255 ? 255 : max(field - 2, 0);
      const float inv = __uint_as_float(static_cast<uint32_t>(254 - min(e8, 253)) << 23);  // 2^(127 - e8)
      float v[8];
      widen(raw[u], v);
#pragma unroll
      for (int e = 0; e < 8; e += 2) {
        const float2 z = __fmul2_rn(make_float2(v[e], v[e + 1]), f2(inv));
        v[e] = z.x;
        v[e + 1] = z.y;
      }
      const uint32_t code = e8 == 255 ? 0u : e2m1x8(v);
      if (row < p.nrows && c < left) {
        *reinterpret_cast<uint32_t*>(q + (at + static_cast<size_t>(row) * cols + c) / 2) = code;
        if ((lane & 3) == 0)
          reinterpret_cast<uint8_t*>(words)[((c / 128 + (lane >> 4)) * kMxRows + row) * 4 + ((lane >> 2) & 3)] =
              static_cast<uint8_t>(e8);
      }
    }
  }
  __syncthreads();
  const int tile = threadIdx.x >> 5;  // of the band, its row lane
  if (p.col0 / 128 + tile < p.tiles) {
    uint8_t* out = scale + (static_cast<size_t>(p.row0 / 128) * p.tiles + p.col0 / 128 + tile) * 512;
    reinterpret_cast<uint32_t*>(out)[lane * 4 + p.row0 % 128 / 32] = words[threadIdx.x];
  }
}

__device__ __forceinline__ void store8(float* p, const float (&v)[8]) {
  *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]);
  *reinterpret_cast<float4*>(p + 4) = make_float4(v[4], v[5], v[6], v[7]);
}
__device__ __forceinline__ void store8(bf16* p, const float (&v)[8]) {
  uint4 raw;
  __nv_bfloat162* h = reinterpret_cast<__nv_bfloat162*>(&raw);
#pragma unroll
  for (int e = 0; e < 4; ++e) h[e] = __floats2bfloat162_rn(v[2 * e], v[2 * e + 1]);
  *reinterpret_cast<uint4*>(p) = raw;
}
__device__ __forceinline__ void store8(f16* p, const float (&v)[8]) {
  uint4 raw;
  __half2* h = reinterpret_cast<__half2*>(&raw);
#pragma unroll
  for (int e = 0; e < 4; ++e) h[e] = __floats2half2_rn(v[2 * e], v[2 * e + 1]);
  *reinterpret_cast<uint4*>(p) = raw;
}

// Two e2m1 codes (a byte, the low nibble first) as f16.
__device__ __forceinline__ float2 e2m1_pair(uint32_t byte) {
  uint32_t h;
  asm("{\n\t.reg .b8 b, z;\n\t"
      "mov.b32 {b, z, z, z}, %1;\n\t"
      "cvt.rn.f16x2.e2m1x2 %0, b;\n\t}"
      : "=r"(h)
      : "r"(byte));
  return __half22float2(*reinterpret_cast<const __half2*>(&h));
}

// y = code * 2^(byte - 127), rounded to T: the quantiser's grid and pieces.
// Memory-bound: 20479 x 4096 to bf16 35.5 us, 6.0 TB/s; 20479 x 1024 11.5 us, 4.6
// TB/s (1.44 waves of three CTAs to an SM).
template <typename T, int SEGS>
__global__ void __launch_bounds__(kMxThreads) dequantize_mxfp4_kernel(const uint8_t* __restrict__ q,
                                                                      const uint8_t* __restrict__ scale,
                                                                      T* __restrict__ y, int rows, int cols) {
  constexpr int kRows = 4;  // rows of a warp: all of them
  const MxPlace p(rows, cols);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint8_t* tiles = scale + (static_cast<size_t>(p.row0 / 128) * p.tiles + p.col0 / 128 + (lane >> 4)) * 512 +
                         p.row0 % 128 / 32 * 4 + ((lane >> 2) & 3);
  const size_t at = static_cast<size_t>(p.row0) * cols + p.col0 + lane * 8;
  const int left = cols - p.col0 - lane * 8;
  uint32_t code[kRows * SEGS], e8[kRows * SEGS];
#pragma unroll
  for (int u = 0; u < kRows * SEGS; ++u) {
    const int row = warp + 8 * (u / SEGS), c = u % SEGS * 256;
    if (row < p.nrows && c < left) {
      code[u] = __ldg(reinterpret_cast<const uint32_t*>(q + (at + static_cast<size_t>(row) * cols + c) / 2));
      e8[u] = __ldg(tiles + c / 128 * 512 + row * 16);
    }
  }
#pragma unroll
  for (int u = 0; u < kRows * SEGS; ++u) {
    const int row = warp + 8 * (u / SEGS), c = u % SEGS * 256;
    if (row < p.nrows && c < left) {
      // 2^(e8 - 127): e8 == 0 is the subnormal 2^-127, e8 == 255 a NaN
      const float s = __uint_as_float(e8[u] == 0 ? 0x00400000u : e8[u] == 255 ? 0x7fffffffu : e8[u] << 23);
      float v[8];
#pragma unroll
      for (int e = 0; e < 8; e += 2) {
        const float2 z = __fmul2_rn(e2m1_pair(code[u] >> (4 * e)), f2(s));
        v[e] = z.x;
        v[e + 1] = z.y;
      }
      store8(y + at + static_cast<size_t>(row) * cols + c, v);
    }
  }
}

// Every 32-row group of the scale tiles, the padding ones too.
unsigned mx_grid(int rows, int cols) {
  return static_cast<unsigned>((rows + 127ll) / 128 * 4 * ((cols + kMxCols - 1ll) / kMxCols));
}

template <typename T>
void launch_quantize(const void* x, uint8_t* q, uint8_t* scale, int rows, int cols, cudaStream_t s) {
  const unsigned grid = mx_grid(rows, cols);
  const T* p = static_cast<const T*>(x);
  switch (std::min(4, (cols + 255) / 256)) {
    case 1: quantize_mxfp4_kernel<T, 1><<<grid, kMxThreads, 0, s>>>(p, q, scale, rows, cols); break;
    case 2: quantize_mxfp4_kernel<T, 2><<<grid, kMxThreads, 0, s>>>(p, q, scale, rows, cols); break;
    case 3: quantize_mxfp4_kernel<T, 3><<<grid, kMxThreads, 0, s>>>(p, q, scale, rows, cols); break;
    default: quantize_mxfp4_kernel<T, 4><<<grid, kMxThreads, 0, s>>>(p, q, scale, rows, cols); break;
  }
}
template <typename T>
void launch_dequantize(const uint8_t* q, const uint8_t* scale, void* y, int rows, int cols, cudaStream_t s) {
  const unsigned grid = mx_grid(rows, cols);
  T* p = static_cast<T*>(y);
  switch (std::min(4, (cols + 255) / 256)) {
    case 1: dequantize_mxfp4_kernel<T, 1><<<grid, kMxThreads, 0, s>>>(q, scale, p, rows, cols); break;
    case 2: dequantize_mxfp4_kernel<T, 2><<<grid, kMxThreads, 0, s>>>(q, scale, p, rows, cols); break;
    case 3: dequantize_mxfp4_kernel<T, 3><<<grid, kMxThreads, 0, s>>>(q, scale, p, rows, cols); break;
    default: dequantize_mxfp4_kernel<T, 4><<<grid, kMxThreads, 0, s>>>(q, scale, p, rows, cols); break;
  }
}

}  // namespace

cudaError_t launch_quantize_mxfp4(const void* x, int dtype, uint8_t* q, uint8_t* scale, int rows, int cols,
                                  cudaStream_t s) {
  if (rows == 0) return cudaSuccess;
  switch (dtype) {
    case JB_DT_F32: launch_quantize<float>(x, q, scale, rows, cols, s); break;
    case JB_DT_BF16: launch_quantize<bf16>(x, q, scale, rows, cols, s); break;
    case JB_DT_F16: launch_quantize<f16>(x, q, scale, rows, cols, s); break;
    default: return cudaErrorInvalidValue;
  }
  return cudaGetLastError();
}

cudaError_t launch_dequantize_mxfp4(const uint8_t* q, const uint8_t* scale, void* y, int dtype, int rows, int cols,
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
