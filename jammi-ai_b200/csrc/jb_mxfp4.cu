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

constexpr int kMxRows = 128;   // rows per CTA: one scale tile
constexpr int kMxCols = 256;   // columns per CTA: two scale tiles, a row per warp and load
constexpr int kMxThreads = 256;
constexpr int kMxAhead = 4;    // a warp's rows in flight

// Eight consecutive elements, widened.
__device__ __forceinline__ void load8(const float* p, float (&v)[8]) {
  const float4 a = *reinterpret_cast<const float4*>(p), b = *reinterpret_cast<const float4*>(p + 4);
  v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
  v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
}
__device__ __forceinline__ void load8(const bf16* p, float (&v)[8]) {
  const uint4 raw = *reinterpret_cast<const uint4*>(p);
  const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    v[2 * e] = __uint_as_float(w[e] << 16);
    v[2 * e + 1] = __uint_as_float(w[e] & 0xffff0000u);
  }
}
__device__ __forceinline__ void load8(const f16* p, float (&v)[8]) {
  const uint4 raw = *reinterpret_cast<const uint4*>(p);
  const __half2* h = reinterpret_cast<const __half2*>(&raw);
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const float2 f = __half22float2(h[e]);
    v[2 * e] = f.x;
    v[2 * e + 1] = f.y;
  }
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

// A CTA per 128 rows x 256 columns; warp w takes rows w, w + 8, ...: its 32
// lanes hold a row's 256 columns, four lanes to a block (two shuffles for the
// block's maximum), 512 bytes read and 128 written per row.  The tile's scale
// bytes are gathered in shared memory and written as one contiguous run.
template <typename T>
__global__ void __launch_bounds__(kMxThreads) quantize_mxfp4_kernel(const T* __restrict__ x, uint8_t* __restrict__ q,
                                                                    uint8_t* __restrict__ scale, int rows, int cols) {
  __shared__ __align__(16) uint8_t tile[1024];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int bands = (cols + kMxCols - 1) / kMxCols;
  const int rt = blockIdx.x / bands, band = blockIdx.x % bands;
  const int row0 = rt * kMxRows;
  const int col = band * kMxCols + lane * 8;
  const int nrows = min(kMxRows, rows - row0);
  reinterpret_cast<uint32_t*>(tile)[threadIdx.x] = 0;  // padding rows and blocks
  __syncthreads();
  const bool in = col < cols;  // cols % 32 == 0: a block's four lanes agree
  for (int r0 = warp; r0 < nrows; r0 += 8 * kMxAhead) {
    float v[kMxAhead][8];
#pragma unroll
    for (int u = 0; u < kMxAhead; ++u) {
#pragma unroll
      for (int e = 0; e < 8; ++e) v[u][e] = 0.f;
      if (in && r0 + 8 * u < nrows) load8(x + static_cast<size_t>(row0 + r0 + 8 * u) * cols + col, v[u]);
    }
#pragma unroll
    for (int u = 0; u < kMxAhead; ++u) {
      const int r = r0 + 8 * u;
      unsigned top = 0;  // bits of |x| order as the values do, NaN above infinity
#pragma unroll
      for (int e = 0; e < 8; ++e) top = max(top, __float_as_uint(v[u][e]) & 0x7fffffffu);
      top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
      top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
      const int field = static_cast<int>(top >> 23);
      const int e8 = field == 255 ? 255 : max(field - 2, 0);
      const float inv = __uint_as_float(static_cast<uint32_t>(254 - min(e8, 253)) << 23);  // 2^(127 - e8)
#pragma unroll
      for (int e = 0; e < 8; ++e) v[u][e] *= inv;
      const uint32_t code = e8 == 255 ? 0u : e2m1x8(v[u]);
      if (in && r < nrows) {
        *reinterpret_cast<uint32_t*>(q + (static_cast<size_t>(row0 + r) * cols + col) / 2) = code;
        const int b = lane >> 2;  // block of the 256 columns
        if ((lane & 3) == 0) tile[(b >> 2) * 512 + (r & 31) * 16 + (r >> 5) * 4 + (b & 3)] = static_cast<uint8_t>(e8);
      }
    }
  }
  __syncthreads();
  const int ct = (cols + 127) / 128;  // scale tiles of a row
  const int words = min(2, ct - 2 * band) * 128;
  uint32_t* out = reinterpret_cast<uint32_t*>(scale) + (static_cast<size_t>(rt) * ct + 2 * band) * 128;
  if (static_cast<int>(threadIdx.x) < words) out[threadIdx.x] = reinterpret_cast<const uint32_t*>(tile)[threadIdx.x];
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

// The value of an e2m1 code's low three bits times its sign, from its bits:
// codes 2..7 are (1 + m / 2) 2^(e - 1); 0 and 1 are 0 and 0.5.
__device__ __forceinline__ float e2m1_value(uint32_t c) {
  const uint32_t mag = c & 7u;
  const float m = mag < 2 ? 0.5f * static_cast<float>(mag) : __uint_as_float((mag << 22) + (126u << 23));
  return __uint_as_float(__float_as_uint(m) | ((c & 8u) << 28));
}

// y = code * 2^(byte - 127), rounded to T: the quantiser's grid and lanes.
template <typename T>
__global__ void __launch_bounds__(kMxThreads) dequantize_mxfp4_kernel(const uint8_t* __restrict__ q,
                                                                      const uint8_t* __restrict__ scale,
                                                                      T* __restrict__ y, int rows, int cols) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int bands = (cols + kMxCols - 1) / kMxCols;
  const int rt = blockIdx.x / bands;
  const int row0 = rt * kMxRows;
  const int col = (blockIdx.x % bands) * kMxCols + lane * 8;
  const int nrows = min(kMxRows, rows - row0);
  if (col >= cols) return;
  const int ct = (cols + 127) / 128, b = col >> 5;
  const uint8_t* tile = scale + (static_cast<size_t>(rt) * ct + (b >> 2)) * 512;
#pragma unroll 4
  for (int r = warp; r < nrows; r += 8) {
    const size_t at = static_cast<size_t>(row0 + r) * cols + col;
    const uint32_t code = *reinterpret_cast<const uint32_t*>(q + at / 2);
    const uint32_t e8 = tile[(r & 31) * 16 + (r >> 5) * 4 + (b & 3)];
    // 2^(e8 - 127): e8 == 0 is the subnormal 2^-127, e8 == 255 a NaN
    const float s = __uint_as_float(e8 == 0 ? 0x00400000u : e8 == 255 ? 0x7fffffffu : e8 << 23);
    float v[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = e2m1_value(code >> (4 * e)) * s;
    store8(y + at, v);
  }
}

unsigned mx_grid(int rows, int cols) {
  return static_cast<unsigned>((cols + kMxCols - 1ll) / kMxCols * ((rows + kMxRows - 1ll) / kMxRows));
}

}  // namespace

cudaError_t launch_quantize_mxfp4(const void* x, int dtype, uint8_t* q, uint8_t* scale, int rows, int cols,
                                  cudaStream_t s) {
  if (rows == 0) return cudaSuccess;
  const unsigned grid = mx_grid(rows, cols);
  switch (dtype) {
    case JB_DT_F32:
      quantize_mxfp4_kernel<<<grid, kMxThreads, 0, s>>>(static_cast<const float*>(x), q, scale, rows, cols);
      break;
    case JB_DT_BF16:
      quantize_mxfp4_kernel<<<grid, kMxThreads, 0, s>>>(static_cast<const bf16*>(x), q, scale, rows, cols);
      break;
    case JB_DT_F16:
      quantize_mxfp4_kernel<<<grid, kMxThreads, 0, s>>>(static_cast<const f16*>(x), q, scale, rows, cols);
      break;
    default: return cudaErrorInvalidValue;
  }
  return cudaGetLastError();
}

cudaError_t launch_dequantize_mxfp4(const uint8_t* q, const uint8_t* scale, void* y, int dtype, int rows, int cols,
                                    cudaStream_t s) {
  if (rows == 0) return cudaSuccess;
  const unsigned grid = mx_grid(rows, cols);
  switch (dtype) {
    case JB_DT_F32:
      dequantize_mxfp4_kernel<<<grid, kMxThreads, 0, s>>>(q, scale, static_cast<float*>(y), rows, cols);
      break;
    case JB_DT_BF16:
      dequantize_mxfp4_kernel<<<grid, kMxThreads, 0, s>>>(q, scale, static_cast<bf16*>(y), rows, cols);
      break;
    case JB_DT_F16:
      dequantize_mxfp4_kernel<<<grid, kMxThreads, 0, s>>>(q, scale, static_cast<f16*>(y), rows, cols);
      break;
    default: return cudaErrorInvalidValue;
  }
  return cudaGetLastError();
}

}  // namespace jb
