// Windowed self-attention over packed rows, with first tokens that stay
// visible.
//
// Query i of a row of n tokens sees key j (0 <= j < n) iff
//     j <= i + right  and  (j >= i - left  or  j < sinks),
// and out = sum_j p_j v_j / sum_j p_j, p_j = 2^((q k_j) log2(e) / sqrt(d) - m)
// over the keys it sees.  left, right >= 0, so every query sees itself and no
// sum is empty.  The keys that a block of queries sees are one range
// [first query - left, last query + right] and, where that has left them
// behind, the `sinks` first keys: both are streamed once with a running
// maximum and sum, and no other key is read.
//
// qkv [T, (heads + 2 kv_heads) * d]: the query heads, then the key heads, then
// the value heads of a token; query head h reads key / value head
// h / (heads / kv_heads).
#include <algorithm>

#include "jb_common.cuh"
#include "jb_internal.h"

namespace jb {
namespace {

struct WinParams {
  const void* qkv;
  const int* cu;
  void* ctx;
  int heads, kv_heads;
  int q_blocks;  // query blocks of the longest row
  int left, right, sinks;
  float scale_log2;
};

// ── any head width, f32 arithmetic ──────────────────────────────────────────
// A CTA per (row, head, kSimtQ queries): LANES lanes share a query's
// dimensions (interleaved by four, so that a warp's reads of a key fall on
// different banks), each thread works on two queries, so that a key read from
// shared memory serves both.  FMA-bound: 4 d per (query, key).
constexpr int kSimtThreads = 128;
constexpr int kSimtKeys = 32;

template <int D>
struct SimtCfg {
  static constexpr int LANES = D >= 64 ? D / 32 : D == 32 ? 2 : 1;
  static constexpr int DL = D / LANES;          // dimensions per lane
  static constexpr int GROUPS = kSimtThreads / LANES;
  static constexpr int QUERIES = 2 * GROUPS;    // queries per CTA
};

template <typename T, int D>
__global__ void __launch_bounds__(kSimtThreads) window_simt_kernel(WinParams p) {
  using C = SimtCfg<D>;
  constexpr int V4 = C::DL / 4;
  __shared__ __align__(16) float Ks[kSimtKeys][D];
  __shared__ __align__(16) float Vs[kSimtKeys][D];
  const int qb = blockIdx.x % p.q_blocks;
  const int h = blockIdx.x / p.q_blocks % p.heads, b = blockIdx.x / p.q_blocks / p.heads;
  const int start = p.cu[b], n = p.cu[b + 1] - start;
  const int q0 = qb * C::QUERIES;
  if (q0 >= n) return;
  const int hk = h / (p.heads / p.kv_heads);
  const int ld = (p.heads + 2 * p.kv_heads) * D;
  const T* row = static_cast<const T*>(p.qkv) + static_cast<size_t>(start) * ld;
  const T* gk = row + (p.heads + hk) * D;
  const T* gv = gk + p.kv_heads * D;
  const int part = threadIdx.x % C::LANES, group = threadIdx.x / C::LANES;
  // queries group and group + GROUPS: a short row fills the first half
  int qi[2], lo[2], hi[2];
  float qv[2][C::DL], o[2][C::DL], m[2], l[2];
#pragma unroll
  for (int u = 0; u < 2; ++u) {
    qi[u] = q0 + group + u * C::GROUPS;
    lo[u] = qi[u] - min(p.left, qi[u]);
    hi[u] = qi[u] < n ? qi[u] + min(p.right, n - 1 - qi[u]) : -1;  // last visible key
    m[u] = -INFINITY;
    l[u] = 0.f;
#pragma unroll
    for (int i = 0; i < V4; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int d = 4 * (i * C::LANES + part) + e;
        qv[u][4 * i + e] = qi[u] < n ? to_f(row[static_cast<size_t>(qi[u]) * ld + h * D + d]) * p.scale_log2 : 0.f;
        o[u][4 * i + e] = 0.f;
      }
  }
  const int q_last = min(n, q0 + C::QUERIES) - 1;
  const int k_end = q_last + min(p.right, n - 1 - q_last) + 1;
  int k_begin = q0 - min(p.left, q0);
  const int s_end = min(p.sinks, k_begin);  // sinks behind the block's window
  // [0, s_end), then [k_begin, k_end)
  for (int k0 = s_end > 0 ? 0 : k_begin; k0 < k_end;) {
    const int stop = k0 < s_end ? s_end : k_end;
    const int kn = min(kSimtKeys, stop - k0);
    __syncthreads();
    for (int i = threadIdx.x; i < kn * D; i += kSimtThreads) {
      const size_t at = static_cast<size_t>(k0 + i / D) * ld + i % D;
      Ks[i / D][i % D] = to_f(gk[at]);
      Vs[i / D][i % D] = to_f(gv[at]);
    }
    __syncthreads();
    for (int j0 = 0; j0 < kn; j0 += 4) {
      float s[2][4];
      bool seen[2][4];  // a hidden value adds nothing, not even 0 * NaN
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        s[0][j] = s[1][j] = 0.f;
        if (j0 + j < kn) {
#pragma unroll
          for (int i = 0; i < V4; ++i) {
            const float4 k4 = *reinterpret_cast<const float4*>(&Ks[j0 + j][4 * (i * C::LANES + part)]);
#pragma unroll
            for (int u = 0; u < 2; ++u) {
              s[u][j] = fmaf(qv[u][4 * i], k4.x, s[u][j]);
              s[u][j] = fmaf(qv[u][4 * i + 1], k4.y, s[u][j]);
              s[u][j] = fmaf(qv[u][4 * i + 2], k4.z, s[u][j]);
              s[u][j] = fmaf(qv[u][4 * i + 3], k4.w, s[u][j]);
            }
          }
        }
#pragma unroll
        for (int w = 1; w < C::LANES; w <<= 1) {
          s[0][j] += __shfl_xor_sync(0xffffffffu, s[0][j], w);
          s[1][j] += __shfl_xor_sync(0xffffffffu, s[1][j], w);
        }
      }
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        float mx = m[u];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int key = k0 + j0 + j;
          seen[u][j] = j0 + j < kn && key <= hi[u] && (key >= lo[u] || key < p.sinks);
          if (!seen[u][j]) s[u][j] = -INFINITY;
          mx = fmaxf(mx, s[u][j]);
        }
        const float ref = mx == -INFINITY ? 0.f : mx;  // nothing seen so far: p stays 0
        const float corr = exp2f(m[u] - ref);
        m[u] = mx;
        l[u] *= corr;
#pragma unroll
        for (int e = 0; e < C::DL; ++e) o[u][e] *= corr;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          s[u][j] = exp2f(s[u][j] - ref);
          l[u] += s[u][j];
        }
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if (j0 + j < kn) {
#pragma unroll
          for (int i = 0; i < V4; ++i) {
            const float4 v4 = *reinterpret_cast<const float4*>(&Vs[j0 + j][4 * (i * C::LANES + part)]);
#pragma unroll
            for (int u = 0; u < 2; ++u) {
              if (!seen[u][j]) continue;
              o[u][4 * i] = fmaf(s[u][j], v4.x, o[u][4 * i]);
              o[u][4 * i + 1] = fmaf(s[u][j], v4.y, o[u][4 * i + 1]);
              o[u][4 * i + 2] = fmaf(s[u][j], v4.z, o[u][4 * i + 2]);
              o[u][4 * i + 3] = fmaf(s[u][j], v4.w, o[u][4 * i + 3]);
            }
          }
        }
      }
    }
    k0 += kn;
    if (k0 == s_end) k0 = k_begin;
  }
#pragma unroll
  for (int u = 0; u < 2; ++u) {
    if (qi[u] < n) {
      const float inv = 1.f / l[u];
      T* out = static_cast<T*>(p.ctx) + (static_cast<size_t>(start + qi[u]) * p.heads + h) * D;
#pragma unroll
      for (int i = 0; i < V4; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) out[4 * (i * C::LANES + part) + e] = from_f<T>(o[u][4 * i + e] * inv);
    }
  }
}

template <typename T, int D>
cudaError_t launch_simt_d(WinParams p, int batch, int max_len, cudaStream_t s, std::string* why) {
  p.q_blocks = (max_len + SimtCfg<D>::QUERIES - 1) / SimtCfg<D>::QUERIES;
  const long long grid = static_cast<long long>(p.q_blocks) * p.heads * batch;
  if (grid > INT32_MAX) {
    if (why) *why = "attention_window: too many (row, head, query block) triples";
    return cudaErrorInvalidValue;
  }
  window_simt_kernel<T, D><<<static_cast<unsigned>(grid), kSimtThreads, 0, s>>>(p);
  return cudaGetLastError();
}
template <typename T>
cudaError_t launch_simt(const WinParams& p, int d, int batch, int max_len, cudaStream_t s, std::string* why) {
  switch (d) {
    case 8: return launch_simt_d<T, 8>(p, batch, max_len, s, why);
    case 16: return launch_simt_d<T, 16>(p, batch, max_len, s, why);
    case 32: return launch_simt_d<T, 32>(p, batch, max_len, s, why);
    case 64: return launch_simt_d<T, 64>(p, batch, max_len, s, why);
    case 128: return launch_simt_d<T, 128>(p, batch, max_len, s, why);
    default:
      if (why) *why = "attention_window: head_dim must be 8, 16, 32, 64 or 128";
      return cudaErrorInvalidValue;
  }
}

}  // namespace

cudaError_t launch_attention_window(const WindowArgs& a, cudaStream_t s, std::string* why) {
  if (a.batch == 0 || a.max_len == 0) return cudaSuccess;
  WinParams p;
  p.qkv = a.qkv;
  p.cu = a.cu;
  p.ctx = a.ctx;
  p.heads = a.heads;
  p.kv_heads = a.kv_heads;
  p.q_blocks = 0;
  p.left = a.left;
  p.right = a.right;
  p.sinks = a.sinks;
  p.scale_log2 = 1.4426950408889634f / sqrtf(static_cast<float>(a.head_dim));
  switch (a.dtype) {
    case JB_DT_F32: return launch_simt<float>(p, a.head_dim, a.batch, a.max_len, s, why);
    case JB_DT_BF16: return launch_simt<bf16>(p, a.head_dim, a.batch, a.max_len, s, why);
    case JB_DT_F16: return launch_simt<f16>(p, a.head_dim, a.batch, a.max_len, s, why);
    default: return cudaErrorInvalidValue;
  }
}

}  // namespace jb
