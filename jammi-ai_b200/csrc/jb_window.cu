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
#include <cudaTypedefs.h>

#include <algorithm>
#include <atomic>
#include <cmath>
#include <type_traits>

#include "jb_common.cuh"
#include "jb_internal.h"

namespace jb {
namespace {

struct WinParams {
  const void* qkv;
  const int* cu;
  void* ctx;
  int heads, kv_heads;
  int rows;      // rows that qkv and ctx hold
  int max_len;   // of a row
  int q_blocks;  // query blocks of the longest row
  int left, right, sinks;
  float scale_log2;
};

// Tokens of row b that lie inside the buffers and max_len, whatever the offsets hold.
__device__ __forceinline__ int row_tokens(const WinParams& p, int b, int start) {
  return start < 0 ? 0 : min(max(0, min(p.cu[b + 1], p.rows)) - start, p.max_len);
}

// ── any head width, f32 arithmetic ──────────────────────────────────────────
// A CTA per (row, head, QUERIES queries): LANES lanes share a query's
// dimensions, 16 each (interleaved by four, so that a warp's reads of a key
// fall on different banks); each thread works on two neighbouring queries, so
// that a key read from shared memory serves both, and a warp skips the key
// tiles that none of its consecutive queries sees.  Two dimensions to an
// instruction (packed f32x2); f32 tiles are
// copied asynchronously, one ahead.  16 rows of 512 tokens, 12 heads of 64, window
// 64 + 64, f32: 228 us, 13 TFLOP/s; 64 rows, 12 heads of 16: f32 324 us, bf16
// 350 us; of 8: bf16 251 us.  No pipe is full (f32, 64: issue 44%, FMA 36%, shared
// memory's data pipe 61%): 14 warps an SM wait in turn for shared loads and
// shuffles, for the FMAs' results and at the two barriers of a key tile; with 16-bit rows,
// whose tiles are not loaded ahead, at the barriers most of all (issue 29%).
constexpr int kSimtThreads = 128;

template <typename T, int D>
struct SimtCfg {
  static constexpr int LANES = D > 16 ? D / 16 : 1;
  static constexpr int DL = D / LANES;          // dimensions per lane
  static constexpr int QUERIES = 2 * kSimtThreads / LANES;
  static constexpr int KEYS = D >= 32 ? 2048 / D : 64;  // of a tile
  static constexpr bool kAsync = sizeof(T) == 4;
  static constexpr int STAGES = kAsync ? 2 : 1;
};

template <typename T, int D>
__global__ void __launch_bounds__(kSimtThreads, 4) window_simt_kernel(WinParams p) {
  using C = SimtCfg<T, D>;
  constexpr int V4 = C::DL / 4;
  __shared__ __align__(16) float Ks[C::STAGES][C::KEYS][D];
  __shared__ __align__(16) float Vs[C::STAGES][C::KEYS][D];
  const int qb = blockIdx.x % p.q_blocks;
  const int h = blockIdx.x / p.q_blocks % p.heads, b = blockIdx.x / p.q_blocks / p.heads;
  const int start = p.cu[b], n = row_tokens(p, b, start);
  const int q0 = qb * C::QUERIES;
  if (q0 >= n) return;
  const int hk = h / (p.heads / p.kv_heads);
  const int ld = (p.heads + 2 * p.kv_heads) * D;
  const T* row = static_cast<const T*>(p.qkv) + static_cast<size_t>(start) * ld;
  const T* gk = row + (p.heads + hk) * D;
  const T* gv = gk + p.kv_heads * D;
  const int part = threadIdx.x % C::LANES, group = threadIdx.x / C::LANES;
  int qi[2], lo[2], hi[2];
  float2 qv[2][C::DL / 2], o[2][C::DL / 2];
  float m[2], l[2];
#pragma unroll
  for (int u = 0; u < 2; ++u) {
    qi[u] = q0 + 2 * group + u;
    lo[u] = qi[u] - min(p.left, qi[u]);
    hi[u] = qi[u] < n ? qi[u] + min(p.right, n - 1 - qi[u]) : -1;  // last visible key
    m[u] = -INFINITY;
    l[u] = 0.f;
#pragma unroll
    for (int i = 0; i < C::DL / 2; ++i) {
      const int d = 4 * (i / 2 * C::LANES + part) + 2 * (i & 1);
      qv[u][i] = o[u][i] = make_float2(0.f, 0.f);
      if (qi[u] < n) {
        const T* q = row + static_cast<size_t>(qi[u]) * ld + h * D + d;
        qv[u][i] = make_float2(to_f(q[0]) * p.scale_log2, to_f(q[1]) * p.scale_log2);
      }
    }
  }
  const int q_last = min(n, q0 + C::QUERIES) - 1;
  const int k_end = q_last + min(p.right, n - 1 - q_last) + 1;
  const int k_begin = q0 - min(p.left, q0);
  const int s_end = min(p.sinks, k_begin);  // sinks behind the block's window
  int see_lo = lo[0], see_hi = max(hi[0], hi[1]);  // of the warp
#pragma unroll
  for (int w = 16; w > 0; w >>= 1) {
    see_lo = min(see_lo, __shfl_xor_sync(0xffffffffu, see_lo, w));
    see_hi = max(see_hi, __shfl_xor_sync(0xffffffffu, see_hi, w));
  }
  // tiles of [0, s_end), then of [k_begin, k_end)
  auto stop_of = [&](int k0) { return min(k0 + C::KEYS, k0 < s_end ? s_end : k_end); };
  auto after = [&](int k1) { return k1 == s_end ? k_begin : k1; };
  auto load = [&](int k0, int st) {
    const int kn = stop_of(k0) - k0;
    if constexpr (C::kAsync) {
      for (int i = threadIdx.x; i < kn * (D / 4); i += kSimtThreads) {
        const size_t at = static_cast<size_t>(k0 + i / (D / 4)) * ld + i % (D / 4) * 4;
        const uint32_t k = smem_u32(&Ks[st][0][0] + 4 * i), v = smem_u32(&Vs[st][0][0] + 4 * i);
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(k), "l"(gk + at) : "memory");
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(v), "l"(gv + at) : "memory");
      }
    } else {
      for (int i = threadIdx.x; i < kn * D; i += kSimtThreads) {
        const size_t at = static_cast<size_t>(k0 + i / D) * ld + i % D;
        (&Ks[st][0][0])[i] = to_f(gk[at]);
        (&Vs[st][0][0])[i] = to_f(gv[at]);
      }
    }
  };
  int k0 = s_end > 0 ? 0 : k_begin, st = 0;
  if constexpr (C::kAsync) {
    load(k0, 0);
    asm volatile("cp.async.commit_group;" ::: "memory");
  }
  while (k0 < k_end) {
    const int k1 = stop_of(k0), next = after(k1), kn = k1 - k0;
    if constexpr (C::kAsync) {
      if (next < k_end) load(next, st ^ 1);  // last read in the turn before, behind its barrier
      asm volatile("cp.async.commit_group;" ::: "memory");
      asm volatile("cp.async.wait_group 1;" ::: "memory");
    } else {
      load(k0, 0);
    }
    __syncthreads();
    if (k0 <= see_hi && (k1 > see_lo || k0 < p.sinks)) {
#pragma unroll 1
      for (int j0 = 0; j0 < kn; j0 += 4) {
        float s[2][4];
        bool seen[2][4];  // a hidden value adds nothing, not even 0 * NaN
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          float2 s2[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
          if (j0 + j < kn) {
#pragma unroll
            for (int i = 0; i < V4; ++i) {
              const float4 k4 = *reinterpret_cast<const float4*>(&Ks[st][j0 + j][4 * (i * C::LANES + part)]);
#pragma unroll
              for (int u = 0; u < 2; ++u) {
                s2[u] = __ffma2_rn(qv[u][2 * i], make_float2(k4.x, k4.y), s2[u]);
                s2[u] = __ffma2_rn(qv[u][2 * i + 1], make_float2(k4.z, k4.w), s2[u]);
              }
            }
          }
#pragma unroll
          for (int u = 0; u < 2; ++u) {
            s[u][j] = s2[u].x + s2[u].y;
#pragma unroll
            for (int w = 1; w < C::LANES; w <<= 1) s[u][j] += __shfl_xor_sync(0xffffffffu, s[u][j], w);
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
          for (int e = 0; e < C::DL / 2; ++e) o[u][e] = __fmul2_rn(o[u][e], f2(corr));
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
              const float4 v4 = *reinterpret_cast<const float4*>(&Vs[st][j0 + j][4 * (i * C::LANES + part)]);
#pragma unroll
              for (int u = 0; u < 2; ++u) {
                if (!seen[u][j]) continue;
                o[u][2 * i] = __ffma2_rn(f2(s[u][j]), make_float2(v4.x, v4.y), o[u][2 * i]);
                o[u][2 * i + 1] = __ffma2_rn(f2(s[u][j]), make_float2(v4.z, v4.w), o[u][2 * i + 1]);
              }
            }
          }
        }
      }
    }
    __syncthreads();  // the tile may be overwritten
    k0 = next;
    if constexpr (C::kAsync) st ^= 1;
  }
#pragma unroll
  for (int u = 0; u < 2; ++u) {
    if (qi[u] < n) {
      const float inv = 1.f / l[u];
      T* out = static_cast<T*>(p.ctx) + (static_cast<size_t>(start + qi[u]) * p.heads + h) * D;
#pragma unroll
      for (int i = 0; i < C::DL / 2; ++i) {
        const int d = 4 * (i / 2 * C::LANES + part) + 2 * (i & 1);
        out[d] = from_f<T>(o[u][i].x * inv);
        out[d + 1] = from_f<T>(o[u][i].y * inv);
      }
    }
  }
}

template <typename T, int D>
cudaError_t launch_simt_d(WinParams p, int batch, int max_len, cudaStream_t s, std::string* why) {
  p.q_blocks = (max_len + SimtCfg<T, D>::QUERIES - 1) / SimtCfg<T, D>::QUERIES;
  const long long grid = static_cast<long long>(p.q_blocks) * p.heads * batch;
  if (grid > INT32_MAX) {
    if (why) *why = "attention_window: too many (row, head, query block) triples";
    return cudaErrorInvalidValue;
  }
  window_simt_kernel<T, D><<<static_cast<unsigned>(grid), kSimtThreads, 0, s>>>(p);
  return cudaGetLastError();
}
// 16-bit rows of head_dim 32 and more run on the tensor cores.
template <typename T>
cudaError_t launch_simt(const WinParams& p, int d, int batch, int max_len, cudaStream_t s, std::string* why) {
  if (d == 8) return launch_simt_d<T, 8>(p, batch, max_len, s, why);
  if (d == 16) return launch_simt_d<T, 16>(p, batch, max_len, s, why);
  if constexpr (sizeof(T) == 4) {
    if (d == 32) return launch_simt_d<T, 32>(p, batch, max_len, s, why);
    if (d == 64) return launch_simt_d<T, 64>(p, batch, max_len, s, why);
    if (d == 128) return launch_simt_d<T, 128>(p, batch, max_len, s, why);
  }
  return cudaErrorInvalidValue;
}

// ── tcgen05, 16-bit rows with head_dim 32, 64 or 128 ────────────────────────
// A persistent CTA per SM runs two independent slots, each on its own items
// (row, head, kq-query block) with its own shared memory and half of TMEM:
//   TMA warp      publishes the slot's items in a ring of four and loads
//                 each one's Q and then, per key block, K and V.
//   MMA warp      S = Q K^T (M = 128, N = the block's keys) into columns
//                 [0, N), then O (+)= P V with P read from TMEM.  The next
//                 item's S comes right behind, before O is read, unless it
//                 is so wide that it would overwrite it.
//   8 softmax     two threads per query row, which take the block's 32-key
//   warps         pieces in turn (even / odd).  Two passes over the scores in
//                 TMEM (maximum, which the two exchange; exponentials and sum),
//                 or one (see ref_col); a warp skips the pieces that none of
//                 its 32 queries sees.  P (16-bit pairs) overwrites the
//                 scores of its own piece: no thread writes where the other
//                 one still reads.
// and four warps for both slots' outputs: O / sum goes out through shared
// memory in whole row segments while the softmax warps are at the next item
// (256 x [32,256]: 8% less than with the softmax warps writing them).
// The keys of an item are its window [k_begin, k_end), padded to 16, then the
// first keys [0, s_end) that the window has left behind, padded to 16.  With
// head_dim 32 or 64, an item of up to 256 keys is ONE block: no running maximum, no
// rescaling, three hand-overs in all (S, P, O); O takes columns of pieces
// 6 and 7 once every score is read, and their P goes to the free halves of
// pieces 0 and 1.  That covers windows of up to left + right = 128 around 128
// queries (and 112 queries with up to 16 sinks), the case this operator is
// for.  Longer ranges go in blocks of 128 keys with a lazily rescaled running
// maximum (raised only by more than 2^8, in f16 2^4).
//
// A masked value contributes 0 * v, which is not 0 when v is not finite.  V
// rows behind the item's last key are zeroed in shared memory; for the rest
// outputs that are not finite are computed again, behind the CTA's last item,
// over the visible keys only (window_rows_exact).
//
// Items are numbered over the query blocks that exist (a prefix sum of the
// rows' blocks in shared memory; beyond kPrefixRows rows an entry stands for a
// group of them, and an item's row is found by a walk through its group) and
// dealt to the slots in turn; no counter in global memory, so calls and
// replayed graphs share nothing.
//
// Measured, bf16 unless said, window 64 + 64 (out of cache):
//   256 rows of 32 to 256 tokens, 12 heads of 64, 1 sink    60 us  3.7 TB/s, f16 76 us
//   8 rows of 4000 to 8192, 16 heads of 64                  82 us  4.5 TB/s, f16 102 us, with 1 sink 95 us
//   256 rows of 4 to 16 tokens, 12 heads of 64              27 us  0.6 TB/s
//   64 x 512 tokens, 12 heads of 64                         47 us  4.3 TB/s, 3 key heads 46 us
//     window 16 + 16: 40 us; 128 + 0: 48; 255 + 0, 4 sinks: 86; 300 + 300: 135
//     unbounded                                            141 us  365 TFLOP/s, f16 the same, causal 91 us
//   64 x 512 tokens, 12 heads of 32                         41 us
//   64 x 512 tokens, 12 heads of 128                        93 us, 6 heads, 3 key heads 52 us
//   one row of 12 tokens                                   6.7 us from launch to launch
// (calls captured into a graph, at 1965 MHz.)
// What bounds it: an item's chain P -> O -> next S leaves the softmax warps
// idle for a third of its time; their exponentials take half of it, 16 a clock
// (two slots' at once).  A row of few tokens costs that chain as a row of 128
// does.  Several blocks: two passes over each block's scores, a meeting of the
// two warps of a row between them, and S of block j + 1 behind P V of block j (one
// S buffer a slot); head_dim 128 has 128-key blocks, so its 64 + 64 window, too.
// More code in any role costs more than it saves (a second, unmasked copy of
// the exponentials: 3% more; P V in two parts, the first behind half of P: 4%;
// an unmasked copy of the maximum: 3%; a call in the output warps' loop and the
// spills around it: 5%): the roles' loops share small instruction caches.  80
// registers, the cap of 768 threads, hold every role without spills.  Items
// dealt by equal cost in contiguous runs instead of in turn: 20% more
// (neighbouring heads of a token are then not read at the same time).  f16
// makes the maximum pass that bf16 saves.
//
// What is rounded: P to the rows' type, which P V on the tensor core asks for
// (scores, sums and O are f32; the sum is of the unrounded weights, since
// unpacking the rounded ones costs bf16 4% of 256 x [32,256] and 12% of the
// unbounded window).  The outputs' relative error against 64 bits: bf16 2.3e-3, of
// which their own rounding is 1.7e-3; f16 2.7e-4 and 2.1e-4.
//
// Every wait is bounded; on a timeout each role stops, copies and MMAs in
// flight are waited for (bounded), the error flag is set and TMEM is freed.
constexpr int kTcWarps = 24;      // 2 TMA, 2 MMA, 16 softmax, 4 output
constexpr int kTcThreads = 32 * kTcWarps;
constexpr int kGroupWarps = 8;    // softmax warps of a slot
constexpr int kSlotBars = 128;    // bytes of a slot's barriers
constexpr int kPrefixRows = 2048;
constexpr int kRounds = (kPrefixRows + kTcThreads - 1) / kTcThreads;
// Lazy-rescaling threshold, log2 units, and how far above the reference's the
// weights of 16-bit P are held: f16 has 2^15 above 1 and 2^-14 below, so one
// block keeps a weight's bits down to 2^-28 of the largest, several down to 2^-25
// (bf16 has f32's range).
template <bool H16> constexpr float kRescale = H16 ? 4.f : 8.f;
constexpr float kLift1 = 14.f, kLift = 11.f;

template <int D>
struct TcCfg {
  static constexpr int ROW = D == 32 ? 64 : 128;           // bytes of a swizzled shared-memory row
  static constexpr int HCOLS = ROW / 2;                    // its elements
  static constexpr int HALVES = D / HCOLS;                 // column blocks of a head
  static constexpr int KEYS = D == 128 ? 128 : 256;        // key rows of a K or V buffer
  static constexpr int Q_BYTES = HALVES * 128 * ROW;
  static constexpr int KV_BYTES = HALVES * KEYS * ROW;
  static constexpr int SLOT_BYTES = Q_BYTES + 2 * KV_BYTES;
  static constexpr int O_COL = 256 - D;                    // O's columns of a slot
  static constexpr int SEG = D == 32 ? 64 : 128;           // bytes of a row that an output warp stores at once
  static constexpr int STAGE_BYTES = 4 * 32 * SEG;
  static constexpr int XCH_BYTES = 2 * 4 * 4 * 2 * 32 * 4;  // [slot][max 0, max 1, sum 0, sum 1][quarter][half][lane]
  static constexpr int META_BYTES = 640;
  static constexpr int USED = 1024 + 2 * SLOT_BYTES + STAGE_BYTES + XCH_BYTES + (kPrefixRows + 4) * 4 + META_BYTES;
  // more than half of an SM's: two CTAs cannot share its TMEM
  static constexpr int SMEM = USED > 120 * 1024 ? USED : 120 * 1024;
  static_assert(SMEM <= 232448, "shared memory");
};

__host__ __device__ constexpr int ceil16(int v) { return (v + 15) & ~15; }
struct TcParams {
  WinParams w;
  int batch;
  int entries, group;  // of the table of query blocks, and the rows of each
  int kq;     // queries per item
  int* err;
};

// A row's tokens and query blocks.
struct TcRow {
  int start, n, blocks;
  __device__ __forceinline__ TcRow(const TcParams& p, int b) : start(p.w.cu[b]), n(row_tokens(p.w, b, start)), blocks(0) {
    if (n > 0) blocks = (n + p.kq - 1) / p.kq;
  }
};
// Item f: its row, head and first query (n = 0: there is none).
struct TcPlace {
  int start = 0, n = 0, h = 0, q0 = 0;
  __device__ __forceinline__ TcPlace() {}
  __device__ __forceinline__ TcPlace(const TcParams& p, const unsigned* prefix, int f) {
    unsigned qb = static_cast<unsigned>(f) / p.w.heads;
    h = f - static_cast<int>(qb) * p.w.heads;
    int lo = 0, hi = p.entries;  // prefix[lo] <= qb < prefix[hi]
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (prefix[mid] <= qb) lo = mid;
      else hi = mid;
    }
    qb -= prefix[lo];
    int b = lo * p.group;
    const int stop = min(p.batch, b + p.group);
    TcRow row(p, b);
    while (qb >= static_cast<unsigned>(row.blocks) && ++b < stop) {
      qb -= row.blocks;
      row = TcRow(p, b);
    }
    if (qb < static_cast<unsigned>(row.blocks)) {  // always, unless the count of blocks wrapped
      q0 = static_cast<int>(qb) * p.kq;
      start = row.start;
      n = row.n;
    }
  }
};
// Its keys: the window's [k_begin, k_begin + nw), the sinks [0, s_end) behind it, in nb blocks.
struct TcKeys {
  int k_begin, nw, s_end, nb;
  __device__ __forceinline__ TcKeys(const WinParams& w, int kq, int n, int q0, int block_keys) {
    const int q_last = min(n, q0 + kq) - 1;
    const int k_end = q_last + min(w.right, n - 1 - q_last) + 1;
    k_begin = q0 - min(w.left, q0);
    // no gap between sinks and window, or a row short enough to read whole
    if (w.sinks >= k_begin || (w.sinks > 0 && k_end <= block_keys)) k_begin = 0;
    s_end = min(w.sinks, k_begin);
    nw = k_end - k_begin;
    const int nv = ceil16(nw) + ceil16(s_end);
    nb = nv <= block_keys ? 1 : (nv + 127) / 128;
  }
};
// A published item.
struct TcItem {
  int live, start, n, h, q0, k_begin, nw, s_end, nb;
};

__device__ __forceinline__ void tmem_st_32x32b_x16(uint32_t taddr, const uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], "
      "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
      "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}
__device__ __forceinline__ void tmem_ld_32x32b_x8(uint32_t taddr, uint32_t (&r)[8]) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7])
               : "r"(taddr));
}
__device__ __forceinline__ float tmem_ld_1(uint32_t taddr) {
  uint32_t r;
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x1.b32 {%0}, [%1];" : "=r"(r) : "r"(taddr));
  tmem_wait_ld();
  return __uint_as_float(r);
}
template <bool H16>
__device__ __forceinline__ uint32_t pack16(float lo, float hi) {
  if constexpr (H16) {
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
  } else {
    const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
}
// bits [0, c) of 32, c clamped to 0 .. 32
__device__ __forceinline__ uint32_t low_bits(int c) {
  return c <= 0 ? 0u : c >= 32 ? 0xffffffffu : (1u << c) - 1u;
}
// First column of the P of keys [16 k, 16 k + 16): the first half of their
// 32-key piece's own score columns; pieces 6 and 7 lie in the second halves of
// pieces 0 and 1 (same parity: the same thread's columns).
__host__ __device__ constexpr uint32_t p_col(int k) {
  const int piece = k >> 1;
  return static_cast<uint32_t>((piece < 6 ? 32 * piece : 32 * (piece - 6) + 16) + 8 * (k & 1));
}

// The score column of a single-block item that a warp's rows take as their
// reference: a key of the window near the middle of the warp's own ones
// (`near`), else a sink.  Its column is one that P never overwrites (the second
// half of a piece, of pieces 2 to 5 where 6 and 7 put P into 0 and 1), since
// the two warps of a row read it at different times.  (Items of 16 columns have
// one piece, and one warp that uses the reference.)
__device__ __forceinline__ int ref_col(int nw, int nw16, int nv, int s_end, int near) {
  if (nw > 16 && (nv <= 192 || nw > 80)) {
    const int piece = min(near >> 5, (nw - 17) >> 5);  // its column 16 is a key
    return 32 * (nv > 192 ? max(piece, 2) : piece) + 16;
  }
  return nv > 192 ? 144 : s_end > 0 ? nw16 : 0;  // nw <= 80, nv > 192: columns 80 to 176 are sinks
}

// The items of a CTA's slot, [its.x, its.y], hold outputs that are not finite: a
// masked value contributed 0 * v, the softmax reference was far from the row's
// scores (those outputs were set to NaN), or they are so.  All warps of the CTA
// take the rows in turn, behind its last item, so that nothing waits for them.
// The columns of a row that are not finite are computed again from global
// memory, in f32, over the visible keys only: a key per lane for 32 scores at
// once, then lane c the columns c, c + 32, .. of their values.  In a row of
// several blocks only a NaN can be wrong, and only if one of its item's hidden
// values is the cause or, in f16, a visible infinity whose weight was rounded
// to 0; and a row ends early where every column it needs is NaN, so that long
// rows of visible values that are not finite cost little.
// Causal row of 8192 tokens, 16 heads of 64, one column infinite: 38 ms (0.41 ms
// without it).  64 x 512 tokens, 12 heads of 64, scores that deviate by 20 from
// one another (many bf16 rows then have a key 2^127 above the reference): 0.55 to
// 0.58 ms; by 8: 50 us, as by 1.
template <typename T, int D>
__device__ __forceinline__ void window_rows_exact(const TcParams& tp, const unsigned* prefix, int slot, int2 its) {
  const WinParams& p = tp.w;
  constexpr int CL = D / 32;  // columns of a lane
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int ld = (p.heads + 2 * p.kv_heads) * D;
  for (long long at = its.x * 128ll + warp; at < (its.y + 1) * 128ll; at += kTcWarps) {
    const TcPlace it(tp, prefix, static_cast<int>(slot * gridDim.x + blockIdx.x + (at >> 7) * 2 * gridDim.x));
    const int qi = it.q0 + static_cast<int>(at & 127), n = it.n, start = it.start;
    if ((at & 127) >= tp.kq || qi >= n) continue;
    const T* row = static_cast<const T*>(p.qkv) + static_cast<size_t>(start) * ld;
    const T* q = row + static_cast<size_t>(qi) * ld + it.h * D;
    const T* k = row + (p.heads + it.h / (p.heads / p.kv_heads)) * D;
    const T* v = k + p.kv_heads * D + lane;
    T* out = static_cast<T*>(p.ctx) + (static_cast<size_t>(start + qi) * p.heads + it.h) * D + lane;
    const TcKeys keys_of(p, tp.kq, n, it.q0, TcCfg<D>::KEYS);
    bool need[CL], any = false;
#pragma unroll
    for (int i = 0; i < CL; ++i) {
      const float y = to_f(out[32 * i]);
      any |= need[i] = y != y || (keys_of.nb == 1 && fabsf(y) == INFINITY);
    }
    if (!__any_sync(0xffffffffu, any)) continue;
    const int lo = qi - min(p.left, qi), hi = qi + min(p.right, n - 1 - qi);
    const int behind = min(p.sinks, lo);  // sinks in front of the window
    const int keys = behind + hi - lo + 1;
    if (keys_of.nb > 1) {  // the item's hidden keys: on both sides of the row's window, and those that pad the sinks
      float zero[CL] = {};
      auto add = [&](int j, int stop) {
        for (; j < stop; ++j)
#pragma unroll
          for (int i = 0; i < CL; ++i) zero[i] = fmaf(to_f(v[static_cast<size_t>(j) * ld + 32 * i]), 0.f, zero[i]);
      };
      add(max(keys_of.k_begin, min(p.sinks, lo)), lo);
      add(hi + 1, keys_of.k_begin + keys_of.nw);
      add(keys_of.s_end, min(ceil16(keys_of.s_end), p.rows - start));
      bool cause = false;
#pragma unroll
      for (int i = 0; i < CL; ++i) cause |= need[i] && zero[i] != 0.f;
      cause = __any_sync(0xffffffffu, cause);
      if constexpr (sizeof(T) == 2 && !std::is_same<T, bf16>::value) {
        for (int t0 = 0; t0 < keys && !cause; t0 += 32) {
#pragma unroll 8
          for (int t = t0; t < min(t0 + 32, keys); ++t) {
            const T* vj = v + static_cast<size_t>(t < behind ? t : lo + (t - behind)) * ld;
#pragma unroll
            for (int i = 0; i < CL; ++i) cause |= need[i] && fabsf(to_f(vj[32 * i])) == INFINITY;
          }
          cause = __any_sync(0xffffffffu, cause);
        }
      }
      if (!cause) continue;
    }
    float o[CL] = {}, l = 0.f, m = -INFINITY;
    bool lost = false;  // every column that is needed is NaN and stays so
    for (int t0 = 0; t0 < keys && !lost; t0 += 32) {
      const int t = min(t0 + lane, keys - 1);
      const int j = t < behind ? t : lo + (t - behind);
      const uint4* kj = reinterpret_cast<const uint4*>(k + static_cast<size_t>(j) * ld);
      const uint4* q4 = reinterpret_cast<const uint4*>(q);
      float s = 0.f;
#pragma unroll 2
      for (int c = 0; c < D / 8; ++c) {
        const uint4 a = q4[c], b = kj[c];
        const T* x = reinterpret_cast<const T*>(&a);
        const T* y = reinterpret_cast<const T*>(&b);
#pragma unroll
        for (int e = 0; e < 8; ++e) s = fmaf(to_f(x[e]), to_f(y[e]), s);
      }
      s = t0 + lane < keys ? s * p.scale_log2 : -INFINITY;
      const float top = fmaxf(m, warp_max(s)), ref = top == -INFINITY ? 0.f : top;
      const float corr = exp2f(m - ref), e = exp2f(s - ref);
      m = top;
      l = l * corr + warp_sum(e);
#pragma unroll
      for (int i = 0; i < CL; ++i) o[i] *= corr;
      const unsigned weighs = __ballot_sync(0xffffffffu, s != -INFINITY);  // the others not even 0 * NaN
#pragma unroll 4
      for (int i = 0; i < 32; ++i) {
        const float ei = __shfl_sync(0xffffffffu, e, i);
        const int ji = __shfl_sync(0xffffffffu, j, i);
        if (weighs >> i & 1) {
#pragma unroll
          for (int c = 0; c < CL; ++c) o[c] = fmaf(ei, to_f(v[static_cast<size_t>(ji) * ld + 32 * c]), o[c]);
        }
      }
      bool nan = true;
#pragma unroll
      for (int i = 0; i < CL; ++i) nan &= !need[i] || o[i] != o[i];
      lost = __all_sync(0xffffffffu, nan);
    }
#pragma unroll
    for (int i = 0; i < CL; ++i)
      if (need[i]) out[32 * i] = from_f<T>(o[i] / l);
  }
}

// Descriptor of a K-major (or, for V, MN-major) tile of 64- or 128-byte
// swizzled rows: 8-row groups contiguous.
template <int ROW>
__device__ __forceinline__ uint64_t tile_desc(uint32_t smem_addr) {
  if constexpr (ROW == 128) return umma_desc_sw128(smem_addr);
  return static_cast<uint64_t>((smem_addr & 0x3FFFF) >> 4) | (static_cast<uint64_t>(1) << 16) |
         (static_cast<uint64_t>(8 * ROW >> 4) << 32) | (static_cast<uint64_t>(1) << 46) |
         (static_cast<uint64_t>(4) << 61);  // SWIZZLE_64B
}

template <int D, bool H16>
__global__ void __launch_bounds__(kTcThreads, 1)
    window_tc_kernel(const __grid_constant__ TcParams p, const __grid_constant__ CUtensorMap tm64,
                     const __grid_constant__ CUtensorMap tm16) {
  using C = TcCfg<D>;
  using T = typename std::conditional<H16, f16, bf16>::type;
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0);  // uniform to the compiler too
  const int lane = threadIdx.x & 31;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw = smem_u32(smem_raw);
  const uint32_t base = (raw + 1023u) & ~1023u;
  const uint32_t staging = base + 2 * C::SLOT_BYTES;
  float* xch = reinterpret_cast<float*>(smem_raw + (staging + C::STAGE_BYTES - raw));
  unsigned* prefix = reinterpret_cast<unsigned*>(xch) + C::XCH_BYTES / 4;  // [entries + 1] query blocks before each group of rows
  uint8_t* meta = reinterpret_cast<uint8_t*>(prefix + kPrefixRows + 4);
  const int g = warp < 4 ? warp & 1 : (warp - 4) / kGroupWarps & 1;  // this warp's slot
  const uint32_t sQ = base + g * C::SLOT_BYTES, sK = sQ + C::Q_BYTES, sV = sK + C::KV_BYTES;
  const uint32_t bars = smem_u32(meta) + g * kSlotBars;
  const uint32_t ifull = bars;         // [2] an item is published
  const uint32_t kfull = bars + 16;    // K (and Q) of a block loaded
  const uint32_t vfull = bars + 24;
  const uint32_t sfull = bars + 32;    // S written: K (and Q) read
  const uint32_t pfull = bars + 40;    // P written
  const uint32_t ofull = bars + 48;    // P V done: V read
  const uint32_t sfree = bars + 56;    // O read
  const uint32_t spare = bars + 64;
  const uint32_t pairs = bars + 72;    // [4] the two warps of a lane quarter meet
  const uint32_t odone = bars + 104;   // an item's last P V done
  const uint32_t lfull = bars + 112;   // [2] an item's sums written
  uint32_t* tslot = reinterpret_cast<uint32_t*>(meta + 2 * kSlotBars);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(meta + 2 * kSlotBars + 4);
  volatile int* ends = reinterpret_cast<volatile int*>(meta + 2 * kSlotBars + 8);  // [2] a slot's number of items
  // four items a slot: the TMA warp is up to two ahead of the output warps
  volatile int* broken = ends + 2;  // [2][first, last item with an output that is not finite]
  volatile TcItem* rings = reinterpret_cast<volatile TcItem*>(meta + 2 * kSlotBars + 32);
  volatile TcItem* ring = rings + 4 * g;
  static_assert(2 * kSlotBars + 32 + 8 * sizeof(TcItem) <= C::META_BYTES, "meta layout");
  const WinParams& w = p.w;
  const int entries = p.entries;

  if (warp == 1 && lane == 0) {
    prefetch_tensormap(&tm64);
    prefetch_tensormap(&tm16);
  }
  // Query blocks before each group of rows: a scan by all warps, kTcThreads entries
  // a round.  (Unsigned: overlapping rows could have more than 32 bits count.)
  unsigned incl[kRounds], mine_blocks[kRounds];
#pragma unroll
  for (int i = 0; i < kRounds; ++i) {
    const int at = i * kTcThreads + threadIdx.x;
    unsigned blocks = 0;
    if (at < entries)
      for (int b = at * p.group, stop = min(p.batch, b + p.group); b < stop; ++b) blocks += TcRow(p, b).blocks;
    mine_blocks[i] = blocks;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const unsigned up = __shfl_up_sync(0xffffffffu, blocks, o);
      if (lane >= o) blocks += up;
    }
    incl[i] = blocks;
    if (lane == 31) reinterpret_cast<unsigned*>(xch)[i * kTcWarps + warp] = blocks;
  }
  __syncthreads();
  {
    unsigned before = 0;  // blocks of the warps before this one
    int w0 = 0;
#pragma unroll
    for (int i = 0; i < kRounds; ++i) {
      if (i * kTcThreads < entries || i == 0) {
        for (; w0 < i * kTcWarps + warp; ++w0) before += reinterpret_cast<unsigned*>(xch)[w0];
        const int at = i * kTcThreads + threadIdx.x;
        if (at < entries) prefix[at] = before + incl[i] - mine_blocks[i];
        if (at == entries - 1) prefix[entries] = before + incl[i];
      }
    }
  }
  if (threadIdx.x == 64) {
    for (int s = 0; s < 2; ++s) {
      const uint32_t b = smem_u32(meta) + s * kSlotBars;
      for (int i = 0; i < 9; ++i) mbar_init(b + 8 * i, i == 5 ? kGroupWarps : i == 7 ? 4 : 1);  // 5: pfull, 7: sfree
      for (int i = 9; i < 13; ++i) mbar_init(b + 8 * i, 2);
      mbar_init(b + 104, 1);
      for (int i = 14; i < 16; ++i) mbar_init(b + 8 * i, kGroupWarps);
    }
    *abort_flag = 0;
    ends[0] = ends[1] = -1;
    broken[0] = broken[2] = INT32_MAX;
    broken[1] = broken[3] = -1;
    fence_barrier_init();
  }
  if (warp == 3) tmem_alloc(smem_u32(tslot), 512);  // all of it (one CTA per SM): the base is column 0
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = static_cast<uint32_t>(g) * 256;
  // keys of block j of an item, in its own order: window, then sinks
  auto block_of = [&](int nv, int nb, int j, int& v0, int& v1) {
    v0 = nb == 1 ? 0 : 128 * j;
    v1 = nb == 1 ? nv : min(nv, v0 + 128);
  };

  // The TMA and MMA warps walk their loops whole and elect one lane around
  // each group of instructions, so that the operands stay in uniform
  // registers (see jb_mxfp4_gemm.cu).
  if (warp < 2) {  // ── TMA
    const long long items = min(static_cast<long long>(prefix[entries]) * w.heads, static_cast<long long>(INT32_MAX));
    const long long stride = 2ll * gridDim.x;
    int bc = 0, m = 0;  // blocks loaded, items published
    bool ok = true;
    const int hk_div = w.heads / w.kv_heads;
    for (long long f0 = static_cast<long long>(g) * gridDim.x + blockIdx.x; f0 < items && ok; f0 += 32 * stride) {
      const long long f = f0 + lane * stride;
      TcPlace mine;  // this lane's candidate
      if (f < items) mine = TcPlace(p, prefix, static_cast<int>(f));
      unsigned todo = __ballot_sync(0xffffffffu, mine.n > 0);
      while (todo && ok) {
        const int src = __ffs(todo) - 1;
        todo &= todo - 1;
        TcItem it;
        it.start = __shfl_sync(0xffffffffu, mine.start, src);
        it.n = __shfl_sync(0xffffffffu, mine.n, src);
        it.h = __shfl_sync(0xffffffffu, mine.h, src);
        it.q0 = __shfl_sync(0xffffffffu, mine.q0, src);
        const TcKeys keys(w, p.kq, it.n, it.q0, C::KEYS);
        it.k_begin = keys.k_begin;
        it.s_end = keys.s_end;
        it.nw = keys.nw;
        it.nb = keys.nb;
        const int nw16 = ceil16(it.nw), nv = nw16 + ceil16(it.s_end);
        const int xk = (w.heads + it.h / hk_div) * D, xv = xk + w.kv_heads * D;
        for (int j = 0; j < it.nb; ++j, ++bc) {
          int v0, v1;
          block_of(nv, it.nb, j, v0, v1);
          // window keys, then sinks, in boxes of 64 and 16 rows
          auto load_keys = [&](uint32_t dst, int x, uint32_t bar) {
            int v = v0;
            while (v < v1) {
              const bool win = v < nw16;
              const int stop = win ? min(v1, nw16) : v1;
              const int y = it.start + (win ? it.k_begin + v : v - nw16);
              const bool big = stop - v >= 64;
#pragma unroll
              for (int half = 0; half < C::HALVES; ++half)
                tma_load_2d(dst + half * (C::KEYS * C::ROW) + (v - v0) * C::ROW, big ? &tm64 : &tm16,
                            x + C::HCOLS * half, y, bar);
              v += big ? 64 : 16;
            }
          };
          if (bc > 0 && !warp_mbar_wait(sfull, (bc - 1) & 1, abort_flag)) { ok = false; break; }
          const uint32_t bytes = static_cast<uint32_t>(v1 - v0) * C::ROW * C::HALVES;
          const int boxes = (min(it.n - it.q0, p.kq) + 63) >> 6;
          if (elect_one()) {
            if (j == 0) {
              volatile TcItem& e = ring[m & 3];
              e.live = 1; e.start = it.start; e.n = it.n; e.h = it.h; e.q0 = it.q0;
              e.k_begin = it.k_begin; e.nw = it.nw; e.s_end = it.s_end; e.nb = it.nb;
              mbar_arrive(ifull + 8 * (m & 1));
              mbar_arrive_expect_tx(kfull, bytes + boxes * 64 * C::ROW * C::HALVES);
              for (int i = 0; i < boxes; ++i)
#pragma unroll
                for (int half = 0; half < C::HALVES; ++half)
                  tma_load_2d(sQ + half * (128 * C::ROW) + i * (64 * C::ROW), &tm64, it.h * D + C::HCOLS * half,
                              it.start + it.q0 + 64 * i, kfull);
            } else {
              mbar_arrive_expect_tx(kfull, bytes);
            }
            load_keys(sK, xk, kfull);
          }
          __syncwarp();
          if (j == 0) ++m;
          if (bc > 0 && !warp_mbar_wait(ofull, (bc - 1) & 1, abort_flag)) {
            volatile int no_abort = 0;
            warp_mbar_wait(kfull, bc & 1, &no_abort);  // this block's copies land (bounded)
            ok = false;
            break;
          }
          if (elect_one()) {
            mbar_arrive_expect_tx(vfull, bytes);
            load_keys(sV, xv, vfull);
          }
          __syncwarp();
        }
      }
    }
    if (lane == 0) {
      if (ok && (bc == 0 || mbar_wait(sfull, (bc - 1) & 1, abort_flag))) {  // no more items
        ring[m & 3].live = 0;
        mbar_arrive(ifull + 8 * (m & 1));
        mbar_arrive(kfull);
      }
      if (*abort_flag && bc > 0) {  // the last copies land before the CTA leaves (bounded)
        volatile int no_abort = 0;
        mbar_wait(kfull, (bc - 1) & 1, &no_abort);
        mbar_wait(vfull, (bc - 1) & 1, &no_abort);
      }
    }
  } else if (warp < 4) {  // ── MMA
    const uint32_t idesc_pv =
        (H16 ? idesc_f16_f32(128, C::HCOLS) : idesc_bf16_f32(128, C::HCOLS)) | (1u << 16);  // V MN-major
    int bc = 0;
    bool ok = true;
    for (int m = 0; ok; ++m) {
      if (!warp_mbar_wait(kfull, bc & 1, abort_flag)) { ok = false; break; }
      const volatile TcItem& e = ring[m & 3];
      if (!e.live) {  // the output warps may go, once all of them have seen the last item
        if (m > 0 && !warp_mbar_wait(sfree, (m - 1) & 1, abort_flag)) ok = false;
        if (ok && lane == 0) {
          ends[g] = m;
          mbar_arrive(odone);
        }
        break;
      }
      const int nv = __shfl_sync(0xffffffffu, ceil16(e.nw) + ceil16(e.s_end), 0);
      const int nb = __shfl_sync(0xffffffffu, e.nb, 0);
      for (int j = 0; j < nb; ++j, ++bc) {
        int v0, v1;
        block_of(nv, nb, j, v0, v1);
        // The first S replaces the P of the item before, which P V has read, and,
        // where it is wide, that item's O.
        if (j == 0 && m > 0 &&
            !(v1 - v0 <= C::O_COL ? warp_mbar_wait(ofull, (bc - 1) & 1, abort_flag)
                                  : warp_mbar_wait(sfree, (m - 1) & 1, abort_flag))) {
          ok = false;
          break;
        }
        // S_j replaces P_{j-1}, which P V has read
        if (j > 0 &&
            (!warp_mbar_wait(kfull, bc & 1, abort_flag) || !warp_mbar_wait(ofull, (bc - 1) & 1, abort_flag))) {
          ok = false;
          break;
        }
        tc_fence_after();
        const uint32_t idesc = H16 ? idesc_f16_f32(128, v1 - v0) : idesc_bf16_f32(128, v1 - v0);
        if (elect_one()) {
#pragma unroll
          for (int half = 0; half < C::HALVES; ++half) {
            const uint64_t dq = tile_desc<C::ROW>(sQ + half * (128 * C::ROW));
            const uint64_t dk = tile_desc<C::ROW>(sK + half * (C::KEYS * C::ROW));
#pragma unroll
            for (int kk = 0; kk < C::HCOLS / 16; ++kk) mma_bf16(tmem, dq + 2u * kk, dk + 2u * kk, idesc, (half | kk) != 0);
          }
          mma_commit(sfull);
        }
        __syncwarp();
        // (P comes last)
        if ((j == 0 && m > 0 && !warp_mbar_wait(sfree, (m - 1) & 1, abort_flag)) ||
            !warp_mbar_wait(vfull, bc & 1, abort_flag) || !warp_mbar_wait(pfull, bc & 1, abort_flag)) {
          ok = false;
          break;
        }
        tc_fence_after();
        const int steps = (v1 - v0) >> 4;
        if (elect_one()) {
#pragma unroll
          for (int half = 0; half < C::HALVES; ++half) {
            const uint64_t dv = tile_desc<C::ROW>(sV + half * (C::KEYS * C::ROW));
#pragma unroll
            for (int c = 0; c < C::KEYS / 16; ++c)
              if (c < steps)
                mma_bf16_ta(tmem + C::O_COL + C::HCOLS * half, tmem + p_col(c), dv + static_cast<uint32_t>(C::ROW) * c, idesc_pv,
                            (j > 0 || c > 0) ? 1u : 0u);
          }
          mma_commit(ofull);
          if (j == nb - 1) mma_commit(odone);
        }
        __syncwarp();
      }
    }
    if (!ok) {  // every MMA issued completes before TMEM is freed (bounded)
      volatile int no_abort = 0;
      if (elect_one()) mma_commit(spare);
      __syncwarp();
      warp_mbar_wait(spare, 0, &no_abort);
    }
  } else if (warp < 4 + 2 * kGroupWarps) {  // ── softmax
    const int quarter = warp & 3, half = ((warp - 4) >> 2) & 1;
    const int r = 32 * quarter + lane;
    const uint32_t trow = tmem + (static_cast<uint32_t>(32 * quarter) << 16);
    const uint32_t pair = pairs + 8 * quarter;
    // [4] max (by block parity), sum (by item parity); then [half][lane]
    float* xq = xch + ((g * 4) * 4 + quarter) * 64 + lane;
    int meets = 0;
    auto meet = [&]() -> bool {  // what both warps wrote before is visible to both
      __syncwarp();
      if (lane == 0) mbar_arrive(pair);
      return warp_mbar_wait(pair, (meets++) & 1, abort_flag);
    };
    int bc = 0;
    bool ok = true;
    for (int m = 0; ok; ++m) {
      if (!warp_mbar_wait(ifull + 8 * (m & 1), (m >> 1) & 1, abort_flag)) break;
      const volatile TcItem& e = ring[m & 3];
      if (!e.live) break;
      const int n = e.n, q0 = e.q0, k_begin = e.k_begin, nw = e.nw, s_end = e.s_end, nb = e.nb;
      const int nw16 = ceil16(nw), nv = nw16 + ceil16(s_end);
      const int qi = q0 + r;
      const int rows = min(p.kq, n - q0) - 32 * quarter;  // rows of this warp's quarter (32 and more: all)
      const bool mine = lane < rows;
      const bool active = rows > 0;
      // visible keys of this row, relative to k_begin
      const int lo = qi - min(w.left, qi) - k_begin;
      const int hi = mine ? qi + min(w.right, n - 1 - qi) - k_begin : -1;
      const int first = min(w.sinks - k_begin, hi + 1);  // sinks inside the window's range
      auto visible = [&](int v) -> uint32_t {  // keys [v, v + 32) of the item's order
        uint32_t bits = 0;
        if (v < nw16) bits = (low_bits(hi + 1 - v) & ~low_bits(lo - v)) | low_bits(first - v);
        if (v + 32 > nw16 && s_end > 0 && mine) {
          const int c = nw16 - v;  // the sinks' first bit
          bits |= c >= 0 ? low_bits(s_end) << c : low_bits(s_end + c);
        }
        return bits;
      };
      float mref = -INFINITY, l = 0.f;
      for (int j = 0; j < nb; ++j, ++bc) {
        int v0, v1;
        block_of(nv, nb, j, v0, v1);
        if (!warp_mbar_wait(sfull, bc & 1, abort_flag)) { ok = false; break; }
        tc_fence_after();
        if (active && !H16 && nb == 1) {
          // The reference is the row's score with one key of the item (see ref_col):
          // bf16 P has f32's range, so any reference within 2^100 of the row's
          // maximum gives the same relative rounding, and no maximum is needed.
          // (A sum outside that range: window_rows_exact.)
          mref = tmem_ld_1(trow + ref_col(nw, nw16, nv, s_end, q0 + 32 * quarter - k_begin + 16)) * w.scale_log2;
        } else if (active) {
          float mx = -INFINITY;
#pragma unroll 1
          for (int c = 32 * half; c < v1 - v0; c += 64) {
            const uint32_t bits = visible(v0 + c);
            if (!__any_sync(0xffffffffu, bits != 0)) continue;
            uint32_t s[32];
            tmem_ld_32x32b_x32(trow + c, s);
            tmem_wait_ld();
#pragma unroll
            for (int i = 0; i < 32; ++i)
              if (bits >> i & 1) mx = fmaxf(mx, __uint_as_float(s[i]));
          }
          float* xm = xq + (bc & 1) * 256;
          xm[32 * half] = mx;
          if (!meet()) { ok = false; break; }
          mx = fmaxf(mx, xm[32 * (half ^ 1)]);
          const float mb = mx * w.scale_log2;
          if (j == 0) {
            mref = mb;
          } else {
            // both threads of a row decide alike; each rescales its half of O
            const bool up = mb > mref + kRescale<H16>;  // always behind scores of -infinity only
            if (__any_sync(0xffffffffu, up)) {
              const float alpha = up ? ex2_approx(mref - mb) : 1.f;
              l *= alpha;
#pragma unroll 1
              for (int c = half * (D / 2); c < (half + 1) * (D / 2); c += 8) {
                uint32_t o8[8];
                tmem_ld_32x32b_x8(trow + C::O_COL + c, o8);
                tmem_wait_ld();
#pragma unroll
                for (int i = 0; i < 8; ++i) o8[i] = __float_as_uint(__uint_as_float(o8[i]) * alpha);
                tmem_st_32x32b_x8(trow + C::O_COL + c, o8);
              }
              tmem_wait_st();
              if (up) mref = mb;
            }
          }
        }
        if (active) {
          float2 l2 = make_float2(0.f, 0.f);
          const float lift = !H16 ? 0.f : nb == 1 ? kLift1 : kLift;
          const float ref = mref == -INFINITY ? 0.f : mref - lift;  // nothing seen so far: p stays 0
#pragma unroll 1
          for (int c = 32 * half; c < v1 - v0; c += 64) {
            const uint32_t bits = visible(v0 + c);
            uint32_t pk[16];
            if (!__any_sync(0xffffffffu, bits != 0)) {
#pragma unroll
              for (int i = 0; i < 16; ++i) pk[i] = 0;
            } else {
              uint32_t s[32];
              tmem_ld_32x32b_x32(trow + c, s);
              tmem_wait_ld();
#pragma unroll
              for (int i = 0; i < 32; i += 2) {
                float2 z = __ffma2_rn(make_float2(__uint_as_float(s[i]), __uint_as_float(s[i + 1])),
                                      f2(w.scale_log2), f2(-ref));
                if (!(bits >> i & 1)) z.x = -INFINITY;
                if (!(bits >> (i + 1) & 1)) z.y = -INFINITY;
                const float2 e2 = make_float2(ex2_approx(z.x), ex2_approx(z.y));
                l2 = __fadd2_rn(l2, e2);
                pk[i >> 1] = pack16<H16>(e2.x, e2.y);
              }
            }
            tmem_st_32x32b_x16(trow + p_col(c >> 4), pk);
          }
          l += l2.x + l2.y;
          tmem_wait_st();
        }
        // V rows [nw, nw16) belong to no key of the item: their product with
        // P = 0 must be 0
        if (nw16 > nw && nw16 > v0 && nw16 <= v1) {
          if (!warp_mbar_wait(vfull, bc & 1, abort_flag)) { ok = false; break; }
          constexpr int kChunks = C::ROW / 16;
          for (int i = r + 128 * half; i < (nw16 - nw) * kChunks * C::HALVES; i += 256) {
            const int row = i / kChunks, blk = row / (nw16 - nw);
            const uint32_t a = sV + blk * (C::KEYS * C::ROW) +
                               static_cast<uint32_t>(nw - v0 + row - blk * (nw16 - nw)) * C::ROW + i % kChunks * 16;
            asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};" ::"r"(a), "r"(0) : "memory");
          }
          fence_proxy_async_smem();
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(pfull);
      }
      if (!ok) break;
      xq[(2 + (m & 1)) * 256 + 32 * half] = l;
      __syncwarp();
      if (lane == 0) mbar_arrive(lfull + 8 * (m & 1));
    }
  } else {  // ── output, of both slots: whichever has an item done
    const int quarter = warp & 3;
    const uint32_t stage = staging + static_cast<uint32_t>(quarter) * 32 * C::SEG;
    int done[2] = {0, 0};
    bool more[2] = {true, true};
    while (more[0] || more[1]) {
      int s = -1;
      uint64_t t0 = 0;
#pragma unroll 1
      for (int i = 0; s < 0; ++i) {
        const bool a = more[0] && mbar_test_wait(smem_u32(meta) + 104, done[0] & 1);
        const bool b = more[1] && mbar_test_wait(smem_u32(meta) + kSlotBars + 104, done[1] & 1);
        if (__all_sync(0xffffffffu, a)) s = 0;
        else if (__all_sync(0xffffffffu, b)) s = 1;
        else if ((i & 63) == 63) {
          bool late = *abort_flag != 0;
          if (t0 == 0) t0 = global_timer_ns();
          else if (global_timer_ns() - t0 > kWaitLimitNs) *abort_flag = 1, late = true;
          if (__any_sync(0xffffffffu, late)) break;
        }
      }
      if (s < 0) break;
      const int m = s ? done[1] : done[0];
      if (s) ++done[1]; else ++done[0];
      if (ends[s] == m) {
        if (s) more[1] = false; else more[0] = false;
        continue;
      }
      const uint32_t sbars = smem_u32(meta) + s * kSlotBars;
      if (!warp_mbar_wait(sbars + 112 + 8 * (m & 1), (m >> 1) & 1, abort_flag)) break;
      const volatile TcItem& e = rings[4 * s + (m & 3)];
      tc_fence_after();
      const int start = e.start, n = e.n, h = e.h, q0 = e.q0, nb = e.nb;
      const int rows = min(p.kq, n - q0) - 32 * quarter;  // rows of this warp's quarter (32 and more: all)
      const uint32_t to = s * 256u + (static_cast<uint32_t>(32 * quarter) << 16) + C::O_COL;
      const float* xs = xch + ((s * 4 + 2 + (m & 1)) * 4 + quarter) * 64 + lane;
      // (NaN: see window_rows_exact.  Of one block the sum is taken only where the
      // reference was near the row's maximum; its outputs may even be 0 otherwise.)
      const float l_row = xs[0] + xs[32];
      const float inv = nb > 1 || (l_row > 0x1p-100f && l_row < INFINITY) ? 1.f / l_row : __int_as_float(0x7fffffff);
      T* out = static_cast<T*>(w.ctx) + (static_cast<size_t>(start + q0 + 32 * quarter) * w.heads + h) * D;
      float2 zero2 = make_float2(0.f, 0.f);  // sum of o * 0: NaN if any output is not finite
      constexpr int kSlots = C::SEG / 16, kShift = kSlots == 4 ? 1 : 0;  // 16-byte slots of a staged row
      constexpr int kRowsPerIns = 32 / kSlots;
      auto slot_at = [&](int row, int q) {
        return stage + row * C::SEG + ((q ^ ((row >> kShift) & (kSlots - 1))) << 4);
      };
#pragma unroll
      for (int c = 0; c < D; c += 32) {
        uint32_t o[32];
        if (rows > 0) {
          tmem_ld_32x32b_x32(to + c, o);
          tmem_wait_ld();
        }
        if (c + 32 == D) {  // the slot's O may be overwritten
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(sbars + 56);
        }
        if (rows > 0) {
          if (c % (C::SEG / 2) == 0) __syncwarp();  // the staged rows before have been read
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            uint32_t pk[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const float2 y = __fmul2_rn(make_float2(__uint_as_float(o[8 * q + 2 * i]),
                                                      __uint_as_float(o[8 * q + 2 * i + 1])), f2(inv));
              zero2 = __ffma2_rn(y, make_float2(0.f, 0.f), zero2);
              pk[i] = pack16<H16>(y.x, y.y);
            }
            asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(slot_at(lane, c % (C::SEG / 2) / 8 + q)),
                         "r"(pk[0]), "r"(pk[1]), "r"(pk[2]), "r"(pk[3])
                         : "memory");
          }
          if ((c + 32) % (C::SEG / 2) == 0) {
            __syncwarp();
#pragma unroll
            for (int i = 0; i < kSlots; ++i) {
              const int row = i * kRowsPerIns + lane / kSlots, q = lane % kSlots;
              uint32_t v0, v1, v2, v3;
              asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];"
                           : "=r"(v0), "=r"(v1), "=r"(v2), "=r"(v3)
                           : "r"(slot_at(row, q))
                           : "memory");
              if (row < rows)
                *reinterpret_cast<uint4*>(out + static_cast<size_t>(row) * w.heads * D + c + 32 - C::SEG / 2 + 8 * q) =
                    make_uint4(v0, v1, v2, v3);
            }
          }
        }
      }
      bool wrong = lane < rows && !(zero2.x + zero2.y == 0.f);
      // A reference far above the row's scores and small values: outputs whose
      // products p v fell to where f32 has few bits left, or none
      const bool far = !H16 && nb == 1 && lane < rows && l_row < 0x1p-24f;
      if (__any_sync(0xffffffffu, far)) {
        __syncwarp();  // the rows' outputs are written
        T* y = out + static_cast<size_t>(lane) * w.heads * D;
#pragma unroll 2
        for (int c = 0; far && c < D; c += 8) {
          uint4 raw = *reinterpret_cast<const uint4*>(y + c);
          T* y8 = reinterpret_cast<T*>(&raw);
          bool low = false;
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            if (fabsf(to_f(y8[i])) * l_row < 0x1p-100f) {
              y8[i] = from_f<T>(__int_as_float(0x7fffffff));
              low = true;
            }
          }
          if (low) *reinterpret_cast<uint4*>(y + c) = raw;
          wrong |= low;
        }
      }
      if (__any_sync(0xffffffffu, wrong) && lane == 0) {
        atomicMin(const_cast<int*>(broken) + 2 * s, m);
        atomicMax(const_cast<int*>(broken) + 2 * s + 1, m);
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  if (threadIdx.x == 0 && *abort_flag && p.err) atomicOr(p.err, kErrTimeout);
  if (warp == 3) {
    __syncwarp();
    tc_fence_after();
    tmem_dealloc(*tslot, 512);
  }
  if (!*abort_flag)
    for (int s = 0; s < 2; ++s) window_rows_exact<T, D>(p, prefix, s, make_int2(broken[2 * s], broken[2 * s + 1]));
}

// Map over qkv [rows, cols] of 16-bit elements with boxes of row_bytes (64 or
// 128, swizzled) x box_rows.
bool make_map(CUtensorMap* map, const void* qkv, bool h16, int rows, int cols, int row_bytes, int box_rows) {
  static const PFN_cuTensorMapEncodeTiled_v12000 enc = [] {
    void* ptr = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &ptr, cudaEnableDefault, &q) != cudaSuccess ||
        q != cudaDriverEntryPointSuccess)
      ptr = nullptr;
    return reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(ptr);
  }();
  if (!enc) return false;
  const cuuint64_t dims[2] = {static_cast<cuuint64_t>(cols), static_cast<cuuint64_t>(rows)};
  const cuuint64_t strides[1] = {static_cast<cuuint64_t>(cols) * 2};
  const cuuint32_t box[2] = {static_cast<cuuint32_t>(row_bytes / 2), static_cast<cuuint32_t>(box_rows)};
  const cuuint32_t estr[2] = {1, 1};
  return enc(map, h16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, const_cast<void*>(qkv),
             dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
             row_bytes == 128 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B,
             CU_TENSOR_MAP_L2_PROMOTION_L2_128B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// Queries per item: 128, or fewer where that keeps a long row's window and
// sinks inside one 256-key block (head_dim 32 or 64).
int queries_per_item(const WindowArgs& a) {
  if (a.head_dim == 128 || a.sinks == 0 || a.max_len <= 256) return 128;
  const long long spare = 256ll - a.left - a.right - ((a.sinks + 15ll) & ~15ll);
  return spare >= 128 || spare < 64 ? 128 : static_cast<int>(spare) & ~15;
}

template <int D, bool H16>
cudaError_t launch_tc(const WindowArgs& a, WinParams w, cudaStream_t s, std::string* why) {
  CUtensorMap tm64, tm16;
  const int cols = (a.heads + 2 * a.kv_heads) * D;
  if (!make_map(&tm64, a.qkv, H16, a.rows, cols, TcCfg<D>::ROW, 64) ||
      !make_map(&tm16, a.qkv, H16, a.rows, cols, TcCfg<D>::ROW, 16)) {
    if (why) *why = "attention_window: cuTensorMapEncodeTiled failed";
    return cudaErrorInvalidValue;
  }
  auto kern = window_tc_kernel<D, H16>;
  int dev = 0;
  cudaGetDevice(&dev);
  // the shared-memory opt-in is a property of each device's context
  static std::atomic<uint8_t> attr_set[64];
  if (dev < 0 || dev >= 64 || !attr_set[dev].load(std::memory_order_acquire)) {
    const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, TcCfg<D>::SMEM);
    if (e != cudaSuccess) return e;
    if (dev >= 0 && dev < 64) attr_set[dev].store(1, std::memory_order_release);
  }
  TcParams p;
  p.kq = queries_per_item(a);
  w.q_blocks = (a.max_len + p.kq - 1) / p.kq;
  p.w = w;
  p.batch = a.batch;
  p.group = (a.batch + kPrefixRows - 1) / kPrefixRows;
  p.entries = (a.batch + p.group - 1) / p.group;
  p.err = a.err;
  const long long most = static_cast<long long>(a.batch) * w.q_blocks * a.heads;
  const int grid = static_cast<int>(std::min<long long>(num_sms(dev), most));
  kern<<<grid, kTcThreads, TcCfg<D>::SMEM, s>>>(p, tm64, tm16);
  return cudaGetLastError();
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
  p.rows = a.rows;
  p.max_len = a.max_len;
  p.q_blocks = 0;
  p.left = a.left;
  p.right = a.right;
  p.sinks = a.sinks;
  p.scale_log2 = 1.4426950408889634f / sqrtf(static_cast<float>(a.head_dim));
  switch (a.dtype) {
    case JB_DT_F32: return launch_simt<float>(p, a.head_dim, a.batch, a.max_len, s, why);
    case JB_DT_BF16:
      switch (a.head_dim) {
        case 32: return launch_tc<32, false>(a, p, s, why);
        case 64: return launch_tc<64, false>(a, p, s, why);
        case 128: return launch_tc<128, false>(a, p, s, why);
        default: return launch_simt<bf16>(p, a.head_dim, a.batch, a.max_len, s, why);
      }
    case JB_DT_F16:
      switch (a.head_dim) {
        case 32: return launch_tc<32, true>(a, p, s, why);
        case 64: return launch_tc<64, true>(a, p, s, why);
        case 128: return launch_tc<128, true>(a, p, s, why);
        default: return launch_simt<f16>(p, a.head_dim, a.batch, a.max_len, s, why);
      }
    default: return cudaErrorInvalidValue;
  }
}

}  // namespace jb
