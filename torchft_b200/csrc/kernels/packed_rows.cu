// What packed batches need besides the attention itself: which keys each token of a row of documents sees, and rotary positions
// that a token brings along, on several axes.
#include <algorithm>
#include <limits.h>

#include "ftb200_common.cuh"

namespace {

// ------------------------------------------------------------------ spans
// A row of `seq` tokens holds documents one after another: runs of equal ids, an id below zero is padding.  What a token sees is
// one range of keys [lo, hi), and who sees a key is one range of queries [from, to):
//   causal      lo = max(start, i - window + 1) or start, hi = max(i + 1, prefix end)
//               from = i < prefix end ? start : i, to = min(end, i + window) or end
//   otherwise   lo = from = start, hi = to = end
// (prefix end = start plus the flagged tokens that open the document).  Empty (0, 0) for padding.  Over the tokens that are not padding no
// bound ever decreases, so that the keys of 128 queries lie in one range, and the queries of 128 keys too: `tiles` holds both.
//
// A block per row; a thread walks over a run of neighbouring tokens three times (backwards for what comes next, forwards for the start,
// then the result), and two scans over the block carry what lies beyond.
constexpr int SPAN_THREADS = 1024;
constexpr int TILE = 128;
constexpr int NONE = INT_MAX;

struct SpanTile {  // of 128 tokens; NONE / 0 where there is nothing
  int lo, hi;            // keys that its queries see: some query sees something in [lo, hi)
  int all_lo, all_hi;    // keys that each of its queries sees; NONE, 0 with padding among them
  int from, to;          // queries that see some of its keys
  int all_from, all_to;  // queries that see each of its keys; NONE, 0 with padding among them or where the row ends inside
};

__device__ __forceinline__ int warp_min_i(int v) { return __reduce_min_sync(0xffffffffu, v); }
__device__ __forceinline__ int warp_max_i(int v) { return __reduce_max_sync(0xffffffffu, v); }

__global__ void __launch_bounds__(SPAN_THREADS) spans_kernel(const int* documents, const unsigned char* prefix, int4* rows, int* positions,
                                                             SpanTile* tiles, int* padded, int seq, int causal, int window) {
  ftb200::wait_for_previous();
  ftb200::start_next();
  __shared__ int2 next_of[32];   // per warp: first start and first unflagged token
  __shared__ int2 start_of[32];  // per warp: last start and the end of its prefix
  __shared__ int any_padding;
  const int b = blockIdx.x, lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
  const long long base = static_cast<long long>(b) * seq;
  const int* id = documents + base;
  const unsigned char* flag = prefix == nullptr ? nullptr : prefix + base;
  const int per = (seq + static_cast<int>(blockDim.x) - 1) / static_cast<int>(blockDim.x);
  const int i0 = static_cast<int>(min(static_cast<long long>(seq), static_cast<long long>(threadIdx.x) * per));
  const int i1 = min(seq, i0 + per);
  auto starts = [&](int i) { return i == 0 || id[i] != id[i - 1]; };
  auto flagged = [&](int i) { return flag != nullptr && flag[i] != 0; };
  if (threadIdx.x == 0) any_padding = 0;

  // the first start and the first unflagged token from each thread's first token on, then of all threads behind it
  int first_start = seq, first_plain = seq;
  for (int i = i1 - 1; i >= i0; --i) {
    if (starts(i)) first_start = i;
    if (!flagged(i)) first_plain = i;
  }
  int s = first_start, u = first_plain;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int s2 = __shfl_down_sync(0xffffffffu, s, o), u2 = __shfl_down_sync(0xffffffffu, u, o);
    if (lane + o < 32) {
      s = min(s, s2);
      u = min(u, u2);
    }
  }
  if (lane == 0) next_of[warp] = make_int2(s, u);
  __syncthreads();
  int next_start = __shfl_down_sync(0xffffffffu, s, 1), next_plain = __shfl_down_sync(0xffffffffu, u, 1);
  if (lane == 31) next_start = next_plain = seq;
  for (int w = warp + 1; w < warps; ++w) {
    next_start = min(next_start, next_of[w].x);
    next_plain = min(next_plain, next_of[w].y);
  }

  // this thread's last start and the end of the prefix that opens there
  int last_start = -1, last_prefix = 0;
  {
    int ns = next_start, np = next_plain;
    for (int i = i1 - 1; i >= i0; --i) {
      if (!flagged(i)) np = i;
      if (starts(i)) {
        if (last_start < 0) {
          last_start = i;
          last_prefix = min(np, ns);
        }
        ns = i;
      }
    }
  }
  int ls = last_start, lp = last_prefix;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int s2 = __shfl_up_sync(0xffffffffu, ls, o), p2 = __shfl_up_sync(0xffffffffu, lp, o);
    if (lane >= o && ls < 0) {
      ls = s2;
      lp = p2;
    }
  }
  if (lane == 31) start_of[warp] = make_int2(ls, lp);
  __syncthreads();
  int start = __shfl_up_sync(0xffffffffu, ls, 1), prefix_end = __shfl_up_sync(0xffffffffu, lp, 1);
  if (lane == 0) start = -1;
  for (int w = warp - 1; w >= 0 && start < 0; --w) {
    start = start_of[w].x;
    prefix_end = start_of[w].y;
  }

  // the spans, from the front: the end of a document is the next start behind it
  int end = -1;
  bool padding = false;
  for (int i = i0; i < i1; ++i) {
    if (starts(i) || end < 0) {
      if (starts(i)) {
        start = i;
        prefix_end = -1;
      }
      end = next_start;
      for (int k = i + 1; k < i1; ++k)
        if (starts(k)) {
          end = k;
          break;
        }
      if (prefix_end < 0) {
        prefix_end = i;
        while (prefix_end < i1 && prefix_end < end && flagged(prefix_end)) ++prefix_end;
        if (prefix_end == i1) prefix_end = min(next_plain, end);
      }
    }
    int4 r = make_int4(start, end, start, end);
    if (causal) {
      if (window > 0) {
        r.x = max(start, i - window + 1);
        r.w = i < end - window ? i + window : end;
      }
      r.y = max(i + 1, prefix_end);
      if (i >= prefix_end) r.z = i;
    }
    if (id[i] < 0) {
      r = make_int4(0, 0, 0, 0);
      padding = true;
    }
    rows[base + i] = r;
    positions[base + i] = i - start;
  }
  if (padding) any_padding = 1;
  __syncthreads();
  if (threadIdx.x == 0) padded[b] = any_padding;

  // a warp per tile, over what the block has just written
  const int n_tiles = (seq + TILE - 1) / TILE;
  for (int t = warp; t < n_tiles; t += warps) {
    SpanTile x = {NONE, 0, 0, NONE, NONE, 0, 0, NONE};
    int all_q = 1, all_k = 1;
#pragma unroll
    for (int k = 0; k < TILE / 32; ++k) {
      const int i = t * TILE + k * 32 + lane;
      if (i >= seq) {
        all_k = 0;
        continue;
      }
      const int4 r = rows[base + i];
      if (r.y <= r.x) {
        all_q = all_k = 0;
        continue;
      }
      x.lo = min(x.lo, r.x), x.hi = max(x.hi, r.y);
      x.all_lo = max(x.all_lo, r.x), x.all_hi = min(x.all_hi, r.y);
      x.from = min(x.from, r.z), x.to = max(x.to, r.w);
      x.all_from = max(x.all_from, r.z), x.all_to = min(x.all_to, r.w);
    }
    x.lo = warp_min_i(x.lo), x.hi = warp_max_i(x.hi);
    x.all_lo = warp_max_i(x.all_lo), x.all_hi = warp_min_i(x.all_hi);
    x.from = warp_min_i(x.from), x.to = warp_max_i(x.to);
    x.all_from = warp_max_i(x.all_from), x.all_to = warp_min_i(x.all_to);
    all_q = __all_sync(0xffffffffu, all_q), all_k = __all_sync(0xffffffffu, all_k);
    if (!all_q) x.all_lo = NONE, x.all_hi = 0;
    if (!all_k) x.all_from = NONE, x.all_to = 0;
    if (lane == 0) tiles[static_cast<long long>(b) * n_tiles + t] = x;
  }
}

// ------------------------------------------------------------------ rotary positions with several axes
// Pair j of every rotated head of token t turns by positions[axis[j]][t] * inv_freq[j], in place; an axis outside [0, axes) leaves
// it.  Pairs are neighbours (2j, 2j + 1) or, with HALF, (j, j + dim / 2).  The angle is a product in 64 bits, brought into one turn there:
// at position 2^20 32 bits are off by 0.06 rad.
//
// Bound by memory.  A block takes `per_block` tokens: each (token, pair) has its sine taken once, into shared memory, while the first
// vectors are on their way, and serves all heads.  8192 tokens, 40 of 48 heads of 128: 65 us.
constexpr int ROPE_THREADS = 256;
constexpr int ROPE_LOADS = 4;  // vectors (pairs of them with HALF) a thread has in flight

template <typename T>
struct alignas(16) Vec16 {
  static constexpr int N = 16 / sizeof(T);
  T v[N];
};
__device__ __forceinline__ float widen(float x) { return x; }
__device__ __forceinline__ float widen(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ void narrow(float x, float& y) { y = x; }
__device__ __forceinline__ void narrow(float x, __nv_bfloat16& y) { y = __float2bfloat16_rn(x); }

template <typename T, bool HALF>
__global__ void __launch_bounds__(ROPE_THREADS) rope_axes_kernel(T* buf, const int* positions, const double* inv_freq, const int* axis,
                                                                 long long tokens, int axes, int n_heads, int dim, long long ld,
                                                                 int per_block, float sign) {
  ftb200::wait_for_previous();
  ftb200::start_next();
  using V = Vec16<T>;
  constexpr int VECS = HALF ? 2 : 1;         // vectors of a unit of work
  constexpr int PAIRS = V::N * VECS / 2;     // pairs in it
  extern __shared__ float2 turn[];           // [per_block][dim / 2], (cos, sin)
  const int half = dim / 2;
  const long long t0 = static_cast<long long>(blockIdx.x) * per_block;
  const int n_tokens = static_cast<int>(min(static_cast<long long>(per_block), tokens - t0));
  const int per_head = half / PAIRS, per_token = n_heads * per_head;
  const int units = n_tokens * per_token;

  V x[ROPE_LOADS][VECS];
  auto place = [&](int unit, int& pair, int& token) {
    token = unit / per_token;
    const int r = unit - token * per_token;
    const int h = r / per_head;
    pair = (r - h * per_head) * PAIRS;
    return buf + (t0 + token) * ld + static_cast<long long>(h) * dim + (HALF ? pair : 2 * pair);
  };
  auto load = [&](int first) {
#pragma unroll
    for (int k = 0; k < ROPE_LOADS; ++k) {
      const int unit = first + k * ROPE_THREADS;
      if (unit >= units) break;
      int pair, token;
      const T* p = place(unit, pair, token);
#pragma unroll
      for (int e = 0; e < VECS; ++e) x[k][e] = *reinterpret_cast<const V*>(p + e * half);
    }
  };
  load(threadIdx.x);
  for (int i = threadIdx.x; i < n_tokens * half; i += ROPE_THREADS) {
    const int token = i / half, j = i - token * half;
    const int a = axis[j];
    float2 cs = make_float2(1.f, 0.f);
    if (a >= 0 && a < axes) {
      const double turns = static_cast<double>(positions[a * tokens + t0 + token]) * inv_freq[j] * 0.15915494309189534;  // 1 / 2 pi
      sincospif(2.f * static_cast<float>(turns - rint(turns)), &cs.y, &cs.x);
    }
    turn[i] = cs;
  }
  __syncthreads();
  for (int first = threadIdx.x; first < units; first += ROPE_LOADS * ROPE_THREADS) {
    if (first != threadIdx.x) load(first);
#pragma unroll
    for (int k = 0; k < ROPE_LOADS; ++k) {
      const int unit = first + k * ROPE_THREADS;
      if (unit >= units) break;
      int pair, token;
      T* p = place(unit, pair, token);
      const float2* cs = turn + token * half + pair;
#pragma unroll
      for (int j = 0; j < PAIRS; ++j) {
        T& px = HALF ? x[k][0].v[j] : x[k][0].v[2 * j];
        T& py = HALF ? x[k][VECS - 1].v[j] : x[k][0].v[2 * j + 1];
        const float c = cs[j].x, s = cs[j].y * sign, a = widen(px), b = widen(py);
        narrow(a * c - b * s, px);
        narrow(a * s + b * c, py);
      }
#pragma unroll
      for (int e = 0; e < VECS; ++e) *reinterpret_cast<V*>(p + e * half) = x[k][e];
    }
  }
}

template <typename T, bool HALF>
int launch_rope_axes(void* buf, const int* positions, const double* inv_freq, const int* axis, long long tokens, int axes, int n_heads, int dim,
                     long long ld, int backward, cudaStream_t stream) {
  constexpr int N = 16 / sizeof(T);
  if (dim % (HALF ? 2 * N : N) != 0 || ld % N != 0) return FTB200_E_ALIGN;
  // As many tokens a block as give each thread its loads, but no fewer than two blocks an SM, and a table of at most 32 KB
  const int per_token = n_heads * (dim / (HALF ? 2 * N : N));
  long long per_block = (ROPE_LOADS * ROPE_THREADS + per_token - 1) / per_token;
  per_block = std::min(per_block, std::max(1LL, tokens / (2 * ftb200::sm_count())));
  per_block = std::max(1LL, std::min(per_block, 32768LL / (dim * 4)));
  const long long blocks = (tokens + per_block - 1) / per_block;
  if (blocks > 0x7fffffffLL) return FTB200_E_TOOBIG;
  ftb200::launch_after(rope_axes_kernel<T, HALF>, static_cast<unsigned>(blocks), ROPE_THREADS, per_block * dim * 4, stream, (T*)buf, positions,
                       inv_freq, axis, tokens, axes, n_heads, dim, ld, static_cast<int>(per_block), backward ? -1.f : 1.f);
  return cudaGetLastError() == cudaSuccess ? 0 : FTB200_E_CUDA;
}

}  // namespace

// documents: [batch, seq] int32; prefix: null or [batch, seq] bytes (non-zero: flagged); rows: [batch, seq] int4 (lo, hi, from, to), positions:
// [batch, seq], tiles: [batch, whole tiles of seq][8], padded: [batch], all int32 and written.  window: 0 or the number of keys, the query's
// own included, that a query sees at most backwards.  Prefix and window go with causal.
FTB200_API int ftb200_attention_spans(const int* documents, const unsigned char* prefix, void* rows, int* positions, void* tiles, int* padded,
                                      int batch, int seq, int causal, int window, cudaStream_t stream) {
  if (batch <= 0 || seq <= 0 || window < 0 || (!causal && (window > 0 || prefix != nullptr))) return FTB200_E_BADARG;
  if ((reinterpret_cast<uintptr_t>(rows) & 15) || (reinterpret_cast<uintptr_t>(tiles) & 15)) return FTB200_E_ALIGN;
  if (seq > (1 << 30)) return FTB200_E_TOOBIG;
  const int threads = std::min(SPAN_THREADS, (seq + 31) / 32 * 32);
  ftb200::launch_after(spans_kernel, static_cast<unsigned>(batch), threads, 0, stream, documents, prefix, (int4*)rows, positions, (SpanTile*)tiles,
                       padded, seq, causal, window);
  return cudaGetLastError() == cudaSuccess ? 0 : FTB200_E_CUDA;
}

// buf: [tokens, ld] bf16 or (f32) fp32, its first n_heads * dim columns are rotated in place; positions: [axes, tokens] int32, inv_freq:
// [dim / 2] fp64, axis: [dim / 2] int32.  half: pairs (j, j + dim / 2) instead of (2j, 2j + 1).
FTB200_API int ftb200_rope_axes(void* buf, const int* positions, const double* inv_freq, const int* axis, long long tokens, int axes, int n_heads,
                                int dim, long long ld, int f32, int half, int backward, cudaStream_t stream) {
  if (tokens <= 0 || axes <= 0 || n_heads <= 0 || dim <= 0 || ld < static_cast<long long>(n_heads) * dim) return FTB200_E_BADARG;
  if (reinterpret_cast<uintptr_t>(buf) & 15) return FTB200_E_ALIGN;
  if (dim > 1024 || n_heads > (1 << 20)) return FTB200_E_TOOBIG;
  if (f32)
    return half ? launch_rope_axes<float, true>(buf, positions, inv_freq, axis, tokens, axes, n_heads, dim, ld, backward, stream)
                : launch_rope_axes<float, false>(buf, positions, inv_freq, axis, tokens, axes, n_heads, dim, ld, backward, stream);
  return half ? launch_rope_axes<__nv_bfloat16, true>(buf, positions, inv_freq, axis, tokens, axes, n_heads, dim, ld, backward, stream)
              : launch_rope_axes<__nv_bfloat16, false>(buf, positions, inv_freq, axis, tokens, axes, n_heads, dim, ld, backward, stream);
}
