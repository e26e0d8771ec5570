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
// A block takes 1024 tokens, a thread one: scans over the block find each token's document and its prefix's end, and where the first document
// began before the block or the last one ends behind it, the block looks there itself, 4096 tokens at a time, so that no block waits for another.
// Bound by latency: 1 x 8192 tokens 5.2 us, 1 x 16384 5.5, documents of 1000 on average.  (One block a row: 68 us for 16384.)
constexpr int SPAN_THREADS = 1024;
constexpr int TILE = 128;
constexpr int NONE = INT_MAX;

struct SpanTile {  // of 128 tokens; NONE / 0 where there is nothing
  int lo, hi;            // keys that its queries see: some query sees something in [lo, hi)
  int all_lo, all_hi;    // keys that each of its queries sees; NONE, 0 with padding among them
  int from, to;          // queries that see some of its keys
  int all_from, all_to;  // queries that see each of its keys; NONE, 0 with padding among them or where the row ends inside
};

__global__ void __launch_bounds__(SPAN_THREADS) spans_kernel(const int* documents, const unsigned char* prefix, int4* rows, int* positions,
                                                             SpanTile* tiles, int* padded, int seq, int causal, int window) {
  ftb200::wait_for_previous();
  ftb200::start_next();
  __shared__ int warp_a[32], warp_b[32], warp_c[32];
  __shared__ int plain_from[SPAN_THREADS];  // the first unflagged token from each on
  __shared__ int found[3];                  // last start before the block, first start behind it, a token to look for
  __shared__ int4 tile_part[32][2];
  const int blocks = (seq + SPAN_THREADS - 1) / SPAN_THREADS;
  const int b = blockIdx.x / blocks, c0 = (blockIdx.x - b * blocks) * SPAN_THREADS, c1 = min(seq, c0 + SPAN_THREADS);
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, warps = blockDim.x >> 5;
  const int* id = documents + static_cast<long long>(b) * seq;
  const unsigned char* flag = prefix == nullptr ? nullptr : prefix + static_cast<long long>(b) * seq;
  const int i = c0 + tid;
  const bool inside = i < c1;
  const int mine = inside ? id[i] : -1;
  auto starts = [&](int k) { return k == 0 || id[k] != id[k - 1]; };
  const bool first = inside && starts(i);
  const bool plain = inside && (flag == nullptr || flag[i] == 0);

  // One walk over the tokens [from, to), in steps of 4096 from the near end: the last (back) or first token with `is`
  auto look = [&](int from, int to, bool back, int slot, int otherwise, auto is) {
    constexpr int STEP = 4;
    const int width = static_cast<int>(blockDim.x) * STEP;
    __syncthreads();
    if (tid == 0) found[slot] = back ? -1 : NONE;
    for (int n = 0; n < to - from; n += width) {
      __syncthreads();
      if (found[slot] != (back ? -1 : NONE)) break;
      int hit = back ? -1 : NONE;
#pragma unroll
      for (int k = 0; k < STEP; ++k) {
        const int d = n + k * static_cast<int>(blockDim.x) + tid;
        if (d >= to - from) break;
        const int at = back ? to - 1 - d : from + d;
        if (is(at)) hit = back ? max(hit, at) : min(hit, at);
      }
      hit = back ? __reduce_max_sync(0xffffffffu, hit) : __reduce_min_sync(0xffffffffu, hit);
      __syncthreads();
      if (lane == 0 && hit != (back ? -1 : NONE)) {
        if (back)
          atomicMax(&found[slot], hit);
        else
          atomicMin(&found[slot], hit);
      }
    }
    __syncthreads();
    const int r = found[slot];
    return r == (back ? -1 : NONE) ? otherwise : r;
  };

  // scans: the last start up to here, the first start behind, the first unflagged token from here on
  int s = first ? i : -1, e = first ? i : NONE, u = plain ? i : NONE;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int s2 = __shfl_up_sync(0xffffffffu, s, o), e2 = __shfl_down_sync(0xffffffffu, e, o), u2 = __shfl_down_sync(0xffffffffu, u, o);
    if (lane >= o) s = max(s, s2);
    if (lane + o < 32) {
      e = min(e, e2);
      u = min(u, u2);
    }
  }
  if (lane == 31) warp_a[warp] = s;
  if (lane == 0) {
    warp_b[warp] = e;
    warp_c[warp] = u;
  }
  __syncthreads();
  {  // what the warps before and behind have
    const int wa = lane < warp ? warp_a[lane] : -1;
    const int wb = lane > warp && lane < warps ? warp_b[lane] : NONE, wc = lane > warp && lane < warps ? warp_c[lane] : NONE;
    s = max(s, __reduce_max_sync(0xffffffffu, wa));
    const int eb = __reduce_min_sync(0xffffffffu, wb);
    int behind = __shfl_down_sync(0xffffffffu, e, 1);
    if (lane == 31) behind = NONE;
    e = min(behind, eb);
    u = min(u, __reduce_min_sync(0xffffffffu, wc));
  }
  plain_from[tid] = u;
  const bool open_back = __syncthreads_or(inside && s < 0);        // its first document began before
  const bool open_ahead = __syncthreads_or(i == c1 - 1 && c1 < seq);  // its last one may go on
  int before = 0, after = seq;
  if (open_back) before = look(0, c0, true, 0, 0, starts);
  if (open_ahead) after = look(c1, seq, false, 1, seq, starts);
  const int start = s >= 0 ? s : before;
  const int end = e != NONE ? e : after;
  int prefix_end = start;
  if (flag != nullptr) {
    auto unflagged = [&](int k) { return flag[k] == 0; };
    // the open first document's prefix ended before the block, or goes on in it; the last document's may go on behind it
    int ended = NONE;
    if (open_back) ended = look(before, c0, false, 2, NONE, unflagged);
    prefix_end = s >= 0 ? plain_from[s - c0] : ended != NONE ? ended : plain_from[0];
    if (__syncthreads_or(inside && prefix_end == NONE)) {
      const int ahead = look(c1, after, false, 2, after, unflagged);
      if (prefix_end == NONE) prefix_end = ahead;
    }
    prefix_end = min(prefix_end, end);
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
  const bool padding = inside && mine < 0;
  if (!inside || padding) r = make_int4(0, 0, 0, 0);
  if (inside) {
    rows[static_cast<long long>(b) * seq + i] = r;
    positions[static_cast<long long>(b) * seq + i] = i - start;
  }
  const bool any_padding = __syncthreads_or(padding);
  if (tid == 0) padded[blockIdx.x] = any_padding;

  // the tiles: four warps each
  const bool live = inside && !padding;
  int4 q, k;
  q.x = __reduce_min_sync(0xffffffffu, live ? r.x : NONE), q.y = __reduce_max_sync(0xffffffffu, r.y);
  q.z = __reduce_max_sync(0xffffffffu, padding ? NONE : r.x), q.w = __reduce_min_sync(0xffffffffu, padding ? 0 : live ? r.y : NONE);
  k.x = __reduce_min_sync(0xffffffffu, live ? r.z : NONE), k.y = __reduce_max_sync(0xffffffffu, r.w);
  k.z = __reduce_max_sync(0xffffffffu, live ? r.z : NONE), k.w = __reduce_min_sync(0xffffffffu, live ? r.w : 0);
  if (lane == 0) {
    tile_part[warp][0] = q;
    tile_part[warp][1] = k;
  }
  __syncthreads();
  const int t = tid;  // of the block's tiles
  if (t < (c1 - c0 + TILE - 1) / TILE) {
    int4 a = make_int4(NONE, 0, 0, NONE), c = a;
    for (int w = t * 4; w < t * 4 + 4; ++w) {
      const bool there = w < warps;
      const int4 x = there ? tile_part[w][0] : make_int4(NONE, 0, 0, NONE), y = there ? tile_part[w][1] : make_int4(NONE, 0, NONE, 0);
      a.x = min(a.x, x.x), a.y = max(a.y, x.y), a.z = max(a.z, x.z), a.w = min(a.w, x.w);
      c.x = min(c.x, y.x), c.y = max(c.y, y.y), c.z = max(c.z, y.z), c.w = min(c.w, y.w);
    }
    if (a.z == NONE) a.w = 0;
    if (c.z == NONE) c.w = 0;
    const long long at = static_cast<long long>(b) * ((seq + TILE - 1) / TILE) + c0 / TILE + t;
    tiles[at] = {a.x, a.y, a.z, a.w, c.x, c.y, c.z, c.w};
  }
}

// ------------------------------------------------------------------ rotary positions with several axes
// Pair j of every rotated head of token t turns by positions[axis[j]][t] * inv_freq[j], in place; an axis outside [0, axes) leaves
// it.  Pairs are neighbours (2j, 2j + 1) or, with HALF, (j, j + dim / 2).  The angle is a product in 64 bits, brought into one turn there:
// at position 2^20 32 bits are off by 0.06 rad.  Sine and cosine are those of its first 24 bits, turned on by the rest (to first order: off by
// 5e-15), so that near a zero they keep their digits; 20000 x 1 head of 256 take 16.1 us for it instead of 15.2, the other shapes the same.
//
// Bound by memory.  A block takes `per_block` tokens: each (token, pair) has its sine taken once, into shared memory, while the first
// vectors are on their way, and serves all heads.  A thread keeps its place in the head and steps over heads and tokens, without a division.
// 8192 tokens, 40 of 48 heads of 128 in bf16, three axes: 30 us (5.6 TB/s); with divisions for the places 63.
constexpr int ROPE_THREADS = 256;
constexpr int ROPE_LOADS = 4;    // vectors a thread has in flight
constexpr int ROPE_VECTORS = 8;  // a thread and block, where there are that many

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
__global__ void __launch_bounds__(ROPE_THREADS, 4) rope_axes_kernel(T* buf, const int* positions, const double* inv_freq, const int* axis,
                                                                    long long tokens, int axes, int n_heads, int dim, long long ld,
                                                                    int per_block, float sign) {
  ftb200::wait_for_previous();
  ftb200::start_next();
  using V = Vec16<T>;
  constexpr int VECS = HALF ? 2 : 1;      // vectors of a unit of work
  constexpr int PAIRS = V::N * VECS / 2;  // pairs in it
  constexpr int UNITS = ROPE_LOADS / VECS;
  extern __shared__ float2 turn[];  // [per_block][dim / 2], (cos, sin)
  const int half = dim / 2;
  const long long t0 = static_cast<long long>(blockIdx.x) * per_block;
  const int n_tokens = static_cast<int>(min(static_cast<long long>(per_block), tokens - t0));
  const int per_head = half / PAIRS;           // units of a head, at most the threads (the host checks)
  const int groups = ROPE_THREADS / per_head;  // heads that the block works on at a time
  const int group = threadIdx.x / per_head, pair = (threadIdx.x - group * per_head) * PAIRS;
  const int step_t = groups / n_heads, step_h = groups - step_t * n_heads;
  struct Place {
    int token, head;
  };
  Place at = {group / n_heads, group % n_heads};
  if (group >= groups) at.token = n_tokens;
  auto next = [&](Place& w) {
    w.token += step_t;
    w.head += step_h;
    if (w.head >= n_heads) {
      w.head -= n_heads;
      ++w.token;
    }
  };
  T* mine = buf + t0 * ld + (HALF ? pair : 2 * pair);
  auto address = [&](const Place& w) { return mine + w.token * ld + w.head * dim; };
  V x[UNITS][VECS];
  auto load = [&](Place w) {
#pragma unroll
    for (int k = 0; k < UNITS; ++k, next(w)) {
      if (w.token >= n_tokens) break;
      const T* p = address(w);
#pragma unroll
      for (int e = 0; e < VECS; ++e) *reinterpret_cast<uint4*>(&x[k][e]) = *reinterpret_cast<const uint4*>(p + e * half);
    }
  };
  load(at);
  for (int i = threadIdx.x; i < n_tokens * half; i += ROPE_THREADS) {
    const int token = i / half, j = i - token * half;
    const int a = axis[j];
    float2 cs = make_float2(1.f, 0.f);
    if (a >= 0 && a < axes) {
      const double turns = static_cast<double>(positions[a * tokens + t0 + token]) * inv_freq[j] * 0.15915494309189534;  // 1 / 2 pi
      const double halves = 2.0 * (turns - rint(turns));
      const float near = static_cast<float>(halves), rest = static_cast<float>(halves - near) * 3.14159265f;  // of 24 bits, and what they leave
      float sine, cosine;
      sincospif(near, &sine, &cosine);
      cs = make_float2(fmaf(-rest, sine, cosine), fmaf(rest, cosine, sine));
    }
    turn[i] = cs;
  }
  __syncthreads();
  while (at.token < n_tokens) {
#pragma unroll
    for (int k = 0; k < UNITS; ++k, next(at)) {
      if (at.token >= n_tokens) break;
      T* p = address(at);
      const float4* cs = reinterpret_cast<const float4*>(turn + at.token * half + pair);
#pragma unroll
      for (int j = 0; j < PAIRS; j += 2) {
        const float4 two = cs[j / 2];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          T& px = HALF ? x[k][0].v[j + e] : x[k][0].v[2 * (j + e)];
          T& py = HALF ? x[k][VECS - 1].v[j + e] : x[k][0].v[2 * (j + e) + 1];
          const float c = e == 0 ? two.x : two.z, s = (e == 0 ? two.y : two.w) * sign, a = widen(px), b = widen(py);
          narrow(a * c - b * s, px);
          narrow(a * s + b * c, py);
        }
      }
#pragma unroll
      for (int e = 0; e < VECS; ++e) *reinterpret_cast<uint4*>(p + e * half) = *reinterpret_cast<const uint4*>(&x[k][e]);
    }
    load(at);
  }
}

template <typename T, bool HALF>
int launch_rope_axes(void* buf, const int* positions, const double* inv_freq, const int* axis, long long tokens, int axes, int n_heads, int dim,
                     long long ld, int backward, cudaStream_t stream) {
  constexpr int N = 16 / sizeof(T);
  if (dim % (HALF ? 2 * N : N) != 0 || ld % N != 0) return FTB200_E_ALIGN;
  // As many tokens a block as give each thread its vectors, but no fewer than two blocks an SM, and a table of at most 32 KB
  const long long per_token = static_cast<long long>(n_heads) * (dim / N);
  long long per_block = (ROPE_VECTORS * ROPE_THREADS + per_token - 1) / per_token;
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
// [batch, seq], tiles: [batch, whole tiles of seq][8], padded: [batch, blocks of 1024 of seq] (whether there is padding), all int32 and written.  window: 0 or the number of keys, the query's
// own included, that a query sees at most backwards.  Prefix and window go with causal.
FTB200_API int ftb200_attention_spans(const int* documents, const unsigned char* prefix, void* rows, int* positions, void* tiles, int* padded,
                                      int batch, int seq, int causal, int window, cudaStream_t stream) {
  if (batch <= 0 || seq <= 0 || window < 0 || (!causal && (window > 0 || prefix != nullptr))) return FTB200_E_BADARG;
  if ((reinterpret_cast<uintptr_t>(rows) & 15) || (reinterpret_cast<uintptr_t>(tiles) & 15)) return FTB200_E_ALIGN;
  if (seq > (1 << 30)) return FTB200_E_TOOBIG;
  const int threads = std::min(SPAN_THREADS, (seq + 31) / 32 * 32);
  const long long blocks = static_cast<long long>(batch) * ((seq + SPAN_THREADS - 1) / SPAN_THREADS);
  if (blocks > 0x7fffffffLL) return FTB200_E_TOOBIG;
  ftb200::launch_after(spans_kernel, static_cast<unsigned>(blocks), threads, 0, stream, documents, prefix, (int4*)rows, positions, (SpanTile*)tiles,
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
