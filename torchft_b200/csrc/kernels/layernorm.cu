// Layer norm, forward and backward, of rows in bf16 or fp32 whose length is a multiple of 8.
//
//   forward    h = x (+ res, rounded to the type: the sum that later passes read), mean = sum h / D, rstd = 1 / sqrt(sum (h - mean)^2 / D + eps)
//              out = (h - mean) rstd w (+ b)
//   backward   xh = (x - mean) rstd, g = dy w:  dx = rstd (g - sum g / D - xh sum(g xh) / D) (+ dres),  dw = sum_rows dy xh,  db = sum_rows dy
//
// Rows are worked on by groups of threads, each thread with VPT vectors of 8 elements that stay in registers, in the rows' own type,
// between the reductions and the second use; all sums are fp32, the variance is that of centred values (no difference of squares).
#include <algorithm>
#include <type_traits>

#include "ftb200_common.cuh"
#include "tcgen05_helpers.cuh"

namespace {

struct alignas(16) f32x8 {
  float4 v[2];
};
template <typename T>
struct Row;  // 8 elements of a row, as they lie in memory
template <>
struct Row<__nv_bfloat16> {
  using V = ftb200::bf16x8;
};
template <>
struct Row<float> {
  using V = f32x8;
};
using ftb200::bf16x8;
using ftb200::unpack8;
__device__ __forceinline__ void unpack8(const f32x8& p, float* f) {
  f[0] = p.v[0].x, f[1] = p.v[0].y, f[2] = p.v[0].z, f[3] = p.v[0].w;
  f[4] = p.v[1].x, f[5] = p.v[1].y, f[6] = p.v[1].z, f[7] = p.v[1].w;
}
__device__ __forceinline__ void store8(const float* f, bf16x8* dst) { *dst = ftb200::pack8(f); }
__device__ __forceinline__ void store8(const float* f, f32x8* dst) {
  dst->v[0] = make_float4(f[0], f[1], f[2], f[3]);
  dst->v[1] = make_float4(f[4], f[5], f[6], f[7]);
}

// Sums over a group of TPR threads, N of them at a time.  `part` holds N floats per warp; who comes here again before the other warps of
// its group can have left takes another set.
template <int TPR, int N>
__device__ __forceinline__ void group_sums(float (&v)[N], float* part) {
#pragma unroll
  for (int n = 0; n < N; ++n) v[n] = ftb200::warp_sum(v[n]);
  if constexpr (TPR > 32) {
    const int g = threadIdx.x / TPR;
    if ((threadIdx.x & 31) == 0) {
#pragma unroll
      for (int n = 0; n < N; ++n) part[(threadIdx.x >> 5) * N + n] = v[n];
    }
    asm volatile("bar.sync %0, %1;" ::"r"(g + 1), "n"(TPR) : "memory");
#pragma unroll
    for (int n = 0; n < N; ++n) v[n] = 0.f;
#pragma unroll
    for (int k = 0; k < TPR / 32; ++k) {
#pragma unroll
      for (int n = 0; n < N; ++n) v[n] += part[(g * (TPR / 32) + k) * N + n];
    }
  }
}

constexpr int FWD_THREADS = 256;

// Every vector is read once and all of a thread's loads are in flight together, but the variance waits for the mean.  Bound by memory: 8192 x 4096
// with a residual 42.9 us (6.3 TB/s), 8192 x 2048 23.3, 2400 x 1024 4.4, 64 x 1024 2.2; in fp32 8192 x 4096 81.5 (6.6 TB/s).
template <typename T, int TPR, int VPT>
__global__ void __launch_bounds__(TPR > FWD_THREADS ? TPR : FWD_THREADS)
layernorm_fwd_kernel(const typename Row<T>::V* x, const typename Row<T>::V* res, typename Row<T>::V* h_out, const typename Row<T>::V* w,
                     const typename Row<T>::V* b, typename Row<T>::V* out, float* mean_out, float* rstd_out, long long rows, int D8, float eps) {
  ftb200::wait_for_previous();
  ftb200::start_next();
  using V = typename Row<T>::V;
  constexpr int THREADS = TPR > FWD_THREADS ? TPR : FWD_THREADS;
  __shared__ float part[2][THREADS / 32];
  const long long row = static_cast<long long>(blockIdx.x) * (THREADS / TPR) + threadIdx.x / TPR;
  if (row >= rows) return;  // a whole group
  const int i0 = threadIdx.x % TPR;
  V a[VPT], c[VPT];
#pragma unroll
  for (int v = 0; v < VPT; ++v) {
    const int i = i0 + v * TPR;
    if (i < D8) {
      a[v] = x[row * D8 + i];
      if (res != nullptr) c[v] = res[row * D8 + i];
    }
  }
  float sum[1] = {0.f};
#pragma unroll
  for (int v = 0; v < VPT; ++v) {
    const int i = i0 + v * TPR;
    if (i < D8) {
      float f[8];
      unpack8(a[v], f);
      if (res != nullptr) {
        float g[8];
        unpack8(c[v], g);
#pragma unroll
        for (int e = 0; e < 8; ++e) f[e] += g[e];
        store8(f, &a[v]);
        h_out[row * D8 + i] = a[v];
        unpack8(a[v], f);  // the rounded value that later passes will read
      }
      c[v] = w[i];  // on its way during the reductions
#pragma unroll
      for (int e = 0; e < 8; ++e) sum[0] += f[e];
    }
  }
  group_sums<TPR>(sum, part[0]);
  const float inv_d = 1.f / (8.f * D8);
  const float mean = sum[0] * inv_d;
  float sq[1] = {0.f};
#pragma unroll
  for (int v = 0; v < VPT; ++v) {
    if (i0 + v * TPR < D8) {
      float f[8];
      unpack8(a[v], f);
#pragma unroll
      for (int e = 0; e < 8; ++e) sq[0] = fmaf(f[e] - mean, f[e] - mean, sq[0]);
    }
  }
  group_sums<TPR>(sq, part[1]);
  const float rstd = rsqrtf(fmaf(sq[0], inv_d, eps));
  if (i0 == 0) {
    mean_out[row] = mean;
    rstd_out[row] = rstd;
  }
#pragma unroll
  for (int v = 0; v < VPT; ++v) {
    const int i = i0 + v * TPR;
    if (i < D8) {
      float f[8], g[8], s[8];
      unpack8(a[v], f);
      unpack8(c[v], g);
      if (b != nullptr) unpack8(b[i], s);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float y = (f[e] - mean) * rstd;
        f[e] = b != nullptr ? fmaf(y, g[e], s[e]) : y * g[e];
      }
      store8(f, &out[row * D8 + i]);
    }
  }
}

constexpr int BWD_THREADS = 512;
constexpr int MAX_STAGES = 8;
constexpr int RING_BYTES = 196608;  // of shared memory, for rows on their way

// A group keeps its columns over all its rows, so dw and db accumulate in registers; the groups of a block meet in shared memory at the
// end and leave one row of partial sums each of dw and db.  One block per SM.  The rows that a group will work on next (dy, x, dres) are on their
// way into a ring of its own, as many as there is room for (bulk copies; 2048 elements of bf16: 4 groups x 4 rows x 12 KB).  With a row's
// loads in registers there was room for one: 8192 x 2048 34.7 us (29.5 now, both kernels, 4.5 TB/s), 8192 x 4096 65.7 (48.1, 5.6 TB/s).
template <typename T, int TPR, int VPT>
__global__ void __launch_bounds__(BWD_THREADS, 1)
layernorm_bwd_kernel(const typename Row<T>::V* dy, const typename Row<T>::V* x, const typename Row<T>::V* w, const float* mean, const float* rstd,
                     const typename Row<T>::V* dres, typename Row<T>::V* dx, float* partial, long long rows, int D8, int stages, int* status) {
  using namespace ftb200::tc;
  using V = typename Row<T>::V;
  constexpr int GROUPS = BWD_THREADS / TPR;
  extern __shared__ __align__(128) uint8_t ring[];  // [group][stage][dy, x, dres][D8]
  __shared__ float part[2][BWD_THREADS / 32 * 2];
  __shared__ float4 meet[BWD_THREADS][2];
  __shared__ uint64_t bars[GROUPS * MAX_STAGES];
  __shared__ volatile int abort_flag;
  const int g = threadIdx.x / TPR, i0 = threadIdx.x % TPR;
  const int n_in = dres != nullptr ? 3 : 2;
  const uint32_t row_bytes = D8 * static_cast<uint32_t>(sizeof(V));
  uint8_t* mine = ring + g * stages * n_in * row_bytes;
  const uint32_t bar = smem_u32(bars + g * MAX_STAGES);
  if (threadIdx.x < GROUPS * MAX_STAGES) mbar_init(smem_u32(bars + threadIdx.x), 1);
  if (threadIdx.x == 0) abort_flag = 0;
  fence_async_smem();
  __syncthreads();
  ftb200::wait_for_previous();
  ftb200::start_next();
  const long long first = blockIdx.x + static_cast<long long>(gridDim.x) * g, step = static_cast<long long>(gridDim.x) * GROUPS;
  auto fetch = [&](long long row, int s) {  // by the group's first thread
    const uint32_t to = smem_u32(mine + s * n_in * row_bytes);
    mbar_expect_tx(bar + 8 * s, n_in * row_bytes);
    bulk_load(to, dy + row * D8, row_bytes, bar + 8 * s);
    bulk_load(to + row_bytes, x + row * D8, row_bytes, bar + 8 * s);
    if (n_in == 3) bulk_load(to + 2 * row_bytes, dres + row * D8, row_bytes, bar + 8 * s);
  };
  if (i0 == 0)
    for (int s = 0; s < stages && first + s * step < rows; ++s) fetch(first + s * step, s);
  float acc[2][VPT][8];  // dw, db
#pragma unroll
  for (int v = 0; v < VPT; ++v)
#pragma unroll
    for (int e = 0; e < 8; ++e) acc[0][v][e] = acc[1][v][e] = 0.f;
  const float inv_d = 1.f / (8.f * D8);
  V wv[VPT];
  auto weights = [&] {
#pragma unroll
    for (int v = 0; v < VPT; ++v)
      if (i0 + v * TPR < D8) wv[v] = w[i0 + v * TPR];
  };
  if constexpr (VPT <= 2) weights();
  int turn = 0, s = 0;
  uint32_t phase = 0;
  float m = 0.f, r = 0.f;
  if (first < rows) m = mean[first], r = rstd[first];
  for (long long row = first; row < rows; row += step) {
    mbar_wait(bar + 8 * s, phase, &abort_flag);  // should it run out, the group goes on together: the status word tells
    V a[VPT], b[VPT], d[VPT];
    const V* from = reinterpret_cast<const V*>(mine + s * n_in * row_bytes);
#pragma unroll
    for (int v = 0; v < VPT; ++v) {
      const int i = i0 + v * TPR;
      if (i < D8) {
        a[v] = from[i];
        b[v] = from[D8 + i];
        if (dres != nullptr) d[v] = from[2 * D8 + i];
      }
    }
    float m_next = 0.f, r_next = 0.f;
    if (row + step < rows) m_next = mean[row + step], r_next = rstd[row + step];
    if constexpr (VPT > 2) weights();
    float sums[2] = {0.f, 0.f};  // of g and of g xh
#pragma unroll
    for (int v = 0; v < VPT; ++v) {
      if (i0 + v * TPR < D8) {
        float fa[8], fb[8], c[8];
        unpack8(a[v], fa);
        unpack8(b[v], fb);
        unpack8(wv[v], c);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float xh = (fb[e] - m) * r, t = fa[e] * c[e];
          sums[0] += t;
          sums[1] = fmaf(t, xh, sums[1]);
          acc[0][v][e] = fmaf(fa[e], xh, acc[0][v][e]);
          acc[1][v][e] += fa[e];
        }
      }
    }
    group_sums<TPR>(sums, part[turn]);
    turn ^= 1;
    if constexpr (TPR == 32) __syncwarp();
    // the group has read the stage
    if (i0 == 0 && row + stages * step < rows) fetch(row + stages * step, s);
    if (++s == stages) {
      s = 0;
      phase ^= 1u;
    }
    const float c0 = sums[0] * inv_d, c1 = sums[1] * inv_d;
    if constexpr (VPT > 2) weights();  // no registers to keep them in
#pragma unroll
    for (int v = 0; v < VPT; ++v) {
      const int i = i0 + v * TPR;
      if (i < D8) {
        float fa[8], fb[8], c[8], o[8];
        unpack8(a[v], fa);
        unpack8(b[v], fb);
        unpack8(wv[v], c);
#pragma unroll
        for (int e = 0; e < 8; ++e) o[e] = r * (fmaf(fa[e], c[e], -c0) - (fb[e] - m) * r * c1);
        if (dres != nullptr) {
          float fd[8];
          unpack8(d[v], fd);
#pragma unroll
          for (int e = 0; e < 8; ++e) o[e] += fd[e];
        }
        store8(o, &dx[row * D8 + i]);
      }
    }
    m = m_next, r = r_next;
  }
  __syncthreads();
  if (abort_flag) {
    if (threadIdx.x == 0 && status != nullptr) atomicExch(status, FTB200_ST_TIMEOUT);
    const uint64_t t0 = ftb200::globaltimer_ns();  // copies in flight land in this block's shared memory
    while (ftb200::globaltimer_ns() - t0 < 200000ull) __nanosleep(1000);
  }
#pragma unroll
  for (int which = 0; which < 2; ++which) {
    float4* dst = reinterpret_cast<float4*>(partial) + (static_cast<long long>(which) * gridDim.x + blockIdx.x) * (2 * D8);
#pragma unroll
    for (int v = 0; v < VPT; ++v) {
      if (which + v > 0) __syncthreads();
      const float* s = acc[which][v];
      meet[threadIdx.x][0] = make_float4(s[0], s[1], s[2], s[3]);
      meet[threadIdx.x][1] = make_float4(s[4], s[5], s[6], s[7]);
      __syncthreads();
      for (int c = threadIdx.x; c < 2 * TPR; c += BWD_THREADS) {  // four columns of the group's 8 TPR
        if (v * 2 * TPR + c >= 2 * D8) break;
        float4 t = meet[c >> 1][c & 1];
#pragma unroll
        for (int k = 1; k < GROUPS; ++k) {
          const float4 z = meet[k * TPR + (c >> 1)][c & 1];
          t.x += z.x, t.y += z.y, t.z += z.z, t.w += z.w;
        }
        dst[v * 2 * TPR + c] = t;
      }
    }
  }
}

// dw[c], db[c] (+)= the blocks' partial sums, in their order.  A block owns 32 columns of one of the two.
template <typename T>
__global__ void __launch_bounds__(1024) layernorm_columns_kernel(const float* partial, T* dw, T* db, int blocks, int D, int accumulate) {
  ftb200::wait_for_previous();
  ftb200::start_next();
  __shared__ float red[32][33];
  const int cx = threadIdx.x & 31, ry = threadIdx.x >> 5;
  const int strips = (D + 31) / 32;
  const int which = static_cast<int>(blockIdx.x) / strips;
  const int c = (static_cast<int>(blockIdx.x) - which * strips) * 32;
  const float* src = partial + static_cast<long long>(which) * blocks * D;
  float s = 0.f;
  if (c + cx < D) {
#pragma unroll 5
    for (int b = ry; b < blocks; b += 32) s += src[static_cast<long long>(b) * D + c + cx];
  }
  red[ry][cx] = s;
  __syncthreads();
  const float t = ftb200::warp_sum(red[cx][ry]);  // warp ry: column ry of the strip
  T* dst = which == 0 ? dw : db;
  if (cx == 0 && c + ry < D) {
    const float before = accumulate ? static_cast<float>(dst[c + ry]) : 0.f;
    dst[c + ry] = static_cast<T>(t + before);
  }
}

// Threads per row and vectors per thread.  Forward: 2 vectors a thread, and 4 for more than 4 M elements of bf16 in rows of more than 2048.  With 4
// instead of 2: 64 x 1024 in bf16 2.9 us instead of 2.2, 2400 x 1024 5.1 (4.4), 600 x 4096 5.3 (4.9), 1200 x 4096 8.8 (8.8), 8192 x 4096 43.1
// (44.9); in fp32 2400 x 1024 12.2 (9.2), 8192 x 4096 85.5 (81.4), 2400 x 8192 56.4 (54.7).
template <bool FOUR, typename F>
int fwd_shape(int D8, bool four, F&& f) {
  auto is = [&](auto tpr, auto vpt) { return f(tpr, vpt); };
#define FTB200_SHAPE(T, V) is(std::integral_constant<int, T>(), std::integral_constant<int, V>())
  if (D8 <= 32) return FTB200_SHAPE(32, 1);
  if (D8 <= 64) return FTB200_SHAPE(32, 2);
  if (D8 <= 128) return FTB200_SHAPE(64, 2);
  if (D8 <= 256) return FTB200_SHAPE(128, 2);
  if constexpr (FOUR) {
    if (D8 <= 512 && four) return FTB200_SHAPE(128, 4);
    if (D8 <= 1024 && four) return FTB200_SHAPE(256, 4);
  }
  if (D8 <= 512) return FTB200_SHAPE(256, 2);
  if (D8 <= 1024) return FTB200_SHAPE(512, 2);
  if (D8 <= 2048) return FTB200_SHAPE(512, 4);
  return FTB200_E_TOOBIG;
}

// Backward: at most 2 vectors a thread up to 8192 elements, for whose two sums there are registers.  (With 4 vectors and half the
// threads 8192 x 2048 in bf16 takes 50 us instead of 30, with one and twice the threads 35.)
template <typename F>
int bwd_shape(int D8, F&& f) {
  auto is = [&](auto tpr, auto vpt) { return f(tpr, vpt); };
  if (D8 <= 32) return FTB200_SHAPE(32, 1);
  if (D8 <= 64) return FTB200_SHAPE(32, 2);
  if (D8 <= 128) return FTB200_SHAPE(64, 2);
  if (D8 <= 256) return FTB200_SHAPE(128, 2);
  if (D8 <= 512) return FTB200_SHAPE(256, 2);
  if (D8 <= 1024) return FTB200_SHAPE(512, 2);
  if (D8 <= 2048) return FTB200_SHAPE(512, 4);
#undef FTB200_SHAPE
  return FTB200_E_TOOBIG;
}

template <typename T>
int layernorm_fwd(const void* x, const void* res, void* h_out, const void* w, const void* b, void* out, float* mean, float* rstd, long long rows,
                  int D, float eps, cudaStream_t stream) {
  using V = typename Row<T>::V;
  const int D8 = D / 8;
  return fwd_shape<sizeof(T) == 2>(D8, rows * D8 > (1 << 19), [&](auto tpr, auto vpt) -> int {
    constexpr int TPR = decltype(tpr)::value, VPT = decltype(vpt)::value, THREADS = TPR > FWD_THREADS ? TPR : FWD_THREADS;
    const long long blocks = (rows + THREADS / TPR - 1) / (THREADS / TPR);
    if (blocks > 0x7fffffffLL) return FTB200_E_TOOBIG;
    ftb200::launch_after(layernorm_fwd_kernel<T, TPR, VPT>, static_cast<unsigned>(blocks), THREADS, 0, stream, (const V*)x, (const V*)res,
                         (V*)h_out, (const V*)w, (const V*)b, (V*)out, mean, rstd, rows, D8, eps);
    return cudaGetLastError() == cudaSuccess ? 0 : FTB200_E_CUDA;
  });
}

int bwd_blocks(long long rows) { return static_cast<int>(std::min<long long>((rows + 3) / 4, ftb200::sm_count())); }

template <typename T>
int layernorm_bwd(const void* dy, const void* x, const void* w, const float* mean, const float* rstd, const void* dres, void* dx, void* dw, void* db,
                  float* partial, long long rows, int D, int accumulate, int* status, cudaStream_t stream) {
  using V = typename Row<T>::V;
  const int D8 = D / 8;
  return bwd_shape(D8, [&](auto tpr, auto vpt) -> int {
    constexpr int TPR = decltype(tpr)::value, VPT = decltype(vpt)::value;
    const int blocks = bwd_blocks(rows);
    const int row_bytes = (dres == nullptr ? 2 : 3) * D * static_cast<int>(sizeof(T)) * (BWD_THREADS / TPR);
    const int stages = std::max(1, std::min(MAX_STAGES, RING_BYTES / row_bytes));
    static std::atomic<unsigned long long> ready{0};  // per device
    if (!ftb200::once_per_device(ready)) {
      if (cudaFuncSetAttribute(layernorm_bwd_kernel<T, TPR, VPT>, cudaFuncAttributeMaxDynamicSharedMemorySize, RING_BYTES) != cudaSuccess)
        return FTB200_E_CUDA;
      ftb200::done_on_device(ready);
    }
    ftb200::launch_after(layernorm_bwd_kernel<T, TPR, VPT>, blocks, BWD_THREADS, stages * row_bytes, stream, (const V*)dy, (const V*)x,
                         (const V*)w, mean, rstd, (const V*)dres, (V*)dx, partial, rows, D8, stages, status);
    ftb200::launch_after(layernorm_columns_kernel<T>, (D + 31) / 32 * (db == nullptr ? 1 : 2), 1024, 0, stream, (const float*)partial, (T*)dw,
                         (T*)db, blocks, D, accumulate);
    return cudaGetLastError() == cudaSuccess ? 0 : FTB200_E_CUDA;
  });
}

bool misaligned(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) != 0; }

}  // namespace

// x, res (may be null), h_out (with res), out: [rows, D]; w, b (may be null): [D]; bf16, or fp32 with `f32`.  mean, rstd: [rows] fp32.
FTB200_API int ftb200_layernorm_fwd(const void* x, const void* res, void* h_out, const void* w, const void* b, void* out, float* mean, float* rstd,
                                    long long rows, int D, float eps, int f32, cudaStream_t stream) {
  if (rows <= 0 || D <= 0 || D % 8 != 0 || (res != nullptr && h_out == nullptr)) return FTB200_E_BADARG;
  for (const void* p : {x, res, (const void*)h_out, w, b, (const void*)out})
    if (misaligned(p)) return FTB200_E_ALIGN;
  return f32 ? layernorm_fwd<float>(x, res, h_out, w, b, out, mean, rstd, rows, D, eps, stream)
             : layernorm_fwd<__nv_bfloat16>(x, res, h_out, w, b, out, mean, rstd, rows, D, eps, stream);
}

// Floats of the partial sums that the backward pass of rows of D elements leaves between its two kernels.
FTB200_API long long ftb200_layernorm_bwd_scratch_floats(int D) { return 2LL * ftb200::sm_count() * D; }

// dy, x (the h of the forward pass), dres (may be null), dx: [rows, D]; w, dw, db (may be null): [D].  dx may be dy, x or dres.
FTB200_API int ftb200_layernorm_bwd(const void* dy, const void* x, const void* w, const float* mean, const float* rstd, const void* dres, void* dx,
                                    void* dw, void* db, float* partial, long long rows, int D, int accumulate, int f32, int* status,
                                    cudaStream_t stream) {
  if (rows <= 0 || D <= 0 || D % 8 != 0) return FTB200_E_BADARG;
  for (const void* p : {dy, x, w, dres, (const void*)dx, (const void*)partial})
    if (misaligned(p)) return FTB200_E_ALIGN;
  return f32 ? layernorm_bwd<float>(dy, x, w, mean, rstd, dres, dx, dw, db, partial, rows, D, accumulate, status, stream)
             : layernorm_bwd<__nv_bfloat16>(dy, x, w, mean, rstd, dres, dx, dw, db, partial, rows, D, accumulate, status, stream);
}
