// Masks and score changes of the attention kernels.
//
// What a query sees is one range of keys [lo, hi), and who sees a key one range of queries [from, to) (packed_rows.cu: documents, prefixes,
// windows, padding).  A tile of 128 queries then has one range of key blocks to look at, a block that each of its queries sees needs no
// mask, and in any other the seen keys of a row are a run of bits.
//
// A score s (the product of query and key) becomes
//
//   y = log2(e) (softcap tanh(scale s / softcap) - slope |query - key|)
//
// tanh(x) is x P(x^2), of degree 3 up to |x| = 0.4 (a relative error of 9.8e-8) and of degree 5 up to 0.8 (5.8e-8; least largest error, by
// Lawson's iteration of weighted least squares): five or seven operations of the FMA pipe, with scale and cap inside the coefficients, while the
// exponential unit, which the softmax wants for itself, stays free.  A warp's scores that go beyond take 1 - 2 / (exp(2x) + 1), with an error
// of about 1e-7 of the cap, which is what counts in a score.
//
// From a cap of about 260 on (head dim 128; of 380 at 64) the last coefficients, the smaller the higher the power of the cap that they are
// divided by, are no normal numbers any more.  There the short form is taken as far as those that it lost would not be seen, and beyond it scores are
// scaled first and each takes the form that its own size asks for: 1e-7 of such a cap would be seen in a small score that shares a warp with a
// large one.  (Scores of a few units under a cap of 1000 take a tenth more time than under one of 50, both passes of 1 x 8192, 32/8 heads of 128.)
#pragma once

#include <float.h>
#include <limits.h>
#include <math.h>

#include "ftb200_common.cuh"
#include "tcgen05_helpers.cuh"

namespace ftb200 {

// Bits [a, b) of a word; a and b may lie outside of it.
__device__ __forceinline__ uint32_t range_bits(int a, int b) {
  const uint32_t below_b = b <= 0 ? 0u : b >= 32 ? 0xffffffffu : (1u << b) - 1u;
  const uint32_t below_a = a <= 0 ? 0u : a >= 32 ? 0xffffffffu : (1u << a) - 1u;
  return below_b & ~below_a;
}

struct KeyRange {
  int lo, hi;
};

// A key's queries [lo, hi), and the queries [all_lo, all_hi) that see every key of its tile.
struct RowMask {
  int lo, hi, all_lo, all_hi;
  __device__ __forceinline__ bool all(int first, int n) const { return all_lo <= first && first + n <= all_hi; }
};

struct MaskParams {
  const int4* rows;  // null, or [batch][seq]: lo, hi, from, to
  const int4* tiles;  // [batch][tiles of 128][2]: (lo, hi, all_lo, all_hi), (from, to, all_from, all_to)
  const int* padded;  // [batch][blocks of 1024]: whether there is padding
  int causal;         // without rows
  int capped;
  const float* slopes;  // null, or [heads]
  float scale_log2;     // log2(e) scale
  float near[4], poly[6];  // of s^2: y = s P(s^2)
  float near_up_to, poly_up_to;  // |s| that they hold for
  int wide;              // a cap beyond that: poly are of scale s / softcap, and hold up to wide_up_to
  float unit, wide_up_to;
  float cap2;           // log2(e) softcap
  float in2;            // 2 log2(e) scale / softcap
  float neg_inv_cap2_sq;  // -1 / cap2^2: 1 - tanh^2 = 1 + y^2 times this (zero for caps that no product of sense reaches, from 6e18 on)

  __device__ __forceinline__ int4 tile(int b, int t, int seq, int which) const {
    return tiles[(static_cast<long long>(b) * ((seq + 127) / 128) + t) * 2 + which];
  }

  // Keys that the `n` tiles of 128 queries from q0 on look at.  (Here and in queries_of the ends are held to the sequence, so that no span, whatever
  // wrote it, leads outside of it.)
  __device__ __forceinline__ KeyRange keys_of(int b, int q0, int n, int seq) const {
    if (rows == nullptr) return {0, causal ? min(seq, q0 + n * 128) : seq};
    KeyRange r = {INT_MAX, 0};
    for (int t = 0; t < n && q0 + t * 128 < seq; ++t) {
      const int4 x = tile(b, q0 / 128 + t, seq, 0);
      r.lo = min(r.lo, x.x);
      r.hi = max(r.hi, x.y);
    }
    return {max(r.lo, 0), min(r.hi, seq)};
  }

  // Keys that each of the 128 queries from q0 on sees (of those inside the sequence).
  __device__ __forceinline__ KeyRange keys_of_all(int b, int q0, int seq) const {
    if (q0 >= seq) return {INT_MAX, 0};
    if (rows == nullptr) return {0, causal ? q0 + 1 : seq};
    const int4 x = tile(b, q0 / 128, seq, 0);
    return {x.z, x.w};
  }

  // A query's keys.
  __device__ __forceinline__ KeyRange row(int b, int query, int seq) const {
    if (query >= seq) return {0, 0};
    if (rows == nullptr) return {0, causal ? query + 1 : seq};
    const int2 r = *reinterpret_cast<const int2*>(rows + static_cast<long long>(b) * seq + query);
    return {r.x, r.y};
  }

  // The other way round: the queries that the block of 128 keys looks at, and those that see a key.
  __device__ __forceinline__ KeyRange queries_of(int b, int t, int seq) const {
    if (rows == nullptr) return {causal ? t * 128 : 0, seq};
    const int4 x = tile(b, t, seq, 1);
    return {max(x.x, 0), min(x.y, seq)};
  }

  __device__ __forceinline__ RowMask column(int b, int key, int seq) const {
    RowMask m = {0, 0, INT_MAX, 0};
    if (key >= seq) return m;
    if (rows == nullptr) {
      m.lo = causal ? key : 0;
      m.hi = seq;
      if ((key | 127) < seq) {
        m.all_lo = causal ? key | 127 : 0;
        m.all_hi = seq;
      }
      return m;
    }
    const int4 r = rows[static_cast<long long>(b) * seq + key];
    const int4 x = tile(b, key / 128, seq, 1);
    return {r.z, r.w, x.z, x.w};
  }

  // By a whole warp: whether there is padding in the sequence.
  __device__ __forceinline__ bool has_padding(int b, int seq, int lane) const {
    if (rows == nullptr) return false;
    const int n = (seq + 1023) / 1024;
    int any = 0;
    for (int i = lane; i < n; i += 32) any |= padded[static_cast<long long>(b) * n + i];
    return __any_sync(0xffffffffu, any);
  }

  // Of a tile in shared memory (slabs of 128 rows x 128 bytes; its first row is row `first` of the sequence) the rows that belong to padding
  // become zeros, by one warp: what stands in padding may be anything, and zero times infinity would reach the tile's other rows.  The
  // products that follow see it.
  __device__ __forceinline__ void clear_padding(uint32_t tile_addr, int slabs, int b, int first, int seq, int lane) const {
    const int2* spans = reinterpret_cast<const int2*>(rows + static_cast<long long>(b) * seq + first + lane);
    const int rest = seq - first - lane;
    uint32_t dead = 0;  // all rows are looked up before the first store
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      int2 x = make_int2(0, 1);
      if (32 * i < rest) x = spans[2 * 32 * i];
      dead |= static_cast<uint32_t>(x.y <= x.x) << i;
    }
    for (int i = 0; dead != 0; ++i, dead >>= 1) {
      const uint32_t at = tile_addr + (lane + 32 * i) * 128;
      if (dead & 1u)
        for (int c = 0; c < slabs * 8; ++c) tc::st_shared_zero16(at + (c >> 3) * (128 * 128) + (c & 7) * 16);
    }
    tc::fence_async_smem();
    __syncwarp();
  }

  __device__ __forceinline__ float slope2(int head) const { return slopes == nullptr ? 0.f : slopes[head] * 1.4426950408889634f; }

  template <int N, int K>
  static __device__ __forceinline__ void by_polynomial(uint32_t* sv, const float* coefficients) {
    using namespace tc;
    unsigned long long k[K];
#pragma unroll
    for (int i = 0; i < K; ++i) k[i] = f2_pack(coefficients[i], coefficients[i]);
#pragma unroll
    for (int c = 0; c < N; c += 2) {
      const unsigned long long s = f2_pack(__uint_as_float(sv[c]), __uint_as_float(sv[c + 1]));
      const unsigned long long u = f2_mul(s, s);
      unsigned long long y = f2_fma(u, k[K - 1], k[K - 2]);
#pragma unroll
      for (int i = K - 3; i >= 0; --i) y = f2_fma(u, y, k[i]);
      float y0, y1;
      f2_unpack(f2_mul(s, y), y0, y1);
      sv[c] = __float_as_uint(y0);
      sv[c + 1] = __float_as_uint(y1);
    }
  }

  __device__ __forceinline__ float by_exponential(float s) const { return fmaf(-2.f * cap2, tc::rcp_approx(exp2f(s * in2) + 1.f), cap2); }

  __device__ __forceinline__ float by_scaled_polynomial(float s) const {
    const float x = s * unit, u = x * x;
    float y = poly[5];
#pragma unroll
    for (int i = 4; i >= 0; --i) y = fmaf(u, y, poly[i]);
    return y * x;
  }

  template <int N>
  static __device__ __forceinline__ float largest(const uint32_t* sv) {
    float big[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int c = 0; c < N; c += 2)
      big[(c >> 1) & 3] = fmaxf(fmaxf(big[(c >> 1) & 3], fabsf(__uint_as_float(sv[c]))), fabsf(__uint_as_float(sv[c + 1])));
    return fmaxf(fmaxf(big[0], big[1]), fmaxf(big[2], big[3]));
  }

  // N products of each thread of a warp become log2(e) softcap tanh(scale s / softcap), or log2(e) scale s without a cap.
  template <int N>
  __device__ __forceinline__ void cap_scores(uint32_t* sv) const {
    if (!capped) {
#pragma unroll
      for (int c = 0; c < N; ++c) sv[c] = __float_as_uint(__uint_as_float(sv[c]) * scale_log2);
    } else if (!wide) {
      const float most = largest<N>(sv);
      if (__all_sync(0xffffffffu, most <= near_up_to)) {
        by_polynomial<N, 4>(sv, near);
      } else if (__all_sync(0xffffffffu, most <= poly_up_to)) {
        by_polynomial<N, 6>(sv, poly);
      } else {
#pragma unroll
        for (int c = 0; c < N; ++c) sv[c] = __float_as_uint(by_exponential(__uint_as_float(sv[c])));
      }
    } else {
      // 32 at a time, each with its vote: the branches keep the work on more of them apart, for which there are no registers
#pragma unroll
      for (int a = 0; a < N; a += 32) {
        if (__all_sync(0xffffffffu, largest<32>(sv + a) <= near_up_to)) {
          by_polynomial<32, 4>(sv + a, near);
        } else {
#pragma unroll
          for (int c = a; c < a + 32; ++c) {
            const float s = __uint_as_float(sv[c]), y = by_scaled_polynomial(s), z = by_exponential(s);
            sv[c] = __float_as_uint(fabsf(s) <= wide_up_to ? y : z);
          }
        }
      }
    }
  }
};

inline int set_mask(MaskParams* m, const void* rows, const void* tiles, const int* padded, const float* slopes, float scale, float softcap, int causal,
                    int seq) {
  if ((rows != nullptr) != (tiles != nullptr) || (rows != nullptr) != (padded != nullptr) || !(softcap == 0.f || (softcap >= 1e-9f && softcap <= 1e30f)))
    return FTB200_E_BADARG;
  if ((reinterpret_cast<uintptr_t>(rows) & 15) || (reinterpret_cast<uintptr_t>(tiles) & 15)) return FTB200_E_ALIGN;
  if (seq > (1 << 30)) return FTB200_E_TOOBIG;
  constexpr double LOG2E = 1.4426950408889634;
  m->rows = static_cast<const int4*>(rows);
  m->tiles = static_cast<const int4*>(tiles);
  m->padded = padded;
  m->causal = causal;
  m->slopes = slopes;
  m->capped = softcap > 0.f;
  m->scale_log2 = static_cast<float>(scale * LOG2E);
  if (softcap > 0.f) {
    constexpr double P[6] = {0.9999999420836679, -0.333326749210523, 0.1332104829082429, -0.05311431573861419, 0.01909330062970014,
                             -0.004355299563624438};
    constexpr double NEAR[4] = {0.9999999019017232, -0.33331362461616354, 0.132709767765151, -0.04755360368917723};
    const double k = static_cast<double>(scale) / softcap, cap2 = softcap * LOG2E;
    double power = cap2 * k;
    bool finite = true;
    int normal = 0;  // coefficients, from the first on
    for (int i = 0; i < 6; ++i, power *= k * k) {
      if (i < 4) m->near[i] = static_cast<float>(NEAR[i] * power);
      m->poly[i] = static_cast<float>(P[i] * power);
      finite = finite && isfinite(m->poly[i]);
      if (normal == i && fabsf(m->poly[i]) >= FLT_MIN && (i >= 4 || fabsf(m->near[i]) >= FLT_MIN)) ++normal;
    }
    // Without its later coefficients the short form holds as far as they would add less than 2e-8; nor may a square overflow.
    const double near = normal >= 4 ? 0.4 : normal == 3 ? 0.08 : normal == 2 ? 0.015 : 1e-4;
    m->near_up_to = finite ? static_cast<float>(fmin(near / k, 1e18)) : -1.f;
    m->wide = normal < 6;
    m->poly_up_to = finite && !m->wide ? static_cast<float>(0.8 / k) : -1.f;
    if (m->wide)
      for (int i = 0; i < 6; ++i) m->poly[i] = static_cast<float>(P[i] * cap2);
    m->wide_up_to = static_cast<float>(0.8 / k);
    m->unit = static_cast<float>(k);
    m->cap2 = static_cast<float>(cap2);
    m->in2 = static_cast<float>(2.0 * LOG2E * k);
    m->neg_inv_cap2_sq = static_cast<float>(-1.0 / (cap2 * cap2));
  }
  return 0;
}

}  // namespace ftb200
