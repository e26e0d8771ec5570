// Grouped-query attention, forward pass, under a mask of ranges and with changed scores (attention_masks.cuh).
//
//   O[b, s, h, :] = softmax(y(Q[b, s, h, :] K[b, :, h / group, :]^T), over the keys that query s sees) V[b, :, h / group, :]
//
// head_dim 64 or 128, bf16 in/out, fp32 accumulation and statistics.  Q, K and V are read in place from a packed
// [batch * seq, n_cols] activation (any row stride).
//
// An item of work is one (batch, pair of tiles of 128 queries): two heads of a group at the same queries where the group's size is even, so that
// the tiles look at the same keys, and two query tiles of a head otherwise (for every group: 120 us instead of 108 for documents of 1000 tokens on
// average in 1 x 8192, 32/8 heads of 128; 78 instead of 65 for 400 in 4 x 2048, heads of 64).  Both walk over blocks of 128 keys, backwards: counted from
// the first key that some query of them sees, the last block first.  Where slopes lower the scores of far keys the running maximum then seldom
// rises.  Documents make items short (8 blocks where 1000 tokens are a document) and unequal, so what surrounds them counts as much
// as their loop: a CTA per SM stays and takes items one after another, in the grid's order, by cancelling CTAs that have not been launched yet
// (cluster launch control), the next one when its current item is nearly done.  The next item's Q, K and first product are under way while
// the current one's output leaves.  As a CTA of its own an item of one block took 8.6 us, of which 1.4 in the softmax.
//
//   warp 0        TMA: Q tiles of an item, K and V blocks into a ring
//   warp 1        tcgen05.mma, in the order P0 V, S0', P1 V, S1' (' = next block): the softmax of a tile has the other's products to hide
//                 under.  (A warp for each tile lets the tiles fall into step: 4480 cycles for two tiles' 128 keys instead of 3630.)
//   warp 2        the next item: launch control, the range of its keys
//   warps 4..7    softmax and output of tile 0, warps 8..11 of tile 1: one thread per query row.  (Four lanes a row in sixteen warps, two rows of
//                 32 scores a thread, are 16 % faster at head dim 64 and 7 % slower at 128.)
//
// P goes back as packed bf16 and is the A operand of P V straight from tensor memory, of its first half while the exponentials of the second are
// computed.  (A quarter of the exponentials by a polynomial instead: 65 us instead of 62 in the last case.)  At head dim 64 it has columns of its
// own, so that S of the next block runs under this one's softmax; at head dim 128 the 512 columns are full (two S, two O) and it takes the place
// of the scores that it came from.  (Scores in two buffers of 64 keys instead read Q twice as often from shared memory: 4900 cycles.)
// The running maximum is only raised (and O in TMEM rescaled) when it grows by more than 2^8.  Blocks that each query sees need no mask; in the
// others a row's seen keys are a run of bits.
//
// Sequences of any length: the tensor maps have the sequence as a dimension of its own, so a tile's rows beyond its end are zeros (not the
// next sequence's); keys there are in no query's range, queries there are not stored.
//
// 1 x 8192, 32/8 heads of 128: documents of 1000 tokens on average 113 us (655 TFLOP/s of the pairs that are seen), with a cap 145; causal with a
// cap 611 (900 TFLOP/s; 441 in the kernel without masks and caps), with slopes 503 (659 with the first block first).
//
// Every mbarrier wait is bounded; on expiry the CTA records FTB200_ST_TIMEOUT in the caller's status word, frees its TMEM and returns.
#include <cuda.h>
#include <math.h>

#include "attention_masks.cuh"
#include "ftb200_common.cuh"
#include "tcgen05_helpers.cuh"
#include "tensor_maps.cuh"

namespace {

using namespace ftb200::tc;

constexpr int BQ = 128;    // queries per tile
constexpr int TILES = 2;   // tiles per item
constexpr int BKV = 128;   // keys per block
constexpr int NUM_THREADS = 384;
// Registers: a CTA is launched with 168 a thread (65536 / 384, checked on the host); the first warpgroup gives most of its own to the two
// softmax warpgroups: 40 + 2 * 232 = 3 * 168.  With these shares nothing is kept in local memory (checked on the host too), and each role ends by
// itself, so that no value is held across a change of shares: what a role needs at its end it reads again.
constexpr int LAUNCH_REGS = 168, ISSUE_REGS = 40, SOFTMAX_REGS = 232;
static_assert(ISSUE_REGS + 2 * SOFTMAX_REGS <= 3 * LAUNCH_REGS, "more registers than the CTA is launched with");
constexpr int ROW_WARPS = 4;                  // softmax warps per tile
constexpr int READERS = 2 + TILES * ROW_WARPS;  // warps that read an item
constexpr int CLAIM_AHEAD = 3;                // blocks before its end at which an item asks for the next one
constexpr uint32_t TMEM_COLS = 512;
constexpr float RESCALE_THRESHOLD = 8.0f;  // in log2 units

template <int D>
struct Cfg {
  static constexpr uint32_t TILE_BYTES = 128 * D * 2;  // a 128-row operand tile
  static constexpr uint32_t SLAB_BYTES = 128 * 128;    // 128 rows x 64 elements (one swizzle atom wide)
  static constexpr int SLABS = D / 64;
  static constexpr int STAGES = D == 128 ? 2 : 4;  // of K and V
  static constexpr bool OWN_P = D == 64;           // P has columns of its own
  static constexpr uint32_t OFF_Q = 0;                    // Q0 Q1
  static constexpr uint32_t OFF_KV = TILES * TILE_BYTES;  // K0 V0 | K1 V1 | ...
  static constexpr uint32_t OFF_O = OFF_KV + STAGES * 2 * TILE_BYTES;  // per softmax warp: 32 rows x 64 elements on their way out
  static constexpr uint32_t OFF_MISC = OFF_O + TILES * ROW_WARPS * 4096;
  static constexpr uint32_t SMEM_BYTES = OFF_MISC + 512 + 1024;
  static_assert(SMEM_BYTES <= 232448, "exceeds the 227 KB of shared memory a CTA can have");
  static constexpr uint32_t COL_S = 0;    // S_t at COL_S + t * 128
  static constexpr uint32_t COL_O = 256;  // O_t at COL_O + t * D
  static constexpr uint32_t COL_P = OWN_P ? 384 : COL_S, P_STEP = OWN_P ? 64 : 128;  // P_t at COL_P + t * P_STEP
};

struct Params {
  int batch, seq, n_heads, n_kv_heads;
  int pair_heads;  // an item's tiles are heads h and h + 1
  float scale_log2;  // softmax scale * log2(e)
  float* lse;        // null, or [batch, n_heads, seq], natural log
  int* status;
  ftb200::MaskParams mask;
};

struct Item {
  int batch;  // below zero: there is none
  int head, query;
  int first, blocks;  // key where the first block, which is the one behind all others, begins; number of blocks
  int all_lo[TILES], all_hi[TILES];  // keys that each query of the tile sees
};

enum : int {
  BAR_Q_FULL = 0,    // +tile
  BAR_Q_EMPTY = 2,   // +tile
  BAR_K_FULL = 4,    // +stage
  BAR_K_EMPTY = 8,   // +stage
  BAR_V_FULL = 12,   // +stage
  BAR_V_EMPTY = 16,  // +stage
  BAR_S_FULL = 20,   // +tile
  BAR_S_READ = 22,   // +tile: the scores are in registers (where P has columns of its own)
  BAR_P_HALF = 24,   // +tile: P of the block's first 64 keys
  BAR_P_FULL = 26,   // +tile
  BAR_O_DONE = 28,   // +tile: P V of a block
  BAR_O_LAST = 30,   // +tile: P V of an item's last block
  BAR_O_FREE = 32,   // +tile: O has been read
  BAR_ITEM_FULL = 34,   // +slot
  BAR_ITEM_EMPTY = 36,  // +slot
  BAR_CLAIM = 38,    // the current item is nearly done
  BAR_CLAIMED = 39,  // the answer of the launch control
  NUM_BARS = 40,
};

// The grid's next CTA that has not been launched, or -1: the answer (16 bytes) arrives in shared memory with the barrier.
__device__ __forceinline__ void claim_next(uint32_t answer, uint32_t bar) {
  asm volatile("clusterlaunchcontrol.try_cancel.async.shared::cta.mbarrier::complete_tx::bytes.b128 [%0], [%1];" ::"r"(answer), "r"(bar) : "memory");
}
__device__ __forceinline__ int claimed(uint32_t answer) {
  uint32_t ok, x;
  asm volatile(
      "{\n"
      ".reg .pred p;\n"
      ".reg .b128 c;\n"
      "ld.shared.b128 c, [%2];\n"
      "clusterlaunchcontrol.query_cancel.is_canceled.pred.b128 p, c;\n"
      "selp.u32 %0, 1, 0, p;\n"
      "mov.u32 %1, 0;\n"
      "@p clusterlaunchcontrol.query_cancel.get_first_ctaid::x.b32.b128 %1, c;\n"
      "}\n"
      : "=r"(ok), "=r"(x)
      : "r"(answer)
      : "memory");
  return ok ? static_cast<int>(x) : -1;
}

template <int D, bool SCORE>
__global__ void __launch_bounds__(NUM_THREADS, 1)
attention_masked_fwd_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV,
                            const __grid_constant__ CUtensorMap tmO, const Params p) {
  using C = Cfg<D>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + C::OFF_MISC);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + C::OFF_MISC + 320);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + C::OFF_MISC + 324);
  Item* items = reinterpret_cast<Item*>(smem + C::OFF_MISC + 336);  // two slots
  static_assert(NUM_BARS * 8 <= 320 && 336 + 2 * sizeof(Item) <= 448, "barriers, slots and the answer overlap");

  const int warp = __shfl_sync(0xffffffffu, static_cast<int>(threadIdx.x >> 5), 0);
  const int lane = threadIdx.x & 31;
  const uint32_t smem_base = smem_u32(smem);
  const uint32_t bar_base = smem_u32(bars);
  const uint32_t answer = smem_base + C::OFF_MISC + 448;
  auto bar = [&](int i) { return bar_base + 8u * i; };
  auto wait = [&](int which, uint32_t parity) { return mbar_wait_warp(bar(which), parity & 1u, abort_flag); };

  const int rep = p.n_heads / p.n_kv_heads;
  const int q_step = p.pair_heads ? 0 : BQ, h_step = p.pair_heads ? 1 : 0;  // from tile 0 to tile 1

  if (threadIdx.x == 0) {
    for (int t = 0; t < TILES; ++t) {
      mbar_init(bar(BAR_Q_FULL + t), 1);
      mbar_init(bar(BAR_Q_EMPTY + t), 1);
      mbar_init(bar(BAR_S_FULL + t), 1);
      mbar_init(bar(BAR_S_READ + t), ROW_WARPS);
      mbar_init(bar(BAR_P_HALF + t), ROW_WARPS);
      mbar_init(bar(BAR_P_FULL + t), ROW_WARPS);
      mbar_init(bar(BAR_O_DONE + t), 1);
      mbar_init(bar(BAR_O_LAST + t), 1);
      mbar_init(bar(BAR_O_FREE + t), ROW_WARPS);
      mbar_init(bar(BAR_ITEM_FULL + t), 1);  // two slots
      mbar_init(bar(BAR_ITEM_EMPTY + t), READERS);
    }
    for (int s = 0; s < C::STAGES; ++s) {
      mbar_init(bar(BAR_K_FULL + s), 1);
      mbar_init(bar(BAR_K_EMPTY + s), 1);
      mbar_init(bar(BAR_V_FULL + s), 1);
      mbar_init(bar(BAR_V_EMPTY + s), 1);
    }
    mbar_init(bar(BAR_CLAIM), 1);
    mbar_init(bar(BAR_CLAIMED), 1);
    *abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    fence_async_smem();
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "r"(TMEM_COLS) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = __shfl_sync(0xffffffffu, *tmem_slot, 0);

  ftb200::wait_for_previous();

  // Item number k of this CTA, for one of the READERS: false where the CTA is aborting.
  auto read_item = [&](int k, Item& it) {
    if (!wait(BAR_ITEM_FULL + (k & 1), k >> 1)) return false;
    const Item& at = items[k & 1];
    it = at;
    mbar_arrive_warp(bar(BAR_ITEM_EMPTY + (k & 1)));
    return true;
  };
  if (warp < 4) {
    regs_dec<ISSUE_REGS>();
    if (warp == 0) {
      // ---------------- TMA producer ----------------
      bool ok = true;
      int blocks = 0, full = 0;  // stages and items with keys, so far
      for (int k = 0; ok; ++k) {
        Item it;
        if (!(ok = read_item(k, it)) || it.batch < 0) break;
        if (it.blocks == 0) continue;
        const int hk = it.head / rep;
        auto load = [&](const CUtensorMap* map, int full_bar, uint32_t dst, int col, int r) {
          if (elect_one()) {
            mbar_expect_tx(bar(full_bar), C::TILE_BYTES);
            for (int s = 0; s < C::SLABS; ++s) tma_load_3d(dst + s * C::SLAB_BYTES, map, bar(full_bar), col * D + s * 64, r, it.batch);
          }
          __syncwarp();
        };
        auto load_q = [&](int t) {
          if (!wait(BAR_Q_EMPTY + t, full ^ 1)) return false;
          load(&tmQ, BAR_Q_FULL + t, smem_base + C::OFF_Q + t * C::TILE_BYTES, it.head + t * h_step, it.query + t * q_step);
          return true;
        };
        ok = load_q(0);
        for (int j = 0; j < it.blocks && ok; ++j, ++blocks) {
          const int st = blocks % C::STAGES, use = blocks / C::STAGES;
          const uint32_t sk = smem_base + C::OFF_KV + st * 2 * C::TILE_BYTES;
          if (!(ok = wait(BAR_K_EMPTY + st, use ^ 1))) break;
          load(&tmK, BAR_K_FULL + st, sk, hk, it.first - j * BKV);
          if (j == 0 && !(ok = load_q(1))) break;
          if (!(ok = wait(BAR_V_EMPTY + st, use ^ 1))) break;
          load(&tmV, BAR_V_FULL + st, sk + C::TILE_BYTES, hk, it.first - j * BKV);
        }
        ++full;
      }
      ftb200::start_next();
      if (!ok) {
        // copies in flight land in this CTA's shared memory: give them time before the CTA exits
        const uint64_t t0 = ftb200::globaltimer_ns();
        while (ftb200::globaltimer_ns() - t0 < 200000ull) __nanosleep(1000);
      }
    } else if (warp == 1) {
      // ---------------- MMA issuer ----------------
      // S = Q K^T: both operands K-major (head dim contiguous), M = N = 128
      const uint32_t F = (1u << 4) | (1u << 7) | (1u << 10) | (static_cast<uint32_t>(BQ >> 4) << 24);
      const uint32_t idesc_s = F | (static_cast<uint32_t>(BKV >> 3) << 17);
      // O += P V: A = P from tensor memory (keys contiguous), B = V MN-major (stored [key][d]), N = D
      const uint32_t idesc_o = F | (1u << 16) | (static_cast<uint32_t>(D >> 3) << 17);
      constexpr uint32_t HI = smem_desc_hi(1024);
      const uint32_t q_lo = smem_desc_lo(smem_base + C::OFF_Q, 16);
      const uint32_t k_lo = smem_desc_lo(smem_base + C::OFF_KV, 16);
      const uint32_t v_lo = smem_desc_lo(smem_base + C::OFF_KV + C::TILE_BYTES, C::SLAB_BYTES);
      constexpr uint32_t STAGE16 = (2 * C::TILE_BYTES) >> 4, QTILE16 = C::TILE_BYTES >> 4;
      // taken from lane 0 where it is used, so that it is known to be the same in all lanes and lies in uniform registers
      auto same = [](uint32_t v) { return __shfl_sync(0xffffffffu, v, 0); };
      bool ok = true;
      int blocks = 0, full = 0;
      for (int k = 0; ok; ++k) {
        Item it;
        if (!(ok = read_item(k, it)) || it.batch < 0) break;
        if (it.blocks == 0) {
          if (elect_one()) mbar_arrive(bar(BAR_CLAIM));
          __syncwarp();
          continue;
        }
        const bool padded = p.mask.has_padding(it.batch, p.seq, lane);
        // what stands in padding reaches neither the products nor the choice of a way for the scores
        auto clear = [&](uint32_t off, int r) {
          if (padded) p.mask.clear_padding(smem_base + off, C::SLABS, it.batch, r, p.seq, lane);
        };
        auto issue_s = [&](int t, int j) {
          const int g = blocks + j, st = g % C::STAGES;
          if (t == 0) {
            if (!wait(BAR_K_FULL + st, g / C::STAGES)) return false;
            clear(C::OFF_KV + st * 2 * C::TILE_BYTES, it.first - j * BKV);
          }
          if (j == 0) {
            if (!wait(BAR_Q_FULL + t, full)) return false;
            clear(C::OFF_Q + t * C::TILE_BYTES, it.query + t * q_step);
          }
          // where P is elsewhere the scores of the block before have to be in registers
          if (C::OWN_P && g > 0 && !wait(BAR_S_READ + t, g - 1)) return false;
          tc_fence_after();
          const uint32_t kb = same(k_lo + st * STAGE16);
          if (elect_one()) {
#pragma unroll
            for (int kk = 0; kk < D / 16; ++kk) {
              const uint32_t off = ((kk >> 2) * C::SLAB_BYTES + (kk & 3) * 32) >> 4;
              umma_bf16_lh(tmem_base + C::COL_S + t * 128, q_lo + t * QTILE16 + off, HI, kb + off, HI, idesc_s, kk != 0);
            }
            umma_commit(bar(BAR_S_FULL + t));
            if (t == 1) umma_commit(bar(BAR_K_EMPTY + st));
            if (j == it.blocks - 1) umma_commit(bar(BAR_Q_EMPTY + t));
          }
          __syncwarp();
          return true;
        };
        auto issue_pv = [&](int t, int j) {
          const int g = blocks + j, st = g % C::STAGES;
          if (t == 0) {
            if (!wait(BAR_V_FULL + st, g / C::STAGES)) return false;
            clear(C::OFF_KV + st * 2 * C::TILE_BYTES + C::TILE_BYTES, it.first - j * BKV);
          }
          if (j == 0 && full > 0 && !wait(BAR_O_FREE + t, full - 1)) return false;
          const uint32_t vb = same(v_lo + st * STAGE16);
#pragma unroll (C::OWN_P ? 2 : 1)  // at head dim 128 both at once would put a word in local memory
          for (int half = 0; half < 2; ++half) {
            if (!wait((half == 0 ? BAR_P_HALF : BAR_P_FULL) + t, g)) return false;
            tc_fence_after();
            if (elect_one()) {
#pragma unroll
              for (int kk = half * 4; kk < half * 4 + 4; ++kk)  // P: keys 2k, 2k+1 in column k
                umma_bf16_tmem_a(tmem_base + C::COL_O + t * D, tmem_base + C::COL_P + t * C::P_STEP + kk * 8, vb + ((kk * 2048) >> 4), HI, idesc_o,
                                 (j | kk) != 0);
              if (half == 1) {
                umma_commit(bar(BAR_O_DONE + t));
                if (t == 1) umma_commit(bar(BAR_V_EMPTY + st));
                if (j == it.blocks - 1) umma_commit(bar(BAR_O_LAST + t));
              }
            }
            __syncwarp();
          }
          return true;
        };
        ok = issue_s(0, 0) && issue_s(1, 0);
        for (int j = 0; j < it.blocks && ok; ++j) {
          if (j == max(0, it.blocks - CLAIM_AHEAD)) {
            if (elect_one()) mbar_arrive(bar(BAR_CLAIM));
            __syncwarp();
          }
          const bool more = j + 1 < it.blocks;
          if constexpr (C::OWN_P) {
            ok = (!more || (issue_s(0, j + 1) && issue_s(1, j + 1))) && issue_pv(0, j) && issue_pv(1, j);
          } else {
            // S held P of this block: its P V was issued before and the tensor pipe runs in order
            ok = issue_pv(0, j) && (!more || issue_s(0, j + 1)) && issue_pv(1, j) && (!more || issue_s(1, j + 1));
          }
        }
        blocks += it.blocks;
        ++full;
      }
    } else if (warp == 2) {
      // ---------------- items ----------------
      const int cta_rows = p.pair_heads ? BQ : BQ * TILES, cta_heads = p.n_heads / (p.pair_heads ? TILES : 1);
      const int n_rows = (p.seq + cta_rows - 1) / cta_rows, per_row = p.batch * cta_heads;
      int next = static_cast<int>(blockIdx.x);
      for (int k = 0;; ++k) {
        Item it = {};
        it.batch = -1;
        if (next >= 0) {
          // late queries first: under a causal mask they see the most
          it.query = (n_rows - 1 - next / per_row) * cta_rows;
          const int bh = next % per_row;
          it.batch = bh / cta_heads;
          it.head = bh % cta_heads * (p.pair_heads ? TILES : 1);
          const ftb200::KeyRange r = p.mask.keys_of(it.batch, it.query, p.pair_heads ? 1 : TILES, p.seq);
          it.blocks = r.hi > r.lo ? (r.hi - r.lo + BKV - 1) / BKV : 0;
          it.first = r.lo + (it.blocks - 1) * BKV;
          for (int t = 0; t < TILES; ++t) {
            const ftb200::KeyRange a = p.mask.keys_of_all(it.batch, it.query + t * q_step, p.seq);
            it.all_lo[t] = a.lo;
            it.all_hi[t] = a.hi;
          }
        }
        if (!wait(BAR_ITEM_EMPTY + (k & 1), (k >> 1) ^ 1)) break;
        if (lane == 0) items[k & 1] = it;
        mbar_arrive_warp(bar(BAR_ITEM_FULL + (k & 1)));
        if (next < 0 || !wait(BAR_CLAIM, k)) break;
        if (elect_one()) {
          mbar_expect_tx(bar(BAR_CLAIMED), 16);
          claim_next(answer, bar(BAR_CLAIMED));
        }
        __syncwarp();
        if (!wait(BAR_CLAIMED, k)) break;
        next = claimed(answer);
        if (next >= n_rows * per_row) next = -1;
        fence_async_smem();  // read before the next answer is written
        __syncwarp();
      }
    }
    __syncwarp();
    tc_fence_before();
    __syncthreads();
    if (warp == 1) {
      tc_fence_after();
      asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(*tmem_slot), "r"(TMEM_COLS) : "memory");
    } else if (warp == 2 && lane == 0 && *abort_flag && p.status != nullptr) {
      atomicExch(p.status, FTB200_ST_TIMEOUT);
    }
  } else {
    // ---------------- softmax + output: one thread per query row ----------------
    regs_inc<SOFTMAX_REGS>();
    const int t = (warp - 4) >> 2;   // tile
    const int quarter = warp & 3;    // TMEM lane quarter this warp may touch
    const int row = quarter * 32 + lane;
    const uint32_t lane_addr = static_cast<uint32_t>(quarter * 32) << 16;
    const uint32_t s_addr = tmem_base + C::COL_S + t * 128 + lane_addr;
    const uint32_t p_addr = tmem_base + C::COL_P + t * C::P_STEP + lane_addr;
    const uint32_t o_addr = tmem_base + C::COL_O + t * D + lane_addr;
    const uint32_t off_stage = C::OFF_O + (warp - 4) * 4096;
    uint8_t* stage = smem + off_stage + lane * 128;
    // with SCORE the scores come scaled, in units of log2
    const float scale_log2 = SCORE ? 1.f : p.scale_log2;
    // The item stays in shared memory while the softmax works on it, and of the row's mask only the ends are kept: registers are scarce.
    int blocks = 0, full = 0;
    bool ok = true;
    for (int k = 0;; ++k) {
      if (!(ok = wait(BAR_ITEM_FULL + (k & 1), k >> 1))) break;
      const Item& it = items[k & 1];
      if (it.batch < 0) break;
      const int query = it.query + t * q_step + row;
      const int head = it.head + t * h_step;
      const ftb200::KeyRange mine = p.mask.row(it.batch, query, p.seq);
      float slope2 = 0.f;
      if constexpr (SCORE) slope2 = p.mask.slope2(head);
      __syncwarp();
      float m_used = -INFINITY, l_sum = 0.f;
      for (int j = 0; j < it.blocks; ++j) {
        const int g = blocks + j;
        if (!(ok = wait(BAR_S_FULL + t, g))) break;
        tc_fence_after();
        uint32_t sv[BKV];
#pragma unroll
        for (int c = 0; c < BKV / 32; ++c) tmem_ld32(s_addr + c * 32, sv + c * 32);
        tmem_wait_ld();
        if constexpr (C::OWN_P) {
          tc_fence_before();
          mbar_arrive_warp(bar(BAR_S_READ + t));
        }
        const int first = it.first - j * BKV;
        if constexpr (SCORE) {
          if (p.mask.capped) p.mask.cap_scores<BKV>(sv);
          const float unit = p.mask.capped ? 1.f : p.scale_log2;
          const float far = static_cast<float>(query - first);
          if (p.mask.slopes == nullptr) {
          } else if (first + BKV - 1 <= it.query + t * q_step) {
            // no key behind a query: the slope's part grows evenly with the key.  Four sums of a slope times eight keys each run through the block
            // (16 additions: off by 5e-7 of it)
            const unsigned long long unit2 = f2_pack(unit, unit), step = f2_pack(8.f * slope2, 8.f * slope2);
            unsigned long long part[4];
#pragma unroll
            for (int c = 0; c < 4; ++c) part[c] = f2_pack(slope2 * (2 * c - far), slope2 * (2 * c + 1 - far));
#pragma unroll
            for (int c = 0; c < BKV / 2; ++c) {
              float y0, y1;
              f2_unpack(f2_fma(f2_pack(__uint_as_float(sv[2 * c]), __uint_as_float(sv[2 * c + 1])), unit2, part[c & 3]), y0, y1);
              part[c & 3] = f2_add(part[c & 3], step);
              sv[2 * c] = __float_as_uint(y0);
              sv[2 * c + 1] = __float_as_uint(y1);
            }
          } else {
#pragma unroll
            for (int c = 0; c < BKV; ++c) sv[c] = __float_as_uint(fmaf(-slope2, fabsf(far - c), __uint_as_float(sv[c]) * unit));
          }
        }
        if (first < it.all_lo[t] || first + BKV > it.all_hi[t]) {
#pragma unroll
          for (int w = 0; w < BKV / 32; ++w) {
            const uint32_t bits = ftb200::range_bits(mine.lo - first - 32 * w, mine.hi - first - 32 * w);
#pragma unroll
            for (int c = 0; c < 32; ++c)
              if (!(bits >> c & 1u)) sv[32 * w + c] = __float_as_uint(-INFINITY);
          }
        }
        float mx4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
        for (int c = 0; c < BKV; c += 2)
          mx4[(c >> 1) & 3] = fmaxf(fmaxf(mx4[(c >> 1) & 3], __uint_as_float(sv[c])), __uint_as_float(sv[c + 1]));
        const float m_new = fmaxf(fmaxf(mx4[0], mx4[1]), fmaxf(mx4[2], mx4[3]));

        // raise the maximum only when it moved far
        float alpha = 1.f;
        const bool raise = m_used > -INFINITY && (m_new - m_used) * scale_log2 > RESCALE_THRESHOLD;
        const bool any_raise = __any_sync(0xffffffffu, raise);
        if (m_used == -INFINITY) {
          m_used = m_new;  // the row has seen nothing yet: O and the sum are zero
        } else if (raise) {
          alpha = exp2f((m_used - m_new) * scale_log2);
          m_used = m_new;
          l_sum *= alpha;
        }
        __syncwarp();  // tensor memory is accessed by whole warps
        // O, and P where it has columns of its own, may only be touched once P V of the previous block is done; P V of this block waits for P
        if ((any_raise || C::OWN_P) && g > 0) {
          if (!(ok = wait(BAR_O_DONE + t, g - 1))) break;
          tc_fence_after();
        }
        if (any_raise) {
#pragma unroll
          for (int c = 0; c < D / 32; ++c) {
            uint32_t ov[32];
            tmem_ld32(o_addr + c * 32, ov);
            tmem_wait_ld();
#pragma unroll
            for (int e = 0; e < 32; ++e) ov[e] = __float_as_uint(__uint_as_float(ov[e]) * alpha);
            tmem_st32(o_addr + c * 32, ov);
          }
        }
        // a row that has seen nothing yet has no maximum
        const float neg_m = m_used == -INFINITY ? 0.f : -m_used * scale_log2;
        const unsigned long long scale2 = f2_pack(scale_log2, scale_log2), neg_m2 = f2_pack(neg_m, neg_m);
        unsigned long long sum2[2] = {0ull, 0ull};
#pragma unroll
        for (int c = 0; c < BKV / 32; ++c) {
          uint32_t packed[16];
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            const unsigned long long x2 =
                f2_fma(f2_pack(__uint_as_float(sv[c * 32 + 2 * e]), __uint_as_float(sv[c * 32 + 2 * e + 1])), scale2, neg_m2);
            float p0, p1;
            f2_unpack(x2, p0, p1);
            p0 = exp2f(p0);
            p1 = exp2f(p1);
            sum2[e & 1] = f2_add(sum2[e & 1], f2_pack(p0, p1));
            // to bf16, as the product takes it next to V: off by up to 2^-8 of itself, where the sum, kept in fp32, has it whole
            __nv_bfloat162 pk = __floats2bfloat162_rn(p0, p1);
            packed[e] = *reinterpret_cast<uint32_t*>(&pk);
          }
          tmem_st16(p_addr + c * 16, packed);  // the scores are in registers
          if (c == 1) {
            tmem_wait_st();
            tc_fence_before();
            mbar_arrive_warp(bar(BAR_P_HALF + t));
          }
        }
        tmem_wait_st();
        tc_fence_before();
        mbar_arrive_warp(bar(BAR_P_FULL + t));
        float sum4[4];
        f2_unpack(sum2[0], sum4[0], sum4[1]);
        f2_unpack(sum2[1], sum4[2], sum4[3]);
        l_sum += (sum4[0] + sum4[1]) + (sum4[2] + sum4[3]);
      }
      if (!ok) break;
      blocks += it.blocks;

      if (it.blocks > 0) {
        if (!(ok = wait(BAR_O_LAST + t, full))) break;
        ++full;
      }
      tc_fence_after();
      const bool nothing = l_sum == 0.f;  // no key is seen: zeros, and a log-sum-exp of -infinity
      const float inv = 1.f / l_sum;
      const int first_row = it.query + t * q_step + quarter * 32;
      // O leaves by TMA, 32 rows of 64 elements at a time
#pragma unroll
      for (int s = 0; s < C::SLABS; ++s) {
        uint32_t ov[64];
        tmem_ld32(o_addr + s * 64, ov);
        tmem_ld32(o_addr + s * 64 + 32, ov + 32);
        tmem_wait_ld();
        if (s == C::SLABS - 1 && it.blocks > 0) {
          tc_fence_before();
          mbar_arrive_warp(bar(BAR_O_FREE + t));
        }
        if (lane == 0) bulk_wait_read();  // what was here has left
        __syncwarp();
#pragma unroll
        for (int c = 0; c < 8; ++c) {
          uint32_t u[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float a = nothing ? 0.f : __uint_as_float(ov[8 * c + 2 * e]) * inv, b = nothing ? 0.f : __uint_as_float(ov[8 * c + 2 * e + 1]) * inv;
            __nv_bfloat162 pk = __floats2bfloat162_rn(a, b);
            u[e] = *reinterpret_cast<uint32_t*>(&pk);
          }
          *reinterpret_cast<uint4*>(stage + ((c ^ (lane & 7)) << 4)) = make_uint4(u[0], u[1], u[2], u[3]);
        }
        fence_async_smem();
        __syncwarp();
        if (lane == 0 && first_row < p.seq) {
          tma_store_3d(&tmO, smem_base + off_stage, head * D + s * 64, first_row, it.batch);
          bulk_commit();
        }
        __syncwarp();
      }
      if (p.lse != nullptr && query < p.seq) {
        p.lse[(static_cast<long long>(it.batch) * p.n_heads + head) * p.seq + query] =
            nothing ? -INFINITY : (m_used * scale_log2 + log2f(l_sum)) * 0.6931471805599453f;
      }
      mbar_arrive_warp(bar(BAR_ITEM_EMPTY + (k & 1)));
    }
    if (lane == 0) bulk_wait_read();
    __syncwarp();
    tc_fence_before();
    __syncthreads();
  }
}

struct Maps {
  CUtensorMap q, k, v, o;
};

template <int D, bool SCORE>
int launch(const Maps& m, const Params& p, long long grid, cudaStream_t stream) {
  auto* kernel = attention_masked_fwd_kernel<D, SCORE>;
  static std::atomic<unsigned long long> ready{0};  // per device
  if (!ftb200::once_per_device(ready)) {
    if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, Cfg<D>::SMEM_BYTES) != cudaSuccess) return FTB200_E_CUDA;
    // The warpgroups' register split assumes this count, which the compiler gives a kernel that moves registers; with fewer the softmax
    // warpgroups would wait for registers that nobody has.
    cudaFuncAttributes attr;
    if (cudaFuncGetAttributes(&attr, kernel) != cudaSuccess) return FTB200_E_CUDA;
    if (attr.numRegs < LAUNCH_REGS || attr.localSizeBytes != 0) return FTB200_E_REGS;
    ftb200::done_on_device(ready);
  }
  ftb200::launch_after(kernel, static_cast<unsigned>(grid), NUM_THREADS, Cfg<D>::SMEM_BYTES, stream, m.q, m.k, m.v, m.o, p);
  return cudaGetLastError() == cudaSuccess ? 0 : FTB200_E_CUDA;
}

}  // namespace

// q: [batch*seq, n_heads*head_dim] view with row stride ld_q; k, v: [batch*seq, n_kv_heads*head_dim] views with row strides ld_k, ld_v; o:
// [batch*seq, n_heads*head_dim] with row stride ld_o.  lse (may be null): [batch, n_heads, seq] fp32.  head_dim 64 or 128, any seq.
// rows, tiles, padded: null, where every query sees the keys up to its own (causal) or all, or what ftb200_attention_spans wrote.
// softcap: 0, or what the scores are capped at, softcap tanh(scale s / softcap).  slopes: null, or [n_heads] fp32: slope |query - key| is
// subtracted from a score.
FTB200_API int ftb200_attention_masked_fwd(const void* q, const void* k, const void* v, void* o, float* lse, const void* rows, const void* tiles,
                                           const int* padded, const float* slopes, int batch, int seq, int n_heads, int n_kv_heads, int head_dim,
                                           long long ld_q, long long ld_k, long long ld_v, long long ld_o, float scale, float softcap, int causal,
                                           int* status, cudaStream_t stream) {
  if ((head_dim != 64 && head_dim != 128) || batch <= 0 || seq <= 0 || n_heads <= 0 || n_kv_heads <= 0 || n_heads % n_kv_heads != 0)
    return FTB200_E_BADARG;
  for (const void* x : {q, k, v, (const void*)o})
    if (reinterpret_cast<uintptr_t>(x) & 15) return FTB200_E_ALIGN;
  for (long long x : {ld_q, ld_k, ld_v, ld_o})
    if (x & 7) return FTB200_E_ALIGN;
  Params p = {};
  Maps m;
  int rc = ftb200::set_mask(&p.mask, rows, tiles, padded, slopes, scale, softcap, causal, seq);
  if (rc == 0) rc = ftb200::encode_rows(&m.q, q, batch, seq, static_cast<long long>(n_heads) * head_dim, ld_q);
  if (rc == 0) rc = ftb200::encode_rows(&m.k, k, batch, seq, static_cast<long long>(n_kv_heads) * head_dim, ld_k);
  if (rc == 0) rc = ftb200::encode_rows(&m.v, v, batch, seq, static_cast<long long>(n_kv_heads) * head_dim, ld_v);
  if (rc == 0) rc = ftb200::encode_rows(&m.o, o, batch, seq, static_cast<long long>(n_heads) * head_dim, ld_o, 64, 32);
  if (rc != 0) return rc;
  p.batch = batch; p.seq = seq; p.n_heads = n_heads; p.n_kv_heads = n_kv_heads;
  p.scale_log2 = scale * 1.4426950408889634f;
  p.lse = lse; p.status = status;
  p.pair_heads = n_heads / n_kv_heads % TILES == 0;
  const long long tiles_q = (static_cast<long long>(seq) + BQ - 1) / BQ;
  const long long grid = p.pair_heads ? batch * (static_cast<long long>(n_heads) / TILES) * tiles_q
                                      : static_cast<long long>(batch) * n_heads * ((tiles_q + TILES - 1) / TILES);
  if (grid > 0x7fffffffLL) return FTB200_E_TOOBIG;
  const bool score = softcap > 0.f || slopes != nullptr;
  if (head_dim == 128) return score ? launch<128, true>(m, p, grid, stream) : launch<128, false>(m, p, grid, stream);
  return score ? launch<64, true>(m, p, grid, stream) : launch<64, false>(m, p, grid, stream);
}
