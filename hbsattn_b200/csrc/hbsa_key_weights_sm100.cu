// Key weights on the tensor cores (tcgen05 + TMEM + TMA), bf16 / fp16, head dimensions up to 256; see hbsa_key_weights.cu for the
// mathematics.  Up to 128 keys of one k-block stay in shared memory; rows of Q of the q-blocks that attend to them are streamed past them in
// tiles, strung together from pieces of 16 rows and more (tokens x GQA heads) that no q-block's end cuts.  The products land in
// tensor memory, and exp2(s scale log2 e - lse log2 e) is summed in registers in one of two ways:
//   keys in lanes (items of more than 64 keys)   S^T = K Q^T, tiles of 64 rows: the thread that owns the lane adds up the columns; no sum
//                  crosses threads
//   rows in lanes (up to 64 keys)                S = Q K^T, tiles of 128 rows: the thread adds to its own sum of every column, tile after tile, and
//                  at the end of the item the sums of 128 rows come together (short k-blocks would leave most lanes idle the other way:
//                  2 x 4096 tokens, 16 heads of 64, 30 % of the blocks: of 64 keys 64 us, keys in lanes 75; of 48 73 and 89; of 16 195 and 248)
// What bounds it: one exponential per pair, 16 a clock and SM, against 2 d FLOP per pair (at d = 128, 1024 clocks for 16384 pairs, and 752
// for their products).
//
// 192 threads, up to four persistent CTAs per SM, items (kv-head, k-block, sub-tile) from a work cursor:
//   warps 0-3     exponentials and sums (thread = TMEM lane)
//   warp 4        work fetch (long items first, see key_weights_order), mask scan, TMA, lse (contiguous copies: the preparation kernel has put it in the order of the tiles)
//   warp 5        TMEM allocation and the thread that issues every tcgen05.mma; two buffers of S
// An item has few tiles (four at a density of 0.1), and finding it takes as long as its exponentials: the CTAs of an SM hide that for each
// other.  One CTA per SM with sixteen exponential warps and two to four loaders that took turns left the exponential unit idle more
// than half of the time (2 x 8192, 16 heads of 128, 10 % of the blocks: 88 us).  Now 78 us, of which 14 are the way to the first sums (schedule, lse, first
// item and tile) and 5 the last CTAs; in between 64 % of the exponential unit.
#include <math.h>

#include "hbsa_key_weights.cuh"
#include "sm100_common.cuh"

namespace hbsa {

namespace {

constexpr int kKwThreads = 192, kKwEwWarps = 4, kKwLoader = 4, kKwMma = 5;
constexpr int kKwSlots = 2, kKwPieces = 8, kKwCols = 64;
constexpr int kKwList = 48;                   // pieces that the loader has found and not issued yet: 32, and the rest of a tile
constexpr int kKwNothing = -0x40000000;       // limit of a piece that is not there
constexpr size_t kKwLeastSmem = 46 * 1024;    // no more than four CTAs on an SM: a fifth would wait for tensor memory

template <int D, bool KEYS> struct Shape {
  static constexpr int kTile = KEYS ? 64 : 128;                 // rows of a streamed tile
  static constexpr int kKeys = KEYS ? 128 : 64;                 // stationary keys
  static constexpr int kStages = D == 64 && KEYS ? 3 : 2;
  // CTAs of an SM, by shared memory (64 columns: registers); four have its tensor memory
  static constexpr int kResident = D == 64 ? (KEYS ? 4 : 3) : D == 128 ? (KEYS ? 3 : 2) : 1;
  // Tiles whose lse is held.  Its Q goes when the product is done, lse is read until the warps free the next tile's buffer of S.  The product
  // that frees a stage for tile T, that of T - kStages, has waited for the buffer of T - kStages - 2: from T - kStages - 3 back lse may
  // be overwritten.
  static constexpr int kRows = 8;
  static_assert(kRows >= kStages + 3, "lse is overwritten too early");
};

struct KwItem {
  int n_tiles;                 // < 0: no more work
  int row0;                    // first key (token) in the packed tensor
  int keys;                    // keys of the item
  int head;                    // kv-head
  int pos0;                    // in-sample position of the first key
};

template <int D, bool KEYS> struct __align__(16) KwControl {
  float neg_lse[Shape<D, KEYS>::kRows][Shape<D, KEYS>::kTile];
  int limit[Shape<D, KEYS>::kRows][kKwPieces];               // last key that the piece's first token sees
  int4 list[kKwList];                         // {token, q-head, limit, offset in neg_lse / 16}
  float sums[2][kKwEwWarps][kKwCols];
  unsigned long long item_full[kKwSlots], item_done[kKwSlots], stat_full, stat_free;
  unsigned long long strm_full[Shape<D, KEYS>::kStages], strm_free[Shape<D, KEYS>::kStages], rows_full[Shape<D, KEYS>::kRows];
  unsigned long long s_full[2], s_free[2], sums_ready[2], drain;
  KwItem slot[kKwSlots];
  uint32_t tmem_base;
  int abort_flag, fill;
};

template <int D, bool KEYS> constexpr size_t kw_smem() {
  const size_t n = (size_t)Shape<D, KEYS>::kKeys * D * 2u + (size_t)Shape<D, KEYS>::kStages * Shape<D, KEYS>::kTile * D * 2u + sizeof(KwControl<D, KEYS>);
  return n < kKwLeastSmem ? kKwLeastSmem : n;
}
static_assert(kw_smem<256, true>() <= 227u * 1024u && kw_smem<256, false>() <= 227u * 1024u, "shared memory of one CTA");
// 228 KB an SM, of which every CTA leaves 1 KB to the system
static_assert(Shape<64, true>::kResident * (kw_smem<64, true>() + 1024u) <= 228u * 1024u && Shape<64, false>::kResident * (kw_smem<64, false>() + 1024u) <= 228u * 1024u &&
              Shape<128, true>::kResident * (kw_smem<128, true>() + 1024u) <= 228u * 1024u && Shape<128, false>::kResident * (kw_smem<128, false>() + 1024u) <= 228u * 1024u,
              "shared memory of an SM");
static_assert(5 * (kKwLeastSmem + 1024u) > 228u * 1024u, "tensor memory of an SM");

__device__ __forceinline__ void tma_load_4d(uint32_t dst, const CUtensorMap* map, uint32_t bar, int c0, int c1, int c2, int c3) {
  asm volatile("cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, %6}], [%2];"
               ::"r"(dst), "l"(reinterpret_cast<uint64_t>(map)), "r"(bar), "r"(c0), "r"(c1), "r"(c2), "r"(c3)
               : "memory");
}
// Contiguous copy global -> shared (16-byte aligned, a multiple of 16 bytes), completion on an mbarrier of this CTA.
__device__ __forceinline__ void bulk_load(uint32_t dst, const void* src, uint32_t bytes, uint32_t bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
               ::"r"(dst), "l"(src), "r"(bytes), "r"(bar) : "memory");
}

// One step of a sum over the lanes of v[0 .. 2 N): lanes that differ in bit N / 2 exchange halves.  After 32, 16, 8, 4, 2 v[0] and v[1] are
// columns 2 lane and 2 lane + 1.
template <int N> __device__ __forceinline__ void fold_columns(float (&v)[kKwCols], int lane) {
  const bool up = (lane & (N / 2)) != 0;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const float keep = up ? v[i + N] : v[i], give = up ? v[i] : v[i + N];
    v[i] = keep + __shfl_xor_sync(0xffffffffu, give, N / 2);
  }
}

template <int D, bool BF16, bool KEYS>
__global__ void __launch_bounds__(kKwThreads, (Shape<D, KEYS>::kResident))
key_weights_sm100_kernel(const __grid_constant__ CUtensorMap tm_k, const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ KeyWeightsParams P) {
  using namespace ptx;
  using S = Shape<D, KEYS>;
  constexpr int PANELS = D / 64, STAGES = S::kStages, ROWS = S::kRows, TILE = S::kTile;
  constexpr uint32_t STAT = (uint32_t)S::kKeys * D * 2u, STRM = (uint32_t)TILE * D * 2u;
  constexpr uint32_t STAT_PANEL = (uint32_t)S::kKeys * 128u, STRM_PANEL = (uint32_t)TILE * 128u;
  const Problem& p = P.p;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  extern __shared__ __align__(1024) uint8_t smem[];
  const uint32_t sStat = smem_u32(smem), sStrm = sStat + STAT;
  auto* const ctl = reinterpret_cast<KwControl<D, KEYS>*>(smem + STAT + STAGES * STRM);
  volatile int* const abort_flag = &ctl->abort_flag;
  const long long budget = P.wait_budget;
  const uint32_t b_item_full = smem_u32(ctl->item_full), b_item_done = smem_u32(ctl->item_done);
  const uint32_t b_stat_full = smem_u32(&ctl->stat_full), b_stat_free = smem_u32(&ctl->stat_free);
  const uint32_t b_strm_full = smem_u32(ctl->strm_full), b_strm_free = smem_u32(ctl->strm_free), b_rows_full = smem_u32(ctl->rows_full);
  const uint32_t b_s_full = smem_u32(ctl->s_full), b_s_free = smem_u32(ctl->s_free), b_sums = smem_u32(ctl->sums_ready);
  if (tid == 0) {
    for (int i = 0; i < 2; ++i) {
      mbar_init(b_item_full + 8 * i, 1);
      mbar_init(b_item_done + 8 * i, kKwEwWarps + 1);
      mbar_init(b_s_full + 8 * i, 1);
      mbar_init(b_s_free + 8 * i, kKwEwWarps);
      mbar_init(b_sums + 8 * i, kKwEwWarps);
    }
    mbar_init(b_stat_full, 1);
    mbar_init(b_stat_free, 1);
    for (int i = 0; i < STAGES; ++i) {
      mbar_init(b_strm_full + 8 * i, 1);
      mbar_init(b_strm_free + 8 * i, 1);
    }
    for (int i = 0; i < ROWS; ++i) mbar_init(b_rows_full + 8 * i, 1);
    mbar_init(smem_u32(&ctl->drain), 1);
    ctl->abort_flag = (sStat & 1023u) != 0 ? 1 : 0;
    fence_barrier_init();
  }
  if (warp == kKwMma) {
    tmem_alloc(smem_u32(&ctl->tmem_base), 2u * kKwCols);
    tmem_relinquish();
  }
  if (tid == kKwLoader * 32) {
    prefetch_tensormap(&tm_k);
    prefetch_tensormap(&tm_q);
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  asm volatile("griddepcontrol.wait;" ::: "memory");            // the schedule, lse in the log2 domain, the cleared cursor
  const uint32_t tmem = ctl->tmem_base;
  const int status = *(volatile int32_t*)&P.ws.status[0];
  const bool idle = status == HBSA_STATUS_BLOCK_COUNT_MISMATCH;  // the preparation kernel has written zeros

  if (idle) {
  } else if (warp == kKwLoader) {
    // =============================== work fetch, mask scan, TMA, lse ===============================
    bool ok = *abort_flag == 0 && P.debug_stall == 0;
    int items = 0, with_tiles = 0, tiles = 0, stage = 0;
    uint32_t stage_par = 1u;
    constexpr int TILE_SHIFT = KEYS ? 6 : 7;
    const int tt_shift = P.piece_shift - P.gp_shift, tt = 1 << tt_shift, per_tile = TILE >> P.piece_shift;     // tokens of a piece, pieces of a tile
    const int per_block = (p.qbs >> tt_shift) * P.n_head_sub;                          // pieces of a full q-block
    const int step_q = 32 / per_block, step_rem = 32 % per_block, q_first = lane / per_block, rem_first = lane % per_block;
    int4* const list = ctl->list;
    while (ok) {
      unsigned idx = 0;
      if (lane == 0) idx = (unsigned)atomicAdd(P.sp.cursor, 1ull);
      idx = __shfl_sync(0xffffffffu, idx, 0);
      const bool last = idx >= (unsigned)P.total_items;
      // item = (kv-head, k-block, sub-tile)
      int n_tiles = -1, hk = 0, kb = 0, k_begin = 0, q_begin = 0, q_len = 0, off = 0, k0 = 0, keys = 0, i_min = 0, qb0 = 0, nqb = 0;
      uint32_t words = 0u;                                 // lane w: which of the q-blocks i_min + 32 w .. + 31 attend
      auto active = [&](int i) -> bool {
        if (i >= nqb) return false;
        if (p.csr_ptr != nullptr) {
          const long long row = (long long)hk * p.num_q_block + qb0 + i;
          const int e1 = p.csr_ptr[row + 1];
          const int e = lower_bound_i32(p.csr_idx, p.csr_ptr[row], e1, kb);
          return e < e1 && p.csr_idx[e] == kb;
        }
        return p.mask[hk * p.mask_s0 + (long long)(qb0 + i) * p.mask_s1 + (long long)kb * p.mask_s2] != 0;
      };
      // pieces of q-block i: token pieces [first, end) x head sub-tiles
      auto sub_range = [&](int i, int& first, int& end) {
        const int rows = min(p.qbs, q_len - i * p.qbs);
        end = (rows + tt - 1) >> tt_shift;
        first = 0;
        if (p.causal) {                                    // a piece counts when its last token reaches key k0
          const int t = k0 - off - i * p.qbs;              // first in-block token that does
          first = t <= 0 ? 0 : t >= rows ? end : t >> tt_shift;
        }
      };
      if (!last) {
        const unsigned rest = P.n_msub == 1 ? idx : idx / (unsigned)P.n_msub;
        const int msub = (int)(idx - rest * (unsigned)P.n_msub);
        if (P.sorted) {
          const unsigned at = rest / (unsigned)p.nhead_k;
          hk = (int)(rest - at * (unsigned)p.nhead_k);
          kb = P.sp.order[at];
        } else {
          hk = (int)(rest / (unsigned)p.num_k_block);
          kb = (int)(rest - (unsigned)hk * (unsigned)p.num_k_block);
        }
        const int b = sample_of_block(P.ws.cnk, p.batch, kb);
        k_begin = p.cu_k[b];
        q_begin = p.cu_q[b];
        const int k_len = p.cu_k[b + 1] - k_begin, blk0 = (kb - P.ws.cnk[b]) * p.kbs;
        q_len = p.cu_q[b + 1] - q_begin;
        off = k_len - q_len;
        k0 = blk0 + msub * P.m_rows;
        keys = min(P.m_rows, min(blk0 + p.kbs, k_len) - k0);
        if (keys <= 0) continue;
        qb0 = P.ws.cnq[b];
        nqb = P.ws.cnq[b + 1] - qb0;
        if (p.causal) {                                    // first q-block whose last row reaches key k0: (i + 1) * qbs - 1 + off >= k0
          const int need = k0 - off + 1 - p.qbs;
          i_min = need > 0 ? min((need + p.qbs - 1) / p.qbs, nqb - 1) : 0;
        }
        int n = 0;
        for (int base = i_min, w = 0; base < nqb; base += 128, w += 4) {       // four loads in flight
          bool on[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) on[e] = active(base + 32 * e + lane);
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const uint32_t bal = __ballot_sync(0xffffffffu, on[e]);
            if (lane == w + e) words = bal;
            int first, end;
            if (on[e]) {
              sub_range(base + 32 * e + lane, first, end);
              n += end - first;
            }
          }
        }
#pragma unroll
        for (int d = 16; d > 0; d >>= 1) n += __shfl_xor_sync(0xffffffffu, n, d);
        n_tiles = (n * P.n_head_sub + per_tile - 1) >> (TILE_SHIFT - P.piece_shift);
        if (n_tiles == 0) {
          for (int j = lane; j < keys; j += 32)
            if (key_is_there(P, k_begin + k0 + j)) P.out[(long long)(k_begin + k0 + j) * p.nhead_k + hk] = 0.f;
          continue;
        }
      }

      if (items >= kKwSlots) ok = warp_wait(bar_of(b_item_done, items), par_of(items - kKwSlots), abort_flag, budget);
      if (!ok) break;
      if (lane == 0) {
        volatile KwItem* sl = &ctl->slot[items & (kKwSlots - 1)];
        sl->n_tiles = n_tiles; sl->row0 = k_begin + k0; sl->keys = keys; sl->head = hk; sl->pos0 = k0;
        mbar_arrive(bar_of(b_item_full, items));
      }
      ++items;
      if (last) break;
      if (with_tiles > 0) ok = warp_wait(b_stat_free, (uint32_t)(with_tiles - 1) & 1u, abort_flag, budget);
      if (!ok) break;
      if (lane == 0) {
        mbar_arrive_expect_tx(b_stat_full, (uint32_t)P.n_cols * D * 2u);
#pragma unroll
        for (int pn = 0; pn < PANELS; ++pn) tma_load_3d(sStat + pn * STAT_PANEL, &tm_k, b_stat_full, pn * 64, hk, k_begin + k0);
      }
      ++with_tiles;

      // The pieces of the q-blocks from i_min on, 32 at a time: lane -> piece `rem` of q-block i_min + q.  Those of active blocks that
      // reach the keys go to the list, from where full tiles go to the ring.
      int np = 0;                                            // pieces in the list
      int q = q_first, rem = rem_first;
      const int blocks = nqb - i_min;
      auto issue = [&](int at, int n) {
        const uint32_t bar = b_strm_full + 8u * stage, dst = sStrm + (uint32_t)stage * STRM;
        const int slot = tiles & (ROWS - 1);
        const uint32_t rows = b_rows_full + 8u * slot;
        if (tiles >= STAGES) ok = quick_wait(b_strm_free + 8u * stage, stage_par, abort_flag, budget);
        if (!ok) return;
        int4 x = make_int4(0, 0, kKwNothing, 0);
        if (lane < n) x = list[at + lane];
        if (lane < per_tile) ctl->limit[slot][lane] = x.z;
        __syncwarp();
        if (lane == 0) {
          mbar_arrive_expect_tx(bar, (uint32_t)(n << P.piece_shift) * 128u * PANELS);
          mbar_arrive_expect_tx(rows, (uint32_t)(n << P.piece_shift) * 4u);
        }
        __syncwarp();
        if (lane < n) {
          const uint32_t to = dst + ((uint32_t)lane << (P.piece_shift + 7));
          if (P.one_box) {
            tma_load_4d(to, &tm_q, bar, 0, x.y, x.x, 0);
          } else {
#pragma unroll
            for (int pn = 0; pn < PANELS; ++pn) tma_load_4d(to + pn * STRM_PANEL, &tm_q, bar, pn * 64, x.y, x.x, 0);
          }
          bulk_load(smem_u32(&ctl->neg_lse[slot][lane << P.piece_shift]), P.sp.neg_lse + (long long)x.w * 16, 4u << P.piece_shift, rows);
        }
        ++tiles;
        if (++stage == STAGES) {
          stage = 0;
          stage_par ^= 1u;
        }
      };
      for (int first_q = 0; first_q < blocks && ok; first_q = __shfl_sync(0xffffffffu, q, 0)) {
        bool on = q < blocks;
        const uint32_t word = __shfl_sync(0xffffffffu, words, (q >> 5) & 31);
        if (on) on = (q >> 5) < 32 ? (word >> (q & 31) & 1u) != 0u : active(i_min + q);
        const int i = i_min + q, s = P.n_head_sub == 1 ? rem : rem / P.n_head_sub, hs = P.n_head_sub == 1 ? 0 : rem - s * P.n_head_sub;
        if (on) {
          int first, end;
          sub_range(i, first, end);
          on = s >= first && s < end;
        }
        const uint32_t bal = __ballot_sync(0xffffffffu, on);
        if (on) {
          const int t0 = s << tt_shift;
          list[np + __popc(bal & ((1u << lane) - 1u))] =
              make_int4(q_begin + i * p.qbs + t0, hk * p.group + hs * P.gp, p.causal ? i * p.qbs + t0 + off : 0x7fffffff - 4096,
                        (int)(((((long long)(hk * P.n_head_sub + hs) * p.num_q_block + qb0 + i) * p.qbs + t0) * P.gp) >> 4));
        }
        np += __popc(bal);
        q += step_q;
        rem += step_rem;
        if (rem >= per_block) {
          rem -= per_block;
          ++q;
        }
        __syncwarp();
        int at = 0;
        for (; np - at >= per_tile && ok; at += per_tile) issue(at, per_tile);
        const int left = np - at;                            // fewer than 8
        int4 x = make_int4(0, 0, 0, 0);
        if (lane < left) x = list[at + lane];
        __syncwarp();
        if (lane < left) list[lane] = x;
        __syncwarp();
        np = left;
      }
      if (np > 0 && ok) issue(0, np);
      __syncwarp();
    }
    // copies still in flight land before the CTA leaves (bounded)
    for (int back = 1; back <= STAGES && tiles - back >= 0; ++back) {
      const int c = tiles - back;
      mbar_wait_clock(b_strm_full + 8u * (uint32_t)(c % STAGES), (uint32_t)(c / STAGES) & 1u, budget >> 4);
      mbar_wait_clock(b_rows_full + 8u * (uint32_t)(c % ROWS), (uint32_t)(c / ROWS) & 1u, budget >> 4);
    }
    if (with_tiles > 0) mbar_wait_clock(b_stat_full, (uint32_t)(with_tiles - 1) & 1u, budget >> 4);
  } else if (warp == kKwMma) {
    // =============================== MMA issuer ===============================
    if (lane == 0 && *abort_flag == 0) {
      const uint32_t idesc = make_idesc(BF16, false, false, 128, KEYS ? TILE : P.n_cols), desc_hi = smem_desc_hi(1024u);
      constexpr uint32_t PANEL_A = (KEYS ? STAT_PANEL : STRM_PANEL) >> 4, PANEL_B = (KEYS ? STRM_PANEL : STAT_PANEL) >> 4;
      bool ok = true;
      int I = 0, T = 0, stage = 0;
      uint32_t par = 0u;
      while (ok) {
        if (!(ok = mbar_wait_bounded(bar_of(b_item_full, I), par_of(I), abort_flag, budget))) break;
        const int n = *(volatile int*)&ctl->slot[I & (kKwSlots - 1)].n_tiles;
        mbar_arrive(bar_of(b_item_done, I));
        if (n < 0) break;
        if (!(ok = mbar_wait_bounded(b_stat_full, (uint32_t)I & 1u, abort_flag, budget))) break;
        for (int t = 0; t < n; ++t, ++T) {
          if (!(ok = mbar_wait_bounded(b_strm_full + 8u * stage, par, abort_flag, budget))) break;
          if (T >= 2 && !(ok = mbar_wait_bounded(bar_of(b_s_free, T), par_of(T - 2), abort_flag, budget))) break;
          tc_fence_after();
          const uint32_t lq = smem_desc_lo(sStrm + (uint32_t)stage * STRM, 16u), lk = smem_desc_lo(sStat, 16u);
          const uint32_t la = KEYS ? lk : lq, lb = KEYS ? lq : lk;
          const uint32_t tS = tmem + (uint32_t)((T & 1) * kKwCols);
#pragma unroll
          for (int ks = 0; ks < D / 16; ++ks) {
            const uint64_t da = smem_desc_join(la + (uint32_t)(ks >> 2) * PANEL_A + (uint32_t)(ks & 3) * 2u, desc_hi);
            const uint64_t db = smem_desc_join(lb + (uint32_t)(ks >> 2) * PANEL_B + (uint32_t)(ks & 3) * 2u, desc_hi);
            if (ks == 0) mma_ss_c<false>(tS, da, db, idesc);
            else mma_ss_c<true>(tS, da, db, idesc);
          }
          tc_commit(bar_of(b_s_full, T));
          tc_commit(b_strm_free + 8u * stage);
          if (t == n - 1) tc_commit(b_stat_free);
          if (++stage == STAGES) {
            stage = 0;
            par ^= 1u;
          }
        }
        ++I;
      }
      tc_commit(smem_u32(&ctl->drain));             // whatever was issued completes before tensor memory is given back
      mbar_wait_clock(smem_u32(&ctl->drain), 0u, budget);
    }
    __syncwarp();
  } else {
    // =============================== exponentials and sums ===============================
    const int row = tid;                             // TMEM lane
    const uint32_t lane_off = (uint32_t)(warp * 32) << 16;
    const uint64_t scale2 = pack_f32x2(P.scale_log2, P.scale_log2);
    const int n_cols = KEYS ? TILE : P.n_cols;
    const int pc = row >> P.piece_shift, in_piece = (row & (P.piece - 1)) >> P.gp_shift;       // rows in lanes
    int I = 0, T = 0;
    bool ok = *abort_flag == 0;
    while (ok) {
      ok = quick_wait(bar_of(b_item_full, I), par_of(I), abort_flag, budget);
      if (!ok) break;
      volatile KwItem* sl = &ctl->slot[I & (kKwSlots - 1)];
      const int n_tiles = sl->n_tiles;
      if (n_tiles < 0) break;
      const int row0 = sl->row0, keys = sl->keys, head = sl->head, pos0 = sl->pos0;
      uint64_t acc[KEYS ? 1 : kKwCols / 2];          // rows in lanes: 64 columns, two a word
#pragma unroll
      for (int j = 0; j < (KEYS ? 1 : kKwCols / 2); ++j) acc[j] = 0ull;
      float total = 0.f;                             // keys in lanes
      const int key = pos0 + row;
      for (int t = 0; t < n_tiles; ++t, ++T) {
        const int slot = T & (ROWS - 1);
        ok = quick_wait(bar_of(b_s_full, T), par_of(T), abort_flag, budget) && quick_wait(b_rows_full + 8u * slot, (uint32_t)(T / ROWS) & 1u, abort_flag, budget);
        if (!ok) break;
        tc_fence_after();
        const uint32_t tS = tmem + (uint32_t)((T & 1) * kKwCols) + lane_off;
        if (KEYS) {
          const float4* nl4 = reinterpret_cast<const float4*>(ctl->neg_lse[slot]);
          const int per_tile = TILE >> P.piece_shift;
          // rows that add nothing, pieces with rows before a key, pieces that are not there
          const float2 nl_mine = reinterpret_cast<const float2*>(ctl->neg_lse[slot])[lane];
          bool edge = fminf(nl_mine.x, nl_mine.y) == -INFINITY;
          if (lane < per_tile) edge |= *(volatile int*)&ctl->limit[slot][lane] < pos0 + keys - 1;
          edge = __any_sync(0xffffffffu, edge);
          uint64_t sum[4] = {0ull, 0ull, 0ull, 0ull};
          uint32_t r[2][32];
          tmem_ld32(tS, r[0]);
          tmem_ld32(tS + 32, r[1]);
          tmem_wait_ld();
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(bar_of(b_s_free, T));         // lse is held on
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            if (!edge) {
#pragma unroll
              for (int i = 0; i < 32; i += 4) {
                const float4 nl = nl4[(32 * h + i) >> 2];
                float x0, x1, x2, x3;
                unpack_f32x2(fma_f32x2(pack_b32x2(r[h][i], r[h][i + 1]), scale2, pack_f32x2(nl.x, nl.y)), x0, x1);
                unpack_f32x2(fma_f32x2(pack_b32x2(r[h][i + 2], r[h][i + 3]), scale2, pack_f32x2(nl.z, nl.w)), x2, x3);
                sum[(i >> 1) & 3] = add_f32x2(sum[(i >> 1) & 3], pack_f32x2(ex2_approx(x0), ex2_approx(x1)));
                sum[((i >> 1) + 1) & 3] = add_f32x2(sum[((i >> 1) + 1) & 3], pack_f32x2(ex2_approx(x2), ex2_approx(x3)));
              }
            } else {
#pragma unroll
              for (int g = 0; g < 32; g += 16) {     // no piece's end in there
                const int at = 32 * h + g, lim = *(volatile int*)&ctl->limit[slot][at >> P.piece_shift];
                // columns below `lo` hold rows before the key
                const int lo = key > lim ? (min(key - lim, 256) << P.gp_shift) - (at & (P.piece - 1)) : 0;
                if (__all_sync(0xffffffffu, lo >= 16)) continue;
#pragma unroll
                for (int i = g; i < g + 16; i += 4) {
                  const float4 nl = nl4[(32 * h + i) >> 2];
                  float x0, x1, x2, x3;
                  unpack_f32x2(fma_f32x2(pack_b32x2(r[h][i], r[h][i + 1]), scale2, pack_f32x2(nl.x, nl.y)), x0, x1);
                  unpack_f32x2(fma_f32x2(pack_b32x2(r[h][i + 2], r[h][i + 3]), scale2, pack_f32x2(nl.z, nl.w)), x2, x3);
                  if (i - g < lo || nl.x == -INFINITY) x0 = -INFINITY;         // selected, not multiplied: what is masked may be NaN
                  if (i - g + 1 < lo || nl.y == -INFINITY) x1 = -INFINITY;
                  if (i - g + 2 < lo || nl.z == -INFINITY) x2 = -INFINITY;
                  if (i - g + 3 < lo || nl.w == -INFINITY) x3 = -INFINITY;
                  sum[(i >> 1) & 3] = add_f32x2(sum[(i >> 1) & 3], pack_f32x2(ex2_approx(x0), ex2_approx(x1)));
                  sum[((i >> 1) + 1) & 3] = add_f32x2(sum[((i >> 1) + 1) & 3], pack_f32x2(ex2_approx(x2), ex2_approx(x3)));
                }
              }
            }
          }
          float a, c;
          unpack_f32x2(add_f32x2(add_f32x2(sum[0], sum[1]), add_f32x2(sum[2], sum[3])), a, c);
          total += a + c;
        } else {
          const float nl = *(volatile float*)&ctl->neg_lse[slot][row];
          int hi_col = -1;                           // last column that this row sees
          if (nl != -INFINITY) hi_col = min(*(volatile int*)&ctl->limit[slot][pc] + in_piece - pos0, keys - 1);
          const bool edge = __any_sync(0xffffffffu, hi_col < keys - 1);
          const uint64_t nl2 = pack_f32x2(nl, nl);
#pragma unroll
          for (int h = 0; h < kKwCols; h += 16) {
            if (h < n_cols) {
              uint32_t r[16];
              tmem_ld16(tS + h, r);
              tmem_wait_ld();
              auto add = [&](int i, bool masked) {
                float x0, x1;
                unpack_f32x2(fma_f32x2(pack_b32x2(r[i], r[i + 1]), scale2, nl2), x0, x1);
                if (masked) {                        // selected, not multiplied: what is masked may be NaN
                  if (h + i > hi_col) x0 = -INFINITY;
                  if (h + i + 1 > hi_col) x1 = -INFINITY;
                }
                uint64_t& to = acc[KEYS ? 0 : (h + i) >> 1];
                to = add_f32x2(to, pack_f32x2(ex2_approx(x0), ex2_approx(x1)));
              };
              if (edge) {
#pragma unroll
                for (int i = 0; i < 16; i += 2) add(i, true);
              } else {
#pragma unroll
                for (int i = 0; i < 16; i += 2) add(i, false);
              }
            }
          }
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(bar_of(b_s_free, T));
        }
      }
      if (!ok) break;
      if (KEYS) {
        if (row < keys && key_is_there(P, row0 + row)) P.out[(long long)(row0 + row) * p.nhead_k + head] = total;
      } else {
        // the sums of the warp's 32 rows, then those of the four warps (the slots see to it that the sums of the item before the last
        // one have been read)
        float v[kKwCols];
#pragma unroll
        for (int j = 0; j < kKwCols / 2; ++j) unpack_f32x2(acc[KEYS ? 0 : j], v[2 * j], v[2 * j + 1]);
        fold_columns<32>(v, lane);
        fold_columns<16>(v, lane);
        fold_columns<8>(v, lane);
        fold_columns<4>(v, lane);
        fold_columns<2>(v, lane);
        *reinterpret_cast<float2*>(&ctl->sums[I & 1][warp][2 * lane]) = make_float2(v[0], v[1]);
        __syncwarp();
        if (lane == 0) mbar_arrive(bar_of(b_sums, I));
        if (warp == 0) {
          ok = quick_wait(bar_of(b_sums, I), par_of(I), abort_flag, budget);
          if (!ok) break;
          float2 sum = make_float2(0.f, 0.f);
#pragma unroll
          for (int w = 0; w < kKwEwWarps; ++w) {
            sum.x += *(volatile float*)&ctl->sums[I & 1][w][2 * lane];
            sum.y += *(volatile float*)&ctl->sums[I & 1][w][2 * lane + 1];
          }
          float* const out = P.out + (long long)(row0 + 2 * lane) * p.nhead_k + head;
          if (2 * lane < keys && key_is_there(P, row0 + 2 * lane)) out[0] = sum.x;
          if (2 * lane + 1 < keys && key_is_there(P, row0 + 2 * lane + 1)) out[p.nhead_k] = sum.y;
        }
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(bar_of(b_item_done, I));
      ++I;
    }
  }

  // ---- teardown: every thread gets here (all waits are bounded)
  tc_fence_before();
  __syncthreads();
  if (warp == kKwMma) {
    tc_fence_after();
    tmem_dealloc(tmem, 2u * kKwCols);
  }
  if (tid == 0) {
    if (ctl->abort_flag) {
      atomicExch(&P.ws.status[0], HBSA_STATUS_WAIT_LIMIT);
      P.ws.status[3] = (int)blockIdx.x;
    }
    __threadfence();
    const bool last = atomicAdd(P.sp.cursor + 1, 1ull) == gridDim.x - 1ull;
    ctl->fill = last && *(volatile int32_t*)&P.ws.status[0] == HBSA_STATUS_WAIT_LIMIT;
  }
  __syncthreads();
  // a launch that gave up: nobody shall take its sums for weights
  if (ctl->fill)
    for (long long i = tid; i < (long long)P.total_k * p.nhead_k; i += kKwThreads) P.out[i] = NAN;
}

template <int D, bool BF16, bool KEYS>
cudaError_t launch_one(const CUtensorMap& tk, const CUtensorMap& tq, const KeyWeightsParams& P, cudaStream_t stream) {
  static SmemOptIn opt_in;
  cudaError_t e = opt_in.once(reinterpret_cast<const void*>(key_weights_sm100_kernel<D, BF16, KEYS>), (int)kw_smem<D, KEYS>());
  if (e != cudaSuccess) return e;
  const long long resident = (long long)Shape<D, KEYS>::kResident * sm100_sm_count();
  cudaLaunchAttribute attr[1] = {};
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(P.total_items < resident ? P.total_items : resident));
  cfg.blockDim = dim3(kKwThreads);
  cfg.dynamicSmemBytes = kw_smem<D, KEYS>();
  cfg.stream = stream;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, key_weights_sm100_kernel<D, BF16, KEYS>, tk, tq, P);
}

// 4-D map over [tokens, heads, headdim]: dims (columns, heads, tokens, panels), box (64, gp, piece / gp, panels).  One copy brings all panels of a
// piece where the piece is the whole tile (the panels of a tile are 128 rows apart) and the columns are whole panels.
bool encode_rows_map(EncodeTiledFn fn, CUtensorMap* map, bool bf16, const hbsa_forward_args& a, const KeyWeightsParams& P) {
  const int panels = P.one_box ? P.p.headdim / 64 : 1, d_tile = P.p.headdim <= 64 ? 64 : P.p.headdim <= 128 ? 128 : 256;
  cuuint64_t dims[4] = {(cuuint64_t)(P.one_box ? 64 : P.p.headdim), (cuuint64_t)P.p.nhead_q, (cuuint64_t)a.total_q, (cuuint64_t)panels};
  cuuint64_t strides[3] = {(cuuint64_t)a.q_stride[1] * 2ull, (cuuint64_t)a.q_stride[0] * 2ull, 128ull};
  cuuint32_t box[4] = {64u, (cuuint32_t)P.gp, (cuuint32_t)(P.piece / P.gp), P.one_box ? (cuuint32_t)(d_tile / 64) : 1u}, estr[4] = {1u, 1u, 1u, 1u};
  return fn(map, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 4, const_cast<void*>(a.q), dims, strides, box, estr,
            CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

}  // namespace

int launch_key_weights_sm100(KeyWeightsParams& P, const hbsa_forward_args& a, cudaStream_t stream, const char** err_text) {
  EncodeTiledFn fn = sm100_encode_fn();
  if (!fn) { *err_text = "cuTensorMapEncodeTiled is not available from the CUDA driver"; return HBSA_ERR_DRIVER; }
  const Problem& p = P.p;
  const bool bf16 = a.dtype == HBSA_DTYPE_BF16;
  P.n_msub = (p.kbs + 127) / 128;
  P.m_rows = ((p.kbs + P.n_msub - 1) / P.n_msub + 15) / 16 * 16;
  P.n_cols = P.m_rows;
  const bool keys = P.n_cols > 64;
  const int tile = keys ? 64 : 128;
  P.piece = 16;                                      // rows: the largest power of two up to a tile that divides those of a q-block
  P.piece_shift = 4;
  while (P.piece < P.gp || (P.piece < tile && (int64_t)p.qbs * P.gp % (2 * P.piece) == 0)) {
    P.piece *= 2;
    ++P.piece_shift;
  }
  P.n_head_sub = p.group / P.gp;
  P.one_box = P.piece == tile && p.headdim % 64 == 0;
  P.total_items = (long long)p.nhead_k * p.num_k_block * P.n_msub;
  if (P.total_items > INT32_MAX) { *err_text = "more than 2^31 (kv-head, k-block) pairs"; return HBSA_ERR_SHAPE; }
  CUtensorMap tk, tq;
  if (!sm100_encode_map(fn, &tk, bf16, a.k, p.headdim, p.nhead_k, a.total_k, a.k_stride[0], a.k_stride[1], 1, P.n_cols) ||
      !encode_rows_map(fn, &tq, bf16, a, P)) {
    *err_text = "cuTensorMapEncodeTiled rejected a q/k layout";
    return HBSA_ERR_UNSUPPORTED;
  }
  cudaError_t e;
#define HBSA_LAUNCH_KW(D_, BF_) (keys ? launch_one<D_, BF_, true>(tk, tq, P, stream) : launch_one<D_, BF_, false>(tk, tq, P, stream))
  if (p.headdim <= 64) e = bf16 ? HBSA_LAUNCH_KW(64, true) : HBSA_LAUNCH_KW(64, false);
  else if (p.headdim <= 128) e = bf16 ? HBSA_LAUNCH_KW(128, true) : HBSA_LAUNCH_KW(128, false);
  else e = bf16 ? HBSA_LAUNCH_KW(256, true) : HBSA_LAUNCH_KW(256, false);
#undef HBSA_LAUNCH_KW
  if (e != cudaSuccess) { *err_text = cudaGetErrorString(e); return (int)e; }
  return 0;
}

}  // namespace hbsa
