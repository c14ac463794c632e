// Key weights on the tensor cores (tcgen05 + TMEM + TMA), bf16 / fp16, head dimensions up to 256; see hbsa_key_weights.cu for the
// mathematics.  Up to 128 keys of one k-block stay in shared memory; Q of the q-blocks that attend to them is streamed past them
// in tiles of up to 128 rows (tokens x GQA heads), S^T = K Q^T lands in tensor memory with one key per lane, and the
// thread that owns the lane adds up exp2(s scale log2 e - lse log2 e) over the tile's columns: no sum ever crosses threads.
//
// 320 threads, one persistent CTA per SM, items (kv-head, k-block, sub-tile) from a work cursor:
//   warps 0-3 / 4-7   the even / odd tiles (thread = TMEM lane = key)
//   warp 8            work fetch, mask scan, TMA, and the rows' lse (asynchronous copies that report to the tile's barrier)
//   warp 9            TMEM allocation and the thread that issues every tcgen05.mma; four buffers of S
#include <math.h>

#include "hbsa_key_weights.cuh"
#include "sm100_common.cuh"

namespace hbsa {

namespace {

constexpr int kKwThreads = 320, kKwEwWarps = 8, kKwProducer = 8, kKwMma = 9;
constexpr int kKwBufs = 4;

template <int D> struct Shape {
  static constexpr int kTile = D == 256 ? 64 : 128;             // rows of a streamed tile, at most
  static constexpr int kStages = D == 64 ? 6 : D == 128 ? 4 : 3;
};

struct KwItem {
  int n_tiles;                 // < 0: no more work
  int row0;                    // first key (token) in the packed tensor
  int keys;                    // keys of the item
  int head;                    // kv-head
  int pos0;                    // in-sample position of the first key
};

template <int TILE, int STAGES> struct __align__(16) KwControl {
  float neg_lse[STAGES][TILE];
  float sums[2][128];
  unsigned long long item_full[2], item_done[2], stat_full[2], stat_free[2];
  unsigned long long strm_full[STAGES], strm_free[STAGES];
  unsigned long long s_full[kKwBufs], s_free[kKwBufs];
  unsigned long long sums_ready[2], drain;
  uint32_t tmem_base;
  int abort_flag, fill;
  int limit[STAGES];           // last key that the tile's first token sees
  KwItem slot[2];
};

template <int D> constexpr size_t kw_smem() {
  return 2u * 128u * D * 2u + (size_t)Shape<D>::kStages * Shape<D>::kTile * D * 2u + sizeof(KwControl<Shape<D>::kTile, Shape<D>::kStages>);
}
static_assert(kw_smem<64>() <= 227u * 1024u && kw_smem<128>() <= 227u * 1024u && kw_smem<256>() <= 227u * 1024u, "shared memory of one CTA");

__device__ __forceinline__ void copy_async4(uint32_t dst, const void* src) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(dst), "l"(src) : "memory");
}
// One arrival (already counted) of this thread once its copies so far have landed.
__device__ __forceinline__ void copy_async_arrive(uint32_t bar) {
  asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(bar) : "memory");
}

template <int D, bool BF16>
__global__ void __launch_bounds__(kKwThreads, 1)
key_weights_sm100_kernel(const __grid_constant__ CUtensorMap tm_k, const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ KeyWeightsParams P) {
  using namespace ptx;
  constexpr int PANELS = D / 64, TILE = Shape<D>::kTile, STAGES = Shape<D>::kStages;
  constexpr uint32_t STAT = 128u * D * 2u, STRM = (uint32_t)TILE * D * 2u;
  const Problem& p = P.p;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int status = *(volatile int32_t*)&P.ws.status[0];
  if (status == HBSA_STATUS_BLOCK_COUNT_MISMATCH) return;       // the preparation kernel has written zeros

  extern __shared__ __align__(1024) uint8_t smem[];
  const uint32_t sStat = smem_u32(smem), sStrm = sStat + 2 * STAT;
  auto* const ctl = reinterpret_cast<KwControl<TILE, STAGES>*>(smem + 2 * STAT + STAGES * STRM);
  volatile int* const abort_flag = &ctl->abort_flag;
  const long long budget = P.wait_budget;
  const uint32_t b_item_full = smem_u32(ctl->item_full), b_item_done = smem_u32(ctl->item_done);
  const uint32_t b_stat_full = smem_u32(ctl->stat_full), b_stat_free = smem_u32(ctl->stat_free);
  const uint32_t b_strm_full = smem_u32(ctl->strm_full), b_strm_free = smem_u32(ctl->strm_free);
  const uint32_t b_s_full = smem_u32(ctl->s_full), b_s_free = smem_u32(ctl->s_free), b_sums = smem_u32(ctl->sums_ready);
  if (tid == 0) {
    for (int i = 0; i < 2; ++i) {
      mbar_init(b_item_full + 8 * i, 1);
      mbar_init(b_item_done + 8 * i, kKwEwWarps + 1);
      mbar_init(b_stat_full + 8 * i, 1);
      mbar_init(b_stat_free + 8 * i, 1);
      mbar_init(b_sums + 8 * i, kKwEwWarps / 2);
    }
    for (int i = 0; i < STAGES; ++i) {
      mbar_init(b_strm_full + 8 * i, 1 + 32);                    // the tile, and the lse copies of 32 lanes
      mbar_init(b_strm_free + 8 * i, 1 + kKwEwWarps / 2);        // the product, and the four warps that read lse
    }
    for (int i = 0; i < kKwBufs; ++i) {
      mbar_init(b_s_full + 8 * i, 1);
      mbar_init(b_s_free + 8 * i, kKwEwWarps / 2);
    }
    mbar_init(smem_u32(&ctl->drain), 1);
    ctl->abort_flag = (sStat & 1023u) != 0 ? 1 : 0;
    fence_barrier_init();
  }
  if (warp == kKwMma) {
    tmem_alloc(smem_u32(&ctl->tmem_base), 512u);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = ctl->tmem_base;
  const int nt = P.nt;
  const uint32_t strm_panel = (uint32_t)nt * 128u;

  if (warp == kKwProducer) {
    // =============================== work fetch, mask scan, TMA, lse ===============================
    if (lane == 0) {
      prefetch_tensormap(&tm_k);
      prefetch_tensormap(&tm_q);
    }
    int I = 0, Iq = 0, T = 0, stage = 0;
    uint32_t stage_par = 1u;
    bool ok = *abort_flag == 0 && P.debug_stall == 0;
    long long next_idx = 0;
    if (lane == 0) next_idx = (long long)atomicAdd(P.sp.cursor, 1ull);
    next_idx = __shfl_sync(0xffffffffu, next_idx, 0);

    auto publish = [&](int n_tiles, int row0, int keys, int head, int pos0) {
      if (I >= 2) ok = warp_wait(bar_of(b_item_done, I), par_of(I - 2), abort_flag, budget);
      if (!ok) return;
      if (lane == 0) {
        volatile KwItem* sl = &ctl->slot[I & 1];
        sl->n_tiles = n_tiles; sl->row0 = row0; sl->keys = keys; sl->head = head; sl->pos0 = pos0;
        __threadfence_block();
        mbar_arrive(bar_of(b_item_full, I));
      }
      ++I;
    };
    auto load_stationary = [&](int row0, int head) {
      if (Iq >= 2) ok = warp_wait(bar_of(b_stat_free, Iq), par_of(Iq - 2), abort_flag, budget);
      if (!ok) return;
      if (lane == 0) {
        const uint32_t bar = bar_of(b_stat_full, Iq), dst = sStat + (uint32_t)(Iq & 1) * STAT;
        mbar_arrive_expect_tx(bar, STAT);
#pragma unroll
        for (int pn = 0; pn < PANELS; ++pn) tma_load_3d(dst + pn * 16384u, &tm_k, bar, pn * 64, head, row0);
      }
      ++Iq;
    };
    // one tile of q rows: `valid` tokens from `tok` on are the block's
    auto load_tile = [&](int tok, int head0, int valid, int limit) {
      if (T >= STAGES) ok = warp_wait(b_strm_free + 8u * stage, stage_par, abort_flag, budget);
      if (!ok) return;
      const uint32_t bar = b_strm_full + 8u * stage, dst = sStrm + (uint32_t)stage * STRM, nl = smem_u32(ctl->neg_lse[stage]);
      for (int c = lane; c < nt; c += 32) {
        const int t = c >> P.gp_shift;
        if (t < valid) {
          copy_async4(nl + 4u * c, P.sp.neg_lse + (long long)(tok + t) * p.nhead_q + head0 + (c & (P.gp - 1)));
        } else {
          ctl->neg_lse[stage][c] = -INFINITY;
        }
      }
      if (lane == 0) {
        ctl->limit[stage] = limit;
        __threadfence_block();
        mbar_arrive_expect_tx(bar, (uint32_t)nt * D * 2u);
#pragma unroll
        for (int pn = 0; pn < PANELS; ++pn) tma_load_3d(dst + pn * strm_panel, &tm_q, bar, pn * 64, head0, tok);
      }
      __threadfence_block();
      copy_async_arrive(bar);
      ++T;
      if (++stage == STAGES) {
        stage = 0;
        stage_par ^= 1u;
      }
    };

    while (ok) {
      const long long idx = next_idx;
      if (idx >= P.total_items) {
        publish(-1, 0, 0, 0, 0);
        break;
      }
      if (lane == 0) next_idx = (long long)atomicAdd(P.sp.cursor, 1ull);
      next_idx = __shfl_sync(0xffffffffu, next_idx, 0);
      // item = (kv-head, k-block, sub-tile); under a causal mask the first k-blocks of a sample have the most work
      const int msub = (int)(idx % P.n_msub);
      const long long rest = idx / P.n_msub;
      const int kb = (int)(rest % p.num_k_block), hk = (int)(rest / p.num_k_block);
      const int b = sample_of_block(P.ws.cnk, p.batch, kb);
      const int k_begin = p.cu_k[b], k_len = p.cu_k[b + 1] - k_begin, q_begin = p.cu_q[b], q_len = p.cu_q[b + 1] - q_begin;
      const int off = k_len - q_len;
      const int blk0 = (kb - P.ws.cnk[b]) * p.kbs;
      const int k0 = blk0 + msub * P.m_rows, k_end = min(blk0 + p.kbs, k_len);
      if (k0 >= k_end) continue;
      const int qb0 = P.ws.cnq[b], nqb = P.ws.cnq[b + 1] - qb0;
      int i_min = 0;
      if (p.causal) {                             // first q-block whose last row reaches key k0: (i + 1) * qbs - 1 + off >= k0
        const int need = k0 - off + 1 - p.qbs;
        i_min = need > 0 ? min((need + p.qbs - 1) / p.qbs, nqb - 1) : 0;
      }
      // tiles of q-block i: token sub-tiles [first, last) x head sub-tiles
      auto sub_range = [&](int i, int& first, int& last) {
        const int rows = min(p.qbs, q_len - i * p.qbs);
        last = (rows + P.tt - 1) / P.tt;
        first = 0;
        if (p.causal) {                           // a sub-tile counts when its last token reaches key k0
          const int t = k0 - off - i * p.qbs;     // first in-block token that does
          first = t <= 0 ? 0 : t >= rows ? last : t / P.tt;
        }
      };
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
      int n_tiles = 0;
      for (int base = i_min; base < nqb; base += 32) {
        const int i = base + lane;
        int first, last;
        if (active(i)) {
          sub_range(i, first, last);
          n_tiles += (last - first) * P.n_head_sub;
        }
      }
#pragma unroll
      for (int d = 16; d > 0; d >>= 1) n_tiles += __shfl_xor_sync(0xffffffffu, n_tiles, d);
      publish(n_tiles, k_begin + k0, min(P.m_rows, k_end - k0), hk, k0);
      if (!ok || n_tiles == 0) continue;
      load_stationary(k_begin + k0, hk);
      for (int base = i_min; base < nqb && ok; base += 32) {
        uint32_t bal = __ballot_sync(0xffffffffu, active(base + lane));
        while (bal != 0 && ok) {
          const int i = base + __ffs(bal) - 1;
          bal &= bal - 1;
          int first, last;
          sub_range(i, first, last);
          const int rows = min(p.qbs, q_len - i * p.qbs);
          for (int s = first; s < last && ok; ++s)
            for (int hs = 0; hs < P.n_head_sub && ok; ++hs) {
              const int t0 = s * P.tt;
              load_tile(q_begin + i * p.qbs + t0, hk * p.group + hs * P.gp, min(P.tt, rows - t0), p.causal ? i * p.qbs + t0 + off : 0x7fffffff - 4096);
            }
        }
      }
    }
    // copies still in flight land before the CTA leaves (bounded)
    for (int back = 1; back <= STAGES && T - back >= 0; ++back) {
      const int c = T - back;
      mbar_wait_clock(b_strm_full + 8u * (uint32_t)(c % STAGES), (uint32_t)(c / STAGES) & 1u, budget >> 4);
    }
    for (int back = 1; back <= 2 && Iq - back >= 0; ++back) mbar_wait_clock(bar_of(b_stat_full, Iq - back), par_of(Iq - back), budget >> 4);
  } else if (warp == kKwMma) {
    // =============================== MMA issuer ===============================
    if (lane == 0 && *abort_flag == 0) {
      const uint32_t idesc = make_idesc(BF16, false, false, 128, nt), desc_hi = smem_desc_hi(1024u);
      const uint32_t panel_units = strm_panel >> 4;
      bool ok = true;
      int I = 0, Iq = 0, T = 0, stage = 0;
      uint32_t par = 0u;
      while (ok) {
        if (!(ok = mbar_wait_bounded(bar_of(b_item_full, I), par_of(I), abort_flag, budget))) break;
        const int n = *(volatile int*)&ctl->slot[I & 1].n_tiles;
        mbar_arrive(bar_of(b_item_done, I));
        ++I;
        if (n < 0) break;
        if (n == 0) continue;
        if (!(ok = mbar_wait_bounded(bar_of(b_stat_full, Iq), par_of(Iq), abort_flag, budget))) break;
        for (int t = 0; t < n; ++t, ++T) {
          const int buf = T & (kKwBufs - 1);
          if (!(ok = mbar_wait_bounded(b_strm_full + 8u * stage, par, abort_flag, budget))) break;
          if (T >= kKwBufs && !(ok = mbar_wait_bounded(b_s_free + 8u * buf, (uint32_t)(T / kKwBufs - 1) & 1u, abort_flag, budget))) break;
          tc_fence_after();
          const uint32_t la = smem_desc_lo(sStat + (uint32_t)(Iq & 1) * STAT, 16u), lx = smem_desc_lo(sStrm + (uint32_t)stage * STRM, 16u);
          const uint32_t tS = tmem + (uint32_t)(buf * TILE);
#pragma unroll
          for (int ks = 0; ks < D / 16; ++ks) {
            const uint64_t da = smem_desc_join(la + (uint32_t)(ks >> 2) * 1024u + (uint32_t)(ks & 3) * 2u, desc_hi);
            const uint64_t dx = smem_desc_join(lx + (uint32_t)(ks >> 2) * panel_units + (uint32_t)(ks & 3) * 2u, desc_hi);
            if (ks == 0) mma_ss_c<false>(tS, da, dx, idesc);
            else mma_ss_c<true>(tS, da, dx, idesc);
          }
          tc_commit(b_s_full + 8u * buf);
          tc_commit(b_strm_free + 8u * stage);
          if (t == n - 1) tc_commit(bar_of(b_stat_free, Iq));
          if (++stage == STAGES) {
            stage = 0;
            par ^= 1u;
          }
        }
        ++Iq;
      }
      tc_commit(smem_u32(&ctl->drain));             // whatever was issued completes before tensor memory is given back
      mbar_wait_clock(smem_u32(&ctl->drain), 0u, budget);
    }
    __syncwarp();
  } else {
    // =============================== exponentials and sums ===============================
    const int wg = warp >> 2, row = tid & 127;
    const uint32_t lane_off = (uint32_t)((warp & 3) * 32) << 16;
    const uint64_t scale2 = pack_f32x2(P.scale_log2, P.scale_log2);
    int I = 0, Iq = 0, T = 0, stage = 0;
    uint32_t par = 0u;
    bool ok = *abort_flag == 0;
    while (ok) {
      ok = warp_wait(bar_of(b_item_full, I), par_of(I), abort_flag, budget);
      if (!ok) break;
      volatile KwItem* sl = &ctl->slot[I & 1];
      const int n_tiles = sl->n_tiles;
      if (n_tiles < 0) break;
      const int row0 = sl->row0, keys = sl->keys, head = sl->head, key = sl->pos0 + row;
      float total = 0.f;
      for (int t = 0; t < n_tiles; ++t, ++T) {
        if ((T & 1) == wg) {
          const int buf = T & (kKwBufs - 1);
          // the tile's barrier too: it is what the lse copies have reported to
          ok = warp_wait(b_strm_full + 8u * stage, par, abort_flag, budget) && warp_wait(b_s_full + 8u * buf, (uint32_t)(T / kKwBufs) & 1u, abort_flag, budget);
          if (!ok) break;
          tc_fence_after();
          const uint32_t tS = tmem + (uint32_t)(buf * TILE) + lane_off;
          const int limit = *(volatile int*)&ctl->limit[stage];
          int lo_col = 0;                           // columns of tokens before the key take no part
          if (key > limit) lo_col = min(key - limit, TILE) << P.gp_shift;
          const float4* nl4 = reinterpret_cast<const float4*>(ctl->neg_lse[stage]);
          bool edge = lo_col > 0;                   // or some rows add nothing
          if (lane * 4 < nt) {
            const float4 nl = nl4[lane];
            edge |= fminf(fminf(nl.x, nl.y), fminf(nl.z, nl.w)) == -INFINITY;
          }
          edge = __any_sync(0xffffffffu, edge);
          uint64_t sum0 = 0ull, sum1 = 0ull;
          for (int c0 = 0; c0 < nt; c0 += 16) {
            uint32_t r[16];
            tmem_ld16(tS + c0, r);
            tmem_wait_ld();
#pragma unroll
            for (int i = 0; i < 16; i += 4) {
              const float4 nl = nl4[(c0 + i) >> 2];
              float x0, x1, x2, x3;
              unpack_f32x2(fma_f32x2(pack_b32x2(r[i], r[i + 1]), scale2, pack_f32x2(nl.x, nl.y)), x0, x1);
              unpack_f32x2(fma_f32x2(pack_b32x2(r[i + 2], r[i + 3]), scale2, pack_f32x2(nl.z, nl.w)), x2, x3);
              if (edge) {                           // selected, not multiplied: what is masked may be NaN
                if (c0 + i < lo_col || nl.x == -INFINITY) x0 = -INFINITY;
                if (c0 + i + 1 < lo_col || nl.y == -INFINITY) x1 = -INFINITY;
                if (c0 + i + 2 < lo_col || nl.z == -INFINITY) x2 = -INFINITY;
                if (c0 + i + 3 < lo_col || nl.w == -INFINITY) x3 = -INFINITY;
              }
              sum0 = add_f32x2(sum0, pack_f32x2(ex2_approx(x0), ex2_approx(x1)));
              sum1 = add_f32x2(sum1, pack_f32x2(ex2_approx(x2), ex2_approx(x3)));
            }
          }
          tc_fence_before();
          __syncwarp();
          if (lane == 0) {
            mbar_arrive(b_s_free + 8u * buf);
            mbar_arrive(b_strm_free + 8u * stage);
          }
          float a, c, d, e;
          unpack_f32x2(sum0, a, c);
          unpack_f32x2(sum1, d, e);
          total += (a + c) + (d + e);
        }
        if (++stage == STAGES) {
          stage = 0;
          par ^= 1u;
        }
      }
      if (!ok) break;
      if (n_tiles > 0) {                             // the odd tiles' sums join the even tiles'
        if (wg == 1) {
          ctl->sums[Iq & 1][row] = total;
          __syncwarp();
          if (lane == 0) mbar_arrive(bar_of(b_sums, Iq));
        } else {
          ok = warp_wait(bar_of(b_sums, Iq), par_of(Iq), abort_flag, budget);
          if (!ok) break;
          total += *(volatile float*)&ctl->sums[Iq & 1][row];
        }
        ++Iq;
      }
      if (wg == 0 && row < keys) P.out[(long long)(row0 + row) * p.nhead_k + head] = total;
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
    tmem_dealloc(tmem, 512u);
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

template <int D, bool BF16>
cudaError_t launch_one(const CUtensorMap& tk, const CUtensorMap& tq, const KeyWeightsParams& P, cudaStream_t stream) {
  static SmemOptIn opt_in;
  cudaError_t e = opt_in.once(reinterpret_cast<const void*>(key_weights_sm100_kernel<D, BF16>), (int)kw_smem<D>());
  if (e != cudaSuccess) return e;
  const long long resident = sm100_sm_count();
  const unsigned grid = (unsigned)(P.total_items < resident ? P.total_items : resident);
  key_weights_sm100_kernel<D, BF16><<<grid, kKwThreads, kw_smem<D>(), stream>>>(tk, tq, P);
  return cudaGetLastError();
}

}  // namespace

int launch_key_weights_sm100(KeyWeightsParams& P, const hbsa_forward_args& a, cudaStream_t stream, const char** err_text) {
  EncodeTiledFn fn = sm100_encode_fn();
  if (!fn) { *err_text = "cuTensorMapEncodeTiled is not available from the CUDA driver"; return HBSA_ERR_DRIVER; }
  const Problem& p = P.p;
  const bool bf16 = a.dtype == HBSA_DTYPE_BF16;
  const int d_tile = p.headdim <= 64 ? 64 : p.headdim <= 128 ? 128 : 256, tile = d_tile == 256 ? 64 : 128;
  P.gp = 1;                                          // largest power of two that divides the group
  P.gp_shift = 0;
  while (P.gp < tile && p.group % (P.gp * 2) == 0) {
    P.gp *= 2;
    ++P.gp_shift;
  }
  P.n_head_sub = p.group / P.gp;
  // rows of a tile: tokens x heads of a q-block, split evenly into the fewest tiles, rounded up to 16
  const int rows = p.qbs * P.gp, n = (rows + tile - 1) / tile;
  P.nt = ((rows + n - 1) / n + 15) / 16 * 16;
  if (P.nt % P.gp != 0) P.nt = (P.nt + P.gp - 1) / P.gp * P.gp;
  P.tt = P.nt / P.gp;
  P.n_msub = (p.kbs + 127) / 128;
  P.m_rows = ((p.kbs + P.n_msub - 1) / P.n_msub + 15) / 16 * 16;
  P.total_items = (long long)p.nhead_k * p.num_k_block * P.n_msub;
  CUtensorMap tk, tq;
  if (!sm100_encode_map(fn, &tk, bf16, a.k, p.headdim, p.nhead_k, a.total_k, a.k_stride[0], a.k_stride[1], 1, 128) ||
      !sm100_encode_map(fn, &tq, bf16, a.q, p.headdim, p.nhead_q, a.total_q, a.q_stride[0], a.q_stride[1], P.gp, P.tt)) {
    *err_text = "cuTensorMapEncodeTiled rejected a q/k layout";
    return HBSA_ERR_UNSUPPORTED;
  }
  cudaError_t e;
  if (d_tile == 64) e = bf16 ? launch_one<64, true>(tk, tq, P, stream) : launch_one<64, false>(tk, tq, P, stream);
  else if (d_tile == 128) e = bf16 ? launch_one<128, true>(tk, tq, P, stream) : launch_one<128, false>(tk, tq, P, stream);
  else e = bf16 ? launch_one<256, true>(tk, tq, P, stream) : launch_one<256, false>(tk, tq, P, stream);
  if (e != cudaSuccess) { *err_text = cudaGetErrorString(e); return (int)e; }
  return 0;
}

}  // namespace hbsa
