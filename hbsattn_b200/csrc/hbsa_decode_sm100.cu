// Main kernel of the paged decode attention for bf16 / fp16: one pass over K and V, see hbsa_decode.cu for the mathematics and
// hbsa_decode.cuh for the split.
//
// What bounds it is the read of K and V: a key of head dimension d is 4 d bytes and 4 d FLOP per q-head, so even 32 heads per kv-head stay
// below 32 FLOP a byte, where the chip has 250.  The products are therefore made with warp-wide mma.sync on fragments: a tcgen05.mma
// works on 128 rows, of which a GQA group fills 1 to 32, and its softmax would have to go through tensor memory and back, while
// a warp here keeps scores, statistics and output in registers and meets no other warp before the row ends.
//
// 288 threads, one persistent CTA per SM:
//   warp 8      walks the CTA's rows, looks the pages up 32 pieces at a time (the next 32 while these are issued) and loads K and V tiles
//               of 64 keys by TMA, 128-byte swizzled, into a ring of as many stages as fit: one box per panel of 64 columns
//               and piece; a piece is the largest power of two up to 64 positions that neither a page nor a block of the mask cuts.
//   warps 0-7   warp w takes keys 16 (w mod 4) .. + 15 of a tile: S = Q K^T (16 heads x 16 keys), running maximum and sum, O += P V.  With up
//               to 16 heads warps 0-3 take the even tiles and 4-7 the odd ones, with up to 32 both take every tile, 16 heads each.
// At the end of a row the warps' parts are put together through shared memory, 64 columns at a time.
// Positions behind the length share the last tile with others and may hold anything: their scores are set to -inf, and their
// rows of V to zero in shared memory (0 x NaN would come out of the product otherwise).
#include <math.h>

#include "hbsa_decode.cuh"
#include "sm100_common.cuh"

namespace hbsa {

namespace {

constexpr int kThreads = 288;
constexpr int kConsumers = 8;
constexpr int kSlabs = 4;                // slabs of 16 keys in a tile
constexpr int kRowSlots = 2;

template <int D> struct Ring { static constexpr int kStages = D == 64 ? 12 : D == 128 ? 6 : 3; };

struct SlabInfo {
  int pos;               // position of the slab's first key
  int n;                 // keys of it that take part
  int hidden;            // keys below the length on a page that does not exist
};

template <int STAGES> struct __align__(16) DecodeControl {
  unsigned long long full[STAGES], free[STAGES];
  unsigned long long row_full[kRowSlots], row_done[kRowSlots], meet;
  DecodeWalk walk;
  long long scratch[16];
  DecodeRow row[kRowSlots];
  SlabInfo slab[STAGES][kSlabs];
  float ml[kConsumers][16][2];
  int abort_flag, bad;
};

template <int D> constexpr size_t decode_smem() {
  return (size_t)Ring<D>::kStages * 2 * kDecodeTile * D * 2 + kConsumers * 16 * 64 * 4 + sizeof(DecodeControl<Ring<D>::kStages>);
}
static_assert(decode_smem<64>() <= 227 * 1024 && decode_smem<128>() <= 227 * 1024 && decode_smem<256>() <= 227 * 1024, "shared memory of one CTA");

__device__ __forceinline__ void tma_load_4d(uint32_t dst, const CUtensorMap* map, uint32_t bar, int c0, int c1, int c2, int c3) {
  asm volatile("cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, %6}], [%2];"
               ::"r"(dst), "l"(reinterpret_cast<uint64_t>(map)), "r"(bar), "r"(c0), "r"(c1), "r"(c2), "r"(c3)
               : "memory");
}
__device__ __forceinline__ void ldmatrix4(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void ldmatrix4_t(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
// c += a (16 x 16) b (16 x 8)
template <bool BF16> __device__ __forceinline__ void mma16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if (BF16)
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// The consumer warps meet; false when one of them has given up (a named barrier would wait for it for good).
__device__ __forceinline__ bool meet(uint32_t bar, uint32_t& par, volatile int* abort_flag, long long budget) {
  __syncwarp();
  if ((threadIdx.x & 31) == 0) ptx::mbar_arrive(bar);
  const bool ok = warp_wait(bar, par, abort_flag, budget);
  __syncwarp();
  par ^= 1u;
  return ok;
}

template <int D, bool BF16>
__global__ void __launch_bounds__(kThreads, 1)
decode_sm100_kernel(const __grid_constant__ CUtensorMap tm_k, const __grid_constant__ CUtensorMap tm_v, const __grid_constant__ DecodeParams P) {
  using namespace ptx;
  constexpr int STAGES = Ring<D>::kStages, PANELS = D / 64, KSTEPS = D / 16;
  constexpr uint32_t PANEL = kDecodeTile * 128u, HALF = PANEL * PANELS, STAGE = 2 * HALF;       // bytes: 64 rows of 128, K or V, both
  using T = typename std::conditional<BF16, __nv_bfloat16, __half>::type;
  extern __shared__ __align__(1024) uint8_t base[];  // 1024-byte aligned tiles for the 128-byte swizzle
  const uint32_t ring = smem_u32(base);
  float* const part = reinterpret_cast<float*>(base + STAGES * STAGE);                           // [kConsumers][16][64]
  auto* const ctl = reinterpret_cast<DecodeControl<STAGES>*>(base + STAGES * STAGE + kConsumers * 16 * 64 * 4);
  volatile int* const abort_flag = &ctl->abort_flag;
  const long long budget = P.wait_budget;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const uint32_t b_full = smem_u32(ctl->full), b_free = smem_u32(ctl->free), b_row_full = smem_u32(ctl->row_full), b_row_done = smem_u32(ctl->row_done);
  const bool wide = P.chunk_heads > 16;            // every tile goes to all eight warps
  if (tid == 0) {
    for (int i = 0; i < STAGES; ++i) {
      mbar_init(b_full + 8 * i, 1);
      mbar_init(b_free + 8 * i, wide ? kConsumers : kSlabs);
    }
    for (int i = 0; i < kRowSlots; ++i) {
      mbar_init(b_row_full + 8 * i, 1);
      mbar_init(b_row_done + 8 * i, kConsumers);
    }
    ctl->abort_flag = (ring & 1023u) != 0 ? 1 : 0;
    ctl->bad = 0;
    mbar_init(smem_u32(&ctl->meet), kConsumers);
    fence_barrier_init();
  }
  if (tid == kThreads - 32) {
    prefetch_tensormap(&tm_k);
    prefetch_tensormap(&tm_v);
  }
  pdl_wait();                                      // the block lists
  decode_locate(P, blockIdx.x, P.grid, blockIdx.x == 0 ? P.sp.entry_start : nullptr, &ctl->walk, ctl->scratch);
  pdl_launch();

  if (warp == kConsumers) {
    // =============================== rows, pages, TMA ===============================
    DecodeWalk walk = ctl->walk;
    if (walk.start >= walk.end && lane == 0) P.sp.cta_start[blockIdx.x] = make_int4(-1, 0, 0, 0);
    bool ok = *abort_flag == 0 && P.debug_stall == 0;
    int stage = 0, n_rows = 0, used = 0;
    uint32_t par = 1u;
    const int per_tile = kDecodeTile / P.unit;                 // pieces of a tile: 1, 2 or 4
    const uint32_t piece_bytes = (uint32_t)P.unit * 128u;
    for (long long t = walk.start; ok;) {
      if (n_rows >= kRowSlots) ok = warp_wait(b_row_done + 8 * (n_rows & 1), (uint32_t)((n_rows >> 1) - 1) & 1u, abort_flag, budget);
      if (!ok) break;
      DecodeRow r;
      r.b = -1;
      if (t < walk.end) r = decode_row_at(P, walk, t);
      if (lane == 0) {
        ctl->row[n_rows & 1] = r;
        if (r.b >= 0 && t == walk.start) decode_note_start(P, r);
        __threadfence_block();
        mbar_arrive(b_row_full + 8 * (n_rows & 1));
      }
      ++n_rows;
      if (r.b < 0) break;
      t += r.tiles;
      // lane i: position and page of piece first + i of the row; page -1: there is none
      const int32_t* const pages = P.table + r.b * P.table_stride;
      const int end = (r.tile0 + r.tiles) * per_tile;
      auto look_up = [&](int piece, int& pos, int& page) {
        pos = -1;
        page = 0;
        if (piece < end) pos = P.mask != nullptr ? decode_piece_position(P, r, piece) : piece * P.unit;
        if (pos >= r.len) pos = -1;
        if (pos >= 0) page = pages[pos / P.page];
      };
      int first = r.tile0 * per_tile, pos, page, next_pos, next_page;
      look_up(first + lane, pos, page);
      while (first < end && ok) {
        look_up(first + 32 + lane, next_pos, next_page);
        const bool bad = pos >= 0 && (page < 0 || page >= P.num_pages);
        if (__any_sync(0xffffffffu, bad) && lane == 0) ctl->bad = 1 + r.b;
        const int n_keys = pos < 0 || bad ? 0 : min(P.unit, r.len - pos), n_hidden = bad ? min(P.unit, r.len - pos) : 0;
        const int slot = pos < 0 ? 0 : pos % P.page;
        for (int g = 0; g < 32 && first + g < end; g += per_tile) {
          if (used >= STAGES) ok = warp_wait(b_free + 8 * stage, par, abort_flag, budget);
          if (!ok) break;
          const bool mine = lane >= g && lane < g + per_tile;
          const uint32_t loads = __ballot_sync(0xffffffffu, mine && n_keys > 0);
          // slabs: 16 keys each, unit / 16 per piece
          if (mine) {
            for (int s = 0; s < P.unit / 16; ++s) {
              SlabInfo* to = &ctl->slab[stage][(lane - g) * (P.unit / 16) + s];
              to->pos = pos + 16 * s;
              to->n = max(0, min(16, n_keys - 16 * s));
              to->hidden = max(0, min(16, n_hidden - 16 * s));
            }
          }
          __syncwarp();
          const uint32_t bar = b_full + 8 * stage;
          if (lane == 0) {
            __threadfence_block();
            if (loads != 0u) mbar_arrive_expect_tx(bar, (uint32_t)__popc(loads) * piece_bytes * 2u * PANELS);
            else mbar_arrive(bar);
          }
          __syncwarp();
          if (mine && n_keys > 0) {
            const uint32_t dst = ring + (uint32_t)stage * STAGE + (uint32_t)(lane - g) * piece_bytes;
#pragma unroll
            for (int pn = 0; pn < PANELS; ++pn) tma_load_4d(dst + pn * PANEL, &tm_k, bar, pn * 64, r.hk, slot, page);
#pragma unroll
            for (int pn = 0; pn < PANELS; ++pn) tma_load_4d(dst + HALF + pn * PANEL, &tm_v, bar, pn * 64, r.hk, slot, page);
          }
          ++used;
          if (++stage == STAGES) {
            stage = 0;
            par ^= 1u;
          }
        }
        first += 32;
        pos = next_pos;
        page = next_page;
      }
    }
    {                                                // copies still in flight land before the CTA leaves (bounded)
      for (int back = 1; back <= STAGES && used - back >= 0; ++back) {
        const int c = used - back;
        mbar_wait_clock(b_full + 8u * (uint32_t)(c % STAGES), (uint32_t)(c / STAGES) & 1u, budget >> 4);
      }
    }
  } else {
    // =============================== products and softmax ===============================
    const int slab = warp & 3, half = warp >> 2, g = lane >> 2, t4 = lane & 3;
    const int head_base = wide ? half * 16 : 0;      // first of the warp's 16 heads in the chunk
    bool ok = *abort_flag == 0;
    int n_rows = 0, stage = 0, tile_count = 0;
    uint32_t par = 0u, meet_par = 0u;
    const uint32_t b_meet = smem_u32(&ctl->meet);
    // ldmatrix addresses: row of the slab and 16-byte column that this lane points at
    const uint32_t k_row = (uint32_t)(slab * 16 + (lane & 7) + ((lane >> 4) << 3)), k_col = (uint32_t)((lane >> 3) & 1);
    const uint32_t v_row = (uint32_t)(slab * 16 + (lane & 15)), v_col = (uint32_t)(lane >> 4);
    while (ok) {
      ok = warp_wait(b_row_full + 8 * (n_rows & 1), (uint32_t)(n_rows >> 1) & 1u, abort_flag, budget);
      if (!ok) break;
      const DecodeRow r = ctl->row[n_rows & 1];
      if (r.b < 0) break;
      const int head0 = r.hk * P.group + r.chunk * P.chunk_heads, heads = min(P.chunk_heads, P.group - r.chunk * P.chunk_heads);
      // Q as left operands: heads g and g + 8 of the warp's 16
      uint32_t q[KSTEPS][4];
#pragma unroll
      for (int ks = 0; ks < KSTEPS; ++ks)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int h = head_base + g + (e & 1) * 8, d = ks * 16 + t4 * 2 + (e >> 1) * 8;
          q[ks][e] = h < heads && d < P.headdim ? *reinterpret_cast<const uint32_t*>(static_cast<const T*>(P.q) + r.b * P.q_s[0] + (head0 + h) * P.q_s[1] + d) : 0u;
        }
      float o[D / 8][4];
#pragma unroll
      for (int i = 0; i < D / 8; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[i][e] = 0.f;
      float m0 = -INFINITY, m1 = -INFINITY, l0 = 0.f, l1 = 0.f;
      float *score0 = nullptr, *score1 = nullptr;
      if (P.weights != nullptr) {
        if (head_base + g < heads) score0 = P.sp.scores + ((long long)r.b * P.nhead_q + head0 + head_base + g) * P.capacity;
        if (head_base + g + 8 < heads) score1 = P.sp.scores + ((long long)r.b * P.nhead_q + head0 + head_base + g + 8) * P.capacity;
      }
      for (int i = 0; i < r.tiles; ++i, ++tile_count) {
        const bool mine = wide || (tile_count & 1) == half;
        if (mine) {
          ok = warp_wait(b_full + 8 * stage, par, abort_flag, budget);
          if (!ok) break;
          const volatile SlabInfo* info = &ctl->slab[stage][slab];
          const int n = info->n, pos = info->pos, hidden = info->hidden;
          if (n > 0) {
            const uint32_t k_at = ring + (uint32_t)stage * STAGE, v_at = k_at + HALF;
            float s[2][4];
#pragma unroll
            for (int e = 0; e < 4; ++e) s[0][e] = s[1][e] = 0.f;
#pragma unroll
            for (int ks = 0; ks < KSTEPS; ++ks) {
              uint32_t f[4];
              const uint32_t col = (uint32_t)(ks & 3) * 2u + k_col;
              ldmatrix4(k_at + (uint32_t)(ks >> 2) * PANEL + k_row * 128u + ((col ^ (k_row & 7u)) << 4), f);
              mma16816<BF16>(s[0], q[ks], f[0], f[1]);
              mma16816<BF16>(s[1], q[ks], f[2], f[3]);
            }
#pragma unroll
            for (int j = 0; j < 2; ++j)
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                s[j][e] *= P.scale_log2;
                if (j * 8 + t4 * 2 + (e & 1) >= n) s[j][e] = -INFINITY;
              }
            if (P.weights != nullptr) {
#pragma unroll
              for (int j = 0; j < 2; ++j)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                  const int key = j * 8 + t4 * 2 + e;
                  if (key < n) {
                    if (score0 != nullptr) score0[pos + key] = s[j][e];
                    if (score1 != nullptr) score1[pos + key] = s[j][2 + e];
                  }
                }
            }
            float x0 = fmaxf(fmaxf(s[0][0], s[0][1]), fmaxf(s[1][0], s[1][1])), x1 = fmaxf(fmaxf(s[0][2], s[0][3]), fmaxf(s[1][2], s[1][3]));
            x0 = fmaxf(x0, __shfl_xor_sync(0xffffffffu, x0, 1));
            x1 = fmaxf(x1, __shfl_xor_sync(0xffffffffu, x1, 1));
            x0 = fmaxf(m0, fmaxf(x0, __shfl_xor_sync(0xffffffffu, x0, 2)));
            x1 = fmaxf(m1, fmaxf(x1, __shfl_xor_sync(0xffffffffu, x1, 2)));
            if (__any_sync(0xffffffffu, x0 > m0 || x1 > m1)) {
              const float a0 = x0 == -INFINITY ? 1.f : ex2_approx(m0 - x0), a1 = x1 == -INFINITY ? 1.f : ex2_approx(m1 - x1);
              l0 *= a0;
              l1 *= a1;
#pragma unroll
              for (int d = 0; d < D / 8; ++d) {
                o[d][0] *= a0;
                o[d][1] *= a0;
                o[d][2] *= a1;
                o[d][3] *= a1;
              }
              m0 = x0;
              m1 = x1;
            }
            const float r0 = m0 == -INFINITY ? 0.f : m0, r1 = m1 == -INFINITY ? 0.f : m1;
            uint32_t p[4];
#pragma unroll
            for (int j = 0; j < 2; ++j) {
              const float p0 = ex2_approx(s[j][0] - r0), p1 = ex2_approx(s[j][1] - r0), p2 = ex2_approx(s[j][2] - r1), p3 = ex2_approx(s[j][3] - r1);
              l0 += p0 + p1;
              l1 += p2 + p3;
              p[2 * j] = pack2<BF16>(p0, p1);
              p[2 * j + 1] = pack2<BF16>(p2, p3);
            }
            if (n < 16) {                            // rows of V behind the length: zeros
              if (lane >= n && lane < 16)
#pragma unroll
                for (int pn = 0; pn < PANELS; ++pn)
#pragma unroll
                  for (int c = 0; c < 8; ++c) st_shared_v4(v_at + pn * PANEL + (uint32_t)(slab * 16 + lane) * 128u + c * 16u, 0u, 0u, 0u, 0u);
              fence_proxy_async();
              __syncwarp();
            }
#pragma unroll
            for (int c = 0; c < D / 16; ++c) {
              uint32_t f[4];
              const uint32_t col = (uint32_t)(c & 3) * 2u + v_col;
              ldmatrix4_t(v_at + (uint32_t)(c >> 2) * PANEL + v_row * 128u + ((col ^ (v_row & 7u)) << 4), f);
              mma16816<BF16>(o[2 * c], p, f[0], f[1]);
              mma16816<BF16>(o[2 * c + 1], p, f[2], f[3]);
            }
          }
          if (hidden > 0 && P.weights != nullptr) {   // keys on a page that does not exist: no weight
            if (t4 == 0)
              for (int key = 0; key < hidden; ++key) {
                if (score0 != nullptr) score0[pos + key] = -INFINITY;
                if (score1 != nullptr) score1[pos + key] = -INFINITY;
              }
          }
          __syncwarp();
          if (lane == 0) mbar_arrive(b_free + 8 * stage);
        }
        if (++stage == STAGES) {
          stage = 0;
          par ^= 1u;
        }
      }
      if (!ok) break;
      // ---- the warps' parts of the row
      l0 += __shfl_xor_sync(0xffffffffu, l0, 1);
      l1 += __shfl_xor_sync(0xffffffffu, l1, 1);
      l0 += __shfl_xor_sync(0xffffffffu, l0, 2);
      l1 += __shfl_xor_sync(0xffffffffu, l1, 2);
      if (t4 == 0) {
        *reinterpret_cast<float2*>(ctl->ml[warp][g]) = make_float2(m0, l0);
        *reinterpret_cast<float2*>(ctl->ml[warp][g + 8]) = make_float2(m1, l1);
      }
      ok = meet(b_meet, meet_par, abort_flag, budget);
      if (ok) {
        const int w0 = wide ? half * 4 : 0, w1 = wide ? w0 + 4 : kConsumers;       // the warps that share this warp's heads
        float t0 = -INFINITY, t1 = -INFINITY;
        for (int w = w0; w < w1; ++w) {
          t0 = fmaxf(t0, ctl->ml[w][g][0]);
          t1 = fmaxf(t1, ctl->ml[w][g + 8][0]);
        }
        const float f0 = m0 == -INFINITY ? 0.f : ex2_approx(m0 - t0), f1 = m1 == -INFINITY ? 0.f : ex2_approx(m1 - t1);
        const long long part_slot = 2ll * blockIdx.x + max(r.slot, 0);
#pragma unroll
        for (int c = 0; c < PANELS; ++c) {
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            float* to = part + (warp * 16 + g) * 64 + (i ^ g) * 8 + t4 * 2;      // groups of 8 columns swapped by row: no bank conflicts
            *reinterpret_cast<float2*>(to) = make_float2(o[c * 8 + i][0] * f0, o[c * 8 + i][1] * f0);
            *reinterpret_cast<float2*>(to + 8 * 64) = make_float2(o[c * 8 + i][2] * f1, o[c * 8 + i][3] * f1);
          }
          if (!(ok = meet(b_meet, meet_par, abort_flag, budget))) break;
          // thread = (head, 4 columns); 32 heads in two goes
          for (int hh = 0; hh < (wide ? 2 : 1); ++hh) {
            const int hl = tid >> 4, col = (tid & 15) * 4, head = hh * 16 + hl;
            const int a = wide ? hh * 4 : 0, b = wide ? a + 4 : kConsumers;
            float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
            float mt = -INFINITY, lt = 0.f;
            for (int w = a; w < b; ++w) mt = fmaxf(mt, ctl->ml[w][hl][0]);
            for (int w = a; w < b; ++w) {
              const float4 y = *reinterpret_cast<const float4*>(part + (w * 16 + hl) * 64 + (((col >> 3) ^ (hl & 7)) << 3) + (col & 7));
              x.x += y.x;
              x.y += y.y;
              x.z += y.z;
              x.w += y.w;
              const float mw = ctl->ml[w][hl][0];
              lt += mw == -INFINITY ? ctl->ml[w][hl][1] : ctl->ml[w][hl][1] * ex2_approx(mw - mt);
            }
            if (head < heads) {
              if (r.slot >= 0) {
                *reinterpret_cast<float4*>(P.sp.part_o + (part_slot * kDecodeHeads + head) * D + c * 64 + col) = x;
                if (c == 0 && col == 0) *reinterpret_cast<float2*>(P.sp.part_ml + (part_slot * kDecodeHeads + head) * 2) = make_float2(mt, lt);
              } else {
                const bool none = mt == -INFINITY && lt == 0.f;
                const float inv = none ? 0.f : 1.f / lt;
                const int d = c * 64 + col;
                if (d < P.headdim)
                  *reinterpret_cast<uint2*>(static_cast<T*>(P.o) + r.b * P.o_s[0] + (head0 + head) * P.o_s[1] + d) =
                      none ? make_uint2(0u, 0u) : make_uint2(pack2<BF16>(x.x * inv, x.y * inv), pack2<BF16>(x.z * inv, x.w * inv));
                if (c == 0 && col == 0 && P.lse != nullptr)
                  P.lse[(long long)r.b * P.nhead_q + head0 + head] = none ? -INFINITY : (mt + log2f(lt)) * kDecodeLn2;
              }
            }
          }
          if (!(ok = meet(b_meet, meet_par, abort_flag, budget))) break;           // before the next columns, or the next row's statistics
        }
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(b_row_done + 8 * (n_rows & 1));
      ++n_rows;
    }
  }
  __syncthreads();
  decode_fill_empty<T>(P, blockIdx.x, P.grid);
  for (int b = blockIdx.x * kThreads + tid; b < P.batch; b += P.grid * kThreads)
    if (P.lens[b] < 0 || P.lens[b] > P.capacity) ctl->bad = 1 + b;
  __syncthreads();
  if (tid == 0) {
    const int bad = ctl->bad;
    decode_note_status(P, ctl->abort_flag != 0 ? (int)HBSA_STATUS_WAIT_LIMIT : bad != 0 ? (int)HBSA_STATUS_CACHE_BOUNDS : (int)HBSA_STATUS_OK, bad - 1);
  }
}

// 4-D map over pages of a cache: dims (headdim, heads, slots, pages), box (64, 1, unit, 1).
bool encode_cache_map(EncodeTiledFn fn, CUtensorMap* map, bool bf16, const void* base, const DecodeParams& P, const long long* s) {
  cuuint64_t dims[4] = {(cuuint64_t)P.headdim, (cuuint64_t)P.nhead_k, (cuuint64_t)P.page, (cuuint64_t)P.num_pages};
  cuuint64_t strides[3] = {(cuuint64_t)s[2] * 2ull, (cuuint64_t)s[1] * 2ull, (cuuint64_t)s[0] * 2ull};
  cuuint32_t box[4] = {64u, 1u, (cuuint32_t)P.unit, 1u}, estr[4] = {1u, 1u, 1u, 1u};
  return fn(map, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 4, const_cast<void*>(base), dims, strides, box, estr,
            CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <int D, bool BF16>
cudaError_t launch_one(const CUtensorMap& tk, const CUtensorMap& tv, const DecodeParams& P, bool dependent, cudaStream_t stream) {
  static SmemOptIn opt_in;
  cudaError_t e = opt_in.once(reinterpret_cast<const void*>(decode_sm100_kernel<D, BF16>), (int)decode_smem<D>());
  if (e != cudaSuccess) return e;
  return launch_kernel(decode_sm100_kernel<D, BF16>, (unsigned)P.grid, kThreads, decode_smem<D>(), dependent, stream, tk, tv, P);
}

}  // namespace

const char* decode_sm100_ineligible_reason(const hbsa_paged_attention_args& a, float scale) {
  const hbsa_cache& c = a.cache;
  if (c.dtype != HBSA_DTYPE_BF16 && c.dtype != HBSA_DTYPE_F16) return "dtype is not bf16/fp16";
  if (c.headdim % 8 != 0 || c.headdim < 16 || c.headdim > 256) return "headdim is not a multiple of 8 between 16 and 256";
  if (c.page_size % 16 != 0) return "page_size is not a multiple of 16";
  if (!(scale > 0.f) || !isfinite(scale)) return "softmax_scale is not a positive finite number";
  if (c.k_stride[3] != 1 || c.v_stride[3] != 1 || a.q_stride[2] != 1 || a.o_stride[2] != 1) return "headdim stride is not 1";
  for (int i = 0; i < 3; ++i)
    for (const int64_t s : {c.k_stride[i], c.v_stride[i]})
      if (s <= 0 || s % 8 != 0 || s >= (1ll << 39)) return "a page/slot/head stride is not a positive multiple of 16 bytes";
  for (int i = 0; i < 2; ++i)
    if (a.q_stride[i] % 8 != 0 || a.o_stride[i] % 8 != 0) return "a stride of q or o is not a multiple of 16 bytes";
  if ((uintptr_t)c.k % 16 != 0 || (uintptr_t)c.v % 16 != 0 || (uintptr_t)a.q % 16 != 0 || (uintptr_t)a.o % 16 != 0) return "a base address is not 16-byte aligned";
  return nullptr;
}

int launch_decode_sm100(const DecodeParams& P, const hbsa_paged_attention_args& a, bool dependent, cudaStream_t stream, const char** err_text) {
  EncodeTiledFn fn = sm100_encode_fn();
  if (!fn) { *err_text = "cuTensorMapEncodeTiled is not available from the CUDA driver"; return HBSA_ERR_DRIVER; }
  const bool bf16 = a.cache.dtype == HBSA_DTYPE_BF16;
  CUtensorMap tk, tv;
  if (!encode_cache_map(fn, &tk, bf16, P.k, P, P.k_s) || !encode_cache_map(fn, &tv, bf16, P.v, P, P.v_s)) {
    *err_text = "cuTensorMapEncodeTiled rejected a cache layout";
    return HBSA_ERR_UNSUPPORTED;
  }
  cudaError_t e;
  if (P.d_pad == 64) e = bf16 ? launch_one<64, true>(tk, tv, P, dependent, stream) : launch_one<64, false>(tk, tv, P, dependent, stream);
  else if (P.d_pad == 128) e = bf16 ? launch_one<128, true>(tk, tv, P, dependent, stream) : launch_one<128, false>(tk, tv, P, dependent, stream);
  else e = bf16 ? launch_one<256, true>(tk, tv, P, dependent, stream) : launch_one<256, false>(tk, tv, P, dependent, stream);
  if (e != cudaSuccess) { *err_text = cudaGetErrorString(e); return (int)e; }
  return 0;
}

}  // namespace hbsa
