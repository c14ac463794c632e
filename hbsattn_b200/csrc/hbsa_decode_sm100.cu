// Main kernel of the paged decode attention for bf16 / fp16: one pass over K and V, see hbsa_decode.cu for the mathematics and
// hbsa_decode.cuh for the split.
//
// What bounds it is the read of K and V: a key of head dimension d is 4 d bytes and 4 d FLOP per q-head, so even 32 heads per kv-head stay
// below 32 FLOP a byte, where the chip has 250.  The products are therefore made with warp-wide mma.sync on fragments: a tcgen05.mma
// works on 128 rows, of which a GQA group fills 1 to 32, and its softmax would have to go through tensor memory and back, while
// a warp here keeps scores, statistics and output in registers and meets no other warp before the row ends.
//
// 320 threads, one persistent CTA per SM:
//   warps 8, 9  walk the CTA's rows, look the pages up 32 pieces at a time (the next 32 while these are issued) and load K (warp 8) and
//               V (warp 9) by TMA, 128-byte swizzled, into a ring of as many stages as fit; a stage is one or two tiles of 64 keys.  A piece
//               is the largest power of two up to 64 positions that neither a page nor a block of the mask cuts; one box brings
//               all of its columns where headdim is a multiple of 64 (x, slot, panel), one per panel of 64 columns otherwise.
//   warps 0-7   warp w takes a slab of 16 or 32 keys of a stage, the (w mod 4)-th: S = Q K^T (16 heads), running maximum and sum, O += P V.
//               With up to 16 heads warps 0-3 take the even stages and 4-7 the odd ones, with up to 32 both take every stage, 16
//               heads each (groups of more take several chunks, each of which reads K and V again: 8 x 16384 keys, 4 kv-heads of 128: 86 us with groups
//               of 32, 133 with 64).  256 columns of O do not fit a warp's registers: there both take every stage, up to 16 heads (chunks of 16:
//               groups of 16 and 32 of 256 columns 101 and 175 us) and half of O's columns each (the scores are made twice), and Q is read from
//               shared memory for every product.
// At the end of a row the warps' parts are put together through shared memory, up to 128 columns at a time.
// P enters P V in the type of V.  With up to 8 heads a chunk it does so in two terms, P rounded and what that leaves (as in the package's backward): rows
// 8 to 15 of the products' left operands, which would be idle, hold the second term, and the two halves of O come together at the end of the row.  That
// costs nothing (16 x 16384..32768 keys, 8 heads of 64, groups of 8: 128.1 us, with one term 128.9; 8 x 16384..65536 at 30 % 100.7 and 100.5; fp16 with
// weights 30.8 and 32.3, as no exponentials are made for the idle rows) and takes P's rounding out of the result: 1.65e-3 (bf16) and 2.1e-4 (fp16) of
// the output against 64 bits, what the output's own rounding makes; 2.1e-3 to 2.2e-3 and 2.7e-4 with one term (8 x 4096..16384 keys).  More heads use
// all rows and have one term, at most 2^-8 or 2^-11 of every p, like the prompts' kernels: a second product would double the tensor work.
// In fp16 such bounds hold for normal numbers only, so P is formed against the maximum less 14 there: the largest is 2^14 (of 2^16 that
// fp16 has), and rounding is by 2^-11 of a term down to 2^-28 of the largest, by at most 2^-39 of the largest below.  Against the maximum itself
// everything below 2^-25 was lost (equal keys 19 nats below sinks that every warp meets: all of their share; now within 2^-10 of it, in the same time).
// The factor is in O, the sums and the maxima that are handed on, and leaves with the division.  Scores, statistics and sums are fp32.
// Measured: 16 x 16384..32768 keys, 8 heads of 64, groups of 8: 125 us, of which 102 are the stream (745 MB, 7.3 TB/s), 6 the way to the first tile, 6
// the join; 8 x 16384..65536 keys, 30 % of the blocks, 8 heads of 128: 98 us (527 MB).  A call without work to speak of: 10.5 us.
// Positions behind the length share the last tile with others and may hold anything: their scores are set to -inf, and their
// rows of V to zero in shared memory (0 x NaN would come out of the product otherwise).
#include <math.h>

#include "hbsa_decode.cuh"
#include "sm100_common.cuh"

namespace hbsa {

namespace {

constexpr int kThreads = 320;
constexpr int kConsumers = 8;
constexpr int kSlabs = 4;                // slabs of a stage
constexpr int kRowSlots = 2;

// Per head dimension of the tiles: keys of a slab in units of 16, stages, columns of O of a warp.
template <int D> struct Shape {
  static constexpr int kUnits = D == 64 ? 2 : 1;
  static constexpr int kStages = D == 256 ? 3 : 6;
  static constexpr int kKeys = kSlabs * kUnits * 16;             // of a stage
  static constexpr bool kHalves = D == 256;                      // warps w and w + 4 share the columns of O
  static constexpr int kColumns = kHalves ? D / 2 : D;
};

struct __align__(16) SlabInfo {          // of 16 keys
  int pos;               // position of the first key
  int n;                 // keys that take part
  int hidden;            // keys below the length on a page that does not exist
  int pad;
};

template <int D> struct __align__(16) DecodeControl {
  SlabInfo slab[Shape<D>::kStages][kSlabs * Shape<D>::kUnits];
  unsigned long long full[Shape<D>::kStages], free[Shape<D>::kStages];
  unsigned long long row_full[kRowSlots], row_done[kRowSlots], part_full, part_free;
  DecodeWalk walk;
  long long scratch[16];
  DecodeRow row[kRowSlots];
  float ml[kConsumers][16][2];
  int abort_flag, bad;   // bad: the first sequence with a length or a page out of range, from the end (0: none)
};

constexpr uint32_t kPartBytes = kConsumers * 16 * 64 * 4;
template <int D> constexpr size_t decode_smem() { return (size_t)Shape<D>::kStages * 2 * Shape<D>::kKeys * D * 2 + kPartBytes + sizeof(DecodeControl<D>); }
static_assert(decode_smem<64>() <= 227 * 1024 && decode_smem<128>() <= 227 * 1024 && decode_smem<256>() <= 227 * 1024, "shared memory of one CTA");

__device__ __forceinline__ void tma_load_5d(uint32_t dst, const CUtensorMap* map, uint32_t bar, int c0, int c1, int c2, int c3, int c4) {
  asm volatile("cp.async.bulk.tensor.5d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, %6, %7}], [%2];"
               ::"r"(dst), "l"(reinterpret_cast<uint64_t>(map)), "r"(bar), "r"(c0), "r"(c1), "r"(c2), "r"(c3), "r"(c4)
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
// PAIRED: up to 8 heads a chunk, rows 8 .. 15 hold what P of rows 0 .. 7 loses in 16 bits.
template <int D, bool BF16, bool PAIRED>
__global__ void __launch_bounds__(kThreads, 1)
decode_sm100_kernel(const __grid_constant__ CUtensorMap tm_k, const __grid_constant__ CUtensorMap tm_v, const __grid_constant__ DecodeParams P) {
  using namespace ptx;
  constexpr int STAGES = Shape<D>::kStages, UNITS = Shape<D>::kUnits, PANELS = D / 64, KSTEPS = D / 16;
  constexpr uint32_t HALF = (uint32_t)Shape<D>::kKeys * D * 2u, STAGE = 2 * HALF;      // bytes of K or V, and of both
  constexpr bool HALVES = Shape<D>::kHalves;
  constexpr int COLUMNS = Shape<D>::kColumns;
  // P = 2^(score - reference(maximum)).  Beyond 2^24 subtracting 14 may subtract 16, and 2^16 is no fp16 number.
  auto reference = [](float m) { return BF16 || fabsf(m) >= 16777216.f ? m : m - 14.f; };
  using T = typename std::conditional<BF16, __nv_bfloat16, __half>::type;
  extern __shared__ __align__(1024) uint8_t base[];  // 1024-byte aligned tiles for the 128-byte swizzle
  const uint32_t ring = smem_u32(base);
  float* const part = reinterpret_cast<float*>(base + STAGES * STAGE);                 // [kConsumers][16][64]
  auto* const ctl = reinterpret_cast<DecodeControl<D>*>(base + STAGES * STAGE + kPartBytes);
  volatile int* const abort_flag = &ctl->abort_flag;
  const long long budget = P.wait_budget;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const uint32_t b_full = smem_u32(ctl->full), b_free = smem_u32(ctl->free), b_row_full = smem_u32(ctl->row_full), b_row_done = smem_u32(ctl->row_done);
  const bool wide = !HALVES && P.chunk_heads > 16; // two times 16 heads
  const bool all = HALVES || wide;                 // every stage goes to all eight warps
  const uint32_t piece_panel = (uint32_t)P.unit * 128u;                                // bytes of a piece's panel of 64 columns
  if (tid == 0) {
    for (int i = 0; i < STAGES; ++i) {
      mbar_init(b_full + 8 * i, 2);
      mbar_init(b_free + 8 * i, all ? kConsumers : kSlabs);
    }
    for (int i = 0; i < kRowSlots; ++i) {
      mbar_init(b_row_full + 8 * i, 1);
      mbar_init(b_row_done + 8 * i, kConsumers);
    }
    mbar_init(smem_u32(&ctl->part_full), kConsumers);
    mbar_init(smem_u32(&ctl->part_free), kConsumers);
    ctl->abort_flag = (ring & 1023u) != 0 ? 1 : 0;
    ctl->bad = 0;
    fence_barrier_init();
  }
  if (tid == kConsumers * 32) prefetch_tensormap(&tm_k);
  if (tid == kConsumers * 32 + 32) prefetch_tensormap(&tm_v);
  pdl_wait();                                      // the block lists
  decode_locate(P, &ctl->walk, ctl->scratch);
  pdl_launch();

  if (warp >= kConsumers) {
    // =============================== rows, pages, TMA: K in the first of the two warps, V in the second ===============================
    const bool first_warp = warp == kConsumers;
    const CUtensorMap* const map = first_warp ? &tm_k : &tm_v;
    DecodeWalk walk = ctl->walk;
    bool ok = *abort_flag == 0 && P.debug_stall == 0;
    int stage = 0, n_rows = 0, used = 0;
    uint32_t par = 1u;
    const int per_tile = kDecodeTile / P.unit, per_stage = Shape<D>::kKeys / P.unit;    // pieces; per_stage <= 8
    for (long long t = walk.start; ok;) {
      DecodeRow r;
      r.b = -1;
      if (t < walk.end) r = decode_row_at(P, walk, t, blockIdx.x);
      if (first_warp) {
        if (n_rows >= kRowSlots) ok = warp_wait(b_row_done + 8 * (n_rows & 1), (uint32_t)((n_rows >> 1) - 1) & 1u, abort_flag, budget);
        if (!ok) break;
        if (lane == 0) {
          ctl->row[n_rows & 1] = r;
          if (r.b >= 0 && t == walk.start) decode_note_start(P, r);
          mbar_arrive(b_row_full + 8 * (n_rows & 1));
        }
        ++n_rows;
      }
      if (r.b < 0) break;
      t += r.tiles;
      // lane i: position and page of piece first + i of the row; position -1: there is none
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
        if (__any_sync(0xffffffffu, bad) && lane == 0) atomicMax(&ctl->bad, P.batch - r.b);
        const int n_keys = pos < 0 || bad ? 0 : min(P.unit, r.len - pos), n_hidden = bad ? min(P.unit, r.len - pos) : 0;
        const int slot = pos < 0 ? 0 : pos % P.page;
        const uint32_t there = __ballot_sync(0xffffffffu, n_keys > 0);
        for (int g = 0; g < 32 && first + g < end; g += per_stage) {
          if (used >= STAGES) ok = quick_wait(b_free + 8 * stage, par, abort_flag, budget);
          if (!ok) break;
          const uint32_t loads = there & (((1u << per_stage) - 1u) << g);      // the pieces behind `end` are not there
          const bool mine = lane >= g && lane < g + per_stage;
          const uint32_t bar = b_full + 8 * stage;
          if (first_warp && mine) {                  // units of 16 keys
            for (int u = 0; u < P.unit / 16; ++u)
              *reinterpret_cast<int4*>(&ctl->slab[stage][(lane - g) * (P.unit / 16) + u]) =
                  make_int4(pos + 16 * u, max(0, min(16, n_keys - 16 * u)), max(0, min(16, n_hidden - 16 * u)), 0);
          }
          __syncwarp();
          if (lane == 0) {
            if (loads != 0u) mbar_arrive_expect_tx(bar, (uint32_t)__popc(loads) * piece_panel * PANELS);
            else mbar_arrive(bar);
          }
          __syncwarp();
          if (mine && n_keys > 0) {
            const uint32_t dst = ring + (uint32_t)stage * STAGE + (first_warp ? 0u : HALF) + (uint32_t)(lane - g) * piece_panel * PANELS;
            if (P.one_box) {
              tma_load_5d(dst, map, bar, 0, slot, 0, r.hk, page);
            } else {
#pragma unroll
              for (int pn = 0; pn < PANELS; ++pn) tma_load_5d(dst + pn * piece_panel, map, bar, pn * 64, slot, 0, r.hk, page);
            }
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
    if (first_warp && lane == 0) decode_note_join(P, ctl->walk);
    // copies still in flight land before the CTA leaves (bounded)
    for (int back = 1; back <= STAGES && used - back >= 0; ++back) {
      const int c = used - back;
      mbar_wait_clock(b_full + 8u * (uint32_t)(c % STAGES), (uint32_t)(c / STAGES) & 1u, budget >> 4);
    }
  } else {
    // =============================== products and softmax ===============================
    const int slab = warp & 3, half = warp >> 2, g = lane >> 2, t4 = lane & 3;
    const int head_base = wide ? half * 16 : 0;      // first of the warp's 16 heads in the chunk
    const uint32_t o_panel = HALVES ? (uint32_t)half * (COLUMNS / 64) : 0u;      // first panel of the warp's columns of O
    bool ok = *abort_flag == 0;
    int n_rows = 0, stage = 0, count = 0;
    uint32_t par = 0u, part_par = 0u;
    const uint32_t b_part_full = smem_u32(&ctl->part_full), b_part_free = smem_u32(&ctl->part_free);
    // The consumer warps take turns with `part` and `ml`: all have written (or may read) when part_full's phase is over, all have read when
    // part_free's is.  Not by a named barrier, which would wait for good for a warp that has given up.
    auto part_arrive = [&](uint32_t bar) {
      __syncwarp();
      if (lane == 0) mbar_arrive(bar);
    };
    auto part_written = [&]() {
      part_arrive(b_part_full);
      return quick_wait(b_part_full, part_par, abort_flag, budget);
    };
    auto part_read = [&]() {
      part_arrive(b_part_free);
      part_par ^= 1u;
    };
    auto part_writable = [&]() { return quick_wait(b_part_free, part_par ^ 1u, abort_flag, budget); };      // (the first time at once)
    // where this lane points at in K and V of a stage for ldmatrix, per unit of 16 keys: a piece holds its panels one behind the other
    const uint32_t k_row = (uint32_t)((lane & 7) + ((lane >> 4) << 3)), k_col = (uint32_t)((lane >> 3) & 1);
    const uint32_t v_row = (uint32_t)(lane & 15), v_col = (uint32_t)(lane >> 4);
    uint32_t unit_at[UNITS];
#pragma unroll
    for (int u = 0; u < UNITS; ++u) {
      const int key = (slab * UNITS + u) * 16;
      unit_at[u] = (uint32_t)(key / P.unit) * piece_panel * PANELS + (uint32_t)(key % P.unit) * 128u;
    }
    const uint32_t q_smem = smem_u32(part) + (uint32_t)(lane & 15) * D * 2u;
    while (ok) {
      ok = quick_wait(b_row_full + 8 * (n_rows & 1), (uint32_t)(n_rows >> 1) & 1u, abort_flag, budget);
      if (!ok) break;
      const DecodeRow r = ctl->row[n_rows & 1];
      if (r.b < 0) break;
      const int head0 = r.hk * P.group + r.chunk * P.chunk_heads, heads = min(P.chunk_heads, P.group - r.chunk * P.chunk_heads);
      // Q as left operands: heads g and g + 8 of the warp's 16
      uint32_t q[HALVES ? 1 : KSTEPS][4];
      const T* const q_row = static_cast<const T*>(P.q) + r.b * P.q_s[0] + head0 * P.q_s[1];
      if (HALVES) {                                  // [16][D] where the parts are exchanged later, 16-byte columns swapped by row
        if (!(ok = part_writable())) break;
        for (int i = tid; i < 16 * (D / 8); i += kConsumers * 32) {
          const int h = i / (D / 8), c = i % (D / 8);
          uint4 x = make_uint4(0u, 0u, 0u, 0u);
          if (h < heads && c * 8 < P.headdim) x = *reinterpret_cast<const uint4*>(q_row + h * P.q_s[1] + c * 8);
          *reinterpret_cast<uint4*>(reinterpret_cast<uint8_t*>(part) + h * (D * 2) + ((c ^ (h & 7)) << 4)) = x;
        }
        if (!(ok = part_written())) break;
      } else {
#pragma unroll
        for (int ks = 0; ks < KSTEPS; ++ks)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int h = head_base + g + (e & 1) * 8, d = ks * 16 + t4 * 2 + (e >> 1) * 8;
            q[HALVES ? 0 : ks][e] = h < heads && d < P.headdim ? *reinterpret_cast<const uint32_t*>(q_row + h * P.q_s[1] + d) : 0u;
          }
      }
      float o[COLUMNS / 8][4];
#pragma unroll
      for (int i = 0; i < COLUMNS / 8; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[i][e] = 0.f;
      float m0 = -INFINITY, m1 = -INFINITY, l0 = 0.f, l1 = 0.f;
      float *score0 = nullptr, *score1 = nullptr;
      if (P.weights != nullptr) {
        if (head_base + g < heads) score0 = P.sp.scores + ((long long)r.b * P.nhead_q + head0 + head_base + g) * P.capacity;
        if (!PAIRED && head_base + g + 8 < heads) score1 = P.sp.scores + ((long long)r.b * P.nhead_q + head0 + head_base + g + 8) * P.capacity;
      }
      // a stage holds the same number of pieces whatever the row's first tile is, so the last one of a row may be half empty, and
      // of every 32 pieces that are looked up together the last stage is full
      const int n_stages = (r.tiles * kDecodeTile + Shape<D>::kKeys - 1) / Shape<D>::kKeys;
      for (int i = 0; i < n_stages; ++i, ++count) {
        const bool mine = all || (count & 1) == half;
        if (mine) {
          ok = quick_wait(b_full + 8 * stage, par, abort_flag, budget);
          if (!ok) break;
          int4 info[UNITS];
          int least = 16, most = 0, hidden = 0;
#pragma unroll
          for (int u = 0; u < UNITS; ++u) {
            info[u] = *reinterpret_cast<const int4*>(&ctl->slab[stage][slab * UNITS + u]);
            least = min(least, info[u].y);
            most = max(most, info[u].y);
            hidden |= info[u].z;
          }
          if (most > 0) {
            const uint32_t k_at = ring + (uint32_t)stage * STAGE, v_at = k_at + HALF;
            float s[2 * UNITS][4];
#pragma unroll
            for (int j = 0; j < 2 * UNITS; ++j)
#pragma unroll
              for (int e = 0; e < 4; ++e) s[j][e] = 0.f;
#pragma unroll
            for (int ks = 0; ks < KSTEPS; ++ks) {
              const uint32_t col = (uint32_t)(ks & 3) * 2u + k_col;
              if (HALVES) ldmatrix4(q_smem + (((uint32_t)(ks * 2) + (uint32_t)(lane >> 4)) ^ (uint32_t)(lane & 7)) * 16u, q[0]);
#pragma unroll
              for (int u = 0; u < UNITS; ++u) {
                uint32_t f[4];
                ldmatrix4(k_at + unit_at[u] + (uint32_t)(ks >> 2) * piece_panel + k_row * 128u + ((col ^ (k_row & 7u)) << 4), f);
                mma16816<BF16>(s[2 * u], q[HALVES ? 0 : ks], f[0], f[1]);
                mma16816<BF16>(s[2 * u + 1], q[HALVES ? 0 : ks], f[2], f[3]);
              }
            }
#pragma unroll
            for (int j = 0; j < 2 * UNITS; ++j)
#pragma unroll
              for (int e = 0; e < 4; ++e) s[j][e] *= P.scale_log2;
            if (least < 16) {
#pragma unroll
              for (int j = 0; j < 2 * UNITS; ++j)
#pragma unroll
                for (int e = 0; e < 4; ++e)
                  if ((j & 1) * 8 + t4 * 2 + (e & 1) >= info[j >> 1].y) s[j][e] = -INFINITY;
            }
            if (P.weights != nullptr && !(HALVES && half)) {
#pragma unroll
              for (int j = 0; j < 2 * UNITS; ++j)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                  const int key = (j & 1) * 8 + t4 * 2 + e;
                  if (key < info[j >> 1].y) {
                    if (score0 != nullptr) score0[info[j >> 1].x + key] = s[j][e];
                    if (score1 != nullptr) score1[info[j >> 1].x + key] = s[j][2 + e];
                  }
                }
            }
            float x0 = m0, x1 = m1;
#pragma unroll
            for (int j = 0; j < 2 * UNITS; ++j) {
              x0 = fmaxf(x0, fmaxf(s[j][0], s[j][1]));
              if (!PAIRED) x1 = fmaxf(x1, fmaxf(s[j][2], s[j][3]));
            }
            if (__any_sync(0xffffffffu, x0 > m0 || x1 > m1)) {       // some row's maximum grows: the quads agree on it, O and the sums follow
              x0 = fmaxf(x0, __shfl_xor_sync(0xffffffffu, x0, 1));
              x1 = fmaxf(x1, __shfl_xor_sync(0xffffffffu, x1, 1));
              x0 = fmaxf(x0, __shfl_xor_sync(0xffffffffu, x0, 2));
              x1 = fmaxf(x1, __shfl_xor_sync(0xffffffffu, x1, 2));
              // (the references' difference is not the maxima's: subtracting 14 may round)
              const float a0 = x0 == -INFINITY ? 1.f : ex2_approx(reference(m0) - reference(x0));
              const float a1 = PAIRED ? a0 : x1 == -INFINITY ? 1.f : ex2_approx(reference(m1) - reference(x1));
              l0 *= a0;
              l1 *= a1;
#pragma unroll
              for (int d = 0; d < COLUMNS / 8; ++d) {
                o[d][0] *= a0;
                o[d][1] *= a0;
                o[d][2] *= a1;
                o[d][3] *= a1;
              }
              m0 = x0;
              m1 = x1;
            }
            const float r0 = m0 == -INFINITY ? 0.f : reference(m0), r1 = m1 == -INFINITY ? 0.f : reference(m1);
            uint32_t p[UNITS][4];
#pragma unroll
            for (int j = 0; j < 2 * UNITS; ++j) {
              const float p0 = ex2_approx(s[j][0] - r0), p1 = ex2_approx(s[j][1] - r0);
              l0 += p0 + p1;
              if (PAIRED) {
                split2<BF16>(p0, p1, p[j >> 1][2 * (j & 1)], p[j >> 1][2 * (j & 1) + 1]);
              } else {
                const float p2 = ex2_approx(s[j][2] - r1), p3 = ex2_approx(s[j][3] - r1);
                l1 += p2 + p3;
                p[j >> 1][2 * (j & 1)] = pack2<BF16>(p0, p1);
                p[j >> 1][2 * (j & 1) + 1] = pack2<BF16>(p2, p3);
              }
            }
            if (least < 16) {                        // rows of V that take no part: zeros
#pragma unroll
              for (int u = 0; u < UNITS; ++u)
                if (lane >= info[u].y && lane < 16)
#pragma unroll
                  for (int pn = 0; pn < PANELS; ++pn)
#pragma unroll
                    for (int c = 0; c < 8; ++c) st_shared_v4(v_at + unit_at[u] + pn * piece_panel + (uint32_t)lane * 128u + c * 16u, 0u, 0u, 0u, 0u);
              fence_proxy_async();
              __syncwarp();
            }
#pragma unroll
            for (int c = 0; c < COLUMNS / 16; ++c) {
              const uint32_t col = (uint32_t)(c & 3) * 2u + v_col;
#pragma unroll
              for (int u = 0; u < UNITS; ++u) {
                uint32_t f[4];
                ldmatrix4_t(v_at + unit_at[u] + ((uint32_t)(c >> 2) + o_panel) * piece_panel + v_row * 128u + ((col ^ (v_row & 7u)) << 4), f);
                mma16816<BF16>(o[2 * c], p[u], f[0], f[1]);
                mma16816<BF16>(o[2 * c + 1], p[u], f[2], f[3]);
              }
            }
          }
          if (hidden != 0 && P.weights != nullptr && t4 == 0) {      // keys on a page that does not exist: no weight
#pragma unroll
            for (int u = 0; u < UNITS; ++u)
              for (int key = 0; key < info[u].z; ++key) {
                if (score0 != nullptr) score0[info[u].x + key] = -INFINITY;
                if (score1 != nullptr) score1[info[u].x + key] = -INFINITY;
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
      // Up to 8 heads: rows 0-7 of each warp, 128 columns (or all) at a time; else 16 rows, 64 columns.  Nobody waits but for the writers: 1.3 us a
      // row, 4.6 with one meeting before and one after every exchange of 64 columns.
      if (HALVES) part_read();                       // Q
      if (PAIRED) {
#pragma unroll
        for (int i = 0; i < COLUMNS / 8; ++i)
#pragma unroll
          for (int e = 0; e < 2; ++e) {              // (an infinite value times a rest that is zero or negative: the first term alone is right)
            const float both = o[i][e] + o[i][2 + e];
            o[i][e] = both == both ? both : o[i][e];
          }
      }
      const bool few = PAIRED || heads <= 8;
      const int width = few && COLUMNS >= 128 ? 128 : 64, rows = few ? 8 : 16;
      const long long part_slot = 2ll * blockIdx.x + max(r.slot, 0);
      for (int c0 = 0; c0 < COLUMNS; c0 += width) {
        if (!(ok = part_writable())) break;
        if (t4 == 0) {
          *reinterpret_cast<float2*>(ctl->ml[warp][g]) = make_float2(reference(m0), l0);
          if (!PAIRED) *reinterpret_cast<float2*>(ctl->ml[warp][g + 8]) = make_float2(reference(m1), l1);
        }
#pragma unroll
        for (int i = 0; i < COLUMNS / 8; ++i) {
          if (i * 8 < c0 || i * 8 >= c0 + width) continue;
          float* to = part + (warp * rows + g) * width + ((i - c0 / 8) ^ g) * 8 + t4 * 2;        // groups of 8 columns swapped by row: no bank conflicts
          *reinterpret_cast<float2*>(to) = make_float2(o[i][0], o[i][1]);
          if (!few) *reinterpret_cast<float2*>(to + 8 * width) = make_float2(o[i][2], o[i][3]);
        }
        if (!(ok = part_written())) break;
        // item = (head, 4 columns); `all`: both 16 heads, or both halves of the columns
        const int quads = width / 4, items = (all ? 2 : 1) * rows * quads;
        for (int item = tid; item < items; item += kConsumers * 32) {
          const int col = item % quads * 4, hl = item / quads % rows, hh = item / quads / rows;
          const int head = HALVES ? hl : hh * 16 + hl, d = (HALVES ? hh * COLUMNS : 0) + c0 + col;
          const int w0 = hh * 4, n_w = all ? 4 : kConsumers;
          if (head >= heads) continue;
          float mt = -INFINITY, lt = 0.f;
          float2 ml[kConsumers];
#pragma unroll
          for (int w = 0; w < kConsumers; ++w) {
            ml[w] = w < n_w ? *reinterpret_cast<const float2*>(ctl->ml[w0 + w][hl]) : make_float2(-INFINITY, 0.f);
            mt = fmaxf(mt, ml[w].x);
          }
          float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
          for (int w = 0; w < kConsumers; ++w) {
            if (w >= n_w) break;
            const float4 y = *reinterpret_cast<const float4*>(part + ((w0 + w) * rows + hl) * width + (((col >> 3) ^ (hl & 7)) << 3) + (col & 7));
            const float f = ml[w].x == -INFINITY ? 0.f : ex2_approx(ml[w].x - mt);
            x.x = fmaf(y.x, f, x.x);
            x.y = fmaf(y.y, f, x.y);
            x.z = fmaf(y.z, f, x.z);
            x.w = fmaf(y.w, f, x.w);
            lt += ml[w].x == -INFINITY ? ml[w].y : ml[w].y * f;      // (a sum of NaN stays one)
          }
          if (r.slot >= 0) {
            *reinterpret_cast<float4*>(P.sp.part_o + (part_slot * kDecodeHeads + head) * D + d) = x;
            if (d == 0) *reinterpret_cast<float2*>(P.sp.part_ml + (part_slot * kDecodeHeads + head) * 2) = make_float2(mt, lt);
          } else {
            const bool none = mt == -INFINITY && lt == 0.f;
            const float inv = none ? 0.f : 1.f / lt;
            if (d < P.headdim)
              *reinterpret_cast<uint2*>(static_cast<T*>(P.o) + r.b * P.o_s[0] + (head0 + head) * P.o_s[1] + d) =
                  none ? make_uint2(0u, 0u) : make_uint2(pack2<BF16>(x.x * inv, x.y * inv), pack2<BF16>(x.z * inv, x.w * inv));
            if (d == 0 && P.lse != nullptr)
              P.lse[(long long)r.b * P.nhead_q + head0 + head] = none ? -INFINITY : (mt + log2f(lt)) * kDecodeLn2;
          }
        }
        part_read();
      }
      if (!ok) break;
      __syncwarp();
      if (lane == 0) mbar_arrive(b_row_done + 8 * (n_rows & 1));
      ++n_rows;
    }
  }
  __syncthreads();
  decode_fill_empty<T>(P, blockIdx.x, P.grid);
  for (int b = blockIdx.x * kThreads + tid; b < P.batch; b += P.grid * kThreads)
    if (P.lens[b] < 0 || P.lens[b] > P.capacity) atomicMax(&ctl->bad, P.batch - b);
  __syncthreads();
  if (tid == 0) {
    const int bad = ctl->bad;
    decode_note_status(P, ctl->abort_flag != 0 ? (int)HBSA_STATUS_WAIT_LIMIT : bad != 0 ? (int)HBSA_STATUS_CACHE_BOUNDS : (int)HBSA_STATUS_OK, P.batch - bad);
  }
}

// 5-D map over the pages of a cache: dims (columns, slots, panels, heads, pages), box (64, unit, panels, 1, 1).  Head dimensions that are no
// multiple of 64 are one panel of headdim columns, so that the hardware fills the columns behind them with zeros.
// The L2 fetches no more than what lies together of a kv-head: with 64 columns and heads inside the slots (128 bytes a row), fetches of
// 256 bytes brought the next head along (16 x 24576 keys, 8 heads: 198 us, 128 bytes as below: 160 us).
bool encode_cache_map(EncodeTiledFn fn, CUtensorMap* map, bool bf16, const void* base, const DecodeParams& P, const long long* s) {
  const int panels = P.one_box ? P.headdim / 64 : 1;
  cuuint64_t dims[5] = {(cuuint64_t)(P.one_box ? 64 : P.headdim), (cuuint64_t)P.page, (cuuint64_t)panels, (cuuint64_t)P.nhead_k, (cuuint64_t)P.num_pages};
  cuuint64_t strides[4] = {(cuuint64_t)s[1] * 2ull, 128ull, (cuuint64_t)s[2] * 2ull, (cuuint64_t)s[0] * 2ull};
  const long long run = (s[1] == P.headdim ? 2ll * P.page : 2ll) * P.headdim;
  const CUtensorMapL2promotion promotion = run >= 256 ? CU_TENSOR_MAP_L2_PROMOTION_L2_256B : run >= 128 ? CU_TENSOR_MAP_L2_PROMOTION_L2_128B : CU_TENSOR_MAP_L2_PROMOTION_L2_64B;
  cuuint32_t box[5] = {64u, (cuuint32_t)P.unit, P.one_box ? (cuuint32_t)(P.d_pad / 64) : 1u, 1u, 1u}, estr[5] = {1u, 1u, 1u, 1u, 1u};
  return fn(map, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 5, const_cast<void*>(base), dims, strides, box, estr,
            CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, promotion, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <int D, bool BF16, bool PAIRED>
cudaError_t launch_one(const CUtensorMap& tk, const CUtensorMap& tv, const DecodeParams& P, bool dependent, cudaStream_t stream) {
  static SmemOptIn opt_in;
  cudaError_t e = opt_in.once(reinterpret_cast<const void*>(decode_sm100_kernel<D, BF16, PAIRED>), (int)decode_smem<D>());
  if (e != cudaSuccess) return e;
  return launch_kernel(decode_sm100_kernel<D, BF16, PAIRED>, (unsigned)P.grid, kThreads, decode_smem<D>(), dependent, stream, tk, tv, P);
}

template <int D, bool BF16>
cudaError_t launch_heads(const CUtensorMap& tk, const CUtensorMap& tv, const DecodeParams& P, bool dependent, cudaStream_t stream) {
  return P.chunk_heads <= 8 ? launch_one<D, BF16, true>(tk, tv, P, dependent, stream) : launch_one<D, BF16, false>(tk, tv, P, dependent, stream);
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
  if (P.d_pad == 64) e = bf16 ? launch_heads<64, true>(tk, tv, P, dependent, stream) : launch_heads<64, false>(tk, tv, P, dependent, stream);
  else if (P.d_pad == 128) e = bf16 ? launch_heads<128, true>(tk, tv, P, dependent, stream) : launch_heads<128, false>(tk, tv, P, dependent, stream);
  else e = bf16 ? launch_heads<256, true>(tk, tv, P, dependent, stream) : launch_heads<256, false>(tk, tv, P, dependent, stream);
  if (e != cudaSuccess) { *err_text = cudaGetErrorString(e); return (int)e; }
  return 0;
}

}  // namespace hbsa
