// What the kernels of the paged decode attention share: the description of a call, the split of its work, and the layout of
// the partial results.
//
// One row = one (sequence, kv-head, chunk of at most 32 q-heads of its group).  A row's keys come in tiles of 64; without a
// block mask tile i holds positions 64 i .. 64 i + 63, with one the tile is strung together from pieces of `unit` positions of the
// active blocks.  The tiles of all rows stand in one line (sequence, kv-head, chunk, tile), which is cut into runs of the same
// length, up to one tile: every CTA reads the same number of keys, whatever the lengths are, and at most its first and its
// last row are shared with neighbours.  Those leave (maximum, sum, unnormalised output) in two slots of the CTA's own, which the
// join kernel puts together in the order of the CTAs, so that results do not depend on timing.
// Without a mask two neighbouring kv-heads (`lanes`; one where their number is odd) are worked on side by side: the line holds
// every other kv-head, and the CTAs lanes * c .. take run c of it, one kv-head each, so that what lies together in memory is read
// at the same time (16 x 24576 keys, 8 heads inside the slots: of 64 157 us with one lane, 133 with two and with four; of 128
// 130 us with any).
#pragma once
#include "hbsa_common.cuh"

namespace hbsa {

constexpr int kDecodeTile = 64;          // keys of a tile
constexpr int kDecodeHeads = 32;         // q-heads of a row, at most
constexpr float kDecodeLog2e = 1.4426950408889634f;
constexpr float kDecodeLn2 = 0.6931471805599453f;

// Carved out of the caller's workspace; all pointers device pointers, each part 256-byte aligned.
struct DecodeSpace {
  int32_t* status;           // [kStatusWords], written by the join kernel
  int32_t* cta_status;       // [G][2] what CTA c has to report: HBSA_STATUS_*, sequence
  int4* cta_start;           // [G] of the CTA's first row {sequence, kv-head / lanes * n_chunk + chunk, its tiles before the CTA's first, its tiles}
  int32_t* cta_join;         // [G] 0, or, where the CTA's first row began with the CTA before: 2 * parts of the row + slot of the first one
  long long* total;          // [1] tiles of the line
  int32_t* pieces;           // [batch * nhead_k] pieces of the active blocks (mask)
  int32_t* list;             // [batch * nhead_k][num_k_block] the active blocks, ascending (mask)
  float* lse;                // [batch, nhead_q] (weights, where the caller wants no lse)
  float* part_ml;            // [2 G][kDecodeHeads][2] what the part is relative to (log2 domain: its maximum, in fp16 14 less) and its sum
  float* part_o;             // [2 G][kDecodeHeads][d_pad]
  float* scores;             // [batch, nhead_q, capacity] scaled scores in the log2 domain (weights)
};

struct DecodeParams {
  DecodeSpace sp;
  const void *k, *v, *q;
  void* o;
  long long k_s[4], v_s[4], q_s[3], o_s[3];
  const int32_t* table;
  long long table_stride;
  const int32_t* lens;
  const uint8_t* mask;
  long long mask_s[3];
  float* lse;                // the caller's, or the workspace's, or NULL
  float* weights;
  long long weights_s[2];
  FastDiv page_div;
  int num_pages, page, capacity, batch, nhead_q, nhead_k, group, headdim, d_pad;
  int n_chunk, chunk_heads;  // chunks of a group, q-heads of every chunk but perhaps the last
  int kbs, num_k_block;
  int unit, pieces_per_block;
  int one_box;               // tensor-core kernel: one copy brings all columns of a piece
  int entries;
  float scale_log2;
  long long wait_budget;
  int debug_stall;
  int grid, lanes, runs;     // G = lanes * runs
};

// The cut of `total` tiles into `grid` runs: the first `rem` have base + 1 tiles, the others base.
struct DecodeCut {
  long long base;
  int rem;
  __device__ __forceinline__ DecodeCut(long long total, int grid) : base(quotient(total, grid)), rem((int)(total - base * grid)) {}
  __device__ __forceinline__ long long first(int c) const { return c * base + min(c, rem); }
  __device__ __forceinline__ int tiles(int c) const { return (int)base + (c < rem ? 1 : 0); }
  // the run that has tile t
  __device__ __forceinline__ int owner(long long t) const {
    const long long front = rem * (base + 1);
    return t < front ? (int)quotient(t, base + 1) : rem + (int)quotient(t - front, base);
  }
};

__device__ __forceinline__ int decode_len(const DecodeParams& P, int b) { return max(0, min(P.lens[b], P.capacity)); }
// Tiles of one row of entry e.
__device__ __forceinline__ int decode_row_tiles(const DecodeParams& P, int e) {
  if (P.mask == nullptr) return (decode_len(P, e) + kDecodeTile - 1) / kDecodeTile;
  return (int)(((long long)P.sp.pieces[e] * P.unit + kDecodeTile - 1) / kDecodeTile);
}
__device__ __forceinline__ int decode_entry_rows(const DecodeParams& P) { return P.mask == nullptr ? P.nhead_k / P.lanes * P.n_chunk : P.n_chunk; }

// One row, and the tiles of it that a CTA works on.
struct DecodeRow {
  int b, hk, chunk;          // b < 0: no more work
  int tile0, tiles, row_tiles;
  int slot;                  // partial slot of the CTA (0, 1), or -1: the row is the CTA's alone
  int len, pieces, entry;
};

// A place on the line of tiles: the entry (a sequence, or a (sequence, kv-head) where there is a mask) and its first tile.
struct DecodeWalk {
  long long start, end, entry_start, total;
  int entry;
};
// Finds the place at which a CTA's run starts; all threads of the block call it.  `scratch`: shared, one word per warp.
__device__ __forceinline__ void decode_locate(const DecodeParams& P, DecodeWalk* walk, long long* scratch) {
  const int tid = threadIdx.x, n_threads = blockDim.x, lane = tid & 31, warp = tid >> 5, n_warps = (n_threads + 31) >> 5;
  const int rows = decode_entry_rows(P);
  const int per = (P.entries + n_threads - 1) / n_threads, e0 = min(per * tid, P.entries), e1 = min(e0 + per, P.entries);
  long long sum = 0;
  for (int e = e0; e < e1; ++e) sum += (long long)decode_row_tiles(P, e) * rows;
  long long incl = sum;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const long long y = __shfl_up_sync(0xffffffffu, incl, d);
    if (lane >= d) incl += y;
  }
  if (lane == 31) scratch[warp] = incl;
  __syncthreads();
  long long before = 0, total = 0;
  for (int w = 0; w < n_warps; ++w) {
    if (w < warp) before += scratch[w];
    total += scratch[w];
  }
  before += incl - sum;
  const DecodeCut cut(total, P.runs);
  const int run = blockIdx.x / P.lanes;
  const long long start = cut.first(run), end = start + cut.tiles(run);
  if (tid == 0) {
    walk->start = start;
    walk->end = end;
    walk->total = total;
    if (blockIdx.x == 0) *P.sp.total = total;
    if (start == end) {
      P.sp.cta_start[blockIdx.x] = make_int4(-1, 0, 0, 0);
      P.sp.cta_join[blockIdx.x] = 0;
    }
  }
  if (start < end && start >= before && start < before + sum) {
    long long at = before;
    for (int e = e0; e < e1; ++e) {
      const long long n = (long long)decode_row_tiles(P, e) * rows;
      if (start >= at && start < at + n) {
        walk->entry = e;
        walk->entry_start = at;
      }
      at += n;
    }
  }
  __syncthreads();
}

// The row of CTA `cta` that holds tile t, and as much of it as lies before `end`; moves `walk` on to the row's entry.
__device__ __forceinline__ DecodeRow decode_row_at(const DecodeParams& P, DecodeWalk& walk, long long t, int cta) {
  DecodeRow r;
  const int rows = decode_entry_rows(P);
  int tiles = decode_row_tiles(P, walk.entry);
  while (t >= walk.entry_start + (long long)tiles * rows) {      // t < end <= total: there is such an entry
    walk.entry_start += (long long)tiles * rows;
    tiles = decode_row_tiles(P, ++walk.entry);
  }
  const int in_entry = (int)quotient(t - walk.entry_start, tiles);
  const long long row0 = walk.entry_start + (long long)in_entry * tiles;
  r.entry = walk.entry;
  r.b = P.mask == nullptr ? walk.entry : walk.entry / P.nhead_k;
  r.hk = P.mask == nullptr ? in_entry / P.n_chunk * P.lanes + cta % P.lanes : walk.entry % P.nhead_k;
  r.chunk = in_entry % P.n_chunk;
  r.row_tiles = tiles;
  r.tile0 = (int)(t - row0);
  r.tiles = (int)(min(walk.end, row0 + tiles) - t);
  r.len = decode_len(P, r.b);
  r.pieces = P.mask == nullptr ? 0 : P.sp.pieces[walk.entry];
  r.slot = r.tiles == tiles ? -1 : t == walk.start ? 0 : 1;
  return r;
}

// Position of piece p of a row with a mask, or -1 behind the last.
__device__ __forceinline__ int decode_piece_position(const DecodeParams& P, const DecodeRow& r, int p) {
  if (p >= r.pieces) return -1;
  return P.sp.list[(long long)r.entry * P.num_k_block + p / P.pieces_per_block] * P.kbs + p % P.pieces_per_block * P.unit;
}

// The output of sequences that see no key: zeros, lse -inf.  All threads of CTA `cta` of `grid`.
template <typename T>
__device__ __forceinline__ void decode_fill_empty(const DecodeParams& P, int cta, int grid) {
  const int heads = P.mask == nullptr ? P.nhead_q : P.group;
  for (int e = cta; e < P.entries; e += grid) {
    if (decode_row_tiles(P, e) != 0) continue;
    const int b = P.mask == nullptr ? e : e / P.nhead_k, h0 = P.mask == nullptr ? 0 : e % P.nhead_k * P.group;
    for (int i = threadIdx.x; i < heads * P.headdim; i += blockDim.x)
      static_cast<T*>(P.o)[b * P.o_s[0] + (h0 + i / P.headdim) * P.o_s[1] + i % P.headdim * P.o_s[2]] = T(0.f);
    if (P.lse != nullptr)
      for (int i = threadIdx.x; i < heads; i += blockDim.x) P.lse[(long long)b * P.nhead_q + h0 + i] = -INFINITY;
  }
}

// A row of the line of tiles that several runs share: its first part is that of run c0, and there are n.
struct DecodeParts {
  int c0, n, slot0, lanes, lane;
  __device__ __forceinline__ DecodeParts(const DecodeCut& cut, long long row0, int row_tiles, int lanes, int lane)
      : c0(cut.owner(row0)), n(cut.owner(row0 + row_tiles - 1) - c0 + 1), slot0(cut.first(c0) == row0 ? 0 : 1), lanes(lanes), lane(lane) {}
  __device__ __forceinline__ long long at(int i) const { return 2ll * ((c0 + i) * lanes + lane) + (i == 0 ? slot0 : 0); }
};

// What every CTA of the main kernel writes down for the join: its first row, and, once its work is under way, what there is to join.
__device__ __forceinline__ void decode_note_start(const DecodeParams& P, const DecodeRow& r) {
  P.sp.cta_start[blockIdx.x] = make_int4(r.b, r.hk / P.lanes * P.n_chunk + r.chunk, r.tile0, r.row_tiles);
}

__device__ __forceinline__ void decode_note_join(const DecodeParams& P, const DecodeWalk& walk) {
  if (walk.start == walk.end) return;
  const int4 st = P.sp.cta_start[blockIdx.x];              // this thread's own
  int info = 0;
  if (st.z != 0) {
    const int run = blockIdx.x / P.lanes, lane = blockIdx.x - run * P.lanes;
    const DecodeParts parts(DecodeCut(walk.total, P.runs), walk.start - st.z, st.w, P.lanes, lane);
    if (run == parts.c0 + 1) info = 2 * parts.n + parts.slot0;
  }
  P.sp.cta_join[blockIdx.x] = info;
}

__device__ __forceinline__ void decode_note_status(const DecodeParams& P, int status, int sequence) {
  P.sp.cta_status[2 * blockIdx.x] = status;
  P.sp.cta_status[2 * blockIdx.x + 1] = sequence;
}

__device__ __forceinline__ void pdl_wait() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void pdl_launch() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }

const char* decode_sm100_ineligible_reason(const hbsa_paged_attention_args& a, float scale);
// The main kernel: every row that one CTA has alone is written, the others leave their parts.
bool decode_f32_eligible(const hbsa_paged_attention_args& a);
cudaError_t launch_decode_f32(const DecodeParams& P, bool dependent, cudaStream_t stream);
cudaError_t launch_decode_generic(const DecodeParams& P, int dtype, bool dependent, cudaStream_t stream);
int launch_decode_sm100(const DecodeParams& P, const hbsa_paged_attention_args& a, bool dependent, cudaStream_t stream, const char** err_text);

// Launch with programmatic stream serialization where `dependent`.
template <typename... K, typename... A>
cudaError_t launch_kernel(void (*kernel)(K...), unsigned grid, unsigned block, size_t smem, bool dependent, cudaStream_t stream, const A&... args) {
  cudaLaunchAttribute attr[1] = {};
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(grid);
  cfg.blockDim = dim3(block);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cfg.attrs = attr;
  cfg.numAttrs = dependent ? 1 : 0;
  return cudaLaunchKernelEx(&cfg, kernel, args...);
}

}  // namespace hbsa
