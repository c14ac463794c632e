// Attention of one new token per sequence over a paged key-value cache: everything but the tensor-core main kernel
// (hbsa_decode_sm100.cu) and the one for fp32 (hbsa_decode_f32.cu).  For every sequence b and q-head h, over the positions j < len_b in active blocks:
//     x_j = scale * q . k_j        o = sum_j exp(x_j - lse) v_j        lse = ln sum_j exp x_j
// and, where wanted, weights[b, kv-head, j] += sum over the heads of the group of exp(x_j - lse).
//
// Two or three kernels (without a mask 10.5 us for a call that reads next to nothing, with one 13), each started while the one before it still runs (programmatic launches):
//   decode_blocks   with a block mask: the list of active blocks of every (sequence, kv-head)
//   main            one pass over K and V with the running maximum and sum of the softmax, split as hbsa_decode.cuh says
//   decode_join     rows that several CTAs have worked on; the weights: exp(score - lse), summed over the group, from the scores that the
//                   main kernel has left (4 bytes per key and q-head, against 4 d bytes per key and kv-head of K and V in 16
//                   bits; reading K again would add half of the traffic); the status words
#include <string.h>

#include "hbsa_decode.cuh"
#include "sm100_common.cuh"

namespace hbsa {

namespace {

// One warp per (sequence, kv-head): its active blocks below the sequence's length, and how many pieces of `unit` positions they
// have (the last block of the sequence may be short).
__global__ void __launch_bounds__(256) decode_blocks_kernel(const __grid_constant__ DecodeParams P) {
  pdl_launch();
  const int row = blockIdx.x * 8 + (threadIdx.x >> 5), lane = threadIdx.x & 31;
  if (row >= P.batch * P.nhead_k) return;
  const int b = row / P.nhead_k, hk = row % P.nhead_k, len = decode_len(P, b);
  const int n = len == 0 ? 0 : min((len - 1) / P.kbs + 1, P.num_k_block);
  const uint8_t* m = P.mask + b * P.mask_s[0] + hk * P.mask_s[1];
  int32_t* list = P.sp.list + (long long)row * P.num_k_block;
  int count = 0;
  bool last = false;
  for (int base = 0; base < n; base += 512) {          // sixteen loads in flight
    bool on[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const int j = base + 32 * i + lane;
      on[i] = j < n && m[j * P.mask_s[2]] != 0;
    }
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const int j = base + 32 * i + lane;
      const uint32_t bal = __ballot_sync(0xffffffffu, on[i]);
      if (on[i]) list[count + __popc(bal & ((1u << lane) - 1u))] = j;
      last |= on[i] && j == n - 1;
      count += __popc(bal);
    }
  }
  last = __any_sync(0xffffffffu, last);
  int pieces = count * P.pieces_per_block;
  if (last) pieces -= P.pieces_per_block - (len - (n - 1) * P.kbs + P.unit - 1) / P.unit;
  if (lane == 0) P.sp.pieces[row] = pieces;
}

// ------------------------------------------------------------------------------------------------------------------
// Main kernel for what the other two do not take: odd strides, page sizes and head dimensions, any type.  A tile of 64 keys is staged in shared
// memory as fp32; thread (key, head mod 4) forms the scores, a warp per head the softmax, thread (dims, heads) adds P V in registers.
// Bound by the way through a tile (five meetings): 8 x 8192..16384 fp32 keys, 8 heads of 128, groups of 4: 490 us, 1.6 TB/s.
constexpr int kGenThreads = 256;

struct DecodeGenericShared {
  DecodeWalk walk;
  long long scratch[8];
  long long k_at[kDecodeTile], v_at[kDecodeTile];      // element offset of every key's row; < 0: no such key
  int pos[kDecodeTile];                                // position in the sequence, or -1
  float m[kDecodeHeads], l[kDecodeHeads], alpha[kDecodeHeads];
  int bad;                                             // the first sequence with a length or a page out of range, from the end (0: none)
};

template <int DP> constexpr size_t generic_smem() {
  return sizeof(float) * (size_t)(kDecodeHeads * DP + kDecodeTile * (DP + 4) + kDecodeTile * DP + kDecodeHeads * kDecodeTile);
}

template <typename T, int DP, int VEC>
__global__ void __launch_bounds__(kGenThreads) decode_generic_kernel(const __grid_constant__ DecodeParams P) {
  constexpr int KS = DP + 4;                           // rows of K 4 floats apart modulo 32: 16-byte reads of 8 keys hit all banks
  constexpr int QUADS = DP / 4, HGROUPS = kGenThreads / QUADS, HPT = kDecodeHeads / HGROUPS;
  extern __shared__ __align__(16) float gsm[];
  float* const sQ = gsm;                               // [kDecodeHeads][DP]
  float* const sK = sQ + kDecodeHeads * DP;            // [tile][KS]
  float* const sV = sK + kDecodeTile * KS;             // [tile][DP]
  float* const sP = sV + kDecodeTile * DP;             // [kDecodeHeads][tile]
  __shared__ DecodeGenericShared sh;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  if (tid == 0) sh.bad = 0;
  pdl_wait();                                          // the block lists
  decode_locate(P, &sh.walk, sh.scratch);
  pdl_launch();
  DecodeWalk walk = sh.walk;
  decode_fill_empty<T>(P, blockIdx.x, P.grid);
  for (int b = blockIdx.x * kGenThreads + tid; b < P.batch; b += P.grid * kGenThreads)
    if (P.lens[b] < 0 || P.lens[b] > P.capacity) atomicMax(&sh.bad, P.batch - b);
  const T* const K = static_cast<const T*>(P.k);
  const T* const V = static_cast<const T*>(P.v);

  if (P.headdim < DP) {                                // the columns beyond headdim stay zero
    for (int i = tid; i < kDecodeTile * KS; i += kGenThreads) sK[i] = 0.f;
    for (int i = tid; i < kDecodeTile * DP; i += kGenThreads) sV[i] = 0.f;
  }
  for (long long t = walk.start; t < walk.end;) {
    const DecodeRow r = decode_row_at(P, walk, t, blockIdx.x);
    if (t == walk.start && tid == 0) decode_note_start(P, r);
    t += r.tiles;
    const int head0 = r.hk * P.group + r.chunk * P.chunk_heads;
    const int heads = min(P.chunk_heads, P.group - r.chunk * P.chunk_heads);
    // threads 0-63: position and place of a key of the tile, found while the tile before is worked on
    int pos = -1, page = 0, slot = 0;
    auto look_up = [&](int tile) {
      if (tid >= kDecodeTile) return;
      pos = tile * kDecodeTile + tid;
      if (P.mask != nullptr) {
        pos = decode_piece_position(P, r, pos / P.unit);
        if (pos >= 0) pos += tid % P.unit;
      }
      if (pos >= r.len) pos = -1;
      if (pos >= 0) {
        const int i = pos / P.page;
        page = P.table[r.b * P.table_stride + i];
        slot = pos - i * P.page;
      }
    };
    look_up(r.tile0);
    __syncthreads();
    for (int i = tid; i < (heads + 1) / 2 * 2 * DP; i += kGenThreads) {
      const int h = i / DP, d = i % DP;
      sQ[i] = h < heads && d < P.headdim ? to_f(static_cast<const T*>(P.q)[r.b * P.q_s[0] + (head0 + h) * P.q_s[1] + d * P.q_s[2]]) : 0.f;
    }
    if (tid < kDecodeHeads) {
      sh.m[tid] = -INFINITY;
      sh.l[tid] = 0.f;
    }
    float acc[HPT][4];
#pragma unroll
    for (int h = 0; h < HPT; ++h)
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[h][e] = 0.f;
    const int quad = tid % QUADS, hg = tid / QUADS;
    for (int tile = r.tile0; tile < r.tile0 + r.tiles; ++tile) {
      __syncthreads();                                 // the tile before is used up
      if (tid < kDecodeTile) {
        long long k_at = -1, v_at = -1;
        if (pos >= 0) {
          if (page >= 0 && page < P.num_pages) {
            k_at = page * P.k_s[0] + slot * P.k_s[1] + r.hk * P.k_s[2];
            v_at = page * P.v_s[0] + slot * P.v_s[1] + r.hk * P.v_s[2];
          } else {
            atomicMax(&sh.bad, P.batch - r.b);
          }
        }
        sh.pos[tid] = pos;
        sh.k_at[tid] = k_at;
        sh.v_at[tid] = v_at;
      }
      if (tile + 1 < r.tile0 + r.tiles) look_up(tile + 1);
      __syncthreads();
      const int vecs = P.headdim / VEC;
#pragma unroll 4
      for (int i = tid; i < kDecodeTile * vecs; i += kGenThreads) {
        const int key = i / vecs, d = (i - key * vecs) * VEC;
        const long long ka = sh.k_at[key], va = sh.v_at[key];
        if (VEC > 1) {
          union { uint4 w; T x[16 / sizeof(T)]; } a, b;
          a.w = b.w = make_uint4(0, 0, 0, 0);
          if (ka >= 0) {
            a.w = *reinterpret_cast<const uint4*>(K + ka + d);
            b.w = *reinterpret_cast<const uint4*>(V + va + d);
          }
#pragma unroll
          for (int e = 0; e < VEC; ++e) {
            sK[key * KS + d + e] = to_f(a.x[e]);
            sV[key * DP + d + e] = to_f(b.x[e]);
          }
        } else {
          sK[key * KS + d] = ka >= 0 ? to_f(K[ka + d * P.k_s[3]]) : 0.f;
          sV[key * DP + d] = ka >= 0 ? to_f(V[va + d * P.v_s[3]]) : 0.f;
        }
      }
      __syncthreads();
      // scores: thread = (key, every fourth pair of heads)
      {
        const int key = tid & 63, at = sh.pos[key];
        const bool there = sh.k_at[key] >= 0;
        const float4* kr = reinterpret_cast<const float4*>(sK + key * KS);
        for (int h = 2 * (tid >> 6); h < heads; h += 8) {
          const float4 *qa = reinterpret_cast<const float4*>(sQ + h * DP), *qb = reinterpret_cast<const float4*>(sQ + (h + 1) * DP);
          float s0 = 0.f, s1 = 0.f;
#pragma unroll 8
          for (int i = 0; i < DP / 4; ++i) {
            const float4 x = kr[i], a = qa[i], c = qb[i];
            s0 = fmaf(x.x, a.x, fmaf(x.y, a.y, fmaf(x.z, a.z, fmaf(x.w, a.w, s0))));
            s1 = fmaf(x.x, c.x, fmaf(x.y, c.y, fmaf(x.z, c.z, fmaf(x.w, c.w, s1))));
          }
          s0 = there ? s0 * P.scale_log2 : -INFINITY;
          s1 = there ? s1 * P.scale_log2 : -INFINITY;
          sP[h * kDecodeTile + key] = s0;
          sP[(h + 1) * kDecodeTile + key] = s1;
          if (P.weights != nullptr && at >= 0) {
            float* to = P.sp.scores + ((long long)r.b * P.nhead_q + head0 + h) * P.capacity + at;
            to[0] = s0;
            if (h + 1 < heads) to[P.capacity] = s1;
          }
        }
      }
      __syncthreads();
      for (int h = warp; h < heads; h += kGenThreads / 32) {
        float* ps = sP + h * kDecodeTile;
        const float a = ps[lane], c = ps[lane + 32], m_old = sh.m[h];
        float mx = fmaxf(a, c);
#pragma unroll
        for (int s = 16; s > 0; s >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, s));
        mx = fmaxf(mx, m_old);
        const float ref = mx == -INFINITY ? 0.f : mx;
        const float p0 = exp2f(a - ref), p1 = exp2f(c - ref);
        float sum = p0 + p1;
#pragma unroll
        for (int s = 16; s > 0; s >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, s);
        ps[lane] = p0;
        ps[lane + 32] = p1;
        if (lane == 0) {
          const float alpha = exp2f(m_old - ref);
          sh.alpha[h] = alpha;
          sh.m[h] = mx;
          sh.l[h] = sh.l[h] * alpha + sum;
        }
      }
      __syncthreads();
#pragma unroll
      for (int h = 0; h < HPT; ++h) {
        const int head = hg + h * HGROUPS;
        if (head < heads) {
          const float alpha = sh.alpha[head];
#pragma unroll
          for (int e = 0; e < 4; ++e) acc[h][e] *= alpha;
        }
      }
#pragma unroll 4
      for (int key = 0; key < kDecodeTile; ++key) {
        const float4 x = *reinterpret_cast<const float4*>(sV + key * DP + quad * 4);
#pragma unroll
        for (int h = 0; h < HPT; ++h) {
          const int head = hg + h * HGROUPS;
          if (head < heads) {
            const float p = sP[head * kDecodeTile + key];
            acc[h][0] = fmaf(p, x.x, acc[h][0]);
            acc[h][1] = fmaf(p, x.y, acc[h][1]);
            acc[h][2] = fmaf(p, x.z, acc[h][2]);
            acc[h][3] = fmaf(p, x.w, acc[h][3]);
          }
        }
      }
    }
    // the row's result, or the CTA's part of it
#pragma unroll
    for (int h = 0; h < HPT; ++h) {
      const int head = hg + h * HGROUPS;
      if (head >= heads) continue;
      const float m = sh.m[head], l = sh.l[head];
      if (r.slot >= 0) {
        const long long slot = 2ll * blockIdx.x + r.slot;
        *reinterpret_cast<float4*>(P.sp.part_o + (slot * kDecodeHeads + head) * P.d_pad + quad * 4) = make_float4(acc[h][0], acc[h][1], acc[h][2], acc[h][3]);
        if (quad == 0) *reinterpret_cast<float2*>(P.sp.part_ml + (slot * kDecodeHeads + head) * 2) = make_float2(m, l);
      } else {
        const bool none = m == -INFINITY && l == 0.f;  // (a NaN score makes the sum NaN)
        const float inv = none ? 0.f : 1.f / l;
        T* o = static_cast<T*>(P.o) + r.b * P.o_s[0] + (head0 + head) * P.o_s[1];
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (quad * 4 + e < P.headdim) o[(quad * 4 + e) * P.o_s[2]] = from_f<T>(none ? 0.f : acc[h][e] * inv);
        if (quad == 0 && P.lse != nullptr) P.lse[(long long)r.b * P.nhead_q + head0 + head] = none ? -INFINITY : (m + log2f(l)) * kDecodeLn2;
      }
    }
  }
  __syncthreads();
  if (tid == 0) decode_note_join(P, sh.walk);
  if (tid == 0) decode_note_status(P, sh.bad != 0 ? (int)HBSA_STATUS_CACHE_BOUNDS : (int)HBSA_STATUS_OK, P.batch - sh.bad);
}

// ------------------------------------------------------------------------------------------------------------------
constexpr int kJoinThreads = 256;
constexpr int kJoinMost = 1024;          // CTAs of the main kernel, at most

// CTA (c, part) of the weights: a quarter of the tiles that CTA c of the main kernel has worked on.  A quarter, because the way to the first
// position is a chain of loads, and few keys wait behind it: a call of 6 x 301..3001 keys, 8 heads, groups of 3 took 33.8, 29.5, 29.5 and 33.8 us
// with 1, 2, 4 and 8 parts.
constexpr int kWeightParts = 4;
__device__ __forceinline__ void add_weights(const DecodeParams& P, const DecodeCut& cut, const int4 st, int c, int part) {
  constexpr int WARPS = kJoinThreads / 32, EARLY = 8;
  __shared__ float s_lse[kJoinMost];     // of the group's heads, in the log2 domain
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  if (st.x < 0) return;
  DecodeWalk walk;
  const long long start = cut.first(c / P.lanes), n_tiles = cut.tiles(c / P.lanes);
  walk.start = start;
  walk.end = start + n_tiles * (part + 1) / kWeightParts;
  const int hk0 = st.y / P.n_chunk, in_entry = P.mask == nullptr ? st.y : st.y % P.n_chunk;
  walk.entry = P.mask == nullptr ? st.x : st.x * P.nhead_k + hk0;
  walk.entry_start = start - st.z - (long long)in_entry * st.w;
  for (long long t = start + n_tiles * part / kWeightParts; t < walk.end;) {
    const DecodeRow r = decode_row_at(P, walk, t, c);
    const long long row0 = t - r.tile0, head0 = (long long)r.b * P.nhead_q + r.hk * P.group;
    t += r.tiles;
    if (r.chunk != 0) continue;          // the first chunk's tiles stand for the whole group
    float* const out = P.weights + r.b * P.weights_s[0] + r.hk * P.weights_s[1];
    for (int h0 = 0; h0 < P.group; h0 += kJoinMost) {
      const int heads = min(kJoinMost, P.group - h0), last = 2 * (r.tile0 + r.tiles);
      const float* const scores = P.sp.scores + (head0 + h0) * P.capacity;
      // half a tile per warp and go; the first one's numbers are on their way while the sums are put together, then the next one's
      int pos = -1;
      float old = 0.f, x[EARLY];
      auto fetch = [&](int i) {
        pos = -1;
        if (i < last) {
          pos = i * 32 + lane;
          if (P.mask != nullptr) {
            const int in = pos;
            pos = decode_piece_position(P, r, in / P.unit);
            if (pos >= 0) pos += in % P.unit;
          }
          if (pos >= r.len) pos = -1;
        }
        if (pos >= 0) {
          old = out[pos];
#pragma unroll
          for (int h = 0; h < EARLY; ++h)
            if (h < heads) x[h] = scores[(long long)h * P.capacity + pos];
        }
      };
      int i = 2 * r.tile0 + warp;
      fetch(i);
      __syncthreads();
      for (int h = warp; h < heads; h += WARPS) {
        const int chunk = (h0 + h) / P.chunk_heads, head = (h0 + h) % P.chunk_heads;
        const DecodeParts parts(cut, row0 + (long long)chunk * r.row_tiles, r.row_tiles, P.lanes, c % P.lanes);
        float lse;
        if (parts.n == 1) {
          lse = P.lse[head0 + h0 + h] * kDecodeLog2e;
        } else {
          float mx = -INFINITY, l = 0.f;
          for (int k = lane; k < parts.n; k += 32) mx = fmaxf(mx, P.sp.part_ml[(parts.at(k) * kDecodeHeads + head) * 2]);
#pragma unroll
          for (int s = 16; s > 0; s >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, s));
          const float ref = mx == -INFINITY ? 0.f : mx;
          for (int k = lane; k < parts.n; k += 32) {
            const float2 ml = *reinterpret_cast<const float2*>(P.sp.part_ml + (parts.at(k) * kDecodeHeads + head) * 2);
            l += exp2f(ml.x - ref) * ml.y;
          }
#pragma unroll
          for (int s = 16; s > 0; s >>= 1) l += __shfl_xor_sync(0xffffffffu, l, s);
          lse = mx == -INFINITY && l == 0.f ? -INFINITY : mx + log2f(l);
        }
        if (lane == 0) s_lse[h] = lse;
      }
      __syncthreads();
      for (; i < last; i += WARPS) {
        const int at = pos;
        float w = 0.f;
        const float before = old;
        if (at >= 0) {
#pragma unroll
          for (int h = 0; h < EARLY; ++h)
            if (h < heads && s_lse[h] != -INFINITY) w += exp2f(x[h] - s_lse[h]);
        }
        fetch(i + WARPS);
        if (at < 0) continue;
#pragma unroll 4
        for (int h = EARLY; h < heads; ++h) {
          const float lse = s_lse[h], y = scores[(long long)h * P.capacity + at];
          if (lse != -INFINITY) w += exp2f(y - lse);
        }
        out[at] = before + w;
      }
    }
  }
}

// Latency, from load to load: it ends 4 to 6 us after the main kernel, with weights 12 (6 x 301..3001 keys, 8 heads, groups of 3; of 14 warps a
// scheduler 4.1 wait at a meeting, 2.8 for global memory, 1.3 for shared).
// CTA (j, y): first the weights, then q-head y of the row whose second part is that of CTA j of the main kernel.  CTA (0, 0) writes the status words.
template <typename T>
__global__ void __launch_bounds__(kJoinThreads, 4) decode_join_kernel(const __grid_constant__ DecodeParams P) {
  __shared__ float s_f[kJoinMost];
  __shared__ float4 s_acc[kJoinThreads];
  __shared__ float s_red[2][kJoinThreads / 32];
  __shared__ int s_first;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, j = blockIdx.x, parts_y = P.weights != nullptr ? kWeightParts : 0;
  const int head = (int)blockIdx.y - parts_y;
  if (tid == 0) s_first = 0x7fffffff;
  pdl_wait();
  const int4 st = P.sp.cta_start[j];
  const int info = P.sp.cta_join[j];
  int codes = 0;
  for (int c = tid; c < P.grid; c += kJoinThreads) codes |= 1 << P.sp.cta_status[2 * c];
  const bool gave_up = __syncthreads_or(codes & (1 << HBSA_STATUS_WAIT_LIMIT)) != 0;
  if (j == 0 && blockIdx.y == 0) {
    const bool bounds = __syncthreads_or(codes & (1 << HBSA_STATUS_CACHE_BOUNDS)) != 0;
    if (bounds)
      for (int c = tid; c < P.grid; c += kJoinThreads)
        if (P.sp.cta_status[2 * c] == HBSA_STATUS_CACHE_BOUNDS) atomicMin(&s_first, P.sp.cta_status[2 * c + 1]);
    __syncthreads();
    if (tid < kStatusWords) {
      int w = 0;
      if (tid == 0) w = gave_up ? (int)HBSA_STATUS_WAIT_LIMIT : bounds ? (int)HBSA_STATUS_CACHE_BOUNDS : (int)HBSA_STATUS_OK;
      if (tid == 1 && !gave_up && bounds) w = s_first;
      P.sp.status[tid] = w;
    }
  }
  if (gave_up) {                         // nobody shall take the output for one
    const long long n = (long long)P.batch * P.nhead_q * P.headdim, step = (long long)gridDim.x * gridDim.y * kJoinThreads;
    for (long long i = ((long long)blockIdx.y * gridDim.x + j) * kJoinThreads + tid; i < n; i += step) {
      const long long row = i / P.headdim, b = row / P.nhead_q, h = row % P.nhead_q, d = i % P.headdim;
      static_cast<T*>(P.o)[b * P.o_s[0] + h * P.o_s[1] + d * P.o_s[2]] = from_f<T>(NAN);
      if (d == 0 && P.lse != nullptr) P.lse[row] = NAN;
    }
    return;
  }
  if (head < 0) {
    add_weights(P, DecodeCut(*P.sp.total, P.runs), st, j, (int)blockIdx.y);
    return;
  }
  if (info == 0) return;
  const int hk = st.y / P.n_chunk * P.lanes + j % P.lanes, chunk = st.y % P.n_chunk, n = info >> 1, slot0 = info & 1;
  if (head >= min(P.chunk_heads, P.group - chunk * P.chunk_heads)) return;
  auto slot_of = [&](int i) { return 2ll * (j + (i - 1) * P.lanes) + (i == 0 ? slot0 : 0); };

  // the outputs of the first parts are on their way while the factors are made
  const int quads = P.d_pad / 4, groups = kJoinThreads / quads, quad = tid % quads, g = tid / quads;
  auto part_of = [&](int i) { return *reinterpret_cast<const float4*>(P.sp.part_o + (slot_of(i) * kDecodeHeads + head) * P.d_pad + quad * 4); };
  constexpr int AHEAD = 4;
  float4 early[AHEAD];
#pragma unroll
  for (int e = 0; e < AHEAD; ++e) early[e] = g + e * groups < n ? part_of(g + e * groups) : make_float4(0.f, 0.f, 0.f, 0.f);
  auto ml_of = [&](int i) { return *reinterpret_cast<const float2*>(P.sp.part_ml + (slot_of(i) * kDecodeHeads + head) * 2); };
  float mx = -INFINITY;
  float2 first = make_float2(-INFINITY, 0.f);
  if (tid < n) first = ml_of(tid);
  for (int i = tid; i < n; i += kJoinThreads) mx = fmaxf(mx, i == tid ? first.x : ml_of(i).x);
#pragma unroll
  for (int s = 16; s > 0; s >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, s));
  if (lane == 0) s_red[0][warp] = mx;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kJoinThreads / 32; ++w) mx = fmaxf(mx, s_red[0][w]);
  const float ref = mx == -INFINITY ? 0.f : mx;
  float l = 0.f;
  for (int i = tid; i < n; i += kJoinThreads) {
    const float2 ml = i == tid ? first : ml_of(i);
    const float f = exp2f(ml.x - ref);
    l += f * ml.y;
    s_f[i] = f;
  }
#pragma unroll
  for (int s = 16; s > 0; s >>= 1) l += __shfl_xor_sync(0xffffffffu, l, s);
  if (lane == 0) s_red[1][warp] = l;
  __syncthreads();
  l = 0.f;
#pragma unroll
  for (int w = 0; w < kJoinThreads / 32; ++w) l += s_red[1][w];
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
  auto add = [&](float f, const float4 x) {
    acc.x = fmaf(f, x.x, acc.x);
    acc.y = fmaf(f, x.y, acc.y);
    acc.z = fmaf(f, x.z, acc.z);
    acc.w = fmaf(f, x.w, acc.w);
  };
#pragma unroll
  for (int e = 0; e < AHEAD; ++e)
    if (g + e * groups < n) add(s_f[g + e * groups], early[e]);
#pragma unroll 4
  for (int i = g + AHEAD * groups; i < n; i += groups) add(s_f[i], part_of(i));
  s_acc[tid] = acc;
  __syncthreads();
  const bool none = mx == -INFINITY && l == 0.f;
  const int hq = hk * P.group + chunk * P.chunk_heads + head;
  if (tid < P.headdim) {
    float x = 0.f;
    for (int i = 0; i < groups; ++i) x += reinterpret_cast<const float*>(s_acc)[i * P.d_pad + tid];
    static_cast<T*>(P.o)[st.x * P.o_s[0] + hq * P.o_s[1] + tid * P.o_s[2]] = from_f<T>(none ? 0.f : x / l);
  }
  if (tid == 0 && P.lse != nullptr) P.lse[(long long)st.x * P.nhead_q + hq] = none ? -INFINITY : (mx + log2f(l)) * kDecodeLn2;
}

template <typename T, int DP, int VEC>
cudaError_t launch_generic(const DecodeParams& P, bool dependent, cudaStream_t stream) {
  static SmemOptIn opt_in;
  cudaError_t e = opt_in.once(reinterpret_cast<const void*>(decode_generic_kernel<T, DP, VEC>), (int)generic_smem<DP>());
  if (e != cudaSuccess) return e;
  return launch_kernel(decode_generic_kernel<T, DP, VEC>, (unsigned)P.grid, kGenThreads, generic_smem<DP>(), dependent, stream, P);
}
template <typename T>
cudaError_t launch_generic_of(const DecodeParams& P, bool dependent, cudaStream_t stream) {
  constexpr int VEC = 16 / (int)sizeof(T);
  bool vec = P.headdim % VEC == 0 && P.k_s[3] == 1 && P.v_s[3] == 1 && (uintptr_t)P.k % 16 == 0 && (uintptr_t)P.v % 16 == 0;
  for (int i = 0; i < 3; ++i) vec = vec && P.k_s[i] % VEC == 0 && P.v_s[i] % VEC == 0;
  if (P.d_pad == 64) return vec ? launch_generic<T, 64, VEC>(P, dependent, stream) : launch_generic<T, 64, 1>(P, dependent, stream);
  if (P.d_pad == 128) return vec ? launch_generic<T, 128, VEC>(P, dependent, stream) : launch_generic<T, 128, 1>(P, dependent, stream);
  return vec ? launch_generic<T, 256, VEC>(P, dependent, stream) : launch_generic<T, 256, 1>(P, dependent, stream);
}

// The main kernel; the generic one where neither is set.
struct DecodeKind {
  bool sm100, f32;
};

size_t align256(size_t x) { return (x + 255) / 256 * 256; }

int gcd(int a, int b) {
  while (b != 0) {
    const int t = a % b;
    a = b;
    b = t;
  }
  return a;
}

// CTAs of the main kernel: one per SM of the tensor-core kernel, as many as fit of the others.
int decode_grid(const DecodeKind& kind, int d_pad) {
  const int per_sm = kind.sm100 ? 1 : kind.f32 ? 2 : d_pad == 64 ? 4 : d_pad == 128 ? 2 : 1;
  const int n = sm100_sm_count() * per_sm;
  return n < kJoinMost ? n : kJoinMost;
}

size_t carve_decode(const DecodeParams& P, char* base, DecodeSpace* s, bool own_lse) {
  char* p = base;
  auto take = [&](size_t bytes) { char* r = p; p += align256(bytes); return r; };
  const size_t rows = (size_t)P.batch * P.nhead_k, heads = (size_t)P.batch * P.nhead_q, slots = 2 * (size_t)P.grid * kDecodeHeads;
  s->status = reinterpret_cast<int32_t*>(take(kStatusWords * 4));
  s->cta_status = reinterpret_cast<int32_t*>(take((size_t)P.grid * 8));
  s->cta_start = reinterpret_cast<int4*>(take((size_t)P.grid * 16));
  s->cta_join = reinterpret_cast<int32_t*>(take((size_t)P.grid * 4));
  s->total = reinterpret_cast<long long*>(take(8));
  s->pieces = reinterpret_cast<int32_t*>(take(P.mask ? rows * 4 : 0));
  s->list = reinterpret_cast<int32_t*>(take(P.mask ? rows * P.num_k_block * 4 : 0));
  s->lse = reinterpret_cast<float*>(take(own_lse ? heads * 4 : 0));
  s->part_ml = reinterpret_cast<float*>(take(slots * 8));
  s->part_o = reinterpret_cast<float*>(take(slots * P.d_pad * 4));
  s->scores = reinterpret_cast<float*>(take(P.weights ? heads * P.capacity * 4 : 0));
  return (size_t)(p - base);
}

// Everything but the launches; also what the workspace's size comes from (need_tensors false: pointers may be missing).
int make_decode(const hbsa_paged_attention_args* a, bool need_tensors, DecodeParams* P, DecodeKind* kind, size_t* bytes) {
  if (!a) return set_last_error("args is NULL"), HBSA_ERR_NULL;
  if (a->struct_bytes != sizeof(*a)) return set_last_error("hbsa_paged_attention_args.struct_bytes does not match this library"), HBSA_ERR_STRUCT;
  const hbsa_cache& c = a->cache;
  if (need_tensors && (!a->q || !a->o || !a->workspace || !c.k || !c.v || !c.block_table || !c.lens))
    return set_last_error("q, o, the cache's k, v, block_table and lens, and workspace must not be NULL"), HBSA_ERR_NULL;
  if (c.batch <= 0 || c.nhead_k <= 0 || c.headdim <= 0 || c.num_pages <= 0 || c.page_size <= 0 || c.max_pages <= 0 || a->nhead_q <= 0)
    return set_last_error("batch, head counts, headdim, num_pages, page_size and max_pages must be positive"), HBSA_ERR_SHAPE;
  if (a->nhead_q % c.nhead_k != 0) return set_last_error("nhead_q must be divisible by nhead_k (for GQA)"), HBSA_ERR_SHAPE;
  if (c.headdim > 256) return set_last_error("headdim above 256 is not supported"), HBSA_ERR_SHAPE;
  if ((int64_t)c.max_pages * c.page_size > INT32_MAX - 4096) return set_last_error("max_pages * page_size does not fit 31 bits"), HBSA_ERR_SHAPE;
  if ((int64_t)c.batch * c.nhead_k > INT32_MAX / 64) return set_last_error("batch * nhead_k is too large"), HBSA_ERR_SHAPE;
  if (c.dtype != HBSA_DTYPE_BF16 && c.dtype != HBSA_DTYPE_F16 && c.dtype != HBSA_DTYPE_F32) return set_last_error("unknown dtype"), HBSA_ERR_DTYPE;
  if (a->impl != HBSA_IMPL_AUTO && a->impl != HBSA_IMPL_GENERIC && a->impl != HBSA_IMPL_SM100) return set_last_error("unknown impl"), HBSA_ERR_DTYPE;
  memset(P, 0, sizeof(*P));
  P->capacity = c.max_pages * c.page_size;
  if (a->block_mask) {
    if (a->k_block_size <= 0 || a->k_block_size % 16 != 0) return set_last_error("k_block_size must be an integer multiple of 16."), HBSA_ERR_BLOCK_SIZE;
    if (a->num_k_block <= 0 || (int64_t)a->num_k_block * a->k_block_size < P->capacity)
      return set_last_error("block_mask must cover max_pages * page_size = %d positions", P->capacity), HBSA_ERR_SHAPE;
  }
  P->k = c.k;
  P->v = c.v;
  P->q = a->q;
  P->o = a->o;
  for (int i = 0; i < 4; ++i) {
    P->k_s[i] = c.k_stride[i];
    P->v_s[i] = c.v_stride[i];
  }
  for (int i = 0; i < 3; ++i) {
    P->q_s[i] = a->q_stride[i];
    P->o_s[i] = a->o_stride[i];
    P->mask_s[i] = a->mask_stride[i];
  }
  P->table = c.block_table;
  P->table_stride = c.table_stride;
  P->lens = c.lens;
  P->mask = a->block_mask;
  P->weights = a->key_weights;
  P->weights_s[0] = a->weights_stride[0];
  P->weights_s[1] = a->weights_stride[1];
  P->num_pages = c.num_pages;
  P->page = c.page_size;
  P->page_div = FastDiv(c.page_size);
  P->batch = c.batch;
  P->nhead_q = a->nhead_q;
  P->nhead_k = c.nhead_k;
  P->group = a->nhead_q / c.nhead_k;
  P->headdim = c.headdim;
  P->d_pad = c.headdim <= 64 ? 64 : c.headdim <= 128 ? 128 : 256;
  P->kbs = a->k_block_size;
  P->num_k_block = a->num_k_block;
  P->entries = a->block_mask ? c.batch * c.nhead_k : c.batch;
  const float scale = a->use_default_scale ? 1.0f / sqrtf((float)c.headdim) : a->softmax_scale;
  P->scale_log2 = scale * kDecodeLog2e;
  P->wait_budget = sm100_wait_budget();
  P->debug_stall = sm100_debug_stall();
  const char* why = decode_sm100_ineligible_reason(*a, scale);
  if (need_tensors && a->impl == HBSA_IMPL_SM100 && why) return set_last_error("the tensor-core kernel cannot run this problem: %s", why), HBSA_ERR_UNSUPPORTED;
  kind->sm100 = !why && a->impl != HBSA_IMPL_GENERIC;
  kind->f32 = decode_f32_eligible(*a);
  const int most_heads = kind->f32 ? (P->d_pad == 256 ? 4 : 8) : kind->sm100 && P->d_pad == 256 ? 16 : kDecodeHeads;
  P->n_chunk = (P->group + most_heads - 1) / most_heads;
  P->chunk_heads = (P->group + P->n_chunk - 1) / P->n_chunk;
  P->unit = kDecodeTile;
  if (kind->sm100) P->unit = gcd(P->unit, P->page);
  if (P->mask) P->unit = gcd(P->unit, P->kbs);
  P->pieces_per_block = P->mask ? P->kbs / P->unit : 0;
  P->one_box = P->headdim % 64 == 0;
  P->lanes = P->mask || P->nhead_k % 2 ? 1 : 2;
  P->runs = decode_grid(*kind, P->d_pad) / P->lanes;
  P->grid = P->runs * P->lanes;
  const bool own_lse = a->key_weights && !a->lse;
  if (!need_tensors) {                                     // enough for whichever kernel the call gets: that depends on addresses and strides
    const int grid = P->grid, all = sm100_sm_count() * (P->d_pad == 64 ? 4 : 2);
    P->grid = all < kJoinMost ? all : kJoinMost;
    *bytes = carve_decode(*P, nullptr, &P->sp, a->key_weights != nullptr);
    P->grid = grid;
    return 0;
  }
  *bytes = carve_decode(*P, static_cast<char*>(a->workspace), &P->sp, own_lse);
  P->lse = own_lse ? P->sp.lse : a->lse;
  return 0;
}

}  // namespace

cudaError_t launch_decode_generic(const DecodeParams& P, int dtype, bool dependent, cudaStream_t stream) {
  if (dtype == HBSA_DTYPE_BF16) return launch_generic_of<__nv_bfloat16>(P, dependent, stream);
  if (dtype == HBSA_DTYPE_F16) return launch_generic_of<__half>(P, dependent, stream);
  return launch_generic_of<float>(P, dependent, stream);
}

}  // namespace hbsa

extern "C" {

size_t hbsa_paged_attention_workspace_bytes(const hbsa_paged_attention_args* args) {
  hbsa::DecodeParams P;
  hbsa::DecodeKind kind;
  size_t bytes;
  return hbsa::make_decode(args, false, &P, &kind, &bytes) == 0 ? bytes : 0;
}

int hbsa_paged_attention(const hbsa_paged_attention_args* args, void* stream_) {
  hbsa::DecodeParams P;
  hbsa::DecodeKind kind;
  size_t bytes;
  int rc = hbsa::make_decode(args, true, &P, &kind, &bytes);
  if (rc != 0) return rc;
  if (args->workspace_bytes < bytes) return hbsa::set_last_error("workspace is smaller than hbsa_paged_attention_workspace_bytes()"), HBSA_ERR_WORKSPACE;
  if ((uintptr_t)args->workspace % 256 != 0) return hbsa::set_last_error("workspace must be 256-byte aligned"), HBSA_ERR_WORKSPACE;
  cudaStream_t stream = static_cast<cudaStream_t>(stream_);
  auto failed = [](cudaError_t e) { return hbsa::set_last_error("hbsa_paged_attention: %s", cudaGetErrorString(e)), (int)e; };
  cudaError_t e = cudaSuccess;
  const bool masked = P.mask != nullptr;
  if (masked && (e = hbsa::launch_kernel(hbsa::decode_blocks_kernel, (unsigned)((P.batch * P.nhead_k + 7) / 8), 256, 0, false, stream, P)) != cudaSuccess) return failed(e);
  if (kind.sm100) {
    const char* text = "";
    rc = hbsa::launch_decode_sm100(P, *args, masked, stream, &text);
    if (rc != 0) return hbsa::set_last_error("hbsa_paged_attention: %s", text), rc;
  } else if ((e = kind.f32 ? hbsa::launch_decode_f32(P, masked, stream) : hbsa::launch_decode_generic(P, args->cache.dtype, masked, stream)) != cudaSuccess) {
    return failed(e);
  }
  auto join = args->cache.dtype == HBSA_DTYPE_BF16  ? hbsa::decode_join_kernel<__nv_bfloat16>
              : args->cache.dtype == HBSA_DTYPE_F16 ? hbsa::decode_join_kernel<__half>
                                                    : hbsa::decode_join_kernel<float>;
  cudaLaunchAttribute attr[1] = {};
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)P.grid, (unsigned)(P.chunk_heads + (P.weights ? hbsa::kWeightParts : 0)));
  cfg.blockDim = dim3(hbsa::kJoinThreads);
  cfg.stream = stream;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  if ((e = cudaLaunchKernelEx(&cfg, join, P)) != cudaSuccess) return failed(e);
  return 0;
}

}  // extern "C"
