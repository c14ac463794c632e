// Main kernel of the paged decode attention for fp32 rows of 16-byte units; see hbsa_decode.cu for the mathematics and hbsa_decode.cuh for the
// split.  Products stay in fp32 on the CUDA cores: a tensor core would round the operands to 10 bits.
//
// A warp works by itself: it reads the rows of K and V of a slab of 2 to 8 keys straight into registers, one 16-byte unit
// per lane (two with 256 columns; with 64 columns half a warp has a key), so every load is one or two whole rows and nothing waits for
// another warp before the row of heads ends.  The products of a slab are sums over the lanes: lanes exchange halves of what they
// have and add, log2(32) times, after which every (key, head) is in a lane of its own: one shuffle a sum, and one exponential a lane.
// Its probability goes back to all lanes by shuffles for O += P V, whose columns stay where V's are.
// Up to 8 heads (4 with 256 columns) share the read of K and V; groups of more take several chunks, each of which reads K and V again (8 x 8192 keys, 4
// kv-heads of 256: 87, 106 and 191 us with groups of 1, 4 and 8).
// With 16 warps an SM, each with up to 8 KB on its way, the read of K and V bounds it for small groups, for larger ones
// the instructions (62 % of the issue slots and 36 % of the FMA pipe with groups of 8, where a slab's read also waits for the products of the one before):
// 8 x 8192..16384 keys, 8 heads of 128, take 123, 154 and 230 us with groups of 1, 4 and 8 (6.4, 5.1 and 3.4 TB/s).  The kernel with tiles
// in shared memory meets five times a tile: 490 us with groups of 4.
#include "hbsa_decode.cuh"

namespace hbsa {

namespace {

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;

struct F32Shared {
  DecodeWalk walk;
  long long scratch[kWarps];
  float2 ml[kWarps][8];
  int bad;                                             // the first sequence with a length or a page out of range, from the end (0: none)
};

template <int DP, int HEADS>
__global__ void __launch_bounds__(kThreads, 2) decode_f32_kernel(const __grid_constant__ DecodeParams P) {
  constexpr int LPK = DP >= 128 ? 32 : DP / 4;         // lanes of a key
  constexpr int UNITS = DP / (4 * LPK);                // 16-byte units of a lane
  // keys of a slab, and of a lane, by measurement (8 heads of 128 with slabs of 8 and 4: 351 and 230 us for 8 x 8192..16384 keys, 4 heads of 256
  // with slabs of 4 and 2: 159 and 134 us for half of them).  Registers hold that nearly: at 128 a thread six of the eleven instances spill, 8 heads of
  // 64 and 128 244 and 188 bytes, the others up to 52.
  constexpr int SLAB = DP == 256 ? (HEADS == 4 ? 2 : 4) : DP == 128 && HEADS == 8 ? 4 : 8, KPL = SLAB / (32 / LPK);
  constexpr int N = KPL * HEADS;                       // sums of a group of LPK lanes: sum v = key * HEADS + head ends in lane v / R * REP
  constexpr int R = N > LPK ? N / LPK : 1, REP = N < LPK ? LPK / N : 1;    // sums of a lane, lanes of a sum
  constexpr int PER_TILE = kDecodeTile / SLAB;
  __shared__ F32Shared sh;
  __shared__ __align__(16) float s_part[kWarps][HEADS][DP];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, sub = lane % LPK, side = lane / LPK;
  if (tid == 0) sh.bad = 0;
  pdl_wait();                                          // the block lists
  decode_locate(P, &sh.walk, sh.scratch);
  pdl_launch();
  DecodeWalk walk = sh.walk;
  const float* const K = static_cast<const float*>(P.k);
  const float* const V = static_cast<const float*>(P.v);
  for (long long t = walk.start; t < walk.end;) {
    const DecodeRow r = decode_row_at(P, walk, t, blockIdx.x);
    if (t == walk.start && tid == 0) decode_note_start(P, r);
    t += r.tiles;
    const int head0 = r.hk * P.group + r.chunk * P.chunk_heads;
    const int heads = min(P.chunk_heads, P.group - r.chunk * P.chunk_heads);
    // position of a slab's first key, how many of its keys there are, its page
    const int first = r.tile0 * PER_TILE, n_slabs = r.tiles * PER_TILE;
    int pos, n = 0, page = 0, slot = 0;
    auto look_up = [&](int slab) {
      pos = (first + slab) * SLAB;
      if (P.mask != nullptr) {
        const int piece = pos / P.unit, p = slab < n_slabs ? decode_piece_position(P, r, piece) : -1;
        pos = p < 0 ? r.len : p + pos - piece * P.unit;
      }
      n = slab < n_slabs ? max(0, min(SLAB, r.len - pos)) : 0;
      if (n > 0) {
        const int i = P.page_div.split(pos, slot);
        page = P.table[r.b * P.table_stride + i];
      }
    };
    look_up(warp);
    float4 q[HEADS][UNITS], o[HEADS][UNITS];
#pragma unroll
    for (int h = 0; h < HEADS; ++h)
#pragma unroll
      for (int u = 0; u < UNITS; ++u) {
        const int d = 4 * (sub + u * LPK);
        const float* from = static_cast<const float*>(P.q) + r.b * P.q_s[0] + (head0 + h) * P.q_s[1] + d * P.q_s[2];
        const bool there = h < heads && d < P.headdim;
        q[h][u] = there ? make_float4(from[0], from[P.q_s[2]], from[2 * P.q_s[2]], from[3 * P.q_s[2]]) : make_float4(0.f, 0.f, 0.f, 0.f);
        o[h][u] = make_float4(0.f, 0.f, 0.f, 0.f);
      }
    float m[R], l[R];                                  // of the head of the lane's sums; the maximum is the warp's
#pragma unroll
    for (int i = 0; i < R; ++i) {
      m[i] = -INFINITY;
      l[i] = 0.f;
    }
    for (int slab = warp; slab < n_slabs; slab += kWarps) {
      const int at = pos, there = n;
      const bool bad = there > 0 && (page < 0 || page >= P.num_pages);
      const long long k_at = page * P.k_s[0] + slot * P.k_s[1] + r.hk * P.k_s[2], v_at = page * P.v_s[0] + slot * P.v_s[1] + r.hk * P.v_s[2];
      const int keys = bad ? 0 : there;
      if (bad && lane == 0) atomicMax(&sh.bad, P.batch - r.b);
      float4 k[KPL][UNITS], v[KPL][UNITS];
#pragma unroll
      for (int e = 0; e < KPL; ++e)
#pragma unroll
        for (int u = 0; u < UNITS; ++u) {
          const int key = e * (32 / LPK) + side, d = 4 * (sub + u * LPK);
          k[e][u] = v[e][u] = make_float4(0.f, 0.f, 0.f, 0.f);
          if (key < keys && d < P.headdim) {
            k[e][u] = *reinterpret_cast<const float4*>(K + k_at + key * P.k_s[1] + d);
            v[e][u] = *reinterpret_cast<const float4*>(V + v_at + key * P.v_s[1] + d);
          }
        }
      look_up(slab + kWarps);
      float s[N];
#pragma unroll
      for (int e = 0; e < KPL; ++e)
#pragma unroll
        for (int h = 0; h < HEADS; ++h) {
          float x = 0.f;
#pragma unroll
          for (int u = 0; u < UNITS; ++u)
            x = fmaf(k[e][u].x, q[h][u].x, fmaf(k[e][u].y, q[h][u].y, fmaf(k[e][u].z, q[h][u].z, fmaf(k[e][u].w, q[h][u].w, x))));
          s[e * HEADS + h] = x;
        }
      // sums over the key's lanes
      constexpr int kSteps = LPK == 32 ? 5 : 4;
#pragma unroll
      for (int step = 0; step < kSteps; ++step) {
        const int mask = LPK >> (step + 1), left = N >> (step + 1);
        if (left > 0) {
          const bool upper = (lane & mask) != 0;
#pragma unroll
          for (int i = 0; i < left; ++i) {
            const float give = upper ? s[i] : s[i + left], have = upper ? s[i + left] : s[i];
            s[i] = have + __shfl_xor_sync(0xffffffffu, give, mask);
          }
        } else {
          s[0] += __shfl_xor_sync(0xffffffffu, s[0], mask);
        }
      }
      bool grows = false;
#pragma unroll
      for (int i = 0; i < R; ++i) {
        const int sum = sub / REP * R + i, key = sum / HEADS * (32 / LPK) + side, head = sum % HEADS;
        s[i] = key < keys ? s[i] * P.scale_log2 : -INFINITY;
        if (P.weights != nullptr && key < there && head < heads && sub % REP == 0)
          P.sp.scores[((long long)r.b * P.nhead_q + head0 + head) * P.capacity + at + key] = s[i];
        grows = grows || s[i] > m[i];
      }
      if (__any_sync(0xffffffffu, grows)) {            // the lanes of a head agree on its maximum; O and the sums follow
        float alpha[R];
#pragma unroll
        for (int i = 0; i < R; ++i) {
          float x = fmaxf(m[i], s[i]);
#pragma unroll
          for (int mask = HEADS * REP / R; mask < 32; mask <<= 1) x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, mask));
          alpha[i] = x == -INFINITY ? 1.f : exp2f(m[i] - x);
          l[i] *= alpha[i];
          m[i] = x;
        }
#pragma unroll
        for (int h = 0; h < HEADS; ++h) {
          const float a = __shfl_sync(0xffffffffu, alpha[h % R], h / R * REP);
#pragma unroll
          for (int u = 0; u < UNITS; ++u) {
            o[h][u].x *= a;
            o[h][u].y *= a;
            o[h][u].z *= a;
            o[h][u].w *= a;
          }
        }
      }
#pragma unroll
      for (int i = 0; i < R; ++i) {
        s[i] = exp2f(s[i] - (m[i] == -INFINITY ? 0.f : m[i]));
        l[i] += s[i];
      }
#pragma unroll
      for (int e = 0; e < KPL; ++e)
#pragma unroll
        for (int h = 0; h < HEADS; ++h) {
          const int sum = e * HEADS + h;
          const float p = __shfl_sync(0xffffffffu, s[sum % R], side * LPK + sum / R * REP);
#pragma unroll
          for (int u = 0; u < UNITS; ++u) {
            o[h][u].x = fmaf(p, v[e][u].x, o[h][u].x);
            o[h][u].y = fmaf(p, v[e][u].y, o[h][u].y);
            o[h][u].z = fmaf(p, v[e][u].z, o[h][u].z);
            o[h][u].w = fmaf(p, v[e][u].w, o[h][u].w);
          }
        }
    }
    // ---- the warps' parts of the row
    __syncthreads();                                   // those of the row before have been read
#pragma unroll
    for (int i = 0; i < R; ++i) {
#pragma unroll
      for (int mask = HEADS * REP / R; mask < 32; mask <<= 1) l[i] += __shfl_xor_sync(0xffffffffu, l[i], mask);
      const int sum = sub / REP * R + i;
      if (sum < HEADS && side == 0 && sub % REP == 0) sh.ml[warp][sum] = make_float2(m[i], l[i]);
    }
#pragma unroll
    for (int h = 0; h < HEADS; ++h)
#pragma unroll
      for (int u = 0; u < UNITS; ++u) {
        float4 x = o[h][u];
        if (LPK < 32) {
          x.x += __shfl_xor_sync(0xffffffffu, x.x, LPK);
          x.y += __shfl_xor_sync(0xffffffffu, x.y, LPK);
          x.z += __shfl_xor_sync(0xffffffffu, x.z, LPK);
          x.w += __shfl_xor_sync(0xffffffffu, x.w, LPK);
        }
        if (side == 0) *reinterpret_cast<float4*>(&s_part[warp][h][4 * (sub + u * LPK)]) = x;
      }
    __syncthreads();
    for (int item = tid; item < heads * (DP / 4); item += kThreads) {
      const int h = item / (DP / 4), d = item % (DP / 4) * 4;
      float2 ml[kWarps];
      float mt = -INFINITY, lt = 0.f;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) {
        ml[w] = sh.ml[w][h];
        mt = fmaxf(mt, ml[w].x);
      }
      float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int w = 0; w < kWarps; ++w) {
        const float4 y = *reinterpret_cast<const float4*>(&s_part[w][h][d]);
        const float f = ml[w].x == -INFINITY ? 0.f : exp2f(ml[w].x - mt);
        x.x = fmaf(y.x, f, x.x);
        x.y = fmaf(y.y, f, x.y);
        x.z = fmaf(y.z, f, x.z);
        x.w = fmaf(y.w, f, x.w);
        lt += ml[w].x == -INFINITY ? ml[w].y : ml[w].y * f;        // (a sum of NaN stays one)
      }
      if (r.slot >= 0) {
        const long long to = (2ll * blockIdx.x + r.slot) * kDecodeHeads + h;
        *reinterpret_cast<float4*>(P.sp.part_o + to * P.d_pad + d) = x;
        if (d == 0) *reinterpret_cast<float2*>(P.sp.part_ml + to * 2) = make_float2(mt, lt);
      } else {
        const bool none = mt == -INFINITY && lt == 0.f;
        const float inv = none ? 0.f : 1.f / lt;
        float* const to = static_cast<float*>(P.o) + r.b * P.o_s[0] + (head0 + h) * P.o_s[1] + d * P.o_s[2];
        if (d < P.headdim) {
          to[0] = none ? 0.f : x.x * inv;
          to[P.o_s[2]] = none ? 0.f : x.y * inv;
          to[2 * P.o_s[2]] = none ? 0.f : x.z * inv;
          to[3 * P.o_s[2]] = none ? 0.f : x.w * inv;
        }
        if (d == 0 && P.lse != nullptr) P.lse[(long long)r.b * P.nhead_q + head0 + h] = none ? -INFINITY : (mt + log2f(lt)) * kDecodeLn2;
      }
    }
  }
  decode_fill_empty<float>(P, blockIdx.x, P.grid);
  for (int b = blockIdx.x * kThreads + tid; b < P.batch; b += P.grid * kThreads)
    if (P.lens[b] < 0 || P.lens[b] > P.capacity) atomicMax(&sh.bad, P.batch - b);
  __syncthreads();
  if (tid == 0) decode_note_join(P, sh.walk);
  if (tid == 0) decode_note_status(P, sh.bad != 0 ? (int)HBSA_STATUS_CACHE_BOUNDS : (int)HBSA_STATUS_OK, P.batch - sh.bad);
}

template <int DP>
cudaError_t launch_heads(const DecodeParams& P, bool dependent, cudaStream_t stream) {
  if (P.chunk_heads == 1) return launch_kernel(decode_f32_kernel<DP, 1>, (unsigned)P.grid, kThreads, 0, dependent, stream, P);
  if (P.chunk_heads == 2) return launch_kernel(decode_f32_kernel<DP, 2>, (unsigned)P.grid, kThreads, 0, dependent, stream, P);
  if constexpr (DP < 256) {                            // (with 256 columns a chunk has up to 4 heads)
    if (P.chunk_heads > 4) return launch_kernel(decode_f32_kernel<DP, 8>, (unsigned)P.grid, kThreads, 0, dependent, stream, P);
  }
  return launch_kernel(decode_f32_kernel<DP, 4>, (unsigned)P.grid, kThreads, 0, dependent, stream, P);
}

}  // namespace

// fp32 rows of 16-byte units, and no slab of 8 keys on two pages.
bool decode_f32_eligible(const hbsa_paged_attention_args& a) {
  const hbsa_cache& c = a.cache;
  if (c.dtype != HBSA_DTYPE_F32 || c.headdim % 4 != 0 || c.page_size % 8 != 0) return false;
  if (c.k_stride[3] != 1 || c.v_stride[3] != 1 || (uintptr_t)c.k % 16 != 0 || (uintptr_t)c.v % 16 != 0) return false;
  for (int i = 0; i < 3; ++i)
    if (c.k_stride[i] % 4 != 0 || c.v_stride[i] % 4 != 0) return false;
  return true;
}

cudaError_t launch_decode_f32(const DecodeParams& P, bool dependent, cudaStream_t stream) {
  if (P.d_pad == 64) return launch_heads<64>(P, dependent, stream);
  if (P.d_pad == 128) return launch_heads<128>(P, dependent, stream);
  return launch_heads<256>(P, dependent, stream);
}

}  // namespace hbsa
