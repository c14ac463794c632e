// Writing into a paged key-value cache, choosing what stays when it is cut down, and moving that together.
// All three are bound by memory: every byte is read once and written once.
#include "sm100_common.cuh"

namespace hbsa {

namespace {

// Rows are copied in units of U: 16 bytes where bases, strides and the row length allow it, one element otherwise.
struct Rows4 { long long s[4]; };        // strides in units: page, slot, head, unit

// ------------------------------------------------------------------------------------------------------------------
// Append: one warp per new token, K and V together, four units of each on their way a lane.  The last block writes the new lengths and the status.
// One token of 16 sequences, 8 heads of 64: 2.6 us (a launch); 8 x 1024..16384 tokens, 8 heads of 128: 78 us (480 MB, 6.2 TB/s).
struct AppendParams {
  const void *k, *v;
  void *k_cache, *v_cache;
  Rows4 kc, vc;
  long long k_s[3], v_s[3];              // token, head, unit
  const int32_t *table, *lens, *cu;
  long long table_stride;
  int32_t *new_lens, *status;
  FastDiv page;
  int num_pages, capacity, batch, heads, units, total;
  int flat;                              // the heads of a token follow one another: one run of heads * units
};

__device__ __forceinline__ int cut(int x, int hi) { return max(0, min(x, hi)); }

__device__ __forceinline__ void append_status(const AppendParams& P) {
  __shared__ int s_bad;
  const int tid = threadIdx.x, threads = blockDim.x;
  if (tid == 0) s_bad = 0x7fffffff;
  __syncthreads();
  int per = 1;                           // threads of a sequence
  while (per < 32 && per * 2 * P.batch <= threads) per *= 2;
  for (int b = tid / per; b < P.batch; b += threads / per) {
    const int raw = P.lens[b], len = cut(raw, P.capacity), c0 = P.cu[b], c1 = P.cu[b + 1], n = max(0, cut(c1, P.total) - cut(c0, P.total));
    const int end = (int)min((long long)len + n, (long long)P.capacity);       // (only rows that are there count: what is read later has been written)
    bool bad = raw != len || (long long)len + n > P.capacity || c0 < 0 || c1 < c0 || c1 > P.total;
    if (end > len)
      for (int i = P.page.quotient(len) + tid % per; i <= P.page.quotient(end - 1); i += per) {
        const int page = P.table[b * P.table_stride + i];
        bad |= page < 0 || page >= P.num_pages;
      }
    if (bad) atomicMin(&s_bad, b);
    if (tid % per == 0) P.new_lens[b] = end;
  }
  __syncthreads();
  if (tid < kStatusWords)
    P.status[tid] = s_bad == 0x7fffffff ? 0 : tid == 0 ? (int)HBSA_STATUS_CACHE_BOUNDS : tid == 1 ? s_bad : 0;
}

template <typename U>
__global__ void __launch_bounds__(256) append_kernel(const __grid_constant__ AppendParams P) {
  if (blockIdx.x == gridDim.x - 1) {
    append_status(P);
    return;
  }
  const int lane = threadIdx.x & 31;
  const U *k = static_cast<const U*>(P.k), *v = static_cast<const U*>(P.v);
  U *kc = static_cast<U*>(P.k_cache), *vc = static_cast<U*>(P.v_cache);
  const int lo = max(0, P.cu[0]), hi = min(P.total, P.cu[P.batch]);
  for (long long tok = lo + (long long)blockIdx.x * 8 + (threadIdx.x >> 5); tok < hi; tok += (gridDim.x - 1) * 8ll) {
    const int b = sample_of_block(P.cu, P.batch, (int)tok);
    const long long pos = (long long)cut(P.lens[b], P.capacity) + (tok - max(0, P.cu[b]));
    if (pos >= P.capacity) continue;                       // (never negative: cu[b] <= tok whatever cu holds)
    int slot;
    const int page = P.table[b * P.table_stride + P.page.split((int)pos, slot)];
    if (page < 0 || page >= P.num_pages) continue;
    const U *ks = k + tok * P.k_s[0], *vs = v + tok * P.v_s[0];
    U *kd = kc + page * P.kc.s[0] + slot * P.kc.s[1], *vd = vc + page * P.vc.s[0] + slot * P.vc.s[1];
    const int n = P.heads * P.units;
    if (P.flat) {
      for (int i = lane; i < n; i += 128) {
        U a[4], c[4];
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (i + 32 * e < n) {
            a[e] = ks[i + 32 * e];
            c[e] = vs[i + 32 * e];
          }
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (i + 32 * e < n) {
            kd[i + 32 * e] = a[e];
            vd[i + 32 * e] = c[e];
          }
      }
    } else {
      for (int i = lane; i < n; i += 32) {
        const int h = i / P.units, u = i % P.units;
        kd[h * P.kc.s[2] + u * P.kc.s[3]] = ks[h * P.k_s[1] + u * P.k_s[2]];
        vd[h * P.vc.s[2] + u * P.vc.s[3]] = vs[h * P.v_s[1] + u * P.v_s[2]];
      }
    }
  }
}

// ------------------------------------------------------------------------------------------------------------------
// Select: radix select of the smallest weight that stays, then one pass that writes positions in order.  The digits are 11 bits of the distance
// from the smallest weight above zero (or, where all of those stay, from the smallest of the rest): that keeps keys that nobody has looked at
// out of the counts, where they would meet in one bin, and spreads weights of one size over many.  Where no more than kSelectRank weights come down
// to the next digit (usual after the first one), each finds its rank among them at once.  Ranking n weights against going on by digits, in us: 128 rows
// of 24576 17.0 and 19.7 (n = 16), 18.0 and 20.0 (100), 19.1 and 20.1 (150), 27.7 and 20.4 (512), 55.5 and 20.6 (1000); 128 rows of 8192 7.6 and 8.9,
// 8.4 and 8.9, 9.4 and 9.0, 17.3 and 9.1, 44.2 and 9.1; 16 rows of 1000 5.3 and 6.3, 5.9 and 6.3, 6.9 and 6.4.
// A cluster of 1 to 4 CTAs per row; counts
// are exchanged through distributed shared memory.  Every warp has its run of positions, in registers where they fit, as numbers that tell by
// themselves whether the position competes; where they do not fit, they are read again for every pass.  Bound by the instructions of its
// passes (20.1 us for 128 rows of 16384 to 32768, 35 us while every pass compared positions): 61 % of the issue slots; no wait stands out, shared
// atomics take 7 % of the cycles, and memory is busy for the first pass only.
constexpr int kSelectBins = 2048;
constexpr int kSelectRank = 128;
constexpr uint32_t kGoes = 0u, kStays = 0xffffffffu, kZero = 0x80000000u;

// Weights as unsigned numbers in the same order, from 0x007fffff to 0xff800000; both zeros are one (0x80000000), NaN is the next above them all.
__device__ __forceinline__ uint32_t order_of(float x) {
  if (x != x) return 0xff800001u;
  const uint32_t u = __float_as_uint(x + 0.f);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}

__device__ __forceinline__ int ld_cluster(uint32_t addr) {
  int x;
  asm volatile("ld.shared::cluster.s32 %0, [%1];" : "=r"(x) : "r"(addr) : "memory");
  return x;
}

// PER: positions of a lane that registers hold, 0: none.
template <int PER, int THREADS>
__global__ void __launch_bounds__(THREADS) select_keys_kernel(const __grid_constant__ hbsa_select_keys_args a, int ctas) {
  constexpr int WARPS = THREADS / 32, BINS = kSelectBins / THREADS, STEP = PER > 0 ? PER : 8;      // bins of a thread, positions of a lane and go
  __shared__ int s_hist[kSelectBins];
  __shared__ int s_more[WARPS], s_ties[WARPS], s_sum[2];
  __shared__ uint32_t s_range[4], s_prefix;
  __shared__ int s_need, s_here, s_found;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int row = blockIdx.x / ctas, rank = blockIdx.x - row * ctas, b = row / a.nhead_k, h = row - b * a.nhead_k;
  const int len = cut(a.lens[b], a.max_len);
  const float* w = a.key_weights + b * a.weights_stride[0] + h * a.weights_stride[1];
  int32_t* kept = a.kept + (long long)row * a.budget;
  if (h == 0 && rank == 0 && tid == 0) a.kept_lens[b] = min(len, a.budget);
  if (len <= a.budget) {                                 // all CTAs of the cluster
    for (int i = rank * THREADS + tid; i < a.budget; i += ctas * THREADS) kept[i] = i < len ? i : -1;
    return;
  }
  const int lo = a.n_sink, hi = len - a.n_recent;        // the positions that compete; n_sink + n_recent <= budget < len
  int need = a.budget - a.n_sink - a.n_recent;
  const int run = ((len + ctas - 1) / ctas + 31) & ~31, p0 = min(rank * run, len), p1 = min(p0 + run, len);      // this CTA's
  const int seg = ((p1 - p0 + WARPS - 1) / WARPS + 31) & ~31, s0 = min(p0 + warp * seg, p1), s1 = min(s0 + seg, p1);     // this warp's
  auto meet = [&]() {
    if (ctas > 1) ptx::cluster_sync();
    else __syncthreads();
  };
  // A number per position: its weight's while it competes; kStays for the first and last ones; kGoes behind the warp's.  Once the range that
  // holds the answer is known, the distance from its low end, plus one, with kGoes below it and kStays above.
  uint32_t u[STEP], low = 0u, high = 0u;
  bool ranged = false;
  auto place = [&](uint32_t x) { return x < low ? kGoes : x > high ? kStays : x - low + 1u; };
  auto read = [&](int from) {
    auto inside = [&](int part) { return from + 32 * part >= lo && from + 32 * part + 256 <= min(hi, s1); };
#pragma unroll
    for (int part = 0; part < STEP; part += 8) {         // all loads first
      const int at = from + 32 * part + lane;
      if (inside(part)) {
#pragma unroll
        for (int e = 0; e < 8; ++e) u[part + e] = __float_as_uint(w[at + 32 * e]);
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) u[part + e] = at + 32 * e >= lo && at + 32 * e < min(hi, s1) ? __float_as_uint(w[at + 32 * e]) : 0u;
      }
    }
#pragma unroll
    for (int part = 0; part < STEP; part += 8) {
#pragma unroll
      for (int e = part; e < part + 8; ++e) u[e] = order_of(__uint_as_float(u[e]));
      if (!inside(part)) {
#pragma unroll
        for (int e = part; e < part + 8; ++e) {
          const int i = from + 32 * e + lane;
          u[e] = i >= s1 ? kGoes : i < lo || i >= hi ? kStays : u[e];
        }
      }
      if (PER == 0 && ranged) {
#pragma unroll
        for (int e = part; e < part + 8; ++e) u[e] = place(u[e]);
      }
    }
  };
  // f(number, position of lane 0) for every 32 positions
  auto each = [&](auto&& f) {
    for (int at = s0; at < s1; at += 32 * STEP) {
      if (PER == 0) read(at);
#pragma unroll
      for (int part = 0; part < STEP; part += 8)
        if (at + 32 * part < s1) {
#pragma unroll
          for (int e = part; e < part + 8; ++e) f(u[e], at + 32 * e);
        }
    }
  };
  if (tid < 4) s_range[tid] = tid < 2 ? 0xffffffffu : 0u;
  if (PER > 0) read(s0);
  uint32_t least = kStays;                               // the smallest number that stays
  int ties = 0x7fffffff;                                 // and how many of it do
  if (need > 0) {
    // smallest of all (kGoes wraps around), smallest above zero (what is not above wraps), largest (kStays wraps), how many above zero
    uint32_t least_all = 0xffffffffu, least_above = 0xffffffffu, most = 0u;
    int above = 0;
    each([&](uint32_t x, int) {
      least_all = min(least_all, x - 1u);
      least_above = min(least_above, x - (kZero + 1u));
      most = max(most, x + 1u);
      above += x > kZero;
    });
    least_all = __reduce_min_sync(0xffffffffu, least_all);
    least_above = __reduce_min_sync(0xffffffffu, least_above);
    most = __reduce_max_sync(0xffffffffu, most);
    above = __reduce_add_sync(0xffffffffu, above);
    __syncthreads();
    if (lane == 0) {
      atomicMin(&s_range[0], least_all);
      atomicMin(&s_range[1], least_above);
      atomicMax(&s_range[2], most);
      atomicAdd(&s_range[3], (uint32_t)above);
    }
    meet();
    least_all = least_above = 0xffffffffu;
    most = 0u;
    above = -a.n_sink - a.n_recent;                      // kStays were counted
    for (int r = 0; r < ctas; ++r) {
      const uint32_t at = ptx::map_to_rank(ptx::smem_u32(s_range), (uint32_t)r);
      least_all = min(least_all, (uint32_t)ld_cluster(at));
      least_above = min(least_above, (uint32_t)ld_cluster(at + 4u));
      most = max(most, (uint32_t)ld_cluster(at + 8u));
      above += ld_cluster(at + 12u);
    }
    if (need <= above) {
      low = least_above + (kZero + 1u);
      high = most - 1u;
    } else {
      need -= above;
      low = least_all + 1u;
      high = kZero;
    }
    ranged = true;
    if (PER > 0) {
#pragma unroll
      for (int e = 0; e < STEP; ++e) u[e] = place(u[e]);
    }
    int left = 32 - __clz((int)(high - low + 1u));       // low bits that are not settled: at most 31
    uint32_t prefix = 0u;
    while (left > 0) {
      const int bits = min(left, 11), shift = left - bits;
      const uint32_t bins = (1u << bits) - 1u, from = max(prefix, 1u), size = prefix + (1u << left) - from;
      left = shift;
      for (int i = tid; i < kSelectBins; i += THREADS) s_hist[i] = 0;
      __syncthreads();
      each([&](uint32_t x, int) {
        if (x - from < size) atomicAdd(&s_hist[(x >> shift) & bins], 1);
      });
      meet();
      // the digit of the need-th largest: thread t holds digits bins - BINS t downwards, over all CTAs
      const int top = (int)bins - BINS * tid;
      int c[BINS], sum = 0;
#pragma unroll
      for (int e = 0; e < BINS; ++e) c[e] = 0;
      if (top >= 0) {
        if (ctas == 1) {
#pragma unroll
          for (int e = 0; e < BINS; ++e) c[e] = top >= e ? s_hist[top - e] : 0;
        } else {
          for (int r = 0; r < ctas; ++r) {
            const uint32_t at = ptx::map_to_rank(ptx::smem_u32(s_hist), (uint32_t)r);
#pragma unroll
            for (int e = 0; e < BINS; ++e) c[e] += top >= e ? ld_cluster(at + 4u * (uint32_t)(top - e)) : 0;
          }
        }
      }
#pragma unroll
      for (int e = 0; e < BINS; ++e) sum += c[e];
      int incl = sum;
#pragma unroll
      for (int d = 1; d < 32; d <<= 1) {
        const int y = __shfl_up_sync(0xffffffffu, incl, d);
        if (lane >= d) incl += y;
      }
      if (lane == 31) s_more[warp] = incl;
      __syncthreads();
      const int others = __reduce_add_sync(0xffffffffu, lane < warp ? s_more[lane < WARPS ? lane : 0] : 0);      // warps before this one
      int before = others + incl - sum;
      if (before < need && before + sum >= need) {       // one thread
#pragma unroll
        for (int e = 0; e < BINS; ++e) {
          if (before < need && before + c[e] >= need) {
            s_prefix = prefix | (uint32_t)(top - e) << shift;
            s_need = need - before;
            s_here = c[e];
            s_found = 0;
            break;
          }
          before += c[e];
        }
      }
      meet();                                            // also: all have read the counts
      prefix = s_prefix;
      need = s_need;
      if (left > 0 && ctas == 1 && s_here <= kSelectRank) {        // few have come down to this digit: a thread for each, which counts those above it
        const uint32_t from = max(prefix, 1u), size = prefix + (1u << left) - from;
        each([&](uint32_t x, int) {
          if (x - from < size) s_hist[atomicAdd(&s_found, 1)] = (int)x;
        });
        __syncthreads();
        const int n = s_found;
        if (tid < n) {
          const uint32_t mine = (uint32_t)s_hist[tid];
          int more = 0, equal = 0;
          for (int i = 0; i < n; ++i) {
            more += (uint32_t)s_hist[i] > mine;
            equal += (uint32_t)s_hist[i] == mine;
          }
          if (more < need && more + equal >= need) {     // all threads with this number
            s_prefix = mine;
            s_need = need - more;
          }
        }
        __syncthreads();
        prefix = s_prefix;
        need = s_need;
        left = 0;
      }
    }
    least = prefix;
    ties = need;
  }
  // every number above `least` stays, and the first `ties` of those equal to it
  int more = 0, equal = 0;
  each([&](uint32_t x, int) {
    more += x > least;
    equal += x == least;
  });
  more = __reduce_add_sync(0xffffffffu, more);
  equal = __reduce_add_sync(0xffffffffu, equal);
  __syncthreads();
  if (lane == 0) {
    s_more[warp] = more;
    s_ties[warp] = equal;
  }
  __syncthreads();
  // ties and positions that stay before this warp's: those of the CTAs before, then those of the warps before
  int out = 0, tie = 0;
  if (ctas > 1) {
    const int m = __reduce_add_sync(0xffffffffu, lane < WARPS ? s_more[lane] : 0), t = __reduce_add_sync(0xffffffffu, lane < WARPS ? s_ties[lane] : 0);
    if (tid == 0) {
      s_sum[0] = m;
      s_sum[1] = t;
    }
    ptx::cluster_sync();
    for (int r = 0; r < rank; ++r) {
      const uint32_t at = ptx::map_to_rank(ptx::smem_u32(s_sum), (uint32_t)r);
      out += ld_cluster(at);
      tie += ld_cluster(at + 4u);
    }
    ptx::cluster_sync();                                 // nobody leaves while its counts are read
  }
  out += __reduce_add_sync(0xffffffffu, lane < warp ? s_more[lane < WARPS ? lane : 0] : 0);
  tie += __reduce_add_sync(0xffffffffu, lane < warp ? s_ties[lane < WARPS ? lane : 0] : 0);
  out += min(tie, ties);
  const uint32_t below = (1u << lane) - 1u;
  const bool all = tie + equal <= ties;                  // of this warp's ties; else none or some
  if (all || tie >= ties || equal == 0) {
    const uint32_t from = all ? least : least + 1u;      // (least is kStays only where all of them do)
    each([&](uint32_t x, int at) {
      const uint32_t bal = __ballot_sync(0xffffffffu, x >= from);
      const int to = out + __popc(bal & below);
      if (x >= from && (PER > 0 || to < a.budget)) kept[to] = at + lane;       // (weights that somebody changes between two reads)
      out += __popc(bal);
    });
  } else {
    each([&](uint32_t x, int at) {
      const uint32_t tied = __ballot_sync(0xffffffffu, x == least);
      const bool stays = x > least || (x == least && tie + __popc(tied & below) < ties);
      const uint32_t bal = __ballot_sync(0xffffffffu, stays);
      const int to = out + __popc(bal & below);
      if (stays && (PER > 0 || to < a.budget)) kept[to] = at + lane;
      out += __popc(bal);
      tie += __popc(tied);
    });
  }
}

template <int PER, int THREADS>
cudaError_t launch_select(const hbsa_select_keys_args& a, int ctas, cudaStream_t stream) {
  cudaLaunchAttribute attr[1] = {};
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = (unsigned)ctas;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(a.batch * a.nhead_k * ctas));
  cfg.blockDim = dim3(THREADS);
  cfg.stream = stream;
  cfg.attrs = attr;
  cfg.numAttrs = ctas > 1 ? 1 : 0;
  return cudaLaunchKernelEx(&cfg, select_keys_kernel<PER, THREADS>, a, ctas);
}

// ------------------------------------------------------------------------------------------------------------------
// Compact: kept positions ascend, so row j comes from row kept[j] >= j, and writing rows [c, d) touches no row that a later chunk still
// reads.  A CTA takes one slice of the columns of one (sequence, kv-head), of K or of V, chunk by chunk: the rows of the next
// chunk are read (their positions one chunk before), all threads meet, then the rows of this one are written.
// Bound by the way from chunk to chunk: of 13.6 warps a scheduler 5.3 wait for gathered rows and 2.3 at the meetings (8 x 4096 rows of 8 heads of 128,
// from 8192 to 32768: 62.4 us, 4.4 TB/s).
struct CompactParams {
  void* cache[2];
  Rows4 rows[2];
  const int32_t *table, *lens, *kept, *kept_lens;
  long long table_stride;
  float* weights;
  long long weights_s[2];
  FastDiv page;
  int num_pages, capacity, batch, heads, units, budget;
  int lanes, slices;                     // units of a slice, slices of K and V together
};
constexpr int kCompactUnroll = 4;

template <typename U> struct Chunk {
  U x[kCompactUnroll];
  int to[kCompactUnroll];                // where it goes: position (weights) or page, -1: nothing moves
};

// `next`: reads the positions of a chunk that load takes one call later.
template <typename U, typename Next, typename Load, typename Store>
__device__ __forceinline__ void compact_rows(int n, int row, int rows, Next next, Load load, Store store) {
  Chunk<U> a, b;
  const int step = rows * kCompactUnroll;
  next(row);
  load(a, row);
  for (int c = 0; c < n; c += 2 * step) {
    load(b, c + step + row);
    __syncthreads();
    store(a, c + row);
    load(a, c + 2 * step + row);
    __syncthreads();
    store(b, c + step + row);
  }
}

// (64 registers, the 16-byte builds spill 52 bytes)
template <typename U, int THREADS>
__global__ void __launch_bounds__(THREADS, 1024 / THREADS) compact_kernel(const __grid_constant__ CompactParams P) {
  const int parts = P.slices + (P.weights != nullptr ? 1 : 0);
  const int part = blockIdx.x % parts, bh = blockIdx.x / parts, b = bh / P.heads, h = bh % P.heads;
  const int len = cut(P.lens[b], P.capacity), n = min(cut(P.kept_lens[b], P.budget), len);
  const int32_t* kept = P.kept + (long long)bh * P.budget;
  const int32_t* table = P.table + b * P.table_stride;
  int src[kCompactUnroll];               // of the chunk that is read next
  if (part == P.slices) {                // the weights: moved alike, zero behind
    float* w = P.weights + b * P.weights_s[0] + h * P.weights_s[1];
    auto next = [&](int j0) {
#pragma unroll
      for (int e = 0; e < kCompactUnroll; ++e) {
        const int j = j0 + e * THREADS;
        src[e] = j < n ? kept[j] : -1;
      }
    };
    auto load = [&](Chunk<float>& c, int j0) {
#pragma unroll
      for (int e = 0; e < kCompactUnroll; ++e) {
        const int j = j0 + e * THREADS;
        c.to[e] = src[e] > j && src[e] < len ? j : -1;
        if (c.to[e] >= 0) c.x[e] = w[src[e]];
      }
      next(j0 + kCompactUnroll * THREADS);
    };
    auto store = [&](const Chunk<float>& c, int) {
#pragma unroll
      for (int e = 0; e < kCompactUnroll; ++e)
        if (c.to[e] >= 0) w[c.to[e]] = c.x[e];
    };
    compact_rows<float>(n, threadIdx.x, THREADS, next, load, store);
    __syncthreads();
    for (int j = n + threadIdx.x; j < len; j += THREADS) w[j] = 0.f;
    return;
  }
  const int per = P.slices / 2, which = part / per, unit = part % per * P.lanes + threadIdx.x % P.lanes;
  const int rows = THREADS / P.lanes;
  const Rows4 s = P.rows[which];
  U* const base = static_cast<U*>(P.cache[which]) + h * s.s[2] + unit * s.s[3];
  const int mine = unit < P.units ? n : 0;
  auto next = [&](int j0) {
#pragma unroll
    for (int e = 0; e < kCompactUnroll; ++e) {
      const int j = j0 + e * rows;
      src[e] = j < mine ? kept[j] : -1;
    }
  };
  auto load = [&](Chunk<U>& c, int j0) {
#pragma unroll
    for (int e = 0; e < kCompactUnroll; ++e) {
      const int j = j0 + e * rows;
      c.to[e] = -1;
      if (src[e] > j && src[e] < len) {
        int slot_from;
        const int from = table[P.page.split(src[e], slot_from)], to = table[P.page.quotient(j)];
        if (from >= 0 && from < P.num_pages && to >= 0 && to < P.num_pages) {
          c.x[e] = base[from * s.s[0] + slot_from * s.s[1]];
          c.to[e] = to;
        }
      }
    }
    next(j0 + kCompactUnroll * rows);
  };
  auto store = [&](const Chunk<U>& c, int j0) {
#pragma unroll
    for (int e = 0; e < kCompactUnroll; ++e)
      if (c.to[e] >= 0) {
        int slot;
        P.page.split(j0 + e * rows, slot);
        base[c.to[e] * s.s[0] + slot * s.s[1]] = c.x[e];
      }
  };
  compact_rows<U>(n, threadIdx.x / P.lanes, rows, next, load, store);
}

int element_bytes(int dtype) { return dtype == HBSA_DTYPE_F32 ? 4 : 2; }

// Whether rows can be moved 16 bytes at a time: base, row length and the strides of all but the last dimension (which is 1).
bool wide_rows(const void* base, const int64_t* strides, int n, int bytes) {
  if ((uintptr_t)base % 16 != 0 || strides[n - 1] != 1) return false;
  for (int i = 0; i < n - 1; ++i)
    if (strides[i] * bytes % 16 != 0) return false;
  return true;
}

int check_cache(const hbsa_cache& c) {
  if (!c.k || !c.v || !c.block_table || !c.lens) return set_last_error("the cache's k, v, block_table and lens must not be NULL"), HBSA_ERR_NULL;
  if (c.batch <= 0 || c.nhead_k <= 0 || c.headdim <= 0 || c.num_pages <= 0 || c.page_size <= 0 || c.max_pages <= 0)
    return set_last_error("batch, nhead_k, headdim, num_pages, page_size and max_pages must be positive"), HBSA_ERR_SHAPE;
  if (c.headdim > 256) return set_last_error("headdim above 256 is not supported"), HBSA_ERR_SHAPE;
  if ((int64_t)c.max_pages * c.page_size > INT32_MAX - 4096) return set_last_error("max_pages * page_size does not fit 31 bits"), HBSA_ERR_SHAPE;
  if ((int64_t)c.batch * c.nhead_k > INT32_MAX / 64) return set_last_error("batch * nhead_k is too large"), HBSA_ERR_SHAPE;
  if (c.dtype != HBSA_DTYPE_BF16 && c.dtype != HBSA_DTYPE_F16 && c.dtype != HBSA_DTYPE_F32) return set_last_error("unknown dtype"), HBSA_ERR_DTYPE;
  return 0;
}

int launched(const char* where) {
  const cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) set_last_error("%s: %s", where, cudaGetErrorString(e));
  return (int)e;
}

}  // namespace

}  // namespace hbsa

using namespace hbsa;

extern "C" {

int hbsa_append_to_cache(const hbsa_append_args* a, void* stream) {
  if (!a) return set_last_error("args is NULL"), HBSA_ERR_NULL;
  if (a->struct_bytes != sizeof(*a)) return set_last_error("hbsa_append_args.struct_bytes does not match this library"), HBSA_ERR_STRUCT;
  const hbsa_cache& c = a->cache;
  const int rc = check_cache(c);
  if (rc != 0) return rc;
  if (!a->cu_seqlens || !a->new_lens || !a->status) return set_last_error("cu_seqlens, new_lens and status must not be NULL"), HBSA_ERR_NULL;
  if (a->total < 0) return set_last_error("total must not be negative"), HBSA_ERR_SHAPE;
  if (a->total > 0 && (!a->k || !a->v)) return set_last_error("k and v must not be NULL"), HBSA_ERR_NULL;
  const int bytes = element_bytes(c.dtype);
  const bool wide = c.headdim * bytes % 16 == 0 && wide_rows(c.k, c.k_stride, 4, bytes) && wide_rows(c.v, c.v_stride, 4, bytes) &&
                    wide_rows(a->k, a->k_stride, 3, bytes) && wide_rows(a->v, a->v_stride, 3, bytes);
  const int per = wide ? 16 / bytes : 1;                 // elements of a unit
  AppendParams P = {};
  P.k = a->k;
  P.v = a->v;
  P.k_cache = c.k;
  P.v_cache = c.v;
  for (int i = 0; i < 4; ++i) {
    P.kc.s[i] = i < 3 ? c.k_stride[i] / per : c.k_stride[i];
    P.vc.s[i] = i < 3 ? c.v_stride[i] / per : c.v_stride[i];
  }
  for (int i = 0; i < 3; ++i) {
    P.k_s[i] = i < 2 ? a->k_stride[i] / per : a->k_stride[i];
    P.v_s[i] = i < 2 ? a->v_stride[i] / per : a->v_stride[i];
  }
  P.table = c.block_table;
  P.lens = c.lens;
  P.cu = a->cu_seqlens;
  P.table_stride = c.table_stride;
  P.new_lens = a->new_lens;
  P.status = a->status;
  P.num_pages = c.num_pages;
  P.page = FastDiv(c.page_size);
  P.capacity = c.max_pages * c.page_size;
  P.batch = c.batch;
  P.heads = c.nhead_k;
  P.units = c.headdim / per;
  P.total = a->total;
  auto run = [&](int64_t s_head, int64_t s_unit) { return s_unit == 1 && (s_head == P.units || P.heads == 1); };
  P.flat = run(P.kc.s[2], P.kc.s[3]) && run(P.vc.s[2], P.vc.s[3]) && run(P.k_s[1], P.k_s[2]) && run(P.v_s[1], P.v_s[2]);
  const int64_t most = 8ll * sm100_sm_count(), need = ((int64_t)a->total + 7) / 8;
  const unsigned grid = (unsigned)(need < most ? need : most) + 1;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (wide) append_kernel<uint4><<<grid, 256, 0, st>>>(P);
  else if (bytes == 2) append_kernel<uint16_t><<<grid, 256, 0, st>>>(P);
  else append_kernel<uint32_t><<<grid, 256, 0, st>>>(P);
  return launched("hbsa_append_to_cache");
}

int hbsa_select_keys(const hbsa_select_keys_args* a, void* stream) {
  if (!a) return set_last_error("args is NULL"), HBSA_ERR_NULL;
  if (a->struct_bytes != sizeof(*a)) return set_last_error("hbsa_select_keys_args.struct_bytes does not match this library"), HBSA_ERR_STRUCT;
  if (!a->key_weights || !a->lens || !a->kept || !a->kept_lens) return set_last_error("key_weights, lens, kept and kept_lens must not be NULL"), HBSA_ERR_NULL;
  if (a->batch <= 0 || a->nhead_k <= 0 || a->max_len <= 0 || a->budget <= 0) return set_last_error("batch, nhead_k, max_len and budget must be positive"), HBSA_ERR_SHAPE;
  if (a->max_len > INT32_MAX - 16384) return set_last_error("max_len does not fit 31 bits"), HBSA_ERR_SHAPE;
  if (a->n_sink < 0 || a->n_recent < 0 || (int64_t)a->n_sink + a->n_recent > a->budget)
    return set_last_error("n_sink and n_recent must not be negative, and together not above budget"), HBSA_ERR_SHAPE;
  if ((int64_t)a->batch * a->nhead_k > INT32_MAX / 64) return set_last_error("batch * nhead_k is too large"), HBSA_ERR_SHAPE;
  // CTAs of a row: as many (up to 4) as bring them down to 8192 positions each where all of them have an SM, else as few as can hold the row.
  // 16 rows of 32768 by 1, 2 and 4 CTAs: 19.7, 22.5 and 15.8 us (by 8: 47, clusters of eight full SMs do not find their places at once);
  // 16 of 9000 by 1 and 2: 15.2 and 13.1 us; 8 of 8192 by 1 and 2: 7.4 and 13.3 us.
  // The lengths are on the device, so this goes by the width of the weights.  Short rows in a wide tensor pay for it: 128 rows of 4000 take 7.7 us
  // in 8192 columns, 13.7 in 32768, 39 in 65536 and 91 in 131072 and more; cut the tensor to the longest sequence where that is known.
  const long long rows = (long long)a->batch * a->nhead_k;
  auto split = [&](int most) {
    int n = 1;
    while (n < 4 && a->max_len > n * most) n *= 2;
    return n;
  };
  int ctas = split(8192);
  if (a->max_len > ctas * 8192 || rows * ctas > sm100_sm_count()) ctas = split(32768);
  // Threads and positions a thread: 10 rows of 1000 by 256 and by 1024 threads 4.7 and 6.8 us, 128 rows 8.2 and 24.9; 128 rows of up to 32768 in
  // registers 20.4, read again for every pass 30.4.
  const int run = ((a->max_len + ctas - 1) / ctas + 31) & ~31;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  cudaError_t e;
  if (run <= 2048) e = launch_select<8, 256>(*a, ctas, st);
  else if (run <= 8192) e = launch_select<8, 1024>(*a, ctas, st);
  else if (run <= 32768) e = launch_select<32, 1024>(*a, ctas, st);
  else e = launch_select<0, 1024>(*a, ctas, st);
  if (e != cudaSuccess) return set_last_error("hbsa_select_keys: %s", cudaGetErrorString(e)), (int)e;
  return 0;
}

int hbsa_compact_cache(const hbsa_compact_args* a, void* stream) {
  if (!a) return set_last_error("args is NULL"), HBSA_ERR_NULL;
  if (a->struct_bytes != sizeof(*a)) return set_last_error("hbsa_compact_args.struct_bytes does not match this library"), HBSA_ERR_STRUCT;
  const hbsa_cache& c = a->cache;
  const int rc = check_cache(c);
  if (rc != 0) return rc;
  if (!a->kept || !a->kept_lens) return set_last_error("kept and kept_lens must not be NULL"), HBSA_ERR_NULL;
  if (a->budget <= 0) return set_last_error("budget must be positive"), HBSA_ERR_SHAPE;
  const int bytes = element_bytes(c.dtype);
  const bool wide = c.headdim * bytes % 16 == 0 && wide_rows(c.k, c.k_stride, 4, bytes) && wide_rows(c.v, c.v_stride, 4, bytes);
  const int per = wide ? 16 / bytes : 1;
  CompactParams P = {};
  P.cache[0] = c.k;
  P.cache[1] = c.v;
  for (int i = 0; i < 4; ++i) {
    P.rows[0].s[i] = i < 3 ? c.k_stride[i] / per : c.k_stride[i];
    P.rows[1].s[i] = i < 3 ? c.v_stride[i] / per : c.v_stride[i];
  }
  P.table = c.block_table;
  P.lens = c.lens;
  P.kept = a->kept;
  P.kept_lens = a->kept_lens;
  P.table_stride = c.table_stride;
  P.weights = a->key_weights;
  P.weights_s[0] = a->weights_stride[0];
  P.weights_s[1] = a->weights_stride[1];
  P.num_pages = c.num_pages;
  P.page = FastDiv(c.page_size);
  P.capacity = c.max_pages * c.page_size;
  P.batch = c.batch;
  P.heads = c.nhead_k;
  P.units = c.headdim / per;
  P.budget = a->budget;
  // Slices of 64 bytes where that gives every SM more than one CTA, else of 32 and, for many rows, CTAs of 1024 threads, whose chunks are longer
  // (chunk by chunk costs a round trip).  64 bytes by 256 threads against the choice, in us: 3 x 2 of 5509 rows of 256 bytes 27.2, 12.3; 1 x 8 33.2,
  // 14.4; 2 x 8 (128 CTAs: 64 bytes by 1024 threads) 41.5, 25.6; 4 x 8 of 1000 rows of 128 bytes (32 bytes by 256 threads) 9.6, 7.1.  Where there are
  // enough CTAs: 8 x 8 of 4096 rows 62.4, with 32 bytes 67.6, with 1024 threads 71.6.
  auto slice = [&](int lanes) {
    while (wide && lanes > 1 && lanes >= 2 * P.units) lanes /= 2;
    P.lanes = lanes;
    P.slices = 2 * ((P.units + lanes - 1) / lanes);
    return (long long)c.batch * c.nhead_k * P.slices;
  };
  const int sms = sm100_sm_count();
  const long long ctas = slice(wide ? 4 : 32);
  const bool few = wide && ctas <= sms, many_rows = few && a->budget > 1024 && a->budget <= 1 << 30;       // (offsets behind the last row stay below 2^31)
  if (few && (!many_rows || 2 * ctas <= sms)) slice(2);
  const unsigned grid = (unsigned)(c.batch * c.nhead_k) * (unsigned)(P.slices + (P.weights ? 1 : 0));
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (many_rows) compact_kernel<uint4, 1024><<<grid, 1024, 0, st>>>(P);
  else if (wide) compact_kernel<uint4, 256><<<grid, 256, 0, st>>>(P);
  else if (bytes == 2) compact_kernel<uint16_t, 256><<<grid, 256, 0, st>>>(P);
  else compact_kernel<uint32_t, 256><<<grid, 256, 0, st>>>(P);
  return launched("hbsa_compact_cache");
}

}  // extern "C"
