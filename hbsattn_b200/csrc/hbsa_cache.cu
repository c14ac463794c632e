// Writing into a paged key-value cache, choosing what stays when it is cut down, and moving that together.
// All three are bound by memory: every byte is read once and written once.
#include <string.h>

#include "sm100_common.cuh"

namespace hbsa {

namespace {

// Rows are copied in units of U: 16 bytes where bases, strides and the row length allow it, one element otherwise.
struct Rows4 { long long s[4]; };        // strides in units: page, slot, head, unit

// ------------------------------------------------------------------------------------------------------------------
// Append: one warp per new token, K and V together.  The last block writes the new lengths and the status.
struct AppendParams {
  const void *k, *v;
  void *k_cache, *v_cache;
  Rows4 kc, vc;
  long long k_s[3], v_s[3];              // token, head, unit
  const int32_t *table, *lens, *cu;
  long long table_stride;
  int32_t *new_lens, *status;
  int num_pages, page, capacity, batch, heads, units, total;
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
    const int raw = P.lens[b], len = cut(raw, P.capacity), n = max(0, P.cu[b + 1] - P.cu[b]);
    const int end = (int)min((long long)len + n, (long long)P.capacity);
    bool bad = raw != len || (long long)len + n > P.capacity;
    if (end > len)
      for (int i = len / P.page + tid % per; i <= (end - 1) / P.page; i += per) {
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
    const long long pos = (long long)cut(P.lens[b], P.capacity) + (tok - P.cu[b]);
    if (pos >= P.capacity) continue;
    const int page = P.table[b * P.table_stride + (int)pos / P.page], slot = (int)pos % P.page;
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
// Select: radix select of the smallest weight that stays, then one pass that writes positions in order.
constexpr int kSelectThreads = 1024;

// Weights as unsigned numbers in the same order; both zeros are one, NaN is the largest.
__device__ __forceinline__ uint32_t order_of(float x) {
  if (x != x) return 0xffffffffu;
  const uint32_t u = __float_as_uint(x + 0.f);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}

__global__ void __launch_bounds__(kSelectThreads) select_keys_kernel(const __grid_constant__ hbsa_select_keys_args a) {
  constexpr int WARPS = kSelectThreads / 32;
  __shared__ int s_hist[256];
  __shared__ int s_more[WARPS], s_ties[WARPS];
  __shared__ uint32_t s_prefix;
  __shared__ int s_need;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int b = blockIdx.x / a.nhead_k, h = blockIdx.x % a.nhead_k;
  const int len = cut(a.lens[b], a.max_len);
  const float* w = a.key_weights + b * a.weights_stride[0] + h * a.weights_stride[1];
  int32_t* kept = a.kept + (long long)blockIdx.x * a.budget;
  if (h == 0 && tid == 0) a.kept_lens[b] = min(len, a.budget);
  if (len <= a.budget) {
    for (int i = tid; i < a.budget; i += kSelectThreads) kept[i] = i < len ? i : -1;
    return;
  }
  const int lo = a.n_sink, hi = len - a.n_recent;        // the positions that compete; n_sink + n_recent <= budget < len
  int need = a.budget - a.n_sink - a.n_recent;
  uint32_t prefix = 0;
  if (need > 0) {
    for (int shift = 24; shift >= 0; shift -= 8) {
      if (tid < 256) s_hist[tid] = 0;
      __syncthreads();
      const uint32_t known = shift == 24 ? 0u : 0xffffffffu << (shift + 8);
      for (int i = lo + tid; i < hi; i += kSelectThreads) {
        const uint32_t u = order_of(w[i]);
        if ((u & known) == prefix) atomicAdd(&s_hist[(u >> shift) & 255u], 1);
      }
      __syncthreads();
      if (warp == 0) {                                   // the digit of the need-th largest: lane l holds digits 255 - 8 l ...
        int c[8], sum = 0;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          c[e] = s_hist[255 - 8 * lane - e];
          sum += c[e];
        }
        int incl = sum;
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
          const int y = __shfl_up_sync(0xffffffffu, incl, d);
          if (lane >= d) incl += y;
        }
        int before = incl - sum;
        if (before < need && incl >= need) {
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            if (before < need && before + c[e] >= need) {
              s_prefix = prefix | (uint32_t)(255 - 8 * lane - e) << shift;
              s_need = need - before;
              break;
            }
            before += c[e];
          }
        }
      }
      __syncthreads();
      prefix = s_prefix;
      need = s_need;
      __syncthreads();
    }
  }
  // every weight above `prefix` stays, and the first `need` of those equal to it (none competes where nothing is needed)
  const bool any = a.budget > a.n_sink + a.n_recent;
  const int seg = (len + WARPS - 1) / WARPS, s0 = min(warp * seg, len), s1 = min(s0 + seg, len);
  auto kind = [&](int i) -> int {                        // 2: stays, 1: a tie, 0: goes
    if (i >= s1) return 0;
    if (i < lo || i >= hi) return 2;
    if (!any) return 0;
    const uint32_t u = order_of(w[i]);
    return u > prefix ? 2 : u == prefix ? 1 : 0;
  };
  int more = 0, ties = 0;
  for (int i = s0 + lane; i < s1; i += 32) {
    const int x = kind(i);
    more += x == 2;
    ties += x == 1;
  }
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) {
    more += __shfl_xor_sync(0xffffffffu, more, d);
    ties += __shfl_xor_sync(0xffffffffu, ties, d);
  }
  if (lane == 0) {
    s_more[warp] = more;
    s_ties[warp] = ties;
  }
  __syncthreads();
  int out = 0, tie = 0;
  for (int i = 0; i < warp; ++i) {
    out += s_more[i] + min(max(need - tie, 0), s_ties[i]);
    tie += s_ties[i];
  }
  for (int base = s0; base < s1; base += 32) {
    const int x = kind(base + lane);
    const uint32_t below = (1u << lane) - 1u, tied = __ballot_sync(0xffffffffu, x == 1);
    const bool stays = x == 2 || (x == 1 && tie + __popc(tied & below) < need);
    const uint32_t bal = __ballot_sync(0xffffffffu, stays);
    if (stays) kept[out + __popc(bal & below)] = base + lane;
    out += __popc(bal);
    tie += __popc(tied);
  }
}

// ------------------------------------------------------------------------------------------------------------------
// Compact: kept positions ascend, so row j comes from row kept[j] >= j, and writing rows [c, d) touches no row that a later chunk still
// reads.  A CTA takes one slice of the columns of one (sequence, kv-head), of K or of V, chunk by chunk: the rows of the next
// chunk are read, all threads meet, then the rows of this one are written.
struct CompactParams {
  void* cache[2];
  Rows4 rows[2];
  const int32_t *table, *lens, *kept, *kept_lens;
  long long table_stride;
  float* weights;
  long long weights_s[2];
  int num_pages, page, capacity, batch, heads, units, budget;
  int lanes, slices;                     // units of a slice, slices of K and V together
};
constexpr int kCompactThreads = 256, kCompactUnroll = 4;

template <typename U> struct Chunk {
  U x[kCompactUnroll];
  long long to[kCompactUnroll];          // offset in units, < 0: nothing moves
};

template <typename U, typename Load, typename Store>
__device__ __forceinline__ void compact_rows(int n, int row, int rows, Load load, Store store) {
  Chunk<U> a, b;
  const int step = rows * kCompactUnroll;
  load(a, row);
  for (int c = 0; c < n; c += 2 * step) {
    load(b, c + step + row);
    __syncthreads();
    store(a);
    load(a, c + 2 * step + row);
    __syncthreads();
    store(b);
  }
}

template <typename U>
__global__ void __launch_bounds__(kCompactThreads) compact_kernel(const __grid_constant__ CompactParams P) {
  const int parts = P.slices + (P.weights != nullptr ? 1 : 0);
  const int part = blockIdx.x % parts, bh = blockIdx.x / parts, b = bh / P.heads, h = bh % P.heads;
  const int len = cut(P.lens[b], P.capacity), n = min(cut(P.kept_lens[b], P.budget), len);
  const int32_t* kept = P.kept + (long long)bh * P.budget;
  const int32_t* table = P.table + b * P.table_stride;
  if (part == P.slices) {                // the weights: moved alike, zero behind
    float* w = P.weights + b * P.weights_s[0] + h * P.weights_s[1];
    auto load = [&](Chunk<float>& c, int j0) {
#pragma unroll
      for (int e = 0; e < kCompactUnroll; ++e) {
        const int j = j0 + e * kCompactThreads, src = j < n ? kept[j] : -1;
        c.to[e] = src > j && src < len ? j : -1;
        if (c.to[e] >= 0) c.x[e] = w[src];
      }
    };
    auto store = [&](const Chunk<float>& c) {
#pragma unroll
      for (int e = 0; e < kCompactUnroll; ++e)
        if (c.to[e] >= 0) w[c.to[e]] = c.x[e];
    };
    compact_rows<float>(n, threadIdx.x, kCompactThreads, load, store);
    __syncthreads();
    for (int j = n + threadIdx.x; j < len; j += kCompactThreads) w[j] = 0.f;
    return;
  }
  const int per = P.slices / 2, which = part / per, unit = part % per * P.lanes + threadIdx.x % P.lanes;
  const int rows = kCompactThreads / P.lanes;
  const Rows4 s = P.rows[which];
  U* const base = static_cast<U*>(P.cache[which]) + h * s.s[2] + unit * s.s[3];
  const bool mine = unit < P.units;
  auto load = [&](Chunk<U>& c, int j0) {
#pragma unroll
    for (int e = 0; e < kCompactUnroll; ++e) {
      const int j = j0 + e * rows, src = mine && j < n ? kept[j] : -1;
      c.to[e] = -1;
      if (src > j && src < len) {
        const int from = table[src / P.page], to = table[j / P.page];
        if (from >= 0 && from < P.num_pages && to >= 0 && to < P.num_pages) {
          c.x[e] = base[from * s.s[0] + src % P.page * s.s[1]];
          c.to[e] = to * s.s[0] + j % P.page * s.s[1];
        }
      }
    }
  };
  auto store = [&](const Chunk<U>& c) {
#pragma unroll
    for (int e = 0; e < kCompactUnroll; ++e)
      if (c.to[e] >= 0) base[c.to[e]] = c.x[e];
  };
  compact_rows<U>(n, threadIdx.x / P.lanes, rows, load, store);
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
  AppendParams P;
  memset(&P, 0, sizeof(P));
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
  P.page = c.page_size;
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
  if (a->max_len > INT32_MAX - 4096) return set_last_error("max_len does not fit 31 bits"), HBSA_ERR_SHAPE;
  if (a->n_sink < 0 || a->n_recent < 0 || (int64_t)a->n_sink + a->n_recent > a->budget)
    return set_last_error("n_sink and n_recent must not be negative, and together not above budget"), HBSA_ERR_SHAPE;
  if ((int64_t)a->batch * a->nhead_k > INT32_MAX / 64) return set_last_error("batch * nhead_k is too large"), HBSA_ERR_SHAPE;
  select_keys_kernel<<<(unsigned)(a->batch * a->nhead_k), kSelectThreads, 0, static_cast<cudaStream_t>(stream)>>>(*a);
  return launched("hbsa_select_keys");
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
  CompactParams P;
  memset(&P, 0, sizeof(P));
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
  P.page = c.page_size;
  P.capacity = c.max_pages * c.page_size;
  P.batch = c.batch;
  P.heads = c.nhead_k;
  P.units = c.headdim / per;
  P.budget = a->budget;
  P.lanes = wide ? 8 : 32;
  while (wide && P.lanes > 1 && P.lanes >= 2 * P.units) P.lanes /= 2;
  P.slices = 2 * ((P.units + P.lanes - 1) / P.lanes);
  const unsigned grid = (unsigned)(c.batch * c.nhead_k) * (unsigned)(P.slices + (P.weights ? 1 : 0));
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (wide) compact_kernel<uint4><<<grid, kCompactThreads, 0, st>>>(P);
  else if (bytes == 2) compact_kernel<uint16_t><<<grid, kCompactThreads, 0, st>>>(P);
  else compact_kernel<uint32_t><<<grid, kCompactThreads, 0, st>>>(P);
  return launched("hbsa_compact_cache");
}

}  // extern "C"
