// The attention weight that the queries of a block-sparse call give to every key:
//     w[j, hk] = sum over rows i that see key j and q-heads h of the group of exp(scale q_ih . k_j - lse_ih)
// with the forward's lse: the column sums of P, which the softmax never holds at one place.  Summed over prompts and decoding steps
// (hbsa_decode.cu) they say which keys of a cache can go (hbsa_select_keys).
//
// exp(scale q.k - lse) is 2^(s scale log2 e - lse log2 e), one multiply-add of fp32 and an exponential (exp2f here, ex2.approx, good to 2^-22, on the
// tensor cores).  lse log2 e is rounded once more when it is prepared, to 2^-24 of it.  Against 64 bits that costs 3.3e-7 and 3.7e-7 where natural
// exponentials in fp32 cost 1.1e-7 and 0.9e-7 (weights of 16-bit prompts); they would take another multiplication for every pair.
//
// This file: the entry point, the preparation kernel, and the CUDA-core kernel for fp32, odd strides and head dimensions.
// One cluster = 64 keys of one (kv-head, k-block).  The rows of the active q-blocks stand in one line, which is cut into tiles of 64 that the
// cluster's CTAs take in turn: thread = 4 keys x 4 rows, whose products it adds up from shared memory.  Bound by the multiplications and the way from
// tile to tile (barriers, loads): 2 x 4096 tokens, 8 heads of 128, 30 % of the blocks: 579 us, 21 TFLOP/s; one CTA per 64 keys with 4 rows x 1 key a
// thread took 1160 us, and with few keys (2048 x 2 kv-heads) 516 instead of 62 us.
#include <string.h>

#include "hbsa_key_weights.cuh"
#include "sm100_common.cuh"

namespace hbsa {

namespace {

constexpr float kLog2e = 1.4426950408889634f;
constexpr int kKeys = 64, kRows = 64, kThreads = 256;

// The k-blocks by the number of rows that may see them, most first, so that the items that end a launch are short.  One CTA, 256 classes, which are
// counted in the workspace: shared memory here would keep CTAs of the next kernel from starting beside this one (4 us of 57).
__device__ __forceinline__ void key_weights_order(const KeyWeightsParams& P) {
  __shared__ int s_warp[8];
  const Problem& p = P.p;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  int* const counts = P.sp.classes;
  counts[tid] = 0;
  int most = 1;
  for (int b = tid; b < p.batch; b += 256) most = max(most, p.cu_q[b + 1] - p.cu_q[b]);
  most = __reduce_max_sync(0xffffffffu, most);
  if (lane == 0) s_warp[warp] = most;
  __syncthreads();
  most = __reduce_max_sync(0xffffffffu, s_warp[lane & 7]);
  auto class_of = [&](int kb) {
    const int b = sample_of_block(P.ws.cnk, p.batch, kb), q_len = p.cu_q[b + 1] - p.cu_q[b], off = p.cu_k[b + 1] - p.cu_k[b] - q_len;
    const int unseen = p.causal ? max(0, (kb - P.ws.cnk[b]) * p.kbs - off) : 0, rows = max(0, q_len - unseen);
    return 255 - (int)(255ll * rows / most);
  };
  for (int kb = tid; kb < p.num_k_block; kb += 256) atomicAdd(counts + class_of(kb), 1);
  __syncthreads();
  const int mine = atomicAdd(counts + tid, 0);
  int incl = mine;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const int y = __shfl_up_sync(0xffffffffu, incl, d);
    if (lane >= d) incl += y;
  }
  if (lane == 31) s_warp[warp] = incl;
  __syncthreads();
  const int before = incl - mine + __reduce_add_sync(0xffffffffu, lane < warp ? s_warp[lane & 7] : 0);
  atomicExch(counts + tid, before);
  __syncthreads();
  for (int kb = tid; kb < p.num_k_block; kb += 256) P.sp.order[atomicAdd(counts + class_of(kb), 1)] = kb;
}

// -lse log2 e of every row in the order of the tiles (-inf: nothing to add), zeros for keys outside every sample, the cleared work cursor, and
// (one CTA more) the order of the k-blocks.
__global__ void __launch_bounds__(256) key_weights_prep_kernel(const __grid_constant__ KeyWeightsParams P, const float* __restrict__ lse) {
  const Problem& p = P.p;
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  if (blockIdx.x == 0 && threadIdx.x < 32) P.sp.cursor[threadIdx.x] = 0;
  asm volatile("griddepcontrol.wait;" ::: "memory");               // the schedule
  const bool ok = P.ws.status[0] == HBSA_STATUS_OK;
  key_weights_outside(P, !ok);
  if (!ok) return;
  if (P.sorted && blockIdx.x == gridDim.x - 1) {
    key_weights_order(P);
    return;
  }
  // a warp takes 256 values of a q-block at a time, in the order of lse (rows, then heads)
  const int lane = threadIdx.x & 31, n = p.qbs * p.nhead_q, chunks = (n + 255) / 256;
  const long long todo = (long long)p.num_q_block * chunks;
  for (long long u = blockIdx.x * 8 + (threadIdx.x >> 5); u < todo; u += (gridDim.x - P.sorted) * 8) {
    const int qb = (int)(u / chunks), first = (int)(u % chunks) * 256 + lane;
    const RowGeom g = row_geometry(p, P.ws.cnq, P.ws.cnk, P.ws.qb2b, qb);
    const float* src = lse + (long long)g.q_begin * p.nhead_q;
    // (rows that cu_q puts outside the tensors add nothing and are not read)
    const int missing = max(0, min(-g.q_begin, p.qbs)) * p.nhead_q, there = max(0, min(g.q_end, P.total_q) - g.q_begin) * p.nhead_q;
    float x[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = first + 32 * e >= missing && first + 32 * e < there ? src[first + 32 * e] : -INFINITY;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const int i = first + 32 * e, tok = i / p.nhead_q, h = i - tok * p.nhead_q;
      if (i < n) P.sp.neg_lse[(((long long)(h >> P.gp_shift) * p.num_q_block + qb) * p.qbs + tok) * P.gp + (h & (P.gp - 1))] = x[e] == -INFINITY ? -INFINITY : -x[e] * kLog2e;
    }
  }
}

struct KeyWeightsStrides { long long q0, q1, q2, k0, k1, k2; };

constexpr int kList = 1024;                      // q-blocks that are looked at together

// VEC: elements of a 16-byte unit, or 1.
template <typename T, int DP, int VEC>
__global__ void __launch_bounds__(kThreads, DP == 256 ? 1 : 2) key_weights_generic_kernel(const __grid_constant__ KeyWeightsParams P, const T* __restrict__ q,
                                                                                          const T* __restrict__ k, KeyWeightsStrides st, int ctas) {
  constexpr int KS = DP + 4;                     // rows 4 floats apart modulo 32: 16-byte reads of 8 rows hit all banks
  const Problem& p = P.p;
  if (P.ws.status[0] != HBSA_STATUS_OK) return;
  extern __shared__ __align__(16) float sm[];
  float* const sK = sm;                          // [kKeys][KS]
  float* const sQ = sK + kKeys * KS;             // [kRows][KS]
  __shared__ long long s_at[kRows];              // element offset of a row of q, or -1
  __shared__ float s_nl[kRows], s_sum[16][kKeys];
  __shared__ int s_pos[kRows], s_list[kList], s_count[kThreads / 32];
  const int subs = (p.kbs + kKeys - 1) / kKeys, item = blockIdx.x / ctas, rank = blockIdx.x - item * ctas, kb = item / subs, sub = item % subs, hk = blockIdx.y;
  const int b = sample_of_block(P.ws.cnk, p.batch, kb);
  const int k_begin = p.cu_k[b], k_len = p.cu_k[b + 1] - k_begin, q_begin = p.cu_q[b], q_len = p.cu_q[b + 1] - q_begin, off = k_len - q_len;
  const int blk0 = (kb - P.ws.cnk[b]) * p.kbs, k0 = blk0 + sub * kKeys, n_keys = min(kKeys, min(blk0 + p.kbs, k_len) - k0);
  if (n_keys <= 0) return;                       // the whole cluster
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, tx = tid & 15, ty = tid >> 4;
  // 64 rows of K or Q: at(row) is the row's offset, or -1
  auto load = [&](float* to, const T* from, long long stride, auto&& at) {
    const int units = DP / VEC, there = p.headdim / VEC;
#pragma unroll 4
    for (int i = tid; i < 64 * units; i += kThreads) {
      const int r = i / units, u = i % units;
      const long long row = at(r);
      float* const dst = to + r * KS + u * VEC;
      const bool on = row >= 0 && u < there;
      if (VEC > 1) {
        union { uint4 w; T x[16 / sizeof(T)]; } in;
        in.w = make_uint4(0u, 0u, 0u, 0u);
        if (on) in.w = *reinterpret_cast<const uint4*>(from + row + u * VEC);
#pragma unroll
        for (int e = 0; e < VEC; ++e) dst[e] = to_f(in.x[e]);
      } else {
        dst[0] = on ? to_f(from[row + u * stride]) : 0.f;
      }
    }
  };
  load(sK, k, st.k2, [&](int r) { return r < n_keys && key_is_there(P, k_begin + k0 + r) ? (long long)(k_begin + k0 + r) * st.k0 + hk * st.k1 : -1ll; });
  const int qb0 = P.ws.cnq[b], n_qb = P.ws.cnq[b + 1] - qb0;
  const long long block_rows = (long long)p.qbs * p.group;        // (token, head) pairs of a q-block, heads innermost
  float sum[4] = {0.f, 0.f, 0.f, 0.f};
  for (int first = 0; first < n_qb; first += kList) {
    // the active q-blocks among the next ones, ascending
    int count = 0;
    for (int i0 = first; i0 < min(first + kList, n_qb); i0 += kThreads) {
      const int i = i0 + tid;
      bool on = false;
      if (i < n_qb && !(p.causal && min((i + 1) * (long long)p.qbs, (long long)q_len) - 1 + off < k0)) {
        if (p.csr_ptr != nullptr) {
          const long long row = (long long)hk * p.num_q_block + qb0 + i;
          const int e1 = p.csr_ptr[row + 1], e = lower_bound_i32(p.csr_idx, p.csr_ptr[row], e1, kb);
          on = e < e1 && p.csr_idx[e] == kb;
        } else {
          on = p.mask[hk * p.mask_s0 + (long long)(qb0 + i) * p.mask_s1 + (long long)kb * p.mask_s2] != 0;
        }
      }
      const uint32_t bal = __ballot_sync(0xffffffffu, on);
      __syncthreads();                           // the counts before, and the list before, have been read
      if (lane == 0) s_count[warp] = __popc(bal);
      __syncthreads();
      int at = count;
#pragma unroll
      for (int w = 0; w < kThreads / 32; ++w) {
        if (w < warp) at += s_count[w];
        count += s_count[w];
      }
      if (on) s_list[at + __popc(bal & ((1u << lane) - 1u))] = i;
    }
    const long long n_tiles = (count * block_rows + kRows - 1) / kRows;
    for (long long tile = rank; tile < n_tiles; tile += ctas) {
      __syncthreads();                           // the list is there, and the tile before is used up
      if (tid < kRows) {
        const long long f = tile * kRows + tid, blk = quotient(f, block_rows);
        long long at = -1;
        float nl = -INFINITY;
        int row = 0;
        if (blk < count) {
          const int i = s_list[blk], r = (int)(f - blk * block_rows), tok = r / p.group, h = hk * p.group + r - tok * p.group;
          row = i * p.qbs + tok;
          if (row < q_len) {
            nl = P.sp.neg_lse[(((long long)(h >> P.gp_shift) * p.num_q_block + qb0 + i) * p.qbs + tok) * P.gp + (h & (P.gp - 1))];
            if (nl != -INFINITY) at = (long long)(q_begin + row) * st.q0 + h * st.q1;
          }
        }
        s_at[tid] = at;
        s_nl[tid] = nl;
        s_pos[tid] = row + off;
      }
      __syncthreads();
      load(sQ, q, st.q2, [&](int r) { return s_at[r]; });
      __syncthreads();
      float s[4][4];
#pragma unroll
      for (int y = 0; y < 4; ++y)
#pragma unroll
        for (int x = 0; x < 4; ++x) s[y][x] = 0.f;
      const float *const kr = sK + tx * KS, *const qr = sQ + ty * KS;
#pragma unroll 2
      for (int d = 0; d < DP; d += 4) {
        float4 a[4], c[4];
#pragma unroll
        for (int x = 0; x < 4; ++x) {
          a[x] = *reinterpret_cast<const float4*>(kr + 16 * x * KS + d);
          c[x] = *reinterpret_cast<const float4*>(qr + 16 * x * KS + d);
        }
#pragma unroll
        for (int y = 0; y < 4; ++y)
#pragma unroll
          for (int x = 0; x < 4; ++x) s[y][x] = fmaf(a[x].x, c[y].x, fmaf(a[x].y, c[y].y, fmaf(a[x].z, c[y].z, fmaf(a[x].w, c[y].w, s[y][x]))));
      }
      float tile_sum[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int y = 0; y < 4; ++y) {
        const int r = ty + 16 * y;
        const float nl = s_nl[r];
        const int pos = s_pos[r];
        if (nl == -INFINITY) continue;
#pragma unroll
        for (int x = 0; x < 4; ++x)
          if (!p.causal || pos >= k0 + tx + 16 * x) tile_sum[x] += exp2f(fmaf(s[y][x], P.scale_log2, nl));
      }
#pragma unroll
      for (int x = 0; x < 4; ++x) sum[x] += tile_sum[x];
    }
  }
#pragma unroll
  for (int x = 0; x < 4; ++x) s_sum[ty][tx + 16 * x] = sum[x];
  __syncthreads();
  float total = 0.f;
  if (tid < kKeys) {
#pragma unroll
    for (int y = 0; y < 16; ++y) total += s_sum[y][tid];
  }
  if (ctas > 1) {                                // the CTAs' sums, in the order of their ranks
    __syncthreads();
    if (tid < kKeys) s_sum[0][tid] = total;
    ptx::cluster_sync();
    if (rank == 0 && tid < kKeys) {
      for (int r = 1; r < ctas; ++r) {
        float x;
        asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(x) : "r"(ptx::map_to_rank(ptx::smem_u32(&s_sum[0][tid]), (uint32_t)r)) : "memory");
        total += x;
      }
    }
    ptx::cluster_sync();                         // nobody leaves while its sums are read
  }
  if (rank == 0 && tid < n_keys && key_is_there(P, k_begin + k0 + tid)) P.out[(long long)(k_begin + k0 + tid) * p.nhead_k + hk] = total;
}

template <typename T, int DP, int VEC>
int launch_generic(const KeyWeightsParams& P, const hbsa_forward_args& a, cudaStream_t stream) {
  constexpr size_t smem = sizeof(float) * (size_t)((kKeys + kRows) * (DP + 4));
  static SmemOptIn opt_in;
  cudaError_t e = opt_in.once(reinterpret_cast<const void*>(key_weights_generic_kernel<T, DP, VEC>), (int)smem);
  if (e != cudaSuccess) return set_last_error("hbsa_key_weights: %s", cudaGetErrorString(e)), (int)e;
  const KeyWeightsStrides st = {a.q_stride[0], a.q_stride[1], a.q_stride[2], a.k_stride[0], a.k_stride[1], a.k_stride[2]};
  // CTAs of a cluster: as long as there are SMs for them, and two tiles for each where all q-blocks are active (with one CTA, four and up to eight:
  // 4096 tokens, 8 on 2 heads of 128 728, 297 and 298 us; 2048 tokens, 4 on 2 heads 205, 80 and 62; 5 x 64..102, 16 on 4 heads 61, 37 and 37)
  const long long pieces = (long long)P.p.num_k_block * ((P.p.kbs + kKeys - 1) / kKeys), items = pieces * P.p.nhead_k;
  if (pieces > INT32_MAX / 8) return set_last_error("num_k_block * k_block_size is too large"), HBSA_ERR_SHAPE;
  const long long tiles = (long long)P.p.num_q_block * P.p.qbs * P.p.group / ((long long)kRows * P.p.batch);
  int ctas = 1;
  while (ctas < 8 && items * ctas < 2ll * sm100_sm_count() && tiles >= 4 * ctas) ctas *= 2;
  cudaLaunchAttribute attr[1] = {};
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = (unsigned)ctas;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(pieces * ctas), (unsigned)P.p.nhead_k);
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cfg.attrs = attr;
  cfg.numAttrs = ctas > 1 ? 1 : 0;
  e = cudaLaunchKernelEx(&cfg, key_weights_generic_kernel<T, DP, VEC>, P, static_cast<const T*>(a.q), static_cast<const T*>(a.k), st, ctas);
  return e == cudaSuccess ? 0 : (set_last_error("hbsa_key_weights: %s", cudaGetErrorString(e)), (int)e);
}
template <typename T>
int launch_generic_of(const KeyWeightsParams& P, const hbsa_forward_args& a, cudaStream_t stream) {
  constexpr int VEC = 16 / (int)sizeof(T);
  bool vec = a.headdim % VEC == 0 && a.q_stride[2] == 1 && a.k_stride[2] == 1 && (uintptr_t)a.q % 16 == 0 && (uintptr_t)a.k % 16 == 0;
  for (int i = 0; i < 2; ++i) vec = vec && a.q_stride[i] % VEC == 0 && a.k_stride[i] % VEC == 0;
  if (a.headdim <= 64) return vec ? launch_generic<T, 64, VEC>(P, a, stream) : launch_generic<T, 64, 1>(P, a, stream);
  if (a.headdim <= 128) return vec ? launch_generic<T, 128, VEC>(P, a, stream) : launch_generic<T, 128, 1>(P, a, stream);
  return vec ? launch_generic<T, 256, VEC>(P, a, stream) : launch_generic<T, 256, 1>(P, a, stream);
}

// A block that holds every packed row there is: larger ones are no different, as every sample is one block of them, and cost workspace.
int32_t block_within(int32_t block, int32_t total) {
  const long long all = ((long long)total + 127) / 128 * 128;
  return total > 0 && block % 16 == 0 && block > all ? (int32_t)all : block;
}

size_t carve_key_weights(const hbsa_forward_args& a, char* base, KeyWeightsSpace* s) {
  char* p = base;
  auto take = [&](size_t bytes) { char* r = p; p += (bytes + 255) / 256 * 256; return r; };
  s->cursor = reinterpret_cast<unsigned long long*>(take(256));
  s->neg_lse = reinterpret_cast<float*>(take((size_t)a.num_q_block * a.q_block_size * a.nhead_q * 4));
  s->classes = reinterpret_cast<int32_t*>(take(256 * 4));
  s->order = reinterpret_cast<int32_t*>(take(a.num_k_block <= kKwSorted ? (size_t)a.num_k_block * 4 : 0));
  return (size_t)(p - base);
}

}  // namespace

}  // namespace hbsa

extern "C" {

size_t hbsa_key_weights_workspace_bytes(const hbsa_key_weights_args* args) {
  if (!args || args->struct_bytes != sizeof(*args) || args->fwd.num_q_block <= 0 || args->fwd.q_block_size <= 0 || args->fwd.nhead_q <= 0) return 0;
  hbsa::KeyWeightsSpace s;
  hbsa_forward_args a = args->fwd;
  a.q_block_size = hbsa::block_within(a.q_block_size, a.total_q);
  return hbsa::carve_key_weights(a, nullptr, &s);
}

int hbsa_key_weights(const hbsa_key_weights_args* args, void* stream_) {
  using namespace hbsa;
  if (!args) return set_last_error("args is NULL"), HBSA_ERR_NULL;
  if (args->struct_bytes != sizeof(*args)) return set_last_error("hbsa_key_weights_args.struct_bytes does not match this library"), HBSA_ERR_STRUCT;
  KeyWeightsParams P;
  memset(&P, 0, sizeof(P));
  hbsa_forward_args a = args->fwd;
  a.q_block_size = block_within(a.q_block_size, a.total_q);
  a.k_block_size = block_within(a.k_block_size, a.total_k);
  a.v = a.k;                                   // not used: the checks of a forward apply to what is there
  a.o = const_cast<void*>(a.q);
  for (int i = 0; i < 3; ++i) {
    a.v_stride[i] = a.k_stride[i];
    a.o_stride[i] = a.q_stride[i];
  }
  int rc = make_problem(&a, true, &P.p);
  if (rc != 0) return rc;
  if ((int64_t)a.q_block_size * a.nhead_q > INT32_MAX - 512) return set_last_error("q-blocks of more than 2^31 rows (tokens x q-heads) are not supported"), HBSA_ERR_SHAPE;
  if (!a.lse || !args->weights || !args->partial_workspace) return set_last_error("lse, weights and partial_workspace must not be NULL"), HBSA_ERR_NULL;
  if (args->partial_workspace_bytes < carve_key_weights(a, static_cast<char*>(args->partial_workspace), &P.sp))
    return set_last_error("partial_workspace is smaller than hbsa_key_weights_workspace_bytes()"), HBSA_ERR_WORKSPACE;
  if ((uintptr_t)args->partial_workspace % 256 != 0) return set_last_error("partial_workspace must be 256-byte aligned"), HBSA_ERR_WORKSPACE;
  const int impl = select_impl(&a, P.p);
  if (impl < 0) return impl;
  P.ws = make_workspace(a.workspace, P.p.nhead_k, P.p.num_q_block, P.p.num_k_block, P.p.batch);
  P.out = args->weights;
  P.total_q = a.total_q;
  P.total_k = a.total_k;
  P.scale_log2 = P.p.scale * kLog2e;
  P.wait_budget = sm100_wait_budget();
  P.debug_stall = sm100_debug_stall();
  cudaStream_t stream = static_cast<cudaStream_t>(stream_);
  auto failed = [](cudaError_t e) { return set_last_error("hbsa_key_weights: %s", cudaGetErrorString(e)), (int)e; };
  cudaError_t e = launch_schedule(P.p, P.ws, nullptr, stream);
  if (e != cudaSuccess) return failed(e);
  P.gp = 1;                                    // q-heads side by side in a tile: the largest power of two that divides the group
  P.gp_shift = 0;
  while (P.gp < 64 && P.p.group % (P.gp * 2) == 0) {
    P.gp *= 2;
    ++P.gp_shift;
  }
  const long long warps = ((long long)a.num_q_block * (((long long)a.q_block_size * a.nhead_q + 255) / 256) + 7) / 8, most = 8ll * sm100_sm_count();
  cudaLaunchAttribute attr[1] = {};
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg = {};
  // Items in order, all heads of a k-block together, where some CTAs get more than one item.  Natural order (head by head) against this one, in us:
  // causal 2 x 8192 at 10 % 86.6, 78.2; 2 x 4096 at 90 % 132, 106; not causal 2 x 1000..8192 58.1, 57.0, 33 x 20..900 56.5, 52.0, blocks of 48
  // 54.9, 49.6; 16384 with 32 heads (134 MB of rows) 209, 199, on 8 kv-heads 258, 214.  Rows beyond the L2 are better read head by head: with 48 heads
  // (201 MB) 296, 298.
  const long long items = (long long)a.num_k_block * P.p.nhead_k * ((a.k_block_size + 127) / 128), streamed = (long long)a.total_q * a.nhead_q * a.headdim * 2;
  P.sorted = impl == HBSA_IMPL_SM100 && a.num_k_block > 1 && a.num_k_block <= kKwSorted && items > 2ll * sm100_sm_count() && streamed <= 160ll << 20;
  cfg.gridDim = dim3((unsigned)(warps < most ? warps : most) + (unsigned)P.sorted);
  cfg.blockDim = dim3(256);
  cfg.stream = stream;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  if ((e = cudaLaunchKernelEx(&cfg, key_weights_prep_kernel, P, static_cast<const float*>(a.lse))) != cudaSuccess) return failed(e);
  if (impl == HBSA_IMPL_SM100) {
    const char* text = "";
    rc = launch_key_weights_sm100(P, a, stream, &text);
    return rc != 0 ? (set_last_error("hbsa_key_weights: %s", text), rc) : 0;
  }
  if (a.dtype == HBSA_DTYPE_BF16) return launch_generic_of<__nv_bfloat16>(P, a, stream);
  if (a.dtype == HBSA_DTYPE_F16) return launch_generic_of<__half>(P, a, stream);
  return launch_generic_of<float>(P, a, stream);
}

}  // extern "C"
