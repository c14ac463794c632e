// The attention weight that the queries of a block-sparse call give to every key:
//     w[j, hk] = sum over rows i that see key j and q-heads h of the group of exp(scale q_ih . k_j - lse_ih)
// with the forward's lse: the column sums of P, which the softmax never holds at one place.  Summed over prompts and decoding steps
// (hbsa_decode.cu) they say which keys of a cache can go (hbsa_select_keys).
//
// This file: the entry point, the preparation kernel, and the CUDA-core kernel for fp32, odd strides and head dimensions.
// One CTA = 64 keys of one (kv-head, k-block); rows of the active q-blocks are streamed past them, 64 at a time.
#include <string.h>

#include "hbsa_key_weights.cuh"
#include "sm100_common.cuh"

namespace hbsa {

namespace {

constexpr float kLog2e = 1.4426950408889634f;
constexpr int kKeys = 64, kRows = 64, kThreads = 256;

template <typename T> __device__ __forceinline__ float to_f(T x);
template <> __device__ __forceinline__ float to_f<float>(float x) { return x; }
template <> __device__ __forceinline__ float to_f<__half>(__half x) { return __half2float(x); }
template <> __device__ __forceinline__ float to_f<__nv_bfloat16>(__nv_bfloat16 x) { return __bfloat162float(x); }

// -lse log2 e of every row in the order of the tiles (-inf: nothing to add), zeros for keys outside every sample, the cleared work cursor.
__global__ void __launch_bounds__(256) key_weights_prep_kernel(const __grid_constant__ KeyWeightsParams P, const float* __restrict__ lse) {
  const Problem& p = P.p;
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  if (blockIdx.x == 0 && threadIdx.x < 32) P.sp.cursor[threadIdx.x] = 0;
  asm volatile("griddepcontrol.wait;" ::: "memory");               // the schedule
  const bool ok = P.ws.status[0] == HBSA_STATUS_OK;
  key_weights_outside(P, !ok);
  if (!ok) return;
  // a warp takes 256 values of a q-block at a time, in the order of lse (rows, then heads)
  const int lane = threadIdx.x & 31, n = p.qbs * p.nhead_q, chunks = (n + 255) / 256;
  const long long todo = (long long)p.num_q_block * chunks;
  for (long long u = blockIdx.x * 8 + (threadIdx.x >> 5); u < todo; u += gridDim.x * 8) {
    const int qb = (int)(u / chunks), first = (int)(u % chunks) * 256 + lane;
    const RowGeom g = row_geometry(p, P.ws.cnq, P.ws.cnk, P.ws.qb2b, qb);
    const float* src = lse + (long long)g.q_begin * p.nhead_q;
    const int there = (g.q_end - g.q_begin) * p.nhead_q;
    float x[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = first + 32 * e < there ? src[first + 32 * e] : -INFINITY;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const int i = first + 32 * e, tok = i / p.nhead_q, h = i - tok * p.nhead_q;
      if (i < n) P.sp.neg_lse[(((long long)(h >> P.gp_shift) * p.num_q_block + qb) * p.qbs + tok) * P.gp + (h & (P.gp - 1))] = x[e] == -INFINITY ? -INFINITY : -x[e] * kLog2e;
    }
  }
}

struct KeyWeightsStrides { long long q0, q1, q2, k0, k1, k2; };

template <typename T, int DP>
__global__ void __launch_bounds__(kThreads) key_weights_generic_kernel(const __grid_constant__ KeyWeightsParams P, const T* __restrict__ q, const T* __restrict__ k,
                                                                       KeyWeightsStrides st) {
  constexpr int KS = DP + 4;
  const Problem& p = P.p;
  if (P.ws.status[0] != HBSA_STATUS_OK) return;
  extern __shared__ __align__(16) float sm[];
  float* const sK = sm;                          // [kKeys][KS]
  float* const sQ = sK + kKeys * KS;             // [kRows][DP]
  __shared__ float s_nl[kRows], s_sum[kThreads];
  const int subs = (p.kbs + kKeys - 1) / kKeys, kb = blockIdx.x / subs, sub = blockIdx.x % subs, hk = blockIdx.y;
  const int b = sample_of_block(P.ws.cnk, p.batch, kb);
  const int k_begin = p.cu_k[b], k_len = p.cu_k[b + 1] - k_begin, q_begin = p.cu_q[b], q_len = p.cu_q[b + 1] - q_begin, off = k_len - q_len;
  const int blk0 = (kb - P.ws.cnk[b]) * p.kbs, k0 = blk0 + sub * kKeys, n_keys = min(kKeys, min(blk0 + p.kbs, k_len) - k0);
  if (n_keys <= 0) return;
  const int tid = threadIdx.x, key = tid & 63, part = tid >> 6;
  for (int i = tid; i < kKeys * DP; i += kThreads) {
    const int r = i / DP, d = i % DP;
    sK[r * KS + d] = r < n_keys && d < p.headdim ? to_f(k[(long long)(k_begin + k0 + r) * st.k0 + hk * st.k1 + d * st.k2]) : 0.f;
  }
  const int qb0 = P.ws.cnq[b], n_qb = P.ws.cnq[b + 1] - qb0;
  float sum = 0.f;
  for (int i = 0; i < n_qb; ++i) {
    bool on;
    if (p.csr_ptr != nullptr) {
      const long long row = (long long)hk * p.num_q_block + qb0 + i;
      const int e1 = p.csr_ptr[row + 1], e = lower_bound_i32(p.csr_idx, p.csr_ptr[row], e1, kb);
      on = e < e1 && p.csr_idx[e] == kb;
    } else {
      on = p.mask[hk * p.mask_s0 + (long long)(qb0 + i) * p.mask_s1 + (long long)kb * p.mask_s2] != 0;
    }
    const int row_end = min((i + 1) * p.qbs, q_len);
    if (!on || (p.causal && row_end - 1 + off < k0)) continue;       // uniform over the CTA
    const int n_rows = (row_end - i * p.qbs) * p.group;              // (token, head) pairs, heads innermost
    for (int r0 = 0; r0 < n_rows; r0 += kRows) {
      __syncthreads();
      for (int j = tid; j < kRows * DP; j += kThreads) {
        const int r = r0 + j / DP, d = j % DP;
        const long long tok = q_begin + i * p.qbs + r / p.group;
        sQ[j] = r < n_rows && d < p.headdim ? to_f(q[tok * st.q0 + (hk * p.group + r % p.group) * st.q1 + d * st.q2]) : 0.f;
      }
      if (tid < kRows) {
        const int r = r0 + tid;
        const int h = hk * p.group + r % p.group;
        s_nl[tid] = r < n_rows ? P.sp.neg_lse[(((long long)(h >> P.gp_shift) * p.num_q_block + qb0 + i) * p.qbs + r / p.group) * P.gp + (h & (P.gp - 1))] : -INFINITY;
      }
      __syncthreads();
      float tile_sum = 0.f;
      for (int rr = part * 16; rr < part * 16 + 16; rr += 4) {
        float s[4] = {0.f, 0.f, 0.f, 0.f};
        const float4* kr = reinterpret_cast<const float4*>(sK + key * KS);
#pragma unroll 4
        for (int d = 0; d < DP / 4; ++d) {
          const float4 x = kr[d];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float4 y = *reinterpret_cast<const float4*>(sQ + (rr + e) * DP + 4 * d);
            s[e] = fmaf(x.x, y.x, fmaf(x.y, y.y, fmaf(x.z, y.z, fmaf(x.w, y.w, s[e]))));
          }
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float nl = s_nl[rr + e];
          const int row = i * p.qbs + (r0 + rr + e) / p.group;
          const bool seen = nl != -INFINITY && (!p.causal || row + off >= k0 + key);
          if (seen) tile_sum += exp2f(fmaf(s[e], P.scale_log2, nl));
        }
      }
      sum += tile_sum;
    }
  }
  s_sum[tid] = sum;
  __syncthreads();
  if (tid < n_keys) P.out[(long long)(k_begin + k0 + tid) * p.nhead_k + hk] = s_sum[tid] + s_sum[tid + 64] + s_sum[tid + 128] + s_sum[tid + 192];
}

template <typename T, int DP>
cudaError_t launch_generic(const KeyWeightsParams& P, const hbsa_forward_args& a, cudaStream_t stream) {
  constexpr size_t smem = sizeof(float) * (size_t)(kKeys * (DP + 4) + kRows * DP);
  static SmemOptIn opt_in;
  cudaError_t e = opt_in.once(reinterpret_cast<const void*>(key_weights_generic_kernel<T, DP>), (int)smem);
  if (e != cudaSuccess) return e;
  const KeyWeightsStrides st = {a.q_stride[0], a.q_stride[1], a.q_stride[2], a.k_stride[0], a.k_stride[1], a.k_stride[2]};
  const dim3 grid((unsigned)(P.p.num_k_block * ((P.p.kbs + kKeys - 1) / kKeys)), (unsigned)P.p.nhead_k);
  key_weights_generic_kernel<T, DP><<<grid, kThreads, smem, stream>>>(P, static_cast<const T*>(a.q), static_cast<const T*>(a.k), st);
  return cudaGetLastError();
}
template <typename T>
cudaError_t launch_generic_of(const KeyWeightsParams& P, const hbsa_forward_args& a, cudaStream_t stream) {
  return a.headdim <= 64 ? launch_generic<T, 64>(P, a, stream) : a.headdim <= 128 ? launch_generic<T, 128>(P, a, stream) : launch_generic<T, 256>(P, a, stream);
}

size_t carve_key_weights(const hbsa_forward_args& a, char* base, KeyWeightsSpace* s) {
  char* p = base;
  auto take = [&](size_t bytes) { char* r = p; p += (bytes + 255) / 256 * 256; return r; };
  s->cursor = reinterpret_cast<unsigned long long*>(take(256));
  s->neg_lse = reinterpret_cast<float*>(take((size_t)a.num_q_block * a.q_block_size * a.nhead_q * 4));
  return (size_t)(p - base);
}

}  // namespace

}  // namespace hbsa

extern "C" {

size_t hbsa_key_weights_workspace_bytes(const hbsa_key_weights_args* args) {
  if (!args || args->struct_bytes != sizeof(*args) || args->fwd.num_q_block <= 0 || args->fwd.q_block_size <= 0 || args->fwd.nhead_q <= 0) return 0;
  hbsa::KeyWeightsSpace s;
  return hbsa::carve_key_weights(args->fwd, nullptr, &s);
}

int hbsa_key_weights(const hbsa_key_weights_args* args, void* stream_) {
  using namespace hbsa;
  if (!args) return set_last_error("args is NULL"), HBSA_ERR_NULL;
  if (args->struct_bytes != sizeof(*args)) return set_last_error("hbsa_key_weights_args.struct_bytes does not match this library"), HBSA_ERR_STRUCT;
  KeyWeightsParams P;
  memset(&P, 0, sizeof(P));
  hbsa_forward_args a = args->fwd;
  a.v = a.k;                                   // not used: the checks of a forward apply to what is there
  a.o = const_cast<void*>(a.q);
  for (int i = 0; i < 3; ++i) {
    a.v_stride[i] = a.k_stride[i];
    a.o_stride[i] = a.q_stride[i];
  }
  int rc = make_problem(&a, true, &P.p);
  if (rc != 0) return rc;
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
  cfg.gridDim = dim3((unsigned)(warps < most ? warps : most));
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
  if (a.dtype == HBSA_DTYPE_BF16) e = launch_generic_of<__nv_bfloat16>(P, a, stream);
  else if (a.dtype == HBSA_DTYPE_F16) e = launch_generic_of<__half>(P, a, stream);
  else e = launch_generic_of<float>(P, a, stream);
  return e == cudaSuccess ? 0 : failed(e);
}

}  // extern "C"
