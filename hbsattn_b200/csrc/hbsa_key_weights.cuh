// What the two kernels of the key weights share (hbsa_key_weights.cu, hbsa_key_weights_sm100.cu).
#pragma once
#include "hbsa_common.cuh"

namespace hbsa {

struct KeyWeightsSpace {
  unsigned long long* cursor;  // [32] word 0: next item, word 1: CTAs that have left
  float* neg_lse;              // -lse log2 e; -inf: the row adds nothing.  [nhead_q / gp][num_q_block][q_block_size][gp], blocks filled up with
                               // -inf: rows in the order of the tiles, every q-block on a 64-byte boundary whatever the samples' lengths
  int32_t* classes;            // [256] what order is made with
  int32_t* order;              // [num_k_block] k-blocks by the rows that may see them, most first (tensor-core kernel, where P.sorted)
};
constexpr int kKwSorted = 8192;              // k-blocks that are put in order, at most

struct KeyWeightsParams {
  Problem p;
  Workspace ws;
  KeyWeightsSpace sp;
  float* out;                  // [total_k, nhead_k]
  int total_q, total_k;
  float scale_log2;
  // tensor-core kernel
  int gp, gp_shift, n_head_sub, piece, piece_shift;      // q-heads of a piece, pieces of heads per group, rows of a piece
  int one_box;                               // one copy brings all columns of a tile
  int m_rows, n_msub, n_cols;                // keys of an item, items per k-block, columns of S
  long long total_items;
  int sorted;                                // items: all heads of a k-block, k-blocks in the order of sp.order; else head by head
  long long wait_budget;
  int debug_stall;
};

// Keys that cu_k puts outside the tensors are neither read nor written.
__device__ __forceinline__ bool key_is_there(const KeyWeightsParams& P, int row) { return (unsigned)row < (unsigned)P.total_k; }

// Keys outside every sample get zeros, and with a block count mismatch all keys do.  All threads of the grid.
__device__ __forceinline__ void key_weights_outside(const KeyWeightsParams& P, bool all) {
  const int lo = all ? 0 : max(0, min(P.p.cu_k[0], P.total_k)), hi = all ? 0 : max(lo, min(P.p.cu_k[P.p.batch], P.total_k));
  const long long n_cta = (long long)gridDim.x * gridDim.y, cta = (long long)blockIdx.y * gridDim.x + blockIdx.x;
  const long long first = (long long)lo * P.p.nhead_k, last = (long long)hi * P.p.nhead_k, n = (long long)P.total_k * P.p.nhead_k;
  for (long long i = cta * blockDim.x + threadIdx.x; i < first + (n - last); i += n_cta * blockDim.x) P.out[i < first ? i : i - first + last] = 0.f;
}

int launch_key_weights_sm100(KeyWeightsParams& P, const hbsa_forward_args& a, cudaStream_t stream, const char** err_text);

}  // namespace hbsa
