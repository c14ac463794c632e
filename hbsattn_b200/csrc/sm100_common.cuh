// Pieces shared by the tensor-core kernels: 16-bit packing, bounded warp-wide barrier waits, and the
// host side of the TMA tensor maps.
#pragma once
#include <cuda.h>
#include <cudaTypedefs.h>

#include "hbsa_common.cuh"
#include "sm100_ptx.cuh"

namespace hbsa {

template <bool BF16> __device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  uint32_t r;
  if (BF16) asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  else asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}

template <bool BF16> __device__ __forceinline__ void unpack16(uint32_t w, float& a, float& b) {
  if (BF16) {
    a = __uint_as_float(w << 16);
    b = __uint_as_float(w & 0xffff0000u);
  } else {
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w));
    a = f.x;
    b = f.y;
  }
}
// x0, x1 = hi + lo, two 16-bit terms each
template <bool BF16> __device__ __forceinline__ void split2(float x0, float x1, uint32_t& hi, uint32_t& lo) {
  hi = pack2<BF16>(x0, x1);
  float h0, h1;
  unpack16<BF16>(hi, h0, h1);
  float l0, l1;
  ptx::unpack_f32x2(ptx::fma_f32x2(ptx::pack_f32x2(h0, h1), ptx::pack_f32x2(-1.f, -1.f), ptx::pack_f32x2(x0, x1)), l0, l1);
  lo = pack2<BF16>(l0, l1);
}

// One lane polls the mbarrier, the rest of the warp sleeps at the shuffle instead of spinning.
__device__ __forceinline__ bool warp_wait(uint32_t bar, uint32_t parity, volatile int* abort_flag, long long budget) {
  int ok = 1;
  if ((threadIdx.x & 31) == 0) ok = ptx::mbar_wait_bounded(bar, parity, abort_flag, budget) ? 1 : 0;
  return __shfl_sync(0xffffffffu, ok, 0) != 0;
}
// A wait of a whole warp that finds the phase complete, or nearly so: all lanes look before one of them waits.  Sixteen looks against one: decoding
// 129.1 and 130.9 us (16 x 16384..32768 keys, 8 heads of 64), 32.3 and 33.2 (6 x 301..3001 with weights); key weights the same within 0.6 us.
__device__ __forceinline__ bool quick_wait(uint32_t bar, uint32_t parity, volatile int* abort_flag, long long budget) {
#pragma unroll 1
  for (int i = 0; i < 16; ++i)
    if (__all_sync(0xffffffffu, ptx::mbar_test(bar, parity))) return true;
  const bool ok = warp_wait(bar, parity, abort_flag, budget);
  __syncwarp();
  return ok;
}
// Barrier entry and parity for the c-th use of a two-entry barrier array.
__device__ __forceinline__ uint32_t bar_of(uint32_t base, int c) { return base + 8u * (uint32_t)(c & 1); }
__device__ __forceinline__ uint32_t par_of(int c) { return (uint32_t)(c >> 1) & 1u; }

typedef CUresult (*EncodeTiledFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                                  const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                                  CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

// cuTensorMapEncodeTiled of the loaded driver, or NULL.
EncodeTiledFn sm100_encode_fn();
// 3-D map over a [tokens, heads, headdim] 16-bit tensor: dims (headdim, heads, tokens), box (64, box_heads, box_tokens).
bool sm100_encode_map(EncodeTiledFn fn, CUtensorMap* map, bool bf16, const void* base, int headdim, int heads, int tokens,
                      long long s_tok, long long s_head, int box_heads, int box_tokens);
int sm100_sm_count();
long long sm100_wait_budget();
int sm100_debug_stall();

}  // namespace hbsa
