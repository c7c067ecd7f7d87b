// Lane helpers of the attention kernels: the transposing LDS read and reductions over the four 16-lane rows of a wave.
#pragma once
#include "common.h"

namespace pp {
#if defined(__HIP_DEVICE_COMPILE__)
typedef __fp16 fp16v4 __attribute__((__vector_size__(4 * sizeof(__fp16))));
typedef __attribute__((address_space(3))) fp16v4 lds_fp16v4;
// ds_read_b64_tr_b16: within each group of 16 lanes, lane i supplies the address of 4 consecutive fp16 (row i / 4, column
// chunk i % 4 of a [4][16] block) and receives column i of that block (4 values, one per row).
static __device__ __forceinline__ f16x4 lds_read_tr16(const _Float16* p) {
  return __builtin_bit_cast(f16x4, __builtin_amdgcn_ds_read_tr16_b64_v4f16((lds_fp16v4*)p));
}

// Reductions over the four 16-lane rows of a wave (lanes l, l ^ 16, l ^ 32, l ^ 48 hold values of the same query) on the VALU:
// v_permlane32_swap / v_permlane16_swap (gfx950) exchange half-waves / odd-even rows between two registers -- with both operands the
// same value, the two results are the value and its partner's.  __shfl_xor is a ds_bpermute: an LDS round trip (~100+ cycles of
// latency each, four in a row per tile of the online softmax).
typedef unsigned int attn_u32x2 __attribute__((ext_vector_type(2)));
// (elements through .x / .y and __uint_as_float: with __builtin_bit_cast(float, r[i]) hipcc 7.2 reads element 0 twice -- max(r0, r1)
//  compiled to r0 and the reduction silently covered one row pair only; tools: grep the ISA for the v_max after the swap)
static __device__ __forceinline__ float rows_max(float v) {
  attn_u32x2 r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  const unsigned a0 = r.x, a1 = r.y;
  v = fmaxf(__uint_as_float(a0), __uint_as_float(a1));
  r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  const unsigned b0 = r.x, b1 = r.y;
  return fmaxf(__uint_as_float(b0), __uint_as_float(b1));
}
static __device__ __forceinline__ float rows_sum(float v) {
  attn_u32x2 r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  const unsigned a0 = r.x, a1 = r.y;
  v = __uint_as_float(a0) + __uint_as_float(a1);
  r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  const unsigned b0 = r.x, b1 = r.y;
  return __uint_as_float(b0) + __uint_as_float(b1);
}
#endif
}  // namespace pp
