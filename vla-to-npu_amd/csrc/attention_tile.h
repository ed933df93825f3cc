// Pieces that the attention kernels share: the LDS tile of 64 keys, its
// transpose read, and maxima over the lanes that hold one query.
#pragma once

#include "svla_common.h"

namespace {

constexpr int D = 64;
constexpr int BKEY = 64;   // keys per LDS stage

// LDS stage = K tile [64 keys][64 d] + V tile [64 keys][64 d], both row-major
// with the 16-byte chunk c of key row r stored in slot c ^ (r & 7), so that
// both the K fragment reads (16 keys x one chunk) and the V transpose reads
// (4 keys x 4 chunks per 16 lanes) spread over the banks.
__device__ __forceinline__ int kv_off(int key, int d) {  // element offset, d % 4 == 0
  return key * D + ((((d >> 3) ^ key) & 7) << 3) + (d & 7);
}

typedef short v4i16 __attribute__((ext_vector_type(4)));
typedef unsigned u32x2_t __attribute__((ext_vector_type(2)));

// Maximum of two scores as IEEE 754-2019 maximum (v_maximum3_f32 on gfx950):
// unlike fmaxf (maxNum), which the compiler must precede with a
// canonicalising v_max of each input, it propagates NaN and needs no quieting,
// so a 16-score row maximum is 8 instructions and a shuffle step 1, not 10
// and 3.  For the non-NaN scores here the two agree (masked scores are -inf).
__device__ __forceinline__ float smax(float a, float b) { return __builtin_elementwise_maximum(a, b); }

// Reductions over lanes l ^ 16 and l ^ 32 with the gfx950 row-swap VALU ops
// (v_permlane16_swap / v_permlane32_swap): called with both operands = x,
// every lane ends up holding {x[l], x[l ^ 16]} (resp. l ^ 32) in some order.
// No LDS round trip, unlike a ds_bpermute shuffle.
__device__ __forceinline__ float max_xor16(float x) {
  const u32x2_t r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return smax(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float max_xor32(float x) {
  const u32x2_t r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return smax(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
typedef __attribute__((address_space(3))) v4i16* lds_v4i16_ptr;

// V^T operand of O^T += V^T . P^T via the LDS transpose read: within each
// 16-lane group, lane j receives element (j & 3) of the 8-byte chunks of
// lanes (j >> 2) + 4t, t = 0..3.  Lane i = 4t + r of the group points at
// V[kbase + t][dbase + 4r], so lane j gets V[kbase + t][dbase + j], t = 0..3:
// 4 consecutive keys of head dim (dbase + j).
__device__ __forceinline__ v4i16 v_tr_read(const bf16* sv, int kbase, int dbase, int i) {
  const int t = i >> 2, r = i & 3;
  const bf16* p = sv + kv_off(kbase + t, dbase + 4 * r);
  return __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4i16_ptr)(p));
}

}  // namespace
