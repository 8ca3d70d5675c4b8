// fp32-accurate products on the bf16 matrix instructions (gfx950, wave64).
//
// An fp32 number is the sum of three bf16 numbers up to 2^-27 of itself (8 + 8 + 8 significand bits and the signs of the
// remainders), so a product of two such operands is the sum of the six partial products whose weights are above 2^-25,
// accumulated in fp32 by the matrix instruction; an operand that is bf16 to begin with needs three.  At 16384 FLOPs in 16
// cycles (v_mfma_f32_16x16x32_bf16) against 2048 in 32 (v_mfma_f32_16x16x4_f32) six of them still cost 2.7 times less
// than the fp32 instruction, three 5.3 times less.
//
// v_mfma_f32_16x16x32_bf16: lane l supplies A[i = l&15][k] and B[k][j = l&15] for the eight k at 8*(l>>4); both operands
// use the same k, so an operand fragment is 16 contiguous bytes of a row whose memory runs along the reduction.  The four
// result registers hold column l&15, rows 4*(l>>4) + reg.
#pragma once
#include "common.h"

namespace hhrl {
namespace sb {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));
typedef float f32x4 __attribute__((ext_vector_type(4)));

// x = h + m + l up to 2^-27 |x|; each term rounded to nearest even, so the remainders are exact in fp32
__device__ __forceinline__ void split3(float x, __bf16& h, __bf16& m, __bf16& l) {
  h = (__bf16)x;
  const float r = x - (float)h;
  m = (__bf16)r;
  l = (__bf16)(r - (float)m);
}

// N terms of x at p[0], p[stride], ...
template <int N>
__device__ __forceinline__ void split_store4(__bf16* p, int stride, const f32x4& x) {
  bf16x4 t[3];
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    __bf16 h, m, l;
    split3(x[e], h, m, l);
    t[0][e] = h; t[1][e] = m; t[2][e] = l;
  }
#pragma unroll
  for (int q = 0; q < N; ++q) *reinterpret_cast<bf16x4*>(p + q * stride) = t[q];
}
template <int N>
__device__ __forceinline__ void split8(const float (&x)[8], bf16x8 (&t)[N]) {
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    __bf16 h, m, l;
    split3(x[e], h, m, l);
    t[0][e] = h;
    if constexpr (N > 1) t[1][e] = m;
    if constexpr (N > 2) t[2][e] = l;
  }
}

// acc += A B from NA and NB terms: the partial products whose weights add up to less than the longer operand's length
// (2^-8 apart), small ones first
template <int NA, int NB>
__device__ __forceinline__ void mma(f32x4& acc, const bf16x8 (&a)[NA], const bf16x8 (&b)[NB]) {
  constexpr int LIM = NA > NB ? NA : NB;
#pragma unroll
  for (int s = LIM - 1; s >= 0; --s)
#pragma unroll
    for (int p = 0; p < NA; ++p)
      if (s - p >= 0 && s - p < NB) acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a[p], b[s - p], acc, 0, 0, 0);
}

// the N terms of a fragment, `stride` elements apart
template <int N>
__device__ __forceinline__ void load_frag(bf16x8 (&f)[N], const __bf16* p, long stride) {
#pragma unroll
  for (int q = 0; q < N; ++q) f[q] = *reinterpret_cast<const bf16x8*>(p + q * stride);
}

}  // namespace sb
}  // namespace hhrl
