// fp32-accurate products on the bf16 matrix instructions (gfx950, wave64).
//
// An fp32 number is the sum of three bf16 numbers up to 2^-27 of itself (8 + 8 + 8 significand bits and the signs of the
// remainders; terms below 2^-126, the least normal number, are lost, so numbers below 2^-109 are kept to 2^-126), so a
// product of two such operands is the sum of the six partial products whose weights are above 2^-25, accumulated in fp32 by
// the matrix instruction; an operand that is bf16 to begin with needs three.  At 16384 FLOPs in 16 cycles
// (v_mfma_f32_16x16x32_bf16) against 2048 in 32 (v_mfma_f32_16x16x4_f32) six of them still cost 2.7 times less than the
// fp32 instruction, three 5.3 times less.
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

typedef float f32x2 __attribute__((ext_vector_type(2)));

// two numbers rounded to bf16 (to nearest even), the first in the low half
__device__ __forceinline__ unsigned pack2(float a, float b) {
  typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
  const f32x2 v = {a, b};
  return __builtin_bit_cast(unsigned, __builtin_convertvector(v, bf16x2));
}
// x = h + m + l up to 2^-27 |x|; each term rounded to nearest even, so the remainders are exact in fp32.  Two numbers at a
// time (one conversion instruction packs a pair): 11 instructions, 15 one by one.
template <int N>
__device__ __forceinline__ void split2(float a, float b, unsigned (&t)[N]) {
#pragma unroll
  for (int q = 0; q < N; ++q) {
    t[q] = pack2(a, b);
    if (q + 1 < N) {
      a -= __uint_as_float(t[q] << 16);
      b -= __uint_as_float(t[q] & 0xffff0000u);
    }
  }
}
__device__ __forceinline__ void split3(float x, __bf16& h, __bf16& m, __bf16& l) {
  h = (__bf16)x;
  const float r = x - (float)h;
  m = (__bf16)r;
  l = (__bf16)(r - (float)m);
}

// N terms of x at p[0], p[stride], ...
template <int N>
__device__ __forceinline__ void split_store4(__bf16* p, int stride, const f32x4& x) {
  unsigned a[N], b[N];
  split2<N>(x[0], x[1], a);
  split2<N>(x[2], x[3], b);
#pragma unroll
  for (int q = 0; q < N; ++q) *reinterpret_cast<uint2*>(p + q * stride) = make_uint2(a[q], b[q]);
}
template <int N>
__device__ __forceinline__ void split8(const float (&x)[8], bf16x8 (&t)[N]) {
  typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
  u32x4 r[N];
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    unsigned a[N];
    split2<N>(x[2 * e], x[2 * e + 1], a);
#pragma unroll
    for (int q = 0; q < N; ++q) r[q][e] = a[q];
  }
#pragma unroll
  for (int q = 0; q < N; ++q) t[q] = __builtin_bit_cast(bf16x8, r[q]);
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
