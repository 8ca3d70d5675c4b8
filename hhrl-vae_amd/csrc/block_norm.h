// Kernels of the norms around a block (block_norm.hip has the operator), a translation unit per element type.
#pragma once
#include "common.h"

namespace hhrl {

struct NormArgs {
  long R;                       // rows = M * H
  int H, D;
  int post, pre, gate_act;
  long gate_rows;               // > 1: row m of x reads gate row m / gate_rows (fp32, H == 1)
  float alpha, scale, eps, inv_d;
  const void *x, *y, *gate;
  long ldx, ldy, ldg;
  const float *w_post, *b_post, *w_pre, *b_pre;
  void *out, *h;
  long ldo, ldh;
  const void *d_out, *d_h;
  long lddo, lddh;
  void *dx, *dy, *dgate;
  long lddx, lddy, lddg;
  long step_m;                  // the advance of a row slot, as tokens and heads
  int step_j;
  // backward: rows are dealt in segments that end with a gate group; a workgroup takes segs_per_block of them
  long group_rows, seg_rows, n_groups;
  int parts;
  long segs_per_block, n_segs;
  float* par_ws;                // [workgroups][n_par][D] partial parameter gradients, order dw_post db_post dw_pre db_pre
  float* gate_ws;               // [n_segs][D] partial gate gradients (parts > 1)
  int par_slot[4], n_par;       // row of each parameter gradient in par_ws, -1: not wanted
  int gate_bcast;
  int bias;                     // a bias or the gradient of one: they cost registers that a norm without them does not pay for
};

// Launches the kernel of a thread layout: tpr threads per row, 16-byte vectors or single elements.
void norm_launch_f32(const NormArgs& a, bool vec, int tpr, int blocks, bool bwd, hipStream_t st);
void norm_launch_bf16(const NormArgs& a, bool vec, int tpr, int blocks, bool bwd, hipStream_t st);

constexpr int kNormE = 8;       // elements of a row per thread

// Waves per SIMD of the kernels, which the launches fill the chip by: workgroups beyond what is resident at once cost a
// second round (bf16 rows of 4096, forward: 56 us with 768 workgroups of 512 threads, 71 us with 1024).  A backward pass
// in bf16 vectors without biases is held to 128 registers for four waves (168 us with one workgroup of 512 threads per CU).
// Rows of 4097 to 8192 elements take 1024 threads, which have 128 registers at most: their backward kernels spill, most of
// all those with biases (both norms of 8192 columns trained: bf16 rms 4.3 TB/s, layer 3.3, fp32 4.7 and 3.0; of 5120, where
// three eighths of the threads idle, 2.9, 2.3, 4.3 and 2.4; of 4096 4.1, 2.9, 4.6 and 4.5).
constexpr int norm_bwd_waves(int el, int vec, bool bias) { return el == 2 && vec > 1 && !bias ? 4 : 2; }
constexpr int norm_fwd_waves(int el, int vec) { return el == 2 && vec > 1 ? 6 : 4; }

// Eight elements of a row as they come from memory: element (c * TPR + lane) * VEC + e of the row for c < 8 / VEC.  The
// request has no condition (a conditional one is waited for where its branch joins): behind the row's end it reads the
// row's last elements, and get() gives 0 there.
template <typename T, int VEC, int TPR>
struct RowRaw;
template <int VEC, int TPR>
struct RowRaw<float, VEC, TPR> {
  float v[kNormE];
  __device__ __forceinline__ void load(const float* p, int lane, int D) {
#pragma unroll
    for (int c = 0; c < kNormE / VEC; ++c) {
      const int at = min((c * TPR + lane) * VEC, D - VEC);
      if constexpr (VEC == 4) {
        const float4 t = *reinterpret_cast<const float4*>(p + at);
        v[4 * c] = t.x; v[4 * c + 1] = t.y; v[4 * c + 2] = t.z; v[4 * c + 3] = t.w;
      } else {
        v[c] = p[at];
      }
    }
  }
  __device__ __forceinline__ void get(float (&x)[kNormE], int lane, int D) const {
#pragma unroll
    for (int e = 0; e < kNormE; ++e) x[e] = ((e / VEC) * TPR + lane) * VEC < D ? v[e] : 0.f;
  }
};
template <int TPR>
struct RowRaw<__bf16, 8, TPR> {
  uint4 v;
  __device__ __forceinline__ void load(const __bf16* p, int lane, int D) { v = *reinterpret_cast<const uint4*>(p + min(lane * 8, D - 8)); }
  __device__ __forceinline__ void get(float (&x)[kNormE], int lane, int D) const {
    const unsigned u[4] = {v.x, v.y, v.z, v.w};
    const bool in = lane * 8 < D;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const unsigned t = in ? u[e] : 0u;
      x[2 * e] = __uint_as_float(t << 16);
      x[2 * e + 1] = __uint_as_float(t & 0xffff0000u);
    }
  }
};
template <int TPR>
struct RowRaw<__bf16, 1, TPR> {
  unsigned v[kNormE];
  __device__ __forceinline__ void load(const __bf16* p, int lane, int D) {
#pragma unroll
    for (int c = 0; c < kNormE; ++c) v[c] = reinterpret_cast<const unsigned short*>(p)[min(c * TPR + lane, D - 1)];
  }
  __device__ __forceinline__ void get(float (&x)[kNormE], int lane, int D) const {
#pragma unroll
    for (int e = 0; e < kNormE; ++e) x[e] = e * TPR + lane < D ? __uint_as_float(v[e] << 16) : 0.f;
  }
};
typedef __bf16 norm_bf16x8 __attribute__((ext_vector_type(8)));
template <typename T, int VEC, int TPR>
__device__ __forceinline__ void row_store(T* p, const float (&x)[kNormE], int lane, int D) {
#pragma unroll
  for (int c = 0; c < kNormE / VEC; ++c) {
    const int at = (c * TPR + lane) * VEC;
    if (at >= D) continue;
    if constexpr (VEC == 8 && sizeof(T) == 2) {          // rounded once, to nearest even
      norm_bf16x8 t;
#pragma unroll
      for (int e = 0; e < 8; ++e) t[e] = (__bf16)x[e];
      *reinterpret_cast<norm_bf16x8*>(p + at) = t;
    } else if constexpr (VEC > 1) {
#pragma unroll
      for (int h = 0; h < VEC / 4; ++h)
        *reinterpret_cast<float4*>(p + at + 4 * h) = make_float4(x[c * VEC + 4 * h], x[c * VEC + 4 * h + 1], x[c * VEC + 4 * h + 2], x[c * VEC + 4 * h + 3]);
    } else {
      p[at] = (T)x[c];
    }
  }
}
// a row of fp32 numbers (parameters, shared gates) in the layout of the activations' vectors
template <int VEC, int TPR>
__device__ __forceinline__ void row_load_f32(const float* p, float (&x)[kNormE], int lane, int D) {
#pragma unroll
  for (int c = 0; c < kNormE / VEC; ++c) {
    const int at = (c * TPR + lane) * VEC;
    const bool in = at < D;
    if constexpr (VEC >= 4) {
#pragma unroll
      for (int h = 0; h < VEC / 4; ++h) {
        const float4 t = *reinterpret_cast<const float4*>(p + min(at, D - VEC) + 4 * h);
        x[c * VEC + 4 * h] = in ? t.x : 0.f; x[c * VEC + 4 * h + 1] = in ? t.y : 0.f;
        x[c * VEC + 4 * h + 2] = in ? t.z : 0.f; x[c * VEC + 4 * h + 3] = in ? t.w : 0.f;
      }
    } else {
      const float t = p[min(at, D - 1)];
      x[c] = in ? t : 0.f;
    }
  }
}

template <int CTRL>
__device__ __forceinline__ float dpp_add(float v) {
  return v + __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), CTRL, 0xf, 0xf, true));
}
// Sums of N values over the TPR threads of a row, the same in all of them.  16 lanes: swaps inside quads, then mirrored
// halves, on the vector unit; the rest of a wave: lane exchanges.  Beyond: the row is a whole workgroup; waves meet
// through one of two LDS buffers in turn (one barrier per sum: the buffer written next was read before the barrier in
// between).
template <int TPR>
struct RowSum {
  float (*red)[16][4];
  int turn;
  template <int N>
  __device__ __forceinline__ void operator()(float (&v)[N]) {
#pragma unroll
    for (int n = 0; n < N; ++n) {
      v[n] = dpp_add<0xB1>(v[n]);        // lane ^ 1
      v[n] = dpp_add<0x4E>(v[n]);        // lane ^ 2
      v[n] = dpp_add<0x141>(v[n]);       // the other quad of eight lanes
      v[n] = dpp_add<0x140>(v[n]);       // the other eight of a row of sixteen
    }
    if constexpr (TPR >= 32) {
#pragma unroll
      for (int n = 0; n < N; ++n) v[n] += __shfl_xor(v[n], 16, 64);
    }
    if constexpr (TPR >= 64) {
#pragma unroll
      for (int n = 0; n < N; ++n) v[n] += __shfl_xor(v[n], 32, 64);
    }
    if constexpr (TPR > 64) {
      const int wave = threadIdx.x / 64 % (TPR / 64), row = threadIdx.x / TPR * (TPR / 64);
      if ((threadIdx.x & 63) == 0) {
#pragma unroll
        for (int n = 0; n < N; ++n) red[turn][row + wave][n] = v[n];
      }
      __syncthreads();
#pragma unroll
      for (int n = 0; n < N; ++n) v[n] = 0.f;
#pragma unroll
      for (int w = 0; w < TPR / 64; ++w)
#pragma unroll
        for (int n = 0; n < N; ++n) v[n] += red[turn][row + w][n];
      turn ^= 1;
    }
  }
};

template <typename T, int VEC, int TPR>
struct RowKernel {
  static constexpr int BT = TPR <= 256 ? 256 : TPR, SLOTS = BT / TPR;
  // rows of more than a wave share barriers, so all row slots of a workgroup take part in every round
  static constexpr bool UNIFORM = TPR > 64;
};
template <int VEC, int TPR>
__device__ __forceinline__ void row_mask(float (&x)[kNormE], int lane, int D) {
  if (D == TPR * kNormE) return;
#pragma unroll
  for (int e = 0; e < kNormE; ++e) x[e] = ((e / VEC) * TPR + lane) * VEC < D ? x[e] : 0.f;
}

// a row's place in the workgroup; the same for a whole wave where a row has one or more (its addresses are scalars then)
template <int TPR>
__device__ __forceinline__ int row_slot() {
  const int s = threadIdx.x / TPR;
  return TPR >= 64 ? __builtin_amdgcn_readfirstlane(s) : s;
}

template <typename T>
struct Gate {
  // s = sigmoid(z) and c = 1 - s, relative 2^-22 each for either type: parameter gradients and shared gates are fp32 results.
  // exp(-z) as the power of two of the rounded product with log2 e, times 1 + what the product and the constant leave out
  // (without it 2^-24 |z|); behind +-88 s and c are at fp32's ends.  Norms of 16384 x 16 heads of 128 with a SiLU gate take 112 us
  // forward and backward, 131 with expf() and a division.
  static __device__ __forceinline__ void sigmoid(float z, float& s, float& c) {
    const float x = __builtin_elementwise_maximum(__builtin_elementwise_minimum(z, 88.f), -88.f);   // (NaN stays)
    const float t = x * -1.44269502f;
    const float r = fmaf(x, -1.92596299e-8f, fmaf(x, -1.44269502f, -t));
    float e = __builtin_amdgcn_exp2f(t);
    e = fmaf(e, r * 0.693147181f, e);
    s = __builtin_amdgcn_rcpf(1.f + e);
    c = e * s;
  }
  // n <- n * value(z)
  static __device__ __forceinline__ void apply(float (&n)[kNormE], const float (&z)[kNormE], int act) {
    if (act == HHRL_ACT_NONE) {
#pragma unroll
      for (int e = 0; e < kNormE; ++e) n[e] *= z[e];
    } else if (act == HHRL_ACT_SILU) {
#pragma unroll
      for (int e = 0; e < kNormE; ++e) {
        float s, c;
        sigmoid(z[e], s, c);
        n[e] *= z[e] * s;
      }
    } else {
#pragma unroll
      for (int e = 0; e < kNormE; ++e) {
        float s, c;
        sigmoid(z[e], s, c);
        n[e] *= s;
      }
    }
  }
  // z <- scale * value(z), slope <- scale * slope of the gate
  static __device__ __forceinline__ void both(float (&z)[kNormE], float (&slope)[kNormE], float scale, int act) {
    if (act == HHRL_ACT_NONE) {
#pragma unroll
      for (int e = 0; e < kNormE; ++e) { z[e] *= scale; slope[e] = scale; }
    } else if (act == HHRL_ACT_SILU) {
#pragma unroll
      for (int e = 0; e < kNormE; ++e) {
        float s, c;
        sigmoid(z[e], s, c);
        const float v = z[e] * s;
        z[e] = scale * v;
        slope[e] = scale * fmaf(v, c, s);
      }
    } else {
#pragma unroll
      for (int e = 0; e < kNormE; ++e) {
        float s, c;
        sigmoid(z[e], s, c);
        z[e] = scale * s;
        slope[e] = scale * (s * c);
      }
    }
  }
};

// v <- v - mean of the row (layer norm; what lies behind the row's end stays 0)
template <int VEC, int TPR>
__device__ __forceinline__ void row_centre(float (&v)[kNormE], int lane, int D, float inv_d, RowSum<TPR>& sum) {
  float s[1] = {0.f};
#pragma unroll
  for (int e = 0; e < kNormE; ++e) s[0] += v[e];
  sum(s);
  const float mean = s[0] * inv_d;
#pragma unroll
  for (int e = 0; e < kNormE; ++e) v[e] -= mean;
  row_mask<VEC, TPR>(v, lane, D);
}
__device__ __forceinline__ float row_rstd(float sq, float inv_d, float eps) { return 1.f / sqrtf(fmaf(sq, inv_d, eps)); }

// The rows of a workgroup's slot, their operands requested a row ahead.
template <typename T, int VEC, int TPR, bool BIAS>
__global__ __launch_bounds__((RowKernel<T, VEC, TPR>::BT)) void block_norm_fwd_kernel(NormArgs a) {
  using RK = RowKernel<T, VEC, TPR>;
  __shared__ float red[2][16][4];
  const int lane = threadIdx.x % TPR, slot = row_slot<TPR>(), D = a.D;
  RowSum<TPR> sum{red, 0};
  const bool has_x = a.x != nullptr, has_y = a.y != nullptr, has_g = a.gate != nullptr, bcast = a.gate_bcast != 0;
  const long step = (long)gridDim.x * RK::SLOTS;
  long row = (long)blockIdx.x * RK::SLOTS + slot;
  long m = row / a.H;
  int j = (int)(row - m * a.H);
  RowRaw<T, VEC, TPR> rx, ry, rz;
  float zb[kNormE];
  auto request = [&](long mm, int jj) {
    const long col = (long)jj * D;
    if (has_x) rx.load(static_cast<const T*>(a.x) + mm * a.ldx + col, lane, D);
    if (has_y) ry.load(static_cast<const T*>(a.y) + mm * a.ldy + col, lane, D);
    if (has_g && !bcast) rz.load(static_cast<const T*>(a.gate) + mm * a.ldg + col, lane, D);
  };
  const long last = a.R - 1;
  const bool any = row <= last;
  if (any) request(m, j);
  float wq[kNormE], bq[kNormE], wp[kNormE], bp[kNormE];
#pragma unroll
  for (int e = 0; e < kNormE; ++e) { wq[e] = wp[e] = 1.f; bq[e] = bp[e] = 0.f; }
  if (a.w_post) row_load_f32<VEC, TPR>(a.w_post, wq, lane, D);
  if (a.w_pre) row_load_f32<VEC, TPR>(a.w_pre, wp, lane, D);
  if (BIAS && a.b_post) row_load_f32<VEC, TPR>(a.b_post, bq, lane, D);
  if (BIAS && a.b_pre) row_load_f32<VEC, TPR>(a.b_pre, bp, lane, D);
  // UNIFORM: every slot goes as many rounds as the first slot of the workgroup
  for (long first = (long)blockIdx.x * RK::SLOTS; RK::UNIFORM ? first <= last : row <= last; first += step) {
    const bool mine = row <= last;
    float r[kNormE], n[kNormE], z[kNormE];
#pragma unroll
    for (int e = 0; e < kNormE; ++e) r[e] = n[e] = z[e] = 0.f;
    if (has_x) rx.get(r, lane, D);
    if (has_y) ry.get(n, lane, D);
    if (has_g) {
      if (bcast) {
        row_load_f32<VEC, TPR>(static_cast<const float*>(a.gate) + (min(m, (a.R - 1) / a.H) / a.gate_rows) * a.ldg, zb, lane, D);
#pragma unroll
        for (int e = 0; e < kNormE; ++e) z[e] = zb[e];
      } else {
        rz.get(z, lane, D);
      }
    }
    long m2 = m + a.step_m;
    int j2 = j + a.step_j;
    if (j2 >= a.H) { j2 -= a.H; ++m2; }
    if (row + step <= last) request(m2, j2);
#pragma unroll
    for (int e = 0; e < kNormE; ++e) r[e] *= a.alpha;
    if (has_y) {
      if (a.post != HHRL_NORM_NONE) {
        if (a.post == HHRL_NORM_LAYER) row_centre<VEC, TPR>(n, lane, D, a.inv_d, sum);
        float q[1] = {0.f};
#pragma unroll
        for (int e = 0; e < kNormE; ++e) q[0] = fmaf(n[e], n[e], q[0]);
        sum(q);
        const float rstd = row_rstd(q[0], a.inv_d, a.eps);
#pragma unroll
        for (int e = 0; e < kNormE; ++e) n[e] = BIAS ? fmaf(n[e] * rstd, wq[e], bq[e]) : n[e] * rstd * wq[e];
      }
      if (has_g) Gate<T>::apply(n, z, a.gate_act);
#pragma unroll
      for (int e = 0; e < kNormE; ++e) r[e] = fmaf(a.scale, n[e], r[e]);
    }
    const long col = (long)j * D;
    if (a.out && mine) row_store<T, VEC, TPR>(static_cast<T*>(a.out) + m * a.ldo + col, r, lane, D);
    if (a.h) {
      if (a.pre != HHRL_NORM_NONE) {
        row_mask<VEC, TPR>(r, lane, D);
        if (a.pre == HHRL_NORM_LAYER) row_centre<VEC, TPR>(r, lane, D, a.inv_d, sum);
        float q[1] = {0.f};
#pragma unroll
        for (int e = 0; e < kNormE; ++e) q[0] = fmaf(r[e], r[e], q[0]);
        sum(q);
        const float rstd = row_rstd(q[0], a.inv_d, a.eps);
#pragma unroll
        for (int e = 0; e < kNormE; ++e) r[e] = BIAS ? fmaf(r[e] * rstd, wp[e], bp[e]) : r[e] * rstd * wp[e];
      }
      if (mine) row_store<T, VEC, TPR>(static_cast<T*>(a.h) + m * a.ldh + col, r, lane, D);
    }
    m = m2;
    j = j2;
    row += step;
  }
}

// GATE: 0 none, 1 an element each, 2 a row for many rows: its values and slopes are formed once.
template <typename T, int VEC, int TPR, bool BIAS, int GATE>
__global__ __launch_bounds__((RowKernel<T, VEC, TPR>::BT), norm_bwd_waves(sizeof(T), VEC, BIAS)) void block_norm_bwd_kernel(NormArgs a) {
  using RK = RowKernel<T, VEC, TPR>;
  __shared__ float red[2][16][4];
  __shared__ float fold[RK::SLOTS > 1 ? RK::BT * kNormE : 1];
  const int lane = threadIdx.x % TPR, slot = row_slot<TPR>(), D = a.D;
  RowSum<TPR> sum{red, 0};
  const bool has_x = a.x != nullptr, has_y = a.y != nullptr;
  const bool has_do = a.d_out != nullptr, has_dh = a.d_h != nullptr, pre = has_dh && a.pre != HHRL_NORM_NONE;
  float wq[kNormE], wp[kNormE], bq[kNormE], aq[kNormE], ap[kNormE], cq[kNormE], cp[kNormE], accg[kNormE];
#pragma unroll
  for (int e = 0; e < kNormE; ++e) { wq[e] = wp[e] = 1.f; bq[e] = aq[e] = ap[e] = cq[e] = cp[e] = 0.f; }
  if (a.w_post) row_load_f32<VEC, TPR>(a.w_post, wq, lane, D);
  if (a.w_pre) row_load_f32<VEC, TPR>(a.w_pre, wp, lane, D);
  if (BIAS && a.b_post) row_load_f32<VEC, TPR>(a.b_post, bq, lane, D);

  // sums a register array over the row slots of the workgroup and stores it as one row of D floats
  auto fold_store = [&](float (&v)[kNormE], float* dst) {
    if constexpr (RK::SLOTS > 1) {
      __syncthreads();
#pragma unroll
      for (int e = 0; e < kNormE; ++e) fold[e * RK::BT + threadIdx.x] = v[e];
      __syncthreads();
      if (slot == 0) {
        for (int s = 1; s < RK::SLOTS; ++s)
#pragma unroll
          for (int e = 0; e < kNormE; ++e) v[e] += fold[e * RK::BT + s * TPR + lane];
      }
    }
    if (slot == 0) row_store<float, VEC, TPR>(dst, v, lane, D);
  };

  const long seg0 = (long)blockIdx.x * a.segs_per_block;
  const long seg1 = min(a.n_segs, seg0 + a.segs_per_block);
  for (long seg = seg0; seg < seg1; ++seg) {
    const long grp = seg / a.parts;
    const long r0 = grp * a.group_rows + (seg - grp * a.parts) * a.seg_rows;
    const long r1 = min(min(a.R, (grp + 1) * a.group_rows), r0 + a.seg_rows);
    float z[kNormE], sl[kNormE];                         // scale * value and scale * slope of the gate
    if constexpr (GATE == 2) {
      row_load_f32<VEC, TPR>(static_cast<const float*>(a.gate) + grp * a.ldg, z, lane, D);
      Gate<T>::both(z, sl, a.scale, a.gate_act);
#pragma unroll
      for (int e = 0; e < kNormE; ++e) accg[e] = 0.f;
    }
    long row = r0 + slot;
    long m = row / a.H;
    int j = (int)(row - m * a.H);
    RowRaw<T, VEC, TPR> rx, ry, rz, ro, rh;
    auto request = [&](long mm, int jj) {
      const long col = (long)jj * D;
      if (has_y) ry.load(static_cast<const T*>(a.y) + mm * a.ldy + col, lane, D);
      if (has_x && pre) rx.load(static_cast<const T*>(a.x) + mm * a.ldx + col, lane, D);
      if (GATE == 1) rz.load(static_cast<const T*>(a.gate) + mm * a.ldg + col, lane, D);
      if (has_dh) rh.load(static_cast<const T*>(a.d_h) + mm * a.lddh + col, lane, D);
      if (has_do) ro.load(static_cast<const T*>(a.d_out) + mm * a.lddo + col, lane, D);
    };
    if (row < r1) request(m, j);
    for (long first = r0; RK::UNIFORM ? first < r1 : row < r1; first += RK::SLOTS) {
      const bool mine = row < r1;
      const bool adds = !RK::UNIFORM || mine;        // a slot without a row of its own adds nothing to the column sums
      float r[kNormE], n[kNormE], dn[kNormE], dr[kNormE];
#pragma unroll
      for (int e = 0; e < kNormE; ++e) r[e] = n[e] = dn[e] = dr[e] = 0.f;
      if (has_y) ry.get(n, lane, D);
      if (has_x && pre) rx.get(r, lane, D);
      if (GATE == 1) rz.get(z, lane, D);
      if (has_dh) rh.get(dn, lane, D);
      if (has_do) ro.get(dr, lane, D);
      long m2 = m + a.step_m;
      int j2 = j + a.step_j;
      if (j2 >= a.H) { j2 -= a.H; ++m2; }
      if (row + RK::SLOTS < r1) request(m2, j2);
      float rq = 1.f;
      if (has_y && a.post != HHRL_NORM_NONE) {
        if (a.post == HHRL_NORM_LAYER) row_centre<VEC, TPR>(n, lane, D, a.inv_d, sum);
        float q[1] = {0.f};
#pragma unroll
        for (int e = 0; e < kNormE; ++e) q[0] = fmaf(n[e], n[e], q[0]);
        sum(q);
        rq = row_rstd(q[0], a.inv_d, a.eps);
#pragma unroll
        for (int e = 0; e < kNormE; ++e) n[e] *= rq;
      }
      if (GATE == 1) Gate<T>::both(z, sl, a.scale, a.gate_act);
      if (pre) {
#pragma unroll
        for (int e = 0; e < kNormE; ++e) {
          r[e] *= a.alpha;
          if (has_y) r[e] = fmaf(GATE ? z[e] : a.scale, BIAS ? fmaf(n[e], wq[e], bq[e]) : n[e] * wq[e], r[e]);
        }
        row_mask<VEC, TPR>(r, lane, D);
        if (a.pre == HHRL_NORM_LAYER) row_centre<VEC, TPR>(r, lane, D, a.inv_d, sum);
        // the row's square sum and the two means of its gradient in one go: sum dn m = rstd * sum dn r
        float q[3] = {0.f, 0.f, 0.f};
#pragma unroll
        for (int e = 0; e < kNormE; ++e) {
          const float d = dn[e] * wp[e];
          q[0] = fmaf(r[e], r[e], q[0]);
          q[1] = fmaf(d, r[e], q[1]);
          q[2] += d;
        }
        sum(q);
        const float rp = row_rstd(q[0], a.inv_d, a.eps);
        const float c1 = rp * q[1] * a.inv_d, c2 = a.pre == HHRL_NORM_LAYER ? q[2] * a.inv_d : 0.f;
#pragma unroll
        for (int e = 0; e < kNormE; ++e) {
          const float mm = r[e] * rp;
          if (adds) {
            ap[e] = fmaf(dn[e], mm, ap[e]);
            if (BIAS) cp[e] += dn[e];
          }
          dr[e] = fmaf(rp, fmaf(-mm, c1, fmaf(dn[e], wp[e], -c2)), dr[e]);
        }
      } else {
#pragma unroll
        for (int e = 0; e < kNormE; ++e) dr[e] += dn[e];
      }
      const long col = (long)j * D;
      if (a.dx && mine) {
#pragma unroll
        for (int e = 0; e < kNormE; ++e) dn[e] = a.alpha * dr[e];
        row_store<T, VEC, TPR>(static_cast<T*>(a.dx) + m * a.lddx + col, dn, lane, D);
      }
      if (has_y) {
        if (GATE && a.dgate) {
#pragma unroll
          for (int e = 0; e < kNormE; ++e) dn[e] = dr[e] * sl[e] * (BIAS ? fmaf(n[e], wq[e], bq[e]) : n[e] * wq[e]);
          if (GATE == 2) {
#pragma unroll
            for (int e = 0; e < kNormE; ++e) accg[e] += adds ? dn[e] : 0.f;
          } else if (mine) {
            row_store<T, VEC, TPR>(static_cast<T*>(a.dgate) + m * a.lddg + col, dn, lane, D);
          }
        }
#pragma unroll
        for (int e = 0; e < kNormE; ++e) dr[e] *= GATE ? z[e] : a.scale;
        if (a.post != HHRL_NORM_NONE) {
          float q[2] = {0.f, 0.f};
          row_mask<VEC, TPR>(dr, lane, D);
#pragma unroll
          for (int e = 0; e < kNormE; ++e) {
            if (adds) {
              aq[e] = fmaf(dr[e], n[e], aq[e]);
              if (BIAS) cq[e] += dr[e];
            }
            dr[e] *= wq[e];
            q[0] = fmaf(dr[e], n[e], q[0]);
            q[1] += dr[e];
          }
          if (a.dy) {
            sum(q);
            const float c1 = q[0] * a.inv_d, c2 = a.post == HHRL_NORM_LAYER ? q[1] * a.inv_d : 0.f;
#pragma unroll
            for (int e = 0; e < kNormE; ++e) dr[e] = rq * fmaf(-n[e], c1, dr[e] - c2);
          }
        }
        if (a.dy && mine) row_store<T, VEC, TPR>(static_cast<T*>(a.dy) + m * a.lddy + col, dr, lane, D);
      }
      m = m2;
      j = j2;
      row += RK::SLOTS;
    }
    if (GATE == 2 && a.dgate) fold_store(accg, a.parts > 1 ? a.gate_ws + seg * D : static_cast<float*>(a.dgate) + grp * a.lddg);
  }
  float* const par = a.par_ws + (long)blockIdx.x * a.n_par * D;
  if (a.par_slot[0] >= 0) fold_store(aq, par + (long)a.par_slot[0] * D);
  if (BIAS && a.par_slot[1] >= 0) fold_store(cq, par + (long)a.par_slot[1] * D);
  if (a.par_slot[2] >= 0) fold_store(ap, par + (long)a.par_slot[2] * D);
  if (BIAS && a.par_slot[3] >= 0) fold_store(cp, par + (long)a.par_slot[3] * D);
}

template <typename T, int VEC, int TPR, bool BIAS>
void norm_launch(const NormArgs& a, int blocks, bool bwd, hipStream_t st) {
  constexpr int BT = RowKernel<T, VEC, TPR>::BT;
  if (bwd && !a.gate) hipLaunchKernelGGL((block_norm_bwd_kernel<T, VEC, TPR, BIAS, 0>), dim3(blocks), dim3(BT), 0, st, a);
  else if (bwd && !a.gate_bcast) hipLaunchKernelGGL((block_norm_bwd_kernel<T, VEC, TPR, BIAS, 1>), dim3(blocks), dim3(BT), 0, st, a);
  else if (bwd) hipLaunchKernelGGL((block_norm_bwd_kernel<T, VEC, TPR, BIAS, 2>), dim3(blocks), dim3(BT), 0, st, a);
  else hipLaunchKernelGGL((block_norm_fwd_kernel<T, VEC, TPR, BIAS>), dim3(blocks), dim3(BT), 0, st, a);
}
template <typename T, int VEC, bool BIAS>
void norm_launch(const NormArgs& a, int tpr, int blocks, bool bwd, hipStream_t st) {
  switch (tpr) {
    case 16: norm_launch<T, VEC, 16, BIAS>(a, blocks, bwd, st); break;
    case 32: norm_launch<T, VEC, 32, BIAS>(a, blocks, bwd, st); break;
    case 64: norm_launch<T, VEC, 64, BIAS>(a, blocks, bwd, st); break;
    case 128: norm_launch<T, VEC, 128, BIAS>(a, blocks, bwd, st); break;
    case 256: norm_launch<T, VEC, 256, BIAS>(a, blocks, bwd, st); break;
    case 512: norm_launch<T, VEC, 512, BIAS>(a, blocks, bwd, st); break;
    default: norm_launch<T, VEC, 1024, BIAS>(a, blocks, bwd, st); break;
  }
}
template <typename T, int VEC>
void norm_launch(const NormArgs& a, bool vec, int tpr, int blocks, bool bwd, hipStream_t st) {
  if (!vec) norm_launch<T, 1, true>(a, tpr, blocks, bwd, st);
  else if (a.bias) norm_launch<T, VEC, true>(a, tpr, blocks, bwd, st);
  else norm_launch<T, VEC, false>(a, tpr, blocks, bwd, st);
}

}  // namespace hhrl
