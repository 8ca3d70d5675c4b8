// Norms before and after a block, fused with the block's gate and residual scale:
//   r = alpha*x + scale * act(gate) * post(y)         h = pre(r)
// x: residual stream, y: a block's output, post / pre: none, RMS norm or layer norm over D elements.
// y absent: the norm in front of the first block; pre = none: the sum behind the last one; x absent: a gated norm
// (per head of a sequence layer: H rows of D elements per token).
//
// What bounds it: memory.  A forward pass reads x, y, gate once and writes r, h once (a row stays in registers between
// its two norms), a backward pass reads x, y, gate, dr, dh once and writes dx, dy, dgate once: r and both norms'
// statistics are formed again from the inputs in registers, which costs no byte and leaves the gradient that of the
// unrounded r.  The column sums of the parameter gradients stay in registers over all rows of a workgroup, leave as one
// partial row per workgroup, and a second launch adds the partial rows in a fixed order (same bits on every run).
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
  int parts, segs_per_block;
  long n_segs;
  float* par_ws;                // [workgroups][n_par][D] partial parameter gradients, order dw_post db_post dw_pre db_pre
  float* gate_ws;               // [n_segs][D] partial gate gradients (parts > 1)
  int par_slot[4], n_par;       // row of each parameter gradient in par_ws, -1: not wanted
  int gate_bcast;
};

template <typename T, int VEC>
struct Vec;
template <> struct Vec<float, 4> {
  static __device__ __forceinline__ void load(const float* p, float* v) {
    const float4 t = *reinterpret_cast<const float4*>(p);
    v[0] = t.x; v[1] = t.y; v[2] = t.z; v[3] = t.w;
  }
  static __device__ __forceinline__ void store(float* p, const float* v) { *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]); }
};
template <> struct Vec<float, 1> {
  static __device__ __forceinline__ void load(const float* p, float* v) { v[0] = *p; }
  static __device__ __forceinline__ void store(float* p, const float* v) { *p = v[0]; }
};
template <> struct Vec<float, 8> {
  static __device__ __forceinline__ void load(const float* p, float* v) { Vec<float, 4>::load(p, v); Vec<float, 4>::load(p + 4, v + 4); }
  static __device__ __forceinline__ void store(float* p, const float* v) { Vec<float, 4>::store(p, v); Vec<float, 4>::store(p + 4, v + 4); }
};
typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));
template <> struct Vec<__bf16, 8> {
  static __device__ __forceinline__ void load(const __bf16* p, float* v) {
    const bf16x8_t t = *reinterpret_cast<const bf16x8_t*>(p);
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = (float)t[e];
  }
  static __device__ __forceinline__ void store(__bf16* p, const float* v) {      // rounded once, to nearest even
    bf16x8_t t;
#pragma unroll
    for (int e = 0; e < 8; ++e) t[e] = (__bf16)v[e];
    *reinterpret_cast<bf16x8_t*>(p) = t;
  }
};
template <> struct Vec<__bf16, 1> {
  static __device__ __forceinline__ void load(const __bf16* p, float* v) { v[0] = (float)*p; }
  static __device__ __forceinline__ void store(__bf16* p, const float* v) { *p = (__bf16)v[0]; }
};

// Sums of two values over the TPR threads of a row.  Up to 64 threads: within the wave.  Beyond: the row is a whole
// workgroup; waves meet through one of two LDS buffers in turn (one barrier per sum: the buffer written next was read
// before the barrier in between).
template <int TPR>
struct RowSum {
  float (*red)[8][2];
  int turn;
  __device__ __forceinline__ void operator()(float& a, float& b) {
#pragma unroll
    for (int off = (TPR < 64 ? TPR : 64) / 2; off > 0; off >>= 1) {
      a += __shfl_xor(a, off, 64);
      b += __shfl_xor(b, off, 64);
    }
    if (TPR > 64) {
      const int wave = threadIdx.x >> 6;
      if ((threadIdx.x & 63) == 0) { red[turn][wave][0] = a; red[turn][wave][1] = b; }
      __syncthreads();
      a = b = 0.f;
#pragma unroll
      for (int w = 0; w < TPR / 64; ++w) { a += red[turn][w][0]; b += red[turn][w][1]; }
      turn ^= 1;
    }
  }
};

template <typename T, int VEC, int TPR, int E>
struct RowKernel {
  static constexpr int BT = TPR <= 256 ? 256 : TPR, SLOTS = BT / TPR, NCH = E / VEC;
  static_assert(E % VEC == 0, "elements per thread are whole vectors");
  int lane, D;
  __device__ __forceinline__ int at(int c) const { return (c * TPR + lane) * VEC; }
  template <typename U>
  __device__ __forceinline__ void load(const U* p, float (&v)[E]) const {
#pragma unroll
    for (int c = 0; c < NCH; ++c) {
      if (at(c) < D) Vec<U, VEC>::load(p + at(c), v + c * VEC);
      else
#pragma unroll
        for (int e = 0; e < VEC; ++e) v[c * VEC + e] = 0.f;
    }
  }
  template <typename U>
  __device__ __forceinline__ void store(U* p, const float (&v)[E]) const {
#pragma unroll
    for (int c = 0; c < NCH; ++c)
      if (at(c) < D) Vec<U, VEC>::store(p + at(c), v + c * VEC);
  }
  __device__ __forceinline__ void param(const float* p, float dflt, float (&v)[E]) const {
    if (p) load(p, v);
    else
#pragma unroll
      for (int e = 0; e < E; ++e) v[e] = dflt;
  }
  // v <- (v - mean) * rstd (layer) or v * rstd (rms); elements beyond D stay 0.  Two passes over the registers for the
  // layer norm's variance (no cancellation of squares).
  __device__ __forceinline__ float normalise(float (&v)[E], int kind, float inv_d, float eps, RowSum<TPR>& sum) const {
    if (kind == HHRL_NORM_LAYER) {
      float s = 0.f, z = 0.f;
#pragma unroll
      for (int e = 0; e < E; ++e) s += v[e];
      sum(s, z);
      const float mean = s * inv_d;
#pragma unroll
      for (int c = 0; c < NCH; ++c)
#pragma unroll
        for (int e = 0; e < VEC; ++e) v[c * VEC + e] = at(c) < D ? v[c * VEC + e] - mean : 0.f;
    }
    float q = 0.f, z = 0.f;
#pragma unroll
    for (int e = 0; e < E; ++e) q = fmaf(v[e], v[e], q);
    sum(q, z);
    const float rstd = 1.f / sqrtf(fmaf(q, inv_d, eps));
#pragma unroll
    for (int e = 0; e < E; ++e) v[e] *= rstd;
    return rstd;
  }
  // dn <- gradient of the normalised row's input, n the normalised row:
  //   rstd * (dn - n mean(dn n) [- mean(dn) for the layer norm])
  __device__ __forceinline__ void normalise_back(float (&dn)[E], const float (&n)[E], float rstd, int kind, float inv_d,
                                                 RowSum<TPR>& sum) const {
    float a = 0.f, b = 0.f;
#pragma unroll
    for (int e = 0; e < E; ++e) { a = fmaf(dn[e], n[e], a); b += dn[e]; }
    sum(a, b);
    a *= inv_d;
    b = kind == HHRL_NORM_LAYER ? b * inv_d : 0.f;
#pragma unroll
    for (int c = 0; c < NCH; ++c)
#pragma unroll
      for (int e = c * VEC; e < c * VEC + VEC; ++e) dn[e] = at(c) < D ? rstd * (dn[e] - n[e] * a - b) : 0.f;
  }
};

__device__ __forceinline__ float gate_value(float z, int act) {
  if (act == HHRL_ACT_NONE) return z;
  const float s = 1.f / (1.f + expf(-z));
  return act == HHRL_ACT_SILU ? z * s : s;
}
__device__ __forceinline__ float gate_slope(float z, int act) {
  if (act == HHRL_ACT_NONE) return 1.f;
  const float s = 1.f / (1.f + expf(-z));
  return act == HHRL_ACT_SILU ? s * (1.f + z * (1.f - s)) : s * (1.f - s);
}

template <typename T, int VEC, int TPR, int E>
__global__ __launch_bounds__((RowKernel<T, VEC, TPR, E>::BT)) void block_norm_fwd_kernel(NormArgs a) {
  using RK = RowKernel<T, VEC, TPR, E>;
  __shared__ float red[2][8][2];
  RK rk{(int)(threadIdx.x % TPR), a.D};
  RowSum<TPR> sum{red, 0};
  const int slot = threadIdx.x / TPR;
  float wq[E], bq[E], wp[E], bp[E];
  rk.param(a.w_post, 1.f, wq);
  rk.param(a.b_post, 0.f, bq);
  rk.param(a.w_pre, 1.f, wp);
  rk.param(a.b_pre, 0.f, bp);
  const long step = (long)gridDim.x * RK::SLOTS;
  long row = (long)blockIdx.x * RK::SLOTS + slot;
  long m = row / a.H;
  int j = (int)(row - m * a.H);
  for (; row < a.R; row += step) {
    const long col = (long)j * a.D;
    float r[E], n[E], z[E];
    if (a.x) rk.load(static_cast<const T*>(a.x) + m * a.ldx + col, r);
    if (a.y) rk.load(static_cast<const T*>(a.y) + m * a.ldy + col, n);
    if (a.gate) {
      if (a.gate_bcast) rk.load(static_cast<const float*>(a.gate) + (m / a.gate_rows) * a.ldg, z);
      else rk.load(static_cast<const T*>(a.gate) + m * a.ldg + col, z);
    }
#pragma unroll
    for (int e = 0; e < E; ++e) r[e] = a.x ? a.alpha * r[e] : 0.f;
    if (a.y) {
      if (a.post != HHRL_NORM_NONE) {
        rk.normalise(n, a.post, a.inv_d, a.eps, sum);
#pragma unroll
        for (int e = 0; e < E; ++e) n[e] = fmaf(n[e], wq[e], bq[e]);
      }
#pragma unroll
      for (int e = 0; e < E; ++e) r[e] = fmaf(a.gate ? a.scale * gate_value(z[e], a.gate_act) : a.scale, n[e], r[e]);
    }
    if (a.out) rk.store(static_cast<T*>(a.out) + m * a.ldo + col, r);
    if (a.h) {
      // elements beyond D: 0 in every array but the affine result of the post norm, which the mask keeps out
#pragma unroll
      for (int c = 0; c < RK::NCH; ++c)
#pragma unroll
        for (int e = 0; e < VEC; ++e) r[c * VEC + e] = rk.at(c) < a.D ? r[c * VEC + e] : 0.f;
      if (a.pre != HHRL_NORM_NONE) {
        rk.normalise(r, a.pre, a.inv_d, a.eps, sum);
#pragma unroll
        for (int e = 0; e < E; ++e) r[e] = fmaf(r[e], wp[e], bp[e]);
      }
      rk.store(static_cast<T*>(a.h) + m * a.ldh + col, r);
    }
    m += a.step_m;
    j += a.step_j;
    if (j >= a.H) { j -= a.H; ++m; }
  }
}

template <typename T, int VEC, int TPR, int E>
__global__ __launch_bounds__((RowKernel<T, VEC, TPR, E>::BT)) void block_norm_bwd_kernel(NormArgs a) {
  using RK = RowKernel<T, VEC, TPR, E>;
  __shared__ float red[2][8][2];
  __shared__ float fold[RK::SLOTS > 1 ? RK::BT * E : 1];
  RK rk{(int)(threadIdx.x % TPR), a.D};
  RowSum<TPR> sum{red, 0};
  const int slot = threadIdx.x / TPR;
  float wq[E], wp[E], bq[E];
  rk.param(a.w_post, 1.f, wq);
  rk.param(a.b_post, 0.f, bq);
  rk.param(a.w_pre, 1.f, wp);
  float acc[4][E], accg[E];
#pragma unroll
  for (int e = 0; e < E; ++e) acc[0][e] = acc[1][e] = acc[2][e] = acc[3][e] = 0.f;

  // sums a register array over the row slots of the workgroup and stores it as one row of D floats
  auto fold_store = [&](float (&v)[E], float* dst) {
    if (RK::SLOTS > 1) {
      __syncthreads();
#pragma unroll
      for (int e = 0; e < E; ++e) fold[e * RK::BT + threadIdx.x] = v[e];
      __syncthreads();
      if (slot == 0) {
        for (int s = 1; s < RK::SLOTS; ++s)
#pragma unroll
          for (int e = 0; e < E; ++e) v[e] += fold[e * RK::BT + s * TPR + rk.lane];
      }
    }
    if (slot == 0) rk.store(dst, v);
  };

  const long seg0 = (long)blockIdx.x * a.segs_per_block;
  const long seg1 = min(a.n_segs, seg0 + a.segs_per_block);
  for (long seg = seg0; seg < seg1; ++seg) {
    const long grp = seg / a.parts;
    const long r0 = grp * a.group_rows + (seg - grp * a.parts) * a.seg_rows;
    const long r1 = min(min(a.R, (grp + 1) * a.group_rows), r0 + a.seg_rows);
    float zg[E], sl[E];
    if (a.gate_bcast) {
      rk.load(static_cast<const float*>(a.gate) + grp * a.ldg, zg);
#pragma unroll
      for (int e = 0; e < E; ++e) accg[e] = 0.f;
    }
    long row = r0 + slot;
    long m = row / a.H;
    int j = (int)(row - m * a.H);
    for (; row < r1; row += RK::SLOTS) {
      const long col = (long)j * a.D;
      float r[E], n[E], g[E], dr[E], dn[E];
      if (a.x) rk.load(static_cast<const T*>(a.x) + m * a.ldx + col, r);
      if (a.y) rk.load(static_cast<const T*>(a.y) + m * a.ldy + col, n);
      if (a.gate && !a.gate_bcast) rk.load(static_cast<const T*>(a.gate) + m * a.ldg + col, zg);
      if (a.d_out) rk.load(static_cast<const T*>(a.d_out) + m * a.lddo + col, dr);
      if (a.d_h) rk.load(static_cast<const T*>(a.d_h) + m * a.lddh + col, dn);
      float rq = 1.f;
#pragma unroll
      for (int e = 0; e < E; ++e) r[e] = a.x ? a.alpha * r[e] : 0.f;
      if (a.y) {
        if (a.post != HHRL_NORM_NONE) rq = rk.normalise(n, a.post, a.inv_d, a.eps, sum);
#pragma unroll
        for (int e = 0; e < E; ++e) {
          g[e] = a.scale;
          sl[e] = 0.f;
          if (a.gate) { g[e] *= gate_value(zg[e], a.gate_act); sl[e] = a.scale * gate_slope(zg[e], a.gate_act); }
        }
      }
#pragma unroll
      for (int e = 0; e < E; ++e) dr[e] = a.d_out ? dr[e] : 0.f;
      if (a.d_h && a.pre != HHRL_NORM_NONE) {
        if (a.y) {
#pragma unroll
          for (int c = 0; c < RK::NCH; ++c)
#pragma unroll
            for (int e0 = 0; e0 < VEC; ++e0) {
              const int e = c * VEC + e0;
              r[e] = rk.at(c) < a.D ? fmaf(g[e], fmaf(n[e], wq[e], bq[e]), r[e]) : 0.f;
            }
        }
        const float rp = rk.normalise(r, a.pre, a.inv_d, a.eps, sum);
#pragma unroll
        for (int e = 0; e < E; ++e) {
          acc[2][e] = fmaf(dn[e], r[e], acc[2][e]);
          acc[3][e] += dn[e];
          dn[e] *= wp[e];
        }
        rk.normalise_back(dn, r, rp, a.pre, a.inv_d, sum);
#pragma unroll
        for (int e = 0; e < E; ++e) dr[e] += dn[e];
      } else if (a.d_h) {
#pragma unroll
        for (int e = 0; e < E; ++e) dr[e] += dn[e];
      }
      if (a.dx) {
#pragma unroll
        for (int e = 0; e < E; ++e) dn[e] = a.alpha * dr[e];
        rk.store(static_cast<T*>(a.dx) + m * a.lddx + col, dn);
      }
      if (a.y) {
        if (a.gate && a.dgate) {
#pragma unroll
          for (int e = 0; e < E; ++e) dn[e] = dr[e] * sl[e] * fmaf(n[e], wq[e], bq[e]);
          if (a.gate_bcast) {
#pragma unroll
            for (int e = 0; e < E; ++e) accg[e] += dn[e];
          } else {
            rk.store(static_cast<T*>(a.dgate) + m * a.lddg + col, dn);
          }
        }
#pragma unroll
        for (int e = 0; e < E; ++e) dr[e] *= g[e];
        if (a.post != HHRL_NORM_NONE) {
#pragma unroll
          for (int e = 0; e < E; ++e) {
            acc[0][e] = fmaf(dr[e], n[e], acc[0][e]);
            acc[1][e] += dr[e];
            dr[e] *= wq[e];
          }
          if (a.dy) rk.normalise_back(dr, n, rq, a.post, a.inv_d, sum);
        }
        if (a.dy) rk.store(static_cast<T*>(a.dy) + m * a.lddy + col, dr);
      }
      m += a.step_m;
      j += a.step_j;
      if (j >= a.H) { j -= a.H; ++m; }
    }
    if (a.gate_bcast && a.dgate) fold_store(accg, a.parts > 1 ? a.gate_ws + seg * a.D : static_cast<float*>(a.dgate) + grp * a.lddg);
  }
#pragma unroll
  for (int q = 0; q < 4; ++q)
    if (a.par_slot[q] >= 0) fold_store(acc[q], a.par_ws + ((long)blockIdx.x * a.n_par + a.par_slot[q]) * a.D);
}

// Sums the partial rows in their order: the parameter gradients (ADDED to dst) over all workgroups, and the gate rows
// (written) over the parts of their group.  32 columns x 8 row lanes per workgroup.
struct NormFoldArgs {
  const float* par_ws;
  const float* gate_ws;
  float* dst[4];
  int n_par, D, blocks, parts;
  float* dgate;
  long lddg, n_groups;
};
__global__ __launch_bounds__(256) void block_norm_fold_kernel(NormFoldArgs a) {
  __shared__ float red[8][33];
  const int cx = threadIdx.x & 31, ry = threadIdx.x >> 5, col = blockIdx.x * 32 + cx;
  for (long job = blockIdx.y; job < a.n_par + a.n_groups; job += gridDim.y) {
    const bool par = job < a.n_par;
    const long grp = job - a.n_par;
    const float* src = par ? a.par_ws + job * a.D : a.gate_ws + grp * a.parts * a.D;
    const long stride = par ? (long)a.n_par * a.D : a.D;
    const int rows = par ? a.blocks : a.parts;
    float s = 0.f;
    if (col < a.D) {
#pragma unroll 8
      for (int r = ry; r < rows; r += 8) s += src[r * stride + col];
    }
    red[ry][cx] = s;
    __syncthreads();
    if (ry == 0 && col < a.D) {
      for (int r = 1; r < 8; ++r) s += red[r][cx];
      if (par) a.dst[job][col] += s;
      else a.dgate[grp * a.lddg + col] = s;
    }
    __syncthreads();
  }
}

namespace {

constexpr int kNormMaxD = 8192;
constexpr int kNormBlocks = 512;           // backward: two workgroups per CU, each with one partial row per parameter

struct NormShape { int tpr, e; };
// Threads per row and elements per thread.  A row of up to 16*16 elements takes 16 lanes (four rows per wave keep all
// lanes busy at the head widths of 64..256), longer ones a wave, 256 or 512 threads; 8 elements per thread where that
// covers the row, 16 otherwise.  Few rows: one wave per row, so that a single row's loads are spread over 64 lanes.
NormShape norm_shape(long R, int D, bool vec) {
  const bool few = R < 2048;
  if (D <= 128 && !few) return {16, 8};
  if (D <= 256 && !few) return {16, 16};
  if (D <= 512) return {64, 8};
  if (D <= 1024 && !few) return {64, 16};
  if (D <= 2048) return {256, 8};
  if (D <= 4096 && (!few || !vec)) return {256, 16};
  if (D <= 4096) return {512, 8};
  return {512, 16};
}

struct NormParts { long group_rows, n_groups, seg_rows, n_segs; int parts, segs_per_block, blocks; };
NormParts norm_parts(long M, int H, long gate_rows, int tpr) {
  NormParts p;
  const long R = M * H;
  const int slots = tpr <= 256 ? 256 / tpr : 1;
  const bool bcast = gate_rows > 1;
  p.group_rows = bcast ? gate_rows : R;
  p.n_groups = (R + p.group_rows - 1) / p.group_rows;
  const long gr = p.group_rows < R ? p.group_rows : R;
  // at least four rows per slot (a partial row costs as much as a row), at most kNormBlocks workgroups
  const long most = (gr + 4L * slots - 1) / (4L * slots);
  long parts = (kNormBlocks + p.n_groups - 1) / p.n_groups;
  if (parts > most) parts = most;
  if (parts < 1) parts = 1;
  p.seg_rows = (gr + parts - 1) / parts;
  p.parts = (int)((gr + p.seg_rows - 1) / p.seg_rows);
  p.n_segs = p.n_groups * p.parts;
  p.segs_per_block = (int)((p.n_segs + kNormBlocks - 1) / kNormBlocks);
  p.blocks = (int)((p.n_segs + p.segs_per_block - 1) / p.segs_per_block);
  return p;
}

bool aligned16(const void* p) { return (reinterpret_cast<unsigned long long>(p) & 15) == 0; }

template <typename T, int VEC, int TPR>
void launch_norm(const NormArgs& a, int e, int blocks, bool bwd, hipStream_t st) {
  constexpr int BT = TPR <= 256 ? 256 : TPR;
  if (bwd) {
    if (e == 8) hipLaunchKernelGGL((block_norm_bwd_kernel<T, VEC, TPR, 8>), dim3(blocks), dim3(BT), 0, st, a);
    else hipLaunchKernelGGL((block_norm_bwd_kernel<T, VEC, TPR, 16>), dim3(blocks), dim3(BT), 0, st, a);
  } else {
    if (e == 8) hipLaunchKernelGGL((block_norm_fwd_kernel<T, VEC, TPR, 8>), dim3(blocks), dim3(BT), 0, st, a);
    else hipLaunchKernelGGL((block_norm_fwd_kernel<T, VEC, TPR, 16>), dim3(blocks), dim3(BT), 0, st, a);
  }
}
template <typename T, int VEC>
void launch_norm(const NormArgs& a, NormShape s, int blocks, bool bwd, hipStream_t st) {
  switch (s.tpr) {
    case 16: launch_norm<T, VEC, 16>(a, s.e, blocks, bwd, st); break;
    case 64: launch_norm<T, VEC, 64>(a, s.e, blocks, bwd, st); break;
    case 256: launch_norm<T, VEC, 256>(a, s.e, blocks, bwd, st); break;
    default: launch_norm<T, VEC, 512>(a, s.e, blocks, bwd, st); break;
  }
}
void launch_norm(const NormArgs& a, int dtype, bool vec, NormShape s, int blocks, bool bwd, hipStream_t st) {
  if (dtype == HHRL_BF16) {
    if (vec) launch_norm<__bf16, 8>(a, s, blocks, bwd, st);
    else launch_norm<__bf16, 1>(a, s, blocks, bwd, st);
  } else {
    if (vec) launch_norm<float, 4>(a, s, blocks, bwd, st);
    else launch_norm<float, 1>(a, s, blocks, bwd, st);
  }
}

int norm_check(const hhrl_block_norm_desc* d, const char* who) {
  HHRL_REQUIRE(d != nullptr, "%s: null descriptor", who);
  HHRL_REQUIRE(d->dtype == HHRL_F32 || d->dtype == HHRL_BF16, "%s: dtype %d", who, d->dtype);
  HHRL_REQUIRE(d->M > 0 && d->H > 0 && d->D > 0, "%s: bad shape M=%ld H=%d D=%d", who, d->M, d->H, d->D);
  HHRL_REQUIRE(d->D <= kNormMaxD, "%s: D=%d (up to %d supported)", who, d->D, kNormMaxD);
  HHRL_REQUIRE(d->M < (1L << 40) / d->H, "%s: M*H too large", who);
  HHRL_REQUIRE(d->post >= HHRL_NORM_NONE && d->post <= HHRL_NORM_LAYER && d->pre >= HHRL_NORM_NONE && d->pre <= HHRL_NORM_LAYER,
               "%s: norm kinds %d, %d", who, d->post, d->pre);
  HHRL_REQUIRE(d->gate_act == HHRL_ACT_NONE || d->gate_act == HHRL_ACT_SIGMOID || d->gate_act == HHRL_ACT_SILU, "%s: gate_act %d", who, d->gate_act);
  HHRL_REQUIRE(d->x || d->y, "%s: neither x nor y", who);
  HHRL_REQUIRE(d->y || (!d->gate && d->post == HHRL_NORM_NONE), "%s: a gate or a post norm without y", who);
  HHRL_REQUIRE(d->gate_rows >= 1, "%s: gate_rows=%ld", who, d->gate_rows);
  HHRL_REQUIRE(d->gate_rows == 1 || d->H == 1, "%s: a gate shared by rows goes with H = 1, not %d", who, d->H);
  HHRL_REQUIRE(d->eps >= 0.f, "%s: eps=%g", who, (double)d->eps);
  HHRL_REQUIRE((d->post != HHRL_NORM_NONE || (!d->w_post && !d->b_post)) && (d->pre != HHRL_NORM_NONE || (!d->w_pre && !d->b_pre)),
               "%s: parameters of a norm that is not there", who);
  const long row = (long)d->H * d->D;
  HHRL_REQUIRE((!d->x || d->ldx >= row) && (!d->y || d->ldy >= row) && (!d->gate || d->ldgate >= row), "%s: leading dimension of an input below H*D=%ld", who, row);
  return HHRL_OK;
}

NormArgs norm_args(const hhrl_block_norm_desc* d) {
  NormArgs a = {};
  a.R = d->M * d->H;
  a.H = d->H; a.D = d->D;
  a.post = d->y ? d->post : HHRL_NORM_NONE;
  a.pre = d->pre;
  a.gate_act = d->gate_act;
  a.gate_rows = d->gate_rows;
  a.gate_bcast = d->gate && d->gate_rows > 1;
  a.alpha = d->alpha; a.scale = d->scale; a.eps = d->eps; a.inv_d = 1.f / d->D;
  a.x = d->x; a.y = d->y; a.gate = d->gate;
  a.ldx = d->ldx; a.ldy = d->ldy; a.ldg = d->ldgate;
  a.w_post = d->w_post; a.b_post = d->b_post; a.w_pre = d->w_pre; a.b_pre = d->b_pre;
  return a;
}

// The 16-byte form reads and writes every operand in vectors: all of them have to allow it.
bool norm_vec(const hhrl_block_norm_desc* d, bool bwd) {
  const int v = d->dtype == HHRL_BF16 ? 8 : 4;
  if (d->D % v) return false;
  auto ok = [&](const void* p, long ld, int el) { return !p || (aligned16(p) && ld % el == 0); };
  const int gv = d->gate_rows > 1 ? 4 : v;
  bool r = ok(d->x, d->ldx, v) && ok(d->y, d->ldy, v) && ok(d->gate, d->ldgate, gv) && ok(d->w_post, 0, 1) && ok(d->b_post, 0, 1) &&
           ok(d->w_pre, 0, 1) && ok(d->b_pre, 0, 1);
  if (!bwd) return r && ok(d->out, d->ldo, v) && ok(d->h, d->ldh, v);
  return r && ok(d->d_out, d->lddo, v) && ok(d->d_h, d->lddh, v) && ok(d->dx, d->lddx, v) && ok(d->dy, d->lddy, v) &&
         ok(d->dgate, d->lddgate, gv) && ok(d->ws, 0, 1);
}

}  // namespace
}  // namespace hhrl

using namespace hhrl;

extern "C" {

long hhrl_block_norm_workspace_floats(long M, int H, int D, long gate_rows) {
  if (M <= 0 || H <= 0 || D <= 0 || D > kNormMaxD || gate_rows < 1 || (gate_rows > 1 && H != 1)) return 0;
  long most = 0;
  for (int tpr : {16, 64, 256, 512}) {                // the thread layout depends on alignment: room for every one
    const NormParts p = norm_parts(M, H, gate_rows, tpr);
    const long n = (long)p.blocks * 4 * D + (p.parts > 1 && gate_rows > 1 ? p.n_segs * D : 0);
    if (n > most) most = n;
  }
  return most;
}

int hhrl_block_norm_forward(const hhrl_block_norm_desc* d, void* stream) {
  HHRL_TRY(norm_check(d, "block_norm_forward"));
  const long row = (long)d->H * d->D;
  HHRL_REQUIRE(d->out || d->h, "block_norm_forward: no output");
  HHRL_REQUIRE(d->pre == HHRL_NORM_NONE || d->h, "block_norm_forward: a pre norm without h");
  HHRL_REQUIRE((!d->out || d->ldo >= row) && (!d->h || d->ldh >= row), "block_norm_forward: leading dimension of an output below H*D=%ld", row);
  NormArgs a = norm_args(d);
  a.out = d->out; a.ldo = d->ldo; a.h = d->h; a.ldh = d->ldh;
  const bool vec = norm_vec(d, false);
  const NormShape s = norm_shape(a.R, a.D, vec);
  const int slots = s.tpr <= 256 ? 256 / s.tpr : 1;
  const long want = (a.R + slots - 1) / slots;
  const int blocks = (int)(want < 2048 ? want : 2048);        // eight workgroups per CU, each over many rows: parameters are read once
  a.step_m = (long)blocks * slots / a.H;
  a.step_j = (int)((long)blocks * slots % a.H);
  const double el = d->dtype == HHRL_BF16 ? 2.0 : 4.0;
  ProfScope ps("block_norm_fwd_kernel", as_stream(stream), 0.0, el * a.R * a.D * ((a.x != nullptr) + (a.y != nullptr) + (a.gate && !a.gate_bcast) + (a.out != nullptr) + (a.h != nullptr)));
  launch_norm(a, d->dtype, vec, s, blocks, false, as_stream(stream));
  return launch_status("block_norm_fwd_kernel");
}

int hhrl_block_norm_backward(const hhrl_block_norm_desc* d, void* stream) {
  HHRL_TRY(norm_check(d, "block_norm_backward"));
  const long row = (long)d->H * d->D;
  HHRL_REQUIRE(d->d_out || d->d_h, "block_norm_backward: no output gradient");
  HHRL_REQUIRE((!d->d_out || d->lddo >= row) && (!d->d_h || d->lddh >= row) && (!d->dx || d->lddx >= row) && (!d->dy || d->lddy >= row) &&
               (!d->dgate || d->lddgate >= row), "block_norm_backward: leading dimension of a gradient below H*D=%ld", row);
  HHRL_REQUIRE((!d->dx || d->x) && (!d->dy || d->y) && (!d->dgate || d->gate), "block_norm_backward: the gradient of an input that is not there");
  HHRL_REQUIRE((!d->dw_post && !d->db_post) || d->post != HHRL_NORM_NONE, "block_norm_backward: parameter gradients of a post norm that is not there");
  HHRL_REQUIRE((!d->dw_pre && !d->db_pre) || (d->pre != HHRL_NORM_NONE && d->d_h), "block_norm_backward: parameter gradients of a pre norm without d_h");
  NormArgs a = norm_args(d);
  a.d_out = d->d_out; a.lddo = d->lddo; a.d_h = d->d_h; a.lddh = d->lddh;
  a.dx = d->dx; a.lddx = d->lddx; a.dy = d->dy; a.lddy = d->lddy; a.dgate = d->dgate; a.lddg = d->lddgate;
  const bool vec = norm_vec(d, true);
  const NormShape s = norm_shape(a.R, a.D, vec);
  const int slots = s.tpr <= 256 ? 256 / s.tpr : 1;
  const NormParts p = norm_parts(d->M, d->H, a.gate_bcast ? d->gate_rows : 1, s.tpr);
  a.group_rows = p.group_rows; a.seg_rows = p.seg_rows; a.n_groups = p.n_groups; a.parts = p.parts;
  a.segs_per_block = p.segs_per_block; a.n_segs = p.n_segs;
  a.step_m = slots / a.H;
  a.step_j = slots % a.H;
  float* const dst[4] = {d->dw_post, d->db_post, d->dw_pre, d->db_pre};
  NormFoldArgs f = {};
  for (int q = 0; q < 4; ++q) {
    a.par_slot[q] = dst[q] ? a.n_par : -1;
    if (dst[q]) f.dst[a.n_par++] = dst[q];
  }
  const bool fold_gate = a.gate_bcast && a.dgate && p.parts > 1;
  const long need = (long)p.blocks * a.n_par * a.D + (fold_gate ? p.n_segs * a.D : 0);
  HHRL_REQUIRE(need == 0 || (d->ws && d->ws_floats >= need), "block_norm_backward: workspace of %ld floats, %ld needed", d->ws ? d->ws_floats : 0L, need);
  a.par_ws = d->ws;
  a.gate_ws = fold_gate ? d->ws + (long)p.blocks * a.n_par * a.D : nullptr;
  const double el = d->dtype == HHRL_BF16 ? 2.0 : 4.0;
  {
    ProfScope ps("block_norm_bwd_kernel", as_stream(stream), 0.0,
                 el * a.R * a.D * ((a.x != nullptr) + (a.y != nullptr) + 2.0 * (a.gate && !a.gate_bcast) + (a.d_out != nullptr) + (a.d_h != nullptr) + (a.dx != nullptr) + (a.dy != nullptr)));
    launch_norm(a, d->dtype, vec, s, p.blocks, true, as_stream(stream));
  }
  HHRL_TRY(launch_status("block_norm_bwd_kernel"));
  if (!a.n_par && !fold_gate) return HHRL_OK;
  f.par_ws = a.par_ws; f.gate_ws = a.gate_ws; f.n_par = a.n_par; f.D = a.D; f.blocks = p.blocks; f.parts = p.parts;
  f.dgate = static_cast<float*>(a.dgate); f.lddg = a.lddg; f.n_groups = fold_gate ? p.n_groups : 0;
  const long jobs = f.n_par + f.n_groups;
  ProfScope ps("block_norm_fold_kernel", as_stream(stream), 0.0, 4.0 * need);
  hipLaunchKernelGGL(block_norm_fold_kernel, dim3(ceil_div(a.D, 32), (unsigned)(jobs < 4096 ? jobs : 4096)), dim3(256), 0, as_stream(stream), f);
  return launch_status("block_norm_fold_kernel");
}

}  // extern "C"
