// The gated delta rule: per value head a matrix state S [K, V],
//   S <- exp(g_t) S;   S <- S + beta_t k_t (v_t - S^T k_t)^T;   o_t = scale * S^T q_t,
// forward and backward over whole sequences, and one token at a time against a pool of states.
//
// Whole sequences go in chunks of 64 tokens.  With G the running sum of g inside a chunk, gam_i = exp(G_i),
// D_ij = exp(G_i - G_j) (i >= j) and S the state in front of the chunk, the recurrence inside the chunk is a unit lower
// triangular system:
//   A = tril(beta_i (k_i.k_j) D_ij, -1),  M = (I + A)^-1,  P = tril((q_i.k_j) D_ij)
//   W = M (beta * (V - gam * (K S)))                      (row i: what token i adds to the state along k_i)
//   o = scale * (gam * (Q S) + P W),   S' = gam_C S + K^T (exp(G_C - G) * W)
// M and P do not depend on the state: one launch forms them for all chunks at once (gdr_prep_kernel).  The launch that
// follows walks the chunks of a sequence (gdr_scan_fwd_kernel); its workgroups hold 32 columns of one head's state in
// registers: columns do not meet.  K and Q are multiplied as they are; decays are applied to fp32 results.
// Backward, with dS' the gradient of the state behind the chunk:
//   Z = scale P^T dO + exp(G_C - G) * (K dS'),   Y = M^T Z,   dV = beta * Y
//   dS = gam_C dS' + Q^T (scale gam * dO) - K^T (gam beta * Y)
// walks the chunks the other way (gdr_scan_bwd_kernel, columns apart again), and everything else is parallel over the
// chunks (gdr_grads_kernel), from the states in front of the chunks, the gradients behind them, W and Y:
//   E1 = dO S^T,  E2 = Y S^T,  E3 = W dS'^T,  R = scale tril(dO W^T) D,  B = -tril(Y W^T, -1) D
//   dq = scale gam E1 + R K
//   H = -gam E2 + B K,   dk = beta H + exp(G_C - G) E3 + (beta B)^T K + R^T Q
//   dbeta_i = Y_i.v_i + k_i.H_i
//   dG_i = q_i.dq_i + beta_i k_i.H_i - k_i.(the other terms of dk_i), dG_C += <dS', S'>, dg = sum of dG from i on.
//
// All products run on the bf16 matrix instruction with fp32 operands as three bf16 terms (split_bf16.h): a decayed,
// corrected state is a difference of numbers much larger than itself, its gradients more so, and dg, dbeta and the
// states are fp32 results.  The decays' sums are kept as two floats from a sum in fp64, so that exp(G_i - G_j) is exact
// to fp32 however far G has run.
#include "common.h"
#include "mfma_tiles.h"
#include "split_bf16.h"

namespace hhrl {

using sb::bf16x4;
using sb::bf16x8;
using sb::f32x4;

constexpr int kC = 64;             // tokens per chunk
constexpr int kVt = 32;            // state columns per workgroup of a scan
constexpr int kLdT = kC + 8;       // row stride of an LDS image that runs along the tokens (16 rows: 16 distinct bank groups)
constexpr int kLdM = kC + 4;       // row stride of the fp32 images of the triangular solve
constexpr float kGMin = -1e4f;     // log decays are clamped here: exp() of it is 0, and infinities would leave NaN differences

struct GdrArgs {
  int n_seq, Hk, Hv, K, V, rep;
  long rows;
  int T, cpt;                      // padded batch: tokens and chunks per sequence
  long n_slots;                    // chunks that have a place in ws
  float scale;
  const int *starts, *lens;
  const void *q, *k, *v;
  long ldq, ldk, ldv;
  const float *g, *beta;
  long ldg, ldbeta;
  void* o;
  long ldo;
  const float *s0, *d_s1;
  float *s1, *d_s0;
  const void* d_o;
  long lddo;
  void *dq, *dk, *dv;
  long lddq, lddk, lddv;
  float *dg, *dbeta;
  long lddg, lddbeta;
  int pack, train, vp, nvt;
  // ws, per chunk and key head: k, q [terms][64][Kp] (pack), their transposes [terms][Kp][64];
  //     per chunk and value head: M, P and their transposes [terms][64][64], five rows of 64 floats, and for the
  //     backward pass W, Y [64][vp] and S, dS [Kp][vp], fp32
  __bf16 *kpk, *qpk, *kt, *qt, *m, *p, *mt, *pt;
  float *vec, *w, *y, *s, *ds;
};
enum { kGam = 0, kTail = 1, kBeta = 2, kGHi = 3, kGLo = 4, kVecs = 5 };

__device__ __forceinline__ long clampl(long v, long lo, long hi) { return v < lo ? lo : v > hi ? hi : v; }

// rows [start, start + len) of sequence n and the place of its first chunk.  Packed sequences of any lengths:
// floor(start/64) + n leaves every sequence at least ceil(len/64) places.
__device__ __forceinline__ void seq_range(const GdrArgs& a, int n, long& start, int& len, long& slot0) {
  if (a.starts) {
    start = clampl(a.starts[n], 0, a.rows);
    len = (int)(clampl(a.starts[n + 1], start, a.rows) - start);
    slot0 = start / kC + n;
  } else {
    start = (long)n * a.T;
    len = a.lens ? (int)clampl(a.lens[n], 0, a.T) : a.T;
    slot0 = (long)n * a.cpt;
  }
}
// the chunk at a place: its first row and its number of tokens (0: nobody's)
__device__ __forceinline__ void slot_chunk(const GdrArgs& a, long slot, long& row0, int& valid) {
  int n = 0;
  if (a.starts) {
    int lo = 0, hi = a.n_seq - 1;                  // the last n whose first place is <= slot
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (clampl(a.starts[mid], 0, a.rows) / kC + mid <= slot) lo = mid;
      else hi = mid - 1;
    }
    n = lo;
  } else {
    n = (int)(slot / a.cpt);
  }
  long start, slot0;
  int len;
  seq_range(a, n, start, len, slot0);
  const long at = (slot - slot0) * kC;
  row0 = start + at;
  valid = at < 0 || at >= len ? 0 : (int)min((long)kC, len - at);
}

// ------------------------------------------------------------------------------------------------------------ prep
// One workgroup per chunk and key head: k k^T and q k^T once, then per value head of the key head the decays, the
// triangular inverse and P.  The inverse goes by blocks: 16 x 16 on the diagonal by substitution (a lane per column), then
// the blocks below them, 16 and 32 wide, as -M22 (L21 M11) on the fp32 matrix instruction.
template <typename T, int NP, int KB2>
__global__ __launch_bounds__(256) void gdr_prep_kernel(GdrArgs a) {
  constexpr int Kp = 64 * KB2, LDK = Kp + 8, KG = Kp / 8;
  extern __shared__ __align__(16) char smem[];
  __bf16* const kl = reinterpret_cast<__bf16*>(smem);          // [NP][64][LDK]
  __bf16* const ql = kl + NP * kC * LDK;
  float* const pm = reinterpret_cast<float*>(smem);            // over kl, once the products are done: P, products of the solve
  float* const tm = pm + kC * kLdM;
  constexpr int kOver = 2 * NP * kC * LDK * 2 > 2 * kC * kLdM * 4 ? 2 * NP * kC * LDK * 2 : 2 * kC * kLdM * 4;
  float* const lm = reinterpret_cast<float*>(smem + kOver);    // [64][kLdM] I + A
  float* const mm = lm + kC * kLdM;                            // [64][kLdM] its inverse
  float* const gh = mm + kC * kLdM;
  float* const gl = gh + kC;
  float* const be = gl + kC;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, lr = lane & 15, lg = lane >> 4;
  const long slot = blockIdx.x;
  const int hk = blockIdx.y;
  long row0;
  int valid;
  slot_chunk(a, slot, row0, valid);
  if (valid == 0) return;
  const long hs = slot * a.Hk + hk;

  // k and q as bf16 terms; what lies beyond the sequence or the head's width becomes 0 and is not read
  for (int side = 0; side < 2; ++side) {
    const T* src = static_cast<const T*>(side ? a.q : a.k) + row0 * (side ? a.ldq : a.ldk) + (long)hk * a.K;
    const long ld = side ? a.ldq : a.ldk;
    __bf16* const dst = side ? ql : kl;
    __bf16* const pk = (side ? a.qpk : a.kpk) + hs * NP * kC * Kp;
    const bool whole = !a.pack;                     // rows of Kp elements, 16-byte aligned
    for (int u = tid; u < kC * KG; u += 256) {
      const int i = u / KG, c = (u - i * KG) * 8;
      bf16x8 t[NP];
      if constexpr (NP == 1) {
        if (whole && i < valid) {
          t[0] = *reinterpret_cast<const bf16x8*>(src + i * ld + c);
        } else {
#pragma unroll
          for (int e = 0; e < 8; ++e) t[0][e] = i < valid && c + e < a.K ? (__bf16)src[i * ld + c + e] : (__bf16)0.f;
        }
      } else {
        float x[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = i < valid && c + e < a.K ? (float)src[i * ld + c + e] : 0.f;
        sb::split8<NP>(x, t);
      }
#pragma unroll
      for (int p = 0; p < NP; ++p) {
        *reinterpret_cast<bf16x8*>(dst + (p * kC + i) * LDK + c) = t[p];
        if (a.pack) *reinterpret_cast<bf16x8*>(pk + ((long)p * kC + i) * Kp + c) = t[p];
      }
    }
  }
  __syncthreads();
  for (int side = 0; side < (a.train ? 2 : 1); ++side) {
    const __bf16* const src = side ? ql : kl;
    __bf16* const dst = (side ? a.qt : a.kt) + hs * NP * Kp * kC;
    for (int u = tid; u < NP * Kp * 8; u += 256) {
      const int k = u % Kp, r = u / Kp, i0 = (r & 7) * 8, p = r >> 3;
      bf16x8 t;
#pragma unroll
      for (int e = 0; e < 8; ++e) t[e] = src[(p * kC + i0 + e) * LDK + k];
      *reinterpret_cast<bf16x8*>(dst + ((long)p * Kp + k) * kC + i0) = t;
    }
  }
  f32x4 kk[4], qk[4];
#pragma unroll
  for (int t = 0; t < 4; ++t) kk[t] = qk[t] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int kb = 0; kb < Kp / 32; ++kb) {
    bf16x8 ka[NP], qa[NP];
    const int off = (16 * wave + lr) * LDK + 32 * kb + 8 * lg;
    sb::load_frag<NP>(ka, kl + off, kC * LDK);
    sb::load_frag<NP>(qa, ql + off, kC * LDK);
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      if (t <= wave) {
        bf16x8 b[NP];
        sb::load_frag<NP>(b, kl + (16 * t + lr) * LDK + 32 * kb + 8 * lg, kC * LDK);
        sb::mma<NP, NP>(kk[t], ka, b);
        sb::mma<NP, NP>(qk[t], qa, b);
      }
    }
  }
  for (int r = 0; r < a.rep; ++r) {
    const int hv = hk * a.rep + r;
    const long vs = slot * a.Hv + hv;
    __syncthreads();                               // kl and ql have been read, the previous head's images too
    // every wave holds token `lane`: running sum of the log decays in fp64, kept as two floats
    {
      const bool in = lane < valid;
      float gi = in ? a.g[(row0 + lane) * a.ldg + hv] : 0.f;
      const float bi = in ? a.beta[(row0 + lane) * a.ldbeta + hv] : 0.f;
      gi = gi < kGMin ? kGMin : gi;
      double G = gi;
#pragma unroll
      for (int off = 1; off < 64; off <<= 1) {
        const double up = __shfl_up(G, off, 64);
        if (lane >= off) G += up;
      }
      const double end = __shfl(G, 63, 64);
      const float hi = (float)G, lo = (float)(G - (double)hi);
      if (wave == 0) {
        gh[lane] = hi; gl[lane] = lo; be[lane] = bi;
        float* const v = a.vec + vs * kVecs * kC + lane;
        v[kGam * kC] = expf(hi) * (1.f + lo);
        v[kTail * kC] = expf((float)(end - G));
        v[kBeta * kC] = bi;
        v[kGHi * kC] = hi;
        v[kGLo * kC] = lo;
      }
    }
    __syncthreads();
    const int ib = 16 * wave + 4 * lg;
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      const int j = 16 * t + lr;
      const float hj = gh[j], lj = gl[j];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int i = ib + e;
        const float d = i >= j ? expf((gh[i] - hj) + (gl[i] - lj)) : 0.f;
        lm[i * kLdM + j] = i > j ? be[i] * kk[t][e] * d : i == j ? 1.f : 0.f;
        pm[i * kLdM + j] = i >= j ? qk[t][e] * d : 0.f;
        mm[i * kLdM + j] = 0.f;
      }
    }
    __syncthreads();
    {
      // diagonal block `wave`: column lr of the inverse by substitution
      const float* const L = lm + 16 * wave * kLdM + 16 * wave;
      float x[16];
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        float s = i == lr ? 1.f : 0.f;
#pragma unroll
        for (int j = 0; j < i; ++j) s = fmaf(-L[i * kLdM + j], x[j], s);
        x[i] = s;
      }
      if (lg == 0) {
#pragma unroll
        for (int i = 0; i < 16; ++i) mm[(16 * wave + i) * kLdM + 16 * wave + lr] = x[i];
      }
    }
    __syncthreads();
    const mt::f32x4 zero = {0.f, 0.f, 0.f, 0.f};
    if (wave < 2) {
      // 16 x 16 below the diagonal of the two 32 x 32 blocks
      const int o1 = 32 * wave, o2 = o1 + 16;
      mt::f32x4 c = mt::wave_mma16<16, kLdM, 1, kLdM, 1>(lm + o2 * kLdM + o1, mm + o1 * kLdM + o1, lane, zero);
      mt::store_block16<kLdM>(tm, o2, 0, c, lane);
      mt::wave_sync();
      c = mt::wave_mma16<16, kLdM, 1, kLdM, 1>(mm + o2 * kLdM + o2, tm + o2 * kLdM, lane, zero);
      mt::store_block16<kLdM>(mm, o2, o1, -c, lane);
    }
    __syncthreads();
    {
      const int ti = 16 * (wave >> 1), tj = 16 * (wave & 1);
      mt::f32x4 c = mt::wave_mma16<32, kLdM, 1, kLdM, 1>(lm + (32 + ti) * kLdM, mm + tj, lane, zero);
      __syncthreads();
      mt::store_block16<kLdM>(tm, ti, tj, c, lane);
      __syncthreads();
      c = mt::wave_mma16<32, kLdM, 1, kLdM, 1>(mm + (32 + ti) * kLdM + 32, tm + tj, lane, zero);
      mt::store_block16<kLdM>(mm, 32 + ti, tj, -c, lane);
    }
    __syncthreads();
    // 16 elements of a row (or of a column, for the transposes the backward scan reads) per thread
    const int row = tid >> 2, c0 = (tid & 3) * 16;
    for (int what = 0; what < (a.train ? 4 : 2); ++what) {
      const float* const src = what & 1 ? pm : mm;
      __bf16* const dst = (what == 0 ? a.m : what == 1 ? a.p : what == 2 ? a.mt : a.pt) + vs * 3 * kC * kC + row * kC + c0;
      const int si = what < 2 ? kLdM : 1, sj = what < 2 ? 1 : kLdM;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        float x[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = src[row * si + (c0 + 8 * h + e) * sj];
        bf16x8 t[3];
        sb::split8<3>(x, t);
#pragma unroll
        for (int p = 0; p < 3; ++p) *reinterpret_cast<bf16x8*>(dst + p * kC * kC + 8 * h) = t[p];
      }
    }
  }
}

// --------------------------------------------------------------------------------------------------------- scans
// Workgroup -> (sequence, value head, column tile).  Workgroups go to the eight XCDs in turn: the column tiles of one
// head read the same k, q, M and P, so they are dealt to one XCD (one L2), eight workgroups apart.
__device__ __forceinline__ bool scan_tile(const GdrArgs& a, int& n, int& hv, int& v0) {
  const int xcd = blockIdx.x & 7, u = blockIdx.x >> 3;
  v0 = (u % a.nvt) * kVt;
  const long pair = (long)(u / a.nvt) * 8 + xcd;
  if (pair >= (long)a.n_seq * a.Hv) return false;
  n = (int)(pair / a.Hv);
  hv = (int)(pair - (long)n * a.Hv);
  return true;
}

template <int NP, int KB2>
struct ScanLds {
  static constexpr int Kp = 64 * KB2, LDS_S = Kp + 8;
  static constexpr int S = 3 * kVt * LDS_S, X = 3 * kVt * kLdT;
  static constexpr int bytes = 2 * (S + 3 * X + (NP == 3 ? X : kVt * kLdT));      // the last: dO as it is (backward)
};

// A-operand rows of k or q: token 16*wave + lr of a chunk, from the packed terms or from the caller's rows
template <int NP, int KB>
__device__ __forceinline__ void load_rows(bf16x8 (&f)[KB][NP], const GdrArgs& a, const void* raw, long ld, const __bf16* packed,
                                          long hs, int hk, long row, bool in, int i, int lg) {
  constexpr int Kp = 32 * KB;
  if (NP == 1 && !a.pack) {
    const __bf16* const p = static_cast<const __bf16*>(raw) + row * ld + (long)hk * Kp + 8 * lg;
#pragma unroll
    for (int kb = 0; kb < KB; ++kb) {
      if (in) {
        f[kb][0] = *reinterpret_cast<const bf16x8*>(p + 32 * kb);
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) f[kb][0][e] = (__bf16)0.f;
      }
    }
  } else {
    const __bf16* const p = packed + (hs * NP * kC + i) * Kp + 8 * lg;
#pragma unroll
    for (int kb = 0; kb < KB; ++kb) sb::load_frag<NP>(f[kb], p + 32 * kb, (long)kC * Kp);
  }
}

template <typename T, int NP, int KB2>
__global__ __launch_bounds__(256, 2) void gdr_scan_fwd_kernel(GdrArgs a) {
  using L = ScanLds<NP, KB2>;
  constexpr int Kp = L::Kp, KB = Kp / 32, LDS_S = L::LDS_S;
  extern __shared__ __align__(16) char smem[];
  __bf16* const sl = reinterpret_cast<__bf16*>(smem);      // [3][32][LDS_S] S, a row per column
  __bf16* const xl = sl + L::S;                            // [3][32][kLdT]  beta (V - gam K S)
  __bf16* const wl = xl + L::X;                            // W
  __bf16* const ul = wl + L::X;                            // exp(G_C - G) W
  int n, hv, v0;
  if (!scan_tile(a, n, hv, v0)) return;
  const int hk = hv / a.rep;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, lr = lane & 15, lg = lane >> 4;
  long start, slot0;
  int len;
  seq_range(a, n, start, len, slot0);
  const int nc = (len + kC - 1) / kC;
  const int ib = 16 * wave + 4 * lg;                       // first of the four tokens of a result register group
  const int nkb = wave < 2 ? 1 : 2;                        // M and P are lower triangular: rows < 32 read 32 columns

  f32x4 S[KB2][2];                                         // rows 16*(KB2*wave + t) + 4*lg + e, columns v0 + 16*c + lr
#pragma unroll
  for (int t = 0; t < KB2; ++t)
#pragma unroll
    for (int c = 0; c < 2; ++c)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int k = 16 * (KB2 * wave + t) + 4 * lg + e, v = v0 + 16 * c + lr;
        S[t][c][e] = a.s0 && k < a.K && v < a.V ? a.s0[(((long)n * a.Hv + hv) * a.K + k) * a.V + v] : 0.f;
      }
  for (int c = 0; c < nc; ++c) {
    const long slot = slot0 + c, hs = slot * a.Hk + hk, vs = slot * a.Hv + hv;
    const long row0 = start + (long)c * kC;
    const int valid = min(kC, len - c * kC);
    const float* const vec = a.vec + vs * kVecs * kC;
    const f32x4 gam = *reinterpret_cast<const f32x4*>(vec + kGam * kC + ib);
    const f32x4 tail = *reinterpret_cast<const f32x4*>(vec + kTail * kC + ib);
    const f32x4 beta = *reinterpret_cast<const f32x4*>(vec + kBeta * kC + ib);
    const float last = vec[kGam * kC + kC - 1];
    bf16x8 kf[KB][NP], qf[KB][NP];
    const int ia = 16 * wave + lr;
    load_rows<NP, KB>(kf, a, a.k, a.ldk, a.kpk, hs, hk, row0 + ia, ia < valid, ia, lg);
    load_rows<NP, KB>(qf, a, a.q, a.ldq, a.qpk, hs, hk, row0 + ia, ia < valid, ia, lg);
    f32x4 vv[2];
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int v = v0 + 16 * t + lr;
        vv[t][e] = ib + e < valid && v < a.V ? (float)static_cast<const T*>(a.v)[(row0 + ib + e) * a.ldv + (long)hv * a.V + v] : 0.f;
      }
#pragma unroll
    for (int t = 0; t < KB2; ++t)
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const int k = 16 * (KB2 * wave + t) + 4 * lg;
        sb::split_store4<3>(sl + (16 * u + lr) * LDS_S + k, kVt * LDS_S, S[t][u]);
        if (a.train) {
#pragma unroll
          for (int e = 0; e < 4; ++e) a.s[(vs * Kp + k + e) * a.vp + v0 + 16 * u + lr] = S[t][u][e];
        }
      }
    lds_barrier();
    f32x4 ks[2], qs[2];
    ks[0] = ks[1] = qs[0] = qs[1] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int kb = 0; kb < KB; ++kb)
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        bf16x8 b[3];
        sb::load_frag<3>(b, sl + (16 * t + lr) * LDS_S + 32 * kb + 8 * lg, kVt * LDS_S);
        sb::mma<NP, 3>(ks[t], kf[kb], b);
        sb::mma<NP, 3>(qs[t], qf[kb], b);
      }
#pragma unroll
    for (int t = 0; t < 2; ++t) sb::split_store4<3>(xl + (16 * t + lr) * kLdT + ib, kVt * kLdT, beta * (vv[t] - gam * ks[t]));
    lds_barrier();
    f32x4 w[2];
    w[0] = w[1] = f32x4{0.f, 0.f, 0.f, 0.f};
    const __bf16* const mrow = a.m + vs * 3 * kC * kC + ia * kC + 8 * lg;
    for (int kb = 0; kb < nkb; ++kb) {
      bf16x8 mf[3];
      sb::load_frag<3>(mf, mrow + 32 * kb, kC * kC);
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        bf16x8 b[3];
        sb::load_frag<3>(b, xl + (16 * t + lr) * kLdT + 32 * kb + 8 * lg, kVt * kLdT);
        sb::mma<3, 3>(w[t], mf, b);
      }
    }
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      sb::split_store4<3>(wl + (16 * t + lr) * kLdT + ib, kVt * kLdT, w[t]);
      sb::split_store4<3>(ul + (16 * t + lr) * kLdT + ib, kVt * kLdT, tail * w[t]);
      if (a.train) {
#pragma unroll
        for (int e = 0; e < 4; ++e) a.w[(vs * kC + ib + e) * a.vp + v0 + 16 * t + lr] = w[t][e];
      }
    }
    lds_barrier();
    const __bf16* const ktr = a.kt + hs * NP * Kp * kC + 8 * lg;
#pragma unroll
    for (int t = 0; t < KB2; ++t) {
      S[t][0] *= last;
      S[t][1] *= last;
#pragma unroll
      for (int kb = 0; kb < 2; ++kb) {
        bf16x8 f[NP];
        sb::load_frag<NP>(f, ktr + (16 * (KB2 * wave + t) + lr) * kC + 32 * kb, Kp * kC);
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          bf16x8 b[3];
          sb::load_frag<3>(b, ul + (16 * u + lr) * kLdT + 32 * kb + 8 * lg, kVt * kLdT);
          sb::mma<NP, 3>(S[t][u], f, b);
        }
      }
    }
    const __bf16* const prow = a.p + vs * 3 * kC * kC + ia * kC + 8 * lg;
#pragma unroll
    for (int t = 0; t < 2; ++t) qs[t] *= gam;
    for (int kb = 0; kb < nkb; ++kb) {
      bf16x8 pf[3];
      sb::load_frag<3>(pf, prow + 32 * kb, kC * kC);
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        bf16x8 b[3];
        sb::load_frag<3>(b, wl + (16 * t + lr) * kLdT + 32 * kb + 8 * lg, kVt * kLdT);
        sb::mma<3, 3>(qs[t], pf, b);
      }
    }
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int v = v0 + 16 * t + lr;
        if (ib + e < valid && v < a.V) static_cast<T*>(a.o)[(row0 + ib + e) * a.ldo + (long)hv * a.V + v] = (T)(a.scale * qs[t][e]);
      }
  }
  if (a.s1) {
#pragma unroll
    for (int t = 0; t < KB2; ++t)
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int k = 16 * (KB2 * wave + t) + 4 * lg + e, v = v0 + 16 * u + lr;
          if (k < a.K && v < a.V) a.s1[(((long)n * a.Hv + hv) * a.K + k) * a.V + v] = S[t][u][e];
        }
  }
}

template <typename T, int NP, int KB2>
__global__ __launch_bounds__(256, 2) void gdr_scan_bwd_kernel(GdrArgs a) {
  using L = ScanLds<NP, KB2>;
  constexpr int Kp = L::Kp, KB = Kp / 32, LDS_S = L::LDS_S;
  extern __shared__ __align__(16) char smem[];
  __bf16* const dl = reinterpret_cast<__bf16*>(smem);      // [3][32][LDS_S] dS'
  __bf16* const gl = dl + L::S;                            // [3][32][kLdT]  scale gam dO
  __bf16* const zl = gl + L::X;                            // Z
  __bf16* const yl = zl + L::X;                            // -gam beta Y
  __bf16* const ol = yl + L::X;                            // [NP][32][kLdT] dO
  int n, hv, v0;
  if (!scan_tile(a, n, hv, v0)) return;
  const int hk = hv / a.rep;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, lr = lane & 15, lg = lane >> 4;
  long start, slot0;
  int len;
  seq_range(a, n, start, len, slot0);
  const int nc = (len + kC - 1) / kC;
  const int ib = 16 * wave + 4 * lg, ia = 16 * wave + lr;
  const int kb0 = wave < 2 ? 0 : 1;                        // P^T and M^T are upper triangular

  f32x4 dS[KB2][2];
#pragma unroll
  for (int t = 0; t < KB2; ++t)
#pragma unroll
    for (int c = 0; c < 2; ++c)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int k = 16 * (KB2 * wave + t) + 4 * lg + e, v = v0 + 16 * c + lr;
        dS[t][c][e] = a.d_s1 && k < a.K && v < a.V ? a.d_s1[(((long)n * a.Hv + hv) * a.K + k) * a.V + v] : 0.f;
      }
  for (int c = nc - 1; c >= 0; --c) {
    const long slot = slot0 + c, hs = slot * a.Hk + hk, vs = slot * a.Hv + hv;
    const long row0 = start + (long)c * kC;
    const int valid = min(kC, len - c * kC);
    const float* const vec = a.vec + vs * kVecs * kC;
    const f32x4 gam = *reinterpret_cast<const f32x4*>(vec + kGam * kC + ib);
    const f32x4 tail = *reinterpret_cast<const f32x4*>(vec + kTail * kC + ib);
    const f32x4 beta = *reinterpret_cast<const f32x4*>(vec + kBeta * kC + ib);
    const float last = vec[kGam * kC + kC - 1];
    bf16x8 kf[KB][NP];
    load_rows<NP, KB>(kf, a, a.k, a.ldk, a.kpk, hs, hk, row0 + ia, ia < valid, ia, lg);
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      f32x4 d;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int v = v0 + 16 * t + lr;
        d[e] = a.d_o && ib + e < valid && v < a.V ? (float)static_cast<const T*>(a.d_o)[(row0 + ib + e) * a.lddo + (long)hv * a.V + v] : 0.f;
      }
      sb::split_store4<NP>(ol + (16 * t + lr) * kLdT + ib, kVt * kLdT, d);
      sb::split_store4<3>(gl + (16 * t + lr) * kLdT + ib, kVt * kLdT, a.scale * gam * d);
    }
#pragma unroll
    for (int t = 0; t < KB2; ++t)
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const int k = 16 * (KB2 * wave + t) + 4 * lg;
        sb::split_store4<3>(dl + (16 * u + lr) * LDS_S + k, kVt * LDS_S, dS[t][u]);
#pragma unroll
        for (int e = 0; e < 4; ++e) a.ds[(vs * Kp + k + e) * a.vp + v0 + 16 * u + lr] = dS[t][u][e];
      }
    lds_barrier();
    f32x4 z[2], y[2];
    z[0] = z[1] = y[0] = y[1] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int kb = 0; kb < KB; ++kb)
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        bf16x8 b[3];
        sb::load_frag<3>(b, dl + (16 * t + lr) * LDS_S + 32 * kb + 8 * lg, kVt * LDS_S);
        sb::mma<NP, 3>(z[t], kf[kb], b);
      }
    const __bf16* const prow = a.pt + vs * 3 * kC * kC + ia * kC + 8 * lg;
    for (int kb = kb0; kb < 2; ++kb) {
      bf16x8 f[3];
      sb::load_frag<3>(f, prow + 32 * kb, kC * kC);
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        bf16x8 b[NP];
        sb::load_frag<NP>(b, ol + (16 * t + lr) * kLdT + 32 * kb + 8 * lg, kVt * kLdT);
        sb::mma<3, NP>(y[t], f, b);
      }
    }
#pragma unroll
    for (int t = 0; t < 2; ++t) sb::split_store4<3>(zl + (16 * t + lr) * kLdT + ib, kVt * kLdT, a.scale * y[t] + tail * z[t]);
    lds_barrier();
    y[0] = y[1] = f32x4{0.f, 0.f, 0.f, 0.f};
    const __bf16* const mrow = a.mt + vs * 3 * kC * kC + ia * kC + 8 * lg;
    for (int kb = kb0; kb < 2; ++kb) {
      bf16x8 f[3];
      sb::load_frag<3>(f, mrow + 32 * kb, kC * kC);
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        bf16x8 b[3];
        sb::load_frag<3>(b, zl + (16 * t + lr) * kLdT + 32 * kb + 8 * lg, kVt * kLdT);
        sb::mma<3, 3>(y[t], f, b);
      }
    }
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      sb::split_store4<3>(yl + (16 * t + lr) * kLdT + ib, kVt * kLdT, -gam * beta * y[t]);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int v = v0 + 16 * t + lr;
        a.y[(vs * kC + ib + e) * a.vp + v] = y[t][e];
        if (ib + e < valid && v < a.V) static_cast<T*>(a.dv)[(row0 + ib + e) * a.lddv + (long)hv * a.V + v] = (T)(beta[e] * y[t][e]);
      }
    }
    lds_barrier();
    const __bf16* const ktr = a.kt + hs * NP * Kp * kC + 8 * lg;
    const __bf16* const qtr = a.qt + hs * NP * Kp * kC + 8 * lg;
#pragma unroll
    for (int t = 0; t < KB2; ++t) {
      dS[t][0] *= last;
      dS[t][1] *= last;
#pragma unroll
      for (int kb = 0; kb < 2; ++kb) {
        bf16x8 f[NP], h[NP];
        const int off = (16 * (KB2 * wave + t) + lr) * kC + 32 * kb;
        sb::load_frag<NP>(f, ktr + off, Kp * kC);
        sb::load_frag<NP>(h, qtr + off, Kp * kC);
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          bf16x8 b[3];
          sb::load_frag<3>(b, gl + (16 * u + lr) * kLdT + 32 * kb + 8 * lg, kVt * kLdT);
          sb::mma<NP, 3>(dS[t][u], h, b);
          sb::load_frag<3>(b, yl + (16 * u + lr) * kLdT + 32 * kb + 8 * lg, kVt * kLdT);
          sb::mma<NP, 3>(dS[t][u], f, b);
        }
      }
    }
    lds_barrier();                                 // gl and yl have been read: the next chunk writes gl before its first barrier
  }
  if (a.d_s0) {
#pragma unroll
    for (int t = 0; t < KB2; ++t)
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int k = 16 * (KB2 * wave + t) + 4 * lg + e, v = v0 + 16 * u + lr;
          if (k < a.K && v < a.V) a.d_s0[(((long)n * a.Hv + hv) * a.K + k) * a.V + v] = dS[t][u][e];
        }
  }
}

// ------------------------------------------------------------------------------------------------------ gradients
// One workgroup per chunk and key head; the value heads of the key head one after the other, so that dq and dk are summed
// in registers in a fixed order.  A wave holds 16 tokens against all of K; S, dS' and W pass through LDS 32 columns at a
// time as bf16 terms.
template <typename T, int NP, int KB2, bool GROUP>
__global__ __launch_bounds__(256, 1) void gdr_grads_kernel(GdrArgs a) {
  constexpr int Kp = 64 * KB2, KT = Kp / 16, LDV = 40;       // 32 columns + 8: 16 rows in 16 distinct bank groups
  extern __shared__ __align__(16) char smem[];
  __bf16* const sl = reinterpret_cast<__bf16*>(smem);        // [3][Kp][LDV]
  __bf16* const dl = sl + 3 * Kp * LDV;                      // [3][Kp][LDV]
  __bf16* const wl = dl + 3 * Kp * LDV;                      // [3][64][LDV]
  __bf16* const rl = reinterpret_cast<__bf16*>(smem);        // over them afterwards: R and B, then their transposes
  __bf16* const bl = rl + 3 * kC * kLdT;                     // [3][64][kLdT]
  constexpr int kOver = 2 * 3 * LDV * (2 * Kp + kC) > 2 * 2 * 3 * kC * kLdT ? 2 * 3 * LDV * (2 * Kp + kC) : 2 * 2 * 3 * kC * kLdT;
  float* const rows = reinterpret_cast<float*>(smem + kOver);      // [4][64]: Y.v, dG without the state's share, dbeta's rest, k.(tail E3)
  float* const red = rows + 4 * kC;                                // [4]
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, lr = lane & 15, lg = lane >> 4;
  const long slot = blockIdx.x;
  const int hk = blockIdx.y;
  long row0;
  int valid;
  slot_chunk(a, slot, row0, valid);
  if (valid == 0) return;
  const long hs = slot * a.Hk + hk;
  const int ib = 16 * wave + 4 * lg, ia = 16 * wave + lr;
  const f32x4 zero = {0.f, 0.f, 0.f, 0.f};

  f32x4 dqs[GROUP ? KT : 1], dks[GROUP ? KT : 1];
  if (GROUP) {
#pragma unroll
    for (int t = 0; t < (GROUP ? KT : 1); ++t) dqs[t] = dks[t] = zero;
  }
  for (int r = 0; r < a.rep; ++r) {
    const int hv = hk * a.rep + r;
    const long vs = slot * a.Hv + hv;
    f32x4 e1[KT], e2[KT], e3[KT], dp[4], da[4];
#pragma unroll
    for (int t = 0; t < KT; ++t) e1[t] = e2[t] = e3[t] = zero;
#pragma unroll
    for (int t = 0; t < 4; ++t) dp[t] = da[t] = zero;
    float sdot = 0.f, yv = 0.f;
    for (int vb = 0; vb < a.vp; vb += 32) {
      __syncthreads();
#pragma unroll
      for (int u0 = 0; u0 < Kp * 4; u0 += 256) {
        const int u = u0 + tid, k = u >> 2, c = (u & 3) * 8;
        const float* const ps = a.s + (vs * Kp + k) * a.vp + vb + c;
        const float* const pd = a.ds + (vs * Kp + k) * a.vp + vb + c;
        float x[8], d[8];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const f32x4 t = *reinterpret_cast<const f32x4*>(ps + 4 * h), w = *reinterpret_cast<const f32x4*>(pd + 4 * h);
#pragma unroll
          for (int e = 0; e < 4; ++e) { x[4 * h + e] = t[e]; d[4 * h + e] = w[e]; sdot = fmaf(t[e], w[e], sdot); }
        }
        bf16x8 t[3];
        sb::split8<3>(x, t);
#pragma unroll
        for (int p = 0; p < 3; ++p) *reinterpret_cast<bf16x8*>(sl + (p * Kp + k) * LDV + c) = t[p];
        sb::split8<3>(d, t);
#pragma unroll
        for (int p = 0; p < 3; ++p) *reinterpret_cast<bf16x8*>(dl + (p * Kp + k) * LDV + c) = t[p];
      }
      {
        const int i = tid >> 2, c = (tid & 3) * 8;
        const float* const pw = a.w + (vs * kC + i) * a.vp + vb + c;
        float x[8];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const f32x4 t = *reinterpret_cast<const f32x4*>(pw + 4 * h);
#pragma unroll
          for (int e = 0; e < 4; ++e) x[4 * h + e] = t[e];
        }
        bf16x8 t[3];
        sb::split8<3>(x, t);
#pragma unroll
        for (int p = 0; p < 3; ++p) *reinterpret_cast<bf16x8*>(wl + (p * kC + i) * LDV + c) = t[p];
      }
      // this wave's rows of dO, Y and W
      bf16x8 of[NP], yf[3], wf[3];
      {
        float x[8], y[8];
        const float* const py = a.y + (vs * kC + ia) * a.vp + vb + 8 * lg;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const f32x4 t = *reinterpret_cast<const f32x4*>(py + 4 * h);
#pragma unroll
          for (int e = 0; e < 4; ++e) y[4 * h + e] = t[e];
        }
        sb::split8<3>(y, yf);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const int v = vb + 8 * lg + e;
          const bool in = ia < valid && v < a.V;
          x[e] = a.d_o && in ? (float)static_cast<const T*>(a.d_o)[(row0 + ia) * a.lddo + (long)hv * a.V + v] : 0.f;
          if (in) yv = fmaf(y[e], (float)static_cast<const T*>(a.v)[(row0 + ia) * a.ldv + (long)hv * a.V + v], yv);
        }
        sb::split8<NP>(x, of);
      }
      __syncthreads();
      sb::load_frag<3>(wf, wl + ia * LDV + 8 * lg, kC * LDV);
#pragma unroll
      for (int t = 0; t < KT; ++t) {
        bf16x8 b[3];
        sb::load_frag<3>(b, sl + (16 * t + lr) * LDV + 8 * lg, Kp * LDV);
        sb::mma<NP, 3>(e1[t], of, b);
        sb::mma<3, 3>(e2[t], yf, b);
        sb::load_frag<3>(b, dl + (16 * t + lr) * LDV + 8 * lg, Kp * LDV);
        sb::mma<3, 3>(e3[t], wf, b);
      }
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        if (t <= wave) {
          bf16x8 b[3];
          sb::load_frag<3>(b, wl + (16 * t + lr) * LDV + 8 * lg, kC * LDV);
          sb::mma<NP, 3>(dp[t], of, b);
          sb::mma<3, 3>(da[t], yf, b);
        }
      }
    }
    yv += __shfl_xor(yv, 16, 64);
    yv += __shfl_xor(yv, 32, 64);
    sdot = wave_sum(sdot);
    const float* const vec = a.vec + vs * kVecs * kC;
    const f32x4 gam = *reinterpret_cast<const f32x4*>(vec + kGam * kC + ib);
    const f32x4 tail = *reinterpret_cast<const f32x4*>(vec + kTail * kC + ib);
    const f32x4 beta = *reinterpret_cast<const f32x4*>(vec + kBeta * kC + ib);
    const f32x4 ghi = *reinterpret_cast<const f32x4*>(vec + kGHi * kC + ib);
    const f32x4 glo = *reinterpret_cast<const f32x4*>(vec + kGLo * kC + ib);
    const float last = vec[kGam * kC + kC - 1];
    __syncthreads();
    if (lg == 0) rows[ia] = yv;
    if (lane == 0) red[wave] = sdot;
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      const int j = 16 * t + lr;
      const float hj = vec[kGHi * kC + j], lj = vec[kGLo * kC + j];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int i = ib + e;
        const float d = i >= j ? expf((ghi[e] - hj) + (glo[e] - lj)) : 0.f;
        dp[t][e] = i >= j ? a.scale * dp[t][e] * d : 0.f;
        da[t][e] = i > j ? -da[t][e] * d : 0.f;
        __bf16 x[3];
        sb::split3(dp[t][e], x[0], x[1], x[2]);
#pragma unroll
        for (int p = 0; p < 3; ++p) rl[(p * kC + i) * kLdT + j] = x[p];
        sb::split3(da[t][e], x[0], x[1], x[2]);
#pragma unroll
        for (int p = 0; p < 3; ++p) bl[(p * kC + i) * kLdT + j] = x[p];
      }
    }
#pragma unroll
    for (int t = 0; t < KT; ++t) {
      e1[t] *= a.scale * gam;
      e2[t] *= -gam;
      e3[t] *= tail;
    }
    __syncthreads();
    const __bf16* const ktr = a.kt + hs * NP * Kp * kC + lr * kC + 8 * lg;
    const __bf16* const qtr = a.qt + hs * NP * Kp * kC + lr * kC + 8 * lg;
    for (int kb = 0; kb < (wave < 2 ? 1 : 2); ++kb) {
      bf16x8 rf[3], bf[3];
      sb::load_frag<3>(rf, rl + ia * kLdT + 32 * kb + 8 * lg, kC * kLdT);
      sb::load_frag<3>(bf, bl + ia * kLdT + 32 * kb + 8 * lg, kC * kLdT);
#pragma unroll
      for (int t = 0; t < KT; ++t) {
        bf16x8 b[NP];
        sb::load_frag<NP>(b, ktr + 16 * t * kC + 32 * kb, Kp * kC);
        sb::mma<3, NP>(e1[t], rf, b);
        sb::mma<3, NP>(e2[t], bf, b);
      }
    }
    __syncthreads();
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      sb::split_store4<3>(rl + (16 * t + lr) * kLdT + ib, kC * kLdT, dp[t]);
      sb::split_store4<3>(bl + (16 * t + lr) * kLdT + ib, kC * kLdT, beta * da[t]);
    }
    // row sums that need k and q as fp32, and k.(tail E3) before the other terms join
    f32x4 dg = zero, db = zero, st = zero;
#pragma unroll
    for (int t = 0; t < KT; ++t)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int k = 16 * t + lr;
        const bool in = ib + e < valid && k < a.K;
        const float kv = in ? (float)static_cast<const T*>(a.k)[(row0 + ib + e) * a.ldk + (long)hk * a.K + k] : 0.f;
        const float qv = in ? (float)static_cast<const T*>(a.q)[(row0 + ib + e) * a.ldq + (long)hk * a.K + k] : 0.f;
        dg[e] = fmaf(qv, e1[t][e], dg[e]);
        db[e] = fmaf(kv, e2[t][e], db[e]);
        st[e] = fmaf(kv, e3[t][e], st[e]);
      }
    __syncthreads();
    for (int kb = wave < 2 ? 0 : 1; kb < 2; ++kb) {
      bf16x8 rf[3], bf[3];
      sb::load_frag<3>(rf, rl + ia * kLdT + 32 * kb + 8 * lg, kC * kLdT);
      sb::load_frag<3>(bf, bl + ia * kLdT + 32 * kb + 8 * lg, kC * kLdT);
#pragma unroll
      for (int t = 0; t < KT; ++t) {
        bf16x8 b[NP];
        sb::load_frag<NP>(b, qtr + 16 * t * kC + 32 * kb, Kp * kC);
        sb::mma<3, NP>(e3[t], rf, b);
        sb::load_frag<NP>(b, ktr + 16 * t * kC + 32 * kb, Kp * kC);
        sb::mma<3, NP>(e3[t], bf, b);
      }
    }
    f32x4 kc = zero;
#pragma unroll
    for (int t = 0; t < KT; ++t) {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int k = 16 * t + lr;
        const bool in = ib + e < valid && k < a.K;
        const float kv = in ? (float)static_cast<const T*>(a.k)[(row0 + ib + e) * a.ldk + (long)hk * a.K + k] : 0.f;
        kc[e] = fmaf(kv, e3[t][e], kc[e]);
      }
      e2[t] = e2[t] * beta + e3[t];                          // dk of this value head
      if (GROUP) { dqs[t] += e1[t]; dks[t] += e2[t]; }
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      float x = dg[e] + beta[e] * db[e] - kc[e], y = db[e], z = st[e];
#pragma unroll
      for (int off = 8; off > 0; off >>= 1) {
        x += __shfl_xor(x, off, 64);
        y += __shfl_xor(y, off, 64);
        z += __shfl_xor(z, off, 64);
      }
      if (lr == 0) { rows[kC + ib + e] = x; rows[2 * kC + ib + e] = y; rows[3 * kC + ib + e] = z; }
    }
    __syncthreads();
    if (wave == 0) {
      // <dS', S'> = gam_C <dS', S> + sum_i k_i.(tail E3)_i reaches every token of the chunk, dG_i those up to i
      double share = rows[3 * kC + lane];
#pragma unroll
      for (int off = 32; off > 0; off >>= 1) share += __shfl_xor(share, off, 64);
      share += (double)last * ((double)red[0] + red[1] + red[2] + red[3]);
      double s = rows[kC + lane];
#pragma unroll
      for (int off = 1; off < 64; off <<= 1) {
        const double down = __shfl_down(s, off, 64);
        if (lane + off < 64) s += down;
      }
      if (lane < valid) {
        a.dg[(row0 + lane) * a.lddg + hv] = (float)(s + share);
        a.dbeta[(row0 + lane) * a.lddbeta + hv] = rows[lane] + rows[2 * kC + lane];
      }
    }
    if (r == a.rep - 1) {
#pragma unroll
      for (int t = 0; t < KT; ++t) {
        const f32x4 dq = GROUP ? dqs[t] : e1[t], dk = GROUP ? dks[t] : e2[t];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int k = 16 * t + lr;
          if (ib + e < valid && k < a.K) {
            static_cast<T*>(a.dq)[(row0 + ib + e) * a.lddq + (long)hk * a.K + k] = (T)dq[e];
            static_cast<T*>(a.dk)[(row0 + ib + e) * a.lddk + (long)hk * a.K + k] = (T)dk[e];
          }
        }
      }
    }
  }
}

// ------------------------------------------------------------------------------------------------------- one token
// A workgroup holds 16 columns (x VEC) of one row's head: 16 threads along the columns, 16 along K.  The two sums over K
// that a token needs, S^T k and S^T q, are taken of the state as it is stored: o = scale (a S^T q + (q.k) u) with
// u = beta (v - a S^T k), so the state is read once, moved in registers and written once, behind one exchange in LDS.
struct GdrStepArgs {
  int Hk, Hv, K, V, rep, n_slots, nvt;
  float scale;
  const void *q, *k, *v;
  long ldq, ldk, ldv;
  const float *g, *beta;
  long ldg, ldbeta;
  void* o;
  long ldo;
  const float* sin;
  float* sout;
  const int* slots;
};
template <typename T, int VEC, int RPT>
__global__ __launch_bounds__(256) void gdr_step_kernel(GdrStepArgs a) {
  constexpr int VB = 16 * VEC;
  __shared__ float ks[16][VB], qs[16][VB], qk16[16];
  __shared__ float kx[16 * RPT], qx[16 * RPT];
  const int tid = threadIdx.x, cx = tid & 15, kg = tid >> 4;
  const int vt = blockIdx.x % a.nvt, hv = (blockIdx.x / a.nvt) % a.Hv;
  const long b = blockIdx.x / ((long)a.nvt * a.Hv);
  const int hk = hv / a.rep, col = vt * VB + cx * VEC;
  long slot = b;
  bool bad = false;
  if (a.slots) {
    slot = a.slots[b];
    int dup = slot >= a.n_slots;
    if (slot >= 0)
      for (long i = tid; i < b; i += 256) dup |= a.slots[i] == slot;
    bad = __syncthreads_or(dup) != 0;
  }
  T* const op = static_cast<T*>(a.o) + b * a.ldo + (long)hv * a.V + col;
  if (slot < 0 || bad) {
    if (kg == 0)
      for (int e = 0; e < VEC; ++e)
        if (col + e < a.V) op[e] = (T)(bad ? __builtin_nanf("") : 0.f);
    return;
  }
  const long base = (slot * a.Hv + hv) * a.K * a.V + col;
  float s[RPT][VEC];
#pragma unroll
  for (int r = 0; r < RPT; ++r) {
    const int k = r * 16 + kg;
    if constexpr (VEC == 4) {
      f32x4 t = {0.f, 0.f, 0.f, 0.f};
      if (k < a.K && col < a.V) t = *reinterpret_cast<const f32x4*>(a.sin + base + (long)k * a.V);
#pragma unroll
      for (int e = 0; e < 4; ++e) s[r][e] = t[e];
    } else {
      s[r][0] = k < a.K && col < a.V ? a.sin[base + (long)k * a.V] : 0.f;
    }
  }
  for (int k = tid; k < 16 * RPT; k += 256) {
    kx[k] = k < a.K ? (float)static_cast<const T*>(a.k)[b * a.ldk + (long)hk * a.K + k] : 0.f;
    qx[k] = k < a.K ? (float)static_cast<const T*>(a.q)[b * a.ldq + (long)hk * a.K + k] : 0.f;
  }
  const float dec = expf(a.g[b * a.ldg + hv]), beta = a.beta[b * a.ldbeta + hv];
  float vv[VEC];
#pragma unroll
  for (int e = 0; e < VEC; ++e) vv[e] = col + e < a.V ? (float)static_cast<const T*>(a.v)[b * a.ldv + (long)hv * a.V + col + e] : 0.f;
  __syncthreads();
  float sk[VEC], sq[VEC], qk = 0.f;
#pragma unroll
  for (int e = 0; e < VEC; ++e) sk[e] = sq[e] = 0.f;
#pragma unroll
  for (int r = 0; r < RPT; ++r) {
    const float kv = kx[r * 16 + kg], qv = qx[r * 16 + kg];
    qk = fmaf(qv, kv, qk);
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
      sk[e] = fmaf(s[r][e], kv, sk[e]);
      sq[e] = fmaf(s[r][e], qv, sq[e]);
    }
  }
#pragma unroll
  for (int e = 0; e < VEC; ++e) { ks[kg][cx * VEC + e] = sk[e]; qs[kg][cx * VEC + e] = sq[e]; }
  if (cx == 0) qk16[kg] = qk;
  __syncthreads();
  float u[VEC];
#pragma unroll
  for (int e = 0; e < VEC; ++e) sk[e] = sq[e] = 0.f;
  qk = 0.f;
#pragma unroll
  for (int r = 0; r < 16; ++r) {
    qk += qk16[r];
#pragma unroll
    for (int e = 0; e < VEC; ++e) { sk[e] += ks[r][cx * VEC + e]; sq[e] += qs[r][cx * VEC + e]; }
  }
#pragma unroll
  for (int e = 0; e < VEC; ++e) u[e] = beta * (vv[e] - dec * sk[e]);
#pragma unroll
  for (int r = 0; r < RPT; ++r) {
    const int k = r * 16 + kg;
    if (k < a.K && col < a.V) {
      const float kv = kx[k];
      if constexpr (VEC == 4) {
        f32x4 t;
#pragma unroll
        for (int e = 0; e < 4; ++e) t[e] = fmaf(kv, u[e], dec * s[r][e]);
        *reinterpret_cast<f32x4*>(a.sout + base + (long)k * a.V) = t;
      } else {
        a.sout[base + (long)k * a.V] = fmaf(kv, u[0], dec * s[r][0]);
      }
    }
  }
  if (kg == 0) {
#pragma unroll
    for (int e = 0; e < VEC; ++e)
      if (col + e < a.V) op[e] = (T)(a.scale * fmaf(qk, u[e], dec * sq[e]));
  }
}

namespace {

bool a16(const void* p) { return (reinterpret_cast<unsigned long long>(p) & 15) == 0; }
int padded_k(int K) { return K <= 64 ? 64 : 128; }
long slots_of(int n_seq, long rows, bool packed) {
  return packed ? rows / kC + n_seq : (long)n_seq * ((rows / n_seq + kC - 1) / kC);
}

// ws: offsets in floats (every array a multiple of 64 floats); returns the total.  Rows that the scans read in place
// (bf16, K = 64 or 128, 16-byte aligned) are not packed; the size leaves room for them where alignment may forbid it.
long carve(GdrArgs* a, float* ws, int dtype, int n_seq, long rows, bool packed, int Hk, int Hv, int K, int V, bool train) {
  const long ns = slots_of(n_seq, rows, packed), kp = padded_k(K), np = dtype == HHRL_BF16 ? 1 : 3, vp = (V + kVt - 1) / kVt * kVt;
  long off = 0;
  auto take = [&](long floats) { float* p = ws ? ws + off : nullptr; off += (floats + 63) & ~63L; return p; };
  auto take16 = [&](long n) { return reinterpret_cast<__bf16*>(take((n + 1) / 2)); };
  GdrArgs t = {};
  t.kpk = take16(ns * Hk * np * kC * kp);
  t.qpk = take16(ns * Hk * np * kC * kp);
  t.kt = take16(ns * Hk * np * kC * kp);
  t.m = take16(ns * Hv * 3 * kC * kC);
  t.p = take16(ns * Hv * 3 * kC * kC);
  t.vec = take(ns * Hv * kVecs * kC);
  if (train) {
    t.qt = take16(ns * Hk * np * kC * kp);
    t.mt = take16(ns * Hv * 3 * kC * kC);
    t.pt = take16(ns * Hv * 3 * kC * kC);
    t.w = take(ns * Hv * kC * vp);
    t.y = take(ns * Hv * kC * vp);
    t.s = take(ns * Hv * kp * vp);
    t.ds = take(ns * Hv * kp * vp);
  }
  if (a) {
    a->kpk = t.kpk; a->qpk = t.qpk; a->kt = t.kt; a->qt = t.qt; a->m = t.m; a->p = t.p; a->mt = t.mt; a->pt = t.pt;
    a->vec = t.vec; a->w = t.w; a->y = t.y; a->s = t.s; a->ds = t.ds;
    a->n_slots = ns; a->vp = (int)vp; a->nvt = (int)(vp / kVt);
  }
  return off;
}

int gdr_check(const hhrl_gdr_desc* d, const char* who) {
  HHRL_REQUIRE(d != nullptr, "%s: null descriptor", who);
  HHRL_REQUIRE(d->dtype == HHRL_F32 || d->dtype == HHRL_BF16, "%s: dtype %d", who, d->dtype);
  HHRL_REQUIRE(d->n_seq > 0 && d->rows > 0 && d->rows < (1L << 31) - kC, "%s: n_seq=%d rows=%ld", who, d->n_seq, d->rows);
  HHRL_REQUIRE(d->starts || d->rows % d->n_seq == 0, "%s: rows=%ld are not n_seq=%d sequences of one length", who, d->rows, d->n_seq);
  HHRL_REQUIRE(!d->starts || !d->lens, "%s: starts and lens", who);
  HHRL_REQUIRE(d->Hk > 0 && d->Hv > 0 && d->Hv % d->Hk == 0, "%s: Hk=%d Hv=%d", who, d->Hk, d->Hv);
  HHRL_REQUIRE(d->Hk <= 65535, "%s: Hk=%d", who, d->Hk);
  HHRL_REQUIRE(d->K > 0 && d->K <= HHRL_GDR_MAX_K && d->V > 0 && d->V <= HHRL_GDR_MAX_V, "%s: K=%d V=%d (up to %d, %d supported)", who,
               d->K, d->V, HHRL_GDR_MAX_K, HHRL_GDR_MAX_V);
  HHRL_REQUIRE(d->q && d->k && d->v && d->g && d->beta, "%s: null input", who);
  HHRL_REQUIRE(d->ldq >= (long)d->Hk * d->K && d->ldk >= (long)d->Hk * d->K && d->ldv >= (long)d->Hv * d->V && d->ldg >= d->Hv && d->ldbeta >= d->Hv,
               "%s: leading dimension of an input too small", who);
  const long ns = slots_of(d->n_seq, d->rows, d->starts != nullptr);
  HHRL_REQUIRE(ns < (1L << 31), "%s: %ld chunks", who, ns);
  const long blocks = ((long)d->n_seq * d->Hv + 7) / 8 * 8 * ((d->V + kVt - 1) / kVt);
  HHRL_REQUIRE(blocks < (1L << 31), "%s: n_seq*Hv too large", who);
  return HHRL_OK;
}

int gdr_fill(const hhrl_gdr_desc* d, GdrArgs& a, bool train, const char* who) {
  const long need = carve(nullptr, nullptr, d->dtype, d->n_seq, d->rows, d->starts != nullptr, d->Hk, d->Hv, d->K, d->V, train);
  HHRL_REQUIRE(d->ws && a16(d->ws) && d->ws_floats >= need, "%s: workspace of %ld floats (16-byte aligned), %ld needed", who, d->ws ? d->ws_floats : 0L, need);
  carve(&a, d->ws, d->dtype, d->n_seq, d->rows, d->starts != nullptr, d->Hk, d->Hv, d->K, d->V, train);
  a.n_seq = d->n_seq; a.Hk = d->Hk; a.Hv = d->Hv; a.K = d->K; a.V = d->V; a.rep = d->Hv / d->Hk;
  a.rows = d->rows;
  a.T = d->starts ? 0 : (int)(d->rows / d->n_seq);
  a.cpt = d->starts ? 1 : (a.T + kC - 1) / kC;
  a.scale = d->scale;
  a.starts = d->starts; a.lens = d->lens;
  a.q = d->q; a.k = d->k; a.v = d->v; a.ldq = d->ldq; a.ldk = d->ldk; a.ldv = d->ldv;
  a.g = d->g; a.beta = d->beta; a.ldg = d->ldg; a.ldbeta = d->ldbeta;
  a.train = train;
  a.pack = !(d->dtype == HHRL_BF16 && d->K == padded_k(d->K) && a16(d->q) && a16(d->k) && d->ldq % 8 == 0 && d->ldk % 8 == 0);
  return HHRL_OK;
}

template <typename T, int NP, int KB2>
int run_fwd(const GdrArgs& a, hipStream_t st, double flops) {
  constexpr int Kp = 64 * KB2;
  constexpr int over = 2 * NP * kC * (Kp + 8) * 2 > 2 * kC * kLdM * 4 ? 2 * NP * kC * (Kp + 8) * 2 : 2 * kC * kLdM * 4;
  constexpr int lds_prep = over + 2 * kC * kLdM * 4 + 3 * kC * 4;
  constexpr int lds_scan = ScanLds<NP, KB2>::bytes;
  const void* prep = reinterpret_cast<const void*>(&gdr_prep_kernel<T, NP, KB2>);
  const void* scan = reinterpret_cast<const void*>(&gdr_scan_fwd_kernel<T, NP, KB2>);
  HHRL_TRY(ensure_dyn_lds(prep, lds_prep, "gdr_forward"));
  HHRL_TRY(ensure_dyn_lds(scan, lds_scan, "gdr_forward"));
  {
    ProfScope ps("gdr_prep_kernel", st, 0.0, 0.0);
    hipLaunchKernelGGL((gdr_prep_kernel<T, NP, KB2>), dim3((unsigned)a.n_slots, a.Hk), dim3(256), lds_prep, st, a);
  }
  HHRL_TRY(launch_status("gdr_prep_kernel"));
  const unsigned grid = (unsigned)(((long)a.n_seq * a.Hv + 7) / 8 * 8 * a.nvt);
  ProfScope ps("gdr_scan_fwd_kernel", st, flops, 0.0);
  hipLaunchKernelGGL((gdr_scan_fwd_kernel<T, NP, KB2>), dim3(grid), dim3(256), lds_scan, st, a);
  return launch_status("gdr_scan_fwd_kernel");
}

template <typename T, int NP, int KB2, bool GROUP>
int run_grads(const GdrArgs& a, hipStream_t st, double flops) {
  constexpr int Kp = 64 * KB2, LDV = 40;
  constexpr int over = 2 * 3 * LDV * (2 * Kp + kC) > 2 * 2 * 3 * kC * kLdT ? 2 * 3 * LDV * (2 * Kp + kC) : 2 * 2 * 3 * kC * kLdT;
  constexpr int lds = over + (4 * kC + 4) * 4;
  HHRL_TRY(ensure_dyn_lds(reinterpret_cast<const void*>(&gdr_grads_kernel<T, NP, KB2, GROUP>), lds, "gdr_backward"));
  ProfScope ps("gdr_grads_kernel", st, flops, 0.0);
  hipLaunchKernelGGL((gdr_grads_kernel<T, NP, KB2, GROUP>), dim3((unsigned)a.n_slots, a.Hk), dim3(256), lds, st, a);
  return launch_status("gdr_grads_kernel");
}

template <typename T, int NP, int KB2>
int run_bwd(const GdrArgs& a, hipStream_t st, double flops) {
  constexpr int lds = ScanLds<NP, KB2>::bytes;
  HHRL_TRY(ensure_dyn_lds(reinterpret_cast<const void*>(&gdr_scan_bwd_kernel<T, NP, KB2>), lds, "gdr_backward"));
  const unsigned grid = (unsigned)(((long)a.n_seq * a.Hv + 7) / 8 * 8 * a.nvt);
  {
    ProfScope ps("gdr_scan_bwd_kernel", st, flops, 0.0);
    hipLaunchKernelGGL((gdr_scan_bwd_kernel<T, NP, KB2>), dim3(grid), dim3(256), lds, st, a);
  }
  HHRL_TRY(launch_status("gdr_scan_bwd_kernel"));
  return a.rep > 1 ? run_grads<T, NP, KB2, true>(a, st, flops) : run_grads<T, NP, KB2, false>(a, st, flops);
}

template <typename T, int VEC>
void launch_step(const GdrStepArgs& a, unsigned grid, hipStream_t st) {
  if (a.K <= 64) hipLaunchKernelGGL((gdr_step_kernel<T, VEC, 4>), dim3(grid), dim3(256), 0, st, a);
  else hipLaunchKernelGGL((gdr_step_kernel<T, VEC, 8>), dim3(grid), dim3(256), 0, st, a);
}

}  // namespace
}  // namespace hhrl

using namespace hhrl;

extern "C" {

long hhrl_gdr_workspace_floats(int dtype, int n_seq, long rows, int packed, int Hk, int Hv, int K, int V, int no_backward) {
  if ((dtype != HHRL_F32 && dtype != HHRL_BF16) || n_seq <= 0 || rows <= 0 || rows >= (1L << 31) || Hk <= 0 || Hv <= 0 || Hv % Hk ||
      K <= 0 || K > HHRL_GDR_MAX_K || V <= 0 || V > HHRL_GDR_MAX_V || (!packed && rows % n_seq))
    return 0;
  return carve(nullptr, nullptr, dtype, n_seq, rows, packed != 0, Hk, Hv, K, V, !no_backward);
}

int hhrl_gdr_forward(const hhrl_gdr_desc* d, void* stream) {
  HHRL_TRY(gdr_check(d, "gdr_forward"));
  HHRL_REQUIRE(d->o && d->ldo >= (long)d->Hv * d->V, "gdr_forward: o null or ldo=%ld too small", d->ldo);
  GdrArgs a = {};
  HHRL_TRY(gdr_fill(d, a, !d->no_backward, "gdr_forward"));
  a.o = d->o; a.ldo = d->ldo; a.s0 = d->s0; a.s1 = d->s1;
  const double flops = 6.0 * d->rows * d->Hv * d->K * d->V;
  hipStream_t st = as_stream(stream);
  if (d->dtype == HHRL_BF16) return d->K <= 64 ? run_fwd<__bf16, 1, 1>(a, st, flops) : run_fwd<__bf16, 1, 2>(a, st, flops);
  return d->K <= 64 ? run_fwd<float, 3, 1>(a, st, flops) : run_fwd<float, 3, 2>(a, st, flops);
}

int hhrl_gdr_backward(const hhrl_gdr_desc* d, void* stream) {
  HHRL_TRY(gdr_check(d, "gdr_backward"));
  HHRL_REQUIRE(d->d_o || d->d_s1, "gdr_backward: no output gradient");
  HHRL_REQUIRE(d->dq && d->dk && d->dv && d->dg && d->dbeta, "gdr_backward: null gradient");
  HHRL_REQUIRE((!d->d_o || d->lddo >= (long)d->Hv * d->V) && d->lddq >= (long)d->Hk * d->K && d->lddk >= (long)d->Hk * d->K && d->lddv >= (long)d->Hv * d->V &&
               d->lddg >= d->Hv && d->lddbeta >= d->Hv, "gdr_backward: leading dimension of a gradient too small");
  GdrArgs a = {};
  HHRL_TRY(gdr_fill(d, a, true, "gdr_backward"));
  a.d_o = d->d_o; a.lddo = d->lddo; a.d_s1 = d->d_s1; a.d_s0 = d->d_s0;
  a.dq = d->dq; a.dk = d->dk; a.dv = d->dv; a.lddq = d->lddq; a.lddk = d->lddk; a.lddv = d->lddv;
  a.dg = d->dg; a.dbeta = d->dbeta; a.lddg = d->lddg; a.lddbeta = d->lddbeta;
  const double flops = 6.0 * d->rows * d->Hv * d->K * d->V;
  hipStream_t st = as_stream(stream);
  if (d->dtype == HHRL_BF16) return d->K <= 64 ? run_bwd<__bf16, 1, 1>(a, st, flops) : run_bwd<__bf16, 1, 2>(a, st, flops);
  return d->K <= 64 ? run_bwd<float, 3, 1>(a, st, flops) : run_bwd<float, 3, 2>(a, st, flops);
}

int hhrl_gdr_step(int dtype, int B, int Hk, int Hv, int K, int V, float scale, const void* q, long ldq, const void* k, long ldk,
                  const void* v, long ldv, const float* g, long ldg, const float* beta, long ldbeta, void* o, long ldo,
                  const float* state_in, float* state_out, int n_slots, const int* slots, void* stream) {
  HHRL_REQUIRE(dtype == HHRL_F32 || dtype == HHRL_BF16, "gdr_step: dtype %d", dtype);
  HHRL_REQUIRE(B > 0 && n_slots > 0 && Hk > 0 && Hv > 0 && Hv % Hk == 0, "gdr_step: B=%d n_slots=%d Hk=%d Hv=%d", B, n_slots, Hk, Hv);
  HHRL_REQUIRE(slots || B <= n_slots, "gdr_step: %d rows for %d states", B, n_slots);
  HHRL_REQUIRE(K > 0 && K <= HHRL_GDR_MAX_K && V > 0 && V <= HHRL_GDR_MAX_V, "gdr_step: K=%d V=%d (up to %d, %d supported)", K, V, HHRL_GDR_MAX_K, HHRL_GDR_MAX_V);
  HHRL_REQUIRE(q && k && v && g && beta && o && state_in && state_out, "gdr_step: null pointer");
  HHRL_REQUIRE(ldq >= (long)Hk * K && ldk >= (long)Hk * K && ldv >= (long)Hv * V && ldo >= (long)Hv * V && ldg >= Hv && ldbeta >= Hv,
               "gdr_step: leading dimension too small");
  const bool vec = V % 4 == 0 && a16(state_in) && a16(state_out);
  GdrStepArgs a = {};
  a.Hk = Hk; a.Hv = Hv; a.K = K; a.V = V; a.rep = Hv / Hk; a.n_slots = n_slots; a.scale = scale;
  a.q = q; a.k = k; a.v = v; a.ldq = ldq; a.ldk = ldk; a.ldv = ldv; a.g = g; a.beta = beta; a.ldg = ldg; a.ldbeta = ldbeta;
  a.o = o; a.ldo = ldo; a.sin = state_in; a.sout = state_out; a.slots = slots;
  a.nvt = ceil_div(V, vec ? 64 : 16);
  const long grid = (long)B * Hv * a.nvt;
  HHRL_REQUIRE(grid < (1L << 31), "gdr_step: B*Hv*V too large");
  hipStream_t st = as_stream(stream);
  ProfScope ps("gdr_step_kernel", st, 6.0 * B * Hv * K * V, 8.0 * B * Hv * K * V);
  if (dtype == HHRL_BF16) {
    if (vec) launch_step<__bf16, 4>(a, (unsigned)grid, st);
    else launch_step<__bf16, 1>(a, (unsigned)grid, st);
  } else {
    if (vec) launch_step<float, 4>(a, (unsigned)grid, st);
    else launch_step<float, 1>(a, (unsigned)grid, st);
  }
  return launch_status("gdr_step_kernel");
}

}  // extern "C"
