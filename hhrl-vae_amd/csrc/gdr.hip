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
// follows walks the chunks of a sequence (gdr_scan_fwd_kernel); its workgroups hold 16 or 32 columns of one head's state in
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
// corrected state is a difference of numbers much larger than itself, its gradients more so, and so may o be; dg, dbeta
// and the states are fp32 results.  The decays' sums are kept as two floats from a sum in fp64, so that exp(G_i - G_j) is exact
// to fp32 however far G has run.
//
// What a whole training call moves: per chunk and head of K = V = 128, bf16, 0.9 MB, of which the caller's tensors are 0.13;
// 4 x 4096 tokens of 16 heads take 0.13 (prep) + 0.26 + 0.24 (scans) + 0.37 ms (gradients), 3.8 GB at 3.7 TB/s (a copy
// reaches 4.85), with the matrix pipes 6 to 24 % busy: neither is full.  Larger chunks would move fewer states, and pay
// for it in the triangles and in accuracy.
#include "common.h"
#include "mfma_tiles.h"
#include "split_bf16.h"

namespace hhrl {

using sb::bf16x4;
using sb::bf16x8;
using sb::f32x4;

constexpr int kC = 64;             // tokens per chunk
constexpr int kLdM = kC + 4;       // row stride of prep's fp32 images
constexpr float kGMin = -1e4f;     // log decays are clamped here: exp() of it is 0, and infinities would leave NaN differences

// Images in LDS that matrix fragments are read from: rows of P pieces of 16 bytes, without padding, the pieces of a row
// exchanged by its number.  A fragment read (lane: row l & 15, piece p + (l >> 4)) goes in four cycles of 16 lanes, rows
// 0-3, 12-15 of one piece with rows 4-11 of the next or the other way round, and the exchange gives these 16 different
// places in the 256 bytes of a cycle; so it does for the 8-byte stores of 16 rows.  Measured per wave: read 4.2 cycles,
// 8.0 from rows padded by 16 bytes; store 8 either way (16 with 32 bytes of padding, which read in 4.2 as well).
template <int P>
__device__ __forceinline__ int place(int row, int piece) {
  static_assert(P == 4 || P == 8 || P == 16, "pieces of a row");
  const int x = row >> 2 & 3;
  return row * P + (piece ^ (P == 16 ? row & 15 : P == 8 ? row >> 1 & 7 : (((x << 1) ^ x) & 2) | x >> 1));
}
// element i of a row of N bf16 (fp32: multiples of 4)
template <int N>
__device__ __forceinline__ int at16(int row, int i) { return place<N / 8>(row, i >> 3) * 8 + (i & 7); }
template <int N>
__device__ __forceinline__ int at32(int row, int i) { return place<N / 4>(row, i >> 2) * 4; }

// Images in the workspace that matrix fragments are read from lie as the fragments do: blocks of 16 rows by 32 columns, the
// 64 lanes' 16 bytes behind each other ([row block][column block][term][lane][8]).  A wave's request for one is 1 KB in a
// row and takes the address unit 16 cycles; from rows of 128 bytes and more (every four lanes four rows) it takes 64,
// and a scan's requests, a hundred per chunk and workgroup, were what bound it.
constexpr int kFrag = 512;         // elements of a block
// where element i .. of row lr (of 16) of a block begins
__device__ __forceinline__ int frag_at(int lr, int i) { return ((i >> 3 & 3) * 16 + lr) * 8 + (i & 7); }

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
  int whole, wide, wide_v, v16, train, vp, nvt, by_length;
  // what ws holds: a number of the shapes whose forward pass was the last one in it, 0 if that was for no backward pass.  A
  // backward pass that finds another number starts its sums from NaN: only the device knows.
  unsigned long long *mark, key;
  // ws behind it, all but vec, w, y, s, ds as operand blocks, per chunk and key head: k, q (rows: tokens) and their transposes (rows: K);
  //     per chunk and value head: M, P and their transposes, five rows of 64 floats, and
  //     for the backward pass W, Y [vp/32][64][32] and S, dS [vp/32][Kp/16][2][64 lanes][4], fp32
  __bf16 *kpk, *qpk, *kt, *qt, *m, *p, *mt, *pt;
  float *vec, *w, *y, *s, *ds;
  // segments of long sequences: segs of seg_chunks chunks each (1: the whole sequence), grid_segs of them in a launch; per
  // value head and segment M and its transpose (operand blocks, fp32), N [Kp][vp], and the state (gradient) it starts from [Kp][vp]
  int segs, seg_chunks, grid_segs;
  float *seg_m, *seg_mt, *seg_n, *seg_s;
};
enum { kGam = 0, kTail = 1, kBeta = 2, kGHi = 3, kGLo = 4, kVecs = 5 };

// exp(x + low), |low| <= 2^-24 |x|, to 2^-22 of itself however large x is: the exponential instruction (base two) takes the
// rounded product with log2 e, and what that, the constant and x leave out multiplies the result.
__device__ __forceinline__ float exp_of(float x, float low) {
  const float t = x * 1.44269502f;
  const float r = fmaf(x, 1.92596299e-8f, fmaf(x, 1.44269502f, -t));
  const float e = __builtin_amdgcn_exp2f(t);
  return fmaf(e, fmaf(r, 0.693147181f, low), e);
}
// exp((a + al) - (b + bl)) for a <= b <= 0, each sum of log decays as two floats.  What a - b leaves out is exact since
// |a| >= |b|, and the sum of both is split anew, so that only the difference matters.
__device__ __forceinline__ float decay(float a, float al, float b, float bl) {
  const float s = a - b, low = (al - bl) + ((a - s) - b), x = s + low;
  return exp_of(x, (s - x) + low);
}
__device__ __forceinline__ float decay(double x) {
  const float hi = (float)x;
  return exp_of(hi, (float)(x - (double)hi));
}

__device__ __forceinline__ long clampl(long v, long lo, long hi) { return v < lo ? lo : v > hi ? hi : v; }

// 0, or NaN for a backward pass without its forward
__device__ __forceinline__ float poison(const GdrArgs& a) { return *a.mark == a.key ? 0.f : __builtin_nanf(""); }

// rows [start, start + len) of sequence n (the same n in the whole wave) and the place of its first chunk.  Packed sequences of any lengths:
// floor(start/64) + n leaves every sequence at least ceil(len/64) places.
__device__ __forceinline__ void seq_range(const GdrArgs& a, int n, long& start, int& len, long& slot0) {
  if (a.starts) {
    start = clampl(__builtin_amdgcn_readfirstlane(a.starts[n]), 0, a.rows);
    len = (int)(clampl(__builtin_amdgcn_readfirstlane(a.starts[n + 1]), start, a.rows) - start);
    slot0 = start / kC + n;
  } else {
    start = (long)n * a.T;
    len = a.lens ? (int)clampl(__builtin_amdgcn_readfirstlane(a.lens[n]), 0, a.T) : a.T;
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

// Rows of the caller's tensors go through buffer descriptors: a base that moves from chunk to chunk in scalar registers, a
// lane's offset that never changes, and the size of what the sequence has left, behind which a load gives 0 and a store is
// dropped.  So rows behind the sequence need no test, no request has a condition (a conditional one would be waited for
// where its branch joins), and a chunk costs no address arithmetic on the vector unit.
typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
typedef unsigned u32x2 __attribute__((ext_vector_type(2)));
constexpr unsigned kNoColumn = 0x80000000u;      // an offset behind every size
__device__ __forceinline__ __amdgpu_buffer_rsrc_t rows_rsrc(const void* base, long offset, long bytes) {
  // (descriptor word 3: 32-bit data, no swizzle)
  return __builtin_amdgcn_make_buffer_rsrc(const_cast<char*>(static_cast<const char*>(base)) + offset, 0, (int)bytes, 0x00027000);
}
// ------------------------------------------------------------------------------------------------------------ prep
// One workgroup per chunk and key head: k k^T and q k^T once, then per value head of the key head the decays, the
// triangular inverse and P.  The inverse goes by blocks: 16 x 16 on the diagonal by substitution (a lane per column), then
// the blocks below them, 16 and 32 wide, as -M22 (L21 M11) on the fp32 matrix instruction.  P is written straight from the
// registers of a product: four elements of a row from k q^T, of a column (for the transpose) from q k^T.  The 32 x 32
// blocks beyond the diagonal are neither written nor read.
// Bound by what it writes where there are many chunks (4 x 4096 tokens, 16 heads, K 128, bf16, for training: 0.58 GB in
// 134 us), else by the latency of its steps (64 chunks in fp32: 17 us, of which the products of the last row of tiles, the
// decays and the substitution are 4 us each).  Three workgroups per CU fill the waits of each other.
template <int NP, int KB2>
struct PrepLds {
  static constexpr int Kp = 64 * KB2;
  static constexpr int kq = 2 * NP * kC * Kp * 2;             // bytes: k and q as terms
  static constexpr int img = (2 * kC + 32) * kLdM * 4;         // I + A, its inverse, a product of the solve: over them once they are used
  static constexpr int over = kq > img ? kq : img;
  static constexpr int bytes = over + 3 * kC * 4;
};
template <typename T, int NP, int KB2>
__global__ __launch_bounds__(256, NP == 1 ? 3 : 2) void gdr_prep_kernel(GdrArgs a) {
  using L = PrepLds<NP, KB2>;
  constexpr int Kp = L::Kp, KG = Kp / 8;
  extern __shared__ __align__(16) char smem[];
  __bf16* const kl = reinterpret_cast<__bf16*>(smem);          // [NP][64][Kp]
  __bf16* const ql = kl + NP * kC * Kp;
  float* const lm = reinterpret_cast<float*>(smem);            // [64][kLdM] I + A
  float* const mm = lm + kC * kLdM;                            // [64][kLdM] its inverse
  float* const tm = mm + kC * kLdM;                            // [32][kLdM]
  float* const gh = reinterpret_cast<float*>(smem + L::over);
  float* const gl = gh + kC;
  float* const be = gl + kC;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lr = lane & 15, lg = lane >> 4;
  const long slot = blockIdx.x;
  const int hk = blockIdx.y;
  if (slot == 0 && hk == 0 && tid == 0) *a.mark = a.train ? a.key : 0;
  long row0;
  int valid;
  slot_chunk(a, slot, row0, valid);
  if (valid == 0) return;
  const long hs = slot * a.Hk + hk;
  // every wave holds token `lane`; a head's g and beta are requested a head ahead
  const long grow = row0 + min(lane, valid - 1);
  float gn = a.g[grow * a.ldg + hk * a.rep], bn = a.beta[grow * a.ldbeta + hk * a.rep];

  // k and q as bf16 terms; what lies beyond the sequence or the head's width becomes 0 and is not read
  if (NP == 1 && a.whole) {                                    // rows of Kp elements, 16-byte aligned
    constexpr int U = kC * KG / 256;
    bf16x8 x[2][U];
#pragma unroll
    for (int side = 0; side < 2; ++side) {
      const long ld = side ? a.ldq : a.ldk;
      const __amdgpu_buffer_rsrc_t r = rows_rsrc(side ? a.q : a.k, (row0 * ld + (long)hk * Kp) * 2, ((valid - 1) * ld + Kp) * 2);
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int g = u * 256 + tid, i = g / KG, c = (g - i * KG) * 8;
        x[side][u] = __builtin_bit_cast(bf16x8, __builtin_amdgcn_raw_buffer_load_b128(r, (i * (unsigned)ld + c) * 2, 0, 0));
      }
    }
#pragma unroll
    for (int side = 0; side < 2; ++side)
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int g = u * 256 + tid, i = g / KG, c = (g - i * KG) * 8;
        *reinterpret_cast<bf16x8*>((side ? ql : kl) + at16<Kp>(i, c)) = x[side][u];
      }
  } else {
    constexpr int U = kC * KG / 256;
    const T* src[2] = {static_cast<const T*>(a.k) + row0 * a.ldk + (long)hk * a.K, static_cast<const T*>(a.q) + row0 * a.ldq + (long)hk * a.K};
    auto convert = [&](int side, int u, const T (&raw)[8]) {
      const int i = (u * 256 + tid) / KG, c = (u * 256 + tid - i * KG) * 8;
      float x[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) x[e] = i < valid && c + e < a.K ? (float)raw[e] : 0.f;
      bf16x8 t[NP];
      sb::split8<NP>(x, t);
#pragma unroll
      for (int p = 0; p < NP; ++p) *reinterpret_cast<bf16x8*>((side ? ql : kl) + p * kC * Kp + at16<Kp>(i, c)) = t[p];
    };
    // (requests of elements that are there, all at once where they come in pieces of 16 bytes, then a choice)
    if (a.wide) {                                              // K % 8 == 0, 16-byte aligned rows
      u32x4 y[2][U][sizeof(T) / 2];
#pragma unroll
      for (int side = 0; side < 2; ++side)
#pragma unroll
        for (int u = 0; u < U; ++u) {
          const int i = (u * 256 + tid) / KG, c = (u * 256 + tid - i * KG) * 8;
          const u32x4* const q = reinterpret_cast<const u32x4*>(src[side] + min(i, valid - 1) * (side ? a.ldq : a.ldk) + min(c, a.K - 8));
#pragma unroll
          for (int h = 0; h < (int)sizeof(T) / 2; ++h) y[side][u][h] = q[h];
        }
#pragma unroll
      for (int side = 0; side < 2; ++side)
#pragma unroll
        for (int u = 0; u < U; ++u) {
          T raw[8];
          __builtin_memcpy(raw, y[side][u], sizeof(raw));
          convert(side, u, raw);
        }
    } else {
      for (int side = 0; side < 2; ++side)
        for (int u = 0; u < U; ++u) {
          const int i = (u * 256 + tid) / KG, c = (u * 256 + tid - i * KG) * 8;
          const T* const q = src[side] + min(i, valid - 1) * (side ? a.ldq : a.ldk);
          T raw[8];
#pragma unroll
          for (int e = 0; e < 8; ++e) raw[e] = q[min(c + e, a.K - 1)];
          convert(side, u, raw);
        }
    }
  }
  lds_barrier();
  // the transposes: two columns of eight tokens per thread
  for (int side = 0; side < (a.train ? 2 : 1); ++side) {
    const __bf16* const src = side ? ql : kl;
    __bf16* const dst = (side ? a.qt : a.kt) + hs * NP * Kp * kC;
#pragma unroll
    for (int v = 0; v < NP * Kp / 64; ++v) {
      const int u = v * 256 + tid, k = u % (Kp / 2) * 2, r = u / (Kp / 2), i0 = (r & 7) * 8, p = r >> 3;
      unsigned x[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) x[e] = *reinterpret_cast<const unsigned*>(src + p * kC * Kp + at16<Kp>(i0 + e, k));
      u32x4 lo, hi;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        lo[e] = __builtin_amdgcn_perm(x[2 * e + 1], x[2 * e], 0x05040100u);       // low halves of two tokens
        hi[e] = __builtin_amdgcn_perm(x[2 * e + 1], x[2 * e], 0x07060302u);       // high halves
      }
      __bf16* const to = dst + ((k >> 4) * 2 + (i0 >> 5)) * NP * kFrag + p * kFrag + frag_at(k & 15, i0);
      *reinterpret_cast<u32x4*>(to) = lo;
      *reinterpret_cast<u32x4*>(to + 8) = hi;
    }
  }
  // rows 16*wave.. against the tiles of columns in front of them: k k^T, q k^T (its transpose's source), and k q^T with the
  // roles changed: rows of the wave's tile are the columns j of P
  f32x4 kk[4], qk[4], kq[4];
#pragma unroll
  for (int t = 0; t < 4; ++t) kk[t] = qk[t] = kq[t] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int kb = 0; kb < Kp / 32; ++kb) {
    bf16x8 ka[NP], qa[NP];
    const int off = at16<Kp>(lr, 32 * kb + 8 * lg);
    sb::load_frag<NP>(ka, kl + 16 * wave * Kp + off, kC * Kp);
    sb::load_frag<NP>(qa, ql + 16 * wave * Kp + off, kC * Kp);
    const long at = hs * kC * NP * Kp + ((wave * (Kp / 32) + kb) * NP) * kFrag + lane * 8;
#pragma unroll
    for (int p = 0; p < NP; ++p) {
      *reinterpret_cast<bf16x8*>(a.kpk + at + p * kFrag) = ka[p];
      *reinterpret_cast<bf16x8*>(a.qpk + at + p * kFrag) = qa[p];
    }
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      if (t <= wave) {
        bf16x8 b[NP];
        sb::load_frag<NP>(b, kl + 16 * t * Kp + off, kC * Kp);
        sb::mma<NP, NP>(kk[t], ka, b);
        if (a.train) sb::mma<NP, NP>(qk[t], qa, b);
        sb::mma<NP, NP>(kq[t], b, qa);                         // row 16*t + ..: k's token j, column 16*wave + lr: q's token i
      }
    }
  }
  for (int r = 0; r < a.rep; ++r) {
    const int hv = hk * a.rep + r;
    const long vs = slot * a.Hv + hv;
    // running sum of the log decays in fp64, kept as two floats
    float gi = gn, bi = bn;
    gi = lane < valid ? gi < kGMin ? kGMin : gi : 0.f;
    bi = lane < valid ? bi : 0.f;
    double G = gi;
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) {
      const double up = __shfl_up(G, off, 64);
      if (lane >= off) G += up;
    }
    const float hi = (float)G, lo = (float)(G - (double)hi);
    lds_barrier();                                 // kl and ql have been read, the previous head's images too
    if (wave == 0) { gh[lane] = hi; gl[lane] = lo; be[lane] = bi; }
    lds_barrier();
    const int hn = hk * a.rep + min(r + 1, a.rep - 1);
    gn = a.g[grow * a.ldg + hn];
    bn = a.beta[grow * a.ldbeta + hn];
    if (wave == 0) {
      const double end = __shfl(G, 63, 64);
      float* const v = a.vec + vs * kVecs * kC + lane;
      v[kGam * kC] = decay(G);
      v[kTail * kC] = decay(end - G);
      v[kBeta * kC] = bi;
      v[kGHi * kC] = hi;
      v[kGLo * kC] = lo;
    }
    const int ib = 16 * wave + 4 * lg, iq = 16 * wave + lr;
    __bf16* const pp = a.p + vs * kC * 3 * kC;
    __bf16* const pt = a.pt + vs * kC * 3 * kC;
    const f32x4 gi4 = *reinterpret_cast<const f32x4*>(gh + ib), li4 = *reinterpret_cast<const f32x4*>(gl + ib), bi4 = *reinterpret_cast<const f32x4*>(be + ib);
    const float gq = gh[iq], lq = gl[iq];
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      const int j = 16 * t + lr, jb = 16 * t + 4 * lg;
      const bool same = t < 2 || wave >= 2;                  // PT rows j >= 32 hold columns i >= 32, P rows i < 32 columns j < 32
      __bf16* const to_p = pp + (wave * 2 + (t >> 1)) * 3 * kFrag + frag_at(lr, jb);
      __bf16* const to_pt = pt + (t * 2 + (wave >> 1)) * 3 * kFrag + frag_at(lr, ib);
      f32x4 x = {0.f, 0.f, 0.f, 0.f};
      if (t <= wave) {
        const float hj = gh[j], lj = gl[j];
        const f32x4 gj4 = *reinterpret_cast<const f32x4*>(gh + jb), lj4 = *reinterpret_cast<const f32x4*>(gl + jb);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int i = ib + e;
          const float d = i >= j ? decay(gi4[e], li4[e], hj, lj) : 0.f;
          lm[i * kLdM + j] = i > j ? bi4[e] * kk[t][e] * d : i == j ? 1.f : 0.f;
          mm[i * kLdM + j] = 0.f;
          x[e] = i >= j ? qk[t][e] * d : 0.f;
        }
        if (a.train && same) sb::split_store4<3>(to_pt, kFrag, x);
#pragma unroll
        for (int e = 0; e < 4; ++e) x[e] = iq >= jb + e ? kq[t][e] * decay(gq, lq, gj4[e], lj4[e]) : 0.f;
        if (same) sb::split_store4<3>(to_p, kFrag, x);
      } else {                                               // above the diagonal: nothing reads it of I + A
#pragma unroll
        for (int e = 0; e < 4; ++e) mm[(ib + e) * kLdM + j] = 0.f;
        if (t >> 1 == wave >> 1) {
          if (a.train) sb::split_store4<3>(to_pt, kFrag, x);
          sb::split_store4<3>(to_p, kFrag, x);
        }
      }
    }
    lds_barrier();
    {
      // diagonal block `wave`: column lr of the inverse by substitution
      const float* const D = lm + 16 * wave * kLdM + 16 * wave;
      float x[16];
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        // (rows of L requested one by one: all at once would not fit the registers)
        if (i > 0) asm volatile("" : "+v"(x[i - 1])::"memory");
        f32x4 row[4];
#pragma unroll
        for (int q = 0; q < 4; ++q)
          if (4 * q < i) row[q] = *reinterpret_cast<const f32x4*>(D + i * kLdM + 4 * q);
        float s0 = i == lr ? 1.f : 0.f, s1 = 0.f;
#pragma unroll
        for (int j = 0; j < i; ++j) {
          if (j & 1) s1 = fmaf(-row[j >> 2][j & 3], x[j], s1);
          else s0 = fmaf(-row[j >> 2][j & 3], x[j], s0);
        }
        x[i] = s0 + s1;
      }
      if (lg == 0) {
#pragma unroll
        for (int i = 0; i < 16; ++i) mm[(16 * wave + i) * kLdM + 16 * wave + lr] = x[i];
      }
    }
    lds_barrier();
    const mt::f32x4 zero = {0.f, 0.f, 0.f, 0.f};
    if (wave < 2) {
      // 16 x 16 below the diagonal of the two 32 x 32 blocks
      const int o1 = 32 * wave, o2 = o1 + 16;
      mt::f32x4 c = mt::wave_mma16<16, kLdM, 1, kLdM, 1>(lm + o2 * kLdM + o1, mm + o1 * kLdM + o1, lane, zero);
      mt::store_block16<kLdM>(tm, 16 * wave, 0, c, lane);
      mt::wave_sync();
      c = mt::wave_mma16<16, kLdM, 1, kLdM, 1>(mm + o2 * kLdM + o2, tm + 16 * wave * kLdM, lane, zero);
      mt::store_block16<kLdM>(mm, o2, o1, -c, lane);
    }
    lds_barrier();
    {
      const int ti = 16 * (wave >> 1), tj = 16 * (wave & 1);
      mt::f32x4 c = mt::wave_mma16<32, kLdM, 1, kLdM, 1>(lm + (32 + ti) * kLdM, mm + tj, lane, zero);
      mt::store_block16<kLdM>(tm, ti, tj, c, lane);
      lds_barrier();
      c = mt::wave_mma16<32, kLdM, 1, kLdM, 1>(mm + (32 + ti) * kLdM + 32, tm + tj, lane, zero);
      mt::store_block16<kLdM>(mm, 32 + ti, tj, -c, lane);
    }
    lds_barrier();
    // 16 elements of a row (or of a column, for the transpose the backward scan reads) per thread
    const int row = 16 * wave + lr, c0 = lg * 16;
    for (int what = 0; what < (a.train ? 2 : 1); ++what) {
      if (what == 0 ? row < 32 && c0 >= 32 : row >= 32 && c0 < 32) continue;
      __bf16* const dst = (what == 0 ? a.m : a.mt) + vs * kC * 3 * kC + (wave * 2 + (lg >> 1)) * 3 * kFrag;
      const int si = what == 0 ? kLdM : 1, sj = what == 0 ? 1 : kLdM;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        float x[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = mm[row * si + (c0 + 8 * h + e) * sj];
        bf16x8 t[3];
        sb::split8<3>(x, t);
#pragma unroll
        for (int p = 0; p < 3; ++p) *reinterpret_cast<bf16x8*>(dst + p * kFrag + frag_at(lr, c0 + 8 * h)) = t[p];
      }
    }
  }
}

// --------------------------------------------------------------------------------------------------------- scans
// the r-th longest of up to 64 sequences (a lane each; equal ones in their order)
__device__ __forceinline__ int longest(const GdrArgs& a, int r) {
  const int lane = threadIdx.x & 63, n = min(lane, a.n_seq - 1);
  int len;
  if (a.starts) {
    const long start = clampl(a.starts[n], 0, a.rows);
    len = (int)(clampl(a.starts[n + 1], start, a.rows) - start);
  } else {
    len = (int)clampl(a.lens[n], 0, a.T);
  }
  int rank = 0;
  for (int j = 0; j < a.n_seq; ++j) {
    const int other = __builtin_amdgcn_readlane(len, j);
    rank += other > len || (other == len && j < lane);
  }
  return __ffsll((unsigned long long)__ballot(lane < a.n_seq && rank == r)) - 1;
}
// Workgroup -> (sequence, value head, segment, column tile).  Sequences of different lengths go from the longest (by_length),
// so that the last workgroups are short ones: 13 sequences of 12345 tokens, 16 heads 182 -> 151 us.  Workgroups go to the
// eight XCDs in turn: the column tiles of one head read the same k, q, M and P, so they are dealt to one XCD (one L2),
// eight workgroups apart.
__device__ __forceinline__ bool scan_tile(const GdrArgs& a, int vt, int& n, int& hv, int& v0, int& seg) {
  const int xcd = blockIdx.x & 7, u = blockIdx.x >> 3;
  v0 = (u % a.nvt) * vt;
  const long unit = (long)(u / a.nvt) * 8 + xcd;
  if (unit >= (long)a.n_seq * a.Hv * a.grid_segs) return false;
  const long pair = unit / a.grid_segs;
  seg = __builtin_amdgcn_readfirstlane((int)(unit - pair * a.grid_segs));
  n = __builtin_amdgcn_readfirstlane((int)(pair / a.Hv));
  hv = __builtin_amdgcn_readfirstlane((int)(pair - (long)n * a.Hv));
  if (a.by_length) n = longest(a, n);
  return true;
}

// LDS of a scan, in bytes: images of bf16 terms run along K (S) or along the tokens (X), fp32 images along the tokens (F);
// a row per state column
template <int NP, int KB2, int NT>
struct ScanLds {
  static constexpr int Kp = 64 * KB2, VT = 16 * NT;
  static constexpr int S = 3 * VT * Kp, X = 3 * VT * kC, F = VT * kC;     // elements
  static constexpr int V = VT * kC * (NP == 1 ? 2 : 4);                            // bytes: rows of v or dO, turned
  static constexpr int chain_bytes = 2 * (S + 2 * X) + V, fwd_bytes = chain_bytes + V + 12 * F;
  static constexpr int bwd_bytes = 2 * (S + 3 * X + NP * VT * kC) + 12 * F + V;
};

// Operand rows of k or q, token 16*w + lr of a chunk
template <int NP, int KB>
__device__ __forceinline__ void load_rows(bf16x8 (&f)[KB][NP], const __bf16* base, unsigned at) {
#pragma unroll
  for (int kb = 0; kb < KB; ++kb)
#pragma unroll
    for (int p = 0; p < NP; ++p) f[kb][p] = *reinterpret_cast<const bf16x8*>(base + (at + (kb * NP + p) * kFrag));
}
// Rows of v, dO, o or dv: lane l holds token 16*w + l/4, columns v0 + 4*NT*(l & 3) + e, so that four lanes read or write
// neighbours (WIDE: in 16-byte pieces, where V is a multiple of those and rows are aligned to them).
template <typename T, int NT, bool WIDE>
struct RowTile {
  static constexpr int N = 4 * NT, R = N * (int)sizeof(T) / 4;
  const char* base;
  long row, width;
  int len, have;                               // have: columns from the lane's first to the end of the head
  unsigned at, x[WIDE ? R : N];
  __device__ __forceinline__ RowTile(const void* src, long ld, long start, int len_, int hv, int V, int v0, int w, int lane)
      : len(len_), have(V - v0 - N * (lane & 3)) {
    base = static_cast<const char*>(src) + (start * ld + (long)hv * V) * sizeof(T);
    row = ld * sizeof(T);
    width = (long)V * sizeof(T);
    at = (16 * w + (lane >> 2)) * (unsigned)row + (v0 + N * (lane & 3)) * (unsigned)sizeof(T);
  }
  __device__ __forceinline__ __amdgpu_buffer_rsrc_t chunk(int c) const {
    return rows_rsrc(base, (long)c * kC * row, (min(kC, len - c * kC) - 1) * row + width);
  }
  __device__ __forceinline__ unsigned place_of(int e) const { return e < have ? at + e * (unsigned)sizeof(T) : kNoColumn; }
  __device__ __forceinline__ void load(int c) {
    const __amdgpu_buffer_rsrc_t r = chunk(c);
    if constexpr (WIDE && R == 2) {
      const u32x2 y = __builtin_amdgcn_raw_buffer_load_b64(r, place_of(0), 0, 0);
      x[0] = y[0]; x[1] = y[1];
    } else if constexpr (WIDE) {
#pragma unroll
      for (int h = 0; h < R; h += 4) {
        const u32x4 y = __builtin_amdgcn_raw_buffer_load_b128(r, place_of(h * 4 / (int)sizeof(T)), 0, 0);
#pragma unroll
        for (int e = 0; e < 4; ++e) x[h + e] = y[e];
      }
    } else {
#pragma unroll
      for (int e = 0; e < N; ++e) {
        if constexpr (sizeof(T) == 2) x[e] = __builtin_amdgcn_raw_buffer_load_b16(r, place_of(e), 0, 0);
        else x[e] = __builtin_amdgcn_raw_buffer_load_b32(r, place_of(e), 0, 0);
      }
    }
  }
  // what was loaded into an image in LDS, columns by tokens
  __device__ __forceinline__ void put(T* img, int w, int lane) const {
    const int i = 16 * w + (lane >> 2);
#pragma unroll
    for (int e = 0; e < N; ++e) {
      const int col = N * (lane & 3) + e;
      if constexpr (sizeof(T) == 2) {
        const unsigned y = WIDE ? e & 1 ? x[e >> 1] >> 16 : x[e >> 1] : x[e];
        reinterpret_cast<unsigned short*>(img)[at16<kC>(col, i)] = (unsigned short)y;
      } else {
        reinterpret_cast<unsigned*>(img)[at32<kC>(col, i) + (i & 3)] = x[e];
      }
    }
  }
  __device__ __forceinline__ void store(int c, const float (&y)[N]) const {
    const __amdgpu_buffer_rsrc_t r = chunk(c);
    if constexpr (WIDE && R == 2) {
      __builtin_amdgcn_raw_buffer_store_b64(u32x2{sb::pack2(y[0], y[1]), sb::pack2(y[2], y[3])}, r, place_of(0), 0, 0);
    } else if constexpr (WIDE) {
#pragma unroll
      for (int h = 0; h < R; h += 4) {
        u32x4 z;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          if constexpr (sizeof(T) == 2) z[e] = sb::pack2(y[2 * e], y[2 * e + 1]);
          else z[e] = __float_as_uint(y[h + e]);
        }
        __builtin_amdgcn_raw_buffer_store_b128(z, r, place_of(h * 4 / (int)sizeof(T)), 0, 0);
      }
    } else {
#pragma unroll
      for (int e = 0; e < N; ++e) {
        if constexpr (sizeof(T) == 2) __builtin_amdgcn_raw_buffer_store_b16(__builtin_bit_cast(unsigned short, (__bf16)y[e]), r, place_of(e), 0, 0);
        else __builtin_amdgcn_raw_buffer_store_b32(__float_as_uint(y[e]), r, place_of(e), 0, 0);
      }
    }
  }
};
// four tokens (i ..) of a column from such an image
template <typename T>
using Four = T __attribute__((ext_vector_type(4)));
template <typename T>
__device__ __forceinline__ Four<T> column4(const T* img, int col, int i) {
  return *reinterpret_cast<const Four<T>*>(img + (sizeof(T) == 2 ? at16<kC>(col, i) : at32<kC>(col, i)));
}
__device__ __forceinline__ f32x4 wide4(const f32x4& x) { return x; }
__device__ __forceinline__ f32x4 wide4(const bf16x4& x) { return f32x4{(float)x[0], (float)x[1], (float)x[2], (float)x[3]}; }
// N columns of token i from an fp32 image of columns by tokens, and into rows of 32 floats
template <int N>
__device__ __forceinline__ void token_row(float (&y)[N], const float* img, int i, int col) {
#pragma unroll
  for (int e = 0; e < N; ++e) y[e] = img[at32<kC>(col + e, i) + (i & 3)];
}
template <int N>
__device__ __forceinline__ void store_row(float* to, const float (&y)[N]) {
#pragma unroll
  for (int h = 0; h < N; h += 4) *reinterpret_cast<f32x4*>(to + h) = f32x4{y[h], y[h + 1], y[h + 2], y[h + 3]};
}
template <int NP, int KB2>
__device__ __forceinline__ void load_kt(bf16x8 (&f)[KB2][2][NP], const __bf16* base, unsigned at) {
#pragma unroll
  for (int t = 0; t < KB2; ++t)
#pragma unroll
    for (int kb = 0; kb < 2; ++kb)
#pragma unroll
      for (int p = 0; p < NP; ++p) f[t][kb][p] = *reinterpret_cast<const bf16x8*>(base + (at + ((t * 2 + kb) * NP + p) * kFrag));
}
// the state tile of a scan's chain wave w: rows 16*(KB2*w + t) + 4*lg + e, columns v0 + 16*u + lr
template <int KB2, int NT>
__device__ __forceinline__ void load_state(f32x4 (&S)[KB2][NT], const float* s, const GdrArgs& a, long nh, int w, int v0, int lr, int lg) {
#pragma unroll
  for (int t = 0; t < KB2; ++t)
#pragma unroll
    for (int u = 0; u < NT; ++u)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int k = 16 * (KB2 * w + t) + 4 * lg + e, v = v0 + 16 * u + lr;
        S[t][u][e] = s && k < a.K && v < a.V ? s[(nh * a.K + k) * a.V + v] : 0.f;
      }
}
template <int KB2, int NT>
__device__ __forceinline__ void store_state(const f32x4 (&S)[KB2][NT], float* s, const GdrArgs& a, long nh, int w, int v0, int lr, int lg) {
#pragma unroll
  for (int t = 0; t < KB2; ++t)
#pragma unroll
    for (int u = 0; u < NT; ++u)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int k = 16 * (KB2 * w + t) + 4 * lg + e, v = v0 + 16 * u + lr;
        if (k < a.K && v < a.V) s[(nh * a.K + k) * a.V + v] = S[t][u][e];
      }
}

// the same tile of a state of a segment, [Kp][ld] without bounds to keep
template <int KB2, int NT>
__device__ __forceinline__ void load_seg(f32x4 (&S)[KB2][NT], const float* s, int ld, int w, int v0, int lr, int lg) {
#pragma unroll
  for (int t = 0; t < KB2; ++t)
#pragma unroll
    for (int u = 0; u < NT; ++u)
#pragma unroll
      for (int e = 0; e < 4; ++e) S[t][u][e] = s[(16 * (KB2 * w + t) + 4 * lg + e) * ld + v0 + 16 * u + lr];
}
template <int KB2, int NT>
__device__ __forceinline__ void store_seg(const f32x4 (&S)[KB2][NT], float* s, int ld, int w, int v0, int lr, int lg) {
#pragma unroll
  for (int t = 0; t < KB2; ++t)
#pragma unroll
    for (int u = 0; u < NT; ++u)
#pragma unroll
      for (int e = 0; e < 4; ++e) s[(16 * (KB2 * w + t) + 4 * lg + e) * ld + v0 + 16 * u + lr] = S[t][u][e];
}

// the tile for the gradients, as the registers hold it: [K/16][2 halves of 32 columns][64 lanes][4]
template <int KB2, int NT>
__device__ __forceinline__ void store_tile(const f32x4 (&S)[KB2][NT], float* s, int w, int lane) {
#pragma unroll
  for (int t = 0; t < KB2; ++t)
#pragma unroll
    for (int u = 0; u < NT; ++u) *reinterpret_cast<f32x4*>(s + ((unsigned)(KB2 * w * 512 + lane * 4) + t * 512 + u * 256)) = S[t][u];
}

// Per-token factors of a chunk, rows ib .. ib + 3
struct ScanVec {
  f32x4 gam, tail, beta;
  float last;
  __device__ __forceinline__ void load(const float* vec, int ib) {
    gam = *reinterpret_cast<const f32x4*>(vec + kGam * kC + ib);
    tail = *reinterpret_cast<const f32x4*>(vec + kTail * kC + ib);
    beta = *reinterpret_cast<const f32x4*>(vec + kBeta * kC + ib);
    last = vec[kGam * kC + kC - 1];
  }
};
// the two 32-wide halves of a row of M, P or a transpose.  Half `f` of a wave whose rows do not reach it reads the other
// one again (from the first-level cache): a request under a condition would be waited for at once.
template <int N>
__device__ __forceinline__ void load_half(bf16x8 (&f)[N], const __bf16* base, unsigned at) {
#pragma unroll
  for (int q = 0; q < N; ++q) f[q] = *reinterpret_cast<const bf16x8*>(base + (at + q * kFrag));
}
template <int N>
__device__ __forceinline__ void load_tri(bf16x8 (&f)[2][N], const __bf16* base, unsigned at, bool low, bool high) {
  load_half<N>(f[0], base, at + (low ? 0 : N * kFrag));
  load_half<N>(f[1], base, at + (high ? N * kFrag : 0));
}

// Requests are counted in their order, so those in front of a loop are made in the order of the loop's: in another one the
// compiler's first wait of every pass would be for what has just been requested.
#define GDR_IN_ORDER __builtin_amdgcn_sched_barrier(0)

// A scan is a chain: state -> K S -> W -> state, chunk after chunk.  Four waves of the workgroup do nothing but the chain,
// and four others what hangs on it: v in front of it and the output o one chunk behind (forward), or what only depends on
// dO, one chunk ahead, and the stores of Y and dV (backward).  Everything a chunk needs from memory is requested while the
// chunk in front of it is worked on, behind the last use of its registers.
// Measured with K = V = 128, bf16: alone 1.4 us per chunk with 16 columns and 2.2 with 32, 2.6 with 32 and the chip full;
// splitting the state and the two right-hand sides into terms, three barriers and the matrix products share it about
// evenly.  Training adds the stores of S and W: 64 chunks of 64 heads take 261 us forward, 0.47 GB written, 240 backward.  Two workgroups
// per CU (128 registers) were slower for all sizes (167 -> 179 us, 256 -> 366 for training): the registers do not hold it.
// The chain: chunks c0 .. c1 - 1 of a sequence, four waves, S in their registers.  BARE: nobody hangs on it (no W is left in
// wl, and v comes into vl by these waves).  vcols: V, or 0 for columns without a v (and v0 what it may).
template <typename T, int NP, int KB2, int NT, bool TRAIN, bool BARE, bool WIDE>
__device__ __forceinline__ void scan_chain(const GdrArgs& a, f32x4 (&S)[KB2][NT], __bf16* sl, __bf16* xl, __bf16* ul, T* vl, float* wl, int hv, int vcols,
                                           int v0, long start, int len, long slot0, int c0, int c1) {
  using L = ScanLds<NP, KB2, NT>;
  constexpr int Kp = L::Kp, KB = Kp / 32, VT = L::VT;
  const int hk = hv / a.rep, lane = threadIdx.x & 63, w = threadIdx.x >> 6, lr = lane & 15, lg = lane >> 4;
  const int ib = 16 * w + 4 * lg;                          // first of four result rows
  const bool high = w >= 2;                                // M is lower triangular: rows < 32 read 32 columns
  const f32x4 zero = {0.f, 0.f, 0.f, 0.f};
  bf16x8 kf[KB][NP], mf[2][3], ktf[KB2][2][NP];
  const __bf16* kp = a.kpk + ((slot0 + c0) * a.Hk + hk) * kC * NP * Kp;
  RowTile<T, NT, WIDE> vp(a.v, a.ldv, start, len, hv, vcols, v0, w, lane);
  ScanVec vn;
  const float* vecp = a.vec + ((slot0 + c0) * a.Hv + hv) * kVecs * kC;
  const __bf16* mp = a.m + ((slot0 + c0) * a.Hv + hv) * 3 * kC * kC;
  const __bf16* ktp = a.kt + ((slot0 + c0) * a.Hk + hk) * Kp * NP * kC;
  const unsigned kat = w * KB * NP * kFrag + lane * 8, mat = w * 2 * 3 * kFrag + lane * 8, ktat = KB2 * w * 2 * NP * kFrag + lane * 8;
  if constexpr (BARE) vp.load(c0);
  GDR_IN_ORDER;
  load_rows<NP, KB>(kf, kp, kat);
  GDR_IN_ORDER;
  vn.load(vecp, ib);
  GDR_IN_ORDER;
  load_tri<3>(mf, mp, mat, true, high);
  GDR_IN_ORDER;
  load_kt<NP, KB2>(ktf, ktp, ktat);
  GDR_IN_ORDER;
  if constexpr (BARE) {
    vp.put(vl, w, lane);
    vp.load(min(c0 + 1, c1 - 1));
  }
  for (int c = c0; c < c1; ++c) {
    const int next = min(c + 1, c1 - 1);
    const long adv = next - c;                         // 0 behind the last chunk: its operands are read again, to no use
    vecp += adv * a.Hv * kVecs * kC;
    mp += adv * a.Hv * 3 * kC * kC;
    ktp += adv * a.Hk * NP * Kp * kC;
    kp += adv * a.Hk * NP * Kp * kC;
    const long vs = (slot0 + c) * a.Hv + hv;
#pragma unroll
    for (int t = 0; t < KB2; ++t)
#pragma unroll
      for (int u = 0; u < NT; ++u)
        sb::split_store4<3>(sl + 16 * u * Kp + at16<Kp>(lr, 16 * (KB2 * w + t) + 4 * lg), VT * Kp, S[t][u]);
    lds_barrier();
    const ScanVec vc = vn;
    f32x4 ks[NT];
    Four<T> vv[NT];
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      ks[t] = zero;
      vv[t] = column4<T>(vl + ((BARE ? 0 : (c & 1) * L::VT) + 16 * t) * kC, lr, ib);
    }
#pragma unroll
    for (int kb = 0; kb < KB; ++kb)
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        bf16x8 b[3];
        sb::load_frag<3>(b, sl + 16 * t * Kp + at16<Kp>(lr, 32 * kb + 8 * lg), VT * Kp);
        sb::mma<NP, 3>(ks[t], kf[kb], b);
      }
    load_rows<NP, KB>(kf, kp, kat);
    vn.load(vecp, ib);
#pragma unroll
    for (int t = 0; t < NT; ++t)
      sb::split_store4<3>(xl + 16 * t * kC + at16<kC>(lr, ib), VT * kC, vc.beta * (wide4(vv[t]) - vc.gam * ks[t]));
    if constexpr (BARE) {                                  // (a wave's tokens are read by nobody else)
      vp.put(vl, w, lane);
      vp.load(min(c + 2, c1 - 1));
    }
    if constexpr (TRAIN) {
      store_tile<KB2, NT>(S, a.s + ((vs * (a.vp / 32) + v0 / 32) * Kp) * 32 + (v0 & 16) * 16, w, lane);
    }
    lds_barrier();
    f32x4 wt[NT];
#pragma unroll
    for (int t = 0; t < NT; ++t) wt[t] = zero;
#pragma unroll
    for (int kb = 0; kb < 2; ++kb)
      if (kb == 0 || high)
#pragma unroll
        for (int t = 0; t < NT; ++t) {
          bf16x8 b[3];
          sb::load_frag<3>(b, xl + 16 * t * kC + at16<kC>(lr, 32 * kb + 8 * lg), VT * kC);
          sb::mma<3, 3>(wt[t], mf[kb], b);
        }
    load_tri<3>(mf, mp, mat, true, high);
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      sb::split_store4<3>(ul + 16 * t * kC + at16<kC>(lr, ib), VT * kC, vc.tail * wt[t]);
      if constexpr (!BARE) *reinterpret_cast<f32x4*>(wl + (c & 1) * L::F + 16 * t * kC + at32<kC>(lr, ib)) = wt[t];
    }
    lds_barrier();
#pragma unroll
    for (int t = 0; t < KB2; ++t)
#pragma unroll
      for (int u = 0; u < NT; ++u) S[t][u] *= vc.last;
#pragma unroll
    for (int kb = 0; kb < 2; ++kb)
#pragma unroll
      for (int u = 0; u < NT; ++u) {
        bf16x8 b[3];
        sb::load_frag<3>(b, ul + 16 * u * kC + at16<kC>(lr, 32 * kb + 8 * lg), VT * kC);
#pragma unroll
        for (int t = 0; t < KB2; ++t) sb::mma<NP, 3>(S[t][u], ktf[t][kb], b);
      }
    load_kt<NP, KB2>(ktf, ktp, ktat);
  }
}

template <typename T, int NP, int KB2, int NT, bool TRAIN, bool WIDE>
__global__ __launch_bounds__(512, 1) void gdr_scan_fwd_kernel(GdrArgs a) {
  using L = ScanLds<NP, KB2, NT>;
  constexpr int Kp = L::Kp, KB = Kp / 32, VT = L::VT;
  extern __shared__ __align__(16) char smem[];
  __bf16* const sl = reinterpret_cast<__bf16*>(smem);      // [3][VT][Kp] S
  __bf16* const xl = sl + L::S;                            // [3][VT][kC]  beta (V - gam K S)
  __bf16* const ul = xl + L::X;                            // [3][VT][kC]  exp(G_C - G) W
  float* const wl = reinterpret_cast<float*>(ul + L::X);   // [2][VT][kC]  W, of the chunk at hand and the one in front of it
  T* const vl = reinterpret_cast<T*>(wl + 2 * L::F);       // [2][VT][kC]  v, of the chunk at hand and the next one
  float* const ot = reinterpret_cast<float*>(vl + 2 * VT * kC);   // [4 waves][16][VT]  o on its way to rows
  int n, hv, v0, seg;
  if (!scan_tile(a, VT, n, hv, v0, seg)) return;
  const int hk = hv / a.rep;
  const int tid = threadIdx.x, lane = tid & 63, w = (tid >> 6) & 3, lr = lane & 15, lg = lane >> 4;
  long start, slot0;
  int len;
  seq_range(a, n, start, len, slot0);
  const int nc = (len + kC - 1) / kC;
  const int c0 = seg * a.seg_chunks, c1 = min(nc, c0 + a.seg_chunks);
  if (seg > 0 && c0 >= nc) return;
  const int ia = 16 * w + lr;                              // operand row
  const bool high = w >= 2;                                // M and P are lower triangular: rows < 32 read 32 columns
  const long nh = (long)n * a.Hv + hv;
  const f32x4 zero = {0.f, 0.f, 0.f, 0.f};

  if (tid < 256) {                                         // ---- the chain
    f32x4 S[KB2][NT];
    if (a.segs == 1) load_state<KB2, NT>(S, a.s0, a, nh, w, v0, lr, lg);
    else load_seg<KB2, NT>(S, a.seg_s + (nh * a.segs + seg) * Kp * a.vp, a.vp, w, v0, lr, lg);   // s0 may be s1 by now
    if (c0 < c1) scan_chain<T, NP, KB2, NT, TRAIN, false, WIDE>(a, S, sl, xl, ul, vl, wl, hv, a.V, v0, start, len, slot0, c0, c1);
    if (a.s1 && c1 == nc) store_state<KB2, NT>(S, a.s1, a, nh, w, v0, lr, lg);
  } else if (c0 < c1) {                                    // ---- the output, between the chain's barriers
    // Chunk c: Q S behind barrier 1, the first half of P W behind barrier 3, the second behind the next chunk's barrier 2,
    // the store behind its barrier 1 after that: no stretch between two barriers is longer than the chain's.
    bf16x8 qf[KB][NP], pf[2][3];
    f32x4 qn[NT], qs[NT], qo[NT];
    const __bf16* const qp = a.qpk + ((slot0 + c0) * a.Hk + hk) * kC * NP * Kp;
    const long qstep = (long)a.Hk * kC * NP * Kp;
    const unsigned qat = w * KB * NP * kFrag + lane * 8;
    const __bf16* const pp = a.p + ((slot0 + c0) * a.Hv + hv) * 3 * kC * kC;
    const long pstep = (long)a.Hv * 3 * kC * kC;
    const unsigned pat = w * 2 * 3 * kFrag + lane * 8;
    // The products are formed turned (S^T Q^T, W^T P^T): a lane then holds four columns of a token, and four lanes' worth of
    // neighbours is one exchange inside the wave away (through its part of ot)
    const RowTile<T, NT, WIDE> op(a.o, a.ldo, start, len, hv, a.V, v0, w, lane);
    RowTile<T, NT, WIDE> vp(a.v, a.ldv, start, len, hv, a.V, v0, w, lane);
    const int ta = 16 * w + (lane >> 2), cb = 4 * NT * (lane & 3);
    float* const ow = ot + 16 * w * VT;
    auto pw = [&](int c, int kb) {                         // qs += P W, columns 32*kb of P; W as the chain left it in wl
      const float* const wc = wl + (c & 1) * L::F;
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        float x[8];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const f32x4 y = *reinterpret_cast<const f32x4*>(wc + 16 * t * kC + at32<kC>(lr, 32 * kb + 8 * lg + 4 * h));
#pragma unroll
          for (int e = 0; e < 4; ++e) x[4 * h + e] = y[e];
        }
        bf16x8 b[3];
        sb::split8<3>(x, b);
        sb::mma<3, 3>(qs[t], b, pf[kb]);
      }
    };
    auto second = [&](int c) {                             // the second half, and W for the backward pass
      if (high) pw(c, 1);
      load_half<3>(pf[1], pp + (min(c + 1, c1 - 1) - c0) * pstep, pat + (high ? 3 * kFrag : 0));
      if constexpr (TRAIN) {
        float* const wp = a.w + ((((slot0 + c) * a.Hv + hv) * (a.vp / 32) + v0 / 32) * kC) * 32 + (v0 & 16);
float y[4 * NT];
        token_row<4 * NT>(y, wl + (c & 1) * L::F, ta, cb);
        store_row<4 * NT>(wp + (unsigned)(ta * 32 + cb), y);
      }
#pragma unroll
      for (int t = 0; t < NT; ++t) qo[t] = qs[t] * a.scale;
    };
    auto store = [&](int c) {
#pragma unroll
      for (int t = 0; t < NT; ++t) *reinterpret_cast<f32x4*>(ow + at32<VT>(lr, 16 * t + 4 * lg)) = qo[t];
      float y[4 * NT];
#pragma unroll
      for (int h = 0; h < NT; ++h) {
        const f32x4 z = *reinterpret_cast<const f32x4*>(ow + at32<VT>(lane >> 2, cb + 4 * h));
#pragma unroll
        for (int e = 0; e < 4; ++e) y[4 * h + e] = z[e];
      }
      op.store(c, y);
    };
    const float* gp = a.vec + ((slot0 + c0) * a.Hv + hv) * kVecs * kC + kGam * kC;
    RowTile<T, NT, WIDE> first = vp;
    first.load(c0);
    GDR_IN_ORDER;
    load_rows<NP, KB>(qf, qp, qat);
    GDR_IN_ORDER;
    vp.load(min(c0 + 1, c1 - 1));
    GDR_IN_ORDER;
    load_half<3>(pf[1], pp, pat + (high ? 3 * kFrag : 0));
    float gam = gp[(unsigned)ia];
    GDR_IN_ORDER;
    load_half<3>(pf[0], pp, pat);
    GDR_IN_ORDER;
    first.put(vl + (c0 & 1) * VT * kC, w, lane);
    for (int c = c0; c < c1; ++c) {
      lds_barrier();
#pragma unroll
      for (int t = 0; t < NT; ++t) qn[t] = zero;
#pragma unroll
      for (int kb = 0; kb < KB; ++kb)
#pragma unroll
        for (int t = 0; t < NT; ++t) {
          bf16x8 b[3];
          sb::load_frag<3>(b, sl + 16 * t * Kp + at16<Kp>(lr, 32 * kb + 8 * lg), VT * Kp);
          sb::mma<3, NP>(qn[t], b, qf[kb]);
        }
      load_rows<NP, KB>(qf, qp + (min(c + 1, c1 - 1) - c0) * qstep, qat);
      if (c > c0 + 1) store(c - 2);
      vp.put(vl + (~c & 1) * VT * kC, w, lane);
      vp.load(min(c + 2, c1 - 1));
      lds_barrier();
      if (c > c0) second(c - 1);
#pragma unroll
      for (int t = 0; t < NT; ++t) qs[t] = qn[t] * gam;
      gp += c + 1 < c1 ? (long)a.Hv * kVecs * kC : 0;
      gam = gp[(unsigned)ia];
      lds_barrier();
      pw(c, 0);
      load_half<3>(pf[0], pp + (min(c + 1, c1 - 1) - c0) * pstep, pat);
    }
    if (c1 - c0 > 1) store(c1 - 2);
    second(c1 - 1);
    store(c1 - 1);
  }
}

// Long sequences with few heads: the chunks of a sequence are cut into segments that all run at once.  A segment moves the
// state it is given to M S + N; one launch finds M and N of every segment but the last (the chain alone, on the columns of
// V from a zero state and on K columns without a v from the unit state), one joins the states along the segments, and the
// scan then runs with every segment's own first state.  The chain is walked twice, and K / V more columns of it the first
// time, by as many times the workgroups.  32768 tokens of 8 heads, 8 segments: 858 us -> 187 + 19 (joining) + 168.
template <typename T, int NP, int KB2, bool WIDE>
__global__ __launch_bounds__(256, 2) void gdr_segment_kernel(GdrArgs a) {
  constexpr int NT = 2;
  using L = ScanLds<NP, KB2, NT>;
  constexpr int Kp = L::Kp, VT = L::VT;
  extern __shared__ __align__(16) char smem[];
  __bf16* const sl = reinterpret_cast<__bf16*>(smem);
  __bf16* const xl = sl + L::S;
  __bf16* const ul = xl + L::X;
  T* const vl = reinterpret_cast<T*>(ul + L::X);
  int n, hv, v0, seg;
  if (!scan_tile(a, VT, n, hv, v0, seg)) return;           // tiles: the columns of V, then Kp of the unit state
  long start, slot0;
  int len;
  seq_range(a, n, start, len, slot0);
  const int nc = (len + kC - 1) / kC, c0 = seg * a.seg_chunks, c1 = c0 + a.seg_chunks;
  if (c1 >= nc) return;                                    // the last segment's end is nobody's beginning
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, lr = lane & 15, lg = lane >> 4;
  const bool unit = v0 >= a.vp;
  const int j0 = v0 - a.vp;
  f32x4 S[KB2][NT];
#pragma unroll
  for (int t = 0; t < KB2; ++t)
#pragma unroll
    for (int u = 0; u < NT; ++u)
#pragma unroll
      for (int e = 0; e < 4; ++e) S[t][u][e] = unit && 16 * (KB2 * w + t) + 4 * lg + e == j0 + 16 * u + lr ? 1.f : 0.f;
  scan_chain<T, NP, KB2, NT, false, true, WIDE>(a, S, sl, xl, ul, vl, nullptr, hv, unit ? 0 : a.V, unit ? 0 : v0, start, len, slot0, c0, c1);
  const long at = ((long)n * a.Hv + hv) * a.segs + seg;
  if (unit) {
    // as operand blocks (fp32), and transposed for the gradients' way back
#pragma unroll
    for (int t = 0; t < KB2; ++t)
#pragma unroll
      for (int u = 0; u < NT; ++u) {
        const int k0 = 16 * (KB2 * w + t), c0 = j0 + 16 * u;
        float* const m = a.seg_m + at * Kp * Kp + ((k0 >> 4) * (Kp / 32) + (c0 >> 5)) * kFrag;
#pragma unroll
        for (int e = 0; e < 4; ++e) m[frag_at(4 * lg + e, (c0 & 16) + lr)] = S[t][u][e];
        if (a.train) *reinterpret_cast<f32x4*>(a.seg_mt + at * Kp * Kp + ((c0 >> 4) * (Kp / 32) + (k0 >> 5)) * kFrag + frag_at(lr, (k0 & 16) + 4 * lg)) = S[t][u];
      }
  } else {
    store_seg<KB2, NT>(S, a.seg_n + at * Kp * a.vp, a.vp, w, v0, lr, lg);
  }
}

// The first states of the segments, one after the other (backward: the gradients behind the segments, from the last):
// S <- M S + N, 16 columns per workgroup.  The scan takes all of them from here, s0 (d_s1) too: the workgroup of another
// segment may have written s1 over it by then.
template <int KB2>
__global__ __launch_bounds__(256) void gdr_join_kernel(GdrArgs a, bool bwd) {
  constexpr int Kp = 64 * KB2, KB = Kp / 32;
  __shared__ __align__(16) __bf16 sl[3 * 16 * Kp];
  int n, hv, v0, seg;
  if (!scan_tile(a, 16, n, hv, v0, seg)) return;
  long start, slot0;
  int len;
  seq_range(a, n, start, len, slot0);
  const int nc = (len + kC - 1) / kC, ns = (nc + a.seg_chunks - 1) / a.seg_chunks;
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, lr = lane & 15, lg = lane >> 4;
  const long nh = (long)n * a.Hv + hv;
  f32x4 S[KB2][1];
  load_state<KB2, 1>(S, bwd ? a.d_s1 : a.s0, a, nh, w, v0, lr, lg);
  store_seg<KB2, 1>(S, a.seg_s + (nh * a.segs + (bwd ? max(ns - 1, 0) : 0)) * Kp * a.vp, a.vp, w, v0, lr, lg);
  int i = 0;
  if (bwd && ns > 1) {                                     // the last segment has been walked from d_s1
    load_seg<KB2, 1>(S, a.seg_n + (nh * a.segs + ns - 1) * Kp * a.vp, a.vp, w, v0, lr, lg);
    store_seg<KB2, 1>(S, a.seg_s + (nh * a.segs + ns - 2) * Kp * a.vp, a.vp, w, v0, lr, lg);
    i = 1;
  }
  if (i + 1 >= ns) return;
  // a step is one chain of latencies: its M and N are requested a step ahead
  f32x4 mn[KB2][KB][2], nn[KB2][1];
  auto request = [&](int j) {
    const long at = nh * a.segs + (bwd ? ns - 1 - j : j);
    const float* const m = (bwd ? a.seg_mt : a.seg_m) + at * Kp * Kp + KB2 * w * KB * kFrag + lane * 8;
#pragma unroll
    for (int t = 0; t < KB2; ++t)
#pragma unroll
      for (int kb = 0; kb < KB; ++kb)
#pragma unroll
        for (int h = 0; h < 2; ++h) mn[t][kb][h] = *reinterpret_cast<const f32x4*>(m + (t * KB + kb) * kFrag + 4 * h);
    load_seg<KB2, 1>(nn, a.seg_n + at * Kp * a.vp, a.vp, w, v0, lr, lg);
  };
  request(i);
  for (; i + 1 < ns; ++i) {
    f32x4 m[KB2][KB][2], next[KB2][1];
#pragma unroll
    for (int t = 0; t < KB2; ++t) {
      next[t][0] = nn[t][0];
#pragma unroll
      for (int kb = 0; kb < KB; ++kb)
#pragma unroll
        for (int h = 0; h < 2; ++h) m[t][kb][h] = mn[t][kb][h];
    }
    request(min(i + 1, ns - 2));
#pragma unroll
    for (int t = 0; t < KB2; ++t) sb::split_store4<3>(sl + at16<Kp>(lr, 16 * (KB2 * w + t) + 4 * lg), 16 * Kp, S[t][0]);
    lds_barrier();
#pragma unroll
    for (int kb = 0; kb < KB; ++kb) {
      bf16x8 b[3];
      sb::load_frag<3>(b, sl + at16<Kp>(lr, 32 * kb + 8 * lg), 16 * Kp);
#pragma unroll
      for (int t = 0; t < KB2; ++t) {
        float x[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = m[t][kb][e >> 2][e & 3];
        bf16x8 f[3];
        sb::split8<3>(x, f);
        sb::mma<3, 3>(next[t][0], f, b);
      }
    }
    lds_barrier();
#pragma unroll
    for (int t = 0; t < KB2; ++t) S[t][0] = next[t][0];
    store_seg<KB2, 1>(S, a.seg_s + (nh * a.segs + (bwd ? ns - 2 - i : i + 1)) * Kp * a.vp, a.vp, w, v0, lr, lg);
  }
}

// BARE: a segment from a zero gradient (the last one: from d_s1), which leaves only the gradient in front of it, in seg_n.
template <typename T, int NP, int KB2, int NT, bool BARE, bool WIDE>
__global__ __launch_bounds__(512, 1) void gdr_scan_bwd_kernel(GdrArgs a) {
  using L = ScanLds<NP, KB2, NT>;
  constexpr int Kp = L::Kp, KB = Kp / 32, VT = L::VT;
  extern __shared__ __align__(16) char smem[];
  __bf16* const dl = reinterpret_cast<__bf16*>(smem);      // [3][VT][Kp] dS'
  __bf16* const gl = dl + L::S;                            // [3][VT][kC]  scale gam dO
  __bf16* const zl = gl + L::X;                            // [3][VT][kC]  Z
  __bf16* const yl = zl + L::X;                            // [3][VT][kC]  -gam beta Y
  __bf16* const ol = yl + L::X;                            // [NP][VT][kC] dO
  float* const zp = reinterpret_cast<float*>(ol + NP * VT * kC);   // [VT][kC] scale P^T dO
  float* const yf = zp + L::F;                             // [2][VT][kC] Y, of the chunk at hand and the one behind it
  T* const rl = reinterpret_cast<T*>(yf + 2 * L::F);       // [VT][kC] dO as it comes
  int n, hv, v0, seg;
  if (!scan_tile(a, VT, n, hv, v0, seg)) return;
  const int hk = hv / a.rep;
  const int tid = threadIdx.x, lane = tid & 63, w = (tid >> 6) & 3, lr = lane & 15, lg = lane >> 4;
  long start, slot0;
  int len;
  seq_range(a, n, start, len, slot0);
  const int nc = (len + kC - 1) / kC;
  if (BARE) ++seg;                                         // in front of the first segment there is none
  const int c0 = seg * a.seg_chunks, c1 = min(nc, c0 + a.seg_chunks);
  if (seg > 0 && c0 >= nc) return;
  const int ib = 16 * w + 4 * lg;
  const bool low = w < 2;                                  // P^T and M^T are upper triangular: rows >= 32 read the last 32 columns
  const long nh = (long)n * a.Hv + hv;
  const long slot1 = slot0 + c1 - 1;                       // the last chunk, where the walk begins
  const f32x4 zero = {0.f, 0.f, 0.f, 0.f};

  // Barriers of a chunk: 1 (dl), 2 (zl), 3 (yl, yf; gl, zp by the others).  Two more in front of the walk.
  if (tid < 256) {                                         // ---- the chain
    f32x4 dS[KB2][NT];
    const float bad = poison(a);
    if (BARE || a.segs == 1) load_state<KB2, NT>(dS, c1 == nc ? a.d_s1 : nullptr, a, nh, w, v0, lr, lg);
    else load_seg<KB2, NT>(dS, a.seg_s + (nh * a.segs + seg) * Kp * a.vp, a.vp, w, v0, lr, lg);
#pragma unroll
    for (int t = 0; t < KB2; ++t)
#pragma unroll
      for (int u = 0; u < NT; ++u) dS[t][u] += bad;          // from here to dv, d_s0 and, through Y and dS', dk, dg and dbeta
    if (c0 < c1) {
      bf16x8 kf[KB][NP], mf[2][3], ktf[KB2][2][NP], qtf[KB2][2][NP];
      const __bf16* kp = a.kpk + (slot1 * a.Hk + hk) * kC * NP * Kp;
      ScanVec vn;
      const float* vecp = a.vec + (slot1 * a.Hv + hv) * kVecs * kC;
      const __bf16* mp = a.mt + (slot1 * a.Hv + hv) * 3 * kC * kC;
      const __bf16 *ktp = a.kt + (slot1 * a.Hk + hk) * Kp * NP * kC, *qtp = a.qt + (slot1 * a.Hk + hk) * Kp * NP * kC;
      const unsigned kat = w * KB * NP * kFrag + lane * 8, mat = w * 2 * 3 * kFrag + lane * 8, ktat = KB2 * w * 2 * NP * kFrag + lane * 8;
      auto load_t = [&]() {
        load_kt<NP, KB2>(qtf, qtp, ktat);
        load_kt<NP, KB2>(ktf, ktp, ktat);
      };
      load_rows<NP, KB>(kf, kp, kat);
      GDR_IN_ORDER;
      vn.load(vecp, ib);
      GDR_IN_ORDER;
      load_tri<3>(mf, mp, mat, low, true);
      GDR_IN_ORDER;
      load_t();
      GDR_IN_ORDER;
      lds_barrier();
      lds_barrier();
      for (int c = c1 - 1; c >= c0; --c) {
        const int next = max(c - 1, c0);
        const long adv = c - next;
        vecp -= adv * a.Hv * kVecs * kC;
        mp -= adv * a.Hv * 3 * kC * kC;
        ktp -= adv * a.Hk * NP * Kp * kC;
        qtp -= adv * a.Hk * NP * Kp * kC;
        kp -= adv * a.Hk * NP * Kp * kC;
        const ScanVec vc = vn;
        const long vs = (slot0 + c) * a.Hv + hv;
#pragma unroll
        for (int t = 0; t < KB2; ++t)
#pragma unroll
          for (int u = 0; u < NT; ++u)
            sb::split_store4<3>(dl + 16 * u * Kp + at16<Kp>(lr, 16 * (KB2 * w + t) + 4 * lg), VT * Kp, dS[t][u]);
        lds_barrier();
        f32x4 z[NT], y[NT];
#pragma unroll
        for (int t = 0; t < NT; ++t) z[t] = y[t] = zero;
#pragma unroll
        for (int kb = 0; kb < KB; ++kb)
#pragma unroll
          for (int t = 0; t < NT; ++t) {
            bf16x8 b[3];
            sb::load_frag<3>(b, dl + 16 * t * Kp + at16<Kp>(lr, 32 * kb + 8 * lg), VT * Kp);
            sb::mma<NP, 3>(z[t], kf[kb], b);
          }
        load_rows<NP, KB>(kf, kp, kat);
#pragma unroll
        for (int t = 0; t < NT; ++t) {
          const f32x4 p = *reinterpret_cast<const f32x4*>(zp + 16 * t * kC + at32<kC>(lr, ib));
          sb::split_store4<3>(zl + 16 * t * kC + at16<kC>(lr, ib), VT * kC, p + vc.tail * z[t]);
        }
        vn.load(vecp, ib);
        if constexpr (!BARE) {
          store_tile<KB2, NT>(dS, a.ds + ((vs * (a.vp / 32) + v0 / 32) * Kp) * 32 + (v0 & 16) * 16, w, lane);
        }
        lds_barrier();
#pragma unroll
        for (int kb = 0; kb < 2; ++kb)
          if (kb == 1 || low)
#pragma unroll
            for (int t = 0; t < NT; ++t) {
              bf16x8 b[3];
              sb::load_frag<3>(b, zl + 16 * t * kC + at16<kC>(lr, 32 * kb + 8 * lg), VT * kC);
              sb::mma<3, 3>(y[t], mf[kb], b);
            }
        load_tri<3>(mf, mp, mat, low, true);
#pragma unroll
        for (int t = 0; t < NT; ++t) {
          sb::split_store4<3>(yl + 16 * t * kC + at16<kC>(lr, ib), VT * kC, -vc.gam * vc.beta * y[t]);
          if constexpr (!BARE) *reinterpret_cast<f32x4*>(yf + (c & 1) * L::F + 16 * t * kC + at32<kC>(lr, ib)) = y[t];
        }
        lds_barrier();
#pragma unroll
        for (int t = 0; t < KB2; ++t)
#pragma unroll
          for (int u = 0; u < NT; ++u) dS[t][u] *= vc.last;
#pragma unroll
        for (int kb = 0; kb < 2; ++kb)
#pragma unroll
          for (int u = 0; u < NT; ++u) {
            bf16x8 b[3], g[3];
            sb::load_frag<3>(g, gl + 16 * u * kC + at16<kC>(lr, 32 * kb + 8 * lg), VT * kC);
            sb::load_frag<3>(b, yl + 16 * u * kC + at16<kC>(lr, 32 * kb + 8 * lg), VT * kC);
#pragma unroll
            for (int t = 0; t < KB2; ++t) {
              sb::mma<NP, 3>(dS[t][u], qtf[t][kb], g);
              sb::mma<NP, 3>(dS[t][u], ktf[t][kb], b);
            }
          }
        load_t();
      }
    }
    if (BARE) store_seg<KB2, NT>(dS, a.seg_n + (nh * a.segs + seg) * Kp * a.vp, a.vp, w, v0, lr, lg);
    else if (a.d_s0 && seg == 0) store_state<KB2, NT>(dS, a.d_s0, a, nh, w, v0, lr, lg);
  } else if (c0 < c1) {                                    // ---- dO's share, ahead of the chain; Y and dV, behind it
    bf16x8 pf[2][3];
    const bool has_do = a.d_o != nullptr;
    RowTile<T, NT, WIDE> dp(has_do ? a.d_o : a.v, has_do ? a.lddo : a.ldv, start, len, hv, has_do ? a.V : 0, has_do ? v0 : 0, w, lane);
    const __bf16* const pt = a.pt + (slot0 * a.Hv + hv) * 3 * kC * kC;
    const unsigned pat = w * 2 * 3 * kFrag + lane * 8;
    const RowTile<T, NT, WIDE> vo(a.dv, a.lddv, start, len, hv, a.V, v0, w, lane);
    const int ta = 16 * w + (lane >> 2), cb = 4 * NT * (lane & 3);
    const float* const vec = a.vec + (slot0 * a.Hv + hv) * kVecs * kC;
    const long pstep = (long)a.Hv * 3 * kC * kC, vstep = (long)a.Hv * kVecs * kC;
    f32x4 d[NT], dn[NT];                                   // dO of the chunk at hand and of the next one
    auto share = [&]() {                                   // zp of the chunk whose dO is in ol and whose P^T is in pf
      f32x4 z[NT];
#pragma unroll
      for (int t = 0; t < NT; ++t) z[t] = zero;
#pragma unroll
      for (int kb = 0; kb < 2; ++kb)
        if (kb == 1 || low)
#pragma unroll
          for (int t = 0; t < NT; ++t) {
            bf16x8 b[NP];
            sb::load_frag<NP>(b, ol + 16 * t * kC + at16<kC>(lr, 32 * kb + 8 * lg), VT * kC);
            sb::mma<3, NP>(z[t], pf[kb], b);
          }
#pragma unroll
      for (int t = 0; t < NT; ++t) *reinterpret_cast<f32x4*>(zp + 16 * t * kC + at32<kC>(lr, ib)) = a.scale * z[t];
    };
    dp.load(c1 - 1);
    load_tri<3>(pf, pt + (c1 - 1) * pstep, pat, low, true);
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      if (t == 0) dp.put(rl, w, lane);                      // (a wave's tokens are read by nobody else)
      dn[t] = wide4(column4<T>(rl + 16 * t * kC, lr, ib));
      sb::split_store4<NP>(ol + 16 * t * kC + at16<kC>(lr, ib), VT * kC, dn[t]);
    }
    dp.load(max(c1 - 2, c0));
    lds_barrier();
    share();
    load_tri<3>(pf, pt + max(c1 - 2, c0) * pstep, pat, low, true);
    lds_barrier();
    // Y and dV of chunk c, which the chain has left in yf
    auto finish = [&](int c, float beta) {
      float* const yp = a.y + ((((slot0 + c) * a.Hv + hv) * (a.vp / 32) + v0 / 32) * kC) * 32 + (v0 & 16);
      float y[4 * NT];
      token_row<4 * NT>(y, yf + (c & 1) * L::F, ta, cb);
      store_row<4 * NT>(yp + (unsigned)(ta * 32 + cb), y);
#pragma unroll
      for (int e = 0; e < 4 * NT; ++e) y[e] *= beta;
      vo.store(c, y);
    };
    f32x4 gam = *reinterpret_cast<const f32x4*>(vec + (c1 - 1) * vstep + kGam * kC + (unsigned)ib);
    float beta = vec[(c1 - 1) * vstep + kBeta * kC + (unsigned)ta], before = 0.f;                                   // beta of the chunk behind
    for (int c = c1 - 1; c >= c0; --c) {
      const int next = max(c - 1, c0), next2 = max(c - 2, c0);
#pragma unroll
      for (int t = 0; t < NT; ++t) d[t] = dn[t];
      dp.put(rl, w, lane);
#pragma unroll
      for (int t = 0; t < NT; ++t) dn[t] = wide4(column4<T>(rl + 16 * t * kC, lr, ib));
      dp.load(next2);
      lds_barrier();                                       // 1: the chain has read the previous chunk's gl
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        sb::split_store4<3>(gl + 16 * t * kC + at16<kC>(lr, ib), VT * kC, a.scale * gam * d[t]);
        sb::split_store4<NP>(ol + 16 * t * kC + at16<kC>(lr, ib), VT * kC, dn[t]);
      }
      gam = *reinterpret_cast<const f32x4*>(vec + next * vstep + kGam * kC + (unsigned)ib);
      lds_barrier();                                       // 2: the chain has read zp
      share();
      load_tri<3>(pf, pt + next2 * pstep, pat, low, true);
      if (!BARE && c < c1 - 1) finish(c + 1, before);
      before = beta;
      beta = vec[next * vstep + kBeta * kC + (unsigned)ta];
      lds_barrier();                                       // 3
    }
    if (!BARE) finish(c0, before);
  }
}

// ------------------------------------------------------------------------------------------------------ gradients
// One workgroup per chunk and key head; the value heads of the key head one after the other, so that dq and dk are summed
// in registers in a fixed order.  Eight waves: 16 tokens against half of K each.  S, dS', W, Y and dO pass through LDS 32
// columns at a time as bf16 terms; the next 32 columns are on their way from memory meanwhile.
// Where the chip is full neither memory nor the matrix pipes are: 4 x 4096 tokens of 16 heads, K = V = 128, bf16, read 1.09 GB
// and write 0.15 in 375 us (3.3 TB/s, two thirds of what a copy reaches); one chunk takes a CU, which it has to itself, 42
// thousand cycles, 11 thousand of them matrix products.  The rest are splits into terms and waits at barriers and for the next columns.
template <int NP, int KB2>
struct GradsLds {
  static constexpr int Kp = 64 * KB2, LDV = 32;              // columns at a time
  static constexpr int cols = 3 * LDV * (2 * Kp + 2 * kC) + NP * LDV * kC;       // elements: S, dS', W, Y, dO
  // afterwards, over them: R, B and their transposes; with three terms 32 tokens of those and of k and q at a time
  static constexpr int LDR = NP == 1 ? kC : 32;
  static constexpr int tri = 4 * 3 * kC * LDR + (NP == 1 ? 0 : 2 * NP * Kp * LDR);
  static constexpr int NB = NP == 1 ? 2 : 1;                 // column images: two where they fit
  static constexpr int over = 2 * (NB * cols > tri ? NB * cols : tri);
  static constexpr int bytes = over + (8 * kC + 8) * 4;
};
template <typename T, int NP, int KB2, bool GROUP>
__global__ __launch_bounds__(512, 1) void gdr_grads_kernel(GdrArgs a) {
  using L = GradsLds<NP, KB2>;
  constexpr int Kp = L::Kp, LDV = L::LDV, KT = Kp / 32;      // k tiles of a wave
  extern __shared__ __align__(16) char smem[];
  __bf16* const img = reinterpret_cast<__bf16*>(smem);
  constexpr int DL = 3 * Kp * LDV, WL = 2 * DL, YL = WL + 3 * kC * LDV, OL = YL + 3 * kC * LDV;   // [3][Kp][LDV] S and dS', [3][64][LDV] W and Y, [NP][64][LDV] dO
  constexpr int LDR = L::LDR;
  __bf16* const rl = reinterpret_cast<__bf16*>(smem);        // [3][64][LDR] each
  __bf16* const bl = rl + 3 * kC * LDR;
  __bf16* const rt = bl + 3 * kC * LDR;
  __bf16* const bt = rt + 3 * kC * LDR;
  // k and q, transposed, 32 tokens at a time ([NP][Kp][32] each; one term comes straight from the workspace)
  __bf16* const kl = bt + 3 * kC * LDR;
  __bf16* const ql = kl + NP * Kp * LDR;
  float* const rows = reinterpret_cast<float*>(smem + L::over);    // [2 halves][3][64]: shares of dG, of dbeta, k.(tail E3)
  float* const yv = rows + 6 * kC;                                 // [64] Y.v
  float* const red = yv + kC;                                      // [8]
  const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), w = wave >> 1, half = wave & 1, kt0 = 16 * KT * half;
  const long slot = blockIdx.x;
  const int hk = blockIdx.y;
  long row0;
  int valid;
  slot_chunk(a, slot, row0, valid);
  if (valid == 0) return;
  const long hs = slot * a.Hk + hk;
  const f32x4 zero = {0.f, 0.f, 0.f, 0.f};
  const bool has_do = a.d_o != nullptr;
  const float bad = poison(a);
  f32x4 dqs[GROUP ? KT : 1], dks[GROUP ? KT : 1];
  if (GROUP) {
#pragma unroll
    for (int t = 0; t < (GROUP ? KT : 1); ++t) dqs[t] = dks[t] = zero;
  }
  for (int r = 0; r < (GROUP ? a.rep : 1); ++r) {
    int lane = tid & 63;
    if (GROUP) asm("" : "+v"(lane));                         // or every address below would be kept over the loop, in registers that are not there
    const int lr = lane & 15, lg = lane >> 4, ib = 16 * w + 4 * lg;
    // cooperative loads: 8 columns of a row per thread
    const int gi = (64 * (wave & 3) + lane) >> 2, gc = (lane & 3) * 8;   // token and columns of W, dO (waves 0 .. 3), Y, v (the others)
    const long rowc = row0 + min(gi, valid - 1);
    const int hv = hk * (GROUP ? a.rep : 1) + r;
    const long vs = slot * a.Hv + hv;
    f32x4 e1[KT], e2[KT], e3[KT], dp[2], da[2];
#pragma unroll
    for (int t = 0; t < KT; ++t) {
      e1[t] = zero + bad;                                    // (dq)
      e2[t] = e3[t] = zero;
    }
#pragma unroll
    for (int t = 0; t < 2; ++t) dp[t] = da[t] = zero;
    float sdot = 0.f, ydot = 0.f;
    const bool has_s = KB2 == 2 || wave < 4;
    // S, dS': two lanes' registers of a 16 x 16 tile, so four rows of two columns
    const long st0 = vs * (a.vp / 32) * Kp * 32 + (64 * wave + lane) % (4 * Kp) * 8;
    const float *const ps = a.s + st0, *const pd = a.ds + st0;
    const int si = at16<LDV>(16 * (wave % (4 * KB2)) + 4 * (lane >> 3 & 3), 16 * (lane >> 5) + 2 * (lane & 7));
    const float* const pw = (wave < 4 ? a.w : a.y) + (vs * (a.vp / 32) * kC + gi) * 32 + gc;
    const T* const px = wave < 4 ? (has_do ? static_cast<const T*>(a.d_o) + rowc * a.lddo + (long)hv * a.V : static_cast<const T*>(a.v))
                                  : static_cast<const T*>(a.v) + rowc * a.ldv + (long)hv * a.V;
    f32x4 xs[2], xd[2], xw[2];
    u32x4 xo[sizeof(T) / 2];                                 // eight columns of dO or v, as they come
    auto request = [&](int vb) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        xs[h] = *reinterpret_cast<const f32x4*>(ps + vb * Kp + 4 * h);
        xd[h] = *reinterpret_cast<const f32x4*>(pd + vb * Kp + 4 * h);
        xw[h] = *reinterpret_cast<const f32x4*>(pw + vb * kC + 4 * h);
      }
      if (a.wide_v) {                                          // V a multiple of 8, 16-byte aligned rows
#pragma unroll
        for (int h = 0; h < (int)sizeof(T) / 2; ++h) xo[h] = *reinterpret_cast<const u32x4*>(px + min(vb + gc, a.V - 8) + 4 * h);
      } else {
        T raw[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) raw[e] = px[min(vb + gc + e, a.V - 1)];
        __builtin_memcpy(xo, raw, sizeof(raw));
      }
    };
    // columns vb .., which have been requested, into an image
    auto stage = [&](int vb, __bf16* im) {
      float x[8];
      bf16x8 t[3];
      if (has_s) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          sdot = fmaf(xs[0][e], xd[0][e], fmaf(xs[1][e], xd[1][e], sdot));
          unsigned u[3], v[3];
          sb::split2<3>(xs[0][e], xs[1][e], u);
          sb::split2<3>(xd[0][e], xd[1][e], v);
#pragma unroll
          for (int p = 0; p < 3; ++p) {
            *reinterpret_cast<unsigned*>(im + p * Kp * LDV + si + e * LDV) = u[p];
            *reinterpret_cast<unsigned*>(im + DL + p * Kp * LDV + si + e * LDV) = v[p];
          }
        }
      }
      float o[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const unsigned y = sizeof(T) == 2 ? e & 1 ? xo[0][e >> 1] & 0xffff0000u : xo[0][e >> 1] << 16 : xo[sizeof(T) / 2 - 1 - (e < 4)][e & 3];
        o[e] = gi < valid && vb + gc + e < a.V ? __uint_as_float(y) : 0.f;
      }
      __bf16* const dst = im + (wave < 4 ? WL : YL) + at16<LDV>(gi, gc);
#pragma unroll
      for (int e = 0; e < 8; ++e) x[e] = xw[e >> 2][e & 3];
      sb::split8<3>(x, t);
#pragma unroll
      for (int p = 0; p < 3; ++p) *reinterpret_cast<bf16x8*>(dst + p * kC * LDV) = t[p];
      if (wave < 4) {
        bf16x8 u[NP];
#pragma unroll
        for (int e = 0; e < 8; ++e) o[e] = has_do ? o[e] : 0.f;
        sb::split8<NP>(o, u);
#pragma unroll
        for (int p = 0; p < NP; ++p) *reinterpret_cast<bf16x8*>(im + OL + p * kC * LDV + at16<LDV>(gi, gc)) = u[p];
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) ydot = fmaf(x[e], o[e], ydot);
      }
    };
    auto products = [&](const __bf16* im) {
      bf16x8 of[NP], yf[3], wf[3];
      const int fr = at16<LDV>(lr, 8 * lg);
      sb::load_frag<NP>(of, im + OL + 16 * w * LDV + fr, kC * LDV);
      sb::load_frag<3>(yf, im + YL + 16 * w * LDV + fr, kC * LDV);
      sb::load_frag<3>(wf, im + WL + 16 * w * LDV + fr, kC * LDV);
#pragma unroll
      for (int t = 0; t < KT; ++t) {
        bf16x8 b[3], d[3];
        sb::load_frag<3>(b, im + (kt0 + 16 * t) * LDV + fr, Kp * LDV);
        sb::load_frag<3>(d, im + DL + (kt0 + 16 * t) * LDV + fr, Kp * LDV);
        sb::mma<NP, 3>(e1[t], of, b);
        sb::mma<3, 3>(e2[t], yf, b);
        sb::mma<3, 3>(e3[t], wf, d);
      }
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        const int jt = 2 * t + half;
        if (jt <= w) {
          bf16x8 b[3];
          sb::load_frag<3>(b, im + WL + 16 * jt * LDV + fr, kC * LDV);
          sb::mma<NP, 3>(dp[t], of, b);
          sb::mma<3, 3>(da[t], yf, b);
        }
      }
    };
    // k and q in the layout of a result: four tokens of one column, from the transposes or (fp32) from the caller's rows
    bf16x4 kr[NP == 1 ? KT : 1], qr[NP == 1 ? KT : 1];
    bf16x8 kf1[2][NP == 1 ? KT : 1], qf1[2][NP == 1 ? KT : 1];   // and as operands of the products below
    unsigned kx[NP == 1 ? 1 : KT][4], qx[NP == 1 ? 1 : KT][4];
    auto own = [&]() {
#pragma unroll
      for (int t = 0; t < KT; ++t) {
        const long at = hs * Kp * kC + (kt0 / 16 + t) * 2 * kFrag;
        kr[t] = *reinterpret_cast<const bf16x4*>(a.kt + at + (w >> 1) * kFrag + frag_at(lr, ib));
        qr[t] = *reinterpret_cast<const bf16x4*>(a.qt + at + (w >> 1) * kFrag + frag_at(lr, ib));
#pragma unroll
        for (int kb = 0; kb < 2; ++kb) {
          kf1[kb][t] = *reinterpret_cast<const bf16x8*>(a.kt + at + kb * kFrag + lane * 8);
          qf1[kb][t] = *reinterpret_cast<const bf16x8*>(a.qt + at + kb * kFrag + lane * 8);
        }
      }
      asm volatile("" ::: "memory");                         // or the requests would move below the products
    };
    request(0);
    if constexpr (L::NB == 2) {
      // Two waves share a SIMD: one of them multiplies while the other splits the next columns, then the other way round.
      stage(0, img);
      request(min(32, a.vp - 32));
      lds_barrier();
      int cur = 0;
      for (int vb = 32; vb < a.vp; vb += 32) {
        if (wave < 4) products(img + cur);
        stage(vb, img + L::cols - cur);
        request(min(vb + 32, a.vp - 32));
        if (wave >= 4) products(img + cur);
        cur = L::cols - cur;
        lds_barrier();
      }
      own();
      products(img + cur);
    } else {
      for (int vb = 0; vb < a.vp; vb += 32) {
        lds_barrier();
        stage(vb, img);
        request(min(vb + 32, a.vp - 32));                    // in front of the barrier: behind it the compiler moves them below the products
        lds_barrier();
        products(img);
      }
    }
    // ---- the chunk's own part
    const float* const vec = a.vec + vs * kVecs * kC;
    const f32x4 gam = *reinterpret_cast<const f32x4*>(vec + kGam * kC + ib);
    const f32x4 tail = *reinterpret_cast<const f32x4*>(vec + kTail * kC + ib);
    const f32x4 beta = *reinterpret_cast<const f32x4*>(vec + kBeta * kC + ib);
    const f32x4 ghi = *reinterpret_cast<const f32x4*>(vec + kGHi * kC + ib);
    const f32x4 glo = *reinterpret_cast<const f32x4*>(vec + kGLo * kC + ib);
    const float last = vec[kGam * kC + kC - 1];
    float hj[2], lj[2];
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      hj[t] = vec[kGHi * kC + 16 * (2 * t + half) + lr];
      lj[t] = vec[kGLo * kC + 16 * (2 * t + half) + lr];
    }
    if constexpr (NP != 1) {
      const __amdgpu_buffer_rsrc_t rk = rows_rsrc(a.k, (row0 * a.ldk + (long)hk * a.K) * 4, ((valid - 1) * a.ldk + a.K) * 4);
      const __amdgpu_buffer_rsrc_t rq = rows_rsrc(a.q, (row0 * a.ldq + (long)hk * a.K) * 4, ((valid - 1) * a.ldq + a.K) * 4);
#pragma unroll
      for (int t = 0; t < KT; ++t)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int k = kt0 + 16 * t + lr;
          kx[t][e] = __builtin_amdgcn_raw_buffer_load_b32(rk, k < a.K ? ((ib + e) * (unsigned)a.ldk + k) * 4 : kNoColumn, 0, 0);
          qx[t][e] = __builtin_amdgcn_raw_buffer_load_b32(rq, k < a.K ? ((ib + e) * (unsigned)a.ldq + k) * 4 : kNoColumn, 0, 0);
        }
    }
    __builtin_amdgcn_sched_barrier(0);                       // all of these requests together, in front of what waits for them
    ydot += __shfl_xor(ydot, 1, 64);
    ydot += __shfl_xor(ydot, 2, 64);
    sdot = wave_sum(sdot);
    f32x4 kv[KT], qv[KT];
#pragma unroll
    for (int t = 0; t < KT; ++t)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        kv[t][e] = NP == 1 ? (float)kr[NP == 1 ? t : 0][e] : __uint_as_float(kx[NP == 1 ? 0 : t][e]);
        qv[t][e] = NP == 1 ? (float)qr[NP == 1 ? t : 0][e] : __uint_as_float(qx[NP == 1 ? 0 : t][e]);
      }
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      const int j = 16 * (2 * t + half) + lr;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int i = ib + e;
        const float d = i >= j ? decay(ghi[e], glo[e], hj[t], lj[t]) : 0.f;
        dp[t][e] = i >= j ? a.scale * dp[t][e] * d : 0.f;
        da[t][e] = i > j ? -da[t][e] * d : 0.f;
      }
    }
    f32x4 dg = zero, db = zero, st = zero, kc = zero;
#pragma unroll
    for (int t = 0; t < KT; ++t) {
      e1[t] *= a.scale * gam;
      e2[t] *= -gam;
      e3[t] *= tail;
      st += kv[t] * e3[t];
    }
    // R and B (columns j0..) and their transposes (rows' tokens i0..) into LDS
    auto put = [&](int t, int j0) {
      const int j = 16 * (2 * t + half) + lr;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        __bf16 x[3];
        sb::split3(dp[t][e], x[0], x[1], x[2]);
#pragma unroll
        for (int p = 0; p < 3; ++p) rl[p * kC * LDR + at16<LDR>(ib + e, j - j0)] = x[p];
        sb::split3(da[t][e], x[0], x[1], x[2]);
#pragma unroll
        for (int p = 0; p < 3; ++p) bl[p * kC * LDR + at16<LDR>(ib + e, j - j0)] = x[p];
      }
    };
    auto put_t = [&](int t, int i0) {
      const int j = 16 * (2 * t + half) + lr;
      sb::split_store4<3>(rt + at16<LDR>(j, ib - i0), kC * LDR, dp[t]);
      sb::split_store4<3>(bt + at16<LDR>(j, ib - i0), kC * LDR, beta * da[t]);
    };
    // the products of 32 tokens: at = where they begin in the images
    auto join = [&](int kb, int at) {
      const int fr = at16<LDR>(lr, at + 8 * lg);
      const __bf16* const kf = kl + kt0 * LDR + fr;
      const __bf16* const qf = ql + kt0 * LDR + fr;
      if (kb == 0 || w >= 2) {
        bf16x8 rf[3], bf[3];
        sb::load_frag<3>(rf, rl + 16 * w * LDR + fr, kC * LDR);
        sb::load_frag<3>(bf, bl + 16 * w * LDR + fr, kC * LDR);
#pragma unroll
        for (int t = 0; t < KT; ++t) {
          bf16x8 b[NP];
          if constexpr (NP == 1) b[0] = kf1[kb][t];
          else sb::load_frag<NP>(b, kf + 16 * t * LDR, Kp * LDR);
          sb::mma<3, NP>(e1[t], rf, b);
          sb::mma<3, NP>(e2[t], bf, b);
        }
      }
      if (kb == 1 || w < 2) {
        bf16x8 rf[3], bf[3];
        sb::load_frag<3>(rf, rt + 16 * w * LDR + fr, kC * LDR);
        sb::load_frag<3>(bf, bt + 16 * w * LDR + fr, kC * LDR);
#pragma unroll
        for (int t = 0; t < KT; ++t) {
          bf16x8 b[NP];
          if constexpr (NP == 1) b[0] = qf1[kb][t];
          else sb::load_frag<NP>(b, qf + 16 * t * LDR, Kp * LDR);
          sb::mma<3, NP>(e3[t], rf, b);
          if constexpr (NP == 1) b[0] = kf1[kb][t];
          else sb::load_frag<NP>(b, kf + 16 * t * LDR, Kp * LDR);
          sb::mma<3, NP>(e3[t], bf, b);
        }
      }
    };
    __syncthreads();
    if (wave >= 4 && (lane & 3) == 0) yv[gi] = ydot;
    if (lane == 0) red[wave] = sdot;
    if constexpr (NP == 1) {
      put(0, 0);
      put(1, 0);
      put_t(0, 0);
      put_t(1, 0);
      __syncthreads();
#pragma unroll
      for (int kb = 0; kb < 2; ++kb) join(kb, 32 * kb);
    } else {
#pragma unroll
      for (int kb = 0; kb < 2; ++kb) {
        // a block of 16 columns of k (q) by 32 tokens per wave
        constexpr int U = (NP * Kp / 16 + 7) / 8;
        bf16x8 x[2][U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
          const int blk = min(u * 8 + wave, NP * Kp / 16 - 1), t = blk / NP, p = blk - t * NP;
          const long at = hs * Kp * NP * kC + ((t * 2 + kb) * NP + p) * kFrag + lane * 8;
          x[0][u] = *reinterpret_cast<const bf16x8*>(a.kt + at);
          x[1][u] = *reinterpret_cast<const bf16x8*>(a.qt + at);
        }
        if (kb) __syncthreads();                             // the first half's images have been read
        put(kb, 32 * kb);
        if ((w >> 1) == kb) {
          put_t(0, 32 * kb);
          put_t(1, 32 * kb);
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
          const int blk = min(u * 8 + wave, NP * Kp / 16 - 1), t = blk / NP, p = blk - t * NP;      // (the last block's copies are the same)
          const int at = at16<LDR>(p * Kp + 16 * t + lr, 8 * lg);
          *reinterpret_cast<bf16x8*>(kl + at) = x[0][u];
          *reinterpret_cast<bf16x8*>(ql + at) = x[1][u];
        }
        __syncthreads();
        join(kb, 0);
      }
    }
#pragma unroll
    for (int t = 0; t < KT; ++t) {
      dg += qv[t] * e1[t];
      db += kv[t] * e2[t];
      kc += kv[t] * e3[t];
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
      if (lr == 0) {
        float* const p = rows + half * 3 * kC + ib + e;
        p[0] = x; p[kC] = y; p[2 * kC] = z;
      }
    }
    __syncthreads();
    if (wave == 0) {
      // <dS', S'> = gam_C <dS', S> + sum_i k_i.(tail E3)_i reaches every token of the chunk, dG_i those up to i
      double share = (double)rows[2 * kC + lane] + rows[5 * kC + lane];
#pragma unroll
      for (int off = 32; off > 0; off >>= 1) share += __shfl_xor(share, off, 64);
      double sd = 0.0;
#pragma unroll
      for (int i = 0; i < 8; ++i) sd += red[i];
      share += (double)last * sd;
      double s = (double)rows[lane] + rows[3 * kC + lane];
#pragma unroll
      for (int off = 1; off < 64; off <<= 1) {
        const double down = __shfl_down(s, off, 64);
        if (lane + off < 64) s += down;
      }
      if (lane < valid) {
        a.dg[(row0 + lane) * a.lddg + hv] = (float)(s + share);
        a.dbeta[(row0 + lane) * a.lddbeta + hv] = yv[lane] + (rows[kC + lane] + rows[4 * kC + lane]);
      }
    }
    if (!GROUP || r == a.rep - 1) {
      T* const pq = static_cast<T*>(a.dq) + (row0 + ib) * a.lddq + (long)hk * a.K + kt0 + lr;
      T* const pk = static_cast<T*>(a.dk) + (row0 + ib) * a.lddk + (long)hk * a.K + kt0 + lr;
#pragma unroll
      for (int t = 0; t < KT; ++t) {
        const f32x4 dq = GROUP ? dqs[t] : e1[t], dk = GROUP ? dks[t] : e2[t];
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (ib + e < valid && kt0 + 16 * t + lr < a.K) {
            pq[e * a.lddq + 16 * t] = (T)dq[e];
            pk[e * a.lddk + 16 * t] = (T)dk[e];
          }
      }
    }
  }
}

// ------------------------------------------------------------------------------------------------------- one token
// A workgroup holds 16 columns (x VEC) of one row's head: 16 threads along the columns, 16 along K.  The two sums over K
// that a token needs, S^T k and S^T q, are taken of the state as it is stored: o = scale (a S^T q + (q.k) u) with
// u = beta (v - a S^T k), so the state is read once, moved in registers and written once, behind one exchange in LDS.
// Bound by the state's way through memory: 192 rows of 32 heads, K = V = 128: 0.81 GB in 161 us, 5.0 TB/s.  One row of 4
// heads takes 4.2 us, two latencies of memory.
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
// rows of V elements that may be taken in 16-byte pieces
int rows16(int dtype, int V, const void* p, long ld) {
  const int n = dtype == HHRL_BF16 ? 8 : 4;
  return V % n == 0 && ld % n == 0 && a16(p);
}
int padded_k(int K) { return K <= 64 ? 64 : 128; }
long slots_of(int n_seq, long rows, bool packed) {
  return packed ? rows / kC + n_seq : (long)n_seq * ((rows / n_seq + kC - 1) / kC);
}

// Segments per sequence and their chunks.  Cutting a sequence in s pays a second walk of 1/s of the chunks with K / V more
// columns and a join of s steps, about one chunk each, so it takes three, of 16 chunks or more, and a chip whose 256 CUs
// hold them side by side (32-column workgroups).  Measured for 32768 tokens, K = V = 128 (no other widths), whole calls: 8
// heads (8 segments) 935 -> 457 us, 12 (5) 1013 -> 701, 16 (4) 1034 -> 822, 20 (3) 1139 -> 1036; 4096 tokens, 8 heads (4 of 16
// chunks) 105 -> 102; two segments would be slower than none.  Packed sequences may all be one.
int segments_of(int n_seq, long rows, bool packed, int Hv, int vp, int* chunks) {
  const long most = packed ? rows / kC + 1 : (rows / n_seq + kC - 1) / kC, wgs = (long)n_seq * Hv * (vp / 32);
  long segs = 256 / wgs;
  if (segs > most / 16) segs = most / 16;
  if (segs > 16) segs = 16;
  if (segs < 3) segs = 1;
  *chunks = (int)((most + segs - 1) / segs);
  return (int)segs;
}

// ws: offsets in floats (every array a multiple of 64 floats); returns the total
long carve(GdrArgs* a, float* ws, int dtype, int n_seq, long rows, bool packed, int Hk, int Hv, int K, int V, bool train) {
  const long ns = slots_of(n_seq, rows, packed), kp = padded_k(K), np = dtype == HHRL_BF16 ? 1 : 3, vp = (V + 31) / 32 * 32;
  long off = 0;
  auto take = [&](long floats) { float* p = ws ? ws + off : nullptr; off += (floats + 63) & ~63L; return p; };
  auto take16 = [&](long n) { return reinterpret_cast<__bf16*>(take((n + 1) / 2)); };
  GdrArgs t = {};
  t.mark = reinterpret_cast<unsigned long long*>(take(2));      // (first, so that a forward pass for no backward pass finds it too)
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
  int chunks;
  const int segs = segments_of(n_seq, rows, packed, Hv, (int)vp, &chunks);
  const long pairs = (long)n_seq * Hv;
  if (segs > 1) {
    t.seg_m = take(pairs * segs * kp * kp);
    t.seg_n = take(pairs * segs * kp * vp);
    t.seg_s = take(pairs * segs * kp * vp);
    if (train) t.seg_mt = take(pairs * segs * kp * kp);
  }
  if (a) {
    a->segs = segs; a->seg_chunks = chunks; a->seg_m = t.seg_m; a->seg_mt = t.seg_mt; a->seg_n = t.seg_n; a->seg_s = t.seg_s;
    a->mark = t.mark; a->kpk = t.kpk; a->qpk = t.qpk; a->kt = t.kt; a->qt = t.qt; a->m = t.m; a->p = t.p; a->mt = t.mt; a->pt = t.pt;
    a->vec = t.vec; a->w = t.w; a->y = t.y; a->s = t.s; a->ds = t.ds;
    a->n_slots = ns; a->vp = (int)vp;
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
  const long most = 1L << 22;                    // offsets inside a chunk are 31-bit byte numbers
  HHRL_REQUIRE(d->ldq < most && d->ldk < most && d->ldv < most, "%s: leading dimension of an input beyond %ld", who, most - 1);
  const long ns = slots_of(d->n_seq, d->rows, d->starts != nullptr);
  const long threads = 1L << 32;                 // a launch has fewer than this; workgroups of a scan (segments and 16-column tiles: few heads only)
  const long scan = (((long)d->n_seq * d->Hv + 7) / 8 * 8) * ((d->V + 31) / 32);
  HHRL_REQUIRE(ns < threads / 512 && scan < threads / 512, "%s: %ld chunks, n_seq*Hv*V/32 = %ld: too many for a launch", who, ns, scan);
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
  a.key = 0xcbf29ce484222325ull;                 // FNV-1a over the shapes
  for (long x : {(long)d->dtype, (long)d->n_seq, d->rows, (long)(d->starts != nullptr), (long)d->Hk, (long)d->Hv, (long)d->K, (long)d->V})
    for (int i = 0; i < 8; ++i) a.key = (a.key ^ (x >> 8 * i & 255)) * 0x100000001b3ull;
  a.v16 = rows16(d->dtype, d->V, d->v, d->ldv);
  a.wide = d->K % 8 == 0 && a16(d->q) && a16(d->k) && d->ldq % 8 == 0 && d->ldk % 8 == 0;
  a.whole = d->K == padded_k(d->K) && a.wide;
  return HHRL_OK;
}

// Columns per workgroup of a scan: 16 where twice the workgroups still have a CU each (the chain from chunk to chunk is
// shorter), else 32.  Measured for 16 chunks, K = V = 128, with 16 / 32 columns: 128 workgroups of 32 30 / 41 us, 144 44 / 42,
// 224 47 / 45, 256 48 / 45; of narrower heads (K <= 64, bf16) two workgroups fit on a CU, and they were not measured apart.
// Segments fill the chip with 32.
int scan_tiles(const GdrArgs& a) { return a.segs > 1 || (long)a.n_seq * a.Hv * (a.vp / 32) > 128 ? 2 : 1; }
unsigned scan_grid(const GdrArgs& a) { return (unsigned)(((long)a.n_seq * a.Hv * a.grid_segs + 7) / 8 * 8 * a.nvt); }

template <typename T, int NP, int KB2, int NT, bool WIDE>
int run_scan(GdrArgs a, bool bwd, hipStream_t st, double flops, bool bare = false) {
  a.nvt = a.vp / (16 * NT);
  a.by_length = (a.starts || a.lens) && a.n_seq > 1 && a.n_seq <= 64 && a.segs == 1 && (long)a.n_seq * a.Hv * a.nvt > 256;    // (else all run at once)
  if (bwd) {
    a.grid_segs = bare ? a.segs - 1 : a.segs;
    constexpr int lds = ScanLds<NP, KB2, NT>::bwd_bytes;
    void (*const fn)(GdrArgs) = bare ? gdr_scan_bwd_kernel<T, NP, KB2, NT, true, WIDE> : gdr_scan_bwd_kernel<T, NP, KB2, NT, false, WIDE>;
    HHRL_TRY(ensure_dyn_lds(reinterpret_cast<const void*>(fn), lds, "gdr_backward"));
    ProfScope ps(bare ? "gdr_segment_bwd_kernel" : "gdr_scan_bwd_kernel", st, flops, 0.0);
    hipLaunchKernelGGL(fn, dim3(scan_grid(a)), dim3(512), lds, st, a);
  } else {
    a.grid_segs = a.segs;
    constexpr int lds = ScanLds<NP, KB2, NT>::fwd_bytes;
    void (*const fn)(GdrArgs) = a.train ? gdr_scan_fwd_kernel<T, NP, KB2, NT, true, WIDE> : gdr_scan_fwd_kernel<T, NP, KB2, NT, false, WIDE>;
    HHRL_TRY(ensure_dyn_lds(reinterpret_cast<const void*>(fn), lds, "gdr_forward"));
    ProfScope ps("gdr_scan_fwd_kernel", st, flops, 0.0);
    hipLaunchKernelGGL(fn, dim3(scan_grid(a)), dim3(512), lds, st, a);
  }
  return launch_status(bwd ? "gdr_scan_bwd_kernel" : "gdr_scan_fwd_kernel");
}
// M and N of the segments
template <typename T, int NP, int KB2, bool WIDE>
int run_segments(GdrArgs a, hipStream_t st) {
  constexpr int lds = ScanLds<NP, KB2, 2>::chain_bytes;
  HHRL_TRY(ensure_dyn_lds(reinterpret_cast<const void*>(&gdr_segment_kernel<T, NP, KB2, WIDE>), lds, "gdr_forward"));
  a.grid_segs = a.segs - 1;
  a.nvt = (a.vp + 64 * KB2) / 32;
  ProfScope ps("gdr_segment_kernel", st, 0.0, 0.0);
  hipLaunchKernelGGL((gdr_segment_kernel<T, NP, KB2, WIDE>), dim3(scan_grid(a)), dim3(256), lds, st, a);
  return launch_status("gdr_segment_kernel");
}
template <int KB2>
int run_join(GdrArgs a, bool bwd, hipStream_t st) {
  a.grid_segs = 1;
  a.nvt = a.vp / 16;
  ProfScope ps("gdr_join_kernel", st, 0.0, 0.0);
  hipLaunchKernelGGL((gdr_join_kernel<KB2>), dim3(scan_grid(a)), dim3(256), 0, st, a, bwd);
  return launch_status("gdr_join_kernel");
}
template <typename T, int NP, int KB2, bool WIDE>
int run_scans(const GdrArgs& a, bool bwd, hipStream_t st, double flops) {
  if (a.segs > 1) {
    if (bwd) HHRL_TRY((run_scan<T, NP, KB2, 2, WIDE>(a, true, st, 0.0, true)));
    else HHRL_TRY((run_segments<T, NP, KB2, WIDE>(a, st)));
    HHRL_TRY(run_join<KB2>(a, bwd, st));
  }
  return scan_tiles(a) == 2 ? run_scan<T, NP, KB2, 2, WIDE>(a, bwd, st, flops) : run_scan<T, NP, KB2, 1, WIDE>(a, bwd, st, flops);
}
template <typename T, int NP, int KB2>
int run_scans(const GdrArgs& a, bool bwd, hipStream_t st, double flops) {
  return a.v16 ? run_scans<T, NP, KB2, true>(a, bwd, st, flops) : run_scans<T, NP, KB2, false>(a, bwd, st, flops);
}

template <typename T, int NP, int KB2>
int run_fwd(const GdrArgs& a, hipStream_t st, double flops) {
  constexpr int lds_prep = PrepLds<NP, KB2>::bytes;
  HHRL_TRY(ensure_dyn_lds(reinterpret_cast<const void*>(&gdr_prep_kernel<T, NP, KB2>), lds_prep, "gdr_forward"));
  {
    ProfScope ps("gdr_prep_kernel", st, 0.0, 0.0);
    hipLaunchKernelGGL((gdr_prep_kernel<T, NP, KB2>), dim3((unsigned)a.n_slots, a.Hk), dim3(256), lds_prep, st, a);
  }
  HHRL_TRY(launch_status("gdr_prep_kernel"));
  return run_scans<T, NP, KB2>(a, false, st, flops);
}

template <typename T, int NP, int KB2, bool GROUP>
int run_grads(const GdrArgs& a, hipStream_t st, double flops) {
  constexpr int lds = GradsLds<NP, KB2>::bytes;
  HHRL_TRY(ensure_dyn_lds(reinterpret_cast<const void*>(&gdr_grads_kernel<T, NP, KB2, GROUP>), lds, "gdr_backward"));
  ProfScope ps("gdr_grads_kernel", st, flops, 0.0);
  hipLaunchKernelGGL((gdr_grads_kernel<T, NP, KB2, GROUP>), dim3((unsigned)a.n_slots, a.Hk), dim3(512), lds, st, a);
  return launch_status("gdr_grads_kernel");
}

template <typename T, int NP, int KB2>
int run_bwd(const GdrArgs& a, hipStream_t st, double flops) {
  HHRL_TRY((run_scans<T, NP, KB2>(a, true, st, flops)));
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
  HHRL_REQUIRE(d->ldo < (1L << 22), "gdr_forward: ldo=%ld too large", d->ldo);
  GdrArgs a = {};
  HHRL_TRY(gdr_fill(d, a, !d->no_backward, "gdr_forward"));
  a.v16 = a.v16 && rows16(d->dtype, d->V, d->o, d->ldo);
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
  HHRL_REQUIRE((!d->d_o || d->lddo < (1L << 22)) && d->lddv < (1L << 22), "gdr_backward: leading dimension of d_o or dv too large");
  GdrArgs a = {};
  HHRL_TRY(gdr_fill(d, a, true, "gdr_backward"));
  a.v16 = (d->d_o ? rows16(d->dtype, d->V, d->d_o, d->lddo) : a.v16) && rows16(d->dtype, d->V, d->dv, d->lddv);
  a.d_o = d->d_o; a.lddo = d->lddo; a.d_s1 = d->d_s1; a.d_s0 = d->d_s0;
  a.dq = d->dq; a.dk = d->dk; a.dv = d->dv; a.lddq = d->lddq; a.lddk = d->lddk; a.lddv = d->lddv;
  a.dg = d->dg; a.dbeta = d->dbeta; a.lddg = d->lddg; a.lddbeta = d->lddbeta;
  a.wide_v = d->V % 8 == 0 && a16(d->v) && d->ldv % 8 == 0 && (!d->d_o || (a16(d->d_o) && d->lddo % 8 == 0));
  const double flops = 6.0 * d->rows * d->Hv * d->K * d->V;
  hipStream_t st = as_stream(stream);
  if (d->dtype == HHRL_BF16) return d->K <= 64 ? run_bwd<__bf16, 1, 1>(a, st, flops) : run_bwd<__bf16, 1, 2>(a, st, flops);
  return d->K <= 64 ? run_bwd<float, 3, 1>(a, st, flops) : run_bwd<float, 3, 2>(a, st, flops);
}

int hhrl_gdr_step(const hhrl_gdr_step_desc* d, void* stream) {
  HHRL_REQUIRE(d != nullptr, "gdr_step: null descriptor");
  HHRL_REQUIRE(d->dtype == HHRL_F32 || d->dtype == HHRL_BF16, "gdr_step: dtype %d", d->dtype);
  HHRL_REQUIRE(d->B > 0 && d->n_slots > 0 && d->Hk > 0 && d->Hv > 0 && d->Hv % d->Hk == 0, "gdr_step: B=%d n_slots=%d Hk=%d Hv=%d", d->B, d->n_slots, d->Hk, d->Hv);
  HHRL_REQUIRE(d->slots || d->B <= d->n_slots, "gdr_step: %d rows for %d states", d->B, d->n_slots);
  HHRL_REQUIRE(d->K > 0 && d->K <= HHRL_GDR_MAX_K && d->V > 0 && d->V <= HHRL_GDR_MAX_V, "gdr_step: K=%d V=%d (up to %d, %d supported)", d->K, d->V, HHRL_GDR_MAX_K, HHRL_GDR_MAX_V);
  HHRL_REQUIRE(d->q && d->k && d->v && d->g && d->beta && d->o && d->state_in && d->state_out, "gdr_step: null pointer");
  HHRL_REQUIRE(d->ldq >= (long)d->Hk * d->K && d->ldk >= (long)d->Hk * d->K && d->ldv >= (long)d->Hv * d->V && d->ldo >= (long)d->Hv * d->V && d->ldg >= d->Hv && d->ldbeta >= d->Hv,
               "gdr_step: leading dimension too small");
  const bool vec = d->V % 4 == 0 && a16(d->state_in) && a16(d->state_out);
  GdrStepArgs a = {};
  a.Hk = d->Hk; a.Hv = d->Hv; a.K = d->K; a.V = d->V; a.rep = d->Hv / d->Hk; a.n_slots = d->n_slots; a.scale = d->scale;
  a.q = d->q; a.k = d->k; a.v = d->v; a.ldq = d->ldq; a.ldk = d->ldk; a.ldv = d->ldv; a.g = d->g; a.beta = d->beta; a.ldg = d->ldg; a.ldbeta = d->ldbeta;
  a.o = d->o; a.ldo = d->ldo; a.sin = d->state_in; a.sout = d->state_out; a.slots = d->slots;
  a.nvt = ceil_div(d->V, vec ? 64 : 16);
  const long grid = (long)d->B * d->Hv < (1L << 24) ? (long)d->B * d->Hv * a.nvt : 1L << 24;
  HHRL_REQUIRE(grid < (1L << 24), "gdr_step: B*Hv*V too large: %ld or more workgroups of 256 threads", grid);
  hipStream_t st = as_stream(stream);
  ProfScope ps("gdr_step_kernel", st, 6.0 * d->B * d->Hv * d->K * d->V, 8.0 * d->B * d->Hv * d->K * d->V);
  if (d->dtype == HHRL_BF16) {
    if (vec) launch_step<__bf16, 4>(a, (unsigned)grid, st);
    else launch_step<__bf16, 1>(a, (unsigned)grid, st);
  } else {
    if (vec) launch_step<float, 4>(a, (unsigned)grid, st);
    else launch_step<float, 1>(a, (unsigned)grid, st);
  }
  return launch_status("gdr_step_kernel");
}

}  // extern "C"
