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
#include "block_norm.h"

namespace hhrl {

void norm_launch_f32(const NormArgs& a, bool vec, int tpr, int blocks, bool bwd, hipStream_t st) { norm_launch<float, 4>(a, vec, tpr, blocks, bwd, st); }

// Sums the partial rows in their order: the parameter gradients (ADDED to dst) over all workgroups, and the gate rows
// (written) over the parts of their group.  Parameters with one gradient (a weight that both norms share) are one job.
// 32 columns x 32 row lanes per workgroup: 1024 rows of 128 columns are few workgroups and a long walk (8 row lanes: 8.0 us).
struct NormFoldArgs {
  const float* par_ws;
  const float* gate_ws;
  float* dst[4];
  int n_par, D, blocks, parts;
  float* dgate;
  long lddg, n_groups;
};
__global__ __launch_bounds__(1024) void block_norm_fold_kernel(NormFoldArgs a) {
  __shared__ float red[32][33];
  const int cx = threadIdx.x & 31, ry = threadIdx.x >> 5, col = blockIdx.x * 32 + cx;
  for (long job = blockIdx.y; job < a.n_par + a.n_groups; job += gridDim.y) {
    const bool par = job < a.n_par;
    const long grp = job - a.n_par;
    float* const dst = par ? a.dst[job] : a.dgate + grp * a.lddg;
    bool first = true;
    for (int q = 0; par && q < job; ++q) first &= a.dst[q] != dst;
    if (!first) continue;
    const long stride = par ? (long)a.n_par * a.D : a.D;
    const int rows = par ? a.blocks : a.parts;
    float s = 0.f;
    for (long q = job; q < (par ? a.n_par : job + 1); ++q) {
      if (par && a.dst[q] != dst) continue;
      const float* const src = par ? a.par_ws + q * a.D : a.gate_ws + grp * a.parts * a.D;
      if (col < a.D) {
#pragma unroll 8
        for (int r = ry; r < rows; r += 32) s += src[r * stride + col];
      }
    }
    red[ry][cx] = s;
    __syncthreads();
    if (ry == 0 && col < a.D) {
      for (int r = 1; r < 32; ++r) s += red[r][cx];
      if (par) dst[col] += s;
      else dst[col] = s;
    }
    __syncthreads();
  }
}

namespace {

constexpr int kNormMaxD = 8192;

// Threads per row: the fewest that hold it at eight elements a thread.
int norm_tpr(int D) {
  int t = 16;
  while (t * kNormE < D) t *= 2;
  return t;
}
int norm_slots(int tpr) { return tpr < 256 ? 256 / tpr : 1; }
// Workgroups that are resident at once on 256 CUs with so many waves per SIMD.  A backward pass has no more: each leaves
// one partial row per parameter.
int norm_resident(int tpr, int waves) {
  const int per_cu = waves * 4 * 64 / (tpr < 256 ? 256 : tpr);
  return 256 * (per_cu > 1 ? per_cu : 1);
}

struct NormParts { long group_rows, n_groups, seg_rows, n_segs, segs_per_block; int parts, blocks; };
NormParts norm_parts(long M, int H, long gate_rows, int tpr, int waves) {
  NormParts p;
  const long R = M * H;
  const int slots = norm_slots(tpr), top = norm_resident(tpr, waves);
  const bool bcast = gate_rows > 1;
  p.group_rows = bcast && gate_rows < R ? gate_rows : R;     // (a gate may be said to be for any number of rows)
  p.n_groups = (R + p.group_rows - 1) / p.group_rows;
  const long gr = p.group_rows;
  // at least four rows per slot (a partial row costs as much as a row)
  const long most = (gr + 4L * slots - 1) / (4L * slots);
  long parts = (top + p.n_groups - 1) / p.n_groups;
  if (parts > most) parts = most;
  if (parts < 1) parts = 1;
  p.seg_rows = (gr + parts - 1) / parts;
  p.parts = (int)((gr + p.seg_rows - 1) / p.seg_rows);
  p.n_segs = p.n_groups * p.parts;
  p.segs_per_block = (p.n_segs + top - 1) / top;
  p.blocks = (int)((p.n_segs + p.segs_per_block - 1) / p.segs_per_block);
  return p;
}

bool norm_rows_ok(long M, int H) { return M < (1L << 40) / H; }

bool aligned16(const void* p) { return (reinterpret_cast<unsigned long long>(p) & 15) == 0; }

void launch_norm(const NormArgs& a, int dtype, bool vec, int tpr, int blocks, bool bwd, hipStream_t st) {
  if (dtype == HHRL_BF16) norm_launch_bf16(a, vec, tpr, blocks, bwd, st);
  else norm_launch_f32(a, vec, tpr, blocks, bwd, st);
}

int norm_check(const hhrl_block_norm_desc* d, const char* who) {
  HHRL_REQUIRE(d != nullptr, "%s: null descriptor", who);
  HHRL_REQUIRE(d->dtype == HHRL_F32 || d->dtype == HHRL_BF16, "%s: dtype %d", who, d->dtype);
  HHRL_REQUIRE(d->M > 0 && d->H > 0 && d->D > 0, "%s: bad shape M=%ld H=%d D=%d", who, d->M, d->H, d->D);
  HHRL_REQUIRE(d->D <= kNormMaxD, "%s: D=%d (up to %d supported)", who, d->D, kNormMaxD);
  HHRL_REQUIRE(norm_rows_ok(d->M, d->H), "%s: M*H too large", who);
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
  if (M <= 0 || H <= 0 || !norm_rows_ok(M, H) || D <= 0 || D > kNormMaxD || gate_rows < 1 || (gate_rows > 1 && H != 1)) return 0;
  long most = 0;
  for (int waves : {2, 4})                            // the backward launch chooses by type, alignment and biases,
    for (long rows : {1L, gate_rows}) {               // and by whether the gate is there
      const NormParts p = norm_parts(M, H, rows, norm_tpr(D), waves);
      const long n = (long)p.blocks * 4 * D + (p.parts > 1 && rows > 1 ? p.n_segs * D : 0);
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
  const int tpr = norm_tpr(a.D), slots = norm_slots(tpr);
  a.bias = a.b_post || a.b_pre;
  const long want = (a.R + slots - 1) / slots;
  const int top = norm_resident(tpr, norm_fwd_waves(d->dtype == HHRL_BF16 ? 2 : 4, vec ? 2 : 1));
  const int blocks = (int)(want < top ? want : top);
  a.step_m = (long)blocks * slots / a.H;
  a.step_j = (int)((long)blocks * slots % a.H);
  const double el = d->dtype == HHRL_BF16 ? 2.0 : 4.0;
  ProfScope ps("block_norm_fwd_kernel", as_stream(stream), 0.0, el * a.R * a.D * ((a.x != nullptr) + (a.y != nullptr) + (a.gate && !a.gate_bcast) + (a.out != nullptr) + (a.h != nullptr)));
  launch_norm(a, d->dtype, vec, tpr, blocks, false, as_stream(stream));
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
  const int tpr = norm_tpr(a.D), slots = norm_slots(tpr);
  a.bias = a.b_post || a.b_pre || d->db_post || d->db_pre;
  const NormParts p = norm_parts(d->M, d->H, a.gate_bcast ? d->gate_rows : 1, tpr, norm_bwd_waves(d->dtype == HHRL_BF16 ? 2 : 4, vec ? 2 : 1, a.bias));
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
  for (int q = 0; q < 4; ++q)
    for (int o = 0; o < q; ++o)
      HHRL_REQUIRE(!dst[q] || !dst[o] || dst[q] == dst[o] || dst[q] + a.D <= dst[o] || dst[o] + a.D <= dst[q],
                   "block_norm_backward: two parameter gradients overlap (they may be the same array)");
  a.par_ws = d->ws;
  a.gate_ws = fold_gate ? d->ws + (long)p.blocks * a.n_par * a.D : nullptr;
  const double el = d->dtype == HHRL_BF16 ? 2.0 : 4.0;
  {
    ProfScope ps("block_norm_bwd_kernel", as_stream(stream), 0.0,
                 el * a.R * a.D * ((a.x != nullptr) + (a.y != nullptr) + 2.0 * (a.gate && !a.gate_bcast) + (a.d_out != nullptr) + (a.d_h != nullptr) + (a.dx != nullptr) + (a.dy != nullptr)));
    launch_norm(a, d->dtype, vec, tpr, p.blocks, true, as_stream(stream));
  }
  HHRL_TRY(launch_status("block_norm_bwd_kernel"));
  if (!a.n_par && !fold_gate) return HHRL_OK;
  f.par_ws = a.par_ws; f.gate_ws = a.gate_ws; f.n_par = a.n_par; f.D = a.D; f.blocks = p.blocks; f.parts = p.parts;
  f.dgate = static_cast<float*>(a.dgate); f.lddg = a.lddg; f.n_groups = fold_gate ? p.n_groups : 0;
  const long jobs = f.n_par + f.n_groups;
  ProfScope ps("block_norm_fold_kernel", as_stream(stream), 0.0, 4.0 * need);
  hipLaunchKernelGGL(block_norm_fold_kernel, dim3(ceil_div(a.D, 32), (unsigned)(jobs < 4096 ? jobs : 4096)), dim3(1024), 0, as_stream(stream), f);
  return launch_status("block_norm_fold_kernel");
}

}  // extern "C"
