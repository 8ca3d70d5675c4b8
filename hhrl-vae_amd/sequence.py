"""Sequence layers beside the BiLSTM of `ops`: the gated delta rule (`GatedDelta`: a matrix state per head, whole
sequences forward and backward, one token per agent against a pool of states) and the norms before and after a block with
its gate and residual scale (`BlockNorm`).

Operands are torch tensors on the current device; every call enqueues on torch's current stream and returns at once.
Outputs, gradients and workspaces are the caller's: a call allocates nothing, so it can be recorded into a HIP graph.
What a call cannot take (type, shape, strides, device) raises ValueError before anything is launched; errors of the
library raise `_lib.HipError`.  A workspace belongs to one forward and its backward at a time: calls that may run at once
(two streams, two graphs) need one each.  Tensors that another stream writes or frees are ordered by the caller, as for
any torch operation."""
from __future__ import annotations

import ctypes as C
import struct
from typing import Optional

import torch

from . import _lib
from ._lib import ACT_NONE, ACT_SIGMOID, ACT_SILU, check

_DTYPES = {torch.float32: 0, torch.bfloat16: 1}            # HHRL_F32, HHRL_BF16
_NORMS = {"none": 0, "rms": 1, "layer": 2}                 # HHRL_NORM_*
# hhrl_gdr_step_desc: acting is bound by the host, and packing a struct takes a third of what setting its fields takes
_STEP = struct.Struct("@6ifi15q")
assert _STEP.size == C.sizeof(_lib.GdrStepDesc)
_GATES = {"none": ACT_NONE, "sigmoid": ACT_SIGMOID, "silu": ACT_SILU}


def _need(ok: bool, msg: str, *args) -> None:
    if not ok:
        raise ValueError(msg % args)


def _dtype_code(dtype) -> int:
    _need(dtype in _DTYPES, "dtype %s: float32 and bfloat16 are supported", dtype)
    return _DTYPES[dtype]


def _fail(name: str, t, shape, dtype, dev: int) -> None:
    """Says what is wrong with an operand that failed a check."""
    _need(isinstance(t, torch.Tensor), "%s is not a tensor", name)
    _need(tuple(t.shape) == tuple(shape), "%s has shape %s, not %s", name, tuple(t.shape), tuple(shape))
    _need(t.dtype == dtype, "%s is %s, not %s", name, t.dtype, dtype)
    _need(t.is_cuda, "%s is on %s, not on a GPU", name, t.device)
    _need(t.get_device() == dev, "%s is on %s, the current device is cuda:%d", name, t.device, dev)


def _tensor(name: str, t, shape, dtype, dev: int) -> int:
    """Checks a contiguous tensor of a given shape; its address."""
    try:
        bad = t.shape != shape or t.dtype is not dtype or t.get_device() != dev
    except AttributeError:
        bad = True
    if bad:
        _fail(name, t, shape, dtype, dev)
    _need(t.is_contiguous(), "%s is not contiguous", name)
    return t.data_ptr()


def _rows(name: str, t, shape, n: int, width: int, dtype, dev: int):
    """Checks a tensor whose first n dimensions are rows of `width` contiguous elements, at one distance from each other
    (a column range of a wider buffer qualifies): its address and that distance in elements."""
    try:
        bad = t.shape != shape or t.dtype is not dtype or t.get_device() != dev
    except AttributeError:
        bad = True
    if bad:
        _fail(name, t, shape, dtype, dev)
    if t.is_contiguous():
        return t.data_ptr(), width
    strides, inner = t.stride(), 1
    for size, stride in zip(reversed(shape[n:]), reversed(strides[n:])):
        _need(size == 1 or stride == inner, "%s: the elements of a row are not contiguous (strides %s)", name, strides)
        inner *= size
    ld, inner = None, 1                           # inner: rows below the dimension at hand
    for size, stride in zip(reversed(shape[:n]), reversed(strides[:n])):
        if size > 1:
            if ld is None and stride % inner == 0:
                ld = stride // inner
            _need(ld is not None and stride == ld * inner, "%s: its rows are not at one distance (strides %s)", name, strides)
        inner *= size
    ld = width if ld is None else ld
    _need(ld >= width, "%s: rows overlap (strides %s)", name, strides)
    return t.data_ptr(), ld


def _device() -> int:
    if not torch.cuda.is_initialized():
        _need(torch.cuda.is_available(), "no GPU")
        torch.cuda.init()
    return torch._C._cuda_getDevice()


def _stream(dev: int) -> int:
    """The raw stream that is current on a device (the current one, which a call has looked up already)."""
    return torch._C._cuda_getCurrentRawStream(dev)


class GatedDelta:
    """Shapes and scale of a gated delta rule layer: Hk key heads of K elements, Hv value heads of V elements (value head
    h reads key head h // (Hv // Hk)).  Per value head, with the log decay g_t <= 0 and the step size beta_t:

        S <- exp(g_t) S;   S <- S + beta_t k_t (v_t - S^T k_t)^T;   o_t = scale * S^T q_t       (scale: K ** -0.5)

    q, k, v, o and their gradients are `dtype`; g, beta, states and their gradients float32.  Sequences come as
    [B, T, heads, width] (`lens`: B int32 numbers of valid tokens, the rest of a row is padding) or packed as
    [rows, heads, width] with `starts` (n + 1 ascending int32 numbers; rows behind starts[n] belong to nobody).  Padding is
    neither read nor written."""

    def __init__(self, Hk: int, Hv: int, K: int, V: int, dtype=torch.float32, scale: Optional[float] = None):
        self.code = _dtype_code(dtype)
        _need(Hk > 0 and 0 < Hv < 1 << 31 and Hv % Hk == 0, "Hv=%d is not a multiple of Hk=%d", Hv, Hk)
        _need(0 < K <= _lib.GDR_MAX_K and 0 < V <= _lib.GDR_MAX_V, "K=%d V=%d: up to %d, %d supported", K, V, _lib.GDR_MAX_K, _lib.GDR_MAX_V)
        self.Hk, self.Hv, self.K, self.V, self.dtype = Hk, Hv, K, V, dtype
        self.scale = float(K) ** -0.5 if scale is None else float(scale)
        d = _lib.GdrDesc()                        # what every call of this layer has in common
        d.dtype, d.Hk, d.Hv, d.K, d.V, d.scale = self.code, Hk, Hv, K, V, self.scale
        self._common = bytes(d)
        self._lib = _lib.load()

    def workspace(self, n_seq: int, rows: int, device, packed: bool = True, no_backward: bool = False) -> torch.Tensor:
        """Workspace for n_seq sequences of `rows` tokens in all (of one padded length if not packed); what serves packed
        sequences serves as many padded ones too."""
        _need(0 < n_seq < 1 << 31 and 0 < rows < 1 << 31, "n_seq=%d rows=%d", n_seq, rows)
        n = self._lib.hhrl_gdr_workspace_floats(self.code, n_seq, rows, int(packed), self.Hk, self.Hv, self.K, self.V, int(no_backward))
        _need(n > 0, "no workspace for n_seq=%d rows=%d", n_seq, rows)
        return torch.empty(n, dtype=torch.float32, device=device)

    def _desc(self, q, k, v, g, beta, ws, starts, lens, dev):
        d = _lib.GdrDesc.from_buffer_copy(self._common)
        _need(isinstance(q, torch.Tensor), "q is not a tensor")
        if starts is not None:
            _need(lens is None, "starts and lens")
            if q.dim() != 3:
                _need(False, "packed q has shape %s, not [rows, Hk, K]", tuple(q.shape))
            lead = (q.shape[0],)
            rows = lead[0]
            _need(isinstance(starts, torch.Tensor) and starts.dim() == 1 and starts.numel() >= 2, "starts: n_seq + 1 numbers")
            n_seq = starts.numel() - 1
            d.starts = _tensor("starts", starts, (n_seq + 1,), torch.int32, dev)
        else:
            if q.dim() != 4:
                _need(False, "q has shape %s, not [B, T, Hk, K]", tuple(q.shape))
            lead = tuple(q.shape[:2])
            n_seq, rows = lead[0], lead[0] * lead[1]
            if lens is not None:
                d.lens = _tensor("lens", lens, (n_seq,), torch.int32, dev)
        _need(rows > 0, "no tokens")
        n = len(lead)
        key, val, head = (lead + (self.Hk, self.K), n, self.Hk * self.K, self.dtype, dev), \
            (lead + (self.Hv, self.V), n, self.Hv * self.V, self.dtype, dev), (lead + (self.Hv,), n, self.Hv, torch.float32, dev)
        d.n_seq, d.rows = n_seq, rows
        d.q, d.ldq = _rows("q", q, *key)
        d.k, d.ldk = _rows("k", k, *key)
        d.v, d.ldv = _rows("v", v, *val)
        d.g, d.ldg = _rows("g", g, *head)
        d.beta, d.ldbeta = _rows("beta", beta, *head)
        _need(isinstance(ws, torch.Tensor), "ws is not a tensor")
        d.ws_floats = ws.numel()
        d.ws = _tensor("ws", ws, (d.ws_floats,), torch.float32, dev)
        return d, n_seq, key, val, head

    def _state(self, name, t, n_seq, dev):
        return _tensor(name, t, (n_seq, self.Hv, self.K, self.V), torch.float32, dev) if t is not None else None

    def fwd(self, q, k, v, g, beta, o, ws, s0=None, s1=None, starts=None, lens=None, no_backward: bool = False) -> None:
        """Writes o and, where given, s1 (states behind the sequences, from s0 or zero; may be s0).  Leaves in ws what `bwd`
        of the same inputs reads, unless no_backward."""
        dev = _device()
        d, n, _, val, _ = self._desc(q, k, v, g, beta, ws, starts, lens, dev)
        d.o, d.ldo = _rows("o", o, *val)
        d.s0, d.s1 = self._state("s0", s0, n, dev), self._state("s1", s1, n, dev)
        d.no_backward = int(no_backward)
        check(self._lib.hhrl_gdr_forward(C.byref(d), _stream(dev)))

    def bwd(self, q, k, v, g, beta, d_o, dq, dk, dv, dg, dbeta, ws, d_s1=None, d_s0=None, starts=None, lens=None) -> None:
        """Gradients of <d_o, o> + <d_s1, s1> (either None: absent), written to dq, dk, dv, dg, dbeta and d_s0; ws as the
        forward call of the same inputs left it (where the last one in it was of other shapes, or with no_backward, every
        gradient is NaN).  d_s0 may be d_s1."""
        dev = _device()
        d, n, key, val, head = self._desc(q, k, v, g, beta, ws, starts, lens, dev)
        if d_o is not None:
            d.d_o, d.lddo = _rows("d_o", d_o, *val)
        d.d_s1, d.d_s0 = self._state("d_s1", d_s1, n, dev), self._state("d_s0", d_s0, n, dev)
        d.dq, d.lddq = _rows("dq", dq, *key)
        d.dk, d.lddk = _rows("dk", dk, *key)
        d.dv, d.lddv = _rows("dv", dv, *val)
        d.dg, d.lddg = _rows("dg", dg, *head)
        d.dbeta, d.lddbeta = _rows("dbeta", dbeta, *head)
        check(self._lib.hhrl_gdr_backward(C.byref(d), _stream(dev)))

    def step(self, q, k, v, g, beta, o, state, state_out=None, slots=None) -> None:
        """One token for each of B rows (q, k [B, Hk, K], v, o [B, Hv, V], g, beta [B, Hv]) against a pool of states
        [n, Hv, K, V]: row b moves state slots[b] (None: state b) into state_out (None: in place).  A negative slot: the
        row is idle, its output 0.  A slot past the pool, or one that an earlier row names: output NaN, no state moves."""
        dev = _device()
        _need(isinstance(q, torch.Tensor) and q.dim() == 3, "q is not [B, Hk, K]")
        _need(isinstance(state, torch.Tensor) and state.dim() == 4, "state is not [n, Hv, K, V]")
        B, n = q.shape[0], state.shape[0]
        _need(B > 0 and n > 0, "%d rows for %d states", B, n)
        Hk, Hv, K, V, dt = self.Hk, self.Hv, self.K, self.V, self.dtype
        key, val, head = ((B, Hk, K), 1, Hk * K, dt, dev), ((B, Hv, V), 1, Hv * V, dt, dev), ((B, Hv), 1, Hv, torch.float32, dev)
        sp = self._state("state", state, n, dev)
        so = sp if state_out is None else self._state("state_out", state_out, n, dev)
        sl = 0
        if slots is not None:
            sl = _tensor("slots", slots, (B,), torch.int32, dev)
        else:
            _need(B <= n, "%d rows for %d states", B, n)
        qp, ldq = _rows("q", q, *key)
        kp, ldk = _rows("k", k, *key)
        vp, ldv = _rows("v", v, *val)
        gp, ldg = _rows("g", g, *head)
        bp, ldb = _rows("beta", beta, *head)
        op, ldo = _rows("o", o, *val)
        check(self._lib.hhrl_gdr_step(_STEP.pack(self.code, B, Hk, Hv, K, V, self.scale, n, qp, kp, vp, ldq, ldk, ldv, gp, bp, ldg, ldb,
                                                 op, ldo, sp, so, sl), _stream(dev)))


class BlockNorm:
    """Norms after a block (`post`) and before the next (`pre`) with the block's gate and residual scale:

        r = alpha * x + scale * a(gate) * post(y);    h = pre(r)

    per group of D elements (H groups per row), in one pass over the rows.  post, pre: "none", "rms", "layer", each with
    optional float32 weight and bias [D]; gate_act a: "none", "sigmoid", "silu".  x, y, gate, out (r), h and their gradients
    are `dtype`, [M, H, D], or [M, D] if H is 1; with gate_rows > 1 (H 1) the gate is float32 [ceil(M / gate_rows), D], a row
    for every gate_rows rows of x.  Without x there is no residual stream, without y only the norm in front of a block."""

    PARAMS = ("w_post", "b_post", "w_pre", "b_pre")

    def __init__(self, D: int, H: int = 1, post: str = "none", pre: str = "none", gate_act: str = "none", gate_rows: int = 1,
                 alpha: float = 1.0, scale: float = 1.0, eps: float = 1e-6, dtype=torch.float32):
        self.code = _dtype_code(dtype)
        _need(post in _NORMS and pre in _NORMS, "norms %r, %r: none, rms or layer", post, pre)
        _need(gate_act in _GATES, "gate_act %r: none, sigmoid or silu", gate_act)
        _need(0 < D <= 8192 and 0 < H < 1 << 31, "H=%d D=%d: D up to 8192", H, D)
        _need(1 <= gate_rows < 1 << 63 and (gate_rows == 1 or H == 1), "gate_rows=%d with H=%d", gate_rows, H)
        _need(eps >= 0, "eps=%g", eps)
        self.D, self.H, self.post, self.pre, self.gate_act, self.gate_rows = D, H, post, pre, gate_act, gate_rows
        self.alpha, self.scale, self.eps, self.dtype = float(alpha), float(scale), float(eps), dtype
        d = _lib.BlockNormDesc()                  # what every call of this plan has in common
        d.dtype, d.H, d.D = self.code, H, D
        d.post, d.pre, d.gate_act, d.gate_rows = _NORMS[post], _NORMS[pre], _GATES[gate_act], gate_rows
        d.alpha, d.scale, d.eps = self.alpha, self.scale, self.eps
        self._common = bytes(d)
        self._lib = _lib.load()

    def workspace(self, M: int, device) -> torch.Tensor:
        """Workspace of `bwd` for M rows."""
        _need(0 < M < 1 << 40, "M=%d", M)
        n = self._lib.hhrl_block_norm_workspace_floats(M, self.H, self.D, self.gate_rows)
        _need(n > 0, "no workspace for M=%d", M)
        return torch.empty(n, dtype=torch.float32, device=device)

    def _shape(self, first, M, dev):
        """What an activation of M rows has to look like: as [M, H, D], or [M, D] if that is how the first one comes."""
        flat = self.H == 1 and isinstance(first, torch.Tensor) and first.dim() == 2
        return ((M, self.D) if flat else (M, self.H, self.D), 1, self.H * self.D, self.dtype, dev)

    def _gate_shape(self, t, M, act, dev):
        if self.gate_rows == 1:
            return act
        n = -(-M // self.gate_rows)
        return ((n, self.D) if isinstance(t, torch.Tensor) and t.dim() == 2 else (n, 1, self.D), 1, self.D, torch.float32, dev)

    def _desc(self, x, y, gate, params, dev):
        d = _lib.BlockNormDesc.from_buffer_copy(self._common)
        first = x if x is not None else y
        _need(isinstance(first, torch.Tensor) and first.dim() > 0, "neither x nor y")
        M = first.shape[0]
        _need(M > 0, "no rows")
        _need(y is not None or (gate is None and self.post == "none"), "a gate or a post norm without y")
        act = self._shape(first, M, dev)
        d.M = M
        if x is not None:
            d.x, d.ldx = _rows("x", x, *act)
        if y is not None:
            d.y, d.ldy = _rows("y", y, *act)
        if gate is not None:
            d.gate, d.ldgate = _rows("gate", gate, *self._gate_shape(gate, M, act, dev))
        w_post, b_post, w_pre, b_pre = params
        if w_post is not None or b_post is not None:
            _need(self.post != "none", "parameters without a post norm")
            if w_post is not None:
                d.w_post = _tensor("w_post", w_post, (self.D,), torch.float32, dev)
            if b_post is not None:
                d.b_post = _tensor("b_post", b_post, (self.D,), torch.float32, dev)
        if w_pre is not None or b_pre is not None:
            _need(self.pre != "none", "parameters without a pre norm")
            if w_pre is not None:
                d.w_pre = _tensor("w_pre", w_pre, (self.D,), torch.float32, dev)
            if b_pre is not None:
                d.b_pre = _tensor("b_pre", b_pre, (self.D,), torch.float32, dev)
        return d, M, act

    def fwd(self, x=None, y=None, gate=None, w_post=None, b_post=None, w_pre=None, b_pre=None, out=None, h=None) -> None:
        """Writes r to out and pre(r) to h (either may be None; both may be x or y)."""
        dev = _device()
        d, M, act = self._desc(x, y, gate, (w_post, b_post, w_pre, b_pre), dev)
        _need(out is not None or h is not None, "neither out nor h")
        _need(self.pre == "none" or h is not None, "a pre norm without h")
        if out is not None:
            d.out, d.ldo = _rows("out", out, *act)
        if h is not None:
            d.h, d.ldh = _rows("h", h, *act)
        check(self._lib.hhrl_block_norm_forward(C.byref(d), _stream(dev)))

    def bwd(self, x=None, y=None, gate=None, w_post=None, b_post=None, w_pre=None, b_pre=None, d_out=None, d_h=None,
            dx=None, dy=None, dgate=None, dw_post=None, db_post=None, dw_pre=None, db_pre=None, ws=None) -> None:
        """Gradients of <d_out, r> + <d_h, h> (either None: absent) from the forward call's inputs: dx, dy, dgate are
        written, parameter gradients added to (two may be one tensor: it gets both); those that are None are skipped.  ws:
        needed for parameter gradients and for the gradient of a gate with gate_rows > 1."""
        dev = _device()
        d, M, act = self._desc(x, y, gate, (w_post, b_post, w_pre, b_pre), dev)
        _need(d_out is not None or d_h is not None, "neither d_out nor d_h")
        for name, t, of in (("dx", dx, x), ("dy", dy, y), ("dgate", dgate, gate)):
            _need(t is None or of is not None, "%s without %s", name, name[1:])
        if d_out is not None:
            d.d_out, d.lddo = _rows("d_out", d_out, *act)
        if d_h is not None:
            d.d_h, d.lddh = _rows("d_h", d_h, *act)
        if dx is not None:
            d.dx, d.lddx = _rows("dx", dx, *act)
        if dy is not None:
            d.dy, d.lddy = _rows("dy", dy, *act)
        if dgate is not None:
            d.dgate, d.lddgate = _rows("dgate", dgate, *self._gate_shape(dgate, M, act, dev))
        for name, t in zip(self.PARAMS, (dw_post, db_post, dw_pre, db_pre)):
            if t is not None:
                _need(getattr(self, name[2:]) != "none" and (name[2:] == "post" or d_h is not None), "d%s without its norm", name)
                setattr(d, "d" + name, _tensor("d" + name, t, (self.D,), torch.float32, dev))
        if ws is not None:
            _need(isinstance(ws, torch.Tensor), "ws is not a tensor")
            d.ws_floats = ws.numel()
            d.ws = _tensor("ws", ws, (d.ws_floats,), torch.float32, dev)
        check(self._lib.hhrl_block_norm_backward(C.byref(d), _stream(dev)))
