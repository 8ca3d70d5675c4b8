"""The sequence layers in 64 bits, straight from their definitions (CPU, autograd): what the kernels are held to.

Tolerances: fp32 results may be off by gamma_n * scale, gamma_n = n * 2^-24, where n counts the roundings on the longest
path to the result (every term of a sum is one) and scale is the largest number of its kind in the tensor, or the size
of the terms that cancel in it where the caller gives one; results in bf16 are rounded once more, by at most 2^-8 of themselves."""
import torch

U32, UBF = 2.0 ** -24, 2.0 ** -8


def gdr(q, k, v, g, beta, scale, s0):
    """One sequence: q, k [T, Hk, K], v [T, Hv, V], g, beta [T, Hv], s0 [Hv, K, V] (all fp64) -> o, s1."""
    rep = v.shape[1] // q.shape[1]
    S, out = s0, []
    for t in range(q.shape[0]):
        qt, kt = (x[t].repeat_interleave(rep, dim=0) for x in (q, k))
        S = S * g[t].exp()[:, None, None]
        u = beta[t][:, None] * (v[t] - (S * kt[:, :, None]).sum(1))
        S = S + kt[:, :, None] * u[:, None, :]
        out.append(scale * (S * qt[:, :, None]).sum(1))
    return (torch.stack(out) if out else v[:0]), S


def gdr_batch(ranges, q, k, v, g, beta, scale, s0):
    """Sequences as row ranges of [rows, ...] -> o [rows, ...] (zero where nobody's), s1 [n, ...]."""
    o, states = torch.zeros_like(v), []
    for n, (a, b) in enumerate(ranges):
        y, S = gdr(q[a:b], k[a:b], v[a:b], g[a:b], beta[a:b], scale, s0[n])
        o = torch.cat([o[:a], y, o[b:]])
        states.append(S)
    return o, torch.stack(states)


def norm(t, kind, w, b, eps):
    if kind == "none":
        return t
    if kind == "layer":
        t = t - t.mean(-1, keepdim=True)
    t = t / ((t * t).mean(-1, keepdim=True) + eps).sqrt()
    if w is not None:
        t = t * w
    return t if b is None else t + b


def block_norm(x, y, gate, w_post, b_post, w_pre, b_pre, post, pre, gate_act, gate_rows, alpha, scale, eps):
    """x, y [M, H, D], gate [M, H, D] or [ceil(M / gate_rows), 1, D] -> r, h."""
    r = 0.0
    if x is not None:
        r = alpha * x
    if y is not None:
        b = norm(y, post, w_post, b_post, eps) * scale
        if gate is not None:
            a = {"none": lambda z: z, "sigmoid": torch.sigmoid, "silu": lambda z: z * torch.sigmoid(z)}[gate_act](gate)
            b = b * a[torch.arange(y.shape[0]) // gate_rows]
        r = r + b
    return r, norm(r, pre, w_pre, b_pre, eps)


def close(name, got, want, n, where=None, size=0.0):
    """got (kernel) against want (fp64): gamma_n of the largest number, and one rounding to got's type."""
    got64 = got.detach().cpu().double()
    assert got64.shape == want.shape, (name, got64.shape, want.shape)
    if where is not None:
        got64, want = got64[where], want[where]
    if not want.numel():
        return
    scale = max(float(want.abs().max()), size)
    tol = n * U32 * scale + (UBF * want.abs() if got.dtype == torch.bfloat16 else 0.0) + 1e-37
    off = (got64 - want).abs()
    assert bool((off <= tol).all()), "%s: off by %g at scale %g (gamma %g)" % (name, float(off.max()), scale, n * U32)
