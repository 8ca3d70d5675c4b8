"""Orders of calls and contents that the sequence layers have to answer or to mark: a backward call without its forward,
non-finite numbers in a token, and gradients against differences along themselves."""
import math

import pytest
import torch

import seq_reference as R

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
F32, BF = torch.float32, torch.bfloat16


@pytest.fixture(scope="module")
def seq():
    from hhrl_vae_amd import sequence
    return sequence


def make(lead, Hk, Hv, K, V, dtype, seed):
    gen = torch.Generator().manual_seed(seed)
    rn = lambda *s: torch.randn(*s, generator=gen)
    unit = lambda t: (t / t.norm(dim=-1, keepdim=True)).to(dtype)
    return [unit(rn(*lead, Hk, K)), unit(rn(*lead, Hk, K)), rn(*lead, Hv, V).to(dtype), -torch.rand(*lead, Hv, generator=gen) ** 2,
            torch.sigmoid(rn(*lead, Hv)), rn(*lead, Hv, V).to(dtype)]


@pytest.mark.parametrize("dtype", [F32, BF])
@pytest.mark.parametrize("K,V,T,Hk,Hv", [(64, 64, 100, 1, 2), (128, 40, 70, 2, 2), (64, 32, 3333, 1, 1)])
def test_gdr_backward_without_its_forward_is_marked(seq, dtype, K, V, T, Hk, Hv):
    """A workspace that holds no forward pass of these shapes for the backward pass (none at all, one with no_backward, one of
    other sequences): every gradient is NaN, rows of nobody stay; after the forward pass it is what it always is."""
    ins = [t.to(DEV) for t in make((T + 3,), Hk, Hv, K, V, dtype, T)]
    *ins, d_o = ins
    layer = seq.GatedDelta(Hk, Hv, K, V, dtype=dtype)
    starts = torch.tensor([0, T // 2, T // 2, T], dtype=torch.int32, device=DEV)
    other = torch.tensor([0, T], dtype=torch.int32, device=DEV)
    d_s1 = torch.randn(3, Hv, K, V, generator=torch.Generator().manual_seed(0)).to(DEV)

    def bwd(ws):
        grads, d_s0 = [torch.full_like(t, 7.0) for t in ins], torch.full_like(d_s1, 7.0)
        layer.bwd(*ins, d_o, *grads, ws, d_s1=d_s1, d_s0=d_s0, starts=starts)
        return grads + [d_s0]
    ws, o = layer.workspace(3, T + 3, DEV), torch.empty_like(ins[2])
    ws.fill_(float("nan"))
    layer.fwd(*ins, o, ws, starts=starts)
    want = bwd(ws)
    for t in want:
        assert bool(torch.isfinite(t).all())
    for t, again in zip(want, bwd(ws)):                       # a second backward pass finds the same workspace
        assert torch.equal(t, again)

    def nothing(w):
        w.zero_()

    def without(w):
        layer.fwd(*ins, o, w, starts=starts)
        layer.fwd(*ins, o, w, starts=starts, no_backward=True)

    def others(w):
        layer.fwd(*ins, o, w, starts=other)
    for before in (nothing, without, others):
        before(ws)
        for i, t in enumerate(bwd(ws)):
            if i < 5:
                assert bool(torch.isnan(t[:T]).all()), (before.__name__, i)
                assert bool((t[T:] == 7.0).all()), (before.__name__, i)
            else:
                assert bool(torch.isnan(t).all()), before.__name__
    layer.fwd(*ins, o, ws, starts=starts)
    for t, again in zip(want, bwd(ws)):
        assert torch.equal(t, again)


@pytest.mark.parametrize("dtype", [F32, BF])
@pytest.mark.parametrize("bad", [math.inf, math.nan])
@pytest.mark.parametrize("which", ["q", "k", "v", "beta", "d_o"])
def test_gdr_non_finite_numbers_stay_in_their_sequence_and_head(seq, dtype, bad, which):
    """One element of one token of the middle sequence's second chunk: other sequences, other key heads and (forward) the chunks
    before it keep their bits; what the definition says is non-finite is (the output of that token or its gradients)."""
    lens, Hk, Hv, K, V = [70, 200, 65], 2, 4, 64, 40
    rows, at = sum(lens), 70 + 64 + 30
    ins = [t.to(DEV) for t in make((rows,), Hk, Hv, K, V, dtype, 5)]
    starts = torch.tensor([0, 70, 270, 335], dtype=torch.int32, device=DEV)
    layer = seq.GatedDelta(Hk, Hv, K, V, dtype=dtype)
    ws = layer.workspace(3, rows, DEV)

    def go(a):
        o, s1, ds0 = torch.empty_like(a[2]), torch.empty(3, Hv, K, V, device=DEV), torch.empty(3, Hv, K, V, device=DEV)
        grads = [torch.empty_like(t) for t in a[:5]]
        layer.fwd(*a[:5], o, ws, s1=s1, starts=starts)
        layer.bwd(*a[:5], a[5], *grads, ws, d_s0=ds0, starts=starts)
        return o, s1, grads, ds0
    clean = go(ins)
    i = ("q", "k", "v", "g", "beta", "d_o").index(which)
    spoilt = list(ins)
    spoilt[i] = ins[i].clone()
    if which in ("q", "k"):
        spoilt[i][at, 1, 3] = bad
        heads, keys = [2, 3], [1]                              # the value heads of key head 1
    elif which == "beta":
        spoilt[i][at, 2] = bad
        heads, keys = [2], [1]
    else:
        spoilt[i][at, 2, 3] = bad
        heads, keys = [2], [1]
    got = go(spoilt)
    o, s1, grads, ds0 = got
    co, cs1, cgrads, cds0 = clean
    out = [r for r in range(rows) if not 70 <= r < 270]
    safe = [h for h in range(Hv) if h not in heads]
    safe_k = [h for h in range(Hk) if h not in keys]
    for a, b in [(o, co)] + list(zip(grads, cgrads)):
        assert torch.equal(a[out], b[out])
        free = safe_k if a.shape[1] == Hk else safe
        assert torch.equal(a[:, free], b[:, free])
    for a, b in ((s1, cs1), (ds0, cds0)):
        assert torch.equal(a[[0, 2]], b[[0, 2]]) and torch.equal(a[:, safe], b[:, safe])
    assert torch.equal(o[: 70 + 64], co[: 70 + 64])            # the chunk in front of the spoilt one
    if which == "d_o":
        assert torch.equal(o, co) and torch.equal(s1, cs1)
        assert not bool(torch.isfinite(grads[0][at, 1]).all())
    elif which == "q":
        assert torch.equal(s1, cs1)
        assert not bool(torch.isfinite(o[at, heads]).all())
    else:
        assert not bool(torch.isfinite(o[at + 1, heads]).all()) and not bool(torch.isfinite(s1[1, heads]).all())


def loss64(ins, d_o, scale):
    o, _ = R.gdr(*ins, scale, torch.zeros(ins[2].shape[1], ins[0].shape[2], ins[2].shape[2], dtype=torch.float64))
    return (o * d_o).sum()


def directions(Hk, Hv, K, V, T, h):
    """fp32 operands, the 64-bit loss's gradient for each, the unit step along it, and how far the 64-bit difference quotient is
    from the 64-bit derivative (what the finite step costs)."""
    ins = [t[0] for t in make((1, T), Hk, Hv, K, V, F32, 11)]
    *ins, d_o = ins
    ins[3] = ins[3] - 0.25                                    # log decays stay below 0 on either side
    leaves = [t.double().requires_grad_(True) for t in ins]
    loss64(leaves, d_o.double(), K ** -0.5).backward()
    steps, slope, cost = [], [], []
    for i, leaf in enumerate(leaves):
        step = leaf.grad / leaf.grad.norm()
        lo, hi = ([t.detach() for t in leaves] for _ in range(2))
        # the operands as the kernels get them, rounded to fp32
        lo[i], hi[i] = (lo[i] - h * step).float().double(), (hi[i] + h * step).float().double()
        quotient = float(loss64(hi, d_o.double(), K ** -0.5) - loss64(lo, d_o.double(), K ** -0.5)) / (2 * h)
        slope.append(float((leaf.grad * step).sum()))
        cost.append(abs(quotient - slope[-1]))
        steps.append(step)
    return ins, d_o, steps, slope, cost


def test_gdr_gradient_against_differences_along_itself(seq):
    """The difference of two losses along the gradient's own direction, fp32.  The tolerance: the loss's rounding (path u
    times its terms' sizes, twice) over 2h, and what the step costs in 64 bits; at most a twentieth of the derivative."""
    Hk, Hv, K, V, T, h = 1, 2, 24, 20, 90, 0.25
    ins, d_o, steps, slope, cost = directions(Hk, Hv, K, V, T, h)
    layer = seq.GatedDelta(Hk, Hv, K, V)
    ws = layer.workspace(1, T, DEV)
    dev, dd = [t[None].to(DEV) for t in ins], d_o[None].to(DEV)
    o = torch.empty_like(dev[2])

    def loss(args):
        layer.fwd(*args, o, ws)
        t = o.double() * dd.double()
        return float(t.sum()), float(t.abs().sum())
    layer.fwd(*dev, o, ws)
    grads = [torch.empty_like(t) for t in dev]
    layer.bwd(*dev, dd, *grads, ws)
    path = 2 * (K + V + 3 * 64 + 5 * (T // 64 + 1))
    for i, step in enumerate(steps):
        lo, hi = list(dev), list(dev)
        lo[i], hi[i] = ((ins[i].double() + s * h * step).float()[None].to(DEV) for s in (-1, 1))
        (a, size), (b, _) = loss(lo), loss(hi)
        got = float((grads[i][0].cpu().double() * step).sum())
        tol = path * R.U32 * size / h + cost[i]
        assert slope[i] >= 20 * tol, (i, slope[i], tol)
        assert abs((b - a) / (2 * h) - got) <= tol, (i, (b - a) / (2 * h), got, tol)
