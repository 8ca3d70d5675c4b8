"""What the sequence layers' results carry: sums, decays and gates of fp32 accuracy for either type, on inputs whose
results show a rounding to fewer bits (differences of equal numbers, decays far from 1), against 64 bits.

u = 2^-24.  The matrix instruction's sums are counted with a whole last place (2 u) for every term that is not zero."""
import math

import pytest
import torch

import seq_reference as R

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
F32, BF = torch.float32, torch.bfloat16
U, UBF = R.U32, R.UBF


@pytest.fixture(scope="module")
def seq():
    from hhrl_vae_amd import sequence
    return sequence


def pairs(T, K, seed):
    """For every token two different rows of k that have been written by then (token 0: the first against nothing)."""
    gen = torch.Generator().manual_seed(seed)
    q = torch.zeros(T, K)
    for t in range(T):
        a = int(torch.randint(0, min(t + 1, K), (1,), generator=gen))
        b = int(torch.randint(0, min(t + 1, K), (1,), generator=gen))
        q[t, a] += 1
        q[t, b] -= 1
    return q


@pytest.mark.parametrize("dtype", [F32, BF])
@pytest.mark.parametrize("K", [64, 128])
@pytest.mark.parametrize("V", [32, 40])
@pytest.mark.parametrize("what", ["state", "tokens", "decays"])
def test_gdr_output_is_a_difference_of_fp32_numbers(seq, dtype, K, V, what):
    """o = a - b with a and b of size 1 that differ by 2^-12 and less, where a and b are rows of the state, what two tokens
    of the chunk have added (beta), or two tokens' decays.  Off by at most: three terms of each number, six sums of
    at most 2 u; the decays 4 u each (exponential 2 u, its correction u, product with q.k u); and o's own rounding."""
    T = 64
    gen = torch.Generator().manual_seed(K + V)
    fine = lambda *s: torch.randint(0, 1 << 11, s, generator=gen).float() * 2.0 ** -24
    q, k, v = pairs(T, K, V), torch.zeros(T, K), torch.ones(T, V)
    g, beta, s0 = torch.zeros(T), torch.zeros(T), torch.zeros(K, V)
    if what == "state":
        s0 = 0.5 + 0.4 * torch.rand(1, V, generator=gen) + fine(K, V)
    else:
        k[torch.arange(T), torch.arange(T)] = 1.0
        beta = 0.8371 + fine(T) if what == "tokens" else torch.ones(T)
        if what == "decays":
            g = -torch.rand(T, generator=gen) * 2.0 ** -13
            g[0] = -0.37
    want, _ = R.gdr(q[:, None].double(), k[:, None].double(), v[:, None].double(), g[:, None].double(), beta[:, None].double(), 1.0, s0[None].double())
    layer = seq.GatedDelta(1, 1, K, V, dtype=dtype, scale=1.0)
    dev = [t[None, :, None].to(dtype).to(DEV) for t in (q, k, v)] + [t[None, :, None].to(DEV) for t in (g, beta)]
    for back in (False, True):
        o = torch.empty_like(dev[2])
        layer.fwd(*dev, o, layer.workspace(1, T, DEV, no_backward=not back), s0=s0[None, None].to(DEV), no_backward=not back)
        off = (o[0].cpu().double() - want).abs()
        tol = 20 * U + (UBF if dtype is BF else 0.0) * want.abs()
        assert bool((off <= tol).all()), "off by %g u" % float(((off - tol) / U).max())


@pytest.mark.parametrize("T", [64, 150])
def test_gdr_decays_far_from_one(seq, T):
    """One token is written and every later one reads it through the decays in between, down to 2^-120: results are one
    product of decays each and carry a relative accuracy.  Inside a chunk: the decay 4 u (its exponential 2, the
    correction 1, the sums behind its argument less than 1), its product with q.k 1, three terms 3, scale 1.  Behind it: the
    decays of the first chunk's end, of the chunks between and of the token, 4 each and 2 for the product, six sums of at most 2.
    And 2^-124: a term of a number is lost where it is below the least normal bf16 number, 2^-126 (the third term of a number
    below 2^-109), which is up to 2^-126 for each number that is split: P or R, or tail W and S, and half of that for W."""
    gen = torch.Generator().manual_seed(T)
    g = -2 * 80.0 / T * torch.rand(T, generator=gen)
    g[1::2] *= 1.0 + 2.0 ** -11
    q, k = torch.zeros(T, 8), torch.zeros(T, 8)
    q[:, 3] = k[0, 3] = 1.0
    beta, v, d_o = torch.zeros(T), torch.ones(T, 1), torch.ones(T, 1)
    beta[0] = 1.0
    G = g.double().cumsum(0)
    want = (G - G[0]).exp()
    layer = seq.GatedDelta(1, 1, 8, 1, scale=1.0)
    dev = [t[None, :, None].contiguous().to(DEV) for t in (q, k, v, g, beta)]
    ws, o = layer.workspace(1, T, DEV), torch.empty(1, T, 1, 1, device=DEV)
    layer.fwd(*dev, o, ws)
    grads = [torch.empty_like(t) for t in dev]
    layer.bwd(*dev, d_o[None, :, None].contiguous().to(DEV), *grads, ws)
    n = 12 if T <= 64 else 12 + 6 * (T // 64)
    for name, got in (("o", o), ("dq", grads[0][..., 3])):          # dq_t = S_t d_o: the same numbers
        off = (got.flatten().cpu().double() - want).abs()
        assert bool((off <= n * U * want + 2.0 ** -124).all()), "%s: %g u" % (name, float((off / want).max() / U))


@pytest.mark.parametrize("dtype", [F32, BF])
@pytest.mark.parametrize("act", ["sigmoid", "silu"])
def test_block_norm_fp32_results_of_gates(seq, dtype, act):
    """A shared gate, its gradient and those of the parameters are fp32 for either type.  Gates down to -80, results of one
    row: sigmoid 6 u (exponential 2, sum 1, quotient 1, argument exact), its slope s (1 - s) 3 more, the products with
    scale, w, n and d_out 5, silu's slope 2: relative, where the factor next to s is of one sign."""
    D = 512
    gen = torch.Generator().manual_seed(1)
    gate = -80 * torch.rand(1, D, generator=gen) - 3.0
    y, d_out = (torch.randn(2, D, generator=gen).to(dtype) for _ in range(2))
    d_out[1] = 0                                                     # two rows share the gate, one of them counts
    plan = seq.BlockNorm(D, gate_act=act, gate_rows=2, dtype=dtype)
    dgate, dy = torch.empty(1, D, device=DEV), torch.empty(2, D, dtype=dtype, device=DEV)
    ws = plan.workspace(2, DEV)
    plan.bwd(y=y.to(DEV), gate=gate.to(DEV), d_out=d_out.to(DEV), dgate=dgate, dy=dy, ws=ws)
    z = gate.double().requires_grad_(True)
    s = torch.sigmoid(z)
    (s if act == "sigmoid" else z * s).sum().backward()
    want = (z.grad * y[:1].double() * d_out[:1].double()).detach()
    assert bool(((dgate.cpu().double() - want).abs() <= 16 * U * want.abs() + 1e-37).all()), float(((dgate.cpu().double() - want).abs() / want.abs()).max() / U)
    # the gradient of the norm's bias: scale * value of the gate * d_out, of one row
    plan = seq.BlockNorm(D, post="rms", gate_act=act, gate_rows=2, dtype=dtype)
    db, b = torch.zeros(D, device=DEV), torch.zeros(D, device=DEV)
    plan.bwd(y=y.to(DEV), gate=gate.to(DEV), b_post=b, d_out=d_out.to(DEV), db_post=db, ws=plan.workspace(2, DEV))
    want = ((s if act == "sigmoid" else z * s).detach() * d_out[:1].double())[0]
    assert bool(((db.cpu().double() - want).abs() <= 16 * U * want.abs() + 1e-37).all()), float(((db.cpu().double() - want).abs() / want.abs()).max() / U)


@pytest.mark.parametrize("dtype", [F32, BF])
@pytest.mark.parametrize("act", ["sigmoid", "silu"])
def test_block_norm_parameter_gradients_behind_a_gate_per_element(seq, dtype, act):
    """The same for a gate with an element for every element: db_post of one row."""
    D = 520
    gen = torch.Generator().manual_seed(2)
    gate = (-80 * torch.rand(1, D, generator=gen) - 3.0).to(dtype)
    y, d_out = (torch.randn(1, D, generator=gen).to(dtype) for _ in range(2))
    plan = seq.BlockNorm(D, post="rms", gate_act=act, dtype=dtype)
    db, b = torch.zeros(D, device=DEV), torch.zeros(D, device=DEV)
    plan.bwd(y=y.to(DEV), gate=gate.to(DEV), b_post=b, d_out=d_out.to(DEV), db_post=db, ws=plan.workspace(1, DEV))
    z = gate.double()
    want = ((torch.sigmoid(z) if act == "sigmoid" else z * torch.sigmoid(z)) * d_out.double())[0]
    assert bool(((db.cpu().double() - want).abs() <= 16 * U * want.abs() + 1e-37).all()), float(((db.cpu().double() - want).abs() / want.abs()).max() / U)


@pytest.mark.parametrize("dtype", [F32, BF])
@pytest.mark.parametrize("gate_rows", [1, 2])
def test_block_norm_gates_at_the_ends(seq, dtype, gate_rows):
    """Gates that are no number stay none, infinite and very large ones give 0, 1 and themselves, and slopes of 0."""
    vals = torch.tensor([math.nan, math.inf, -math.inf, 200.0, -200.0, 88.5, -88.5, 0.0] * 8)
    D = vals.numel()
    y = torch.ones(1, D, dtype=dtype, device=DEV)
    gate = vals[None].to(DEV) if gate_rows > 1 else vals[None].to(dtype).to(DEV)
    for act in ("sigmoid", "silu"):
        plan = seq.BlockNorm(D, gate_act=act, gate_rows=gate_rows, dtype=dtype)
        out, dgate = torch.empty_like(y), torch.empty_like(gate)
        plan.fwd(y=y, gate=gate, out=out)
        plan.bwd(y=y, gate=gate, d_out=y, dgate=dgate, ws=plan.workspace(1, DEV))
        o, d = out.float().cpu()[0], dgate.float().cpu()[0]
        assert bool(torch.isnan(o[0::8]).all()) and bool(torch.isnan(d[0::8]).all())
        # 88.5 and -200 are multiples of their own last places in bf16 too
        want = torch.tensor([1.0, 0.0, 1.0, 0.0, 1.0, 0.0, 0.5] if act == "sigmoid" else [math.inf, math.nan, 200.0, 0.0, 88.5, 0.0, 0.0])
        slope = torch.tensor([0.0, 0.0, 0.0, 0.0, 0.0, 0.0, 0.25] if act == "sigmoid" else [math.nan, math.nan, 1.0, 0.0, 1.0, 0.0, 0.5])
        for got, ref in ((o, want), (d, slope)):
            for i in range(7):
                if not math.isnan(ref[i]):             # (infinity times 0 at the far end: no value that is asked for)
                    assert bool(torch.isclose(got[i + 1::8], ref[i], rtol=0, atol=1e-35).all()), (act, i, got[i + 1], ref[i])
