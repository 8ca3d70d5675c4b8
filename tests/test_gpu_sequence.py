"""The sequence layers (hhrl_vae_amd.sequence) against their definitions in 64 bits: odd widths, ragged and padded
sequences, shared key heads, strides, states, gradients, single tokens, captured graphs, and a run of them together."""
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


def path(K, V, T):
    """Roundings on the longest path through the chunked form: sums over K, V and three times over a chunk, and the state's
    own recurrence with five roundings a chunk; gradients pass the same way back."""
    return 2 * (K + V + 3 * 64 + 5 * (T // 64 + 1))


def make(lead, Hk, Hv, K, V, dtype, seed, gscale=1.0):
    gen = torch.Generator().manual_seed(seed)
    rn = lambda *s: torch.randn(*s, generator=gen)
    unit = lambda t: t / t.norm(dim=-1, keepdim=True).clamp(min=1e-6)
    q, k = unit(rn(*lead, Hk, K)).to(dtype), unit(rn(*lead, Hk, K)).to(dtype)
    v = rn(*lead, Hv, V).to(dtype)
    g = -gscale * torch.rand(*lead, Hv, generator=gen) ** 2
    beta = torch.sigmoid(rn(*lead, Hv))
    return q, k, v, g, beta, rn(*lead, Hv, V).to(dtype)


def reference(ranges, ins, scale, s0, d_o, d_s1):
    leaves = [t.double().reshape(-1, *t.shape[-(2 if i < 3 else 1):]).requires_grad_(True) for i, t in enumerate(ins)]
    s0 = s0.double().requires_grad_(True)
    o, s1 = R.gdr_batch(ranges, *leaves, scale, s0)
    loss = (o * d_o.double().reshape(o.shape)).sum() + (s1 * d_s1.double()).sum()
    loss.backward()
    zero = lambda t: t.grad if t.grad is not None else torch.zeros_like(t)
    return o.detach(), s1.detach(), [zero(t) for t in leaves], zero(s0)


def check_gdr(seq, dtype, Hk, Hv, K, V, ranges, lead, starts=None, lens=None, seed=0, gscale=1.0, edit=None, wide=0):
    rows = 1
    for s in lead:
        rows *= s
    q, k, v, g, beta, d_o = make(lead, Hk, Hv, K, V, dtype, seed, gscale)
    if edit:
        edit(q, k, v, g, beta)
    n = len(ranges)
    gen = torch.Generator().manual_seed(seed + 1)
    s0, d_s1 = 0.5 * torch.randn(n, Hv, K, V, generator=gen), torch.randn(n, Hv, K, V, generator=gen)
    scale = K ** -0.5
    clean = [t.clone() for t in (q, k, v, g, beta)]
    used = torch.zeros(rows, dtype=torch.bool)
    for a, b in ranges:
        used[a:b] = True
    for t in clean:
        t.view(rows, *t.shape[len(lead):])[~used] = 0
    dclean = d_o.clone()
    dclean.view(rows, Hv, V)[~used] = 0
    o_r, s1_r, grads_r, ds0_r = reference(ranges, clean, scale, s0, dclean, d_s1)

    def to_dev(t, junk=float("nan")):
        """On the GPU, as a column range of a wider buffer if asked for; rows of nobody hold NaN."""
        t = t.clone()
        t.view(rows, *t.shape[len(lead):])[~used] = junk
        if not wide:
            return t.to(DEV)
        flat = t.reshape(rows, -1)
        buf = torch.full((rows, flat.shape[1] + 2 * wide), float("nan"), dtype=t.dtype, device=DEV)
        buf[:, wide: wide + flat.shape[1]] = flat.to(DEV)
        view = buf[:, wide: wide + flat.shape[1]]
        return view.as_strided(t.shape, [buf.shape[1] * math.prod(lead[i + 1:]) for i in range(len(lead))]
                               + [math.prod(t.shape[i + 1:]) for i in range(len(lead), t.dim())], view.storage_offset())

    layer = seq.GatedDelta(Hk, Hv, K, V, dtype=dtype)
    dev = [to_dev(t) for t in (q, k, v, g, beta)]
    out = [to_dev(torch.full_like(t, 7.0), 7.0) for t in (v, q, k, v, g, beta)]
    o, dq, dk, dv, dg, dbeta = out
    ws = layer.workspace(n, rows, DEV, packed=starts is not None)
    ws.fill_(float("nan"))
    s1, ds0 = torch.full((n, Hv, K, V), 7.0, device=DEV), torch.full((n, Hv, K, V), 7.0, device=DEV)
    st = torch.tensor(starts, dtype=torch.int32, device=DEV) if starts is not None else None
    ln = torch.tensor(lens, dtype=torch.int32, device=DEV) if lens is not None else None
    s0d = s0.to(DEV)
    layer.fwd(*dev, o, ws, s0=s0d, s1=s1, starts=st, lens=ln)
    layer.bwd(*dev, to_dev(d_o), dq, dk, dv, dg, dbeta, ws, d_s1=d_s1.to(DEV), d_s0=ds0, starts=st, lens=ln)
    o2, s12 = torch.full_like(o, 7.0), torch.empty_like(s1)
    ws2 = layer.workspace(n, rows, DEV, packed=starts is not None, no_backward=True)
    ws2.fill_(float("nan"))
    layer.fwd(*dev, o2, ws2, s0=s0d, s1=s12, starts=st, lens=ln, no_backward=True)
    torch.cuda.synchronize()
    T = max([b - a for a, b in ranges] + [1])
    m = path(K, V, T)
    flat = lambda t: t.reshape(rows, *t.shape[len(lead):])
    assert torch.equal(flat(o2)[used], flat(o)[used]) and torch.equal(s12, s1)
    for name, got, want in (("o", o, o_r), ("dq", dq, grads_r[0]), ("dk", dk, grads_r[1]), ("dv", dv, grads_r[2]),
                            ("dg", dg, grads_r[3]), ("dbeta", dbeta, grads_r[4])):
        got = flat(got).cpu()
        R.close(name, got, want, m, where=used)
        assert bool((got[~used] == 7.0).all()), name + ": a row of nobody was written"
    R.close("s1", s1, s1_r, m)
    R.close("d_s0", ds0, ds0_r, m)


def packed(lens, tail=0):
    starts = [0]
    for n in lens:
        starts.append(starts[-1] + n)
    return [(a, b) for a, b in zip(starts, starts[1:])], (starts[-1] + tail,), starts


@pytest.mark.parametrize("dtype", [F32, BF])
@pytest.mark.parametrize("Hk,Hv,K,V,lens", [
    (1, 1, 1, 1, [1]), (1, 1, 64, 32, [1]), (2, 2, 64, 64, [63]), (1, 2, 128, 128, [64]), (1, 1, 128, 128, [65]),
    (2, 4, 61, 72, [130, 0, 1, 77]), (1, 3, 128, 33, [200]), (1, 1, 65, 160, [129]), (3, 3, 8, 31, [5, 64, 128, 0]),
    (1, 1, 17, 512, [70]), (1, 1, 128, 5, [0, 0, 3]),
])
def test_gdr_packed(seq, dtype, Hk, Hv, K, V, lens):
    ranges, lead, starts = packed(lens, tail=3)
    check_gdr(seq, dtype, Hk, Hv, K, V, ranges, lead, starts=starts, seed=K + V)


@pytest.mark.parametrize("dtype", [F32, BF])
@pytest.mark.parametrize("T,lens", [(70, None), (130, [130, 0, 64, 1]), (3, [1, 2, 3]), (3201, [3201, 1601, 0])])
def test_gdr_padded(seq, dtype, T, lens):
    B = 4 if lens is None else len(lens)
    ranges = [(b * T, b * T + (T if lens is None else lens[b])) for b in range(B)]
    check_gdr(seq, dtype, 2, 2, 64, 48, ranges, (B, T), lens=lens, seed=T)


@pytest.mark.parametrize("dtype", [F32, BF])
@pytest.mark.parametrize("K,V,Hv,lens", [(64, 32, 2, [3333]), (65, 40, 1, [70, 0, 3200, 1]), (16, 128, 2, [5000])])
def test_gdr_long_sequences_with_few_heads(seq, dtype, K, V, Hv, lens):
    """Long enough for the walk over the chunks to be cut into segments that run side by side."""
    ranges, lead, starts = packed(lens, tail=1)
    check_gdr(seq, dtype, 1, Hv, K, V, ranges, lead, starts=starts, seed=K + V, gscale=0.05)


@pytest.mark.parametrize("dtype", [F32, BF])
@pytest.mark.parametrize("lens", [[70, 0, 1, 64, 65, 130, 3, 3, 200], [1] * 64, [3] * 65 + [70]])
def test_gdr_more_sequences_than_run_at_once(seq, dtype, lens):
    """Enough workgroups for the order of the sequences to matter (the longest go first, up to 64 of them)."""
    Hv = 576 // (2 * len(lens)) + 1 if len(lens) > 9 else 32
    ranges, lead, starts = packed(lens)
    check_gdr(seq, dtype, 1, Hv, 8, 33, ranges, lead, starts=starts, seed=len(lens))
    T = max(lens)
    check_gdr(seq, dtype, 1, Hv, 8, 33, [(i * T, i * T + n) for i, n in enumerate(lens)], (len(lens), T), lens=lens, seed=1 + len(lens))


@pytest.mark.parametrize("T", [100, 3333])
def test_gdr_states_in_place(seq, T):
    """s1 over s0 and d_s0 over d_s1, of one walk and of segments that run side by side: the same bits as apart."""
    q, k, v, g, beta, d_o = (t.to(DEV) for t in make((2, T), 1, 1, 64, 32, BF, T, 0.05))
    layer = seq.GatedDelta(1, 1, 64, 32, dtype=BF)
    ws = layer.workspace(2, 2 * T, DEV, packed=False)
    gen = torch.Generator().manual_seed(T)
    s0, d_s1 = (torch.randn(2, 1, 64, 32, generator=gen).to(DEV) for _ in range(2))

    def go(s, s1, d, d0):
        o, grads = torch.empty_like(v), [torch.empty_like(t) for t in (q, k, v, g, beta)]
        layer.fwd(q, k, v, g, beta, o, ws, s0=s, s1=s1)
        layer.bwd(q, k, v, g, beta, d_o, *grads, ws, d_s1=d, d_s0=d0)
        return [o, s1, d0] + grads
    want = go(s0, torch.empty_like(s0), d_s1, torch.empty_like(d_s1))
    for _ in range(3):
        s, d = s0.clone(), d_s1.clone()
        for a, b in zip(go(s, s, d, d), want):
            assert torch.equal(a, b)


@pytest.mark.parametrize("dtype", [F32, BF])
@pytest.mark.parametrize("wide", [8, 3])
def test_gdr_columns_of_wider_buffers(seq, dtype, wide):
    ranges, lead, starts = packed([100, 30])
    check_gdr(seq, dtype, 1, 2, 128, 64, ranges, lead, starts=starts, seed=wide, wide=wide)
    check_gdr(seq, dtype, 1, 2, 64, 64, [(0, 70), (70, 140)], (2, 70), seed=wide, wide=wide)


@pytest.mark.parametrize("dtype", [F32, BF])
@pytest.mark.parametrize("what", ["reset", "strong", "none", "one"])
def test_gdr_decays(seq, dtype, what):
    """Log decays of -infinity (the state is forgotten), sums of log decays in the thousands, no decay, and beta = 1 on equal
    keys (the largest entries of the triangular inverse)."""
    def edit(q, k, v, g, beta):
        if what == "reset":
            g[10] = -math.inf
            g[70:72] = -math.inf
        elif what == "strong":
            g.mul_(80.0)
        elif what == "none":
            g.zero_()
        else:
            g.zero_()
            beta.fill_(1.0)
            k[1:] = k[:1]
    ranges, lead, starts = packed([150])
    if what == "reset":
        # the reference's own gradient of exp() at -infinity is 0 * infinity: a decay of -2000 is the same number, 0
        inner = edit

        def edit(q, k, v, g, beta):
            inner(q, k, v, g, beta)
            g.clamp_(min=-2000.0)
    check_gdr(seq, dtype, 1, 1, 64, 64, ranges, lead, starts=starts, seed=5, edit=edit)


def test_gdr_minus_infinity_is_a_decay_of_zero(seq):
    q, k, v, g, beta, d_o = (t.to(DEV) for t in make((1, 100), 1, 1, 64, 64, F32, 3))
    layer = seq.GatedDelta(1, 1, 64, 64)
    res = []
    for low in (-math.inf, -3000.0):
        g[0, 40] = low
        g[0, 41] = low
        ws = layer.workspace(1, 100, DEV)
        outs = [torch.empty_like(t) for t in (v, q, k, v, g, beta)]
        layer.fwd(q, k, v, g, beta, outs[0], ws)
        layer.bwd(q, k, v, g, beta, d_o, *outs[1:], ws)
        res.append(outs)
    for a, b in zip(*res):
        assert torch.isfinite(a).all() and torch.equal(a, b)


def test_gdr_gradient_against_differences(seq):
    """<d_o, o> + <d_s1, s1> moved by +-h along a direction, fp32: the loss's own rounding (gamma of its path times the sum
    of its terms' sizes) over 2h, and h^2 of the third derivative, which is kept below it by h = 2^-7 on inputs of size 1/8."""
    Hk, Hv, K, V, T = 1, 2, 24, 20, 90
    ins = list(make((1, T), Hk, Hv, K, V, F32, 11))
    d_o = ins.pop().to(DEV)
    ins = [t.to(DEV) for t in ins]
    layer = seq.GatedDelta(Hk, Hv, K, V)
    ws = layer.workspace(1, T, DEV)
    o = torch.empty_like(ins[2])

    def loss(args):
        layer.fwd(*args, o, ws)
        return float((o.double() * d_o.double()).sum()), float((o.double() * d_o.double()).abs().sum())
    layer.fwd(*ins, o, ws)
    grads = [torch.empty_like(t) for t in ins]
    layer.bwd(*ins, d_o, *grads, ws)
    h = 2.0 ** -7
    for i in range(5):
        step = torch.randn(ins[i].shape, generator=torch.Generator().manual_seed(i)).to(DEV) / 8
        lo, hi = list(ins), list(ins)
        lo[i], hi[i] = ins[i] - h * step, ins[i] + h * step
        (a, size), (b, _) = loss(lo), loss(hi)
        want = float((grads[i].double() * step.double()).sum())
        tol = path(K, V, T) * R.U32 * size / (2 * h) + h * h * size
        assert abs((b - a) / (2 * h) - want) <= tol, (i, (b - a) / (2 * h), want, tol)


def test_gdr_only_state_gradient_and_no_initial_state(seq):
    q, k, v, g, beta, _ = make((1, 66), 1, 1, 32, 40, F32, 2)
    d_s1 = torch.randn(1, 1, 32, 40, generator=torch.Generator().manual_seed(1))
    _, _, want, ds0 = reference([(0, 66)], (q, k, v, g, beta), 32 ** -0.5, torch.zeros(1, 1, 32, 40), torch.zeros(1, 66, 1, 40), d_s1)
    layer = seq.GatedDelta(1, 1, 32, 40)
    dev = [t.to(DEV) for t in (q, k, v, g, beta)]
    ws = layer.workspace(1, 66, DEV)
    o, grads = torch.empty_like(dev[2]), [torch.empty_like(t) for t in dev]
    layer.fwd(*dev, o, ws)
    layer.bwd(*dev, None, *grads, ws, d_s1=d_s1.to(DEV))
    for name, a, b in zip("q k v g beta".split(), grads, want):
        R.close(name, a.reshape(b.shape), b, path(32, 40, 66))


def test_gdr_same_bits_and_state_handed_on(seq):
    """A sequence in two halves, the state of the first handed to the second in place, gives what it gives in one
    (to rounding; halves at a chunk's end form the same sums), and every run the same bits."""
    q, k, v, g, beta, _ = (t.to(DEV) for t in make((1, 192), 2, 2, 64, 64, BF, 9))
    layer = seq.GatedDelta(2, 2, 64, 64, dtype=BF)
    ws = layer.workspace(1, 192, DEV, no_backward=True)
    o, s1 = torch.empty_like(v), torch.empty(1, 2, 64, 64, device=DEV)
    layer.fwd(q, k, v, g, beta, o, ws, s1=s1, no_backward=True)
    for _ in range(2):
        o2, s = torch.empty_like(v), torch.zeros(1, 2, 64, 64, device=DEV)
        for a, b in ((0, 128), (128, 192)):
            part = [t[:, a:b] for t in (q, k, v, g, beta)]
            layer.fwd(*part, o2[:, a:b], ws, s0=s, s1=s, no_backward=True)
        assert torch.equal(o, o2) and torch.equal(s, s1)


@pytest.mark.parametrize("dtype", [F32, BF])
def test_gdr_captured_and_replayed(seq, dtype):
    B, T = 3, 100
    layer = seq.GatedDelta(1, 2, 64, 64, dtype=dtype)
    ws = layer.workspace(B, B * T, DEV)
    ins = [t.to(DEV) for t in make((B, T), 1, 2, 64, 64, dtype, 1)]
    outs = [torch.zeros_like(t) for t in (ins[2], ins[0], ins[1], ins[2], ins[3], ins[4])]
    lens = torch.tensor([100, 3, 64], dtype=torch.int32, device=DEV)

    def go(i, o, w, ln):
        layer.fwd(*i[:5], o[0], w, lens=ln)
        layer.bwd(*i[:5], i[5], *o[1:], w, lens=ln)
    go(ins, outs, ws, lens)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        go(ins, outs, ws, lens)
    for r in range(4):
        new = [t.to(DEV) for t in make((B, T), 1, 2, 64, 64, dtype, 20 + r)]
        for a, b in zip(ins, new):
            a.copy_(b)
        lens.copy_(torch.tensor([[100, 3, 64], [1, 0, 99], [64, 65, 63], [100, 100, 100]][r], dtype=torch.int32))
        for t in outs:
            t.zero_()
        graph.replay()
        eager = [torch.zeros_like(t) for t in outs]
        go(new, eager, layer.workspace(B, B * T, DEV), lens)
        torch.cuda.synchronize()
        for a, b in zip(outs, eager):
            assert torch.equal(a, b) and torch.isfinite(a).all()


@pytest.mark.parametrize("dtype", [F32, BF])
def test_gdr_two_streams(seq, dtype):
    """Two calls at once, each with its own workspace, on streams that are not torch's default."""
    sets = [[t.to(DEV) for t in make((2, 300), 1, 1, 64, 64, dtype, s)] for s in (1, 2)]
    layer = seq.GatedDelta(1, 1, 64, 64, dtype=dtype)
    want = []
    for ins in sets:
        outs = [torch.zeros_like(t) for t in (ins[2], ins[0], ins[1], ins[2], ins[3], ins[4])]
        ws = layer.workspace(2, 600, DEV)
        layer.fwd(*ins[:5], outs[0], ws)
        layer.bwd(*ins[:5], ins[5], *outs[1:], ws)
        want.append(outs)
    torch.cuda.synchronize()
    got, keep = [], []
    for ins in sets:
        st = torch.cuda.Stream()
        outs = [torch.zeros_like(t) for t in (ins[2], ins[0], ins[1], ins[2], ins[3], ins[4])]
        ws = layer.workspace(2, 600, DEV)
        st.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(st):
            layer.fwd(*ins[:5], outs[0], ws)
            layer.bwd(*ins[:5], ins[5], *outs[1:], ws)
        got.append(outs)
        keep.append((st, ws))
    torch.cuda.synchronize()
    for a, b in zip(want, got):
        for x, y in zip(a, b):
            assert torch.equal(x, y)


# ------------------------------------------------------------------------------------------------------- one token
@pytest.mark.parametrize("dtype", [F32, BF])
@pytest.mark.parametrize("Hk,Hv,K,V", [(1, 1, 1, 1), (2, 4, 64, 64), (1, 2, 128, 128), (1, 3, 61, 72), (1, 1, 128, 33), (2, 2, 5, 512)])
def test_gdr_step(seq, dtype, Hk, Hv, K, V):
    B, n = 5, 9
    q, k, v, g, beta, _ = make((B,), Hk, Hv, K, V, dtype, K + V)
    pool = torch.randn(n, Hv, K, V, generator=torch.Generator().manual_seed(1))
    slots = [7, -1, 0, 3, -5]
    layer = seq.GatedDelta(Hk, Hv, K, V, dtype=dtype)
    dev = [t.to(DEV) for t in (q, k, v, g, beta)]
    o, state = torch.full_like(dev[2], 7.0), pool.to(DEV)
    out = torch.full_like(state, 7.0)
    sl = torch.tensor(slots, dtype=torch.int32, device=DEV)
    layer.step(*dev, o, state, state_out=out, slots=sl)
    assert torch.equal(state.cpu(), pool)
    o_in = torch.empty_like(o)
    layer.step(*dev, o_in, state, slots=sl)
    n_round = 2 * K + 16
    for b, s in enumerate(slots):
        if s < 0:
            assert bool((o[b] == 0).all())
            continue
        y, S = R.gdr(*[t[b: b + 1].double() for t in (q, k, v, g, beta)], K ** -0.5, pool[s].double())
        R.close("o", o[b], y[0], n_round)
        R.close("state", out[s], S, n_round)
        assert torch.equal(out[s], state[s])
    assert torch.equal(o, o_in)
    for s in range(n):
        if s not in slots:
            assert bool((out[s] == 7.0).all()) and torch.equal(state[s].cpu(), pool[s])
    # without slots: row b and state b
    first = pool[:B].to(DEV)
    layer.step(*dev, o, first)
    y, S = R.gdr(*[t[2:3].double() for t in (q, k, v, g, beta)], K ** -0.5, pool[2].double())
    R.close("state", first[2], S, n_round)


def test_gdr_step_bad_slots(seq):
    """A slot past the pool and a slot named twice: NaN for that row, nothing moved for it, the others as they should be."""
    layer = seq.GatedDelta(1, 1, 64, 64)
    B, n = 4, 6
    q, k, v, g, beta, _ = (t.to(DEV) for t in make((B,), 1, 1, 64, 64, F32, 4))
    pool = torch.randn(n, 1, 64, 64, device=DEV)
    ok, o_ok = pool.clone(), torch.empty_like(v)
    layer.step(q, k, v, g, beta, o_ok, ok, slots=torch.tensor([2, 5, -1, 0], dtype=torch.int32, device=DEV))
    bad, o = pool.clone(), torch.empty_like(v)
    layer.step(q, k, v, g, beta, o, bad, slots=torch.tensor([2, n, 2, 0], dtype=torch.int32, device=DEV))
    assert torch.isnan(o[1]).all() and torch.isnan(o[2]).all()
    assert torch.equal(o[0], o_ok[0]) and torch.equal(o[3], o_ok[3])
    assert torch.equal(bad[2], ok[2]) and torch.equal(bad[0], ok[0]) and torch.equal(bad[5], pool[5])


def test_gdr_steps_follow_the_sequence(seq):
    """Prefill, then token by token from the state it leaves: the outputs of the whole sequence."""
    Hk, Hv, K, V, T, P = 2, 4, 64, 96, 90, 70
    q, k, v, g, beta, _ = make((1, T), Hk, Hv, K, V, F32, 8)
    o_r, s1_r = R.gdr_batch([(0, T)], *[t[0].double() for t in (q, k, v, g, beta)], K ** -0.5, torch.zeros(1, Hv, K, V, dtype=torch.float64))
    layer = seq.GatedDelta(Hk, Hv, K, V)
    dev = [t.to(DEV) for t in (q, k, v, g, beta)]
    state = torch.empty(1, Hv, K, V, device=DEV)
    o = torch.empty(1, T, Hv, V, device=DEV)
    layer.fwd(*[t[:, :P] for t in dev], o[:, :P], layer.workspace(1, P, DEV, no_backward=True), s1=state, no_backward=True)
    for t in range(P, T):
        layer.step(*[x[:, t] for x in dev], o[:, t], state)
    R.close("o", o[0], o_r, path(K, V, T) + (T - P) * (2 * K + 16))
    R.close("s1", state, s1_r, path(K, V, T) + (T - P) * (2 * K + 16))


# ------------------------------------------------------------------------------------------------------------ norms
def check_norm(seq, dtype, M, H, D, post, pre, x, y, gate, gate_rows, bias=True, weight=True, seed=0, d_out=True, d_h=True, wide=0):
    gen = torch.Generator().manual_seed(seed)
    rn = lambda *s: torch.randn(*s, generator=gen)
    t = {"x": rn(M, H, D).to(dtype) if x else None, "y": (0.3 + rn(M, H, D)).to(dtype) if y else None}
    t["gate"] = None if gate == "off" else rn(M, H, D).to(dtype) if gate_rows == 1 else rn(-(-M // gate_rows), 1, D)
    for which, kind in (("post", post), ("pre", pre)):
        t["w_" + which] = 1 + 0.3 * rn(D) if kind != "none" and weight else None
        t["b_" + which] = rn(D) if kind != "none" and bias else None
    alpha, scale, eps = 0.75, 1.25, 1e-5
    act = "none" if gate == "off" else gate
    leaf = {k: v.double().requires_grad_(True) if v is not None else None for k, v in t.items()}
    r, h = R.block_norm(*[leaf[k] for k in ("x", "y", "gate", "w_post", "b_post", "w_pre", "b_pre")], post, pre, act, gate_rows, alpha, scale, eps)
    go, gh = rn(M, H, D).to(dtype), rn(M, H, D).to(dtype)
    loss = (r * go.double()).sum() * float(d_out) + (h * gh.double()).sum() * float(d_h)
    loss.backward()
    plan = seq.BlockNorm(D, H=H, post=post, pre=pre, gate_act=act, gate_rows=gate_rows, alpha=alpha, scale=scale, eps=eps, dtype=dtype)

    def place(v):
        if not wide or v.dim() != 3:
            return v.to(DEV)
        buf = torch.full((v.shape[0], v.shape[1] * v.shape[2] + 2 * wide), 7.0, dtype=v.dtype, device=DEV)
        at = buf[:, wide: wide + v.shape[1] * v.shape[2]].unflatten(1, v.shape[1:])
        at.copy_(v)
        return at
    dev = {k: place(v) if v is not None else None for k, v in t.items()}
    out, hh = place(torch.zeros(M, H, D, dtype=dtype)), place(torch.zeros(M, H, D, dtype=dtype))
    plan.fwd(out=out, h=hh, **dev)
    grads = {"d" + k: (place(torch.full_like(v, 2.0)) if v is not None else None) for k, v in t.items()}
    if not d_h:
        grads["dw_pre"] = grads["db_pre"] = None
    ws = plan.workspace(M, DEV)
    ws.fill_(float("nan"))
    plan.bwd(d_out=place(go) if d_out else None, d_h=place(gh) if d_h else None, ws=ws, **dev, **grads)
    torch.cuda.synchronize()
    # a row: sums of up to 16 elements a thread and a tree over the row's threads, twice each norm, about 40 further roundings;
    # column sums: rows per thread, row slots, then partial rows in eight lanes
    n_row, n_col = 128, 128 + M * H // 16 + 64 + 16
    # the sizes of what cancels: a normalised row carries the rounding of its input times 1/std, a norm's gradient is the
    # difference of terms of the size dn/std and n mean(dn n)/std
    with torch.no_grad():
        big = lambda v: float(v.abs().max()) if v is not None else 0.0

        def stats(v, kind):
            if kind == "none":
                return 1.0, 1.0
            c = v - v.mean(-1, keepdim=True) if kind == "layer" else v
            rstd = big(1 / ((c * c).mean(-1) + eps).sqrt())
            return rstd, max(1.0, rstd * big(v))
        rp, mp = stats(r, pre)
        wp = big(leaf["w_pre"]) if pre != "none" and weight else 1.0
        size_r = big(go) + big(gh) * wp * rp * (1 + mp)
        sizes = {"x": alpha * size_r, "w_pre": big(gh) * mp, "b_pre": big(gh)}
        if y:
            rq, mq = stats(leaf["y"], post)
            wq = big(leaf["w_post"]) if post != "none" and weight else 1.0
            zg = max(1.0, big(leaf["gate"]))
            body = mq * wq + big(leaf["b_post"])
            sizes.update(y=size_r * scale * zg * wq * rq * (1 + mq), gate=size_r * scale * body * 2, w_post=size_r * scale * zg * mq, b_post=size_r * scale * zg)
        size_out = alpha * big(leaf["x"]) + (scale * zg * body if y else 0.0)
    R.close("out", out, r.detach(), n_row, size=size_out)
    R.close("h", hh, h.detach(), n_row, size=size_out * rp * wp)
    for k, v in leaf.items():
        got = grads["d" + k]
        if got is None:
            continue
        want = v.grad if v.grad is not None else torch.zeros_like(v)
        par = "_" in k
        R.close("d" + k, got - 2.0 if par else got, want, n_col if par or (k == "gate" and gate_rows > 1) else n_row, size=sizes[k] + (2.0 if par else 0.0))


@pytest.mark.parametrize("dtype", [F32, BF])
@pytest.mark.parametrize("M,H,D", [(1, 1, 1), (3, 1, 256), (33, 1, 100), (700, 3, 17), (300, 8, 128), (9, 2, 1000), (70, 1, 2048), (5, 1, 4096), (3, 1, 8192),
                                   (2100, 1, 640), (2050, 1, 1504), (2049, 1, 2056), (4, 1, 5001)])
@pytest.mark.parametrize("post,pre,gate", [("rms", "rms", "silu"), ("layer", "layer", "sigmoid"), ("none", "rms", "none")])
def test_block_norm(seq, dtype, M, H, D, post, pre, gate):
    check_norm(seq, dtype, M, H, D, post, pre, True, True, gate, 1, seed=D)


@pytest.mark.parametrize("dtype", [F32, BF])
@pytest.mark.parametrize("post,pre,x,y,gate", [("none", "rms", True, False, "off"), ("none", "layer", True, False, "off"), ("rms", "none", False, True, "silu"),
                                               ("layer", "none", True, True, "off"), ("none", "none", True, True, "sigmoid"), ("rms", "layer", False, True, "off")])
def test_block_norm_parts(seq, dtype, post, pre, x, y, gate):
    check_norm(seq, dtype, 37, 1, 264, post, pre, x, y, gate, 1, seed=1)
    check_norm(seq, dtype, 37, 2, 51, post, pre, x, y, gate, 1, seed=2, weight=False, bias=False)
    check_norm(seq, dtype, 37, 2, 64, post, pre, x, y, gate, 1, seed=3, wide=8)
    check_norm(seq, dtype, 37, 2, 64, post, pre, x, y, gate, 1, seed=4, wide=1, d_out=False)
    check_norm(seq, dtype, 37, 1, 64, post, pre, x, y, gate, 1, seed=5, d_h=False)


@pytest.mark.parametrize("dtype", [F32, BF])
@pytest.mark.parametrize("M,gate_rows,D", [(10, 3, 40), (10, 10, 256), (10, 64, 33), (2500, 2500, 72), (2500, 2, 16), (3000, 700, 1024), (5000, 3, 64), (1030, 1029, 4096)])
def test_block_norm_shared_gate(seq, dtype, M, gate_rows, D):
    check_norm(seq, dtype, M, 1, D, "rms", "rms", True, True, "silu", gate_rows, seed=M + D)


def test_block_norm_in_place_and_same_bits(seq):
    M, D = 500, 512
    x, y, w, w2 = (torch.randn(*s, device=DEV) for s in ((M, D), (M, D), (D,), (D,)))
    plan = seq.BlockNorm(D, post="rms", pre="layer")
    out, h = torch.empty_like(x), torch.empty_like(x)
    plan.fwd(x=x, y=y, w_post=w, w_pre=w2, out=out, h=h)
    a, b = x.clone(), y.clone()
    plan.fwd(x=a, y=b, w_post=w, w_pre=w2, out=a, h=b)
    assert torch.equal(a, out) and torch.equal(b, h)
    res = []
    for _ in range(2):
        dw = torch.zeros(D, device=DEV)
        plan.bwd(x=x, y=y, w_post=w, w_pre=w2, d_out=y, d_h=x, dw_post=dw, ws=plan.workspace(M, DEV))
        res.append(dw)
    assert torch.equal(*res)


def test_block_norm_captured_and_replayed(seq):
    M, D = 2300, 384
    plan = seq.BlockNorm(D, post="rms", pre="rms", gate_act="silu", gate_rows=M, dtype=BF)
    names = ("x", "y", "d_out", "d_h")
    ins = {k: torch.randn(M, D, device=DEV).to(BF) for k in names}
    ins.update(gate=torch.randn(1, D, device=DEV), w_post=torch.randn(D, device=DEV), w_pre=torch.randn(D, device=DEV))
    outs = {"out": torch.zeros(M, D, device=DEV, dtype=BF), "h": torch.zeros(M, D, device=DEV, dtype=BF)}
    grads = {"d" + k: torch.zeros_like(ins[k]) for k in ("x", "y", "gate", "w_post", "w_pre")}
    ws = plan.workspace(M, DEV)

    def go(i, o, g, w):
        f = {k: i[k] for k in ("x", "y", "gate", "w_post", "w_pre")}
        plan.fwd(**f, **o)
        for k in ("dw_post", "dw_pre"):
            g[k].zero_()
        plan.bwd(**f, d_out=i["d_out"], d_h=i["d_h"], ws=w, **g)
    go(ins, outs, grads, ws)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        go(ins, outs, grads, ws)
    for r in range(3):
        for k in names:
            ins[k].copy_(torch.randn(M, D, generator=torch.Generator().manual_seed(r)).to(BF))
        graph.replay()
        o2, g2 = {k: torch.zeros_like(v) for k, v in outs.items()}, {k: torch.zeros_like(v) for k, v in grads.items()}
        go(ins, o2, g2, plan.workspace(M, DEV))
        torch.cuda.synchronize()
        for k in outs:
            assert torch.equal(outs[k], o2[k])
        for k in grads:
            assert torch.equal(grads[k], g2[k])


# --------------------------------------------------------------------------------------------------------- refusals
def test_offsets_beyond_32_bits(seq):
    """Rows 8 MB apart (the last ones begin 9 GB behind the first), as columns of one buffer: the bits of contiguous rows."""
    T, ld = 1100, (1 << 22) - 64
    big = torch.empty(T * ld, dtype=BF, device=DEV)
    at = iter(range(0, ld, 64))
    far = lambda: big.as_strided((1, T, 1, 64), (T * ld, ld, 64, 1), next(at))
    near = [t.to(DEV) for t in make((1, T), 1, 1, 64, 64, BF, 3, 0.05)]
    layer = seq.GatedDelta(1, 1, 64, 64, dtype=BF)
    ws = layer.workspace(1, T, DEV, packed=False)
    g, beta, got = near[3], near[4], []
    for new in (lambda t: torch.empty_like(t), lambda t: far()):
        q, k, v, d_o = (new(t) for t in (near[0], near[1], near[2], near[5]))
        for a, b in zip((q, k, v, d_o), (near[0], near[1], near[2], near[5])):
            a.copy_(b)
        o, dq, dk, dv = (new(t) for t in (v, q, k, v))
        dg, db = torch.empty_like(g), torch.empty_like(beta)
        layer.fwd(q, k, v, g, beta, o, ws)
        layer.bwd(q, k, v, g, beta, d_o, dq, dk, dv, dg, db, ws)
        n = seq.BlockNorm(64, post="rms", pre="layer", dtype=BF)
        r, h, dx, dy = (new(v) for _ in range(4))
        flat = lambda t: t.view(T, 64) if t.is_contiguous() else t.as_strided((T, 64), (ld, 1), t.storage_offset())
        n.fwd(x=flat(v), y=flat(o), out=flat(r), h=flat(h))
        n.bwd(x=flat(v), y=flat(o), d_out=flat(d_o), d_h=flat(dv), dx=flat(dx), dy=flat(dy))
        got.append([t.clone() for t in (o, dq, dk, dv, dg, db, r, h, dx, dy)])
    for a, b in zip(*got):
        assert torch.equal(a, b)


def test_step_in_a_pool_beyond_32_bits(seq):
    """2^31 state elements and more: the last states of the pool move as the first."""
    n = (1 << 31) // (2 * 128 * 128) + 3
    pool = torch.empty(n, 2, 128, 128, device=DEV)
    layer = seq.GatedDelta(1, 2, 128, 128, dtype=BF)
    q, k, v, g, beta, _ = (t[0].to(DEV) for t in make((1, 2), 1, 2, 128, 128, BF, 8))
    s0 = torch.randn(2, 2, 128, 128, generator=torch.Generator().manual_seed(0)).to(DEV)
    want, small = torch.empty_like(v), s0.clone()
    layer.step(q, k, v, g, beta, want, small)
    slots = [n - 1, n - 2]
    for i, p in enumerate(slots):
        pool[p] = s0[i]
    o = torch.empty_like(v)
    layer.step(q, k, v, g, beta, o, pool, slots=torch.tensor(slots, dtype=torch.int32, device=DEV))
    assert torch.equal(o, want)
    for i, p in enumerate(slots):
        assert torch.equal(pool[p], small[i])


def test_refusals_on_the_gpu(seq):
    """Wrong types, shapes, strides and places raise ValueError, too small a workspace HipError, before anything is launched."""
    from hhrl_vae_amd._lib import HipError
    layer = seq.GatedDelta(1, 1, 64, 64, dtype=BF)
    q, k, v, g, beta, d_o = (t.to(DEV) for t in make((1, 70), 1, 1, 64, 64, BF, 0))
    o, ws = torch.full_like(v, 7.0), layer.workspace(1, 70, DEV)
    good = dict(q=q, k=k, v=v, g=g, beta=beta, o=o, ws=ws)
    for bad in (dict(q=q.float()), dict(q=q.cpu()), dict(q=q[0]), dict(v=v[:, :69]), dict(g=g.to(BF)), dict(k=k.transpose(2, 3)), dict(o=None),
                dict(beta=beta[..., None]), dict(starts=torch.tensor([0, 70], device=DEV)), dict(lens=torch.tensor([70], dtype=torch.int32)),
                dict(lens=torch.tensor([70, 1], dtype=torch.int32, device=DEV)), dict(s0=torch.zeros(2, 1, 64, 64, device=DEV)),
                dict(s1=torch.zeros(1, 1, 64, 64, device=DEV, dtype=BF)), dict(ws=ws.view(-1, 1)), dict(ws=None)):
        with pytest.raises(ValueError):
            layer.fwd(**{**good, **bad})
    for small in (ws[:1000], ws[1:]):
        with pytest.raises(HipError):
            layer.fwd(**{**good, "ws": small})
    with pytest.raises(HipError):                   # a forward pass alone leaves no room for the backward pass
        layer.fwd(**{**good, "ws": layer.workspace(1, 70, DEV, no_backward=True)})
    with pytest.raises(HipError):
        layer.bwd(q, k, v, g, beta, None, *[torch.empty_like(t) for t in (q, k, v, g, beta)], ws)
    pool = torch.zeros(3, 1, 64, 64, device=DEV)
    row = [t[0, :4].contiguous() for t in (q, k, v, g, beta, v)]
    for bad in (dict(state=pool[:, 0]), dict(state=pool.to(BF)), dict(slots=torch.zeros(4, dtype=torch.int64, device=DEV)), dict(slots=None),
                dict(state_out=torch.zeros(4, 1, 64, 64, device=DEV)), dict(slots=torch.zeros(3, dtype=torch.int32, device=DEV))):
        with pytest.raises(ValueError):
            layer.step(*row, **{**dict(state=pool, slots=torch.zeros(4, dtype=torch.int32, device=DEV)), **bad})
    x = torch.zeros(5, 64, device=DEV)
    w = torch.ones(64, device=DEV)
    plan = seq.BlockNorm(64, post="rms", pre="rms", gate_act="silu", gate_rows=2)
    ok = dict(x=x, y=x, gate=x[:3], out=torch.full_like(x, 7.0), h=torch.empty_like(x), w_post=w, w_pre=w)
    for bad in (dict(x=x.to(BF)), dict(y=x[:4]), dict(gate=x[:2]), dict(gate=x[:3].to(BF)), dict(w_post=w[:63]), dict(w_pre=w.to(BF)), dict(h=None), dict(y=None),
                dict(out=x.t().contiguous().t()), dict(x=None, y=None)):
        with pytest.raises(ValueError):
            plan.fwd(**{**ok, **bad})
    back = {k_: v_ for k_, v_ in ok.items() if k_ not in ("out", "h")}
    for bad in (dict(), dict(d_out=x, d_h=x, dw_pre=w[:3]), dict(d_out=x, dw_pre=w), dict(d_out=x[:4]), dict(d_out=x, ws=torch.zeros(4, dtype=torch.int32, device=DEV))):
        with pytest.raises(ValueError):
            plan.bwd(**back, **bad)
    for ws_ in (None, torch.zeros(16, device=DEV)):
        with pytest.raises(HipError):
            plan.bwd(**back, d_out=x, dw_post=w.clone(), ws=ws_)
    torch.cuda.synchronize()
    assert bool((o == 7.0).all()) and bool((ok["out"] == 7.0).all())


# ---------------------------------------------------------------------------------------------------------- together
def test_layer_of_all_of_them(seq):
    """A residual layer as it would be built: norm before the block, q, k, v, gate and output projections (hhrl_linear_*),
    q and k normalised per head, gated delta rule, gated norm per head, norm after the block and residual sum, with the
    gradients of all parameters, against 64-bit autograd."""
    from hhrl_vae_amd import _lib as L
    lib = L.load()
    B, T, D, H, K, V = 2, 70, 48, 2, 32, 40
    M = B * T
    gen = torch.Generator().manual_seed(0)
    rn = lambda *s: torch.randn(*s, generator=gen)
    W = H * (2 * K + 2 * V)
    p = {"w_in": rn(W, D) / D ** 0.5, "w_out": rn(D, H * V) / (H * V) ** 0.5, "n1": 1 + 0.1 * rn(D), "nh": 1 + 0.1 * rn(V), "n2": 1 + 0.1 * rn(D)}
    x, g, beta, d_out = rn(M, D), -0.3 * torch.rand(B, T, H, generator=gen), torch.sigmoid(rn(B, T, H)), rn(M, D)
    # 64 bits
    P = {k: v.double().requires_grad_(True) for k, v in p.items()}
    X = x.double().requires_grad_(True)
    h = R.norm(X, "rms", P["n1"], None, 1e-6)
    z = h @ P["w_in"].t()
    q, k, v, gt = z.split([H * K, H * K, H * V, H * V], dim=1)
    l2 = lambda t: R.norm(t.reshape(M, H, K), "rms", None, None, 1e-6) * K ** -0.5
    o, _ = R.gdr_batch([(b * T, b * T + T) for b in range(B)], l2(q), l2(k), v.reshape(M, H, V), g.double().reshape(M, H), beta.double().reshape(M, H), K ** -0.5,
                       torch.zeros(B, H, K, V, dtype=torch.float64))
    og = R.norm(o, "rms", P["nh"], None, 1e-6) * torch.nn.functional.silu(gt.reshape(M, H, V))
    y = og.reshape(M, H * V) @ P["w_out"].t()
    r = X + 0.5 * R.norm(y, "rms", P["n2"], None, 1e-6)
    (r * d_out.double()).sum().backward()
    # kernels
    d = {k_: v_.to(DEV) for k_, v_ in p.items()}
    gd = {k_: torch.zeros_like(v_) for k_, v_ in d.items()}
    new = lambda *s: torch.empty(*s, device=DEV)
    x_, dout_ = x.to(DEV), d_out.to(DEV)
    pre, unit = seq.BlockNorm(D, pre="rms"), seq.BlockNorm(K, H=H, post="rms", scale=K ** -0.5)
    heads, after = seq.BlockNorm(V, H=H, post="rms", gate_act="silu"), seq.BlockNorm(D, post="rms", scale=0.5)
    rule = seq.GatedDelta(H, H, K, V)
    h_, z_, qn, kn, o_, og_, y_, r_ = new(M, D), new(M, W), new(M, H, K), new(M, H, K), new(M, H, V), new(M, H, V), new(M, D), new(M, D)
    q_, k_, v_, gt_ = (t.unflatten(1, (H, -1)) for t in z_.split([H * K, H * K, H * V, H * V], dim=1))
    st = L.stream_ptr()
    seqs = lambda t: t.unflatten(0, (B, T))
    ws = rule.workspace(B, M, DEV)
    gb = [t.to(DEV) for t in (g, beta)]
    pre.fwd(x=x_, h=h_, w_pre=d["n1"])
    L.check(lib.hhrl_linear_forward(h_.data_ptr(), D, d["w_in"].data_ptr(), None, z_.data_ptr(), W, M, D, W, 0, 0, st))
    unit.fwd(y=q_, out=qn)
    unit.fwd(y=k_, out=kn)
    rule.fwd(seqs(qn), seqs(kn), seqs(v_), *gb, seqs(o_), ws)
    heads.fwd(y=o_, gate=gt_, w_post=d["nh"], out=og_)
    L.check(lib.hhrl_linear_forward(og_.data_ptr(), H * V, d["w_out"].data_ptr(), None, y_.data_ptr(), D, M, H * V, D, 0, 0, st))
    after.fwd(x=x_, y=y_, w_post=d["n2"], out=r_)
    dz, dqn, dkn, do, dog, dy, dx, dh, dx2 = new(M, W), new(M, H, K), new(M, H, K), new(M, H, V), new(M, H, V), new(M, D), new(M, D), new(M, D), new(M, D)
    dq_, dk_, dv_, dgt_ = (t.unflatten(1, (H, -1)) for t in dz.split([H * K, H * K, H * V, H * V], dim=1))
    dg, dbeta = new(B, T, H), new(B, T, H)
    after.bwd(x=x_, y=y_, w_post=d["n2"], d_out=dout_, dx=dx, dy=dy, dw_post=gd["n2"], ws=after.workspace(M, DEV))
    L.check(lib.hhrl_linear_backward(og_.data_ptr(), H * V, d["w_out"].data_ptr(), None, 0, dy.data_ptr(), D, dog.data_ptr(), H * V, 0, gd["w_out"].data_ptr(), None, M, H * V, D, 0, st))
    heads.bwd(y=o_, gate=gt_, w_post=d["nh"], d_out=dog, dy=do, dgate=dgt_, dw_post=gd["nh"], ws=heads.workspace(M, DEV))
    rule.bwd(seqs(qn), seqs(kn), seqs(v_), *gb, seqs(do), seqs(dqn), seqs(dkn), seqs(dv_), dg, dbeta, ws)
    unit.bwd(y=q_, d_out=dqn, dy=dq_)
    unit.bwd(y=k_, d_out=dkn, dy=dk_)
    L.check(lib.hhrl_linear_backward(h_.data_ptr(), D, d["w_in"].data_ptr(), None, 0, dz.data_ptr(), W, dh.data_ptr(), D, 0, gd["w_in"].data_ptr(), None, M, D, W, 0, st))
    pre.bwd(x=x_, w_pre=d["n1"], d_h=dh, dx=dx2, dw_pre=gd["n1"], ws=pre.workspace(M, DEV))
    torch.cuda.synchronize()
    n = 2 * (path(K, V, T) + D + W + H * V + M + 6 * 128)         # the roundings of all stages, there and back
    R.close("r", r_, r.detach(), n)
    R.close("dx", dx + dx2, X.grad, n)
    for name in p:
        R.close("d" + name, gd[name], P[name].grad, n)
