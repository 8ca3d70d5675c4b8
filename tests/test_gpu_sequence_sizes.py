"""Norms around a block at the ends of what a plan may be asked for."""
import pytest
import torch

import seq_reference as R

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.mark.parametrize("M", [1, 70, 3000])
def test_block_norm_gate_for_any_number_of_rows(M):
    """A gate said to be shared by more rows than there are: the bits of one shared by all of them."""
    from hhrl_vae_amd import sequence
    D, gen = 72, torch.Generator().manual_seed(M)
    x, y, d_out, d_h = (torch.randn(M, D, generator=gen).to(DEV) for _ in range(4))
    gate, w = torch.randn(1, D, generator=gen).to(DEV), torch.rand(D, generator=gen).to(DEV)
    want = None
    for rows in (max(M, 2), M + 1, (1 << 63) - 1):
        plan = sequence.BlockNorm(D, post="rms", pre="layer", gate_act="silu", gate_rows=rows)
        ins = dict(x=x, y=y, gate=gate, w_post=w)
        out, h, dx, dy, dgate, dw = torch.empty_like(x), torch.empty_like(x), torch.empty_like(x), torch.empty_like(x), torch.empty_like(gate), torch.zeros_like(w)
        plan.fwd(out=out, h=h, **ins)
        plan.bwd(d_out=d_out, d_h=d_h, dx=dx, dy=dy, dgate=dgate, dw_post=dw, ws=plan.workspace(M, DEV), **ins)
        got = (out, h, dx, dy, dgate, dw)
        want = want or got
        for a, b in zip(got, want):
            assert torch.equal(a, b) and bool(torch.isfinite(a).all())


def test_block_norm_shared_gate_plan_without_its_gate():
    """A plan whose gate is shared by 4465 rows, called without the gate in the workspace it gives: the bits of a plan without one."""
    from hhrl_vae_amd import sequence
    M, D, gen = 9201, 8192, torch.Generator(device=DEV).manual_seed(0)
    y, d_out = (torch.randn(M, D, generator=gen, device=DEV).bfloat16() for _ in range(2))
    got = []
    for rows in (4465, 1):
        plan = sequence.BlockNorm(D, post="layer", gate_rows=rows, dtype=torch.bfloat16)
        dy, dw, db = torch.empty_like(y), torch.zeros(D, device=DEV), torch.zeros(D, device=DEV)
        ws = plan.workspace(M, DEV)
        ws.fill_(float("nan"))
        plan.bwd(y=y, d_out=d_out, dy=dy, dw_post=dw, db_post=db, ws=ws)
        got.append((dy, dw, db))
    for a, b in zip(*got):
        assert torch.equal(a, b) and bool(torch.isfinite(a).all())


@pytest.mark.parametrize("M,D,gate_rows", [(1, 33, 1), (700, 72, 1), (5000, 4096, 1), (3000, 64, 700)])
def test_block_norm_parameters_shared_by_both_norms(M, D, gate_rows):
    """One array for the gradients of both norms' weights and one for those of both biases: each gets both, the same bits on
    every run."""
    from hhrl_vae_amd import sequence
    gen = torch.Generator().manual_seed(D)
    rn = lambda *s: torch.randn(*s, generator=gen).to(DEV)
    ins = dict(x=rn(M, D), y=rn(M, D), gate=rn(-(-M // gate_rows), D), w_post=rn(D), b_post=rn(D))
    ins.update(w_pre=ins["w_post"], b_pre=ins["b_post"])
    plan = sequence.BlockNorm(D, post="rms", pre="layer", gate_act="sigmoid", gate_rows=gate_rows)
    ws, d_out, d_h = plan.workspace(M, DEV), rn(M, D), rn(M, D)

    def grads(shared):
        w, b = torch.zeros(D, device=DEV), torch.zeros(D, device=DEV)
        w2, b2 = (w, b) if shared else (torch.zeros(D, device=DEV), torch.zeros(D, device=DEV))
        dgate = torch.empty_like(ins["gate"])
        plan.bwd(d_out=d_out, d_h=d_h, dgate=dgate, dw_post=w, db_post=b, dw_pre=w2, db_pre=b2, ws=ws, **ins)
        return w, b, w2, b2, dgate
    *_, dgate = grads(False)
    first = grads(True)
    for r in range(4):
        sw, sb, _, _, sg = grads(True) if r else first
        assert torch.equal(sw, first[0]) and torch.equal(sb, first[1]) and torch.equal(sg, dgate)
    # what the terms of both add up to in size, in 64 bits; either way a thread's rows, its slots, 32 lanes of partial rows and
    # at last the two parameters: fewer than M / 8 + 256 sums, and the terms' own 128 roundings
    d64 = {k: v.double() for k, v in ins.items()}
    act = torch.sigmoid(d64["gate"])[torch.arange(M, device=DEV) // gate_rows]
    n = R.norm(d64["y"], "rms", None, None, 1e-6)
    r = (d64["x"] + act * (n * d64["w_post"] + d64["b_post"])).requires_grad_(True)
    m = R.norm(r, "layer", None, None, 1e-6)
    ((r * d_out.double()).sum() + ((m * d64["w_pre"] + d64["b_pre"]) * d_h.double()).sum()).backward()
    db = r.grad * act
    for got, parts in ((first[0], (db * n, d_h.double() * m.detach())), (first[1], (db, d_h.double()))):
        want, size = sum(p.sum(0) for p in parts), sum(p.abs().sum(0) for p in parts) + 128 / max(M, 128) * sum(p.abs().max() for p in parts)
        assert bool(((got.double() - want).abs() <= (M / 8 + 384) * R.U32 * size).all())
