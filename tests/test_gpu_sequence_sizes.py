"""Norms around a block at the ends of what a plan may be asked for."""
import pytest
import torch

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
