"""Input and parameter gradients of the norms around a block, every thread layout, row by row against 64 bits."""
import pytest
import torch

import seq_bounds as B

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("M,H,D", B.SHAPES)
@pytest.mark.parametrize("kind", ["rms", "layer"])
@pytest.mark.parametrize("bias", [False, True])
def test_block_norm_gradients_row_by_row(M, H, D, kind, bias, dtype):
    from hhrl_vae_amd import sequence
    x, w, d_out = B.inputs(M, H, D, dtype, D)
    want, size, n = B.gradient(x, w, d_out, kind, 1.25)
    tol = B.tolerance(want, size, dtype)
    terms = 1.25 * d_out.double() * n
    want_w, want_b = terms.sum((0, 1)), 1.25 * d_out.double().sum((0, 1))
    # a column: the row's own roundings (those of n, 70 relative to the row's numbers in units of its deviation), rows one after
    # the other in a thread and over row slots, and partial rows in 32 lanes: fewer than M H / 8 + 256 in any split
    n_col = M * H / 8 + 256
    top = x.double().abs().amax(-1, keepdim=True) / x.double().std(-1, unbiased=False, keepdim=True).clamp(min=B.EPS ** 0.5) if D > 1 else 1.0 / B.EPS ** 0.5
    tol_w = B.U32 * ((n_col + 70) * terms.abs() + 70 * 1.25 * d_out.double().abs() * (1 + top)).sum((0, 1))
    tol_b = B.U32 * n_col * 1.25 * d_out.double().abs().sum((0, 1))
    dev = x.to(DEV), w.to(DEV), d_out.to(DEV)
    b = torch.randn(D, generator=torch.Generator().manual_seed(1)).to(DEV) if bias else None
    grad = lambda: (torch.full_like(dev[0], 7.0), torch.zeros(D, device=DEV), torch.zeros(D, device=DEV) if bias else None)
    # behind the block: scale * post(y)
    post = sequence.BlockNorm(D, H=H, post=kind, scale=1.25, eps=B.EPS, dtype=dtype)
    dy, dw, db = grad()
    post.bwd(y=dev[0], w_post=dev[1], b_post=b, d_out=dev[2], dy=dy, dw_post=dw, db_post=db, ws=post.workspace(M, DEV))
    # in front of it: pre(alpha x) with alpha = 1, whose gradient has no scale, so the weight carries it
    pre = sequence.BlockNorm(D, H=H, pre=kind, eps=B.EPS, dtype=dtype)
    dx, dw2, db2 = grad()
    pre.bwd(x=dev[0], w_pre=1.25 * dev[1], b_pre=b, d_h=dev[2], dx=dx, dw_pre=dw2, db_pre=db2, ws=pre.workspace(M, DEV))
    for name, got in (("dy", dy), ("dx", dx)):
        off = (got.cpu().double() - want).abs()
        assert bool((off <= tol).all()), "%s: %g of its bound" % (name, float((off / tol).max()))
    for name, got, ref, t in (("dw_post", dw, want_w, tol_w), ("dw_pre", dw2, want_w / 1.25, tol_w / 1.25), ("db_post", db, want_b, tol_b), ("db_pre", db2, want_b / 1.25, tol_b / 1.25)):
        if got is not None:
            off = (got.cpu().double() - ref).abs()
            assert bool((off <= t).all()), "%s: %g of its bound" % (name, float((off / t).max()))
