"""The bounds of the norms' gradients have the power they are meant to have: a gradient without one of its means is outside."""
import pytest
import torch

import seq_bounds as B


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("M,H,D", [s for s in B.SHAPES if s[2] > 1])
@pytest.mark.parametrize("kind", ["rms", "layer"])
def test_a_missing_mean_is_beyond_the_bounds(M, H, D, kind, dtype):
    x, w, d_out = B.inputs(M, H, D, dtype, D)
    want, size, _ = B.gradient(x, w, d_out, kind, 1.25)
    tol = B.tolerance(want, size, dtype)
    for without in ("along", "mean") if kind == "layer" else ("along",):
        wrong, _, _ = B.gradient(x, w, d_out, kind, 1.25, without=without)
        rows = ((wrong - want).abs() > 4 * tol).any(-1)
        assert bool(rows.float().mean() > 0.5), "%s: %d of %d rows" % (without, int(rows.sum()), rows.numel())


@pytest.mark.parametrize("kind", ["rms", "layer"])
def test_the_formula_is_autograds(kind):
    x, w, d_out = B.inputs(7, 2, 33, torch.float32, 3)
    leaf = x.double().requires_grad_(True)
    c = leaf - leaf.mean(-1, keepdim=True) if kind == "layer" else leaf
    n = c / ((c * c).mean(-1, keepdim=True) + B.EPS).sqrt()
    (1.25 * n * w.double() * d_out.double()).sum().backward()
    got, _, _ = B.gradient(x, w, d_out, kind, 1.25)
    assert torch.allclose(got, leaf.grad, rtol=1e-12, atol=1e-12)
