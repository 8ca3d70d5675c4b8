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
