"""Bounds of the norms' input gradients row by row (64 bits, CPU), tight enough that a gradient without one of its two means is
beyond them: d_out has a mean of its own and one along the normalised row, so both means are of the size of d_out itself.

A row's gradient is rstd (d - mean(d) - n mean(d n)) with d = scale w d_out, n the normalised row (layer norm; without
mean(d) for the RMS norm).  Roundings, u = 2^-24 each: a sum over a row is 8 elements a thread, 6 steps in a wave and up to
16 waves one after the other, 30 in all; mean and square sum behind each other 62, the root and quotient 4, n 2, d 3, the second
sums 30 and the last combination 4: fewer than 128.  What they are relative to, of the row itself: every term of the
bracket, and the row's numbers in units of its deviation, which is what a centred number's rounding is relative to."""
import torch

U32, UBF = 2.0 ** -24, 2.0 ** -8
N_ROW = 128
EPS = 1e-5
SHAPES = [(1, 1, 1), (3, 1, 256), (33, 1, 100), (700, 3, 17), (300, 8, 128), (9, 2, 1000), (70, 1, 2048), (5, 1, 4096), (3, 1, 8192),
          (2100, 1, 640), (2050, 1, 1504), (2049, 1, 2056), (4, 1, 5001), (6, 1, 2), (3, 1, 6144)]


def inputs(M, H, D, dtype, seed):
    gen = torch.Generator().manual_seed(seed)
    rn = lambda *s: torch.randn(*s, generator=gen)
    x = (0.3 + rn(M, H, D)).to(dtype)
    w = 1 + 0.25 * torch.rand(D, generator=gen)
    d_out = (0.7 + 0.5 * x.float() + 0.5 * rn(M, H, D)).to(dtype)
    return x, w, d_out


def gradient(x, w, d_out, kind, scale, without=None):
    """The row gradients in 64 bits (`without`: one of the means left out), and the size the roundings are relative to."""
    v, d = x.double(), scale * w.double() * d_out.double()
    c = v - v.mean(-1, keepdim=True) if kind == "layer" else v
    rstd = 1 / ((c * c).mean(-1, keepdim=True) + EPS).sqrt()
    n = c * rstd
    m1, m2 = (d * n).mean(-1, keepdim=True), d.mean(-1, keepdim=True)
    g = d.clone()
    if without != "along":
        g = g - n * m1
    if kind == "layer" and without != "mean":
        g = g - m2
    top = lambda t: t.abs().amax(-1, keepdim=True)
    size = rstd * (1 + rstd * top(v)) * (top(d) + d.abs().mean(-1, keepdim=True) + top(n) * (d * n).abs().mean(-1, keepdim=True))
    return rstd * g, size, n


def tolerance(want, size, dtype):
    return N_ROW * U32 * size + (UBF * want.abs() if dtype == torch.bfloat16 else 0.0)
