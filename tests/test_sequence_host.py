"""The sequence layers' checks of arguments and workspace sizes, which need no GPU: what a call refuses it refuses before
anything is launched."""
import ctypes as C

import pytest
import torch

F32, BF = torch.float32, torch.bfloat16


@pytest.fixture(scope="module")
def lib():
    from hhrl_vae_amd import _lib
    return _lib.load()


@pytest.fixture(scope="module")
def seq():
    from hhrl_vae_amd import sequence
    return sequence


FAKE = 1 << 20                     # an address that no check looks behind


def gdr_desc(**over):
    from hhrl_vae_amd import _lib
    d = _lib.GdrDesc()
    f = dict(dtype=1, n_seq=2, rows=200, Hk=2, Hv=4, K=64, V=64, scale=0.1, q=FAKE, k=FAKE, v=FAKE, ldq=128, ldk=128, ldv=256, g=FAKE, beta=FAKE, ldg=4,
             ldbeta=4, o=FAKE, ldo=256, ws=FAKE, ws_floats=1 << 40, d_o=FAKE, lddo=256, dq=FAKE, dk=FAKE, dv=FAKE, lddq=128, lddk=128, lddv=256, dg=FAKE,
             dbeta=FAKE, lddg=4, lddbeta=4)
    f.update(over)
    for k, v in f.items():
        setattr(d, k, v)
    return d


@pytest.mark.parametrize("over,word", [
    (dict(dtype=2), b"dtype"), (dict(n_seq=0), b"n_seq"), (dict(rows=0), b"rows"), (dict(rows=201), b"one length"), (dict(rows=1 << 31), b"rows"),
    (dict(Hk=3), b"Hk"), (dict(Hk=0), b"Hk"), (dict(K=129), b"K="), (dict(K=0), b"K="), (dict(V=513), b"V="), (dict(q=None), b"null input"),
    (dict(beta=None), b"null input"), (dict(ldq=127), b"leading dimension"), (dict(ldv=255), b"leading dimension"), (dict(ldg=3), b"leading dimension"),
    (dict(ldk=1 << 22), b"leading dimension"), (dict(starts=FAKE, lens=FAKE), b"starts and lens"), (dict(ws=None), b"workspace"),
    (dict(ws=FAKE + 4), b"workspace"), (dict(ws_floats=1000), b"workspace"),
])
def test_gdr_refuses(lib, over, word):
    for fn in (lib.hhrl_gdr_forward, lib.hhrl_gdr_backward):
        assert fn(C.byref(gdr_desc(**over)), None) == 1
        assert word in lib.hhrl_last_error(), lib.hhrl_last_error()


@pytest.mark.parametrize("over", [dict(n_seq=1 << 23, rows=1 << 23), dict(n_seq=4096, rows=4096, Hk=1, Hv=128, V=512, K=1, ldv=1 << 16, ldg=128, ldbeta=128)])
def test_gdr_refuses_more_than_a_launch_holds(lib, over):
    """A launch has fewer than 2^32 threads: 512 for each chunk, and for each 32 columns of a sequence's head."""
    for fn in (lib.hhrl_gdr_forward, lib.hhrl_gdr_backward):
        assert fn(C.byref(gdr_desc(ldo=1 << 16, lddo=1 << 16, lddv=1 << 16, lddg=128, lddbeta=128, **over)), None) == 1
        assert b"too many" in lib.hhrl_last_error(), lib.hhrl_last_error()


def test_gdr_step_refuses_more_than_a_launch_holds(lib):
    assert lib.hhrl_gdr_step(step_desc(B=8192, Hk=1, Hv=256, K=32, V=512, ldv=1 << 17, ldg=256, ldbeta=256, ldo=1 << 17, n_slots=8192, slots=None), None) == 1
    assert b"too large" in lib.hhrl_last_error(), lib.hhrl_last_error()


@pytest.mark.parametrize("over", [dict(o=None), dict(ldo=255), dict(ldo=1 << 22)])
def test_gdr_forward_refuses(lib, over):
    assert lib.hhrl_gdr_forward(C.byref(gdr_desc(**over)), None) == 1


@pytest.mark.parametrize("over", [dict(d_o=None), dict(dq=None), dict(dbeta=None), dict(lddq=1), dict(lddv=1), dict(lddo=1), dict(lddg=3), dict(lddv=1 << 22)])
def test_gdr_backward_refuses(lib, over):
    assert lib.hhrl_gdr_backward(C.byref(gdr_desc(**over)), None) == 1


def test_null_descriptors(lib):
    for fn in (lib.hhrl_gdr_forward, lib.hhrl_gdr_backward, lib.hhrl_block_norm_forward, lib.hhrl_block_norm_backward):
        assert fn(None, None) == 1 and b"descriptor" in lib.hhrl_last_error()


def step_desc(**over):
    from hhrl_vae_amd import _lib
    d = _lib.GdrStepDesc()
    f = dict(dtype=1, B=3, Hk=2, Hv=4, K=64, V=64, scale=0.1, n_slots=8, q=FAKE, k=FAKE, v=FAKE, ldq=128, ldk=128, ldv=256, g=FAKE, beta=FAKE, ldg=4,
             ldbeta=4, o=FAKE, ldo=256, state_in=FAKE, state_out=FAKE, slots=FAKE)
    f.update(over)
    for k, v in f.items():
        setattr(d, k, v)
    return C.byref(d)


@pytest.mark.parametrize("over", [dict(dtype=5), dict(B=0), dict(Hk=0), dict(Hv=5), dict(K=129), dict(V=513), dict(q=None), dict(k=None), dict(ldq=127), dict(ldv=255),
                                  dict(ldo=255), dict(state_in=None), dict(state_out=None), dict(n_slots=0)])
def test_gdr_step_refuses(lib, over):
    assert lib.hhrl_gdr_step(step_desc(**over), None) == 1


def test_gdr_step_refuses_more_rows_than_states(lib):
    assert lib.hhrl_gdr_step(step_desc(B=9, slots=None), None) == 1 and lib.hhrl_gdr_step(None, None) == 1


def norm_desc(**over):
    from hhrl_vae_amd import _lib
    d = _lib.BlockNormDesc()
    f = dict(dtype=0, M=10, H=1, D=64, post=1, pre=2, gate_act=4, gate_rows=1, alpha=1.0, scale=1.0, eps=1e-6, x=FAKE, y=FAKE, gate=FAKE, ldx=64, ldy=64,
             ldgate=64, w_post=FAKE, w_pre=FAKE, b_pre=FAKE, out=FAKE, h=FAKE, ldo=64, ldh=64, d_out=FAKE, d_h=FAKE, lddo=64, lddh=64, dx=FAKE, dy=FAKE,
             dgate=FAKE, lddx=64, lddy=64, lddgate=64, dw_post=FAKE, dw_pre=FAKE, ws=FAKE, ws_floats=1 << 30)
    f.update(over)
    for k, v in f.items():
        setattr(d, k, v)
    return d


@pytest.mark.parametrize("over", [dict(dtype=3), dict(M=0), dict(D=0), dict(D=8193), dict(H=0), dict(post=3), dict(pre=-1), dict(gate_act=1), dict(gate_act=2),
                                  dict(gate_rows=0), dict(gate_rows=2, H=2, ldx=128, ldy=128, ldgate=128), dict(eps=-1.0), dict(x=None, y=None), dict(y=None),
                                  dict(ldx=63), dict(ldy=63), dict(ldgate=63), dict(post=0), dict(M=1 << 40)])
def test_block_norm_refuses(lib, over):
    for fn in (lib.hhrl_block_norm_forward, lib.hhrl_block_norm_backward):
        assert fn(C.byref(norm_desc(**over)), None) == 1


@pytest.mark.parametrize("over", [dict(out=None, h=None), dict(h=None), dict(ldo=63), dict(ldh=63)])
def test_block_norm_forward_refuses(lib, over):
    assert lib.hhrl_block_norm_forward(C.byref(norm_desc(**over)), None) == 1


@pytest.mark.parametrize("over", [dict(d_out=None, d_h=None), dict(lddo=1), dict(lddx=1), dict(x=None), dict(gate=None), dict(ws=None), dict(ws_floats=64),
                                  dict(d_h=None), dict(pre=0, w_pre=None, b_pre=None)])
def test_block_norm_backward_refuses(lib, over):
    assert lib.hhrl_block_norm_backward(C.byref(norm_desc(**over)), None) == 1


def test_workspace_sizes(lib, seq):
    size = lib.hhrl_gdr_workspace_floats
    assert size(1, 2, 200, 0, 2, 4, 64, 64, 1) > 0
    assert size(1, 2, 200, 0, 2, 4, 64, 64, 0) > size(1, 2, 200, 0, 2, 4, 64, 64, 1)
    for bad in ((2, 2, 200, 0, 2, 4, 64, 64, 0), (1, 0, 200, 0, 2, 4, 64, 64, 0), (1, 2, 201, 0, 2, 4, 64, 64, 0), (1, 2, 200, 0, 3, 4, 64, 64, 0),
                (1, 2, 200, 0, 2, 4, 129, 64, 0), (1, 2, 200, 0, 2, 4, 64, 513, 0)):
        assert size(*bad) == 0
    # what serves packed sequences serves as many padded ones of the same rows
    for n, T in ((1, 1), (3, 63), (3, 64), (7, 65), (2, 130), (1, 6400), (5, 2049)):
        for back in (0, 1):
            assert size(0, n, n * T, 1, 1, 2, 32, 40, back) >= size(0, n, n * T, 0, 1, 2, 32, 40, back), (n, T)
    norm = lib.hhrl_block_norm_workspace_floats
    assert norm(10, 1, 64, 1) > 0 and norm(0, 1, 64, 1) == norm(10, 1, 8193, 1) == norm(10, 2, 64, 3) == norm(10, 1, 64, 0) == 0


@pytest.mark.parametrize("make", [
    lambda s: s.GatedDelta(2, 3, 64, 64), lambda s: s.GatedDelta(0, 0, 64, 64), lambda s: s.GatedDelta(1, 1, 129, 64), lambda s: s.GatedDelta(1, 1, 64, 513),
    lambda s: s.GatedDelta(1, 1, 64, 64, dtype=torch.float16), lambda s: s.GatedDelta(1, 1, 64, 64).workspace(0, 10, "cpu"),
    lambda s: s.BlockNorm(0), lambda s: s.BlockNorm(8193), lambda s: s.BlockNorm(64, post="batch"), lambda s: s.BlockNorm(64, gate_act="relu"),
    lambda s: s.BlockNorm(64, H=2, gate_rows=3), lambda s: s.BlockNorm(64, eps=-1.0), lambda s: s.BlockNorm(64, dtype=torch.float64),
    lambda s: s.BlockNorm(64).workspace(0, "cpu"),
])
def test_plans_refuse(seq, make):
    with pytest.raises(ValueError):
        make(seq)


def test_rows_of_tensors(seq):
    """The strides a call takes (host tensors stand in: their device number is -1)."""
    rows = lambda t, n=1, shape=None, dtype=F32: seq._rows("t", t, t.shape if shape is None else shape, n, t.shape[n:].numel(), dtype, -1)
    a = torch.zeros(6, 2, 4)
    assert rows(a) == (a.data_ptr(), 8)
    wide = torch.zeros(6, 20)[:, 3:11].unflatten(1, (2, 4))
    assert rows(wide) == (wide.data_ptr(), 20)
    batch = torch.zeros(3, 5, 20)[:, :, 3:11].unflatten(2, (2, 4))
    assert rows(batch, 2)[1] == 20
    assert rows(torch.zeros(1, 5, 8).unflatten(2, (2, 4))[:, 2:4], 2)[1] == 8            # one sequence: any part of it
    assert rows(torch.zeros(3, 5, 20)[:, :1, :8].unflatten(2, (2, 4)), 2)[1] == 100      # one token each
    assert rows(torch.zeros(1, 1, 2, 4), 2)[1] == 8
    for bad in (torch.zeros(6, 4, 2).transpose(1, 2), torch.zeros(2, 6, 4).transpose(0, 1), torch.zeros(6, 2, 8)[:, :, ::2], torch.zeros(1, 2, 4).expand(6, 2, 4)):
        with pytest.raises(ValueError):
            rows(bad)
    with pytest.raises(ValueError):
        rows(torch.zeros(3, 7, 2, 4)[:, :5], 2)                                          # rows at two distances
    for kw in (dict(shape=(6, 2, 5)), dict(dtype=BF)):
        with pytest.raises(ValueError):
            rows(a, **kw)
    with pytest.raises(ValueError):
        seq._rows("t", a, a.shape, 1, 8, F32, 0)                                         # not on device 0
    with pytest.raises(ValueError):
        seq._rows("t", None, (6, 2, 4), 1, 8, F32, -1)
    with pytest.raises(ValueError):
        seq._tensor("t", a.transpose(0, 1), (2, 6, 4), F32, -1)


def test_calls_refuse_without_gpu(seq):
    if torch.cuda.is_available():
        pytest.skip("GPU present")
    layer, z = seq.GatedDelta(1, 1, 4, 4), torch.zeros
    with pytest.raises(ValueError):
        layer.fwd(z(1, 3, 1, 4), z(1, 3, 1, 4), z(1, 3, 1, 4), z(1, 3, 1), z(1, 3, 1), z(1, 3, 1, 4), z(100))
    with pytest.raises(ValueError):
        seq.BlockNorm(4, pre="rms").fwd(x=z(3, 4), h=z(3, 4))
