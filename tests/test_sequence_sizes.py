"""Sizes at the ends of their ranges, on the host: what the norms' workspace function and checks answer, without a GPU."""
import ctypes as C
import random
import re
import subprocess
import sys

import pytest

FAKE = 1 << 20                     # an address that no check looks behind
LONG_MAX = (1 << 63) - 1


@pytest.fixture(scope="module")
def lib():
    from hhrl_vae_amd import _lib
    return _lib.load()


def norm_desc(M, D, gate_rows, ws_floats, gate=FAKE, **over):
    from hhrl_vae_amd import _lib
    d = _lib.BlockNormDesc()
    f = dict(dtype=0, M=M, H=1, D=D, post=2, pre=2, gate_act=0, gate_rows=gate_rows, alpha=1.0, scale=1.0, eps=1e-6, x=FAKE, y=FAKE, gate=gate, ldx=D, ldy=D,
             ldgate=D, d_out=FAKE, d_h=FAKE, lddo=D, lddh=D, dx=FAKE, dy=FAKE, lddx=D, lddy=D, dw_post=1 * FAKE, db_post=2 * FAKE, dw_pre=3 * FAKE,
             db_pre=4 * FAKE, ws=FAKE, ws_floats=ws_floats)
    f.update(over)
    for k, v in f.items():
        setattr(d, k, v)
    return d


def run(code):
    """In a process of its own, which a mistake here would end."""
    p = subprocess.run([sys.executable, "-c", "import sys; sys.path[:0] = ['.', 'tests']\nimport test_sequence_sizes as t, ctypes as C\n"
                        "from hhrl_vae_amd import _lib, sequence\nlib = _lib.load()\n" + code], capture_output=True, text=True, timeout=120)
    assert p.returncode == 0, (p.returncode, p.stderr[-500:])
    return p.stdout.split()


def test_a_gate_shared_by_more_rows_than_there_are():
    """One learned gate per channel, however many rows it is said to be for: as for the rows that there are."""
    rows = (LONG_MAX, LONG_MAX - 9, 1 << 62, 101, 100)
    sizes = run("for r in %r: print(lib.hhrl_block_norm_workspace_floats(100, 1, 64, r), sequence.BlockNorm(64, gate_rows=r).workspace(100, 'cpu').numel())" % (rows,))
    assert len(set(sizes)) == 1 and len(sizes) == 2 * len(rows) and int(sizes[0]) > 0
    # the backward call divides the rows the same way, and asks for its workspace
    for line in run("for r in %r: print(lib.hhrl_block_norm_backward(C.byref(t.norm_desc(100, 64, r, 16)), None), 'workspace' in lib.hhrl_last_error().decode(), sep=',')" % (rows,)):
        assert line == "1,True"


def test_more_rows_than_a_call_takes(lib):
    size = lib.hhrl_block_norm_workspace_floats
    for M, H in ((1 << 40, 1), (1 << 30, 1 << 10), (LONG_MAX, 1), (LONG_MAX, (1 << 31) - 1)):
        assert size(M, H, 64, 1) == 0
    for M, gate_rows in (((1 << 40) - 1, 1), ((1 << 40) - 1, 2), ((1 << 40) - 1, LONG_MAX)):
        assert 0 < size(M, 1, 64, gate_rows) < 1 << 60


@pytest.mark.parametrize("rows", [1 << 63, (1 << 64) + 3, -(1 << 64) + 1])
def test_rows_of_a_gate_that_no_long_holds(rows):
    from hhrl_vae_amd import sequence
    with pytest.raises(ValueError):
        sequence.BlockNorm(64, post="rms", gate_rows=rows)


def test_workspace_serves_a_call_without_the_optional_gate(lib):
    """A plan with a shared gate, called without one: its rows are dealt as one group, and the workspace holds those parts too.
    (A workspace one float short of what the call needs is refused and says how many that is, before anything is launched.)"""
    rng = random.Random(7)
    cases = [(9201, 8192, 4465), (10400, 8192, 40), (1002, 4096, 1001), (70, 64, 3), (1, 1, 1 << 40)]
    cases += [(rng.randint(1, 20000), rng.choice([1, 17, 100, 512, 1024, 2056, 4096, 8192]), rng.randint(2, 20000)) for _ in range(3000)]
    for M, D, gate_rows in cases:
        size = lib.hhrl_block_norm_workspace_floats(M, 1, D, gate_rows)
        for dtype in (0, 1):
            for over in (dict(), dict(db_post=None, db_pre=None)):
                for gate in (None, FAKE):
                    d = norm_desc(M, D, gate_rows, 0, gate=gate, dtype=dtype, dgate=gate, lddgate=D, **over)
                    assert lib.hhrl_block_norm_backward(C.byref(d), None) == 1
                    need = int(re.search(rb"(\d+) needed", lib.hhrl_last_error()).group(1))
                    assert need <= size, (M, D, gate_rows, dtype, gate, need, size)


@pytest.mark.parametrize("a,b", [("dw_post", "dw_pre"), ("dw_post", "db_post"), ("db_post", "db_pre"), ("dw_pre", "db_pre"), ("dw_post", "db_pre")])
@pytest.mark.parametrize("apart", [4, -4, 63 * 4, -63 * 4])
def test_parameter_gradients_that_overlap_are_refused(lib, a, b, apart):
    """Two parameter gradients are added to by different workgroups at once: arrays that overlap in part would lose sums."""
    base = 16 * FAKE
    d = norm_desc(10, 64, 1, 1 << 40, **{a: base, b: base + apart})
    assert lib.hhrl_block_norm_backward(C.byref(d), None) == 1 and b"overlap" in lib.hhrl_last_error(), lib.hhrl_last_error()


BIG = (1 << 32) + 1                # what an int of 32 bits takes for 1


@pytest.mark.parametrize("make", [
    lambda s: s.BlockNorm(64, H=BIG), lambda s: s.GatedDelta(BIG, BIG, 64, 64), lambda s: s.GatedDelta(1, BIG, 64, 64),
    lambda s: s.GatedDelta(1, 1, 64, 64).workspace(BIG, 10, "cpu"), lambda s: s.GatedDelta(1, 1, 64, 64).workspace(1, (1 << 64) + 10, "cpu"),
    lambda s: s.BlockNorm(64).workspace((1 << 64) + 10, "cpu"),
])
def test_numbers_that_the_library_would_cut_off_are_refused(make):
    from hhrl_vae_amd import sequence
    with pytest.raises(ValueError):
        make(sequence)


def test_gdr_step_counts_its_workgroups_without_overflow(lib):
    """2^30 rows of 2^30 heads of 16 column tiles are 2^64 workgroups, which a long takes for none."""
    from hhrl_vae_amd import _lib
    d = _lib.GdrStepDesc()
    n, V = 1 << 30, 256
    for k, v in dict(dtype=0, B=n, Hk=1, Hv=n, K=1, V=V - 1, scale=1.0, n_slots=n, q=FAKE, k=FAKE, v=FAKE, ldq=1, ldk=1, ldv=n * V, g=FAKE, beta=FAKE, ldg=n,
                     ldbeta=n, o=FAKE, ldo=n * V, state_in=FAKE, state_out=FAKE).items():
        setattr(d, k, v)
    assert lib.hhrl_gdr_step(C.byref(d), None) == 1 and b"too large" in lib.hhrl_last_error(), lib.hhrl_last_error()
