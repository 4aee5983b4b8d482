"""What the rotary positions refuse before any launch: by the class's own checks and by the C entry point."""
import ctypes

import pytest
import torch


def test_constructor_arguments():
    import kch_b200
    for args, kw, what in (((60,), {}, "c=60"), ((264,), {}, "c=264"), ((4,), {}, "c=4"), ((True,), {}, "c=True"), ((64.0,), {}, "c=64.0"),
                           ((64,), dict(rotary_dim=66), "rotary_dim=66"), ((64,), dict(rotary_dim=31), "even"), ((64,), dict(rotary_dim=0), "rotary_dim=0"),
                           ((64,), dict(sections=(16, 15)), "31 pairs"), ((64,), dict(sections=()), "1 to 4 axes"),
                           ((64,), dict(sections=(8, 8, 8, 4, 4)), "1 to 4 axes"), ((64,), dict(sections=(40, -8)), "pairs of an axis"),
                           ((64,), dict(base=0.0), "base"), ((64,), dict(base=float("inf")), "base"), ((64,), dict(base=-3), "base"),
                           ((64,), dict(inv_freq=[1.0] * 31), "32 finite"), ((64,), dict(inv_freq=[float("nan")] * 32), "32 finite")):
        with pytest.raises(ValueError, match=what):
            kch_b200.RotaryPositions(*args, "cuda", **kw)
    with pytest.raises(RuntimeError, match="CUDA"):
        kch_b200.RotaryPositions(64, "cpu")


# q_out and k_out behind q [3, 4, 64] and k [3, 2, 64] of bf16
Q, K, QO, KO = 4096, 8192, 12288, 16384


def _args(lib_mod, **over):
    v = dict(q=Q, k=K, q_out=QO, k_out=KO, ld_q=256, ld_k=128, ld_q_out=256, ld_k_out=128, N=3, nh=4, n_kv=2, c=64, dtype=1, positions=4096,
             ld_positions=2, axes=2, sections=(20, 12, 0, 0), turns=4096, rotary_dim=64, neighbours=0, inverse=0)
    v.update(over)
    a = lib_mod.RotaryArgs()
    for name, x in v.items():
        setattr(a, name, x)
    return a


@pytest.mark.parametrize("over,what", [
    (dict(dtype=2), "dtype"), (dict(c=60), "c=60"), (dict(c=264), "c=264"), (dict(rotary_dim=0), "rotary_dim=0"), (dict(rotary_dim=63), "rotary_dim=63"),
    (dict(rotary_dim=66), "rotary_dim=66"), (dict(nh=0), "nh=0"), (dict(n_kv=-1), "n_kv=-1"), (dict(axes=0), "axes=0"), (dict(axes=5), "axes=5"),
    (dict(sections=(20, 11, 0, 0)), "31 pairs"), (dict(sections=(-1, 33, 0, 0)), "sections\\[0\\]"), (dict(N=-1), "N=-1"), (dict(N=1 << 31), "N="),
    (dict(positions=None), "null positions"), (dict(turns=None), "null positions"), (dict(ld_positions=1), "1 apart"), (dict(q=None), "null q"),
    (dict(k=None), "null q"), (dict(q_out=None), "null q"), (dict(k_out=None), "null q"), (dict(q=4098), "q must be 16-byte"),
    (dict(ld_k=127), "k must be"), (dict(ld_q_out=260), "q_out must be"), (dict(ld_q=248), "q must be"),
    (dict(q_out=Q + 16), "q_out overlaps q"), (dict(q_out=K), "q_out overlaps k"), (dict(k_out=Q), "k_out overlaps q"), (dict(k_out=QO), "k_out overlaps q_out|q_out overlaps k_out"),
    (dict(q_out=Q, ld_q_out=264), "q_out overlaps q"), (dict(k_out=K + 2 * (2 * 128 + 120)), "k_out overlaps k")])
def test_arguments_are_refused_by_name(over, what):
    from kch_b200 import _lib
    lib = _lib.load()
    with pytest.raises(ValueError, match=what):
        _lib.check(lib.kch_rotary(_args(_lib, **over), None))


def test_slices_of_a_fused_projection_that_meet_are_refused():
    """Tokens 512 elements apart: q the first 256 of them, k the next 128; outputs that reach into the other's columns, from either side."""
    from kch_b200 import _lib
    lib = _lib.load()
    fused = dict(ld_q=512, ld_k=512, q=Q, k=Q + 2 * 256, ld_q_out=512, ld_k_out=512)
    for over, what in ((dict(q_out=Q, k_out=Q + 2 * 248), "overlaps"), (dict(q_out=Q + 2 * 384, k_out=Q + 2 * 256), "q_out overlaps q"),
                       (dict(q_out=Q + 2 * 512, k_out=Q + 2 * 256), "q_out overlaps q")):
        with pytest.raises(ValueError, match=what):
            _lib.check(lib.kch_rotary(_args(_lib, **fused, **over), None))


def test_no_rows_are_no_work_and_null_arguments_are_refused():
    from kch_b200 import _lib
    lib = _lib.load()
    assert lib.kch_rotary(_args(_lib, N=0, q=None, k=None, positions=None), None) == 0
    with pytest.raises(ValueError, match="null arguments"):
        _lib.check(lib.kch_rotary(None, None))
    assert ctypes.sizeof(_lib.RotaryArgs) == 152


def test_cpu_tensors_are_refused():
    import kch_b200
    rope = object.__new__(kch_b200.RotaryPositions)
    rope.c, rope.device, rope._index, rope.sections, rope._axes = 64, torch.device("cuda:0"), 0, (32,), 1
    with pytest.raises(RuntimeError, match="CUDA"):
        rope.rotate(torch.zeros(3, 4, 64), None, torch.zeros(3, dtype=torch.int32))
    with pytest.raises(ValueError, match="q must be"):
        rope.rotate(torch.zeros(3, 4, 32), None, torch.zeros(3, dtype=torch.int32))
