"""What the attention of prompts refuses before any launch: in Python and by the C entry point."""
import ctypes

import pytest
import torch


def _args(lib_mod, **over):
    """Arguments of kch_prompt_attend that pass every check up to the workspace's; the pointers are never followed."""
    v = dict(q=4096, k=8192, v=12288, ld_q=256, ld_k=128, ld_v=128, cu_seqlens=4096, B=1, N=3, dtype=1, nh=4, n_kv=2, c=64, scale=0.125,
             sliding_window=0, sink=None, sink_dtype=0, out=16384, zero_rest=1, workspace=4096, workspace_bytes=0)
    v.update(over)
    a = lib_mod.PromptAttendArgs()
    for name, x in v.items():
        setattr(a, name, x)
    return a


@pytest.mark.parametrize("over,what", [
    (dict(dtype=2), "dtype"), (dict(c=60), "c=60"), (dict(c=0), "c=0"), (dict(c=264), "c=264"), (dict(n_kv=0), "n_kv=0"), (dict(nh=3), "nh=3"), (dict(nh=0), "nh=0"),
    (dict(B=0), "B=0"), (dict(B=4097), "B=4097"), (dict(N=-1), "N=-1"), (dict(N=1 << 31), "N="), (dict(cu_seqlens=None), "null cu_seqlens"),
    (dict(sliding_window=-1), "sliding_window"), (dict(scale=float("inf")), "scale"), (dict(scale=3e38), "scale"), (dict(sink=4096, sink_dtype=2), "sink"),
    (dict(q=None), "null q"), (dict(k=None), "null q"), (dict(v=None), "null q"), (dict(out=None), "null q"), (dict(q=4098), "q must be"),
    (dict(k=8200), "k must be"), (dict(ld_v=127), "v must be"), (dict(ld_k=132), "k must be"), (dict(ld_q=248), "q must be"), (dict(out=16392), "out must be"),
    (dict(out=4096 + 2 * 256 * 2), "out overlaps q"), (dict(out=8192 - 16), "out overlaps k"), (dict(out=12288 + 2 * 2 * 128 + 240), "out overlaps v"),
    (dict(ld_v=1 << 20, out=12288 + 2 * (1 << 20)), "out overlaps v"),
    (dict(), "workspace"), (dict(workspace=None, workspace_bytes=1 << 40), "workspace"), (dict(workspace=4112, workspace_bytes=1 << 40), "workspace"),
    (dict(N=1 << 24, nh=32, ld_q=32 * 64, q=1 << 20, k=1 << 40, v=1 << 41, out=1 << 42, workspace_bytes=1 << 40), "more than a call takes"),
    (dict(N=1 << 30), "N \\* nh")])
def test_arguments_are_refused_by_name(over, what):
    from kch_b200 import _lib
    lib = _lib.load()
    with pytest.raises(ValueError, match=what):
        _lib.check(lib.kch_prompt_attend(_args(_lib, **over), None))


def test_no_rows_are_no_work_and_the_workspace_grows_with_the_width():
    from kch_b200 import _lib
    lib = _lib.load()
    assert lib.kch_prompt_attend(_args(_lib, N=0, q=None, out=None), None) == 0
    with pytest.raises(ValueError, match="null arguments"):
        _lib.check(lib.kch_prompt_attend(None, None))
    sizes = [int(lib.kch_prompt_attend_workspace_bytes(_args(_lib, c=c))) for c in (64, 128, 256)]
    assert 0 < sizes[0] < sizes[1] < sizes[2]
    assert lib.kch_prompt_attend_workspace_bytes(None) == 0 and lib.kch_prompt_attend_workspace_bytes(_args(_lib, n_kv=0)) == 0
    assert ctypes.sizeof(_lib.PromptAttendArgs) == 144


def test_cpu_tensors_and_shapes_are_refused():
    from kch_b200 import prompt_attention
    q, k, cu = torch.zeros(3, 4, 64), torch.zeros(3, 2, 64), torch.tensor([0, 3], dtype=torch.int32)
    with pytest.raises(RuntimeError, match="CUDA"):
        prompt_attention(q, k, k, cu)
    with pytest.raises(TypeError, match="float16"):
        prompt_attention(q.half(), k.half(), k.half(), cu)
