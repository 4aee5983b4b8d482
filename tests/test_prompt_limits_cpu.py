"""How many tokens a call of the attention of prompts takes, as the header has it."""
import pytest

from test_prompt_cpu import _args


@pytest.mark.parametrize("dtype,most", [(1, 2096895), (0, 741439)])
def test_the_tokens_of_a_call(dtype, most):
    """16 heads of 128 on 4 key heads, one sequence.  (A call below the limit gets as far as its workspace, which is missing.)"""
    from kch_b200 import _lib
    lib = _lib.load()
    size = dict(dtype=dtype, nh=16, n_kv=4, c=128, ld_q=16 * 128, ld_k=4 * 128, ld_v=4 * 128, q=1 << 20, k=1 << 40, v=1 << 41, out=1 << 42, workspace=None)
    for n, what in ((most, "workspace"), (most + 1, "more than a call takes")):
        with pytest.raises(ValueError, match=what):
            _lib.check(lib.kch_prompt_attend(_args(_lib, N=n, **size), None))
