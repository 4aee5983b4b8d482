"""Any number of heads of a key head: blocks of whole tokens are then any number of rows, an odd one of a warpgroup's among them.  Items in parts, in one piece, and
both in a call; oracles and tolerances are those of test_gpu_paged.py."""
import pytest
import torch

from test_gpu_paged import DEV, close, reference
from test_gpu_paged_int4 import Batch4
from test_gpu_prompt import Prompts

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def kch():
    import kch_b200
    from kch_b200 import _lib
    _lib.load()
    yield kch_b200
    assert _lib.device_status() == 0, "a device-side status was raised"


HEADS = [5, 6, 9, 11, 13, 15, 17, 25, 31, 41, 63, 65, 127, 128, 129]


@pytest.mark.parametrize("G", HEADS)
@pytest.mark.parametrize("c,n_kv,new", [(128, 2, [700, 33, 1]), (64, 1, [1500]), (128, 1, [300] * 9), (64, 3, [130, 257])])
def test_prompts(kch, c, n_kv, new, G):
    m = Prompts(new, nh=G * n_kv, n_kv=n_kv, c=c)
    sink = torch.randn(G * n_kv, generator=m.g, device=DEV)
    for kw in (dict(), dict(scale=-0.3, window=200, sink=sink)):
        want, tol = reference(m, m.q, **kw)
        got = kch.prompt_attention(*m.args, scale=kw.get("scale"), sliding_window=kw.get("window", 0), sink_logits=kw.get("sink"))
        close(got, want, tol)


@pytest.mark.parametrize("G", HEADS)
@pytest.mark.parametrize("c,n_kv,new,past", [(128, 2, [200, 33, 1], [900, 2000, 50]), (64, 1, [100], [7000]), (128, 1, [40] * 9, [300] * 9)])
def test_chunks_over_4_bit_pages(kch, c, n_kv, new, past, G):
    m = Batch4(kch, new, past, c=c, n_kv=n_kv, page=32)
    q = m.randn(m.N, G * n_kv, c)
    sink = torch.randn(G * n_kv, generator=m.g, device=DEV)
    for kw in (dict(), dict(scale=-0.3, window=200, sink=sink)):
        want, tol = reference(m, q, **kw)
        got = m.cache.forward_step(q, *m.args, scale=kw.get("scale"), sliding_window=kw.get("window", 0), sink_logits=kw.get("sink"))
        close(got, want, tol)
