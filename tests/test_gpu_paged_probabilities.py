"""Steps of up to 16 rows of a key head carry the bits that rounding a probability to bf16 leaves, whatever the pages hold.

The keys of a sequence are in turns one of logit 0 and one of logit log(1 - e), e between 2^-10 and 2^-9: a probability 1 - e lies less than half a
step of bf16 (2^-8 below 1) from 1, and alone it would be 1.  Values are 7 and -7, so that an output is 7 e / 2 or so, and it would be 0 (or what an odd number of
keys leaves).  Tolerance: a probability in two terms of bf16 is off by 2^-18 of itself; logits, powers and sums as in test_gpu_paged.py (d and (n + 64)
2^-24); 8-bit pages: the product with a value's scale rounds once, 2^-24; the output rounds by half a step, 2^-8 of itself."""
import math

import pytest
import torch

from test_gpu_paged import Batch, DEV
from test_gpu_paged_int4 import Batch4

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def kch():
    import kch_b200
    from kch_b200 import _lib
    _lib.load()
    yield kch_b200
    assert _lib.device_status() == 0, "a device-side status was raised"


@pytest.mark.parametrize("new,past", [([1, 1, 1], [0, 129, 700]), ([2, 1, 2], [31, 400, 5]), ([4, 4, 3], [300, 64, 1000]), ([1], [5000])])
@pytest.mark.parametrize("nh", [1, 3, 4, 5, 7, 8, 9, 12, 16])
@pytest.mark.parametrize("kind", [None, "fp8", "int8", "int4"])
@pytest.mark.parametrize("c", [64, 128])
def test_what_rounding_a_probability_leaves_is_not_lost(kch, c, kind, nh, new, past):
    if nh * sum(new) > 16 * len(new):
        pytest.skip("more than 16 rows a sequence: another form")
    m = Batch4(kch, new, past, c=c, n_kv=1, page=32) if kind == "int4" else Batch(kch, new, past, c=c, n_kv=1, page=32, kind=kind)
    total = [n + p for n, p in zip(new, past)]
    low = torch.cat([torch.arange(n, device=DEV) % 2 for n in total]).bool()
    k, v = (torch.zeros(len(low), 1, c, dtype=torch.bfloat16, device=DEV) for _ in range(2))
    k[low, 0, 0] = 7.
    v[:] = torch.where(low, -7., 7.)[:, None, None]
    cu = torch.tensor([sum(total[:i]) for i in range(len(total) + 1)], dtype=torch.int32, device=DEV)
    m.cache.append_step(k, v, m.table, torch.zeros_like(m.t0), cu)
    q = torch.zeros(m.N, nh, c, dtype=torch.bfloat16, device=DEV)
    q[:, :, 0] = math.log(1 - 2.0 ** -10) / 7 * (1 + torch.arange(nh, device=DEV) / 17)
    got = m.cache.forward_step(q, *m.args, scale=1.0).double()
    for b, (n, p) in enumerate(zip(new, past)):
        kk, vv = m.values("k", b, p + n)[0], m.values("v", b, p + n)[0]
        hidden = torch.arange(p + n, device=DEV) > torch.arange(p, p + n, device=DEV)[:, None]
        for h in range(nh):
            qq = q[sum(new[:b]):sum(new[:b + 1]), h].double()
            w = (qq @ kk.T).masked_fill(hidden, -torch.inf).softmax(1)
            want, weight = w @ vv, w @ vv.abs()
            d = (c + 4) * 2.0 ** -24 * (qq.abs() @ kk.abs().T).amax(1, keepdim=True)
            tol = (2 * d + (p + n + 64) * 2.0 ** -24 + 2.0 ** -18 + 2.0 ** -24) * weight + 2.0 ** -8 * want.abs()
            off = (got[sum(new[:b]):sum(new[:b + 1]), h] - want).abs()
            assert (off <= tol).all(), f"sequence {b}, head {h}: {float((off / tol).max()):.2f} of the tolerance"
