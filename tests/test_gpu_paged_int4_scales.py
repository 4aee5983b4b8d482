"""Scales that no append writes, in places of a 4-bit pool that no query sees: memory that something else has left behind a sequence's end, before
its window and in pages that are not its own.  Oracle and tolerances are those of test_gpu_paged.py."""
import pytest
import torch

from test_gpu_paged import DEV, close, reference
from test_gpu_paged_int4 import Batch4

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def kch():
    import kch_b200
    from kch_b200 import _lib
    _lib.load()
    yield kch_b200
    assert _lib.device_status() == 0, "a device-side status was raised"


LARGEST = torch.finfo(torch.bfloat16).max
ODD = [torch.nan, torch.inf, -torch.inf, LARGEST, -LARGEST, 1.5 * 2.0 ** 123]
FORMS = [(torch.bfloat16, 128), (torch.bfloat16, 64), (torch.float32, 64), (torch.bfloat16, 96)]


def seen_by_some(m, window):
    """[pool, page]: the rows of the pool that some query of the batch sees."""
    seen = torch.zeros(m.cache.num_pages, m.page, dtype=torch.bool, device=DEV)
    for b, (n, p) in enumerate(zip(m.new, m.past)):
        pos = torch.arange(max(p - window + 1, 0) if window else 0, n + p, device=DEV)
        seen[m.table[b].long()[pos // m.page], pos % m.page] = True
    return seen


# (2, 8 and 14 rows of a key head, which are the steps' forms, and chunks)
@pytest.mark.parametrize("odd", ODD)
@pytest.mark.parametrize("new", [[1, 1, 1], [3, 4, 1], [3, 150, 1]])
@pytest.mark.parametrize("window", [0, 50])
@pytest.mark.parametrize("dtype,c", FORMS)
@pytest.mark.parametrize("nh,n_kv", [(4, 2), (14, 1)])
def test_what_lies_where_no_query_sees_reaches_none(kch, nh, n_kv, dtype, c, window, new, odd):
    m = Batch4(kch, new, [200, 67, 300], dtype=dtype, c=c, n_kv=n_kv, page=16)
    q = m.randn(m.N, nh, c)
    want, tol = reference(m, q, window=window)
    hidden = (~seen_by_some(m, window))[:, None, :, None]
    for scales in (m.cache.k_scales, m.cache.v_scales):
        scales.masked_fill_(hidden.expand_as(scales), odd)
    got = m.cache.forward_step(q, *m.args, sliding_window=window)
    assert got.isfinite().all()
    close(got, want, tol)


@pytest.mark.parametrize("odd", [torch.inf, -torch.inf])
@pytest.mark.parametrize("new", [[3, 4, 1], [3, 150, 1]])
@pytest.mark.parametrize("dtype,c", FORMS)
@pytest.mark.parametrize("nh,n_kv", [(4, 2), (6, 2)])
def test_an_infinity_among_the_scales_of_values_reaches_those_that_see_it_alone(kch, nh, n_kv, dtype, c, new, odd):
    m = Batch4(kch, new, [200, 64, 300], dtype=dtype, c=c, n_kv=n_kv, page=16)
    i, head, group = (40 if new[1] > 40 else 2), 1, c // 32 - 1
    pg, at = int(m.table[1, (64 + i) // 16]), (64 + i) % 16
    q = m.randn(m.N, nh, c)
    want, tol = reference(m, q)
    m.cache.v_scales[pg, head, at, group] = odd
    got = m.cache.forward_step(q, *m.args)
    reached = torch.zeros(m.N, nh, c, dtype=torch.bool, device=DEV)
    reached[3 + i:3 + new[1], head * nh // n_kv:(head + 1) * nh // n_kv, 32 * group:] = True
    assert got[~reached].isfinite().all() and not got[reached].isfinite().any()
    close(torch.where(reached, 0., got), torch.where(reached, 0., want), tol)


def test_a_pool_whose_last_page_holds_anything_behind_its_rows(kch):
    """Bytes of every kind: codes and scales from all 16 bits, behind the ends of a page's rows and in the pages of nobody."""
    m = Batch4(kch, [1] * 40, [7 * i % 333 for i in range(40)], c=128, n_kv=2, page=64, spare=9)
    q = m.randn(m.N, 8, 128)
    want, tol = reference(m, q)
    hidden = (~seen_by_some(m, 0))[:, None, :, None]
    for x in ("k", "v"):
        for part, dt, most in (("_pages", torch.uint8, 2 ** 8), ("_scales", torch.int16, 2 ** 16)):
            t = getattr(m.cache, x + part).view(dt)
            t.copy_(torch.where(hidden, torch.randint(0, most, t.shape, generator=m.g, device=DEV).to(dt), t))
    close(m.cache.forward_step(q, *m.args), want, tol)
