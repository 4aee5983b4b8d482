"""The paged cache in 4 bits against its definitions in 64 bits: rows written and read back, attention of ragged batches over the pages.

What is stored is compared bit by bit.  Tolerances of the attention as in test_gpu_paged.py: a stored value, (u - 8) s with s of 5 bits, has 8
bits at most and is exact in bf16, so that the sums are the only thing that rounds, as over bf16 pages.
"""
import types

import pytest
import torch

from test_gpu_paged import Batch, DEV, GEOMETRY, LENGTHS, close, reference
from test_gpu_paged_edges import by_rows

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def kch():
    import kch_b200
    from kch_b200 import _lib
    _lib.load()
    yield kch_b200
    assert _lib.device_status() == 0, "a device-side status was raised"


def codes4(x):
    """(values that are stored, bytes, scales) by their definition, in 64 bits.  Scales: candidates of 5 bits around a seventh of the largest
    value, the smallest that reaches it; codes: the nearest of -7 .. 7, ties to the even one."""
    y = x.double().unflatten(-1, (-1, 32))
    amax = y.abs().amax(-1)
    there = amax > 0
    power = torch.floor(torch.log2(torch.where(there, amax, 1.0) / 7)).long() - 4
    two = ((power + 1023) << 52).view(torch.double)          # (2^power by its bits: torch.ldexp goes by pow, which rounds)
    sizes = torch.tensor([15, *range(16, 33), 34], device=x.device).double() * two[..., None]
    scale = torch.where(sizes * 7 >= amax[..., None], sizes, torch.inf).amin(-1).clamp_min(2.0 ** -126)
    scale = torch.where(there, scale, 1.0)
    q = y / scale[..., None]
    low = torch.floor(q)
    up = (q - low > 0.5) | ((q - low == 0.5) & (low % 2 != 0))
    code = (low + up).flatten(-2)
    u = (code + 8).to(torch.uint8).unflatten(-1, (-1, 2))
    value = code * scale.repeat_interleave(32, -1)
    assert code.abs().max() <= 7 and torch.equal(scale.bfloat16().double(), scale) and torch.equal(value.bfloat16().double(), value)
    return value, u[..., 0] + 16 * u[..., 1], scale.bfloat16()


class Batch4(Batch):
    """Batch over a cache in 4 bits: every code and odd ones of the scales that an append can write."""

    def __init__(self, kch, new, past, **kw):
        super().__init__(_Int4(kch), new, past, **kw)
        self.cache = self.cache.real
        pool = self.cache.num_pages
        for x in ("k", "v"):
            _, byte, scale = codes4(torch.randn(pool, self.n_kv, self.page, self.c, generator=self.g, device=DEV).to(self.dtype))
            getattr(self.cache, x + "_pages").copy_(byte)
            getattr(self.cache, x + "_scales").copy_(scale)

    def values(self, x, b, n):
        ids = self.table[b, :-(-n // self.page)].long()
        byte, scale = getattr(self.cache, x + "_pages")[ids], getattr(self.cache, x + "_scales")[ids]
        code = torch.stack((byte % 16, byte // 16), -1).flatten(-2).double() - 8
        return (code * scale.double().repeat_interleave(32, -1)).transpose(0, 1).flatten(1, 2)[:, :n]


class _Int4:
    """The package as Batch calls it, which fills pages with rows: room for those beside a cache in 4 bits, whose pages Batch4 fills."""

    def __init__(self, kch):
        self.kch = kch

    def PagedKVCache(self, pages, page, n_kv, c, *a, kv_quant=None):
        room = torch.empty(pages, n_kv, page, c, device=DEV)
        return types.SimpleNamespace(k_pages=room, v_pages=room, real=self.kch.PagedKVCache(pages, page, n_kv, c, *a, kv_quant="int4"))


# ---- rows ------------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("new,past", [([1], [0]), ([1, 1, 1], [0, 15, 16]), ([0, 5, 0, 33, 17], [3, 0, 9, 31, 100]), ([300, 1, 64], [7, 8, 64])])
@pytest.mark.parametrize("dtype,c,page,n_kv", [(torch.bfloat16, 128, 16, 2), (torch.float32, 64, 32, 1), (torch.bfloat16, 96, 8, 3),
                                               (torch.float32, 256, 64, 2), (torch.bfloat16, 32, 128, 5), (torch.bfloat16, 160, 16, 1)])
def test_rows_are_written_where_they_belong_and_read_back(kch, new, past, dtype, c, page, n_kv):
    m = Batch4(kch, new, past, dtype=dtype, c=c, page=page, n_kv=n_kv, first_row=2, rows_behind=3)
    both = m.randn(m.N, 2 * n_kv * c + 8)
    k, v = (both[:, i * n_kv * c:(i + 1) * n_kv * c].unflatten(1, (n_kv, c)) for i in range(2))
    k[m.first, :, :32] = 0.          # 32 channels of zeros
    k[m.first, :, c - 1] = 1e4       # and one above all others of its 32
    want = {}
    for x, rows in (("k", k), ("v", v)):
        value, byte, scale = codes4(rows)
        pages, scales = getattr(m.cache, x + "_pages").clone(), getattr(m.cache, x + "_scales").clone()
        for b, (n, p) in enumerate(zip(new, past)):
            for i in range(n):
                row, pg, at = m.first + sum(new[:b]) + i, int(m.table[b, (p + i) // page]), (p + i) % page
                pages[pg, :, at], scales[pg, :, at] = byte[row], scale[row]
        want[x] = value, pages, scales
    m.cache.append_step(k, v, *m.args)
    got = m.cache.read_step(*m.args, n_rows=m.N)
    mine = [torch.full_like(g, 7.) for g in got]
    assert m.cache.read_step(*m.args, n_rows=m.N, out=mine)[0] is mine[0]
    live = slice(m.first, m.first + sum(new))
    for x, out, kept in zip("kv", got, mine):
        value, pages, scales = want[x]
        assert torch.equal(getattr(m.cache, x + "_pages"), pages) and torch.equal(getattr(m.cache, x + "_scales"), scales)
        assert torch.equal(out[live].double(), value[live])
        outside = torch.cat((out[:m.first], out[live.stop:]))
        assert not outside.any() and not torch.signbit(outside).any()
        assert torch.equal(kept[live], out[live]) and (kept[:m.first] == 7).all() and (kept[live.stop:] == 7).all()


def test_values_in_the_middle_between_two_codes_and_scales_next_to_5_bits(kch):
    """Quotients on, or within one rounding of, the middle between two codes; largest values on, or next to, 7 times a number of 5 bits."""
    m = Batch4(kch, [8192], [0], dtype=torch.float32, c=32, page=64, n_kv=1)
    g = torch.Generator(device=DEV).manual_seed(5)
    n = 8192
    scale = torch.ldexp(torch.randint(16, 32, (n, 1, 1), generator=g, device=DEV).float(), torch.randint(-90, 90, (n, 1, 1), generator=g, device=DEV).float())
    x = (torch.randint(-7, 7, (n, 1, 32), generator=g, device=DEV) + 0.5) * scale
    side = torch.rand(x.shape, generator=g, device=DEV)
    x = torch.where(side < 0.3, torch.nextafter(x, torch.zeros_like(x)), torch.where(side < 0.6, torch.nextafter(x, x.sign() * torch.inf), x))
    top = 7 * scale[:, :, 0]
    side = torch.rand(top.shape, generator=g, device=DEV)
    top = torch.where(side < 0.3, torch.nextafter(top, torch.zeros_like(top)), torch.where(side < 0.6, torch.nextafter(top, 2 * top), top))
    x[:, :, 9] = -top
    m.cache.append_step(x, x, *m.args)
    _, byte, want = codes4(x)
    at = m.table[0].long()
    assert torch.equal(m.cache.k_scales[at].flatten(), want.flatten()) and torch.equal(m.cache.k_pages[at].flatten(), byte.flatten())
    assert torch.equal(m.cache.v_pages[at].flatten(), byte.flatten())


def test_channels_that_are_not_finite_read_as_nan_and_the_smallest_and_largest_ones(kch):
    m = Batch4(kch, [7], [3], dtype=torch.float32, c=64, n_kv=1)
    x = m.randn(7, 1, 64)
    x[0, 0, 5], x[1, 0, 36] = torch.inf, torch.nan
    x[2] = 1e-44
    x[3, 0, :32] *= 2.0 ** -127
    x[4, 0, 0] = 7 * 2.0 ** 122
    x[5, 0, 40] = -torch.nextafter(torch.tensor(7 * 2.0 ** 122), torch.tensor(torch.inf))
    m.cache.append_step(x, x, *m.args)
    k = m.cache.read_step(*m.args, n_rows=7)[0][:, 0]
    odd = torch.zeros(7, 64, dtype=torch.bool, device=DEV)
    odd[0, :32] = odd[1, 32:] = odd[5, 32:] = True
    assert torch.equal(k.isnan(), odd) and k[~odd].isfinite().all()
    assert (k[2] - x[2, 0]).abs().max() <= 2.0 ** -127 and (k[3, :32] - x[3, 0, :32]).abs().max() <= 2.0 ** -126 / 2
    assert k[4, 0] == x[4, 0, 0]
    assert torch.equal(k[6].double(), codes4(x[6])[0][0])


# ---- attention --------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("new,past", LENGTHS)
@pytest.mark.parametrize("dtype,c,nh,n_kv,page", [g for g in GEOMETRY if g[1] % 32 == 0] + [(torch.bfloat16, 96, 6, 3, 16), (torch.float32, 160, 2, 2, 16),
                                                                                          (torch.bfloat16, 32, 2, 1, 8), (torch.bfloat16, 128, 8, 1, 8)])
def test_attention_over_the_pages(kch, new, past, dtype, c, nh, n_kv, page):
    m = Batch4(kch, new, past, dtype=dtype, c=c, n_kv=n_kv, page=page)
    q = m.randn(m.N, nh, c)
    want, tol = reference(m, q)
    got = m.cache.forward_step(q, *m.args)
    assert got.dtype == dtype
    close(got, want, tol)
    sink = torch.randn(nh, generator=m.g, device=DEV)
    want, tol = reference(m, q, scale=-0.3, window=37, sink=sink)
    close(m.cache.forward_step(q, *m.args, scale=-0.3, sliding_window=37, sink_logits=sink), want, tol)


@pytest.mark.parametrize("nh,n_kv", [(2, 2), (8, 1), (14, 1), (16, 2), (32, 1), (48, 2), (9, 3), (16, 4)])
@pytest.mark.parametrize("c", [64, 128])
def test_steps_of_one_to_four_tokens(kch, nh, n_kv, c):
    """From one row of a key head to a hundred: each form of the attention over few rows, and the one behind them."""
    for new, past in (([1, 1, 1], [400, 0, 129]), ([4, 3, 1, 4], [1000, 5, 64, 333]), ([4], [2000])):
        m = Batch4(kch, new, past, c=c, n_kv=n_kv, page=32)
        q = m.randn(m.N, nh, c)
        sink = torch.randn(nh, generator=m.g, device=DEV)
        want, tol = reference(m, q, sink=sink, window=700)
        close(m.cache.forward_step(q, *m.args, sink_logits=sink, sliding_window=700), want, tol)


@pytest.mark.parametrize("c,nh,n_kv", [(128, 8, 2), (64, 4, 1), (128, 16, 1), (64, 2, 2), (128, 14, 2)])
def test_batches_of_few_rows_with_one_long_chunk_among_them(kch, c, nh, n_kv):
    new, past = [1] * 20 + [60] + [2] * 19, [31 * i % 700 for i in range(40)]
    m = Batch4(kch, new, past, c=c, n_kv=n_kv, page=16)
    q = m.randn(m.N, nh, c)
    want, tol = reference(m, q, window=300)
    close(m.cache.forward_step(q, *m.args, sliding_window=300), want, tol)
    want, tol = reference(m, q)
    close(m.cache.forward_step(q[:20], m.table[:20], m.t0[:20], m.cu[:21]), want[:20], tol[:20])


def test_large_batches_and_long_sequences(kch):
    new, past = [1 + (i % 7 == 0) * 40 for i in range(700)], [(i * 37) % 500 for i in range(700)]
    m = Batch4(kch, new, past, n_kv=1, c=64, page=32)
    q = m.randn(m.N, 4, 64)
    want, tol = reference(m, q)
    close(m.cache.forward_step(q, *m.args), want, tol)
    m = Batch4(kch, [2], [70001], n_kv=2, page=64)
    q = m.randn(2, 8, 128)
    for window in (0, 5000):
        want, tol = reference(m, q, window=window)
        close(m.cache.forward_step(q, *m.args, sliding_window=window), want, tol)


@pytest.mark.parametrize("new", [[3, 150, 1], [3, 4, 1]])
@pytest.mark.parametrize("window", [0, 50])
@pytest.mark.parametrize("dtype,c", [(torch.bfloat16, 128), (torch.bfloat16, 64), (torch.float32, 64), (torch.bfloat16, 96)])
def test_what_a_query_does_not_see_does_not_reach_it(kch, dtype, c, window, new):
    """Scales of NaN in other pages, behind a sequence's end, ahead of a query and behind its window; those that it sees reach it."""
    past = [200, 64, 300]
    m = Batch4(kch, new, past, dtype=dtype, c=c, page=16)
    owned = torch.zeros(m.cache.num_pages, 16, dtype=torch.bool, device=DEV)
    for b, (n, p) in enumerate(zip(new, past)):
        pos = torch.arange(n + p, device=DEV)
        owned[m.table[b].long()[pos // 16], pos % 16] = True
    for scales in (m.cache.k_scales, m.cache.v_scales):
        scales.masked_fill_((~owned)[:, None, :, None].expand_as(scales), torch.nan)
    i = 40 if new[1] > 40 else 2
    q = m.randn(m.N, 4, c)
    for head, group, far in ((0, 0, 0), (1, c // 32 - 1, 0), (0, 1, 60)):      # a value's, at the chunk's token i or 60 before that
        pg, at = int(m.table[1, (64 + i - far) // 16]), (64 + i - far) % 16
        was = m.cache.v_scales[pg, head, at, group].clone()
        m.cache.v_scales[pg, head, at, group] = torch.nan
        want, tol = by_rows(m, q, window=window)
        got = m.cache.forward_step(q, *m.args, sliding_window=window)
        assert want[:3].isfinite().all()
        close(got, want, tol)
        m.cache.v_scales[pg, head, at, group] = was
    pg, at = int(m.table[1, (64 + i) // 16]), (64 + i) % 16                 # a key's
    m.cache.k_scales[pg, 1, at, 0] = torch.nan
    want, tol = by_rows(m, q, window=window)
    got = m.cache.forward_step(q, *m.args, sliding_window=window)
    assert want[:3].isfinite().all() and want[3 + i, 2:].isnan().all() and want[3 + i, :2].isfinite().all()
    close(got, want, tol)


@pytest.mark.parametrize("dtype,c", [(torch.bfloat16, 128), (torch.bfloat16, 64), (torch.float32, 64)])
def test_rows_of_no_sequence(kch, dtype, c):
    for new in ([0, 5, 0, 130, 0], [0, 1, 0, 2, 0]):
        m = Batch4(kch, new, [4, 60, 0, 3, 9], dtype=dtype, c=c, first_row=3, rows_behind=7)
        q = m.randn(m.N, 4, c)
        want, tol = reference(m, q)
        got = m.cache.forward_step(q, *m.args)
        close(got, want, tol)                               # (zeros outside)
        out = torch.full_like(q, 5.)
        assert m.cache.forward_step(q, *m.args, out=out) is out
        live = slice(3, 3 + sum(new))
        assert torch.equal(out[live], got[live]) and (out[:3] == 5).all() and (out[live.stop:] == 5).all()
        empty = torch.zeros_like(m.cu)
        assert not m.cache.forward_step(q, m.table, m.t0, empty).any()


@pytest.mark.parametrize("dtype,c", [(torch.bfloat16, 128), (torch.float32, 64)])
def test_tables_that_name_no_page_raise_the_status_and_touch_nothing_else(kch, dtype, c):
    from kch_b200 import _lib
    assert _lib.device_status() == 0
    for new in ([20, 3], [2, 1]):
        for bad in (-1, 1 << 20, -2 ** 31, 2 ** 31 - 1):
            m = Batch4(kch, new, [0, 70], dtype=dtype, c=c)
            q = m.randn(m.N, 4, c)
            m.table[1, 1] = bad
            before = m.cache.k_pages.clone()
            want, tol = by_rows(m, q, missing=[(1, 1)])
            close(m.cache.forward_step(q, *m.args), want, tol)
            torch.cuda.synchronize()
            assert _lib.device_status(reset=True) == _lib.STATUS_PAGED_TABLE
            m.table[1, 4] = bad
            k = m.randn(m.N, 2, c)
            m.cache.append_step(k, k, *m.args)
            torch.cuda.synchronize()
            assert _lib.device_status(reset=True) == _lib.STATUS_PAGED_TABLE
            changed = (m.cache.k_pages != before).flatten(1).any(1).nonzero()[:, 0]
            assert set(changed.tolist()) <= set(m.table[0].tolist())
            assert not m.cache.read_step(*m.args, n_rows=m.N)[0][new[0]:].any()
            assert _lib.device_status(reset=True) == _lib.STATUS_PAGED_TABLE


@pytest.mark.parametrize("dtype,c", [(torch.bfloat16, 128), (torch.bfloat16, 64), (torch.float32, 64)])
def test_a_captured_step_replays_with_other_lengths(kch, dtype, c):
    m = Batch4(kch, [1, 1, 1], [500, 40, 300], dtype=dtype, c=c, n_kv=2, wider=5)
    q, k, v = m.randn(3, 8, c), m.randn(3, 2, c), m.randn(3, 2, c)
    t0 = m.t0.clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        m.cache.append_step(k, v, m.table, t0, m.cu)
        m.cache.forward_step(q, m.table, t0, m.cu)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        m.cache.append_step(k, v, m.table, t0, m.cu)
        out = m.cache.forward_step(q, m.table, t0, m.cu)
    for past in ([500, 40, 300], [7, 0, 77], [499, 39, 2]):
        t0.copy_(torch.tensor(past, dtype=torch.int32))
        for x in (q, k, v):
            x.copy_(m.randn(*x.shape))
        graph.replay()
        m.past = past
        want, tol = reference(m, q)
        close(out, want, tol)
        assert torch.equal(out, m.cache.forward_step(q, m.table, t0, m.cu))


@pytest.mark.parametrize("new,past", [([1, 3, 1], [300, 40, 129]), ([40, 200], [100, 64])])
@pytest.mark.parametrize("dtype,c", [(torch.bfloat16, 128), (torch.bfloat16, 64), (torch.float32, 64)])
def test_a_pool_from_elsewhere_with_codes_of_0_and_scales_of_both_signs(kch, dtype, c, new, past):
    """Code 0 stands for -8 scales, which no append writes; a scale below 0 turns its 32 channels over."""
    m = Batch4(kch, new, past, dtype=dtype, c=c, page=16)
    for x in ("k", "v"):
        pages, scales = getattr(m.cache, x + "_pages"), getattr(m.cache, x + "_scales")
        pages.copy_(torch.randint(0, 256, pages.shape, generator=m.g, device=DEV, dtype=torch.uint8))
        scales.mul_(torch.where(torch.rand(scales.shape, generator=m.g, device=DEV) < 0.5, -1., 1.))
    q = m.randn(m.N, 4, c)
    want, tol = reference(m, q, window=200)
    close(m.cache.forward_step(q, *m.args, sliding_window=200), want, tol)
    got = m.cache.read_step(*m.args, n_rows=m.N)[0]
    for b, (n, p) in enumerate(zip(new, past)):
        rows = got[sum(new[:b]):sum(new[:b + 1])]
        assert torch.equal(rows.double(), m.values("k", b, p + n)[:, p:].transpose(0, 1))


@pytest.mark.parametrize("new,past", [([1, 1], [33, 700]), ([40, 300], [100, 900])])
@pytest.mark.parametrize("dtype,c", [(torch.bfloat16, 128), (torch.bfloat16, 64), (torch.float32, 64)])
def test_strided_queries_and_outputs_and_rows_that_begin_on_16_bytes_and_no_more(kch, dtype, c, new, past):
    m = Batch4(kch, new, past, dtype=dtype, c=c)
    q = m.randn(m.N, 6, c)
    want = m.cache.forward_step(q, *m.args)
    ahead = 16 // want.element_size()
    room = torch.full((ahead + want.numel() + ahead,), 7.0, dtype=dtype, device=DEV)
    out = room[ahead:ahead + want.numel()].view(want.shape)
    assert out.data_ptr() % 32 == 16
    m.cache.forward_step(q, *m.args, out=out)
    assert torch.equal(out, want) and (room[:ahead] == 7).all() and (room[-ahead:] == 7).all()
    wide = torch.randn(m.N, 6 * c + 3 * ahead, device=DEV).to(dtype)
    wide[:, ahead:ahead + 6 * c] = q.flatten(1)
    assert torch.equal(m.cache.forward_step(wide[:, ahead:ahead + 6 * c].unflatten(1, (6, c)), *m.args), want)
    rows = m.cache.read_step(*m.args, n_rows=m.N)
    rooms = [torch.full((ahead + rows[0].numel() + ahead,), 7.0, dtype=dtype, device=DEV) for _ in range(2)]
    outs = tuple(r[ahead:ahead + rows[0].numel()].view(rows[0].shape) for r in rooms)
    m.cache.read_step(*m.args, n_rows=m.N, out=outs)
    for got, kept, r in zip(rows, outs, rooms):
        assert torch.equal(got, kept) and (r[:ahead] == 7).all() and (r[-ahead:] == 7).all()


@pytest.mark.parametrize("B,N,n_kv", [(4096, 4096, 16), (4096, 16400, 16), (32, 65536, 128)])
def test_lengths_that_fall_and_rise_again_beyond_what_is_counted_do_nothing(kch, B, N, n_kv):
    """Every other sequence has all rows: more steps in all than 32 bits hold, which the host, who sees N alone, cannot know."""
    from kch_b200 import _lib
    assert _lib.device_status() == 0
    cache = kch.PagedKVCache(1, 256, n_kv, 64, DEV, torch.bfloat16, kv_quant="int4")
    table = torch.zeros(B, 4096, dtype=torch.int32, device=DEV)
    t0 = torch.full((B,), 4096 * 256 - N, dtype=torch.int32, device=DEV)
    cu = (torch.arange(B + 1, device=DEV) % 2 * N).int()
    q, out = torch.zeros(N, n_kv, 64, dtype=torch.bfloat16, device=DEV), torch.full((N, n_kv, 64), 7.0, dtype=torch.bfloat16, device=DEV)
    cache.forward_step(q, table, t0, cu, out=out)
    torch.cuda.synchronize()
    assert _lib.device_status(reset=True) == _lib.STATUS_PAGED_TABLE
    assert (out == 7).all()


def test_calls_on_two_streams_at_once_and_again(kch):
    a, b = (Batch4(kch, new, [97 * i for i in range(20)], n_kv=2, seed=s) for s, new in ((1, [1] * 20), (2, [1] * 10 + [50] * 10)))
    qa, qb = a.randn(a.N, 16, 128), b.randn(b.N, 16, 128)
    want = [a.cache.forward_step(qa, *a.args), b.cache.forward_step(qb, *b.args)]
    torch.cuda.synchronize()
    s, got = [torch.cuda.Stream(), torch.cuda.Stream()], [[], []]
    for _ in range(10):
        for i, (m, q) in enumerate(((a, qa), (b, qb))):
            with torch.cuda.stream(s[i]):
                got[i].append(m.cache.forward_step(q, *m.args))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(g, want[i]) for g in got[i])


def test_offsets_that_pass_32_bits(kch):
    """A pool whose rows lie beyond 2^32 bytes, and twice that in codes."""
    pages, page, c = 2 ** 32 // (64 * 64) + 40, 64, 128
    k, v = (torch.empty(pages, 1, page, c // 2, dtype=torch.uint8, device=DEV) for _ in range(2))
    ks, vs = (torch.empty(pages, 1, page, c // 32, dtype=torch.bfloat16, device=DEV) for _ in range(2))
    cache = kch.PagedKVCache(pages, page, 1, c, DEV, torch.bfloat16, kv_quant="int4", storage=(k, v, ks, vs))
    table = torch.arange(pages - 1, pages - 6, -1, dtype=torch.int32, device=DEV)[None]
    x = torch.randn(300, 1, c, device=DEV).bfloat16()
    for n in (300, 2):                                      # a chunk, and a step
        t0, cu = torch.tensor([300 - n], dtype=torch.int32, device=DEV), torch.tensor([0, n], dtype=torch.int32, device=DEV)
        cache.append_step(x[300 - n:], x[300 - n:], table, t0, cu)
        got = cache.read_step(table, t0, cu, n_rows=n)
        value = codes4(x)[0]
        assert torch.equal(got[0].double(), value[300 - n:]) and torch.equal(got[1], got[0])
        q = torch.randn(n, 2, c, device=DEV).bfloat16()
        o = cache.forward_step(q, table, t0, cu)
        hidden = torch.arange(300, device=DEV) > torch.arange(300 - n, 300, device=DEV)[:, None]
        p = (q[:, 1].double() @ value[:, 0].T * c ** -0.5).masked_fill(hidden, -torch.inf).softmax(1)
        assert ((o[:, 1].double() - p @ value[:, 0]).abs() <= 2.0 ** -7 * (p @ value[:, 0].abs()) + 2.0 ** -8).all()


def test_a_prompt_turned_attended_kept_in_4_bits_and_continued(kch):
    """A run of the operators together: queries and keys of two prompts turned by their positions, attended as a whole, kept in 4 bits, and
    three steps of tokens behind them, whose attention runs over what was kept."""
    nh, n_kv, c, page = 8, 2, 128, 16
    g = torch.Generator(device=DEV).manual_seed(9)
    rope = kch.RotaryPositions(c, DEV, sections=(16, 24, 24))
    cache = kch.PagedKVCache(64, page, n_kv, c, DEV, torch.bfloat16, kv_quant="int4")
    table = torch.randperm(64, generator=g, device=DEV).view(2, 32).to(torch.int32)
    lengths, kept = [300, 77], [[], []]
    t0 = torch.zeros(2, dtype=torch.int32, device=DEV)
    for step in range(4):
        new = lengths if step == 0 else [1, 1]
        n = sum(new)
        cu = torch.tensor([0, new[0], n], dtype=torch.int32, device=DEV)
        both = torch.randn(n, (nh + 2 * n_kv) * c, generator=g, device=DEV).bfloat16()
        q, k, v = (x.unflatten(1, (-1, c)) for x in both.split((nh * c, n_kv * c, n_kv * c), 1))
        pos = torch.cat([torch.arange(a, device=DEV) + b for a, b in zip(new, t0.tolist())])[:, None].expand(-1, 3).to(torch.int32)
        q, k = rope.rotate(q, k, pos)
        cache.append_step(k, v, table, t0, cu)
        o = kch.prompt_attention(q, k, v, cu) if step == 0 else cache.forward_step(q, table, t0, cu)
        for b in range(2):
            r = slice(int(cu[b]), int(cu[b + 1]))
            old = kept[b]
            kept[b] = [torch.cat([*(old[i:i + 1] if old else []), codes4(x[r])[0]]) for i, x in enumerate((k, v))]
            keys, values = (k[r].double(), v[r].double()) if step == 0 else kept[b]
            total = keys.shape[0]
            hidden = torch.arange(total, device=DEV) > torch.arange(total - new[b], total, device=DEV)[:, None]
            for h in range(nh):
                l = (q[r, h].double() @ keys[:, h // 4].T * c ** -0.5).masked_fill(hidden, -torch.inf)
                p = l.softmax(1)
                size = c ** -0.5 * (q[r, h].double().abs() @ keys[:, h // 4].abs().T).masked_fill(hidden, 0.).amax(1, keepdim=True)
                rel = 2 * (c + 4) * 2.0 ** -24 * size + (total + 64) * 2.0 ** -24 + 2.0 ** -8
                want, weight = p @ values[:, h // 4], p @ values[:, h // 4].abs()
                assert ((o[r, h].double() - want).abs() <= rel * weight + 2.0 ** -8 * want.abs()).all()
        t0 += torch.tensor(new, dtype=torch.int32, device=DEV)
    got = cache.read_step(table, torch.zeros_like(t0), torch.tensor([0, 303, 383], dtype=torch.int32, device=DEV), n_rows=383)
    for i in range(2):
        assert torch.equal(got[i].double(), torch.cat([kept[0][i], kept[1][i]]))


def test_what_python_refuses(kch):
    with pytest.raises(ValueError, match="multiple of 32"):
        kch.PagedKVCache(4, 16, 1, 72, DEV, torch.bfloat16, kv_quant="int4")
    k, s = torch.zeros(4, 1, 16, 32, dtype=torch.uint8, device=DEV), torch.ones(4, 1, 16, 2, dtype=torch.bfloat16, device=DEV)
    kch.PagedKVCache(4, 16, 1, 64, DEV, torch.bfloat16, kv_quant="int4", storage=(k, k, s, s))
    for storage, what in (((k.view(torch.int8), k, s, s), "k_pages"), ((k, k[:, :, :, :16], s, s), "v_pages"), ((k, k, s.float(), s), "k_scales"),
                          ((k, k, s, s[..., :1]), "v_scales"), ((k, k, None, None), "k_scales")):
        with pytest.raises(ValueError, match=what):
            kch.PagedKVCache(4, 16, 1, 64, DEV, torch.bfloat16, kv_quant="int4", storage=storage)
    fresh = kch.PagedKVCache(4, 16, 1, 64, DEV, torch.float32, kv_quant="int4")
    table, zero = torch.zeros(1, 1, dtype=torch.int32, device=DEV), torch.zeros(1, dtype=torch.int32, device=DEV)
    rows = fresh.read_step(table, zero, torch.tensor([0, 16], dtype=torch.int32, device=DEV), n_rows=16)
    assert not rows[0].any() and not rows[1].any()          # a new cache holds zeros
