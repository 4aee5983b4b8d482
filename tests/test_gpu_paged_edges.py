"""The paged cache where numbers, masks, tables and lengths run out: what a query sees reaches it whatever it is, what it does not see
does not, and a batch with an entry at fault leaves the others alone.

The reference takes a row's visible keys alone, in 64 bits, and takes nothing out of them.  Tolerances as in test_gpu_paged.py.
"""
import pytest
import torch

from test_gpu_paged import Batch, DEV, close

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def kch():
    import kch_b200
    from kch_b200 import _lib
    _lib.load()
    yield kch_b200
    assert _lib.device_status() == 0, "a device-side status was raised"


def by_rows(m, q, *, window=0, missing=()):
    """(outputs, tolerances) in 64 bits, a row at a time over the keys that it sees.  missing: (sequence, page index) pairs whose table entry
    names no page: zeros."""
    G, scale = q.shape[1] // m.n_kv, m.c ** -0.5
    out = torch.zeros(q.shape, dtype=torch.double, device=DEV)
    tol = torch.zeros_like(out)
    for b, (n, p) in enumerate(zip(m.new, m.past)):
        r0 = m.first + sum(m.new[:b])
        if n == 0:
            continue
        whole = m.table.clone()
        m.table = m.table.clamp(0, m.cache.num_pages - 1)
        k, v = (m.values(x, b, p + n).clone() for x in "kv")
        m.table = whole
        for s, page in missing:
            if s == b:
                k[:, page * m.page:(page + 1) * m.page] = 0.
                v[:, page * m.page:(page + 1) * m.page] = 0.
        for i in range(n):
            lo, hi = max(0, p + i + 1 - window) if window else 0, p + i + 1
            kk, vv = (x[:, lo:hi].repeat_interleave(G, 0) for x in (k, v))              # [nh, keys, c]
            qq = q[r0 + i].double()[:, None]
            l = scale * (qq * kk).sum(-1)
            w = (l - l.amax(-1, keepdim=True)).exp()
            w = w / w.sum(-1, keepdim=True)
            out[r0 + i] = (w[..., None] * vv).sum(1)
            size = scale * (qq.abs() * kk.abs()).sum(-1).nan_to_num(0., 0., 0.).amax(-1)
            rel = 2 * (m.c + 4) * 2.0 ** -24 * size + (hi - lo + 64) * 2.0 ** -24
            if m.dtype == torch.bfloat16:
                rel = rel + 2.0 ** -8
            tol[r0 + i] = rel[:, None] * (w[..., None] * vv.abs()).nan_to_num(0., 0., 0.).sum(1)
            if m.dtype == torch.bfloat16:
                tol[r0 + i] += 2.0 ** -8 * out[r0 + i].nan_to_num(0., 0., 0.).abs()
    return out, tol


def at(m, b, pos):
    return int(m.table[b, pos // m.page]), pos % m.page


# ---- numbers ---------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("col", range(8))
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), float("-inf")])
@pytest.mark.parametrize("dtype,c", [(torch.bfloat16, 128), (torch.bfloat16, 64), (torch.float32, 64)])
def test_a_visible_key_that_is_not_finite(kch, dtype, c, bad, col):
    """A logit that is NaN or +inf makes the rows that see it NaN, one that is -inf takes its key out, at every place of a tile's words."""
    m = Batch(kch, [140], [60], dtype=dtype, c=c, n_kv=1, page=16)
    q = m.randn(m.N, 2, c)
    q[..., 3] = 1.
    pg, row = at(m, 0, 96 + col)
    m.cache.k_pages[pg, 0, row, 3] = bad
    m.cache.v_pages[pg, 0, row, 5] = 1e36          # (large and finite: nothing of it where its weight is 0)
    want, tol = by_rows(m, q)
    assert want[:36 + col].isfinite().all()
    assert want[36 + col:].isfinite().all() if bad == float("-inf") else want[36 + col:].isnan().all()
    close(m.cache.forward_step(q, *m.args), want, tol)


@pytest.mark.parametrize("window", [0, 40])
@pytest.mark.parametrize("dtype,c", [(torch.bfloat16, 128), (torch.bfloat16, 64), (torch.float32, 64)])
def test_a_large_finite_value_that_is_hidden_adds_nothing(kch, dtype, c, window):
    m = Batch(kch, [150], [50], dtype=dtype, c=c, n_kv=1, page=16)
    q = m.randn(m.N, 2, c)
    want, tol = by_rows(m, q, window=window)
    for key in (118, 119, 126, 127):               # one after the other: what a row that sees them gets is not compared
        pg, row = at(m, 0, key)
        m.cache.v_pages[pg, 0, row] = 3e38
    got = m.cache.forward_step(q, *m.args, sliding_window=window)
    rows = torch.arange(50, 200, device=DEV)
    hidden = rows < 118
    if window:
        hidden |= rows - 127 >= window
    close(got[hidden], want[hidden], tol[hidden])


@pytest.mark.parametrize("dtype,c", [(torch.bfloat16, 128), (torch.bfloat16, 64), (torch.float32, 64)])
def test_rows_behind_a_table_that_ends_too_early_and_whose_window_ends_there_too_are_zero(kch, dtype, c):
    """They see no key, in tiles of which other rows see some."""
    from kch_b200 import _lib
    m = Batch(kch, [150], [20], dtype=dtype, c=c, n_kv=1, page=16)
    q = m.randn(m.N, 2, c)
    want, tol = by_rows(m, q, window=30)
    got = m.cache.forward_step(q, m.table[:, :5], m.t0, m.cu, sliding_window=30)        # 80 positions
    torch.cuda.synchronize()
    assert _lib.device_status(reset=True) == _lib.STATUS_PAGED_TABLE
    close(got[:60], want[:60], tol[:60])
    assert (got[109 - 20:] == 0).all()


# ---- batches ---------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype,kind,c", [(torch.bfloat16, None, 128), (torch.bfloat16, "fp8", 128), (torch.float32, "int8", 64)])
@pytest.mark.parametrize("first,last", [(-1, 30), (-2 ** 31, 30), (0, 2 ** 31 - 1), (-2 ** 31, 2 ** 31 - 1)])
def test_rows_in_front_of_the_packed_tensors_and_behind_them_count_as_their_ends(kch, dtype, kind, c, first, last):
    a, b = (Batch(kch, [13, 17], [40, 3], dtype=dtype, kind=kind, c=c, seed=3) for _ in range(2))
    k, v, q = a.randn(30, 2, c), a.randn(30, 2, c), a.randn(30, 4, c)
    cu = torch.tensor([first, 13, last], dtype=torch.int32, device=DEV)
    a.cache.append_step(k, v, *a.args)
    b.cache.append_step(k, v, b.table, b.t0, cu)
    for x in ("k_pages", "v_pages", "k_scales", "v_scales"):
        one, other = getattr(a.cache, x), getattr(b.cache, x)
        assert one is None or torch.equal(one.view(torch.uint8), other.view(torch.uint8))
    for one, other in zip(a.cache.read_step(*a.args, n_rows=30), b.cache.read_step(b.table, b.t0, cu, n_rows=30)):
        assert torch.equal(one, other)
    assert torch.equal(a.cache.forward_step(q, *a.args), b.cache.forward_step(q, b.table, b.t0, cu))


@pytest.mark.parametrize("B", [4, 40])
@pytest.mark.parametrize("dtype,kind,c", [(torch.bfloat16, None, 128), (torch.bfloat16, "fp8", 128), (torch.float32, None, 64)])
def test_sequences_without_new_tokens_need_no_page(kch, dtype, kind, c, B):
    """Idle places of a captured batch: lengths of long ago, far behind the table."""
    from kch_b200 import _lib
    m = Batch(kch, [1 + b % 3 if b % 2 else 0 for b in range(B)], [40 + b if b % 2 else 0 for b in range(B)], dtype=dtype, kind=kind, c=c, page=16)
    q, k = m.randn(m.N, 4, c), m.randn(m.N, 2, c)
    for far in (200, 10 ** 6, 2 ** 31 - 1):
        m.t0[::2] = far
        m.cache.append_step(k, k, *m.args)
        got = m.cache.forward_step(q, *m.args)
        torch.cuda.synchronize()
        assert _lib.device_status(reset=True) == 0
        want, tol = by_rows(m, q)
        close(got, want, tol)


@pytest.mark.parametrize("new,past", [([1, 3, 1], [1000, 700, 90]), ([1, 150], [3, 1000]), ([300], [777])])
@pytest.mark.parametrize("dtype,kind,c,page", [(torch.bfloat16, None, 128, 16), (torch.bfloat16, None, 64, 8), (torch.bfloat16, "fp8", 128, 16),
                                               (torch.bfloat16, "int8", 64, 32), (torch.float32, None, 64, 16), (torch.float32, "fp8", 128, 8),
                                               (torch.bfloat16, None, 128, 256)])
def test_pages_that_every_window_has_left_behind_may_be_gone(kch, dtype, kind, c, page, new, past):
    """The caller gives them to other sequences and takes them out of the table."""
    from kch_b200 import _lib
    m = Batch(kch, new, past, dtype=dtype, kind=kind, c=c, page=page)
    q, window = m.randn(m.N, 4, c), 100
    want, tol = by_rows(m, q, window=window)
    for b, p in enumerate(past):
        gone = max(p - window + 1, 0) // page
        for x in ("k_pages", "v_pages") if kind is None else ("k_scales", "v_scales"):
            getattr(m.cache, x)[m.table[b, :gone].long()] = torch.nan
        m.table[b, :gone] = -1
    got = m.cache.forward_step(q, *m.args, sliding_window=window)
    torch.cuda.synchronize()
    assert _lib.device_status(reset=True) == 0
    close(got, want, tol)


def test_a_table_at_fault_cuts_no_wait_short(kch):
    """The status it raises is the caller's to read; kernels that wait for their copies do not give up because of it."""
    from kch_b200 import _lib
    m = Batch(kch, [3], [70])
    m.table[0, 1] = -1
    m.cache.forward_step(m.randn(3, 4, 128), *m.args)
    torch.cuda.synchronize()
    assert _lib.device_status() == _lib.STATUS_PAGED_TABLE
    _lib.check(_lib.load().kch_selftest_bounded_wait(4096, None, _lib.stream()))       # a wait that nothing ends: to its own limit
    torch.cuda.synchronize()
    assert _lib.device_status(reset=True) == _lib.STATUS_SELFTEST_WAIT                 # (and it is reported first)
    assert _lib.device_status() == 0
    m.cache.forward_step(m.randn(3, 4, 128), *m.args)
    with pytest.raises(RuntimeError, match="block table"):
        _lib.raise_on_device_status("test")


@pytest.mark.parametrize("new", [[1, 2, 1], [200, 130, 5]])
@pytest.mark.parametrize("dtype,kind,c", [(torch.bfloat16, None, 128), (torch.bfloat16, "fp8", 128), (torch.bfloat16, "int8", 64), (torch.float32, None, 64)])
def test_a_table_at_fault_leaves_the_other_sequences_alone(kch, dtype, kind, c, new):
    from kch_b200 import _lib
    m = Batch(kch, new, [1500, 700, 3], dtype=dtype, kind=kind, c=c)
    q = m.randn(m.N, 4, c)
    m.table[1, 20] = 1 << 30
    want, tol = by_rows(m, q, missing=[(1, 20)])           # (what it does not name reads as zeros)
    for _ in range(3):
        got = m.cache.forward_step(q, *m.args)
        torch.cuda.synchronize()
        assert _lib.device_status() == _lib.STATUS_PAGED_TABLE
        close(got, want, tol)
    assert _lib.device_status(reset=True) == _lib.STATUS_PAGED_TABLE


@pytest.mark.parametrize("new", [[1, 2, 1], [8, 8, 8], [200, 130, 5]])
@pytest.mark.parametrize("kind,c", [("fp8", 128), ("int8", 64), ("fp8", 72)])
def test_pages_that_are_missing_have_scales_of_zero_not_those_of_another_page(kch, kind, c, new):
    from kch_b200 import _lib
    for page in (16, 128):
        m = Batch(kch, new, [1500, 700, 3], kind=kind, c=c, page=page)
        held = set(m.table[m.table >= 0].tolist())
        if 0 in held:                                      # page 0 is nobody's
            spare = next(i for i in range(m.cache.num_pages) if i not in held)
            m.table[m.table == 0] = spare
        for scales in (m.cache.k_scales, m.cache.v_scales):
            scales[0] = torch.nan
        q = m.randn(m.N, 4, c)
        m.table[1, 4] = -1
        want, tol = by_rows(m, q, missing=[(1, 4)])
        got = m.cache.forward_step(q, *m.args)
        torch.cuda.synchronize()
        assert _lib.device_status(reset=True) == _lib.STATUS_PAGED_TABLE
        close(got, want, tol)


@pytest.mark.parametrize("low", [0., 0.6])
@pytest.mark.parametrize("new,past", [([1], [400]), ([1], [30000]), ([4, 1], [700, 250]), ([40], [9000]), ([150, 90], [300, 1000])])
@pytest.mark.parametrize("dtype,kind,c", [(torch.bfloat16, None, 128), (torch.bfloat16, None, 64), (torch.bfloat16, "fp8", 128), (torch.bfloat16, "int8", 64),
                                          (torch.float32, None, 64), (torch.float32, "int8", 72)])
def test_a_value_that_is_not_a_number_reaches_the_rows_that_see_it_however_little_it_weighs(kch, dtype, kind, c, new, past, low):
    """NaN values of keys far below the others (less than 2^-1000 of the weight), among others or, with `low`, among their like: 0 times a NaN is
    one, whatever tile, warp or part of a row has it."""
    m = Batch(kch, new, past, dtype=dtype, kind=kind, c=c, n_kv=1, page=16)
    q = m.randn(m.N, 2, c)
    q[..., 0] = 1000.
    for b, (n, p) in enumerate(zip(new, past)):
        pos = torch.arange(p + n, device=DEV)
        bad = torch.tensor([1, p // 2, p - 1] if b == 0 and not low else [p // 3], device=DEV)
        down = (pos < low * p) | torch.isin(pos, bad)
        pages, rows = m.table[b].long()[pos // 16], pos % 16
        if kind is None:
            m.cache.k_pages[pages, 0, rows, 0] = torch.where(down, -60., 0.).to(dtype)
            m.cache.v_pages[pages[bad], 0, rows[bad], 5] = torch.nan
        else:
            m.cache.k_pages.view(torch.uint8)[pages, 0, rows, 0] = torch.where(down, 0x81 if kind == "int8" else 0xF6, 0).byte()
            m.cache.k_scales[pages[down], 0, rows[down]] = 0.3
            m.cache.v_scales[pages[bad], 0, rows[bad]] = torch.nan
    want, tol = by_rows(m, q)
    assert want[..., 5].isnan().any()
    close(m.cache.forward_step(q, *m.args), want, tol)


@pytest.mark.parametrize("new", [[2, 3, 1], [90, 140, 20]])
@pytest.mark.parametrize("dtype,kind,c", [(torch.bfloat16, None, 128), (torch.bfloat16, "fp8", 128), (torch.bfloat16, "int8", 64), (torch.float32, None, 64)])
@pytest.mark.parametrize("t0", [-1, -100, -2 ** 31])
def test_a_negative_count_of_earlier_tokens_is_the_callers_mistake_and_touches_nothing(kch, dtype, kind, c, new, t0):
    from kch_b200 import _lib
    m = Batch(kch, new, [70, 0, 33], dtype=dtype, kind=kind, c=c)
    k, q = m.randn(m.N, 2, c), m.randn(m.N, 4, c)
    before = m.cache.k_pages.clone().view(torch.uint8)
    m.t0[1] = t0
    mine = slice(new[0], new[0] + new[1])
    for call in (lambda: m.cache.append_step(k, k, *m.args), lambda: m.cache.read_step(*m.args, n_rows=m.N), lambda: m.cache.forward_step(q, *m.args)):
        got = call()
        torch.cuda.synchronize()
        assert _lib.device_status(reset=True) == _lib.STATUS_PAGED_TABLE
        if isinstance(got, tuple):
            assert not got[0][mine].any() and got[0][:new[0]].any()
    held = m.table[1][m.table[1] >= 0].long()
    assert torch.equal(m.cache.k_pages.view(torch.uint8)[held], before[held])
    assert (got[mine] == 0).all()
    want, tol = by_rows(m, q)
    rows = torch.cat([torch.arange(0, new[0]), torch.arange(new[0] + new[1], m.N)]).to(DEV)
    close(got[rows], want[rows], tol[rows])


@pytest.mark.parametrize("window", [0, 90])
@pytest.mark.parametrize("where", ["nowhere", "key", "value", "both"])
@pytest.mark.parametrize("new,past", [([1, 1], [300, 4000]), ([4, 2], [700, 31]), ([140, 3], [60, 500]), ([70], [2000])])
@pytest.mark.parametrize("dtype,c,nh,n_kv", [(torch.bfloat16, 128, 4, 2), (torch.bfloat16, 64, 16, 1), (torch.bfloat16, 128, 24, 1), (torch.float32, 64, 4, 2)])
def test_a_pool_that_holds_codes_of_nan(kch, dtype, c, nh, n_kv, new, past, where, window):
    """e4m3 has two codes of NaN.  Rows written here have none, but a pool that existed already may: what sees one is what read_step's values give,
    and what does not see it is as ever."""
    m = Batch(kch, new, past, dtype=dtype, kind="fp8", c=c, n_kv=n_kv, page=16)
    m.cache = kch.PagedKVCache(m.cache.num_pages, 16, n_kv, c, DEV, dtype, kv_quant="fp8",
                               storage=(m.cache.k_pages, m.cache.v_pages, m.cache.k_scales, m.cache.v_scales))
    owned = torch.zeros(m.cache.num_pages, 16, dtype=torch.bool, device=DEV)
    for b, (n, p) in enumerate(zip(new, past)):
        lo = max(p + 1 - window, 0) if window else 0
        pos = torch.arange(lo, n + p, device=DEV)
        owned[m.table[b].long()[pos // 16], pos % 16] = True
    raw = [x.view(torch.uint8) for x in (m.cache.k_pages, m.cache.v_pages)]
    for x in raw:                                          # behind the ends, before the windows and in pages of nobody: anything
        x.masked_fill_((~owned)[:, None, :, None].expand_as(x), 0x7F)
        x[:, :, ::3].masked_fill_((~owned)[:, None, ::3, None].expand_as(x[:, :, ::3]), 0xFF)
    pg, row = at(m, 0, past[0] - 3)
    if where in ("key", "both"):
        raw[0][pg, n_kv - 1, row, c - 1] = 0xFF
    if where in ("value", "both"):
        raw[1][pg, 0, row, 9], raw[1][pg, 0, row, c - 2] = 0x7F, 0xFF
        pg, row = at(m, 0, past[0] + new[0] - 1)           # the newest token's: its own query alone sees it
        raw[1][pg, n_kv - 1, row, 40] = 0x7F
    if where != "nowhere":
        first = torch.tensor([past[0] - 3], dtype=torch.int32, device=DEV)
        k, v = m.cache.read_step(m.table[:1], first, torch.tensor([0, new[0] + 3], dtype=torch.int32, device=DEV), n_rows=new[0] + 3)
        want_k, want_v = (m.values(x, 0, past[0] + new[0])[:, past[0] - 3:].transpose(0, 1).to(dtype) for x in "kv")
        for got, want in ((k, want_k), (v, want_v)):
            assert torch.equal(got.isnan(), want.isnan()) and torch.equal(got.nan_to_num(), want.nan_to_num())
    q = m.randn(m.N, nh, c)
    want, tol = by_rows(m, q, window=window)
    assert bool(want.isnan().any()) == (where != "nowhere")
    for _ in range(2):
        close(m.cache.forward_step(q, *m.args, sliding_window=window), want, tol)


@pytest.mark.parametrize("kind", [None, "fp8"])
def test_rows_that_are_summed_again_over_a_long_sequence_do_not_run_the_others_waits_out(kch, kind):
    """A NaN at the start of 131072 keys: every row of a chunk of 4096 tokens has one, and all of them are summed key by key."""
    from kch_b200 import _lib
    new, past = 4096, 131072 - 4096
    n = 131072 // 64
    cache = kch.PagedKVCache(n, 64, 4, 128, DEV, torch.bfloat16, kv_quant=kind)
    g = torch.Generator(device=DEV).manual_seed(9)
    for x in (cache.k_pages, cache.v_pages):
        x.normal_(generator=g) if kind is None else x.view(torch.uint8).random_(0, 0x60, generator=g)
    if kind is None:
        cache.v_pages[0, :, 3, 5] = torch.nan
    else:
        cache.v_pages.view(torch.uint8)[0, :, 3, 5] = 0x7F
    table = torch.arange(n, dtype=torch.int32, device=DEV)[None]
    t0, cu = torch.tensor([past], dtype=torch.int32, device=DEV), torch.tensor([0, new], dtype=torch.int32, device=DEV)
    q = torch.randn(new, 16, 128, generator=g, device=DEV).bfloat16()
    got = cache.forward_step(q, table, t0, cu)
    torch.cuda.synchronize()
    assert _lib.device_status(reset=True) == 0
    assert got[..., 5].isnan().all() and got.isnan().sum() == new * 16
    # the same without the NaN, the other channels: P (2^-8 of the weighed sizes of the values) and the output are rounded in either call
    pages = cache.v_pages.view(torch.uint8) if kind else cache.v_pages
    pages[0, :, 3, 5] = 0
    want = cache.forward_step(q, table, t0, cu).float()
    pages.copy_(pages & 0x7F if kind else pages.abs())
    size = cache.forward_step(q, table, t0, cu).float()
    rest = torch.arange(128, device=DEV) != 5
    assert ((got.float() - want).abs() <= 2.0 ** -7 * (1 + 2.0 ** -7) * (size + want.abs()) + 2.0 ** -14 * size)[..., rest].all()
