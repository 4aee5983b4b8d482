"""The paged cache against its definitions in 64 bits: rows written and read back, attention of ragged batches over the pages.

Tolerances.  A logit is a sum of c products in fp32, off by d = (c + 4) 2^-24 scale sum|q||k| at most (products of bf16 values
are exact, the sum is not); a probability is then off by 2 d of itself, numerator and denominator together, and by the error of
exp2 and of the running sums, (n + 64) 2^-24 for n keys.  bf16: probabilities are rounded before the product (2^-8) and the output
once (2^-8 of itself).  All of it weighs values of sum p |v|.
"""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
QUANT = {"fp8": (torch.float8_e4m3fn, 448.0), "int8": (torch.int8, 127.0)}


@pytest.fixture(scope="module")
def kch():
    import kch_b200
    from kch_b200 import _lib
    _lib.load()
    yield kch_b200
    assert _lib.device_status() == 0, "a device-side status was raised"


def codes(x, kind):
    """Stored values and scales by their definition, in 64 bits: the nearest value of the type, ties to the even code."""
    store, most = QUANT[kind]
    amax = x.double().abs().amax(-1)
    scale = torch.where(amax > 0, (amax / most).clamp_min(2.0 ** -126), 1.0).float()
    size = (x.double() / scale.double()[..., None]).abs()
    held = torch.arange(int(most) + 1 if kind == "int8" else 127, device=x.device).to(torch.uint8).view(store).double()
    above = torch.searchsorted(held, size).clamp_(1, len(held) - 1)
    low, high = size - held[above - 1], held[above] - size
    up = (high < low) | ((high == low) & (above % 2 == 0))
    return torch.where(up, held[above], held[above - 1]).copysign(x.double()), scale


class Batch:
    """A cache with pages scattered over its pool, and a ragged batch of it."""

    def __init__(self, kch, new, past, *, dtype=torch.bfloat16, kind=None, n_kv=2, c=128, page=16, seed=0, spare=3, first_row=0, rows_behind=0,
                 wider=0):
        g = torch.Generator(device=DEV).manual_seed(seed)
        self.new, self.past, self.page, self.n_kv, self.c, self.dtype, self.kind = new, past, page, n_kv, c, dtype, kind
        held = [-(-(n + p) // page) for n, p in zip(new, past)]
        pool = sum(held) + spare
        self.cache = kch.PagedKVCache(pool, page, n_kv, c, DEV, dtype, kv_quant=kind)
        ids = torch.randperm(pool, generator=g, device=DEV)[:sum(held)].to(torch.int32)
        table = torch.full((len(new), max(max(held), 1) + wider), -1, dtype=torch.int32, device=DEV)
        at = 0
        for b, h in enumerate(held):
            table[b, :h] = ids[at:at + h]
            at += h
        self.table = table
        self.t0 = torch.tensor(past, dtype=torch.int32, device=DEV)
        self.cu = torch.tensor([first_row + sum(new[:i]) for i in range(len(new) + 1)], dtype=torch.int32, device=DEV)
        self.N = first_row + sum(new) + rows_behind
        self.first = first_row
        # everything the pool holds, of this batch or not
        for x in ("k", "v"):
            rows = torch.randn(pool, n_kv, page, c, generator=g, device=DEV).to(dtype)
            if kind is None:
                getattr(self.cache, x + "_pages").copy_(rows)
            else:
                payload, scale = codes(rows, kind)
                getattr(self.cache, x + "_pages").copy_(payload.to(QUANT[kind][0]))
                getattr(self.cache, x + "_scales").copy_(scale)
        self.g = g

    @property
    def args(self):
        return self.table, self.t0, self.cu

    def randn(self, *shape):
        return torch.randn(*shape, generator=self.g, device=DEV).to(self.dtype)

    def values(self, x, b, n):
        """The first n rows of sequence b in 64 bits, [n_kv, n, c]."""
        ids = self.table[b, :-(-n // self.page)].long()
        got = getattr(self.cache, x + "_pages")[ids].double()
        if self.kind:
            got = got * getattr(self.cache, x + "_scales")[ids].double()[..., None]
        return got.transpose(0, 1).flatten(1, 2)[:, :n]


def reference(m, q, *, scale=None, window=0, sink=None):
    """(outputs, tolerances) of the batch's rows in 64 bits; a key that a query does not see does not reach it."""
    scale = m.c ** -0.5 if scale is None else scale
    G = q.shape[1] // m.n_kv
    out = torch.zeros(q.shape, dtype=torch.double, device=DEV)
    tol = torch.zeros_like(out)
    for b, (n, p) in enumerate(zip(m.new, m.past)):
        if n == 0:
            continue
        r = slice(m.first + sum(m.new[:b]), m.first + sum(m.new[:b + 1]))
        k, v = m.values("k", b, p + n), m.values("v", b, p + n)
        far = torch.arange(p, p + n, device=DEV)[:, None] - torch.arange(p + n, device=DEV)
        sees = (far >= 0) & ((far < window) if window else True)
        for h in range(q.shape[1]):
            qq, kk, vv = q[r, h].double(), k[h // G], v[h // G]
            l = (scale * (qq @ kk.nan_to_num().T)).masked_fill(~sees, -torch.inf)
            size = (abs(scale) * (qq.abs() @ kk.nan_to_num().abs().T)).masked_fill(~sees, 0.).amax(1, keepdim=True)
            z = torch.logsumexp(l, 1, keepdim=True)
            if sink is not None:
                z = torch.logaddexp(z, sink[h].double().expand_as(z))
            w = (l - z).exp()
            w = w.masked_fill(~sees, 0.)
            finite = vv.isfinite().all(1)
            out[r, h] = w[:, finite] @ vv[finite]
            for j in (~finite).nonzero()[:, 0].tolist():              # only the rows that see it
                i = sees[:, j].nonzero()[:, 0]
                out[r.start + i, h] += w[i, j, None] * vv[j]
            d = (m.c + 4) * 2.0 ** -24 * size
            rel = 2 * d + (p + n + 64) * 2.0 ** -24
            weight = w[:, finite] @ vv[finite].abs()
            if m.dtype == torch.bfloat16:
                tol[r, h] = (rel + 2.0 ** -8) * weight + 2.0 ** -8 * out[r, h].nan_to_num().abs()
            else:
                tol[r, h] = rel * weight
    return out, tol


def close(got, want, tol):
    fine = want.isfinite()
    assert torch.equal(got.isnan(), want.isnan())
    assert torch.equal(got.double()[~fine & ~want.isnan()], want[~fine & ~want.isnan()])
    off = (got.double() - want).abs()[fine]
    assert (off <= tol[fine] + 1e-30).all(), f"{float((off - tol[fine]).max()):.3e} beyond, {float((off / (tol[fine] + 1e-30)).max()):.2f} of the tolerance"


# ---- rows ------------------------------------------------------------------------------------------------------------------
ROWS = [([1], [0]), ([1, 1, 1], [0, 15, 16]), ([0, 5, 0, 33, 17], [3, 0, 9, 31, 100]), ([300, 1, 64], [7, 8, 64])]


@pytest.mark.parametrize("new,past", ROWS)
@pytest.mark.parametrize("kind", [None, "fp8", "int8"])
@pytest.mark.parametrize("dtype,c,page,n_kv", [(torch.bfloat16, 128, 16, 2), (torch.float32, 64, 32, 1), (torch.bfloat16, 72, 8, 3),
                                               (torch.float32, 256, 64, 2), (torch.bfloat16, 8, 128, 5)])
def test_rows_are_written_where_they_belong_and_read_back(kch, new, past, kind, dtype, c, page, n_kv):
    m = Batch(kch, new, past, dtype=dtype, kind=kind, c=c, page=page, n_kv=n_kv, first_row=2, rows_behind=3)
    before = [t.clone() for t in (m.cache.k_pages, m.cache.v_pages)]
    scales = [t.clone() for t in (m.cache.k_scales, m.cache.v_scales)] if kind else [None, None]
    # heads dense within a token, tokens apart: slices of a fused projection
    both = m.randn(m.N, 2 * n_kv * c + 8)
    k, v = (both[:, i * n_kv * c:(i + 1) * n_kv * c].unflatten(1, (n_kv, c)) for i in range(2))
    if n_kv == 2:
        k[m.first] = 0.          # a row of zeros
    m.cache.append_step(k, v, *m.args)
    got = m.cache.read_step(*m.args, n_rows=m.N)
    mine = [torch.full_like(g, 7.) for g in got]
    back = m.cache.read_step(*m.args, n_rows=m.N, out=mine)
    assert back[0] is mine[0]
    live = slice(m.first, m.first + sum(new))
    for x, pages, was, scale_was, rows, out, kept in zip("kv", (m.cache.k_pages, m.cache.v_pages), before, scales, (k, v), got, mine):
        want_pages = was.double()
        want_scales = scale_was
        payload, s = (rows.double(), None) if kind is None else codes(rows, kind)
        if kind:
            want_scales = scale_was.clone()
        for b, (n, p) in enumerate(zip(new, past)):
            for i in range(n):
                row, pg, at = m.first + sum(new[:b]) + i, int(m.table[b, (p + i) // page]), (p + i) % page
                want_pages[pg, :, at] = payload[row]
                if kind:
                    want_scales[pg, :, at] = s[row]
        assert torch.equal(pages.double(), want_pages)
        if kind:
            assert torch.equal(getattr(m.cache, x + "_scales"), want_scales)
        value = payload if kind is None else payload.float() * s[..., None]
        assert torch.equal(out[live], value.to(dtype)[live])
        assert not out[:m.first].any() and not out[m.first + sum(new):].any()
        assert torch.equal(kept[live], out[live])
        assert (kept[:m.first] == 7).all() and (kept[m.first + sum(new):] == 7).all()


@pytest.mark.parametrize("kind", ["fp8", "int8"])
def test_values_in_the_middle_between_two_codes(kch, kind):
    """Quotients that lie on, or within one rounding of, the middle between two codes: the nearest code, ties to the even one."""
    m = Batch(kch, [4096], [0], dtype=torch.float32, kind=kind, c=64, page=64, n_kv=1)
    g = torch.Generator(device=DEV).manual_seed(5)
    most = QUANT[kind][1]
    held = torch.arange(int(most) + 1 if kind == "int8" else 127, device=DEV).to(torch.uint8).view(QUANT[kind][0]).float()
    middle = (held[1:] + held[:-1]) / 2
    amax = torch.exp(torch.randn(4096, 1, 1, generator=g, device=DEV))
    amax = torch.where(torch.rand(4096, 1, 1, generator=g, device=DEV) < 0.5, amax.bfloat16().float(), amax)
    pick = middle[torch.randint(len(middle), (4096, 1, 64), generator=g, device=DEV)]
    x = pick * (amax / most)
    x = torch.where(torch.rand(x.shape, generator=g, device=DEV) < 0.3, x.bfloat16().float(), x)
    x = torch.nextafter(x, torch.where(torch.rand(x.shape, generator=g, device=DEV) < 0.5, 0., 1e30)) if kind == "int8" else x
    x[:, :, :1] = -amax
    m.cache.append_step(x, x, *m.args)
    payload, scale = codes(x, kind)
    at = m.table[0].long()
    assert torch.equal(m.cache.k_scales[at].flatten(), scale.flatten())
    assert torch.equal(m.cache.k_pages[at].double().flatten(), payload.flatten())


def test_rows_that_are_not_finite_read_as_nan_and_the_smallest_ones_as_zero_or_themselves(kch):
    for kind in ("fp8", "int8"):
        m = Batch(kch, [4], [3], dtype=torch.float32, kind=kind, c=64, n_kv=1)
        x = m.randn(4, 1, 64)
        x[0, 0, 5], x[1, 0, 6] = torch.inf, torch.nan
        x[2] = 1e-44
        m.cache.append_step(x, x, *m.args)
        k, v = m.cache.read_step(*m.args, n_rows=4)
        assert k[:2].isnan().all() and v[:2].isnan().all()
        assert k[2].isfinite().all() and (k[2] - x[2]).abs().max() <= 2.0 ** -126
        assert k[3].isfinite().all()


# ---- attention --------------------------------------------------------------------------------------------------------------
GEOMETRY = [(torch.bfloat16, 128, 16, 4, 16), (torch.bfloat16, 64, 4, 4, 32), (torch.float32, 64, 4, 2, 16), (torch.float32, 128, 8, 1, 8),
            (torch.bfloat16, 128, 12, 4, 64), (torch.bfloat16, 64, 14, 2, 128), (torch.bfloat16, 128, 16, 1, 256), (torch.bfloat16, 72, 6, 3, 16),
            (torch.float32, 200, 2, 2, 16), (torch.bfloat16, 256, 4, 1, 16), (torch.bfloat16, 8, 2, 1, 8)]
LENGTHS = [([1], [0]), ([1], [130]), ([1, 1, 1, 1], [0, 15, 400, 1025]), ([3, 0, 1, 200], [64, 9, 0, 77]), ([130, 17], [0, 1000])]


@pytest.mark.parametrize("new,past", LENGTHS)
@pytest.mark.parametrize("kind", [None, "fp8", "int8"])
@pytest.mark.parametrize("dtype,c,nh,n_kv,page", GEOMETRY)
def test_attention_over_the_pages(kch, new, past, kind, dtype, c, nh, n_kv, page):
    m = Batch(kch, new, past, dtype=dtype, kind=kind, c=c, n_kv=n_kv, page=page)
    q = m.randn(m.N, nh, c)
    want, tol = reference(m, q)
    got = m.cache.forward_step(q, *m.args)
    assert got.dtype == dtype
    close(got, want, tol)
    # a window, a sink, another scale; rows that belong to no sequence
    sink = torch.randn(nh, generator=m.g, device=DEV)
    want, tol = reference(m, q, scale=-0.3, window=37, sink=sink)
    close(m.cache.forward_step(q, *m.args, scale=-0.3, sliding_window=37, sink_logits=sink), want, tol)


@pytest.mark.parametrize("dtype,kind,c", [(torch.bfloat16, None, 128), (torch.bfloat16, "fp8", 128), (torch.bfloat16, "int8", 64), (torch.float32, None, 64)])
def test_rows_of_no_sequence(kch, dtype, kind, c):
    m = Batch(kch, [0, 5, 0, 130, 0], [4, 60, 0, 3, 9], dtype=dtype, kind=kind, c=c, first_row=3, rows_behind=70)
    q = m.randn(m.N, 4, c)
    want, tol = reference(m, q)
    got = m.cache.forward_step(q, *m.args)
    close(got, want, tol)                                   # (zeros outside)
    out = torch.full_like(q, 5.)
    assert m.cache.forward_step(q, *m.args, out=out) is out
    live = slice(3, 3 + 135)
    assert torch.equal(out[live], got[live]) and (out[:3] == 5).all() and (out[138:] == 5).all()
    # nothing at all
    empty = torch.zeros_like(m.cu)
    assert not m.cache.forward_step(q, m.table, m.t0, empty).any()
    assert m.cache.forward_step(q[:0], m.table, m.t0, empty).shape == (0, 4, c)
    m.cache.append_step(q[:0, :2], q[:0, :2], m.table, m.t0, empty)


@pytest.mark.parametrize("window", [0, 50])
@pytest.mark.parametrize("dtype,kind,c", [(torch.bfloat16, None, 128), (torch.bfloat16, None, 64), (torch.float32, None, 64), (torch.bfloat16, "fp8", 128),
                                          (torch.bfloat16, "int8", 64), (torch.bfloat16, None, 72)])
def test_what_a_query_does_not_see_does_not_reach_it(kch, dtype, kind, c, window):
    """Infinities and NaN in other pages, behind a sequence's end, ahead of a query and behind its window."""
    new, past = [3, 150, 1], [200, 64, 300]
    m = Batch(kch, new, past, dtype=dtype, kind=kind, c=c, page=16)
    owned = torch.zeros(m.cache.num_pages, 16, dtype=torch.bool, device=DEV)
    for b, (n, p) in enumerate(zip(new, past)):
        pos = torch.arange(n + p, device=DEV)
        owned[m.table[b].long()[pos // 16], pos % 16] = True
    for pages, scales in ((m.cache.k_pages, m.cache.k_scales), (m.cache.v_pages, m.cache.v_scales)):
        bad = (~owned)[:, None, :, None].expand_as(pages)
        if kind is None:
            pages.masked_fill_(bad, torch.nan)
            pages[:, :, 1::2].masked_fill_(bad[:, :, 1::2], torch.inf)
        else:
            scales.masked_fill_((~owned)[:, None].expand_as(scales), torch.nan)
    # the value row of the chunk's token 40 is infinite: the queries before it do not see it, nor those 50 behind it
    pg, at = int(m.table[1, (64 + 40) // 16]), (64 + 40) % 16
    if kind is None:
        m.cache.v_pages[pg, 0, at, 3] = torch.inf
    else:
        m.cache.v_scales[pg, 0, at] = torch.nan
    q = m.randn(m.N, 4, c)
    want, tol = reference(m, q, window=window)
    assert want[3:3 + 40].isfinite().all() and not want[3 + 40, 0].isfinite().all()
    close(m.cache.forward_step(q, *m.args, sliding_window=window), want, tol)


def test_large_and_infinite_sinks_and_large_logits(kch):
    for dtype in (torch.bfloat16, torch.float32):
        m = Batch(kch, [5, 1], [100, 700], dtype=dtype, c=64, n_kv=2)
        q = m.randn(6, 4, 64) * 30
        sink = torch.tensor([-torch.inf, 50., 1000., torch.inf], device=DEV)
        want, tol = reference(m, q, sink=sink)
        got = m.cache.forward_step(q, *m.args, sink_logits=sink)
        close(got[:, :3], want[:, :3], tol[:, :3])
        assert not got[:, 3].any()                          # an infinite sink leaves nothing
        half = sink[:3].tolist()[:2] + [0.5, -2.]
        half = torch.tensor(half, device=DEV).bfloat16()
        want, tol = reference(m, q, sink=half)
        close(m.cache.forward_step(q, *m.args, sink_logits=half), want, tol)


@pytest.mark.parametrize("kind", [None, "fp8"])
def test_a_session_appended_and_attended_step_by_step_is_the_whole_attention(kch, kind):
    """Prompts in chunks, then tokens one by one, sequences that join and leave: as one causal attention over what was stored."""
    m = Batch(kch, [57, 90, 23], [0, 0, 0], kind=kind, c=128, n_kv=2, page=16)
    nh, total = 8, m.new
    data = {x: [m.randn(n, 2 if x != "q" else nh, 128) for n in total] for x in "qkv"}
    outs = [[] for _ in total]
    seen = [0, 0, 0]
    for take in ([20, 0, 23], [30, 64, 0], [1, 1, 0], [1, 17, 0], [1, 1, 0], [4, 7, 0]):
        who = [b for b in range(3) if take[b]]
        cu = torch.tensor([0] + [sum(take[b] for b in who[:i + 1]) for i in range(len(who))], dtype=torch.int32, device=DEV)
        t0 = torch.tensor([seen[b] for b in who], dtype=torch.int32, device=DEV)
        part = {x: torch.cat([data[x][b][seen[b]:seen[b] + take[b]] for b in who]) for x in "qkv"}
        m.cache.append_step(part["k"], part["v"], m.table[who], t0, cu)
        o = m.cache.forward_step(part["q"], m.table[who], t0, cu)
        for i, b in enumerate(who):
            outs[b].append(o[int(cu[i]):int(cu[i + 1])])
            seen[b] += take[b]
    assert seen == total
    for b, x in enumerate("kv"):
        k = m.cache.read_step(*m.args, n_rows=m.N)[b]
        rows = torch.cat(data[x])
        assert torch.equal(k, rows if kind is None else (lambda p, s: (p.float() * s[..., None]).bfloat16())(*codes(rows, kind)))
    q = torch.cat(data["q"])
    want, tol = reference(m, q)
    close(torch.cat([torch.cat(o) for o in outs]), want, tol)


@pytest.mark.parametrize("dtype,kind,c", [(torch.bfloat16, None, 128), (torch.bfloat16, "int8", 64), (torch.float32, None, 64)])
def test_a_captured_step_replays_with_other_lengths(kch, dtype, kind, c):
    m = Batch(kch, [1, 1, 1], [500, 40, 300], dtype=dtype, kind=kind, c=c, n_kv=2, wider=5)
    q, k, v = m.randn(3, 8, c), m.randn(3, 2, c), m.randn(3, 2, c)
    t0 = m.t0.clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):                           # (the first calls of a process resolve addresses)
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
        assert torch.equal(out, m.cache.forward_step(q, m.table, t0, m.cu))      # the same bits as an eager call


def test_calls_on_two_streams_at_once_and_again(kch):
    a, b = (Batch(kch, [1] * 20, [97 * i for i in range(20)], kind=k, n_kv=2, seed=s) for k, s in ((None, 1), ("fp8", 2)))
    qa, qb = a.randn(20, 16, 128), b.randn(20, 16, 128)
    want = [a.cache.forward_step(qa, *a.args), b.cache.forward_step(qb, *b.args)]
    torch.cuda.synchronize()
    s = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = [[], []]
    for _ in range(10):
        for i, (m, q) in enumerate(((a, qa), (b, qb))):
            with torch.cuda.stream(s[i]):
                got[i].append(m.cache.forward_step(q, *m.args))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(g, want[i]) for g in got[i])


def test_strided_operands_and_tables(kch):
    m = Batch(kch, [5, 40], [33, 100], n_kv=2)
    q = m.randn(m.N, 4, 128)
    want = m.cache.forward_step(q, *m.args)
    wide = torch.randn(m.N, 4 * 128 + 24, device=DEV).bfloat16()
    wide[:, 8:8 + 512] = q.flatten(1)
    assert torch.equal(m.cache.forward_step(wide[:, 8:8 + 512].unflatten(1, (4, 128)), *m.args), want)
    assert torch.equal(m.cache.forward_step(q.transpose(0, 1).contiguous().transpose(0, 1), *m.args), want)
    odd = torch.empty(m.N * 512 + 1, device=DEV).bfloat16()[1:].view(m.N, 4, 128).copy_(q)      # not on 16 bytes
    assert torch.equal(m.cache.forward_step(odd, *m.args), want)
    big = torch.full((2, 64), -1, dtype=torch.int32, device=DEV)
    big[:, 3:3 + m.table.shape[1]] = m.table
    assert torch.equal(m.cache.forward_step(q, big[:, 3:3 + m.table.shape[1]], m.t0, m.cu), want)
    assert torch.equal(m.cache.forward_step(q, m.table.t().contiguous().t(), m.t0, m.cu), want)
    pairs = torch.stack([m.t0, m.t0], 1)
    assert torch.equal(m.cache.forward_step(q, m.table, pairs[:, 0], m.cu), want)


@pytest.mark.parametrize("new,past", [([1, 1], [33, 700]), ([40, 300], [100, 900])])
@pytest.mark.parametrize("dtype,kind,c", [(torch.bfloat16, None, 128), (torch.bfloat16, "fp8", 64), (torch.bfloat16, "int8", 128), (torch.float32, None, 64)])
def test_an_output_that_begins_on_16_bytes_and_no_more(kch, dtype, kind, c, new, past):
    m = Batch(kch, new, past, dtype=dtype, kind=kind, c=c)
    q = m.randn(m.N, 6, c)
    want = m.cache.forward_step(q, *m.args)
    ahead = 16 // want.element_size()
    room = torch.full((ahead + want.numel() + ahead,), 7.0, dtype=dtype, device=DEV)
    out = room[ahead:ahead + want.numel()].view(want.shape)
    assert out.data_ptr() % 32 == 16
    m.cache.forward_step(q, *m.args, out=out)
    assert torch.equal(out, want) and torch.equal(room[:ahead], room[-ahead:]) and (room[:ahead] == 7).all()


def test_offsets_that_pass_32_bits(kch):
    """A pool whose rows lie beyond 2^32 elements."""
    pages, page, c = 2 ** 32 // (64 * 128) + 40, 64, 128
    for kind in ("fp8", "int8"):
        cache = kch.PagedKVCache(pages, page, 1, c, DEV, torch.bfloat16, kv_quant=kind)
        table = torch.arange(pages - 1, pages - 6, -1, dtype=torch.int32, device=DEV)[None]
        t0, cu = torch.zeros(1, dtype=torch.int32, device=DEV), torch.tensor([0, 300], dtype=torch.int32, device=DEV)
        x = torch.randn(300, 1, c, device=DEV).bfloat16()
        cache.append_step(x, x, table, t0, cu)
        payload, scale = codes(x, kind)
        k, v = cache.read_step(table, t0, cu, n_rows=300)
        want = (payload.float() * scale[..., None]).bfloat16()
        assert torch.equal(k, want) and torch.equal(v, want)
        q = torch.randn(300, 2, c, device=DEV).bfloat16()
        o = cache.forward_step(q, table, t0, cu)
        value = payload[:, 0] * scale.double()
        p = (q[:, 1].double() @ value.T * c ** -0.5).masked_fill(torch.ones(300, 300, device=DEV).triu(1).bool(), -torch.inf).softmax(1)
        assert ((o[:, 1].double() - p @ value).abs() <= 2.0 ** -7 * (p @ value.abs()) + 2.0 ** -8).all()
        del cache


def test_tables_that_name_no_page_raise_the_status_and_touch_nothing(kch):
    from kch_b200 import _lib
    assert _lib.device_status() == 0
    for dtype, c in ((torch.bfloat16, 128), (torch.float32, 64)):
        for bad in (-1, 1 << 20, -2 ** 31, 2 ** 31 - 1):
            m = Batch(kch, [20, 3], [0, 70], dtype=dtype, c=c)
            m.table[1, 4] = bad
            before = m.cache.k_pages.clone()
            k = m.randn(23, 2, c)
            m.cache.append_step(k, k, *m.args)
            torch.cuda.synchronize()
            assert _lib.device_status(reset=True) == _lib.STATUS_PAGED_TABLE
            changed = (m.cache.k_pages != before).flatten(1).any(1).nonzero()[:, 0]
            assert set(changed.tolist()) <= set(m.table[0].tolist())
            assert not m.cache.read_step(*m.args, n_rows=23)[0][20:].any()
            assert _lib.device_status(reset=True) == _lib.STATUS_PAGED_TABLE
            m.cache.forward_step(m.randn(23, 4, c), *m.args)
            torch.cuda.synchronize()
            assert _lib.device_status(reset=True) == _lib.STATUS_PAGED_TABLE
        # a table that ends before its sequence does
        m = Batch(kch, [20, 3], [0, 70], dtype=dtype, c=c)
        k = m.randn(23, 2, c)
        for call in (lambda t: m.cache.append_step(k, k, t, m.t0, m.cu), lambda t: m.cache.forward_step(m.randn(23, 4, c), t, m.t0, m.cu)):
            call(m.table[:, :3])
            torch.cuda.synchronize()
            assert _lib.device_status(reset=True) == _lib.STATUS_PAGED_TABLE


@pytest.mark.parametrize("dtype,kind,B,N,n_kv", [(torch.bfloat16, None, 4096, 4096, 16), (torch.bfloat16, "fp8", 4096, 4096, 16),
                                                 (torch.float32, None, 4096, 4096, 16), (torch.bfloat16, None, 4096, 16400, 16),
                                                 (torch.bfloat16, None, 32, 65536, 128)])
def test_lengths_that_fall_and_rise_again_beyond_what_is_counted_do_nothing(kch, dtype, kind, B, N, n_kv):
    """Every other sequence has all rows: more steps in all than 32 bits hold, which the host, who sees N alone, cannot know."""
    from kch_b200 import _lib
    assert _lib.device_status() == 0
    cache = kch.PagedKVCache(1, 256, n_kv, 64, DEV, dtype, kv_quant=kind)
    table = torch.zeros(B, 4096, dtype=torch.int32, device=DEV)
    t0 = torch.full((B,), 4096 * 256 - N, dtype=torch.int32, device=DEV)
    cu = (torch.arange(B + 1, device=DEV) % 2 * N).int()
    q, out = torch.zeros(N, n_kv, 64, dtype=dtype, device=DEV), torch.full((N, n_kv, 64), 7.0, dtype=dtype, device=DEV)
    cache.forward_step(q, table, t0, cu, out=out)
    torch.cuda.synchronize()
    assert _lib.device_status(reset=True) == _lib.STATUS_PAGED_TABLE
    assert (out == 7).all()


def test_what_python_refuses(kch):
    m = Batch(kch, [2, 3], [5, 6])
    q, k = m.randn(5, 4, 128), m.randn(5, 2, 128)
    t, t0, cu = m.args
    for call, error, what in (
            (lambda: m.cache.forward_step(q[:, :3], t, t0, cu), ValueError, "multiple of n_kv"),
            (lambda: m.cache.forward_step(q.float(), t, t0, cu), ValueError, "dtype"),
            (lambda: m.cache.forward_step(q.cpu(), t, t0, cu), RuntimeError, "CUDA"),
            (lambda: m.cache.forward_step(q[..., :64], t, t0, cu), ValueError, "q must be"),
            (lambda: m.cache.forward_step(q, t.long(), t0, cu), TypeError, "table must be int32"),
            (lambda: m.cache.forward_step(q, t, t0[:1], cu), ValueError, "entries"),
            (lambda: m.cache.forward_step(q, t, t0, cu.cpu()), ValueError, "cu_seqlens is on cpu"),
            (lambda: m.cache.forward_step(q, t[0], t0, cu), ValueError, "rank 2"),
            (lambda: m.cache.forward_step(q, t[:, :0], t0, cu), ValueError, "no columns"),
            (lambda: m.cache.forward_step(q, t, t0, cu, sliding_window=-1), ValueError, "sliding_window"),
            (lambda: m.cache.forward_step(q, t, t0, cu, sink_logits=torch.zeros(3, device=DEV)), ValueError, "sink_logits"),
            (lambda: m.cache.forward_step(q, t, t0, cu, out=q[:4]), ValueError, "out must be"),
            (lambda: m.cache.append_step(q, k, t, t0, cu), ValueError, "k_new must be"),
            (lambda: m.cache.append_step(k, k[:4], t, t0, cu), ValueError, "v_new has 4"),
            (lambda: m.cache.read_step(t, t0, cu, n_rows=-1), ValueError, "n_rows"),
            (lambda: m.cache.read_step(t, t0, cu, n_rows=5, out=(k[:4], k[:4])), ValueError, "out"),
            (lambda: kch.PagedKVCache(m.cache.num_pages, 16, 2, 128, DEV, torch.bfloat16, storage=(m.cache.k_pages[1:], m.cache.v_pages, None, None)),
             ValueError, "k_pages")):
        with pytest.raises(error, match=what):
            call()


def test_large_batches_and_long_sequences(kch):
    """More sequences than a block has threads, lengths over three orders; one sequence split over every CTA."""
    new, past = [1 + (i % 7 == 0) * 40 for i in range(700)], [(i * 37) % 500 for i in range(700)]
    m = Batch(kch, new, past, n_kv=1, c=64, page=32)
    q = m.randn(m.N, 4, 64)
    want, tol = reference(m, q)
    close(m.cache.forward_step(q, *m.args), want, tol)
    for kind in (None, "fp8"):
        m = Batch(kch, [2], [70001], n_kv=2, kind=kind, page=64)
        q = m.randn(2, 8, 128)
        want, tol = reference(m, q)
        close(m.cache.forward_step(q, *m.args), want, tol)
        want, tol = reference(m, q, window=5000)
        close(m.cache.forward_step(q, *m.args, sliding_window=5000), want, tol)


@pytest.mark.parametrize("kind", [None, "fp8", "int8"])
@pytest.mark.parametrize("c,nh,n_kv", [(128, 8, 2), (64, 4, 1), (128, 16, 1), (64, 2, 2), (128, 14, 2)])
def test_batches_of_few_rows_with_one_long_chunk_among_them(kch, kind, c, nh, n_kv):
    """What a batch is on average decides on the form of the attention; every form takes every batch."""
    new, past = [1] * 20 + [60] + [2] * 19, [31 * i % 700 for i in range(40)]
    m = Batch(kch, new, past, kind=kind, c=c, n_kv=n_kv, page=16)
    q = m.randn(m.N, nh, c)
    want, tol = reference(m, q, window=300)
    close(m.cache.forward_step(q, *m.args, sliding_window=300), want, tol)
    # rows that do not depend on their company: the same bits in a batch of their own kind
    one = m.cache.forward_step(q[:20], m.table[:20], m.t0[:20], m.cu[:21])
    want, tol = reference(m, q)
    close(one, want[:20], tol[:20])


@pytest.mark.parametrize("page", [8, 16, 256])
def test_values_of_earlier_tokens_behind_a_sequence_are_cleared_not_summed_around(kch, page):
    """NaN in the last page of every sequence, in the rows behind its end."""
    m = Batch(kch, [1, 40, 1, 300], [6, 129, 1000, 500], page=page, n_kv=2, c=128)
    for b, (n, p) in enumerate(zip(m.new, m.past)):
        left = (n + p) % page
        if left:
            m.cache.v_pages[int(m.table[b, (n + p) // page]), :, left:] = torch.nan
    q = m.randn(m.N, 8, 128)
    want, tol = reference(m, q)
    close(m.cache.forward_step(q, *m.args), want, tol)
    # single tokens of the same sequences
    last = torch.tensor([n + p - 1 for n, p in zip(m.new, m.past)], dtype=torch.int32, device=DEV)
    ends = torch.tensor([sum(m.new[:i + 1]) - 1 for i in range(4)], device=DEV)
    got = m.cache.forward_step(q[ends], m.table, last, torch.arange(5, dtype=torch.int32, device=DEV))
    close(got, want[ends], tol[ends])


@pytest.mark.parametrize("kind", [None, "fp8", "int8"])
@pytest.mark.parametrize("nh,n_kv", [(2, 2), (8, 1), (14, 1), (16, 2), (32, 1), (48, 2), (9, 3)])
@pytest.mark.parametrize("c", [64, 128])
def test_steps_of_one_to_four_tokens(kch, kind, nh, n_kv, c):
    """From one row of a key head to a hundred: each form of the attention over few rows, and the one behind them."""
    for new, past in (([1, 1, 1], [400, 0, 129]), ([4, 3, 1, 4], [1000, 5, 64, 333]), ([4], [2000])):
        m = Batch(kch, new, past, kind=kind, c=c, n_kv=n_kv, page=32)
        q = m.randn(m.N, nh, c)
        sink = torch.randn(nh, generator=m.g, device=DEV)
        want, tol = reference(m, q, sink=sink, window=700)
        close(m.cache.forward_step(q, *m.args, sink_logits=sink, sliding_window=700), want, tol)
