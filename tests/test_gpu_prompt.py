"""Attention of whole prompts against its definition in 64 bits.  Oracle and tolerances are those of the paged attention's tests
(test_gpu_paged.py): the same sums, over keys and values that are packed rows."""
import pytest
import torch

from test_gpu_paged import DEV, close, reference

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def kch():
    import kch_b200
    from kch_b200 import _lib
    _lib.load()
    yield kch_b200
    assert _lib.device_status() == 0, "a device-side status was raised"


class Prompts:
    """Packed prompts, column slices of a fused projection."""

    def __init__(self, new, *, dtype=torch.bfloat16, nh=4, n_kv=2, c=128, seed=0, first_row=0, rows_behind=0, pad=8):
        self.g = torch.Generator(device=DEV).manual_seed(seed)
        self.new, self.past, self.dtype, self.n_kv, self.c, self.first = new, [0] * len(new), dtype, n_kv, c, first_row
        self.N = first_row + sum(new) + rows_behind
        self.cu = torch.tensor([first_row + sum(new[:i]) for i in range(len(new) + 1)], dtype=torch.int32, device=DEV)
        self.both = torch.randn(self.N, (nh + 2 * n_kv) * c + pad, generator=self.g, device=DEV).to(dtype)
        cuts = [pad, pad + nh * c, pad + (nh + n_kv) * c, pad + (nh + 2 * n_kv) * c]
        self.q, self.k, self.v = (self.both[:, a:b].unflatten(1, (-1, c)) for a, b in zip(cuts, cuts[1:]))

    def values(self, x, b, n):
        r = self.first + sum(self.new[:b])
        return getattr(self, x)[r:r + n].double().transpose(0, 1)

    @property
    def args(self):
        return self.q, self.k, self.v, self.cu


GEOMETRY = [(torch.bfloat16, 64, 150, 1), (torch.bfloat16, 128, 35, 5), (torch.bfloat16, 128, 100, 1), (torch.bfloat16, 128, 16, 4), (torch.bfloat16, 64, 4, 4), (torch.float32, 64, 4, 2), (torch.float32, 128, 8, 1), (torch.bfloat16, 128, 12, 4),
            (torch.bfloat16, 64, 14, 2), (torch.bfloat16, 128, 16, 1), (torch.bfloat16, 72, 6, 3), (torch.float32, 200, 2, 2), (torch.bfloat16, 256, 4, 1),
            (torch.bfloat16, 8, 2, 1), (torch.bfloat16, 128, 1, 1)]
LENGTHS = [[1], [2, 1, 1], [100], [128, 127, 129], [0, 300, 0, 0, 1, 64], [700, 33], [1] * 70 + [17] * 5]


@pytest.mark.parametrize("new", LENGTHS, ids=[str(sum(n)) + "x" + str(len(n)) for n in LENGTHS])
@pytest.mark.parametrize("dtype,c,nh,n_kv", GEOMETRY)
def test_prompts(kch, new, dtype, c, nh, n_kv):
    m = Prompts(new, dtype=dtype, nh=nh, n_kv=n_kv, c=c)
    want, tol = reference(m, m.q)
    got = kch.prompt_attention(*m.args)
    assert got.dtype == dtype and got.is_contiguous()
    close(got, want, tol)
    sink = torch.randn(nh, generator=m.g, device=DEV)
    want, tol = reference(m, m.q, scale=-0.3, window=37, sink=sink)
    close(kch.prompt_attention(*m.args, scale=-0.3, sliding_window=37, sink_logits=sink), want, tol)


@pytest.mark.parametrize("window", [1, 128, 1000])
@pytest.mark.parametrize("dtype,nh,n_kv,c", [(torch.bfloat16, 16, 4, 128), (torch.bfloat16, 8, 8, 64), (torch.float32, 2, 1, 64)])
def test_longer_prompts_and_windows(kch, dtype, nh, n_kv, c, window):
    m = Prompts([2500, 1, 1300], dtype=dtype, nh=nh, n_kv=n_kv, c=c, seed=window)
    for w in (0, window):
        want, tol = reference(m, m.q, window=w)
        close(kch.prompt_attention(*m.args, sliding_window=w), want, tol)


@pytest.mark.parametrize("dtype,c", [(torch.bfloat16, 128), (torch.bfloat16, 72), (torch.float32, 64)])
def test_rows_of_no_sequence(kch, dtype, c):
    m = Prompts([0, 5, 0, 130, 0], dtype=dtype, c=c, first_row=3, rows_behind=70)
    for x in (m.q, m.k, m.v):
        x[:3], x[138:] = torch.nan, torch.inf
    want, tol = reference(m, m.q)
    got = kch.prompt_attention(*m.args)
    close(got, want, tol)                                   # (zeros outside)
    out = torch.full((m.N, 4, c), 5., dtype=dtype, device=DEV)
    assert kch.prompt_attention(*m.args, out=out) is out
    assert torch.equal(out[3:138], got[3:138]) and (out[:3] == 5).all() and (out[138:] == 5).all()
    empty = torch.zeros_like(m.cu)
    assert not kch.prompt_attention(m.q, m.k, m.v, empty).any()
    assert kch.prompt_attention(m.q[:0], m.k[:0], m.v[:0], empty).shape == (0, 4, c)


@pytest.mark.parametrize("window", [0, 50])
@pytest.mark.parametrize("dtype,c", [(torch.bfloat16, 128), (torch.bfloat16, 64), (torch.float32, 64), (torch.bfloat16, 72)])
def test_what_a_query_does_not_see_does_not_reach_it(kch, dtype, c, window):
    """Infinities and NaN in other prompts, ahead of a query and behind its window."""
    m = Prompts([150, 200, 90], dtype=dtype, c=c, seed=4)
    m.k[:150], m.v[:150:2], m.v[1:150:2] = torch.nan, torch.nan, torch.inf
    m.k[350:], m.v[350:] = torch.inf, torch.nan
    m.v[150 + 40, 0, 3] = torch.inf
    want, tol = reference(m, m.q, window=window)
    got = kch.prompt_attention(*m.args, sliding_window=window)
    assert want[150:190].isfinite().all() and not want[190, 0].isfinite().all()
    close(got[150:350], want[150:350], tol[150:350])
    # a key that is NaN makes those that see it NaN, and no other
    m.v[190, 0, 3], m.k[150 + 77, 1] = 0., torch.nan
    got = kch.prompt_attention(*m.args, sliding_window=window)[150:350]
    sees = torch.zeros(200, dtype=torch.bool, device=DEV)
    sees[77:77 + window if window else None] = True
    assert got[:, :2].isfinite().all() and got[~sees].isfinite().all() and got[sees][:, 2:].isnan().all()


def test_large_logits_and_sinks(kch):
    for dtype in (torch.bfloat16, torch.float32):
        m = Prompts([5, 300], dtype=dtype, c=64)
        m.q *= 30
        sink = torch.tensor([-torch.inf, 50., 1000., torch.inf], device=DEV)
        want, tol = reference(m, m.q, sink=sink)
        got = kch.prompt_attention(*m.args, sink_logits=sink)
        close(got[:, :3], want[:, :3], tol[:, :3])
        assert not got[:, 3].any()


@pytest.mark.parametrize("dtype,nh,n_kv,c,page", [(torch.bfloat16, 16, 4, 128, 128), (torch.bfloat16, 4, 2, 64, 16), (torch.float32, 4, 2, 64, 32)])
def test_a_prompt_is_what_the_cache_attends(kch, dtype, nh, n_kv, c, page):
    """The same rows as pages, which are divided over the chip in another way: within both calls' roundings."""
    m = Prompts([700, 40, 1], dtype=dtype, nh=nh, n_kv=n_kv, c=c)
    pages = -(-700 // page)
    cache = kch.PagedKVCache(3 * pages, page, n_kv, c, DEV, dtype)
    table = torch.randperm(3 * pages, generator=m.g, device=DEV).view(3, pages).to(torch.int32)
    t0 = torch.zeros(3, dtype=torch.int32, device=DEV)
    cache.append_step(m.k, m.v, table, t0, m.cu)
    want, tol = reference(m, m.q, window=300)
    close(kch.prompt_attention(*m.args, sliding_window=300), want, tol)
    close(cache.forward_step(m.q, table, t0, m.cu, sliding_window=300), want, tol)


def test_operands_of_other_strides_and_outputs_on_16_bytes(kch):
    for c in (128, 64):
        m = Prompts([200, 33], c=c, nh=6, n_kv=2, pad=8)
        want = kch.prompt_attention(*m.args)
        q, k, v = (x.contiguous() for x in (m.q, m.k, m.v))
        assert torch.equal(kch.prompt_attention(q, k, v, m.cu), want)
        assert torch.equal(kch.prompt_attention(q.transpose(0, 1).contiguous().transpose(0, 1), k, v, m.cu), want)
        odd = torch.empty(m.N * 2 * c + 1, device=DEV).bfloat16()[1:].view(m.N, 2, c).copy_(k)      # not on 16 bytes
        assert torch.equal(kch.prompt_attention(q, odd, v, torch.stack([m.cu, m.cu], 1)[:, 0]), want)
        room = torch.full((8 + want.numel() + 8,), 7.0, dtype=want.dtype, device=DEV)
        out = room[8:8 + want.numel()].view(want.shape)
        assert out.data_ptr() % 32 == 16
        kch.prompt_attention(*m.args, out=out)
        assert torch.equal(out, want) and (room[:8] == 7).all() and (room[-8:] == 7).all()


@pytest.mark.parametrize("dtype,c", [(torch.bfloat16, 128), (torch.float32, 64)])
def test_a_captured_call_replays_with_other_lengths(kch, dtype, c):
    m = Prompts([300, 0, 100], dtype=dtype, c=c)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        kch.prompt_attention(*m.args)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = kch.prompt_attention(*m.args)
    for new in ([300, 0, 100], [1, 398, 1], [133, 133, 100]):
        m.new = new
        m.cu.copy_(torch.tensor([sum(new[:i]) for i in range(4)], dtype=torch.int32))
        m.both.normal_(generator=m.g)
        graph.replay()
        want, tol = reference(m, m.q)
        close(out, want, tol)
        assert torch.equal(out, kch.prompt_attention(*m.args))


def test_calls_on_two_streams_at_once(kch):
    ms = [Prompts([400, 30, 1000], seed=s, nh=8, n_kv=2) for s in (1, 2)]
    want = [kch.prompt_attention(*m.args) for m in ms]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream(), torch.cuda.Stream()], [[], []]
    for _ in range(10):
        for i, m in enumerate(ms):
            with torch.cuda.stream(streams[i]):
                got[i].append(kch.prompt_attention(*m.args))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(g, want[i]) for g in got[i])


def test_lengths_out_of_range_stay_in_the_tensors(kch):
    """cu_seqlens that begins in front of the rows, ends behind them, or falls: rows outside are left alone, nothing else is touched."""
    m = Prompts([40, 60], c=64)
    room = torch.full((300, 4, 64), 5., dtype=torch.bfloat16, device=DEV)
    out = room[100:200]
    want = kch.prompt_attention(*m.args)
    kch.prompt_attention(m.q, m.k, m.v, torch.tensor([0, 40, 5000], dtype=torch.int32, device=DEV), out=out)
    assert torch.equal(out, want) and (room[:100] == 5).all() and (room[200:] == 5).all()
    kch.prompt_attention(m.q, m.k, m.v, torch.tensor([-7, 40, 100], dtype=torch.int32, device=DEV), out=out)
    assert torch.equal(out, want) and (room[:100] == 5).all() and (room[200:] == 5).all()


def test_lengths_that_fall_and_rise_again_beyond_what_is_counted_do_nothing(kch):
    """Every other prompt has all rows: more steps in all than 32 bits hold, which the host, who sees N alone, cannot know."""
    from kch_b200 import _lib
    assert _lib.device_status() == 0
    N, B, n_kv = 65536, 4096, 32
    cu = (torch.arange(B + 1, device=DEV) % 2 * N).int()
    q, out = torch.zeros(N, n_kv, 64, dtype=torch.bfloat16, device=DEV), torch.full((N, n_kv, 64), 7.0, dtype=torch.bfloat16, device=DEV)
    kch.prompt_attention(q, q, q, cu, out=out)
    torch.cuda.synchronize()
    assert _lib.device_status(reset=True) == _lib.STATUS_PAGED_TABLE
    assert (out == 7).all()


def test_many_prompts_of_a_token_and_a_few(kch):
    """More prompts than a block has threads; one key head and as many as there are query heads."""
    for nh, n_kv in ((4, 1), (3, 3)):
        m = Prompts([1 + i % 5 + (i % 97 == 0) * 200 for i in range(900)], nh=nh, n_kv=n_kv, c=64, seed=nh)
        want, tol = reference(m, m.q)
        close(kch.prompt_attention(*m.args), want, tol)


def test_rows_beyond_32_bits_of_elements(kch):
    """Keys and values whose last rows lie behind 2^32 elements."""
    N, c = 2 ** 17, 128
    wide = torch.empty(N, 2 ** 15 + 2 * c, device=DEV, dtype=torch.bfloat16)          # 8.7 GB: tokens 33 024 elements apart
    k, v = (wide[:, 2 ** 15 + i * c:2 ** 15 + (i + 1) * c].unflatten(1, (1, c)) for i in range(2))
    q = torch.randn(N, 1, c, device=DEV).bfloat16()
    k.normal_(), v.normal_()
    got = kch.prompt_attention(q, k, v, torch.tensor([N - 300, N], dtype=torch.int32, device=DEV))
    m = Prompts([300], nh=1, n_kv=1)
    m.q, m.k, m.v = q[-300:], k[-300:], v[-300:]
    want, tol = reference(m, m.q)
    close(got[-300:], want, tol)
    assert not got[:-300].any()


def test_what_python_refuses(kch):
    m = Prompts([2, 3], c=64)
    q, k, v, cu = m.args
    call = kch.prompt_attention
    for args, kw, error, what in (
            ((q[:, :3], k, v, cu), {}, ValueError, "multiple of n_kv"), ((q, k.float(), v, cu), {}, ValueError, "dtype"), ((q, k.cpu(), v, cu), {}, RuntimeError, "CUDA"),
            ((q, k[..., :32], v, cu), {}, ValueError, "heads of 32"), ((q, k, v[:, :1], cu), {}, ValueError, "shape of k"), ((q, k[:4], v[:4], cu), {}, ValueError, "k must be"),
            ((q, k, v, cu.long()), {}, TypeError, "int32"), ((q, k, v, cu[:1]), {}, ValueError, "2 to 4097"), ((q, k, v, cu.cpu()), {}, ValueError, "cu_seqlens is on"),
            ((q, k, v, cu), dict(sliding_window=-1), ValueError, "sliding_window"), ((q, k, v, cu), dict(sliding_window=True), ValueError, "sliding_window"),
            ((q, k, v, cu), dict(sink_logits=torch.zeros(3, device=DEV)), ValueError, "sink_logits"), ((q, k, v, cu), dict(out=q[:4]), ValueError, "out must be"),
            ((q, k, v, cu), dict(scale=float("nan")), ValueError, "scale"), ((q[0], k, v, cu), {}, ValueError, "q must be")):
        with pytest.raises(error, match=what):
            call(*args, **kw)
    flat = torch.zeros(5, 4, 64, dtype=torch.bfloat16, device=DEV)
    with pytest.raises(ValueError, match="overlaps"):
        call(flat, k, v, cu, out=flat)
