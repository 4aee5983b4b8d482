"""Rotary positions against complex products in 64 bits.

Tolerances.  The angle's remainder is off by 2^-53 of the turns (twice: the frequency's rounding and the product's) and by the rounding of
twice it to 32 bits, pi 2^-25; sine and cosine by 2 units of the last place at most, 2^-23; a product and a sum round by 2^-24 each.  All
of it weighs |x_a| + |x_b|; the output's rounding is half a step of its own value.
"""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.fixture(scope="module")
def kch():
    import kch_b200
    yield kch_b200


def oracle(x, positions, *, r, sections, inv_freq, neighbours=False, inverse=False):
    """(turned, tolerance) of x [N, heads, c] in 64 bits."""
    place = torch.cat([positions[:, a:a + 1].double().expand(-1, n) for a, n in enumerate(sections)], 1)
    angle = place * torch.tensor(inv_freq, dtype=torch.double, device=x.device)
    turn = torch.polar(torch.ones_like(angle), -angle if inverse else angle)[:, None]
    first, second = (slice(0, r, 2), slice(1, r, 2)) if neighbours else (slice(0, r // 2), slice(r // 2, r))
    y, tol = x.double().clone(), torch.zeros(x.shape, dtype=torch.double, device=x.device)
    z = torch.complex(y[..., first].contiguous(), y[..., second].contiguous())
    size = (z.real.abs() + z.imag.abs()) * (math.pi * 2.0 ** -25 + 2.0 ** -23 + 2 * 2.0 ** -24 + 3 * 2.0 ** -53 * angle.abs()[:, None])
    y[..., first], y[..., second] = (z * turn).real, (z * turn).imag
    tol[..., first] = tol[..., second] = size
    tol[..., :r] += torch.finfo(x.dtype).eps / 2 * y[..., :r].abs()
    return y, tol


def near(got, x, positions, **kw):
    want, tol = oracle(x, positions, **kw)
    off = (got.double() - want).abs()
    assert got.dtype == x.dtype and (off <= tol).all(), f"{float((off - tol).max()):.3e} beyond"


def freqs(r, base=10000.0):
    return [base ** (-2.0 * i / r) for i in range(r // 2)]


def positions_of(N, axes, g, far):
    return torch.randint(-3, far, (N, axes), generator=g, device=DEV, dtype=torch.int32)


CASES = [(torch.bfloat16, 128, 128, (64,), 16, 4), (torch.float32, 64, 64, (32,), 4, 2), (torch.bfloat16, 128, 128, (16, 24, 24), 12, 1),
         (torch.float32, 128, 96, (24, 24), 3, 3), (torch.bfloat16, 64, 32, (4, 6, 6), 4, 4), (torch.bfloat16, 72, 72, (36,), 5, 1),
         (torch.float32, 80, 20, (1, 2, 3, 4), 2, 1), (torch.bfloat16, 8, 2, (1,), 1, 1), (torch.bfloat16, 256, 256, (0, 128), 1, 1),
         (torch.float32, 256, 250, (125,), 7, 2), (torch.bfloat16, 8, 8, (4,), 1, 0), (torch.bfloat16, 128, 16, (8,), 40, 40)]


@pytest.mark.parametrize("N", [1, 3, 64, 1000, 5003])
@pytest.mark.parametrize("neighbours", [False, True])
@pytest.mark.parametrize("dtype,c,r,sections,nh,n_kv", CASES)
def test_queries_and_keys_are_turned_by_their_positions(kch, dtype, c, r, sections, nh, n_kv, neighbours, N):
    g = torch.Generator(device=DEV).manual_seed(N + c)
    rope = kch.RotaryPositions(c, DEV, rotary_dim=r, sections=sections, neighbours=neighbours)
    q = torch.randn(N, nh, c, generator=g, device=DEV).to(dtype)
    k = torch.randn(N, n_kv, c, generator=g, device=DEV).to(dtype) if n_kv else None
    pos = positions_of(N, len(sections), g, 40000)
    for inverse in (False, True):
        got = rope.rotate(q, k, pos, inverse=inverse)
        for x, y in zip((q, k), got):
            if x is None:
                assert y is None
                continue
            near(y, x, pos, r=r, sections=sections, inv_freq=freqs(r), neighbours=neighbours, inverse=inverse)
            assert torch.equal(y[..., r:], x[..., r:])


def test_far_positions_and_other_frequencies(kch):
    g = torch.Generator(device=DEV).manual_seed(1)
    pos = torch.tensor([0, 1, -1, 2 ** 31 - 1, -2 ** 31, 10 ** 9, 123456789, 2 ** 24 + 1], dtype=torch.int32, device=DEV)[:, None]
    for dtype in (torch.float32, torch.bfloat16):
        q = torch.randn(8, 3, 64, generator=g, device=DEV).to(dtype)
        rope = kch.RotaryPositions(64, DEV)
        near(rope.rotate(q, None, pos)[0], q, pos, r=64, sections=(32,), inv_freq=freqs(64))
        assert torch.equal(rope.rotate(q[:1], None, pos[:1])[0], q[:1])      # position 0 changes nothing
        near(kch.RotaryPositions(64, DEV, base=5e5).rotate(q, None, pos)[0], q, pos, r=64, sections=(32,), inv_freq=freqs(64, 5e5))
        own = torch.rand(16, generator=g, device=DEV) * 3 - 1
        near(kch.RotaryPositions(64, DEV, rotary_dim=32, inv_freq=own).rotate(q, None, pos[:, 0])[0], q, pos, r=32, sections=(16,),
             inv_freq=own.double().tolist())


def test_the_gradient_is_the_turn_back(kch):
    """Of a sum weighed by w, against differences in 64 bits of the formula."""
    g = torch.Generator(device=DEV).manual_seed(2)
    rope = kch.RotaryPositions(16, DEV, sections=(3, 5), neighbours=True)
    x, w = (torch.randn(5, 2, 16, generator=g, device=DEV) for _ in range(2))
    pos = positions_of(5, 2, g, 900)
    grad = rope.rotate(w, None, pos, inverse=True)[0].double()
    kw = dict(r=16, sections=(3, 5), inv_freq=freqs(16), neighbours=True)
    for at in ((0, 0, 0), (1, 1, 7), (4, 0, 15), (3, 1, 8)):
        up, down = x.double(), x.double()
        up[at] += 1e-3
        down[at] -= 1e-3
        slope = ((oracle(up, pos, **kw)[0] - oracle(down, pos, **kw)[0]) * w.double()).sum() / 2e-3
        # (linear: the difference is exact but for 64-bit rounding over 2e-3)
        assert abs(float(slope - grad[at])) <= 4e-6


@pytest.mark.parametrize("dtype,c", [(torch.bfloat16, 128), (torch.float32, 72), (torch.bfloat16, 24)])
def test_slices_of_a_fused_projection_in_place_and_out_of_place(kch, dtype, c):
    g = torch.Generator(device=DEV).manual_seed(3)
    N, nh, n_kv = 77, 6, 2
    both = torch.randn(N, (nh + 2 * n_kv) * c + 8, generator=g, device=DEV).to(dtype)
    cut = lambda t: (t[:, 8:8 + nh * c].unflatten(1, (nh, c)), t[:, 8 + nh * c:8 + (nh + n_kv) * c].unflatten(1, (n_kv, c)))      # noqa: E731
    r = 16 if c == 24 else c
    rope, pos = kch.RotaryPositions(c, DEV, rotary_dim=r), positions_of(N, 1, g, 5000)
    q, k = cut(both)
    want = rope.rotate(q, k, pos)
    near(want[0], q, pos, r=r, sections=(r // 2,), inv_freq=freqs(r))
    mine = both.clone()
    out = cut(mine)
    got = rope.rotate(*out, pos, out=out)
    assert got[0] is out[0] and got[1] is out[1]
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    assert torch.equal(mine[:, :8], both[:, :8]) and torch.equal(mine[:, 8 + (nh + n_kv) * c:], both[:, 8 + (nh + n_kv) * c:])
    # other strides, heads apart, addresses off 16 bytes: copied first
    assert torch.equal(rope.rotate(q.transpose(0, 1).contiguous().transpose(0, 1), k, pos)[0], want[0])
    odd = torch.empty(N * nh * c + 1, device=DEV, dtype=dtype)[1:].view(N, nh, c).copy_(q)
    assert torch.equal(rope.rotate(odd, k, pos)[0], want[0])
    wide = torch.stack([pos[:, 0]] * 3, 1)
    assert torch.equal(rope.rotate(q, k, wide[:, 1])[1], want[1]) and torch.equal(rope.rotate(q, k, wide[:, 1:2])[1], want[1])
    one = pos[:1, 0].expand(N)
    assert torch.equal(rope.rotate(q, k, one)[0], rope.rotate(q, k, one.contiguous())[0])


def test_infinities_and_nan_stay_in_their_pairs(kch):
    rope = kch.RotaryPositions(64, DEV)
    for dtype in (torch.bfloat16, torch.float32):
        q = torch.ones(4, 2, 64, device=DEV, dtype=dtype)
        q[2, 1, 5], q[1, 0, 40] = torch.nan, torch.inf
        got = rope.rotate(q, None, torch.arange(4, dtype=torch.int32, device=DEV))[0]
        odd = ~got.isfinite()
        want = torch.zeros_like(odd)
        want[2, 1, 5] = want[2, 1, 37] = want[1, 0, 40] = want[1, 0, 8] = True
        assert torch.equal(odd, want)


def test_no_rows(kch):
    rope = kch.RotaryPositions(64, DEV)
    q, k = rope.rotate(torch.empty(0, 4, 64, device=DEV), torch.empty(0, 2, 64, device=DEV), torch.empty(0, dtype=torch.int32, device=DEV))
    assert q.shape == (0, 4, 64) and k.shape == (0, 2, 64)


def test_a_captured_turn_replays_with_other_positions_and_streams_do_not_meet(kch):
    g = torch.Generator(device=DEV).manual_seed(4)
    rope = kch.RotaryPositions(128, DEV, sections=(16, 24, 24))
    q, k, pos = torch.randn(9, 8, 128, generator=g, device=DEV).bfloat16(), torch.randn(9, 2, 128, generator=g, device=DEV).bfloat16(), positions_of(9, 3, g, 100)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        rope.rotate(q, k, pos)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = rope.rotate(q, k, pos)
    for seed in range(3):
        pos.copy_(positions_of(9, 3, g, 9000))
        graph.replay()
        want = rope.rotate(q, k, pos)
        assert torch.equal(out[0], want[0]) and torch.equal(out[1], want[1])
        near(out[0], q, pos, r=128, sections=(16, 24, 24), inv_freq=freqs(128))


def test_more_elements_than_32_bits_count(kch):
    """q of 2^32 elements and more in place; the last tokens."""
    N, nh, c = 2 ** 17 + 3, 256, 128
    g = torch.Generator(device=DEV).manual_seed(5)
    q = torch.empty(N, nh, c, device=DEV, dtype=torch.bfloat16)
    q[:2].normal_(generator=g)
    q[-5:].normal_(generator=g)
    was = q[-5:].clone()
    pos = torch.arange(N, dtype=torch.int32, device=DEV)
    kch.RotaryPositions(c, DEV).rotate(q, None, pos, out=(q, None))
    near(q[-5:], was, pos[-5:, None], r=c, sections=(64,), inv_freq=freqs(c))


def test_what_python_refuses(kch):
    rope = kch.RotaryPositions(64, DEV, sections=(20, 12))
    q, k, pos = torch.zeros(3, 4, 64, device=DEV), torch.zeros(3, 2, 64, device=DEV), torch.zeros(3, 2, dtype=torch.int32, device=DEV)
    for call, error, what in (
            (lambda: rope.rotate(q[0], k, pos), ValueError, "q must be"), (lambda: rope.rotate(q, k[:2], pos), ValueError, "k must be"),
            (lambda: rope.rotate(q[:, :0], k, pos), ValueError, "q must be"), (lambda: rope.rotate(q, k.bfloat16(), pos), ValueError, "dtype"),
            (lambda: rope.rotate(q.half(), None, pos), TypeError, "float16"), (lambda: rope.rotate(q.cpu(), None, pos), RuntimeError, "CUDA"),
            (lambda: rope.rotate(q, k, pos.long()), TypeError, "int32"), (lambda: rope.rotate(q, k, pos[:, :1]), ValueError, "positions must be"),
            (lambda: rope.rotate(q, k, pos[:2]), ValueError, "positions must be"), (lambda: rope.rotate(q, k, pos.cpu()), ValueError, "positions is on"),
            (lambda: rope.rotate(q, k, pos, out=(q, None)), ValueError, "out needs"), (lambda: rope.rotate(q, None, pos, out=(q, k)), ValueError, "out has"),
            (lambda: rope.rotate(q, k, pos, out=(k, k)), ValueError, "out \\(q\\)"),
            (lambda: rope.rotate(q, k, pos, out=(q.transpose(0, 1).contiguous().transpose(0, 1), k)), ValueError, "dense"),
            (lambda: rope.rotate(q[1:], k[1:], pos[1:], out=(q[:2], k[1:])), ValueError, "overlaps")):
        with pytest.raises(error, match=what):
            call()
