"""Rotary positions between tensors whose tokens lie differently far apart: slices of one projection turned into slices of another.  Oracle and
tolerances are those of test_gpu_rotary.py."""
import pytest
import torch

from test_gpu_rotary import DEV, freqs, near, positions_of

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def kch():
    import kch_b200
    yield kch_b200


@pytest.mark.parametrize("N", [1, 2, 77, 1500])
@pytest.mark.parametrize("neighbours", [False, True])
@pytest.mark.parametrize("dtype,c,r,nh,n_kv", [(torch.bfloat16, 128, 128, 6, 2), (torch.bfloat16, 128, 64, 5, 1), (torch.float32, 64, 64, 3, 3),
                                               (torch.float32, 80, 24, 2, 4), (torch.bfloat16, 24, 10, 7, 1), (torch.bfloat16, 256, 32, 1, 1)])
def test_slices_into_slices_of_other_strides(kch, dtype, c, r, nh, n_kv, neighbours, N):
    g = torch.Generator(device=DEV).manual_seed(N + c)
    rope, pos = kch.RotaryPositions(c, DEV, rotary_dim=r, neighbours=neighbours), positions_of(N, 1, g, 5000)
    wide = torch.randn(N, (nh + 2 * n_kv) * c + 16, generator=g, device=DEV).to(dtype)
    q, k = wide[:, 8:8 + nh * c].unflatten(1, (nh, c)), wide[:, 8 + nh * c:8 + (nh + n_kv) * c].unflatten(1, (n_kv, c))
    was = wide.clone()
    kw = dict(r=r, sections=(r // 2,), inv_freq=freqs(r), neighbours=neighbours)
    want = rope.rotate(q, k, pos)
    near(want[0], q, pos, **kw)
    near(want[1], k, pos, **kw)
    # k's tokens further apart than q's, behind one another's, in one buffer and in two; what lies between them stays
    room = torch.full((N, (nh + 3 * n_kv) * c + 24), 7., dtype=dtype, device=DEV)
    to_q, to_k = room[:, :nh * c].unflatten(1, (nh, c)), room[:, 16 + nh * c:16 + (nh + n_kv) * c].unflatten(1, (n_kv, c))
    got = rope.rotate(q, k, pos, out=(to_q, to_k))
    assert got[0] is to_q and got[1] is to_k and torch.equal(to_q, want[0]) and torch.equal(to_k, want[1])
    assert (room[:, nh * c:16 + nh * c] == 7).all() and (room[:, 16 + (nh + n_kv) * c:] == 7).all() and torch.equal(wide, was)
    apart = torch.full((2 * N, n_kv, c), 7., dtype=dtype, device=DEV)
    dense = torch.empty_like(want[0])
    rope.rotate(q, k, pos, out=(dense, apart[::2]))
    assert torch.equal(dense, want[0]) and torch.equal(apart[::2], want[1]) and (apart[1::2] == 7).all()
    # a dense k beside a sliced q, turned in place, and q alone
    mine, own_k = wide.clone(), k.contiguous()
    own_q = mine[:, 8:8 + nh * c].unflatten(1, (nh, c))
    rope.rotate(own_q, own_k, pos, out=(own_q, own_k))
    assert torch.equal(own_q, want[0]) and torch.equal(own_k, want[1])
    mine[:, 8:8 + nh * c] = was[:, 8:8 + nh * c]
    assert torch.equal(mine, was)
    assert torch.equal(rope.rotate(q, None, pos, out=(to_q.zero_(), None))[0], want[0])
