"""What the paged cache in 4 bits refuses before any launch."""
import pytest
import torch

from test_paged_cpu import _args


@pytest.mark.parametrize("over,what", [(dict(c=72), "multiple of 32"), (dict(c=8), "multiple of 32"), (dict(ks=None), "scales"), (dict(vs=4104), "scales"),
                                       (dict(k=4104), "16-byte"), (dict(kind=5), "kind=5"), (dict(), "workspace")])
def test_arguments_are_refused_by_name(over, what):
    from kch_b200 import _lib
    lib = _lib.load()
    a = _args(_lib, **{"kind": 4, **over})
    with pytest.raises(ValueError, match=what):
        _lib.check(lib.kch_paged_attend(a, None))
    if what != "workspace":
        with pytest.raises(ValueError, match=what):
            _lib.check(lib.kch_paged_append(a.cache, a.batch, 4096, 128, 4096, 128, 1, None))
        with pytest.raises(ValueError, match=what):
            _lib.check(lib.kch_paged_read(a.cache, a.batch, 4096, 128, 4096, 128, 1, 0, None))


def test_constructor_arguments():
    import kch_b200
    with pytest.raises(ValueError, match="multiple of 32"):
        kch_b200.PagedKVCache(4, 16, 1, 40, "cuda", torch.bfloat16, kv_quant="int4")
    k, s = torch.zeros(4, 1, 16, 32, dtype=torch.uint8), torch.ones(4, 1, 16, 2, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="is on cpu"):
        kch_b200.PagedKVCache(4, 16, 1, 64, "cuda", torch.bfloat16, kv_quant="int4", storage=(k, k, s, s))
    with pytest.raises(ValueError, match="k_scales"):
        kch_b200.PagedKVCache(4, 16, 1, 64, "cuda", torch.bfloat16, kv_quant="int4", storage=(k, k, None, None))
    with pytest.raises(ValueError, match="kv_quant"):
        kch_b200.CSADecodingCache(1, 8, 4, 4, 4, "cuda", torch.bfloat16, kv_quant="int4")
