"""What the paged cache refuses before any launch: by the class's own checks and by the C entry points."""
import ctypes

import pytest
import torch


def test_constructor_arguments():
    import kch_b200
    for args, what in (((0, 16, 1, 64), "num_pages"), ((4, 12, 1, 64), "page_size"), ((4, 4, 1, 64), "page_size"), ((4, 512, 1, 64), "page_size"),
                       ((4, 16, 0, 64), "n_kv"), ((4, 16, 1, 60), "c=60"), ((4, 16, 1, 264), "c=264"), ((True, 16, 1, 64), "num_pages"),
                       ((2 ** 31, 16, 1, 64), "num_pages"), ((4, 16.0, 1, 64), "page_size")):
        with pytest.raises(ValueError, match=what):
            kch_b200.PagedKVCache(*args, "cuda", torch.bfloat16)
    with pytest.raises(ValueError, match="kv_quant"):
        kch_b200.PagedKVCache(4, 16, 1, 64, "cuda", torch.bfloat16, kv_quant="fp4")
    with pytest.raises(TypeError):
        kch_b200.PagedKVCache(4, 16, 1, 64, "cuda", torch.float16)
    with pytest.raises(RuntimeError, match="CUDA"):
        kch_b200.PagedKVCache(4, 16, 1, 64, "cpu", torch.bfloat16)
    k = torch.zeros(4, 1, 16, 64)
    with pytest.raises(ValueError, match="storage"):
        kch_b200.PagedKVCache(4, 16, 1, 64, "cuda", torch.float32, storage=(k, k))
    with pytest.raises(ValueError, match="k_pages"):
        kch_b200.PagedKVCache(4, 16, 1, 64, "cuda", torch.bfloat16, storage=(k, k, None, None))
    with pytest.raises(ValueError, match="k_scales"):
        kch_b200.PagedKVCache(4, 16, 1, 64, "cuda", torch.float32, storage=(k, k, k, None))
    with pytest.raises(ValueError, match="is on cpu"):
        kch_b200.PagedKVCache(4, 16, 1, 64, "cuda", torch.float32, storage=(k, k, None, None))


def _args(lib_mod, **over):
    """Arguments of kch_paged_attend that pass every check up to the workspace's; the pointers are never followed."""
    v = dict(k=4096, v=4096, ks=4096, vs=4096, kind=1, num_pages=4, page_size=16, n_kv=2, c=64, table=4096, ld_table=2, max_pages=2, t0=4096,
             cu=4096, B=1, N=3, q=4096, ld_q=256, dtype=1, nh=4, scale=0.125, window=0, sink=None, sink_dtype=0, out=4096, ws=4096, ws_bytes=0)
    v.update(over)
    a = lib_mod.PagedAttendArgs()
    a.cache = lib_mod.PagedCache(v["k"], v["v"], v["ks"], v["vs"], v["kind"], v["num_pages"], v["page_size"], v["n_kv"], v["c"])
    a.batch = lib_mod.PagedBatch(v["table"], v["ld_table"], v["max_pages"], v["t0"], v["cu"], v["B"], v["N"])
    a.q, a.ld_q, a.dtype, a.nh, a.scale, a.sliding_window = v["q"], v["ld_q"], v["dtype"], v["nh"], v["scale"], v["window"]
    a.sink, a.sink_dtype, a.out, a.workspace, a.workspace_bytes = v["sink"], v["sink_dtype"], v["out"], v["ws"], v["ws_bytes"]
    return a


@pytest.mark.parametrize("over,what", [
    (dict(dtype=2), "dtype"), (dict(kind=0), "kind"), (dict(c=60), "c=60"), (dict(c=0), "c=0"), (dict(page_size=24), "page_size"),
    (dict(n_kv=0), "n_kv"), (dict(num_pages=0), "num_pages"), (dict(B=0), "B=0"), (dict(B=5000), "B=5000"), (dict(N=-1), "N=-1"),
    (dict(max_pages=0), "max_pages"), (dict(ld_table=1), "apart"), (dict(table=None), "null table"), (dict(t0=None), "null table"),
    (dict(cu=None), "null table"), (dict(k=None), "pages"), (dict(v=4104), "16-byte"), (dict(kind=2, ks=None), "scales"),
    (dict(nh=3), "nh=3"), (dict(nh=0), "nh=0"), (dict(window=-1), "sliding_window"), (dict(scale=float("nan")), "scale"),
    (dict(sink=4096, sink_dtype=3), "sink"), (dict(q=None), "null q"), (dict(ld_q=255), "ld_q=255"), (dict(ld_q=260), "ld_q=260"),
    (dict(out=4100), "16-byte"), (dict(), "workspace"), (dict(ws=None, ws_bytes=1 << 40), "workspace"), (dict(ws=4112, ws_bytes=1 << 40), "workspace"),
    (dict(N=1 << 24, nh=32, ld_q=32 * 64, max_pages=1 << 26, ld_table=1 << 26, ws_bytes=1 << 40), "more than a call takes"),
    (dict(N=1 << 30, nh=4, ws_bytes=1 << 40), "N \\* nh")])
def test_attend_arguments_are_refused_by_name(over, what):
    from kch_b200 import _lib
    lib = _lib.load()
    with pytest.raises(ValueError, match=what):
        _lib.check(lib.kch_paged_attend(_args(_lib, **over), None))


def test_rows_arguments_are_refused_by_name():
    from kch_b200 import _lib
    lib = _lib.load()
    a = _args(_lib)
    good = (4096, 128, 4096, 128)
    for rows, what in (((None, 128, 4096, 128), "null k"), ((4096, 127, 4096, 128), "ld_k=127"), ((4096, 128, 4096, 132), "ld_v=132"),
                       ((4098, 128, 4096, 128), "16-byte")):
        with pytest.raises(ValueError, match=what):
            _lib.check(lib.kch_paged_append(a.cache, a.batch, *rows, 1, None))
        with pytest.raises(ValueError, match=what):
            _lib.check(lib.kch_paged_read(a.cache, a.batch, *rows, 1, 0, None))
    with pytest.raises(ValueError, match="kind"):
        _lib.check(lib.kch_paged_append(a.cache, a.batch, *good, 0, None))
    for fn in (lambda: lib.kch_paged_append(None, a.batch, *good, 1, None), lambda: lib.kch_paged_read(a.cache, None, *good, 1, 0, None),
               lambda: lib.kch_paged_attend(None, None)):
        with pytest.raises(ValueError, match="null"):
            _lib.check(fn())


def test_workspace_grows_with_the_width_and_asks_for_nothing_where_the_arguments_are_empty():
    from kch_b200 import _lib
    lib = _lib.load()
    sizes = [int(lib.kch_paged_attend_workspace_bytes(_args(_lib, c=c))) for c in (64, 128, 256)]
    assert 0 < sizes[0] < sizes[1] < sizes[2]
    assert lib.kch_paged_attend_workspace_bytes(None) == 0
    assert lib.kch_paged_attend_workspace_bytes(_args(_lib, n_kv=0)) == 0
    assert ctypes.sizeof(_lib.PagedAttendArgs) == ctypes.sizeof(_lib.PagedCache) + ctypes.sizeof(_lib.PagedBatch) + 80


@pytest.mark.parametrize("over", [dict(), dict(out=4096 + 2 * 256 * 2 + 2 * 248), dict(q=4096 + 2 * 256 * 3 - 16), dict(N=1, ld_q=1 << 20, out=4096 + 2 * 240)])
def test_an_output_over_the_queries_is_refused(over):
    from kch_b200 import _lib
    lib = _lib.load()
    with pytest.raises(ValueError, match="overlaps"):
        _lib.check(lib.kch_paged_attend(_args(_lib, ws_bytes=1 << 40, **over), None))


def test_more_rows_and_columns_than_32_bits_count_are_refused():
    from kch_b200 import _lib
    lib = _lib.load()
    for over in (dict(N=0x7FFFFE00 // 4 + 1), dict(nh=1 << 26, ld_q=1 << 32, N=1)):
        with pytest.raises(ValueError, match="N \\* nh"):
            _lib.check(lib.kch_paged_attend(_args(_lib, ws_bytes=1 << 40, **over), None))


def test_the_storage_of_a_cache_cannot_be_exchanged():
    import kch_b200
    cache = object.__new__(kch_b200.PagedKVCache)
    for name in ("k_pages", "v_pages", "k_scales", "v_scales"):
        with pytest.raises(AttributeError):
            setattr(cache, name, torch.zeros(1))
