"""Causal softmax attention of whole prompts, packed one behind the other, beside the stack's own layers.

Not in the reference.  What :class:`PagedKVCache` attends in its pages, with the keys and values still the activations that a projection
has left: the prompt is then attended as it is, whatever kind of cache keeps it (its 8- or 4-bit rows serve the tokens that follow,
``PagedKVCache.forward_step``).  Forward only: tensors that require a gradient are refused while gradients are enabled.
"""
from __future__ import annotations

import torch

from . import _lib
from .paged_cache import _packed

_ws_bytes = {}                  # of calls, by their sizes


def _error(q, k, v, cu_seqlens, sink_logits):
    fn = "prompt_attention"
    for name, x in (("q", q), ("k", k), ("v", v)):
        if x.dim() != 3 or x.shape[0] != q.shape[0] or x.shape[1] < 1:
            raise ValueError(f"{fn}: {name} must be [{'N' if x is q else q.shape[0]}, heads, c], got {tuple(x.shape)}")
        if not x.is_cuda:
            raise RuntimeError(f"{fn}: backend 'b200' requires CUDA tensors (got a {x.device} tensor); there is no CPU fallback")
        if x.device != q.device:
            raise ValueError(f"{fn}: {name} is on {x.device}, q on {q.device}")
        if x.dtype != q.dtype:
            raise ValueError(f"{fn}: {name}.dtype={x.dtype} does not match q's {q.dtype}")
        if x.shape[2] != q.shape[2]:
            raise ValueError(f"{fn}: {name} has heads of {x.shape[2]}, q of {q.shape[2]}")
    if k.shape != v.shape:
        raise ValueError(f"{fn}: v {tuple(v.shape)} must have the shape of k, {tuple(k.shape)}")
    if cu_seqlens.dim() != 1 or not 2 <= cu_seqlens.shape[0] <= 4097:
        raise ValueError(f"{fn}: cu_seqlens must have 2 to 4097 entries, got shape {tuple(cu_seqlens.shape)}")
    if cu_seqlens.dtype != torch.int32:
        raise TypeError(f"{fn}: cu_seqlens must be int32, got {cu_seqlens.dtype}")
    if cu_seqlens.device != q.device:
        raise ValueError(f"{fn}: cu_seqlens is on {cu_seqlens.device}, q on {q.device}")
    raise ValueError(f"{fn}: sink_logits must be [{q.shape[1]}] on {q.device}, got {tuple(sink_logits.shape)} on {sink_logits.device}")


def prompt_attention(q, k, v, cu_seqlens, *, scale=None, sink_logits=None, sliding_window=0, out=None):
    """``q [N, nh, c]``, ``k`` and ``v`` ``[N, n_kv, c]`` (fp32 or bf16; ``nh`` a multiple of ``n_kv``, query head h reads key head
    ``h // (nh // n_kv)``; column slices of a fused projection are read where they lie) -> ``[N, nh, c]`` in their dtype.

    Rows ``cu_seqlens[b] .. cu_seqlens[b + 1]`` (int32 ``[B + 1]`` on the device, at most 4096 sequences) are sequence b, and a token sees
    its sequence up to itself, or the last ``sliding_window`` tokens of that.  ``scale``: ``c ** -0.5`` unless given; ``sink_logits [nh]`` adds
    ``exp(sink)`` to the denominator.  Rows of no sequence are zeros, and stay as they are in a tensor given as ``out``, which overlaps
    none of the others.  The lengths stay on the device: a captured call replays with other ones."""
    if q.requires_grad or k.requires_grad or v.requires_grad or (sink_logits is not None and sink_logits.requires_grad):
        _lib.forward_only("prompt_attention")
    shape, kv, index, dtype = q.shape, k.shape, q.get_device(), q.dtype
    tag = _lib.dtype_tag(dtype)
    if not (len(shape) == len(kv) == 3 and kv == v.shape and shape[0] == kv[0] and shape[2] == kv[2] and shape[1] > 0 and kv[1] > 0 and index >= 0
            and k.dtype is v.dtype is dtype and k.get_device() == index == v.get_device() and cu_seqlens.get_device() == index
            and cu_seqlens.dtype is torch.int32 and cu_seqlens.dim() == 1 and 2 <= cu_seqlens.shape[0] <= 4097
            and (sink_logits is None or (sink_logits.shape == shape[1:2] and sink_logits.get_device() == index))):
        _error(q, k, v, cu_seqlens, sink_logits)
    (N, nh, c), n_kv, B = shape, kv[1], cu_seqlens.shape[0] - 1
    if nh % n_kv:
        raise ValueError(f"prompt_attention: nh={nh} must be a multiple of n_kv={n_kv}")
    if not isinstance(sliding_window, int) or isinstance(sliding_window, bool) or sliding_window < 0:
        raise ValueError(f"prompt_attention: sliding_window={sliding_window!r} must be an int >= 0 (0: every key)")
    lib = _lib.load()
    with _lib.device(q.device):
        sink, sink_tag = None, 0
        if sink_logits is not None:
            sink_logits = sink_logits.contiguous()
            sink, sink_tag = sink_logits.data_ptr(), _lib.dtype_tag(sink_logits.dtype)
        if not cu_seqlens.is_contiguous():
            cu_seqlens = cu_seqlens.contiguous()
        if out is None:
            o = torch.empty_strided(shape, (nh * c, c, 1), dtype=dtype, device=q.device)
        else:
            o = out
            if o.shape != shape or o.dtype is not dtype or o.get_device() != index or not o.is_contiguous() or o.data_ptr() % 16:
                raise ValueError(f"prompt_attention: out must be a contiguous {tuple(shape)} tensor on 16 bytes in {dtype} on {q.device}, got "
                                 f"{tuple(o.shape)} in {o.dtype} on {o.device}")
        (q, at_q, ld_q), (k, at_k, ld_k), (v, at_v, ld_v) = _packed(q), _packed(k), _packed(v)
        a = _lib.PromptAttendArgs(at_q, at_k, at_v, ld_q, ld_k, ld_v, cu_seqlens.data_ptr(), B, N, tag, nh, n_kv, c,
                                  c ** -0.5 if scale is None else float(scale), min(sliding_window, 0x7FFFFFFF), sink, sink_tag, o.data_ptr(),
                                  int(out is None))
        sizes = (N, nh, n_kv, c, B, tag)
        nbytes = _ws_bytes.get(sizes)
        if nbytes is None:
            if len(_ws_bytes) > 4096:
                _ws_bytes.clear()
            nbytes = _ws_bytes[sizes] = int(lib.kch_prompt_attend_workspace_bytes(a))
        ws = torch.empty_strided((nbytes,), (1,), dtype=torch.uint8, device=q.device)
        a.workspace, a.workspace_bytes = ws.data_ptr(), nbytes
        _lib.check(lib.kch_prompt_attend(a, _lib.stream()))
    return o
