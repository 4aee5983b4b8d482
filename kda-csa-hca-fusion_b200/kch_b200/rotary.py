"""Rotary positions for the softmax attention beside the stack's own layers (:mod:`paged_cache`).

Not in the reference, whose layers carry no positions.  Queries and keys of packed tokens are turned in one launch, by positions on
one to four axes (a token's place in a text; or its time, height and width in a picture or a film).
"""
from __future__ import annotations

import ctypes
import math

import torch

from . import _lib
from .paged_cache import _packed


def _whole(name, v, least, most):
    if not isinstance(v, int) or isinstance(v, bool) or not least <= v <= most:
        raise ValueError(f"RotaryPositions: {name}={v!r} must be an int from {least} to {most}")


class RotaryPositions:
    """Heads of ``c`` channels (a multiple of 8 up to 256), of which the first ``rotary_dim`` (all of them) are turned in pairs.

    Pair i is ``(i, i + rotary_dim / 2)``, or ``(2 i, 2 i + 1)`` with ``neighbours``, and turns by its token's position on an axis times
    ``base ** (-2 i / rotary_dim)``, or times ``inv_freq[i]`` (``rotary_dim / 2`` numbers: frequencies that are scaled, or that begin anew on
    each axis).  ``sections``: how many pairs each axis has, the first axis' first; without it there is one axis.
    """

    def __init__(self, c, device, *, rotary_dim=None, sections=None, base=10000.0, inv_freq=None, neighbours=False):
        _whole("c", c, 8, 256)
        if c % 8:
            raise ValueError(f"RotaryPositions: c={c} must be a multiple of 8")
        rotary_dim = c if rotary_dim is None else rotary_dim
        _whole("rotary_dim", rotary_dim, 2, c)
        if rotary_dim % 2:
            raise ValueError(f"RotaryPositions: rotary_dim={rotary_dim} must be even")
        pairs = rotary_dim // 2
        sections = (pairs,) if sections is None else tuple(sections)
        if not 1 <= len(sections) <= 4:
            raise ValueError(f"RotaryPositions: sections={sections} must name 1 to 4 axes")
        for n in sections:
            _whole("sections: pairs of an axis", n, 0, pairs)
        if sum(sections) != pairs:
            raise ValueError(f"RotaryPositions: sections={sections} have {sum(sections)} pairs, rotary_dim={rotary_dim} has {pairs}")
        if inv_freq is None:
            base = float(base)
            if not (base > 0 and math.isfinite(base)):
                raise ValueError(f"RotaryPositions: base={base!r} must be a positive number")
            inv_freq = [base ** (-2.0 * i / rotary_dim) for i in range(pairs)]
        inv_freq = [float(f) for f in (inv_freq.tolist() if isinstance(inv_freq, torch.Tensor) else inv_freq)]
        if len(inv_freq) != pairs or not all(math.isfinite(f) for f in inv_freq):
            raise ValueError(f"RotaryPositions: inv_freq must be {pairs} finite numbers")
        device = torch.device(device)
        if device.type != "cuda":
            raise RuntimeError(f"RotaryPositions: backend 'b200' requires a CUDA device, got {device}")
        self.c, self.rotary_dim, self.sections, self.neighbours = c, rotary_dim, sections, bool(neighbours)
        self._turns = torch.tensor([f / (2.0 * math.pi) for f in inv_freq], dtype=torch.float64, device=device)
        self.device, self._index, self._lib = self._turns.device, self._turns.get_device(), _lib.load()
        self._axes, self._table = len(sections), self._turns.data_ptr()
        self._sections = (ctypes.c_int * 4)(*sections)

    # A call of a decode step takes the host longer than the GPU: the checks compare what they can in one expression, and name the
    # argument at fault only where it fails.
    def _error(self, q, k, positions):
        for name, x in (("q", q), ("k", k)):
            if x is None:
                continue
            if x.dim() != 3 or x.shape[2] != self.c or x.shape[1] < 1 or x.shape[0] != q.shape[0]:
                raise ValueError(f"rotate: {name} must be [{'N' if x is q else q.shape[0]}, heads, {self.c}], got {tuple(x.shape)}")
            if x.get_device() != self._index:
                raise (ValueError if x.is_cuda else RuntimeError)(f"rotate: {name} is on {x.device}, the CUDA table on {self.device}")
            if x.dtype != q.dtype:
                raise ValueError(f"rotate: k.dtype={x.dtype} does not match q's {q.dtype}")
        N, axes = q.shape[0], len(self.sections)
        if positions.dtype != torch.int32:
            raise TypeError(f"rotate: positions must be int32, got {positions.dtype}")
        if tuple(positions.shape) != (N, axes) and not (axes == 1 and tuple(positions.shape) == (N,)):
            raise ValueError(f"rotate: positions must be [{N}, {axes}], got {tuple(positions.shape)}")
        raise ValueError(f"rotate: positions is on {positions.device}, the table on {self.device}")

    def _own_out(self, name, out, x):
        """``(its address, elements between tokens)`` of an output that has been given."""
        if x is None:
            if out is not None:
                raise ValueError("rotate: out has a tensor for k, which is None")
            return None, 0
        if out is None:
            raise ValueError(f"rotate: out needs a tensor for {name}")
        if out.shape != x.shape or out.dtype != x.dtype or out.device != x.device:
            raise ValueError(f"rotate: out ({name}) must be {tuple(x.shape)} in {x.dtype} on {x.device}, got {tuple(out.shape)} in {out.dtype} on {out.device}")
        y, at, ld = _packed(out)
        if y is not out:
            raise ValueError(f"rotate: out ({name}) must be dense within a token, begin on 16 bytes and have tokens a multiple of 16 bytes apart")
        return at, ld

    def rotate(self, q, k, positions, *, inverse=False, out=None):
        """``q [N, nh, c]`` and ``k [N, n_kv, c]`` (or None) turned by ``positions``, int32 ``[N, axes]`` (or ``[N]`` where there is
        one axis) on the device: ``(q', k')``.  ``inverse`` turns back, which is the gradient too; the call itself records none, and refuses
        tensors that require one while gradients are enabled.  ``out=(q', k')``: tensors to store to, which may be ``q`` and ``k`` themselves
        (column slices of a fused projection, say) and overlap nothing else."""
        if q.requires_grad or (k is not None and k.requires_grad):
            _lib.forward_only("rotate")
        shape, index, axes, dtype, c = q.shape, self._index, self._axes, q.dtype, self.c
        tag = _lib.dtype_tag(dtype)
        at, n_kv = positions.shape, 0
        if not (len(shape) == 3 and shape[2] == c and shape[1] > 0 and q.get_device() == index == positions.get_device()
                and positions.dtype is torch.int32 and (at == (shape[0], axes) or (axes == 1 and at == shape[:1]))):
            self._error(q, k, positions)
        N, nh, _ = shape
        if k is not None:
            other = k.shape
            if not (len(other) == 3 and other[0] == N and other[2] == c and other[1] > 0 and k.dtype is dtype and k.get_device() == index):
                self._error(q, k, positions)
            n_kv = other[1]
        ld = positions.stride(0) if N > 1 else axes
        if (axes > 1 and positions.stride(1) != 1) or ld < axes:
            positions = positions.contiguous()
            ld = axes
        with _lib.device(self.device):
            if out is None:
                ld_to_q, ld_to_k, to_k = nh * c, n_kv * c, None
                y = (torch.empty_strided(shape, (ld_to_q, c, 1), dtype=dtype, device=self.device),
                     None if k is None else torch.empty_strided(other, (ld_to_k, c, 1), dtype=dtype, device=self.device))
                to_q, to_k = y[0].data_ptr(), _lib.ptr(y[1])
            else:
                y = (out[0], out[1])
                (to_q, ld_to_q), (to_k, ld_to_k) = self._own_out("q", y[0], q), self._own_out("k", y[1], k)
            q, at_q, ld_q = _packed(q)
            k, at_k, ld_k = (None, None, 0) if k is None else _packed(k)
            a = _lib.RotaryArgs(at_q, at_k, to_q, to_k, ld_q, ld_k, ld_to_q, ld_to_k, N, nh, n_kv, c, tag, positions.data_ptr(), ld, axes,
                                self._sections, self._table, self.rotary_dim, self.neighbours, 1 if inverse else 0)
            _lib.check(self._lib.kch_rotary(a, _lib.stream()))
        return y
