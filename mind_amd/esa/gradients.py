"""The gradient norm over many tensors, and clipping by it (esa_grad_norm / esa_grad_clip).

The reference sums its gradient norm on the host, one ``.item()`` per parameter
(core/pretraining_model.py:606-612), and its trainer clips; here the norm of
all tensors together stays on the device and nothing synchronises.
"""
from __future__ import annotations

import ctypes
import math

import numpy as np
import torch

from .. import _lib

_CODES = {torch.float32: _lib.ESA_F32, torch.bfloat16: _lib.ESA_BF16}
_BYTES = np.array([4, 2], dtype=np.int64)   # by code


def _infinity(norm_type) -> int:
    norm_type = float(norm_type)
    if norm_type not in (2.0, math.inf):
        raise ValueError(f"norm_type must be 2 or inf (got {norm_type})")
    return int(norm_type == math.inf)


class _Lists:
    """The C ABI's arrays over tensors: pointers, counts and dtypes of the tensors themselves or, where one is not
    contiguous, of what ``held`` makes of it (kept in ``tensors``).  One list comprehension for each property: with
    hundreds of small tensors the host's time is the call's."""

    def __init__(self, name, given, held):
        dtypes = [t.dtype for t in given]
        for dt in set(dtypes):
            if dt not in _CODES:
                raise TypeError(f"{name} must be float32 or bfloat16 (got {dt})")
        devices = {t.get_device() for t in given}
        if min(devices) < 0:
            _lib.require_gpu(*given)
        if len(devices) > 1:
            _lib.require_one_device(*given)
        self.tensors = given
        if not all([t.is_contiguous() for t in given]):
            self.tensors = [t if t.is_contiguous() else held(t) for t in given]
        self.n, self.device = len(given), given[0].device
        self.at = [t.data_ptr() for t in self.tensors]
        self.size = [t.numel() for t in self.tensors]
        self.codes = [_CODES[dt] for dt in dtypes]
        self.ptrs = (ctypes.c_void_p * self.n)(*self.at)
        self.counts = (ctypes.c_longlong * self.n)(*self.size)
        self.dtypes = (ctypes.c_int * self.n)(*self.codes)

    def spans(self):
        """(first bytes, ends) of the tensors' memory."""
        first = np.array(self.at, dtype=np.int64)
        return first, first + np.array(self.size, dtype=np.int64) * _BYTES[self.codes]


def _listed(tensors) -> list[torch.Tensor]:
    return [tensors] if isinstance(tensors, torch.Tensor) else list(tensors)


def _norm(x: _Lists, infinity: int) -> torch.Tensor:
    first = x.tensors[0]
    norm = torch.empty((), dtype=torch.float32, device=x.device)
    lib, need = _lib.load(), ctypes.c_size_t(0)
    _lib.check(lib.esa_grad_norm_workspace_size(x.n, x.counts, ctypes.byref(need)), "esa_grad_norm_workspace_size")
    ws = torch.empty(max(int(need.value), 256), dtype=torch.uint8, device=x.device)
    _lib.check(lib.esa_grad_norm(x.n, x.ptrs, x.counts, x.dtypes, infinity, norm.data_ptr(), ws.data_ptr(), ws.numel(),
                                 _lib.stream_of(first)), "esa_grad_norm")
    return norm


@torch.no_grad()
def grad_norm(tensors, norm_type: float = 2.0) -> torch.Tensor:
    """The norm of all values of the float32 and bfloat16 tensors together, a float32 scalar on their device: sqrt of the
    sum of squares (norm_type 2, summed in float64 in a fixed order) or the largest magnitude (inf; a NaN gives NaN).
    No tensors: 0, on the host."""
    infinity = _infinity(norm_type)
    tensors = _listed(tensors)
    if not tensors:
        return torch.zeros(())
    lists = _Lists("tensors", tensors, torch.Tensor.contiguous)
    with _lib.on_device(tensors[0]):
        return _norm(lists, infinity)


def _separate(dst: _Lists, src: _Lists) -> bool:
    """Whether every written tensor keeps to itself: no byte of it is another written tensor's, nor another's gradient
    (its own gradient may lie exactly there)."""
    first, ends = dst.spans()
    some = np.flatnonzero(ends > first)
    some = some[np.argsort(first[some], kind="stable")]
    first, ends = first[some], ends[some]
    if np.any(ends[:-1] > first[1:]):
        return False
    if src is dst:
        return True
    read, read_ends = src.spans()
    lo, hi = np.searchsorted(ends, read, side="right"), np.searchsorted(first, read_ends, side="left")
    met = (hi > lo) & (read_ends > read)   # written tensors lo .. hi - 1 share bytes with the gradient
    at = np.minimum(lo, max(len(some) - 1, 0))
    if not met.any():
        return True
    own = (hi - lo == 1) & (some[at] == np.arange(src.n)) & (first[at] == read) & (ends[at] == read_ends)
    return bool(np.all(own | ~met))


@torch.no_grad()
def clip_gradients(grads, max_norm: float, norm_type: float = 2.0, out=None, error_if_nonfinite: bool = False) -> torch.Tensor:
    """The gradients times min(1, max_norm / (norm + 1e-6)), their norm (``grad_norm``) returned as a scalar on the
    device.

    grads: a list of float32 and bfloat16 tensors.  out: None (in place), or a list of tensors of the same sizes that
    take the clipped gradients, each of its gradient's dtype or float32 (bfloat16 gradients into float32 master
    gradients).  Tensors may be of any layout: what is not contiguous goes through a copy.  No two tensors written may
    share memory, nor a tensor written and another's gradient.  A NaN norm gives NaN throughout, an infinite one zeros
    (NaN where a gradient is infinite); with error_if_nonfinite such a norm raises before anything is written (that
    waits for the device).  Values are rounded once.  Nothing here is recorded by autograd.
    """
    infinity, max_norm = _infinity(norm_type), float(max_norm)
    if not max_norm >= 0.0:
        raise ValueError(f"max_norm must not be negative (got {max_norm})")
    grads = _listed(grads)
    targets = grads if out is None else _listed(out)
    if len(targets) != len(grads):
        raise ValueError(f"out has {len(targets)} tensors for {len(grads)} gradients")
    if not grads:
        return torch.zeros(())
    src = _Lists("grads", grads, torch.Tensor.contiguous)
    if out is None:
        dst = src
    else:
        dst = _Lists("out", targets, lambda o: torch.empty(o.shape, dtype=o.dtype, device=o.device))
        _lib.require_one_device(grads[0], targets[0])
        if src.size != dst.size:
            raise ValueError("out must have its gradients' numbers of values")
        if any(o != g and o != _lib.ESA_F32 for o, g in zip(dst.codes, src.codes)):
            raise TypeError("out must have its gradients' dtypes or be float32")
    if not _separate(dst, src):
        raise ValueError("tensors that are written share memory with others of the call")
    with _lib.on_device(grads[0]):
        norm = _norm(src, infinity)
        if error_if_nonfinite and not math.isfinite(float(norm)):
            raise RuntimeError(f"the gradients' norm is {float(norm)}: they are not clipped")
        _lib.check(_lib.load().esa_grad_clip(src.n, src.ptrs, dst.ptrs, src.counts, src.dtypes, dst.dtypes,
                                             max_norm, norm.data_ptr(), _lib.stream_of(grads[0])), "esa_grad_clip")
        for target, held in zip(targets, dst.tensors) if dst.tensors is not targets else ():
            if held is not target:
                target.copy_(held.view(target.shape))
        torch.autograd.graph.increment_version(targets)
    return norm


def clip_grad_norm_(parameters, max_norm: float, norm_type: float = 2.0, error_if_nonfinite: bool = False) -> torch.Tensor:
    """Clips the parameters' gradients in place by their norm together and returns it, as
    ``torch.nn.utils.clip_grad_norm_``; parameters without a gradient are passed over."""
    parameters = [parameters] if isinstance(parameters, torch.Tensor) else list(parameters)
    return clip_gradients([p.grad for p in parameters if p.grad is not None], max_norm, norm_type,
                          error_if_nonfinite=error_if_nonfinite)
