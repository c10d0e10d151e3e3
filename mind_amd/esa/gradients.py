"""The gradient norm over many tensors, and clipping by it (esa_grad_norm / esa_grad_clip).

The reference sums its gradient norm on the host, one ``.item()`` per parameter
(core/pretraining_model.py:606-612), and its trainer clips; here the norm of
all tensors together stays on the device and nothing synchronises.
"""
from __future__ import annotations

import ctypes
import math

import torch

from .. import _lib

def _infinity(norm_type) -> int:
    norm_type = float(norm_type)
    if norm_type not in (2.0, math.inf):
        raise ValueError(f"norm_type must be 2 or inf (got {norm_type})")
    return int(norm_type == math.inf)


class _Lists:
    """The C ABI's arrays over tensors (as bytes): pointers, counts and dtypes of the tensors themselves or, where they
    are not all contiguous, of what ``held`` makes of those that are not (kept in ``tensors``)."""

    def __init__(self, given, held):
        describe = _lib.tensors().describe
        self.tensors = given
        self.ptrs, self.counts, self.dtypes, device, contiguous = describe(given)
        if device < 0:
            _lib.require_gpu(*given)
            _lib.require_one_device(*given)
        if not contiguous:
            self.tensors = [t if t.is_contiguous() and not t.is_neg() else held(t) for t in given]
            self.ptrs, self.counts, self.dtypes, _, _ = describe(self.tensors)
        self.n, self.device = len(given), given[0].device

    @property
    def arrays(self):
        return self.ptrs, self.counts, self.dtypes


def _copy(t: torch.Tensor) -> torch.Tensor:
    return t.resolve_neg().contiguous()


def _listed(tensors) -> list[torch.Tensor]:
    return [tensors] if isinstance(tensors, torch.Tensor) else list(tensors)


def _outputs(x: _Lists, clip: int):
    """(the norm's scalar, the workspace)."""
    need = ctypes.c_size_t(0)
    _lib.check(_lib.load().esa_grad_workspace_size(x.n, x.counts, clip, ctypes.byref(need)), "esa_grad_workspace_size")
    return (torch.empty((), dtype=torch.float32, device=x.device),
            torch.empty(max(int(need.value), 256), dtype=torch.uint8, device=x.device))


def _norm(x: _Lists, infinity: int) -> torch.Tensor:
    norm, ws = _outputs(x, 0)
    _lib.check(_lib.load().esa_grad_norm(x.n, x.ptrs, x.counts, x.dtypes, infinity, norm.data_ptr(), ws.data_ptr(), ws.numel(),
                                         _lib.stream_of(norm)), "esa_grad_norm")
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
    lists = _Lists(tensors, _copy)
    with _lib.on_device(tensors[0]):
        return _norm(lists, infinity)


def clip_gradients(grads, max_norm: float, norm_type: float = 2.0, out=None, error_if_nonfinite: bool = False) -> torch.Tensor:
    """The gradients times min(1, max_norm / (norm + 1e-6)), their norm (``grad_norm``) returned as a scalar on the
    device.

    grads: a list of float32 and bfloat16 tensors.  out: None (in place), or a list of tensors of the same shapes that
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
    if not error_if_nonfinite and isinstance(grads[0], torch.Tensor) and grads[0].is_cuda:
        done = _lib.tensors().clip(_lib.address("esa_grad_clip"), _lib.address("esa_grad_workspace_size"),
                                   _lib.stream_of(grads[0]), grads, targets, infinity, max_norm)
        if done is not None:
            _lib.check(done[0], "esa_grad_clip")
            return done[1]
    return _clip_with_copies(grads, targets, max_norm, infinity, error_if_nonfinite)


@torch.no_grad()
def _clip_with_copies(grads, targets, max_norm: float, infinity: int, error_if_nonfinite: bool) -> torch.Tensor:
    """``clip_gradients`` for lists of any layout, and what says why a call is refused."""
    src = _Lists(grads, _copy)
    if targets is grads:
        dst = src
    else:
        dst = _Lists(targets, lambda o: torch.empty(o.shape, dtype=o.dtype, device=o.device))
        _lib.require_one_device(grads[0], targets[0])
        misfit = _lib.tensors().misfit(grads, targets)
        if misfit == "shapes":
            raise ValueError("out must have its gradients' shapes")
        if misfit == "dtypes":
            raise TypeError("out must have its gradients' dtypes or be float32")
    if not _lib.tensors().separate(dst.arrays, None if dst is src else src.arrays):
        raise ValueError("tensors that are written share memory with others of the call")
    with _lib.on_device(grads[0]):
        if error_if_nonfinite:
            value = float(_norm(src, infinity))
            if not math.isfinite(value):
                raise RuntimeError(f"the gradients' norm is {value}: they are not clipped")
        norm, ws = _outputs(src, 1)
        _lib.check(_lib.load().esa_grad_clip(src.n, src.ptrs, dst.ptrs, src.counts, src.dtypes, dst.dtypes, infinity, max_norm,
                                             norm.data_ptr(), ws.data_ptr(), ws.numel(), _lib.stream_of(norm)),
                   "esa_grad_clip")
        for target, held in zip(targets, dst.tensors) if dst.tensors is not targets else ():
            if held is not target:
                target.copy_(held)
        _lib.tensors().changed(targets)
    return norm


def clip_grad_norm_(parameters, max_norm: float, norm_type: float = 2.0, error_if_nonfinite: bool = False) -> torch.Tensor:
    """Clips the parameters' gradients in place by their norm together and returns it, as
    ``torch.nn.utils.clip_grad_norm_``; parameters without a gradient are passed over."""
    parameters = [parameters] if isinstance(parameters, torch.Tensor) else list(parameters)
    return clip_gradients([p.grad for p in parameters if p.grad is not None], max_norm, norm_type,
                          error_if_nonfinite=error_if_nonfinite)
