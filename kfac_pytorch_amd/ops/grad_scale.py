"""Rescaling a whole model's gradients by one number that they give.

* ``global_norm`` / ``clip_by_global_norm`` / ``clip_grad_norm_``: the norm
  over all tensors and clipping by it, as ``torch.nn.utils.clip_grad_norm_``.
* ``kl_clip``: K-FAC's trust region,
  ``nu = min(1, sqrt(kl_clip / |lr^2 sum_i <update_i, grad_i>|))``
  (reference: kfac/kfac_preconditioner_inv.py:188-217).

On the GPU two passes over the data, a few launches whatever the number of
tensors (``csrc/grad_scale.hip``), and no wait for the device: norms and
factors stay there.  On the CPU the plain expressions run.  None of them is
differentiated: results require no gradient, and tensors with a forward-mode
tangent raise.
"""

from __future__ import annotations

import bisect
import math
from typing import Iterable, List, Optional, Sequence, Tuple, Union

import torch
from torch.autograd import forward_ad

__all__ = ["global_norm", "clip_by_global_norm", "clip_grad_norm_",
           "kl_clip"]

_KINDS = {2.0: 0, 1.0: 1, math.inf: 2}
Tensors = Union[torch.Tensor, Iterable[torch.Tensor]]


def _as_list(tensors: Tensors) -> List[torch.Tensor]:
    if isinstance(tensors, torch.Tensor):
        return [tensors]
    return list(tensors)


# The GPU calls make the same checks in C++, where hundreds of tensors take
# some microseconds.
def _check_lists(name: str, *lists: Sequence[torch.Tensor]) -> None:
    first = lists[0]
    for other in lists[1:]:
        if len(other) != len(first):
            raise ValueError(f"{name}: lists of {len(first)} and "
                             f"{len(other)} tensors")
        for a, b in zip(first, other):
            if a.shape != b.shape:
                raise ValueError(f"{name}: shapes {tuple(a.shape)} and "
                                 f"{tuple(b.shape)} differ")
    device = first[0].device
    for group in lists:
        for t in group:
            if t.device != device:
                raise ValueError(f"{name}: tensors on {device} and "
                                 f"{t.device}")
            if not t.dtype.is_floating_point or t.layout != torch.strided:
                raise TypeError(f"{name}: dense floating tensors expected, "
                                f"got {t.dtype}, {t.layout}")
            if forward_ad.unpack_dual(t).tangent is not None:
                raise NotImplementedError(f"{name} has no forward-mode "
                                          "derivative")


def _span(t: torch.Tensor) -> Tuple[int, int]:
    """First byte and end; of a tensor with gaps its first value alone."""
    n = 1 + sum((size - 1) * stride
                for size, stride in zip(t.shape, t.stride()))
    return (t.data_ptr(), t.data_ptr()
            + (n if n == t.numel() else 1) * t.element_size())


def _check_outputs(name: str, tensors: Sequence[torch.Tensor],
                   out: Sequence[torch.Tensor]) -> None:
    """Each output is written by workgroups of its own, while others read:
    none may be there twice, or lie in another's input."""
    written = sorted(_span(t) for t in out if t.numel())
    for (_, end), (begin, _) in zip(written, written[1:]):
        if begin < end:
            raise ValueError(f"{name}: the same memory is to be written "
                             "twice")
    for t, o in zip(tensors, out):
        if not t.numel() or (t.data_ptr() == o.data_ptr()
                             and t.dtype == o.dtype
                             and t.stride() == o.stride()):
            continue
        begin, end = _span(t)
        at = bisect.bisect_left(written, (end, 0))
        if at and written[at - 1][1] > begin:
            raise ValueError(f"{name}: an output shares memory with another "
                             "input")


def _kind(name: str, norm_type: float) -> int:
    try:
        return _KINDS[float(norm_type)]
    except KeyError:
        raise ValueError(f"{name}: norm_type must be 1, 2 or inf, got "
                         f"{norm_type}") from None


def _cpu_norm(tensors, norm_type: float) -> torch.Tensor:
    parts = [torch.linalg.vector_norm(t.detach().double(), norm_type)
             for t in tensors if t.numel()]
    if not parts:
        return torch.zeros(())
    return torch.linalg.vector_norm(torch.stack(parts), norm_type).float()


@torch.no_grad()
def global_norm(tensors: Tensors, norm_type: float = 2.0) -> torch.Tensor:
    """``(sum |t|^p)^(1/p)`` over all values of all tensors; p = 1, 2 or inf.

    fp32, a scalar on the tensors' device (0 on the CPU for no tensors).
    Sums are in double, so no square overflows or vanishes.
    """
    tensors = _as_list(tensors)
    kind = _kind("global_norm", norm_type)
    if not tensors:
        return torch.zeros(())
    if tensors[0].is_cuda:
        from kfac_pytorch_amd.ops import _ext
        return _ext.grad_norm(tensors, None, math.inf, kind)[0]
    _check_lists("global_norm", tensors)
    return _cpu_norm(tensors, float(norm_type))


@torch.no_grad()
def clip_by_global_norm(
        tensors: Tensors, max_norm: float, norm_type: float = 2.0,
        out: Optional[Sequence[torch.Tensor]] = None,
) -> Tuple[List[torch.Tensor], torch.Tensor]:
    """The tensors times ``min(1, max_norm / (norm + 1e-6))``, and the norm.

    ``out``: tensors to write, of the same shapes (any of the types); the
    inputs themselves clip in place, and are then left untouched where the
    factor is 1.  Otherwise an output must not share memory with an input or
    another output.  New tensors by default.  A norm that is not finite gives
    what the expression gives (0 or NaN times the values).
    """
    tensors = _as_list(tensors)
    kind = _kind("clip_by_global_norm", norm_type)
    max_norm = float(max_norm)
    if not max_norm >= 0:
        raise ValueError(f"clip_by_global_norm: max_norm must not be "
                         f"negative, got {max_norm}")
    out = [torch.empty_like(t) for t in tensors] if out is None \
        else _as_list(out)
    if not tensors:
        if out:
            raise ValueError("clip_by_global_norm: out without tensors")
        return out, torch.zeros(())
    if tensors[0].is_cuda:
        from kfac_pytorch_amd.ops import _ext
        return out, _ext.grad_norm(tensors, out, max_norm, kind)[0]
    _check_lists("clip_by_global_norm", tensors, out)
    _check_outputs("clip_by_global_norm", tensors, out)
    norm = _cpu_norm(tensors, float(norm_type))
    factor = (max_norm / (norm.double() + 1e-6)).clamp(max=1.0).float()
    for t, o in zip(tensors, out):
        o.copy_(t * factor.to(t.dtype) if t.dtype == torch.float64
                else t.float() * factor)
    return out, norm


def clip_grad_norm_(parameters: Tensors, max_norm: float,
                    norm_type: float = 2.0,
                    error_if_nonfinite: bool = False) -> torch.Tensor:
    """Clip the gradients of ``parameters`` in place; returns their norm.

    ``torch.nn.utils.clip_grad_norm_`` for one device, with an fp32 norm and
    without a wait for the device (``error_if_nonfinite`` does wait, and
    raises before anything is written).
    """
    # a parameter given twice counts once
    grads = list({id(p): p.grad for p in _as_list(parameters)
                  if p.grad is not None}.values())
    if error_if_nonfinite:
        norm = global_norm(grads, norm_type)
        if not math.isfinite(float(norm)):
            raise RuntimeError(f"clip_grad_norm_: the gradients' norm is "
                               f"{float(norm)}")
    return clip_by_global_norm([g.detach() for g in grads], max_norm,
                               norm_type, out=[g.detach() for g in grads])[1]


@torch.no_grad()
def kl_clip(updates: Sequence[torch.Tensor], grads: Sequence[torch.Tensor], *,
            lr: float, kl_clip: float,
            out: Optional[Sequence[torch.Tensor]] = None,
            ) -> Tuple[List[torch.Tensor], torch.Tensor]:
    """The updates times ``nu = min(1, sqrt(kl_clip / |lr^2 <u, g>|))``.

    ``<u, g>`` is the inner product over all tensors, summed in double.
    ``out``: tensors to write, of the same shapes (any of the types), which
    may be the updates or the gradients themselves, but not share memory with
    another's update.  New tensors like the gradients by default.  Returns them and nu (fp32, on the device).
    """
    updates, grads = _as_list(updates), _as_list(grads)
    lr, kl = float(lr), float(kl_clip)
    if not kl > 0:
        raise ValueError(f"kl_clip: kl_clip must be positive, got {kl}")
    if out is None:
        out = [torch.empty_like(g) for g in grads]
    out = _as_list(out)
    if not updates:
        if grads or out:
            raise ValueError("kl_clip: gradients without updates")
        return out, torch.ones(())
    if updates[0].is_cuda:
        from kfac_pytorch_amd.ops import _ext
        return out, _ext.trust_region(updates, grads, out, lr, kl)
    _check_lists("kl_clip", updates, grads, out)
    _check_outputs("kl_clip", updates, out)
    total = sum((u.double() * g.double()).sum()
                for u, g in zip(updates, grads)) * lr ** 2
    nu = (kl / total.abs().clamp_min(1e-30)).sqrt().clamp(max=1.0).float()
    for u, o in zip(updates, out):
        o.copy_(u * nu.to(u.dtype) if u.dtype == torch.float64
                else u.float() * nu)
    return out, nu
