"""Cross entropy of a vocabulary projection, without the logits in memory.

``linear_cross_entropy(hidden, weight, target, bias)`` is
``F.cross_entropy(F.linear(hidden, weight, bias), target)``: the output layer
and the loss of a language model in one operator.  K-FAC leaves that layer out
(``exclude_vocabulary_size``), so nothing needs its input and output as
tensors of their own.

    z[n, v] = sum_d hidden[n, d] weight[v, d] + bias[v]
    loss[n] = log sum_v exp z[n, v] - (1 - eps) z[n, target[n]]
              - eps / V sum_v z[n, v]

On the GPU, hand-written MFMA kernels (``csrc/vocab_loss.hip``) make the logits
tile by tile in registers.  Where gradients are asked for, the forward pass of
a reduced loss computes them in the same go; otherwise the backward pass makes
the logits once more, piece by piece of the vocabulary.  Products are of the
inputs' type, sums, losses and the log-sum-exp fp32.  On the CPU the plain
expression above runs.
"""

from __future__ import annotations

from typing import Optional

import torch
import torch.nn.functional as F
from torch.nn.modules import module

__all__ = ["linear_cross_entropy", "projection_loss"]

_REDUCTIONS = {"none": 0, "mean": 1, "sum": 2}


def _check(hidden, weight, target, bias, label_smoothing):
    if not 0.0 <= label_smoothing <= 1.0:
        raise ValueError("linear_cross_entropy: label_smoothing must be in "
                         f"[0, 1], got {label_smoothing}")
    if hidden.dim() < 1 or weight.dim() != 2 \
            or hidden.size(-1) != weight.size(1):
        raise ValueError("linear_cross_entropy: hidden (..., d) and weight "
                         f"(V, d) expected, got {tuple(hidden.shape)} and "
                         f"{tuple(weight.shape)}")
    if target.shape != hidden.shape[:-1]:
        raise ValueError("linear_cross_entropy: target must have the shape "
                         f"{tuple(hidden.shape[:-1])}, got "
                         f"{tuple(target.shape)}")
    if bias is not None and bias.shape != weight.shape[:1]:
        raise ValueError("linear_cross_entropy: bias must have the shape "
                         f"{tuple(weight.shape[:1])}, got "
                         f"{tuple(bias.shape)}")
    if target.dtype not in (torch.int64, torch.int32):
        raise TypeError("linear_cross_entropy: target must be int64 or "
                        f"int32, got {target.dtype}")
    if weight.size(0) == 0 or weight.size(1) == 0:
        raise ValueError("linear_cross_entropy: weight is empty")
    for name, t in (("weight", weight), ("target", target), ("bias", bias)):
        if t is not None and t.device != hidden.device:
            raise ValueError(f"linear_cross_entropy: {name} is on "
                             f"{t.device}, hidden on {hidden.device}")


def linear_cross_entropy(hidden: torch.Tensor, weight: torch.Tensor,
                         target: torch.Tensor,
                         bias: Optional[torch.Tensor] = None, *,
                         ignore_index: int = -100,
                         label_smoothing: float = 0.0,
                         reduction: str = "mean") -> torch.Tensor:
    """Cross entropy of ``F.linear(hidden, weight, bias)`` against ``target``.

    Args:
      hidden: (..., d), bf16, fp16 or fp32, any strides.
      weight: (V, d), the type of ``hidden``.
      target: (...), int64 or int32; rows with ``ignore_index`` count for
        nothing, whatever their hidden states hold, and get zero gradients.
      bias: (V,), or None.
      label_smoothing: as in ``F.cross_entropy``: the target keeps
        ``1 - eps``, and ``eps`` is spread over the whole vocabulary.
      reduction: ``"mean"`` over the rows that count (NaN if none does, with
        zero gradients), ``"sum"``, or ``"none"`` (ignored rows are 0).

    Returns fp32 (a scalar, or one loss for each row).  Under autocast the
    floating arguments are cast as ``F.linear`` casts them.  A target outside
    the vocabulary raises on the CPU; on the GPU, where raising would mean to
    wait for the device, that row's loss and the gradients become NaN.
    On the GPU there is no double backward and no forward-mode derivative;
    both raise.

    On the GPU a reduced loss computes its gradients in the forward pass if
    any is asked for (evaluate under ``torch.no_grad()``), and scales them
    by the upstream factor in the first backward pass.  A bf16 gradient of
    the weight may be rounded twice then, to bf16 before and after a factor
    that is no power of two.

    Memory on the GPU.  While a call lasts: a packed copy of ``hidden``, one
    of ``weight`` unless its rows are whole 16-byte chunks, 8 or 12 bytes
    for each row and 32 to 128 entries of the vocabulary, and, for gradients
    of a reduced loss, rows x V values of the inputs' type if that is 4 GiB
    at most.  From there to the first backward pass, which allocates the
    gradients beside it: the weight's gradient, in fp32 for fp16; the fp32
    partial sums of the hidden states' gradient, one to 64 times rows x d (4
    at most where that is over 70 MB); of the bias's, V for each 4 to 64 rows;
    and, where the weight's gradient has too few tiles for the GPU, up to 16
    of its partial sums instead (some 60 MB at most).  Beyond 4 GiB, for
    ``"none"`` and for a second backward pass nothing is kept: the backward
    pass makes the logits again, 256 MB of them at a time (64 to 256 entries
    of the vocabulary at least).
    """
    if reduction not in _REDUCTIONS:
        raise ValueError(f"linear_cross_entropy: reduction must be one of "
                         f"{tuple(_REDUCTIONS)}, got {reduction!r}")
    if hidden.is_cuda and target.numel():
        # the same checks, autocast and autograd are behind this call: a
        # step's last operator is short enough for Python to be seen
        from kfac_pytorch_amd.ops import _ext
        return _ext.linear_cross_entropy(hidden, weight, target, bias,
                                         ignore_index, label_smoothing,
                                         _REDUCTIONS[reduction])

    _check(hidden, weight, target, bias, label_smoothing)
    kind = hidden.device.type
    if torch.is_autocast_enabled(kind):
        t = torch.get_autocast_dtype(kind)
        # autocast leaves float64 alone
        cast = (lambda a: a if a is None or a.dtype == torch.float64
                else a.to(t))
        hidden, weight, bias = cast(hidden), cast(weight), cast(bias)
    if hidden.dtype != weight.dtype or (
            bias is not None and bias.dtype != weight.dtype):
        raise TypeError("linear_cross_entropy: hidden, weight and bias must "
                        f"have one dtype, got {hidden.dtype}, {weight.dtype}"
                        + (f", {bias.dtype}" if bias is not None else ""))
    # what an ignored row holds must not meet its gradients' zeros
    hidden = hidden.masked_fill((target == ignore_index).unsqueeze(-1), 0.0)
    wide = (lambda a: a if a is None or a.dtype == torch.float64
            else a.float())
    with torch.autocast(kind, enabled=False):
        z = F.linear(wide(hidden), wide(weight), wide(bias))
        loss = F.cross_entropy(
            z.reshape(-1, z.size(-1)), target.reshape(-1).long(),
            ignore_index=ignore_index, label_smoothing=label_smoothing,
            reduction=reduction)
    return loss.view(target.shape) if reduction == "none" else loss


def projection_loss(layer: torch.nn.Linear, hidden: torch.Tensor,
                    target: torch.Tensor, **kw) -> torch.Tensor:
    """``linear_cross_entropy`` with an output layer's weight and bias.

    The layer itself is not called, so nothing that hangs on its calls may
    be left waiting, and the call may be nothing else than ``F.linear``: a
    layer with hooks (K-FAC's, of a preconditioner that does not leave the
    vocabulary projection out; hooks on all modules too) or with a forward
    pass of its own (an adapter, a scaled or quantised head) is refused.
    """
    plain = getattr(layer, "_orig_mod", layer)  # of torch.compile(layer)
    if any(getattr(m, name) for m in {layer, plain}
           for name in ("_forward_pre_hooks", "_forward_hooks",
                        "_backward_hooks", "_backward_pre_hooks")) or any(
            getattr(module, "_global" + name, None)
            for name in ("_forward_pre_hooks", "_forward_hooks",
                         "_backward_hooks", "_backward_pre_hooks")):
        raise RuntimeError(
            "the vocabulary projection carries hooks, which a loss without "
            "logits does not run; leave the layer out of K-FAC "
            f"(exclude_vocabulary_size={plain.weight.size(0)}) or take the "
            "loss from the logits")
    if (getattr(type(plain), "forward", None) is not torch.nn.Linear.forward
            or type(plain).__call__ is not torch.nn.Module.__call__
            or "forward" in vars(plain)):
        raise RuntimeError(
            f"the vocabulary projection, a {type(plain).__name__}, has a "
            "forward pass of its own, which a loss without logits does not "
            "run; take the loss from the logits")
    return linear_cross_entropy(hidden, plain.weight, target,
                                bias=plain.bias, **kw)
