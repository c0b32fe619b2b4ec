"""Group normalisation with its activation on channels_last tensors, forward and backward.

``y = act((x - mean) * rstd * weight + bias)`` with the mean and the (biased)
variance of each group of C / G channels over the pixels of each sample: the
normalisation of a network that trains with few images a GPU, in one pass over
the activation.  float16 and bfloat16; ``weight`` and ``bias`` in the tensor's
type or float32; statistics and sums in float32, in a fixed order.
``act``: "none", "relu", "gelu" (exact erf form) or "silu".

With ``checkpoint=True`` the forward pass also writes the 8-bit checkpoint of its
input (``act8_ops``), from which the backward pass then works, so that the graph
keeps 1 + 1/32 bytes a value instead of 2.  The statistics are those of the
input itself in both cases.

Everything here checks its tensors and calls the C ABI on the current stream
(through the compiled module ``_train_bind``); there is no CPU or PyTorch fallback.  The reference's networks normalise with an
inference BatchNorm (convmixer/convmixer.py:93-127) and have no counterpart.

Torch op (differentiable in input, weight and bias):
``depthwise::group_norm_act(Tensor input, int num_groups, Tensor? weight, Tensor? bias, float eps, int act,
bool checkpoint) -> (Tensor output, Tensor mean, Tensor rstd, Tensor codes, Tensor scales)``; mean and rstd are
float32 [B, G]; without a checkpoint codes and scales are empty.
"""
from __future__ import annotations

import torch

from . import _lib
from .act8_ops import after_launch, bind, empty_checkpoint, first_order, incoming, no_checkpoint, will_differentiate

ACT_CODES = _lib.NORM_ACT_CODES


def _act_code(act) -> int:
    if isinstance(act, str):
        if act not in ACT_CODES:
            raise RuntimeError(f"act must be one of {sorted(ACT_CODES)}, got {act!r}")
        return ACT_CODES[act]
    return int(act)


def group_norm_act_forward(x: torch.Tensor, num_groups: int, weight=None, bias=None, eps: float = 1e-5,
                           act: int | str = 0, checkpoint: bool = False):
    """(y, mean, rstd), with ``checkpoint`` (y, mean, rstd, codes, scales).

    x: channels_last [B, C, H, W], float16 or bfloat16, C % 8 == 0; y like x; mean, rstd: float32 [B, num_groups]."""
    out = bind().group_norm_act_forward(x, num_groups, weight, bias, eps, _act_code(act), checkpoint)
    after_launch(x, "depthwise group_norm_act")
    return out


def group_norm_act_backward(dy: torch.Tensor, saved, mean: torch.Tensor, rstd: torch.Tensor, num_groups: int,
                            weight=None, bias=None, act: int | str = 0):
    """(dx, dweight, dbias) of the forward pass; dweight, dbias in the parameters' type, None where there is none.

    ``saved``: the forward pass's input, or the (codes, scales) of its checkpoint."""
    x, codes, scales = (saved, None, None) if isinstance(saved, torch.Tensor) else (None, *saved)
    out = bind().group_norm_act_backward(dy, x, codes, scales, mean, rstd, num_groups, weight, bias, _act_code(act))
    after_launch(dy, "depthwise group_norm_act gradient")
    return out


def group_norm_act(x: torch.Tensor, num_groups: int, weight=None, bias=None, eps: float = 1e-5, act: int | str = 0,
                   checkpoint: bool = False) -> torch.Tensor:
    """act(group_norm(x)), differentiable; ``checkpoint``: keep the input for the backward pass in 8 bits.

    Where there will be no backward pass no checkpoint is made; the result is the same bits."""
    return torch.ops.depthwise.group_norm_act(x, int(num_groups), weight, bias, float(eps), _act_code(act),
                                              bool(checkpoint) and will_differentiate(x, weight, bias))[0]


torch.library.define(
    "depthwise::group_norm_act",
    "(Tensor input, int num_groups, Tensor? weight, Tensor? bias, float eps, int act, bool checkpoint) -> "
    "(Tensor output, Tensor mean, Tensor rstd, Tensor codes, Tensor scales)",
)


@torch.library.impl("depthwise::group_norm_act", "default")
def _group_norm_act_impl(input, num_groups, weight, bias, eps, act, checkpoint):
    out = group_norm_act_forward(input, num_groups, weight, bias, eps, act, checkpoint)
    return out if checkpoint else (*out, *no_checkpoint(input))


@torch.library.register_fake("depthwise::group_norm_act")
def _group_norm_act_fake(input, num_groups, weight, bias, eps, act, checkpoint):
    mean = input.new_empty((input.shape[0], num_groups), dtype=torch.float32)
    kept = empty_checkpoint(input) if checkpoint else no_checkpoint(input)
    return torch.empty_like(input), mean, torch.empty_like(mean), *kept


def _group_norm_act_setup(ctx, inputs, output):
    x, num_groups, weight, bias, _, act, checkpoint = inputs
    _, mean, rstd, codes, scales = output
    ctx.save_for_backward(None if checkpoint else x, weight, bias, mean, rstd, codes, scales)
    ctx.num_groups, ctx.act, ctx.checkpoint = num_groups, act, checkpoint
    ctx.mark_non_differentiable(mean, rstd, codes, scales)
    ctx.set_materialize_grads(False)


def _group_norm_act_backward(ctx, grad, *_):
    if grad is None:
        return (None,) * 7
    x, weight, bias, mean, rstd, codes, scales = ctx.saved_tensors
    dx, dweight, dbias = group_norm_act_backward(incoming(grad), (codes, scales) if ctx.checkpoint else x, mean, rstd,
                                                 ctx.num_groups, weight, bias, ctx.act)
    need = ctx.needs_input_grad
    dx, dweight, dbias = first_order("group_norm_act", dx if need[0] else None, dweight if need[2] else None,
                                     dbias if need[3] else None)
    return dx, None, dweight, dbias, None, None, None


torch.library.register_autograd("depthwise::group_norm_act", _group_norm_act_backward,
                                setup_context=_group_norm_act_setup)
