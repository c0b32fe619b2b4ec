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

Everything here validates tensors and calls the C ABI on the current stream;
there is no CPU or PyTorch fallback.  The reference's networks normalise with an
inference BatchNorm (convmixer/convmixer.py:93-127) and have no counterpart.

Torch op (differentiable in input, weight and bias):
``depthwise::group_norm_act(Tensor input, int num_groups, Tensor? weight, Tensor? bias, float eps, int act,
bool checkpoint) -> (Tensor output, Tensor mean, Tensor rstd, Tensor codes, Tensor scales)``; mean and rstd are
float32 [B, G]; without a checkpoint codes and scales are empty.
"""
from __future__ import annotations

import ctypes
import functools

import torch

from . import _lib
from .act8_ops import check_checkpoint, check_nhwc, empty_checkpoint, launch

ACT_CODES = _lib.NORM_ACT_CODES


def _act_code(act) -> int:
    if isinstance(act, str):
        if act not in ACT_CODES:
            raise RuntimeError(f"act must be one of {sorted(ACT_CODES)}, got {act!r}")
        return ACT_CODES[act]
    return int(act)


def _check_param(name: str, t, like: torch.Tensor) -> None:
    if not t.is_cuda or t.dtype not in (like.dtype, torch.float32) or t.shape != like.shape[1:2] or not t.is_contiguous():
        raise RuntimeError(f"{name} must be a contiguous {like.dtype} or float32 CUDA tensor with {like.shape[1]} elements, "
                           f"got {t.dtype} {tuple(t.shape)}")
    if t.device != like.device:
        raise RuntimeError(f"{name} is on {t.device}, input on {like.device}")


def _check_params(weight, bias, like: torch.Tensor, dtype_code: int):
    """Pointers of the parameter vectors and their dwb_dtype."""
    wp = bp = None
    if weight is not None:
        _check_param("weight", weight, like)
        wp = weight.data_ptr()
    if bias is not None:
        _check_param("bias", bias, like)
        bp = bias.data_ptr()
        if weight is not None and weight.dtype != bias.dtype:
            raise RuntimeError(f"weight and bias must have one type, got {weight.dtype} and {bias.dtype}")
    first = bias if weight is None else weight
    return wp, bp, _lib.F32 if first is not None and first.dtype == torch.float32 else dtype_code


@functools.lru_cache(maxsize=1024)
def _workspace_bytes(B: int, H: int, W: int, C: int, G: int, backward: int) -> int:
    n = ctypes.c_int64(0)
    _lib.call("dwb_group_norm_act_workspace", B, H, W, C, G, backward, ctypes.byref(n))
    return n.value


def _workspace(x: torch.Tensor, B: int, H: int, W: int, C: int, G: int, backward: int):
    n = _workspace_bytes(B, H, W, C, G, backward)
    return (x.new_empty((n,), dtype=torch.uint8) if n else None), n


def group_norm_act_forward(x: torch.Tensor, num_groups: int, weight=None, bias=None, eps: float = 1e-5,
                           act: int | str = 0, checkpoint: bool = False):
    """(y, mean, rstd), with ``checkpoint`` (y, mean, rstd, codes, scales).

    x: channels_last [B, C, H, W], float16 or bfloat16, C % 8 == 0; y like x; mean, rstd: float32 [B, num_groups]."""
    dtype = check_nhwc(x)
    B, C, H, W = x.shape
    G, act_code = int(num_groups), _act_code(act)
    wp, bp, param_dtype = _check_params(weight, bias, x, dtype)
    ws, nbytes = _workspace(x, B, H, W, C, G, 0)
    y = torch.empty_like(x)  # keeps the strides
    mean = x.new_empty((B, G), dtype=torch.float32)
    rstd = torch.empty_like(mean)
    codes, scales = empty_checkpoint(x) if checkpoint else (None, None)
    launch("dwb_group_norm_act_nhwc_fwd", "depthwise group_norm_act", x.device, x.data_ptr(), wp, bp, y.data_ptr(),
           mean.data_ptr(), rstd.data_ptr(), codes.data_ptr() if checkpoint else None,
           scales.data_ptr() if checkpoint else None, ws.data_ptr() if nbytes else None, nbytes, B, H, W, C, G, float(eps),
           act_code, dtype, param_dtype)
    return (y, mean, rstd, codes, scales) if checkpoint else (y, mean, rstd)


def group_norm_act_backward(dy: torch.Tensor, saved, mean: torch.Tensor, rstd: torch.Tensor, num_groups: int,
                            weight=None, bias=None, act: int | str = 0):
    """(dx, dweight, dbias) of the forward pass; dweight, dbias in the parameters' type, None where there is none.

    ``saved``: the forward pass's input, or the (codes, scales) of its checkpoint."""
    dtype = check_nhwc(dy, "grad_output")
    B, C, H, W = dy.shape
    G, act_code = int(num_groups), _act_code(act)
    if isinstance(saved, torch.Tensor):
        check_nhwc(saved, "saved input")
        if saved.dtype != dy.dtype:
            raise RuntimeError(f"saved input is {saved.dtype}, grad_output {dy.dtype}")
        first, xp, qp, sp = saved, saved.data_ptr(), None, None
    else:
        codes, scales = saved
        check_checkpoint(codes, scales)
        first, xp, qp, sp = codes, None, codes.data_ptr(), scales.data_ptr()
    if first.shape != dy.shape or first.device != dy.device:
        raise RuntimeError("what was saved must match grad_output in shape and device")
    wp, bp, param_dtype = _check_params(weight, bias, dy, dtype)
    for name, t in (("mean", mean), ("rstd", rstd)):
        if t.dtype != torch.float32 or t.shape != (B, G) or not t.is_contiguous() or t.device != dy.device:
            raise RuntimeError(f"{name} must be a contiguous float32 tensor [{B}, {G}] on {dy.device}")
    ws, nbytes = _workspace(dy, B, H, W, C, G, 1)
    dx = torch.empty_like(dy)
    dweight = torch.empty_like(weight) if weight is not None else None
    dbias = torch.empty_like(bias) if bias is not None else None
    launch("dwb_group_norm_act_nhwc_bwd", "depthwise group_norm_act gradient", dy.device, dy.data_ptr(), xp, qp, sp,
           mean.data_ptr(), rstd.data_ptr(), wp, bp, dx.data_ptr(), dweight.data_ptr() if dweight is not None else None,
           dbias.data_ptr() if dbias is not None else None, ws.data_ptr() if nbytes else None, nbytes, B, H, W, C, G,
           act_code, dtype, param_dtype)
    return dx, dweight, dbias


def group_norm_act(x: torch.Tensor, num_groups: int, weight=None, bias=None, eps: float = 1e-5, act: int | str = 0,
                   checkpoint: bool = False) -> torch.Tensor:
    """act(group_norm(x)), differentiable; ``checkpoint``: keep the input for the backward pass in 8 bits."""
    return torch.ops.depthwise.group_norm_act(x, int(num_groups), weight, bias, float(eps), _act_code(act),
                                              bool(checkpoint))[0]


torch.library.define(
    "depthwise::group_norm_act",
    "(Tensor input, int num_groups, Tensor? weight, Tensor? bias, float eps, int act, bool checkpoint) -> "
    "(Tensor output, Tensor mean, Tensor rstd, Tensor codes, Tensor scales)",
)


def _no_checkpoint(x):
    return x.new_empty((0,), dtype=torch.int8), x.new_empty((0,), dtype=torch.uint8)


@torch.library.impl("depthwise::group_norm_act", "default")
def _group_norm_act_impl(input, num_groups, weight, bias, eps, act, checkpoint):
    out = group_norm_act_forward(input, num_groups, weight, bias, eps, act, checkpoint)
    return out if checkpoint else (*out, *_no_checkpoint(input))


@torch.library.register_fake("depthwise::group_norm_act")
def _group_norm_act_fake(input, num_groups, weight, bias, eps, act, checkpoint):
    mean = input.new_empty((input.shape[0], num_groups), dtype=torch.float32)
    kept = empty_checkpoint(input) if checkpoint else _no_checkpoint(input)
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
    g = grad if grad.is_contiguous(memory_format=torch.channels_last) else grad.contiguous(
        memory_format=torch.channels_last)
    dx, dweight, dbias = group_norm_act_backward(g, (codes, scales) if ctx.checkpoint else x, mean, rstd, ctx.num_groups,
                                                 weight, bias, ctx.act)
    need = ctx.needs_input_grad
    return (dx if need[0] else None, None, dweight if need[2] else None, dbias if need[3] else None, None, None, None)


torch.library.register_autograd("depthwise::group_norm_act", _group_norm_act_backward,
                                setup_context=_group_norm_act_setup)
