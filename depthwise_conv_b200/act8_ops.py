"""8-bit activation checkpoints: the codec, and the weight gradient that reads them.

A training step keeps the input of every depthwise convolution for the weight
gradient (and the input of every norm, ``norm_ops``).  Kept as a checkpoint it
takes 1 + 1/32 bytes a value instead of 2: for every pixel and block of 32
channels one exponent byte E, and a signed code q of 8 bits a channel; the value
is ``q * 2^(E - 127)``.  The exponent is the smallest one with which 127 steps
reach the block's largest magnitude, so a value is off by at most half a step,
``amax / 127`` or less; what a checkpoint stands for is exact in the 16-bit type
it came from.  A block that holds an infinity or a NaN reads back as NaN.

``codes``: int8, the activation's shape, channels_last.  ``scales``: uint8
[B, H, W, ceil(C / 32)], contiguous.

Everything here checks its tensors and calls the C ABI on the current stream
(through the compiled module ``_train_bind``); there is no CPU or PyTorch fallback.  The reference's ops are inference-only
(convmixer/kernels/depthwise_torch_ops.py:157-159) and keep nothing.

Torch ops:

* ``depthwise::act8_encode(Tensor input) -> (Tensor codes, Tensor scales)``
* ``depthwise::act8_decode(Tensor codes, Tensor scales, ScalarType dtype) -> Tensor``
* ``depthwise::conv2d_nhwc_act8(Tensor input, Tensor weight, Tensor? bias=None,
  bool checkpoint=True) -> (Tensor output, Tensor codes, Tensor scales)``:
  ``depthwise::conv2d_nhwc`` whose backward pass takes the weight gradient from the
  checkpoint, so that the graph does not keep the input.  The input gradient does not
  read the input and is the same as the other op's.  Without a checkpoint codes and
  scales are empty and there is no weight gradient.
"""
from __future__ import annotations

import torch

from . import _lib, dw_ops

BLOCK = 32
DTYPE_CODES = {torch.float16: _lib.F16, torch.bfloat16: _lib.BF16}

_bind = None


def bind():
    """The compiled host side of the training ops (checks, allocation, the C ABI's call); loaded once."""
    global _bind
    if _bind is None:
        _lib.load()
        try:
            from . import _train_bind
        except ImportError as e:
            raise RuntimeError("depthwise_conv_b200: _train_bind.so is missing or does not load; build it with "
                               "`python -m depthwise_conv_b200.csrc.build` (there is no fallback)") from e
        _bind = _train_bind
    return _bind


def after_launch(t: torch.Tensor, where: str) -> None:
    """The opt-in check of the device error word behind a launch on the tensor's device."""
    if _lib.check_device_error_enabled():
        with dw_ops._DeviceGuard(t.device):
            _lib.after_launch(dw_ops._stream_of(t), where)


def incoming(grad: torch.Tensor) -> torch.Tensor:
    """A gradient from autograd as the kernels take it: channels_last, on a 16-byte boundary."""
    g = grad.contiguous(memory_format=torch.channels_last)
    return g if g.data_ptr() % 16 == 0 else g.clone()


def first_order(name: str, *grads):
    """The gradients a backward pass returns; differentiating them again raises instead of leaving terms out."""
    if torch.is_grad_enabled():  # under create_graph=True
        refuse = torch._C._functions.DelayedError(f"{name}: the backward pass is not differentiable", 1)
        grads = tuple(g if g is None else refuse(g.requires_grad_()) for g in grads)
    return grads


def act8_encode(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """(codes, scales) of a channels_last float16 or bfloat16 activation."""
    kept = bind().act8_encode(x)
    after_launch(x, "depthwise act8_encode")
    return kept


def act8_decode(codes: torch.Tensor, scales: torch.Tensor, dtype: torch.dtype = torch.float16) -> torch.Tensor:
    """The activation a checkpoint stands for, channels_last; ``dtype``: the type it was made from."""
    if dtype not in DTYPE_CODES:
        raise RuntimeError(f"dtype must be float16 or bfloat16, got {dtype}")
    x = bind().act8_decode(codes, scales, DTYPE_CODES[dtype])
    after_launch(x, "depthwise act8_decode")
    return x


def conv2d_nhwc_backward_weight_act8(codes: torch.Tensor, scales: torch.Tensor, dy: torch.Tensor, K: int) -> torch.Tensor:
    """dw of y = conv(x, w) as [K, K, C] float32 from the checkpoint of x (a float16 activation).

    The sums have a fixed order: the same bits on every call.  An infinity or a NaN
    in ``dy`` or the checkpoint may spread to every tap of its channel."""
    dw = bind().backward_weight_act8(codes, scales, dy, int(K))
    after_launch(dw, "depthwise conv2d_nhwc weight gradient from a checkpoint")
    return dw


def empty_checkpoint(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """Unwritten codes and scales for an activation like ``x`` (the fake impls' outputs)."""
    B, C, H, W = x.shape
    return torch.empty_like(x, dtype=torch.int8), x.new_empty((B, H, W, -(-C // BLOCK)), dtype=torch.uint8)


def no_checkpoint(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """The empty codes and scales of an op that was not asked for a checkpoint."""
    return x.new_empty((0,), dtype=torch.int8), x.new_empty((0,), dtype=torch.uint8)


def will_differentiate(*tensors) -> bool:
    """Whether the graph will hold a call with these inputs (some of them None)."""
    return torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors)


def conv2d_nhwc_act8(x: torch.Tensor, w: torch.Tensor, bias=None) -> torch.Tensor:
    """y = conv(x, w) (+ bias), differentiable; keeps the 8-bit checkpoint of x for the weight gradient.

    Where no weight gradient will be taken (grad mode off, a weight that requires none) no checkpoint is made."""
    return torch.ops.depthwise.conv2d_nhwc_act8(x, w, bias, will_differentiate(w))[0]


torch.library.define("depthwise::act8_encode", "(Tensor input) -> (Tensor codes, Tensor scales)")
torch.library.define("depthwise::act8_decode", "(Tensor codes, Tensor scales, ScalarType dtype) -> Tensor")
torch.library.define("depthwise::conv2d_nhwc_act8",
                     "(Tensor input, Tensor weight, Tensor? bias=None, bool checkpoint=True) -> "
                     "(Tensor output, Tensor codes, Tensor scales)")


@torch.library.impl("depthwise::act8_encode", "default")
def _act8_encode_impl(input):
    return act8_encode(input)


@torch.library.register_fake("depthwise::act8_encode")
def _act8_encode_fake(input):
    return empty_checkpoint(input)


@torch.library.impl("depthwise::act8_decode", "default")
def _act8_decode_impl(codes, scales, dtype):
    return act8_decode(codes, scales, dtype)


@torch.library.register_fake("depthwise::act8_decode")
def _act8_decode_fake(codes, scales, dtype):
    return torch.empty_like(codes, dtype=dtype)


@torch.library.impl("depthwise::conv2d_nhwc_act8", "default")
def _conv2d_nhwc_act8_impl(input, weight, bias=None, checkpoint=True):
    y = dw_ops.conv2d_nhwc_fused(input, weight, bias=bias)
    return y, *(act8_encode(input) if checkpoint else no_checkpoint(input))


@torch.library.register_fake("depthwise::conv2d_nhwc_act8")
def _conv2d_nhwc_act8_fake(input, weight, bias=None, checkpoint=True):
    return torch.empty_like(input), *(empty_checkpoint(input) if checkpoint else no_checkpoint(input))


def _conv2d_nhwc_act8_setup(ctx, inputs, output):
    _, w, bias, checkpoint = inputs
    _, codes, scales = output
    ctx.save_for_backward(w, codes, scales)
    ctx.has_bias, ctx.checkpoint = bias is not None, checkpoint
    ctx.mark_non_differentiable(codes, scales)
    ctx.set_materialize_grads(False)


def _conv2d_nhwc_act8_backward(ctx, grad, _codes, _scales):
    if grad is None:
        return None, None, None, None
    w, codes, scales = ctx.saved_tensors
    if ctx.needs_input_grad[1] and not ctx.checkpoint:
        raise RuntimeError("conv2d_nhwc_act8: the weight gradient needs a checkpoint of the input (checkpoint=True)")
    g = incoming(grad)
    dx = dw_ops.conv2d_nhwc_backward_input(g, w) if ctx.needs_input_grad[0] else None
    dw = conv2d_nhwc_backward_weight_act8(codes, scales, g, w.shape[0]).to(w.dtype) if ctx.needs_input_grad[1] else None
    db = g.float().sum(dim=(0, 2, 3)).to(g.dtype).detach() if ctx.has_bias and ctx.needs_input_grad[2] else None
    return *first_order("conv2d_nhwc_act8", dx, dw, db), None


torch.library.register_autograd("depthwise::conv2d_nhwc_act8", _conv2d_nhwc_act8_backward,
                                setup_context=_conv2d_nhwc_act8_setup)
