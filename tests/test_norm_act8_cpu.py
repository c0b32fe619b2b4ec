"""Group norm with an activation and the 8-bit checkpoints without a GPU: the float64 oracle against
PyTorch, the entry points' refusals, the fake impls, and workspace sizes."""
from __future__ import annotations

import ctypes
import importlib.metadata
import importlib.util

import pytest
import torch
import torch.nn.functional as F

from oracle import train_ref as R


@pytest.fixture(scope="module")
def L():
    from depthwise_conv_b200 import _lib
    _lib.load()
    return _lib


@pytest.mark.parametrize("act", ["none", "relu", "gelu", "silu"])
@pytest.mark.parametrize("B,H,W,C,G", [(2, 5, 3, 24, 8), (1, 1, 4, 16, 16), (3, 4, 4, 8, 1)])
def test_oracle_matches_torch_autograd(act, B, H, W, C, G):
    g = torch.Generator().manual_seed(C + G)
    x = torch.randn(B, C, H, W, dtype=torch.float64, generator=g).requires_grad_()
    w = (1 + 0.3 * torch.randn(C, dtype=torch.float64, generator=g)).requires_grad_()
    b = (0.3 * torch.randn(C, dtype=torch.float64, generator=g)).requires_grad_()
    dy = torch.randn(B, C, H, W, dtype=torch.float64, generator=g)
    fn = {"none": lambda t: t, "relu": F.relu, "gelu": F.gelu, "silu": F.silu}[act]
    y = fn(F.group_norm(x, G, w, b, 1e-5))
    y.backward(dy)
    yr, mean, rstd, _ = R.group_norm_act(x.detach(), G, w.detach(), b.detach(), 1e-5, act)
    got = R.group_norm_act_grad(dy, x.detach(), mean, rstd, G, w.detach(), b.detach(), act)
    torch.testing.assert_close(yr, y.detach(), rtol=1e-11, atol=1e-11)
    torch.testing.assert_close(got["dx"], x.grad, rtol=1e-9, atol=1e-10)
    torch.testing.assert_close(got["dweight"], w.grad, rtol=1e-10, atol=1e-10)
    torch.testing.assert_close(got["dbias"], b.grad, rtol=1e-10, atol=1e-10)


def test_oracle_gradient_against_differences():
    """dx of the whole chain by central differences of sum(y * dy) in float64."""
    g = torch.Generator().manual_seed(5)
    B, C, H, W, G, h = 1, 8, 2, 3, 2, 1e-6
    x = torch.randn(B, C, H, W, dtype=torch.float64, generator=g)
    dy = torch.randn(B, C, H, W, dtype=torch.float64, generator=g)
    mean, rstd = R.stats(x, G, 1e-5)
    dx = R.group_norm_act_grad(dy, x, mean, rstd, G, act="gelu")["dx"].reshape(-1)
    for i in range(x.numel()):
        lo, hi = x.clone().reshape(-1), x.clone().reshape(-1)
        lo[i] -= h
        hi[i] += h
        d = [(R.group_norm_act(t.view_as(x), G, act="gelu")[0] * dy).sum() for t in (lo, hi)]
        assert abs((d[1] - d[0]) / (2 * h) - dx[i]) < 1e-7


@pytest.mark.parametrize("dtype,tiny,huge", [(torch.float16, 2.0**-24, 65504.0), (torch.bfloat16, 2.0**-133, 3.3e38)])
def test_oracle_codec_error_bound(dtype, tiny, huge):
    """Every value is within half a step, the step at most 2 amax / 127 (or the type's finest code step);
    what the codes stand for is exact in the type; an infinity or a NaN takes its block along."""
    g = torch.Generator().manual_seed(1)
    x = (torch.randn(2, 72, 3, 5, generator=g) * torch.exp(4 * torch.randn(2, 1, 3, 5, generator=g))).to(dtype)
    x[0, :32, 0, 0] = 0
    x[0, 3, 0, 1] = tiny
    x[0, 32:64, 0, 1] = -huge
    x[1, 40, 2, 2] = float("inf")
    x[1, 70, 2, 3] = float("nan")
    codes, scales = R.act8_encode(x)
    v = R.act8_decode(codes, scales)
    assert torch.isnan(v[1, 32:64, 2, 2]).all() and torch.isfinite(v[1, :32, 2, 2]).all()
    assert torch.isnan(v[1, 64:, 2, 3]).all() and torch.isfinite(v[1, :64, 2, 3]).all()
    bad = torch.isnan(v)
    assert torch.equal(v.to(dtype).double()[~bad], v[~bad])
    low = 2.0 ** R.EXPONENTS[dtype][0]
    for at in range(0, 72, 32):
        d, part = (v - x.double())[:, at:at + 32], x.double()[:, at:at + 32]
        fine = ~bad[:, at:at + 32]
        limit = torch.maximum(part.abs().amax(dim=1, keepdim=True) / 127, torch.tensor(low / 2)).expand_as(d)
        assert (d.abs()[fine] <= limit[fine]).all()


def test_oracle_weight_gradient_matches_conv_backward():
    g = torch.Generator().manual_seed(2)
    x = torch.randn(2, 8, 5, 7, dtype=torch.float64, generator=g)
    w = torch.randn(8, 1, 5, 5, dtype=torch.float64, generator=g).requires_grad_()
    dy = torch.randn(2, 8, 5, 7, dtype=torch.float64, generator=g)
    F.conv2d(x, w, padding=2, groups=8).backward(dy)
    dw, _ = R.dw_weight_grad(x, dy, 5)
    torch.testing.assert_close(dw, w.grad[:, 0].permute(1, 2, 0), rtol=1e-11, atol=1e-11)


# Addresses that are never read: each call is refused before any CUDA call.
X, Y, Q, S, M, WS = (ctypes.c_void_p(256 * i) for i in range(1, 7))


def test_codec_refusals(L):
    for name in ("dwb_act8_encode_nhwc", "dwb_act8_decode_nhwc"):
        f = getattr(L.load(), name)
        a, b, c = (X, Q, S) if "encode" in name else (Q, S, X)
        assert f(a, b, c, 10, 64, 2, None) == L.ERR_BAD_ARG         # fp32
        assert f(a, b, c, 10, 60, 0, None) == L.ERR_BAD_SHAPE       # C % 8
        assert f(a, b, c, 10, 0, 0, None) == L.ERR_BAD_SHAPE
        assert f(a, b, c, -1, 64, 0, None) == L.ERR_BAD_SHAPE
        assert f(None, b, c, 10, 64, 0, None) == L.ERR_NULL_POINTER
        assert f(a, b, None, 10, 64, 0, None) == L.ERR_NULL_POINTER
        assert f(None, None, None, 0, 64, 0, None) == L.OK          # no pixel: nothing to do
        odd = ctypes.c_void_p(260)
        args = (odd, b, c) if "encode" in name else (a, b, odd)
        assert f(*args, 10, 64, 1, None) == L.ERR_BAD_ALIGN


def test_weight_gradient_refusals(L):
    f = L.load().dwb_conv2d_nhwc_bwd_weight_act8
    big = 1 << 40
    assert f(Q, S, X, Y, WS, big, 1, 8, 8, 64, 8, None) == L.ERR_BAD_SHAPE      # even K
    assert f(Q, S, X, Y, WS, big, 1, 8, 8, 64, 33, None) == L.ERR_BAD_SHAPE
    assert f(Q, S, X, Y, WS, big, 1, 8, 8, 12, 7, None) == L.ERR_BAD_SHAPE
    assert f(Q, S, X, Y, WS, big, 1, 0, 8, 64, 7, None) == L.ERR_BAD_SHAPE
    assert f(None, S, X, Y, WS, big, 1, 8, 8, 64, 7, None) == L.ERR_NULL_POINTER
    assert f(Q, S, X, None, WS, big, 1, 8, 8, 64, 7, None) == L.ERR_NULL_POINTER
    assert f(Q, S, X, Y, None, big, 1, 8, 8, 64, 7, None) == L.ERR_NULL_POINTER
    assert f(Q, S, ctypes.c_void_p(258), Y, WS, big, 1, 8, 8, 64, 7, None) == L.ERR_BAD_ALIGN
    n = ctypes.c_int64(-1)
    assert L.load().dwb_conv2d_nhwc_bwd_weight_act8_workspace(1, 8, 8, 64, 7, ctypes.byref(n)) == L.OK and n.value > 0
    assert f(Q, S, X, Y, WS, n.value - 1, 1, 8, 8, 64, 7, None) == L.ERR_BAD_ARG
    assert L.load().dwb_conv2d_nhwc_bwd_weight_act8_workspace(1, 8, 8, 64, 7, None) == L.ERR_NULL_POINTER
    assert L.load().dwb_conv2d_nhwc_bwd_weight_act8_workspace(1, 8, 8, 64, 6, ctypes.byref(n)) == L.ERR_BAD_SHAPE


def _fwd(L, x=X, w=None, b=None, y=Y, mean=M, rstd=M, q=None, s=None, ws=WS, nws=1 << 50, B=1, H=8, W=8, C=64, G=8,
         eps=1e-5, act=0, dtype=0, pdtype=0):
    return L.load().dwb_group_norm_act_nhwc_fwd(x, w, b, y, mean, rstd, q, s, ws, nws, B, H, W, C, G, eps, act, dtype,
                                                pdtype, None)


def _bwd(L, dy=X, x=X, q=None, s=None, mean=M, rstd=M, w=None, b=None, dx=Y, dw=None, db=None, ws=WS, nws=1 << 50, B=1,
         H=8, W=8, C=64, G=8, act=0, dtype=0, pdtype=0):
    return L.load().dwb_group_norm_act_nhwc_bwd(dy, x, q, s, mean, rstd, w, b, dx, dw, db, ws, nws, B, H, W, C, G, act,
                                                dtype, pdtype, None)


@pytest.mark.parametrize("call", [_fwd, _bwd])
def test_group_norm_refusals(L, call):
    for kw, code in [(dict(C=60), L.ERR_BAD_SHAPE), (dict(G=7), L.ERR_BAD_SHAPE), (dict(G=0), L.ERR_BAD_SHAPE),
                     (dict(G=128), L.ERR_BAD_SHAPE), (dict(H=0), L.ERR_BAD_SHAPE), (dict(B=-1), L.ERR_BAD_SHAPE),
                     (dict(C=1 << 17), L.ERR_BAD_SHAPE), (dict(H=1 << 16, W=1 << 16), L.ERR_BAD_SHAPE),
                     (dict(act=4), L.ERR_BAD_ARG), (dict(act=-1), L.ERR_BAD_ARG), (dict(dtype=2), L.ERR_BAD_ARG),
                     (dict(dtype=0, pdtype=1), L.ERR_BAD_ARG), (dict(x=None), L.ERR_NULL_POINTER),
                     (dict(mean=None), L.ERR_NULL_POINTER), (dict(q=Q, x=None if call is _bwd else X), L.ERR_NULL_POINTER),
                     (dict(x=ctypes.c_void_p(264)), L.ERR_BAD_ALIGN), (dict(w=ctypes.c_void_p(258), pdtype=2), L.ERR_BAD_ALIGN)]:
        assert call(L, **kw) == code, kw


def test_group_norm_refuses_a_bad_eps_and_an_ambiguous_source(L):
    for eps in (-1e-9, float("nan"), float("inf")):
        assert _fwd(L, eps=eps) == L.ERR_BAD_ARG
    assert _bwd(L, x=X, q=Q, s=S) == L.ERR_BAD_ARG
    assert _bwd(L, dx=None) == L.ERR_NULL_POINTER
    assert _fwd(L, B=0) == L.OK


def test_group_norm_workspace(L):
    n = ctypes.c_int64(-1)
    f = L.load().dwb_group_norm_act_workspace
    for shape in [(1, 7, 7, 1024, 32), (64, 56, 56, 1024, 32), (2, 300, 300, 64, 1), (1, 1, 1, 8, 8)]:
        for backward in (0, 1):
            assert f(*shape, backward, ctypes.byref(n)) == L.OK and n.value >= 0
            if n.value:
                call = _bwd if backward else _fwd
                B, H, W, C, G = shape
                assert call(L, nws=n.value - 1, B=B, H=H, W=W, C=C, G=G) == L.ERR_BAD_ARG
                assert call(L, ws=None, B=B, H=H, W=W, C=C, G=G) == L.ERR_NULL_POINTER
    assert f(0, 7, 7, 64, 8, 0, ctypes.byref(n)) == L.OK and n.value == 0
    assert f(1, 7, 7, 60, 6, 0, ctypes.byref(n)) == L.ERR_BAD_SHAPE
    assert f(1, 7, 7, 64, 8, 0, None) == L.ERR_NULL_POINTER


def test_python_refusals_on_cpu():
    import depthwise_conv_b200 as d
    x = torch.zeros(1, 64, 4, 4, dtype=torch.float16).contiguous(memory_format=torch.channels_last)
    q, s = torch.zeros(1, 64, 4, 4, dtype=torch.int8), torch.zeros(1, 4, 4, 2, dtype=torch.uint8)
    for call in (lambda: d.act8_encode(x), lambda: d.act8_decode(q, s), lambda: d.group_norm_act(x, 8),
                 lambda: d.act8_ops.conv2d_nhwc_backward_weight_act8(q, s, x, 3),
                 lambda: d.conv2d_nhwc_act8(x, torch.zeros(3, 3, 64, dtype=torch.float16)),
                 lambda: d.norm_ops.group_norm_act_backward(x, x, x, x, 8)):
        with pytest.raises(RuntimeError, match="CUDA"):
            call()
    with pytest.raises(RuntimeError, match="act must be"):
        d.norm_ops._act_code("tanh")


def test_fake_impls():
    import depthwise_conv_b200  # noqa: F401
    from torch._subclasses.fake_tensor import FakeTensorMode
    with FakeTensorMode():
        x = torch.empty(2, 72, 5, 6, dtype=torch.float16, device="cuda").contiguous(memory_format=torch.channels_last)
        w = torch.empty(5, 5, 72, dtype=torch.float16, device="cuda")
        v = torch.empty(72, device="cuda")
        y, mean, rstd, codes, scales = torch.ops.depthwise.group_norm_act(x, 8, v, v, 1e-5, 3, True)
        assert y.shape == x.shape and y.stride() == x.stride() and mean.shape == rstd.shape == (2, 8)
        assert codes.dtype == torch.int8 and codes.stride() == x.stride() and scales.shape == (2, 5, 6, 3)
        assert torch.ops.depthwise.group_norm_act(x, 8, None, None, 1e-5, 0, False)[3].numel() == 0
        codes, scales = torch.ops.depthwise.act8_encode(x)
        back = torch.ops.depthwise.act8_decode(codes, scales, torch.bfloat16)
        assert back.dtype == torch.bfloat16 and back.stride() == x.stride()
        y, codes, scales = torch.ops.depthwise.conv2d_nhwc_act8(x, w)
        assert y.stride() == x.stride() and codes.shape == x.shape and scales.dtype == torch.uint8


def test_trainable_block_on_cpu_fails_loudly():
    from depthwise_conv_b200.convmixer import TrainableDWBlock
    x = torch.zeros(1, 64, 8, 8, dtype=torch.float16).contiguous(memory_format=torch.channels_last)
    for checkpoint8 in (False, True):
        with pytest.raises(RuntimeError, match="CUDA"):
            TrainableDWBlock(64, 5, 8, checkpoint8=checkpoint8)(x)


def _wgrad_workspace(L, *shape):
    n = ctypes.c_int64(-1)
    assert L.load().dwb_conv2d_nhwc_bwd_weight_act8_workspace(*shape, ctypes.byref(n)) == L.OK, shape
    return n.value


@pytest.mark.parametrize("H,W,C", [(56, 56, 1024), (56, 56, 128), (32, 32, 768), (14, 14, 512), (7, 7, 1024), (224, 224, 128)])
def test_weight_gradient_workspace_does_not_grow_with_the_batch(L, H, W, C):
    """At most 12 turns of the CTAs that run at once (148 SMs, 3 CTAs each at K <= 7, 2 at K <= 15), each with 32
    channels of K * K sums, and beyond that a slice for every 256 chains of 128 products of 16 columns: 123 KB at most
    for 16.8 M values, 0.75% of a byte for each (2.3 times that at 7 columns of a tile of 16)."""
    for K in (3, 7, 9, 13, 15, 21, 27, 31):
        turns = 12 * 148 * (3 if K <= 7 else 2 if K <= 15 else 1) * 32 * K * K * 4
        for B in (64, 1024, 4096):
            assert _wgrad_workspace(L, B, H, W, C, K) <= turns + 0.02 * B * H * W * C
    assert _wgrad_workspace(L, 64, 56, 56, 1024, 31) <= 40e6


def test_weight_gradient_takes_long_batches(L):
    """As many images as the tensors may have: their number limits neither the ranges nor the workspace."""
    for B, H, W, C, K in [(1 << 20, 512, 64, 8, 31), (1 << 30, 1, 16, 8, 3), (1 << 18, 56, 56, 128, 31), (1, 1 << 24, 64, 8, 17)]:
        assert 0 < _wgrad_workspace(L, B, H, W, C, K) <= 0.01 * B * H * W * C + 12 * 148 * 3 * 32 * K * K * 4


def test_no_checkpoint_where_no_gradient_is_taken(monkeypatch):
    """The differentiable ops with the kernels' calls replaced: who asks for a checkpoint, and when."""
    import depthwise_conv_b200 as d
    made = []

    def encode(x):
        made.append("conv")
        return d.act8_ops.empty_checkpoint(x)

    def norm(x, num_groups, weight, bias, eps, act, checkpoint):
        stats = torch.zeros(x.shape[0], num_groups)
        out = (x.clone(memory_format=torch.preserve_format), stats, stats.clone())
        if checkpoint:
            made.append("norm")
        return (*out, *d.act8_ops.empty_checkpoint(x)) if checkpoint else out

    monkeypatch.setattr(d.act8_ops, "act8_encode", encode)
    monkeypatch.setattr(d.norm_ops, "group_norm_act_forward", norm)
    monkeypatch.setattr(d.dw_ops, "conv2d_nhwc_fused", lambda x, w, bias=None: x.clone(memory_format=torch.preserve_format))
    monkeypatch.setattr(d.dw_ops, "conv2d_nhwc_backward_input", lambda g, w: 2 * g)
    monkeypatch.setattr(d.act8_ops, "conv2d_nhwc_backward_weight_act8",
                        lambda codes, scales, g, K: torch.ones(K, K, g.shape[1]))

    def call(f, *args):
        made.clear()
        return f(*args)

    x = torch.zeros(2, 64, 4, 4, dtype=torch.float16).contiguous(memory_format=torch.channels_last)
    w, v = torch.zeros(3, 3, 64, dtype=torch.float16), torch.ones(64)
    conv = lambda *a: call(d.conv2d_nhwc_act8, *a)  # noqa: E731
    gn = lambda *a: call(lambda *b: d.group_norm_act(b[0], 8, b[1], b[2], checkpoint=True), *a)  # noqa: E731
    grad = lambda t: t.clone(memory_format=torch.preserve_format).requires_grad_()  # noqa: E731
    # nothing to differentiate: grad mode off, or no input that requires it
    with torch.no_grad():
        conv(grad(x), grad(w))
        assert made == []
        gn(grad(x), grad(v), grad(v))
        assert made == []
    with torch.inference_mode():
        conv(x, w)
        assert made == []
    conv(x, w)
    assert made == []
    gn(x, v, v)
    assert made == []
    # a frozen weight: the input gradient alone, which reads no input
    xg = grad(x)
    conv(xg, w).backward(torch.ones_like(x))
    assert made == [] and (xg.grad == 2).all()
    # a weight gradient
    wg = grad(w)
    conv(x, wg).backward(torch.ones_like(x))
    assert made == ["conv"] and (wg.grad == 1).all()
    # every gradient of the norm reads its input
    for args in ((grad(x), v, v), (x, grad(v), None), (x, None, grad(v))):
        gn(*args)
        assert made == ["norm"]
    # the op itself does what its argument says, which is to make one unless told otherwise
    wg = grad(w)
    call(torch.ops.depthwise.conv2d_nhwc_act8, x, wg)[0].backward(torch.ones_like(x))
    assert made == ["conv"] and (wg.grad == 1).all()
    assert torch.ops.depthwise.conv2d_nhwc_act8(x, w)[1].shape == x.shape
    y, codes, scales = torch.ops.depthwise.conv2d_nhwc_act8(x, grad(w), None, False)
    assert codes.numel() == scales.numel() == 0
    with pytest.raises(RuntimeError, match="needs a checkpoint"):
        y.backward(torch.ones_like(x))


@pytest.fixture
def bind_build(monkeypatch, tmp_path):
    """csrc/build.py with the Python module's files in tmp_path and a compiler that only notes its calls."""
    from depthwise_conv_b200.csrc import build as b
    calls = []

    class Done:
        returncode, stdout, stderr = 0, "", ""

    def run(cmd, **_):
        calls.append(cmd)
        (tmp_path / "bind.so").write_text("")
        return Done

    monkeypatch.setattr(b, "BIND", str(tmp_path / "bind.so"))
    monkeypatch.setattr(b, "BUILD", str(tmp_path / "objects"))
    monkeypatch.setattr(b, "BIND_VERSIONS", str(tmp_path / "objects" / "versions"), raising=False)
    monkeypatch.setattr(b.subprocess, "run", run)
    return b, calls


def test_build_without_pytorch(bind_build, monkeypatch):
    """The library is built without PyTorch; its Python module is left out then."""
    import sys
    b, calls = bind_build
    monkeypatch.setitem(sys.modules, "torch", None)  # `import torch` raises
    real = importlib.util.find_spec
    monkeypatch.setattr(importlib.util, "find_spec", lambda name, *a: None if name == "torch" else real(name, *a))
    assert b.build_bind() is None and calls == []


def test_the_python_module_is_rebuilt_for_another_pytorch(bind_build, monkeypatch):
    b, calls = bind_build
    assert b.build_bind() == b.BIND and len(calls) == 1
    assert b.build_bind() == b.BIND and len(calls) == 1  # nothing has changed
    real = importlib.metadata.version
    monkeypatch.setattr(importlib.metadata, "version", lambda name: "0.0" if name == "torch" else real(name))
    b.build_bind()
    assert len(calls) == 2
    b.build_bind()
    assert len(calls) == 2


def test_group_norm_takes_a_group_for_each_of_65536_channels(L):
    n = ctypes.c_int64(-1)
    for backward in (0, 1):
        assert L.load().dwb_group_norm_act_workspace(2, 3, 3, 65536, 65536, backward, ctypes.byref(n)) == L.OK
    assert _fwd(L, C=65536, G=65536, x=None) == _bwd(L, C=65536, G=65536, dy=None) == L.ERR_NULL_POINTER
