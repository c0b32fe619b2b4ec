"""Group norm with an activation, 8-bit activation checkpoints and the weight gradient that reads them, on
the GPU against the float64 restatements in oracle/train_ref.py.

Bounds.  u = one rounding to the output's type, eps/2 of its value (fp16 2^-11, bf16 2^-8) plus half its
finest step; e32 = 2^-24.  In fp32 a value passes through fewer than 64 roundings between its inputs and the
output, each at most e32 of the largest term at that point (for x_hat that includes mean * rstd: the mean is
a rounded fp32), and the GELU's and its slope's approximation adds at most 3e-7 < 8 e32 of the gradient's
size, so 64 e32 times the sum of the terms' magnitudes bounds it.  Sums of many terms: a chain of at most
2^8 additions between roundings to one partial sum (rows of a thread, threads, chunks, samples), so
2^8 e32 = 2^-16 times the sum of the magnitudes.
"""
from __future__ import annotations

import ctypes

import pytest
import torch

from oracle import train_ref as R

pytestmark = pytest.mark.gpu

E32 = 2.0**-24
HALF = {torch.float16: 2.0**-11, torch.bfloat16: 2.0**-8, torch.float32: E32}
FINEST = {torch.float16: 2.0**-25, torch.bfloat16: 2.0**-134, torch.float32: 2.0**-150}


@pytest.fixture(scope="module")
def eng():
    import depthwise_conv_b200 as d
    return d


def nhwc(B, C, H, W, seed, dtype, spread=1.0, offset=0.5):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn(B, H, W, C, device="cuda", generator=g) * spread
    x = x * (0.5 + torch.rand(C, device="cuda", generator=g)) + offset * torch.randn(C, device="cuda", generator=g)
    return x.to(dtype).permute(0, 3, 1, 2)


def params(C, seed, dtype):
    g = torch.Generator(device="cuda").manual_seed(seed)
    w = (1 + 0.3 * torch.randn(C, device="cuda", generator=g)).to(dtype)
    return w, (0.3 * torch.randn(C, device="cuda", generator=g)).to(dtype)


def rounded(ref, dtype):
    return HALF[dtype] * ref.abs() + FINEST[dtype]


# groups inside a vector, of 9 channels, one channel, the whole sample; one pixel; a ragged last block of 32
# channels; samples too large for one SM; more groups than a grid's SMs
SHAPES = [(2, 7, 5, 64, 8), (1, 1, 1, 8, 1), (3, 1, 1, 24, 3), (2, 23, 17, 72, 8), (1, 9, 9, 40, 5), (2, 5, 6, 48, 16),
          (2, 3, 3, 8, 8), (2, 16, 16, 1536, 32), (1, 32, 32, 768, 1), (1, 130, 70, 64, 4), (5, 14, 14, 512, 32),
          (1, 3, 2, 4104, 3), (1, 200, 200, 64, 1), (70, 2, 3, 16, 2), (1, 7, 7, 1024, 32), (1, 57, 1, 200, 25)]
# tensors that go through memory twice: groups larger than a tile, of 257 channels, of 9, of 4, of 3 in a ragged last
# tile and of one channel; few long rows; a batch in several groups of samples
LARGE = [(2, 61, 47, 1536, 2), (2, 31, 33, 2056, 8), (5, 120, 119, 72, 8), (8, 100, 90, 128, 32), (3, 128, 127, 264, 88),
         (2, 180, 170, 104, 104), (1, 1, 40000, 40, 1), (6, 97, 96, 776, 97)]
ACTS = ["gelu", "none", "silu", "relu"]


def check_forward(got, x, G, w, b, eps, act):
    y, mean, rstd = got[:3]
    C = x.shape[1]
    yr, mr, rr, u = R.group_norm_act(x, G, w, b, eps, act)
    v = x.double().reshape(x.shape[0], G, -1)
    far = (v - mr[..., None]).abs().amax(dim=2)
    assert ((mean.double() - mr).abs() <= 16 * E32 * far + 2 * E32 * mr.abs()).all()
    # var's relative error is at most 64 e32, and that of eps's and the root's roundings less
    assert ((rstd.double() - rr).abs() <= 64 * E32 * rr).all()
    wd = torch.ones(C, dtype=torch.float64, device=x.device) if w is None else w.double().abs()
    bd = torch.zeros_like(wd) if b is None else b.double().abs()
    xh = R.normalised(x, mr, rr)
    size = wd[:, None, None] * (xh.abs() + R._per_channel((mr * rr).abs(), C)) + bd[:, None, None]
    limit = rounded(yr, y.dtype) + 64 * E32 * size
    assert y.dtype == x.dtype and y.is_contiguous(memory_format=torch.channels_last)
    assert ((y.double() - yr).abs() <= limit).all(), ((y.double() - yr).abs() / limit).max()


def check_backward(got, dy, saved, mean, rstd, G, w, b, act):
    r = R.group_norm_act_grad(dy, saved, mean, rstd, G, w, b, act)
    if act == "relu":  # at the corner both slopes are right: the inputs stay clear of it
        assert r["u"].abs().min() > 4e-6
    dx, dw, db = got
    # u enters the slope: act'' <= 0.8 times u's error, with mean * rstd among its terms
    far = 1 + R._per_channel((mean.double() * rstd.double()).abs(), dy.shape[1])
    limit = rounded(r["dx"], dx.dtype) + 64 * E32 * far * r["dx_size"]
    assert dx.dtype == dy.dtype and dx.is_contiguous(memory_format=torch.channels_last)
    assert ((dx.double() - r["dx"]).abs() <= limit).all(), ((dx.double() - r["dx"]).abs() / limit).max()
    top = float(far.max())
    for v, p, name in ((dw, w, "dweight"), (db, b, "dbias")):
        if p is None:
            assert v is None
            continue
        size = r[name + "_size"] + (r["dbias_size"] * (top - 1) if name == "dweight" else 0)
        limit = rounded(r[name], p.dtype) + (2.0**-16 + 64 * E32 * top) * size
        assert v.dtype == p.dtype and v.shape == p.shape
        assert ((v.double() - r[name]).abs() <= limit).all(), name


@pytest.mark.parametrize("i,shape", list(enumerate(SHAPES)))
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_forward(eng, i, shape, dtype):
    B, H, W, C, G = shape
    x = nhwc(B, C, H, W, i, dtype)
    w, b = params(C, i, torch.float32 if i % 2 else dtype)
    act = ACTS[i % 4]
    check_forward(eng.norm_ops.group_norm_act_forward(x, G, w, b, 1e-5, act), x, G, w, b, 1e-5, act)
    check_forward(eng.norm_ops.group_norm_act_forward(x, G, None, b, 1e-3, "none"), x, G, None, b, 1e-3, "none")


@pytest.mark.parametrize("i,shape", list(enumerate(SHAPES)))
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_forward_with_checkpoint(eng, i, shape, dtype):
    """The same y, mean and rstd bit for bit, and the checkpoint that the codec itself writes."""
    B, H, W, C, G = shape
    x = nhwc(B, C, H, W, i + 50, dtype)
    w, b = params(C, i, dtype)
    plain = eng.norm_ops.group_norm_act_forward(x, G, w, b, 1e-5, ACTS[i % 4])
    kept = eng.norm_ops.group_norm_act_forward(x, G, w, b, 1e-5, ACTS[i % 4], checkpoint=True)
    for a, c in zip(plain, kept[:3]):
        assert torch.equal(a, c)
    codes, scales = R.act8_encode(x)
    assert torch.equal(kept[3], codes) and torch.equal(kept[4], scales)


@pytest.mark.parametrize("i,shape", list(enumerate(SHAPES)))
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("kept", ["input", "checkpoint"])
def test_backward(eng, i, shape, dtype, kept):
    B, H, W, C, G = shape
    # seeds at which no ReLU input lies at the corner; GELU and SiLU elsewhere
    act = ACTS[i % 4] if B * H * W * C < 40000 else ACTS[i % 3]
    x = nhwc(B, C, H, W, i + 100, dtype)
    w, b = params(C, i, torch.float32 if i % 2 else dtype)
    mean, rstd = (t.float() for t in R.stats(x, G, 1e-5))
    dy = nhwc(B, C, H, W, i + 200, dtype, spread=0.3, offset=0.1)
    codes, scales = R.act8_encode(x)
    saved, values = (x, x) if kept == "input" else ((codes, scales), R.act8_decode(codes, scales))
    got = eng.norm_ops.group_norm_act_backward(dy, saved, mean, rstd, G, w, b, act)
    check_backward(got, dy, values, mean, rstd, G, w, b, act)
    again = eng.norm_ops.group_norm_act_backward(dy, saved, mean, rstd, G, w, b, act)
    assert all(torch.equal(p, q) for p, q in zip(got, again))
    got = eng.norm_ops.group_norm_act_backward(dy, saved, mean, rstd, G, None, None, "none")
    check_backward(got, dy, values, mean, rstd, G, None, None, "none")


@pytest.mark.parametrize("i,shape", list(enumerate(LARGE)))
def test_large_tensors(eng, i, shape):
    """Forward with and without a checkpoint, backward from both."""
    B, H, W, C, G = shape
    dtype = [torch.float16, torch.bfloat16][i % 2]
    act = ["gelu", "silu", "none"][i % 3]
    x, dy = nhwc(B, C, H, W, i + 300, dtype), nhwc(B, C, H, W, i + 400, dtype, spread=0.3, offset=0.1)
    w, b = params(C, i, torch.float32 if i % 2 else dtype)
    got = eng.norm_ops.group_norm_act_forward(x, G, w, b, 1e-5, act, checkpoint=True)
    check_forward(got, x, G, w, b, 1e-5, act)
    plain = eng.norm_ops.group_norm_act_forward(x, G, w, b, 1e-5, act)
    assert all(torch.equal(p, q) for p, q in zip(got, plain))
    codes, scales = R.act8_encode(x)
    assert torch.equal(got[3], codes) and torch.equal(got[4], scales)
    del got, plain
    mean, rstd = (t.float() for t in R.stats(x, G, 1e-5))
    for saved, values in ((x, x), ((codes, scales), R.act8_decode(codes, scales))):
        back = eng.norm_ops.group_norm_act_backward(dy, saved, mean, rstd, G, w, b, act)
        check_backward(back, dy, values, mean, rstd, G, w, b, act)
        again = eng.norm_ops.group_norm_act_backward(dy, saved, mean, rstd, G, w, b, act)
        assert all(torch.equal(p, q) for p, q in zip(back, again))


@pytest.mark.parametrize("offset,spread", [(1000.0, 1.0), (0.0, 1e-3), (0.0, 3000.0)])
def test_statistics_far_from_zero(eng, offset, spread):
    """A mean a thousand times the deviation, tiny and large values: var without cancellation."""
    g = torch.Generator(device="cuda").manual_seed(9)
    x = (offset + spread * torch.randn(2, 31, 17, 64, device="cuda", generator=g)).half().permute(0, 3, 1, 2)
    check_forward(eng.norm_ops.group_norm_act_forward(x, 4, act="silu"), x, 4, None, None, 1e-5, "silu")


def test_an_outlier_in_the_first_pixel(eng):
    x = nhwc(1, 64, 40, 40, 3, torch.float16)
    x[0, :, 0, 0] = 60000.0
    check_forward(eng.norm_ops.group_norm_act_forward(x, 8), x, 8, None, None, 1e-5, "none")


def test_constant_groups_and_zero_eps(eng):
    x = torch.full((2, 32, 3, 3), 2.5, dtype=torch.float16, device="cuda").contiguous(memory_format=torch.channels_last)
    y, mean, rstd = eng.norm_ops.group_norm_act_forward(x, 4, eps=1e-5)
    assert (y == 0).all() and (mean == 2.5).all()
    assert torch.allclose(rstd, torch.full_like(rstd, 1e-5**-0.5), rtol=1e-6)
    _, _, rstd = eng.norm_ops.group_norm_act_forward(x, 4, eps=0.0)
    assert torch.isinf(rstd).all()


@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_not_a_number_stays_in_its_group(eng, bad):
    x = nhwc(2, 64, 6, 6, 4, torch.bfloat16)
    x[1, 17, 2, 3] = bad
    for act in ("none", "gelu", "silu", "relu"):
        y, mean, rstd, codes, scales = eng.norm_ops.group_norm_act_forward(x, 4, act=act, checkpoint=True)
        assert torch.isnan(y[1, 16:32]).all() or act != "none"
        assert torch.isnan(y[1, 16:32].float()).any()
        rest = torch.cat([y[0].flatten(), y[1, :16].flatten(), y[1, 32:].flatten()])
        assert torch.isfinite(rest).all()
        assert (scales == 255).sum() == 1 and scales[1, 2, 3, 0] == 255
        dx, _, _ = eng.norm_ops.group_norm_act_backward(torch.ones_like(x), (codes, scales), mean, rstd, 4, act=act)
        assert torch.isnan(dx[1, 16:32]).any() and torch.isfinite(dx[0]).all()


# ---- codec ------------------------------------------------------------------------------------------

CODEC_SHAPES = [(1, 1, 1, 8), (2, 3, 5, 32), (1, 7, 7, 72), (3, 13, 11, 200), (2, 17, 19, 1024), (1, 1, 3, 2056), (4, 32, 32, 96)]


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("B,H,W,C", CODEC_SHAPES)
def test_codec(eng, B, H, W, C, dtype):
    x = nhwc(B, C, H, W, C, dtype)
    scale = torch.exp2(torch.randint(-30, 12, (B, 1, H, W), device="cuda").float())
    x = (x.float() * scale).clamp(-6e4, 6e4).to(dtype)
    x[0, : C // 2, 0, 0] = 0
    codes, scales = eng.act8_encode(x)
    cr, sr = R.act8_encode(x)
    assert torch.equal(scales, sr) and torch.equal(codes, cr)
    assert codes.is_contiguous(memory_format=torch.channels_last)
    back = eng.act8_decode(codes, scales, dtype)
    assert torch.equal(back.double(), R.act8_decode(codes, scales))
    assert back.is_contiguous(memory_format=torch.channels_last)
    # what a checkpoint stands for has itself as its checkpoint's values
    assert torch.equal(eng.act8_decode(*eng.act8_encode(back), dtype), back)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_codec_over_every_16_bit_pattern(eng, dtype):
    """All 65536 patterns as the largest value of a block, next to smaller ones."""
    top = torch.arange(65536, device="cuda", dtype=torch.int32).to(torch.int16).view(dtype)
    x = torch.zeros(1, 256, 256, 32, dtype=dtype, device="cuda")
    x[0, :, :, 5] = top.view(256, 256)
    x[0, :, :, 6] = (top.float() * 0.37).to(dtype).view(256, 256)
    x[0, :, :, 31] = (top.float() * -0.004).to(dtype).view(256, 256)
    x = x.permute(0, 3, 1, 2)
    codes, scales = eng.act8_encode(x)
    cr, sr = R.act8_encode(x)
    assert torch.equal(scales, sr)
    fine = (sr != 255)
    q = codes.permute(0, 2, 3, 1)
    assert torch.equal(q[fine[..., 0]], cr.permute(0, 2, 3, 1)[fine[..., 0]])
    back, want = eng.act8_decode(codes, scales, dtype), R.act8_decode(cr, sr)
    assert torch.equal(torch.isnan(back), torch.isnan(want))
    assert torch.equal(back.double().nan_to_num(7), want.nan_to_num(7))


# ---- weight gradient --------------------------------------------------------------------------------

WGRAD_SHAPES = [(2, 19, 21, 72, 7), (1, 9, 30, 64, 31), (3, 5, 11, 64, 9), (1, 14, 14, 512, 27), (2, 1, 1, 8, 1),
                (2, 23, 17, 136, 13), (1, 3, 40, 16, 29), (1, 6, 100, 64, 7), (2, 5, 130, 72, 31), (1, 1, 1, 32, 31),
                (4, 7, 7, 96, 13), (1, 40, 3, 40, 3), (2, 33, 64, 32, 5), (3, 16, 16, 32, 17), (1, 64, 65, 24, 15),
                (9, 2, 15, 8, 23), (1, 28, 28, 256, 29), (2, 32, 32, 64, 9), (5, 8, 16, 160, 19), (1, 12, 48, 8, 25)]


def _wgrad_problem(B, H, W, C, K):
    x = nhwc(B, C, H, W, 10 * K + C, torch.float16)
    dy = nhwc(B, C, H, W, 10 * K + C + 1, torch.float16, spread=0.3, offset=0.05)
    return R.act8_encode(x), dy


@pytest.mark.parametrize("B,H,W,C,K", WGRAD_SHAPES)
def test_weight_gradient_from_checkpoint(eng, B, H, W, C, K):
    (codes, scales), dy = _wgrad_problem(B, H, W, C, K)
    dw = eng.act8_ops.conv2d_nhwc_backward_weight_act8(codes, scales, dy, K)
    ref, size = R.dw_weight_grad(R.act8_decode(codes, scales), dy, K)
    assert dw.dtype == torch.float32 and dw.shape == (K, K, C)
    # exact products, fp32 partial sums of at most 2^8 additions in a chain
    assert ((dw.double() - ref).abs() <= 2.0**-16 * size).all()
    assert (dw.double() - ref).norm() <= 1e-5 * ref.norm()  # the bar of the 16-bit weight gradient
    assert torch.equal(dw, eng.act8_ops.conv2d_nhwc_backward_weight_act8(codes, scales, dy, K))
    assert eng.device_error() == 0


def test_weight_gradient_ignores_what_lies_outside_the_tensors(eng):
    """Codes, scales and dy cut out of larger buffers full of NaN patterns: nothing around them is used."""
    B, H, W, C, K = 2, 5, 9, 40, 11
    (codes, scales), dy = _wgrad_problem(B, H, W, C, K)
    want = eng.act8_ops.conv2d_nhwc_backward_weight_act8(codes, scales, dy, K)
    n = B * H * W

    def inside(t, fill, per):
        flat = torch.full((n * per + 2 * 1024,), fill, dtype=t.dtype, device="cuda")
        flat[1024:1024 + n * per] = t.reshape(-1)
        return flat[1024:1024 + n * per]

    q = inside(codes.permute(0, 2, 3, 1), 127, C).view(B, H, W, C).permute(0, 3, 1, 2)
    s = inside(scales, 255, 2).view(B, H, W, 2)
    g = inside(dy.permute(0, 2, 3, 1), float("nan"), C).view(B, H, W, C).permute(0, 3, 1, 2)
    assert torch.equal(eng.act8_ops.conv2d_nhwc_backward_weight_act8(q, s, g, K), want)


def test_weight_gradient_keeps_a_nan_in_its_channels(eng):
    (codes, scales), dy = _wgrad_problem(2, 12, 20, 96, 7)
    clean = eng.act8_ops.conv2d_nhwc_backward_weight_act8(codes, scales, dy, 7)
    scales[1, 3, 4, 1] = 255
    dw = eng.act8_ops.conv2d_nhwc_backward_weight_act8(codes, scales, dy, 7)
    assert torch.isnan(dw[3, 3, 32:64]).all()
    assert torch.equal(dw[..., :32], clean[..., :32]) and torch.equal(dw[..., 64:], clean[..., 64:])


# ---- refusals -----------------------------------------------------------------------------------------

def test_refusals(eng):
    x = nhwc(2, 64, 4, 4, 0, torch.float16)
    w, b = params(64, 0, torch.float16)
    n, a = eng.norm_ops, eng.act8_ops
    mean, rstd = (t.float() for t in R.stats(x, 8, 1e-5))
    codes, scales = eng.act8_encode(x)
    cases = [
        (lambda: n.group_norm_act_forward(x.float(), 8), "float16 or bfloat16"),
        (lambda: n.group_norm_act_forward(x.contiguous(), 8), "channels_last"),
        (lambda: n.group_norm_act_forward(x[0], 8), "4-D"),
        (lambda: n.group_norm_act_forward(x, 7), "shape"),
        (lambda: n.group_norm_act_forward(x, 8, w[:32]), "weight must be"),
        (lambda: n.group_norm_act_forward(x, 8, w, b.float()), "one type"),
        (lambda: n.group_norm_act_forward(x, 8, w.bfloat16()), "weight must be"),
        (lambda: n.group_norm_act_forward(x, 8, w.cpu()), "weight must be"),
        (lambda: n.group_norm_act_forward(x, 8, eps=-1.0), "argument"),
        (lambda: n.group_norm_act_forward(x, 8, act="tanh"), "act must be"),
        (lambda: n.group_norm_act_forward(x, 8, act=9), "argument"),
        (lambda: n.group_norm_act_backward(x, x.bfloat16(), mean, rstd, 8), "saved input is"),
        (lambda: n.group_norm_act_backward(x, x[:1], mean, rstd, 8), "must match"),
        (lambda: n.group_norm_act_backward(x, x, mean[:1], rstd, 8), "mean must be"),
        (lambda: n.group_norm_act_backward(x, x, mean, rstd.half(), 8), "rstd must be"),
        (lambda: n.group_norm_act_backward(x, (codes, scales[:1]), mean, rstd, 8), "scales must be"),
        (lambda: eng.act8_decode(codes, scales, torch.float32), "dtype must be"),
        (lambda: eng.act8_decode(codes.contiguous(), scales), "channels_last"),
        (lambda: a.conv2d_nhwc_backward_weight_act8(codes, scales, x.bfloat16(), 3), "float16"),
        (lambda: a.conv2d_nhwc_backward_weight_act8(codes, scales, x[:, :, :2], 3), "channels_last|shape"),
        (lambda: a.conv2d_nhwc_backward_weight_act8(codes, scales, x, 4), "shape"),
    ]
    for call, text in cases:
        with pytest.raises(RuntimeError, match=text):
            call()
    assert eng.conv2d_nhwc(x, torch.zeros(3, 3, 64, dtype=torch.float16, device="cuda")).abs().max() == 0


def test_empty_batch(eng):
    x = nhwc(0, 64, 4, 4, 0, torch.float16)
    w, b = params(64, 0, torch.float32)
    y, mean, rstd, codes, scales = eng.norm_ops.group_norm_act_forward(x, 8, w, b, checkpoint=True)
    assert y.shape == x.shape and mean.shape == (0, 8)
    for saved in (x, (codes, scales)):
        dx, dw, db = eng.norm_ops.group_norm_act_backward(x, saved, mean, rstd, 8, w, b)
        assert dx.numel() == 0 and (dw == 0).all() and (db == 0).all()
    assert (eng.act8_ops.conv2d_nhwc_backward_weight_act8(codes, scales, x, 5) == 0).all()
    assert eng.act8_decode(*eng.act8_encode(x)).shape == x.shape


# ---- streams, graphs, buffers --------------------------------------------------------------------------

def _all(eng, x, dy, w, b, K=5, G=8):
    y, mean, rstd, codes, scales = eng.norm_ops.group_norm_act_forward(x, G, w, b, 1e-5, "gelu", checkpoint=True)
    back = eng.norm_ops.group_norm_act_backward(dy, (codes, scales), mean, rstd, G, w, b, "gelu")
    full = eng.norm_ops.group_norm_act_backward(dy, x, mean, rstd, G, w, b, "gelu")
    dw = eng.act8_ops.conv2d_nhwc_backward_weight_act8(codes, scales, dy, K)
    return [y, mean, rstd, codes, scales, *back, *full, dw, eng.act8_decode(codes, scales, x.dtype)]


@pytest.mark.parametrize("shape", [(2, 12, 11, 64), (1, 96, 96, 64)])
def test_two_streams_and_graphs_give_the_same_bits(eng, shape):
    """Two streams at once on their own data, then both captured and replayed together with new data."""
    B, H, W, C = shape
    w, b = params(C, 1, torch.float16)
    data = [(nhwc(B, C, H, W, s, torch.float16), nhwc(B, C, H, W, s + 1, torch.float16)) for s in (10, 20, 30, 40)]
    want = [_all(eng, x, dy, w, b) for x, dy in data]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [None, None]
    for _ in range(3):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i] = _all(eng, *data[i], w, b)
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(p, q) for p, q in zip(got[i], want[i]))
    graphs, held = [], []
    for i in range(2):
        x, dy = data[i][0].clone(memory_format=torch.preserve_format), data[i][1].clone(memory_format=torch.preserve_format)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = _all(eng, x, dy, w, b)
        graphs.append(g)
        held.append((x, dy, out))
    for i in range(2):  # data the capture has not seen
        held[i][0].copy_(data[i + 2][0])
        held[i][1].copy_(data[i + 2][1])
    torch.cuda.synchronize()
    for _ in range(3):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                graphs[i].replay()
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(p, q) for p, q in zip(held[i][2], want[i + 2]))


@pytest.mark.parametrize("shape", [(2, 12, 11, 64, 8), (1, 200, 200, 64, 1)])
def test_dx_in_the_buffer_of_dy(eng, shape):
    """dwb_group_norm_act_nhwc_bwd documents dx == dy."""
    from depthwise_conv_b200 import _lib
    B, H, W, C, G = shape
    x, dy = nhwc(B, C, H, W, 1, torch.float16), nhwc(B, C, H, W, 2, torch.float16)
    mean, rstd = (t.float() for t in R.stats(x, G, 1e-5))
    want = eng.norm_ops.group_norm_act_backward(dy, x, mean, rstd, G, act="silu")[0]
    n = ctypes.c_int64(0)
    _lib.call("dwb_group_norm_act_workspace", B, H, W, C, G, 1, ctypes.byref(n))
    ws = torch.empty(max(16, n.value), dtype=torch.uint8, device="cuda")
    _lib.call("dwb_group_norm_act_nhwc_bwd", dy.data_ptr(), x.data_ptr(), None, None, mean.data_ptr(), rstd.data_ptr(), None,
              None, dy.data_ptr(), None, None, ws.data_ptr(), n.value, B, H, W, C, G, 3, 0, 0,
              torch.cuda.current_stream().cuda_stream)
    torch.cuda.synchronize()
    assert torch.equal(dy, want)


def test_nothing_is_written_around_the_outputs(eng):
    """Outputs in the middle of buffers of a known pattern: ragged channels, pixels and a partial block."""
    from depthwise_conv_b200 import _lib
    B, H, W, C, G = 2, 5, 3, 40, 5
    n, pad = B * H * W, 512
    x = nhwc(B, C, H, W, 6, torch.float16)

    def guarded(count, dtype):
        return torch.full((count + 2 * pad,), 77, dtype=dtype, device="cuda")

    y, q, s = guarded(n * C, torch.float16), guarded(n * C, torch.int8), guarded(n * 2, torch.uint8)
    mean, rstd = guarded(B * G, torch.float32), guarded(B * G, torch.float32)
    b = ctypes.c_int64(0)
    _lib.call("dwb_group_norm_act_workspace", B, H, W, C, G, 0, ctypes.byref(b))
    ws = torch.full((b.value + 1024,), 77, dtype=torch.uint8, device="cuda")
    at = lambda t: t.data_ptr() + pad * t.element_size()  # noqa: E731
    _lib.call("dwb_group_norm_act_nhwc_fwd", x.data_ptr(), None, None, at(y), at(mean), at(rstd), at(q), at(s),
              ws.data_ptr() if b.value else None, b.value, B, H, W, C, G, 1e-5, 2, 0, 0,
              torch.cuda.current_stream().cuda_stream)
    torch.cuda.synchronize()
    for t in (y, q, s, mean, rstd):
        assert (t[:pad] == 77).all() and (t[-pad:] == 77).all()
    assert (ws[b.value:] == 77).all()
    want = eng.norm_ops.group_norm_act_forward(x, G, act="gelu", checkpoint=True)
    assert torch.equal(y[pad:-pad], want[0].permute(0, 2, 3, 1).reshape(-1))
    assert torch.equal(s[pad:-pad], want[4].reshape(-1))


# ---- autograd -------------------------------------------------------------------------------------------

@pytest.mark.parametrize("checkpoint", [False, True])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_group_norm_autograd(eng, checkpoint, dtype):
    B, H, W, C, G = 2, 10, 7, 96, 12
    x = nhwc(B, C, H, W, 1, dtype).requires_grad_()
    w, b = (t.requires_grad_() for t in params(C, 2, torch.float32))
    y = eng.group_norm_act(x, G, w, b, act="gelu", checkpoint=checkpoint)
    dy = torch.randn_like(y).contiguous()  # not channels_last: the op takes any gradient
    y.backward(dy)
    mean, rstd = (t.float() for t in R.stats(x.detach(), G, 1e-5))
    values = R.act8_decode(*R.act8_encode(x.detach())) if checkpoint else x.detach()
    check_backward((x.grad, w.grad, b.grad), dy, values, mean, rstd, G, w.detach(), b.detach(), "gelu")


def test_conv_autograd_with_checkpoint(eng):
    """The same y and dx as depthwise::conv2d_nhwc, dw from the checkpoint, and the input is not kept."""
    B, H, W, C, K = 2, 15, 18, 64, 9
    x = nhwc(B, C, H, W, 1, torch.float16).requires_grad_()
    g = torch.Generator(device="cuda").manual_seed(3)
    w = (torch.randn(K, K, C, device="cuda", generator=g) / K).half().requires_grad_()
    b = (0.1 * torch.randn(C, device="cuda", generator=g)).half().requires_grad_()
    dy = nhwc(B, C, H, W, 2, torch.float16)
    y0 = torch.ops.depthwise.conv2d_nhwc(x, w, b)
    dx0, dw0, db0 = torch.autograd.grad(y0, (x, w, b), dy)
    y1 = eng.conv2d_nhwc_act8(x, w, b)
    dx1, dw1, db1 = torch.autograd.grad(y1, (x, w, b), dy)
    assert torch.equal(y0, y1) and torch.equal(dx0, dx1) and torch.equal(db0, db1)
    ref, size = R.dw_weight_grad(R.act8_decode(*R.act8_encode(x.detach())), dy, K)
    assert dw1.dtype == torch.float16
    assert ((dw1.double() - ref).abs() <= rounded(ref, torch.float16) + 2.0**-16 * size).all()
    # how far the checkpoint itself moves the gradient: its values are within 1/127 of their block's maximum
    assert (dw1.double() - dw0.double()).norm() <= 2e-2 * dw0.double().norm()


def test_gradients_against_differences(eng):
    """d loss along a direction by the ops' gradients and by float64 differences of the oracle's forward."""
    B, H, W, C, G = 1, 6, 5, 32, 4
    x = nhwc(B, C, H, W, 11, torch.float16).requires_grad_()
    w, b = (t.requires_grad_() for t in params(C, 12, torch.float32))
    dy = nhwc(B, C, H, W, 13, torch.float16)
    eng.group_norm_act(x, G, w, b, act="silu").backward(dy)
    h = 1e-5
    for leaf in (x, w, b):
        g = torch.Generator(device="cuda").manual_seed(14)
        d = torch.randn(leaf.shape, device="cuda", generator=g, dtype=torch.float64)
        loss = []
        for s in (-h, h):
            v = [(t.detach().double() + s * d if t is leaf else t.detach().double()) for t in (x, w, b)]
            loss.append((R.group_norm_act(v[0], G, v[1], v[2], 1e-5, "silu")[0] * dy.double()).sum())
        slope = (loss[1] - loss[0]) / (2 * h)
        got = (leaf.grad.double() * d).sum()
        # fp16 dx: each of the 960 products within 2^-11 of itself
        assert abs(got - slope) <= (2.0**-11 * (leaf.grad.double() * d).abs().sum() + 1e-4)


def test_a_training_block(eng):
    """conv -> group norm + GELU -> conv -> group norm, both with checkpoints, forward and backward in one run:
    every gradient against float64 autograd of the same block; what the graph keeps is about half."""
    import torch.nn.functional as F
    B, H, W, C, G, K = 4, 24, 20, 64, 8, 7

    def leaves():
        g = torch.Generator(device="cuda").manual_seed(21)
        r = lambda *s: torch.randn(*s, device="cuda", generator=g)  # noqa: E731
        x = r(B, H, W, C).half().permute(0, 3, 1, 2)
        return [x, (r(K, K, C) / K).half(), (r(K, K, C) / K).half(), 1 + 0.2 * r(C), 0.2 * r(C), 1 + 0.2 * r(C), 0.2 * r(C)]

    def block(conv, checkpoint, x, w1, w2, g1, b1, g2, b2):
        z = eng.group_norm_act(conv(x, w1), G, g1, b1, act="gelu", checkpoint=checkpoint)
        return eng.group_norm_act(conv(z, w2), G, g2, b2, act="silu", checkpoint=checkpoint)

    dy = nhwc(B, C, H, W, 22, torch.float16)
    grads, kept = {}, {}
    for name, conv, ck in (("16", torch.ops.depthwise.conv2d_nhwc, False), ("8", eng.conv2d_nhwc_act8, True)):
        t = [v.requires_grad_() for v in leaves()]
        torch.cuda.synchronize()
        before = torch.cuda.memory_allocated()
        y = block(conv, ck, *t)
        kept[name] = torch.cuda.memory_allocated() - before
        y.backward(dy)
        grads[name] = [v.grad.double() for v in t]
    r = [v.double().requires_grad_() for v in leaves()]

    def ref_conv(x, w):
        return F.conv2d(x, w.permute(2, 0, 1).unsqueeze(1), padding=K // 2, groups=C)

    z = F.gelu(F.group_norm(ref_conv(r[0], r[1]), G, r[3], r[4]))
    F.silu(F.group_norm(ref_conv(z, r[2]), G, r[5], r[6])).backward(dy.double())
    # 16 bits: the convolution's own bar (1e-3 of the result) through two convolutions and their gradients;
    # 8 bits: four checkpoints, each off by at most amax / 127 / 2 per step of a power of two, 1e-2 of its norm
    for name, bar in (("16", 5e-3), ("8", 4e-2)):
        for v, ref in zip(grads[name], r):
            assert (v - ref.grad).norm() <= bar * ref.grad.norm(), name
    n = B * H * W * C
    assert kept["16"] >= 2 * n * 3 and kept["8"] <= 0.72 * kept["16"]
    assert eng.device_error() == 0


@pytest.mark.parametrize("checkpoint8", [False, True])
def test_trainable_blocks_in_a_model(eng, checkpoint8):
    """Two ConvMixer training blocks: every gradient against float64 autograd of the same blocks, and one
    gradient step that changes every parameter."""
    import torch.nn.functional as F

    from depthwise_conv_b200.convmixer import TrainableDWBlock
    torch.manual_seed(5)
    B, C, H, W, K = 2, 96, 16, 18, 9
    blocks = torch.nn.Sequential(*(TrainableDWBlock(C, K, 12, act, checkpoint8=checkpoint8) for act in ("gelu", "silu"))).cuda()
    x = nhwc(B, C, H, W, 31, torch.float16).requires_grad_()
    dy = nhwc(B, C, H, W, 32, torch.float16)
    y = blocks(x)
    assert y.is_contiguous(memory_format=torch.channels_last) and y.dtype == torch.float16
    y.backward(dy)
    r = x.detach().double().requires_grad_()
    z, leaves = r, []
    for b in blocks:
        p = [t.detach().double().requires_grad_() for t in (b.weight, b.norm_weight, b.norm_bias)]
        leaves.append(p)
        u = F.group_norm(F.conv2d(z, p[0].permute(2, 0, 1).unsqueeze(1), padding=K // 2, groups=C), 12, p[1], p[2], b.eps)
        z = z + (F.gelu(u) if b.activation == "gelu" else F.silu(u))
    z.backward(dy.double())
    bar = 4e-2 if checkpoint8 else 5e-3  # as in test_a_training_block
    assert (x.grad.double() - r.grad).norm() <= bar * r.grad.norm()
    for b, p in zip(blocks, leaves):
        for v, ref in zip((b.weight, b.norm_weight, b.norm_bias), p):
            assert (v.grad.double() - ref.grad).norm() <= bar * ref.grad.norm()
    before = [p.detach().clone() for p in blocks.parameters()]
    torch.optim.SGD(blocks.parameters(), lr=0.1).step()
    assert all(not torch.equal(a, b.detach()) for a, b in zip(before, blocks.parameters()))


@pytest.mark.parametrize("checkpoint8", [False, True])
def test_training_step_captured_and_replayed(eng, checkpoint8):
    """Forward and backward of a block captured into a graph on leaves of their own, replayed with new data:
    the gradients of an eager step on that data, bit for bit."""
    from depthwise_conv_b200.convmixer import TrainableDWBlock
    torch.manual_seed(6)
    B, C, H, W = 2, 64, 20, 20
    block = TrainableDWBlock(C, 7, 8, "gelu", checkpoint8=checkpoint8).cuda()
    data = [(nhwc(B, C, H, W, s, torch.float16), nhwc(B, C, H, W, s + 1, torch.float16)) for s in (50, 60)]

    def step(module, x, dy):
        return torch.autograd.grad(module(x), list(module.parameters()), dy)

    prev = torch.are_deterministic_algorithms_enabled()
    torch.use_deterministic_algorithms(True, warn_only=True)  # the 16-bit weight gradient in a fixed order
    try:
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step(block, *data[0])  # warm-up
        torch.cuda.current_stream().wait_stream(side)
        torch.cuda.synchronize()
        x, dy = data[0][0].clone(memory_format=torch.preserve_format), data[0][1].clone(memory_format=torch.preserve_format)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            grads = step(block, x, dy)
        x.copy_(data[1][0])
        dy.copy_(data[1][1])
        graph.replay()
        torch.cuda.synchronize()
        want = step(block, *data[1])
    finally:
        torch.use_deterministic_algorithms(prev)
    assert all(torch.equal(g, w) for g, w in zip(grads, want))


# ---- calls at the edges of what the ops take -------------------------------------------------------------

@pytest.mark.parametrize("K", [1, 5, 7, 9, 11, 15, 17, 23, 25, 31])
def test_weight_gradient_over_kernel_sizes_and_widths(eng, K):
    """Every width of a tile, just below, at and above it, with heights that end inside a step."""
    for i, W in enumerate((4, 16, 17, 32, 33, 48, 49, 64, 65)):
        B, H, C = 2 + i % 2, 1 + (5 * i + K) % 11, (24, 40, 64)[i % 3]
        (codes, scales), dy = _wgrad_problem(B, H, W, C, K)
        dw = eng.act8_ops.conv2d_nhwc_backward_weight_act8(codes, scales, dy, K)
        ref, size = R.dw_weight_grad(R.act8_decode(codes, scales), dy, K)
        assert ((dw.double() - ref).abs() <= 2.0**-16 * size).all(), (B, H, W, C)


@pytest.mark.parametrize("act", ["gelu", "none"])
def test_many_small_samples(eng, act):
    """More samples than a grid's second dimension takes: forward, backward and the checkpoint."""
    B, H, W, C, G = 70000, 1, 2, 16, 2
    x, dy = nhwc(B, C, H, W, 1, torch.float16), nhwc(B, C, H, W, 2, torch.float16, offset=0.1)
    w, b = params(C, 3, torch.float32)
    out = eng.norm_ops.group_norm_act_forward(x, G, w, b, act=act, checkpoint=True)
    check_forward(out, x, G, w, b, 1e-5, act)
    assert all(torch.equal(i, j) for i, j in zip(out[3:], eng.act8_encode(x)))
    mean, rstd = (t.float() for t in R.stats(x, G, 1e-5))
    dx = eng.norm_ops.group_norm_act_backward(dy, x, mean, rstd, G, w, b, act)[0]
    r = R.group_norm_act_grad(dy, x, mean, rstd, G, w, b, act)
    far = 1 + R._per_channel((mean.double() * rstd.double()).abs(), C)
    assert ((dx.double() - r["dx"]).abs() <= rounded(r["dx"], dx.dtype) + 64 * E32 * far * r["dx_size"]).all()


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
@pytest.mark.parametrize("shape", [(2, 9, 7, 72, 8), (2, 61, 47, 1536, 2)])
def test_parameters_at_any_offset(eng, shape, dtype):
    """Slices of one flat buffer, each a value further than a vector load could start: the same bits."""
    B, H, W, C, G = shape
    x, dy = nhwc(B, C, H, W, 1, torch.float16), nhwc(B, C, H, W, 2, torch.float16)
    w, b = params(C, 3, dtype)
    flat = torch.zeros(2 * C + 8, dtype=dtype, device="cuda")
    wv, bv = flat[1:1 + C].copy_(w), flat[C + 3:2 * C + 3].copy_(b)
    n = eng.norm_ops
    want, got = n.group_norm_act_forward(x, G, w, b, act="gelu"), n.group_norm_act_forward(x, G, wv, bv, act="gelu")
    assert all(torch.equal(i, j) for i, j in zip(want, got))
    want, got = (n.group_norm_act_backward(dy, x, *want[1:], G, p, q, "gelu") for p, q in ((w, b), (wv, bv)))
    assert all(torch.equal(i, j) for i, j in zip(want, got))


def test_offsets_past_32_bits(eng):
    """One image of 2^31 values and more, most of them zero: its last rows against the same rows by themselves."""
    H, W, C, G, K, tail = 8200, 8200, 32, 2, 3, 5
    x = torch.zeros(1, H, W, C, dtype=torch.float16, device="cuda").permute(0, 3, 1, 2)
    dy = torch.zeros_like(x)
    x[:, :, -tail:] = nhwc(1, C, tail, W, 1, torch.float16)
    dy[:, :, -tail:] = nhwc(1, C, tail, W, 2, torch.float16)
    w, b = params(C, 3, torch.float32)
    xt, dyt = x[:, :, -tail:], dy[:, :, -tail:]
    y, mean, rstd, codes, scales = eng.norm_ops.group_norm_act_forward(x, G, w, b, act="silu", checkpoint=True)
    small = eng.act8_encode(xt)
    assert torch.equal(codes[:, :, -tail:], small[0]) and torch.equal(scales[:, -tail:], small[1])
    assert not codes[:, :, :-tail].any()
    kept = eng.act8_encode(x)
    assert torch.equal(kept[0], codes) and torch.equal(kept[1], scales)
    assert torch.equal(eng.act8_decode(codes, scales)[:, :, -tail:], eng.act8_decode(*small))
    # a thread adds up to 2^10 values that are not zero: 2^10 e32 of the sum of the magnitudes
    v = xt.double().reshape(G, -1)
    n = H * W * C // G
    mr = v.sum(1) / n
    rr = (((v - mr[:, None])**2).sum(1) / n + (1 - v.shape[1] / n) * mr**2 + 1e-5).rsqrt()
    assert ((mean[0].double() - mr).abs() <= 2.0**-14 * v.abs().sum(1) / n + 2 * E32 * mr.abs()).all()
    assert ((rstd[0].double() - rr).abs() <= 2.0**-14 * rr).all()
    md, rd = mean.double(), rstd.double()
    u = R.normalised(xt, md, rd) * w.double()[:, None, None] + b.double()[:, None, None]
    yr, _ = R.act_and_slope(u, "silu")
    xh = R.normalised(xt, md, rd)
    size = w.double().abs()[:, None, None] * (xh.abs() + R._per_channel((md * rd).abs(), C)) + b.double().abs()[:, None, None]
    assert ((y[:, :, -tail:].double() - yr).abs() <= rounded(yr, y.dtype) + 64 * E32 * size).all()
    assert (y[:, :, :-tail] == y[:, :, :1, :1]).all()
    del y, kept
    # the input gradient: the sums over the rows with a gradient, then every pixel by itself
    d = [eng.norm_ops.group_norm_act_backward(dy, saved, mean, rstd, G, w, b, "none")[0] for saved in (x, (codes, scales))]
    for dx, values in zip(d, (xt, eng.act8_decode(*small))):
        xh, g = R.normalised(values, md, rd), dyt.double() * w.double()[:, None, None]
        m1, m2 = (R._per_channel(t.reshape(1, G, -1).sum(2) / n, C) for t in (g, g * xh))
        s1, s2 = (R._per_channel(t.abs().reshape(1, G, -1).sum(2) / n, C) for t in (g, g * xh))
        rc = R._per_channel(rd, C)
        ref, size = rc * (g - m1 - xh * m2), rc * (g.abs() + s1 + xh.abs() * s2)
        far = 1 + R._per_channel((md * rd).abs(), C)
        assert ((dx[:, :, -tail:].double() - ref).abs() <= rounded(ref, dx.dtype) + 2.0**-13 * far * size).all()
    del d
    dw = eng.act8_ops.conv2d_nhwc_backward_weight_act8(codes, scales, dy, K)
    ref, size = R.dw_weight_grad(R.act8_decode(*small), dyt, K)
    assert ((dw.double() - ref).abs() <= 2.0**-16 * size).all()
    assert eng.device_error() == 0


def test_a_second_derivative_is_refused(eng):
    """The backward passes are not differentiable: a gradient of a gradient raises, a first one with a graph does not."""
    x = nhwc(1, 32, 6, 5, 1, torch.float16).requires_grad_()
    w = torch.ones(3, 3, 32, dtype=torch.float16, device="cuda", requires_grad=True)
    for f in (lambda: eng.group_norm_act(x, 4, act="gelu"), lambda: eng.conv2d_nhwc_act8(x, w)):
        plain, = torch.autograd.grad(f().sum(), x)
        first, = torch.autograd.grad(f().sum(), x, create_graph=True)
        assert torch.equal(first, plain)
        with pytest.raises(RuntimeError, match="not differentiable"):
            (first.square().sum() + x.sum()).backward()


def test_a_gradient_off_the_vector_boundary(eng):
    """A gradient that autograd cuts out of a larger one at an odd place is copied, not refused."""
    x = nhwc(3, 32, 1, 1, 1, torch.float16).requires_grad_()
    y = eng.group_norm_act(x, 4, act="gelu")
    odd = torch.zeros(3, device="cuda", dtype=torch.float16, requires_grad=True)
    dy = torch.randn(99, device="cuda").half()
    torch.cat([odd, y.flatten()]).backward(dy)
    want = torch.autograd.grad(eng.group_norm_act(x, 4, act="gelu"), x, dy[3:].clone().view(3, 32, 1, 1))[0]
    assert torch.equal(x.grad, want)


@pytest.mark.parametrize("shape", [(1, 36, 18, 1208, 4), (4, 28, 28, 1544, 8), (1, 5, 3, 1032, 2), (2, 90, 70, 4104, 8)])
def test_large_groups_of_odd_sizes(eng, shape):
    """Groups too large for a tile and no multiple of 8 channels: an entry a channel, few groups of many entries."""
    B, H, W, C, G = shape
    x, dy = nhwc(B, C, H, W, 1, torch.float16), nhwc(B, C, H, W, 2, torch.float16, offset=0.1)
    w, b = params(C, 3, torch.float32)
    out = eng.norm_ops.group_norm_act_forward(x, G, w, b, act="gelu", checkpoint=True)
    check_forward(out, x, G, w, b, 1e-5, "gelu")
    assert all(torch.equal(i, j) for i, j in zip(out[3:], eng.act8_encode(x)))
    mean, rstd = (t.float() for t in R.stats(x, G, 1e-5))
    for kept, values in ((x, x), (out[3:], R.act8_decode(*R.act8_encode(x)))):
        got = eng.norm_ops.group_norm_act_backward(dy, kept, mean, rstd, G, w, b, "gelu")
        check_backward(got, dy, values, mean, rstd, G, w, b, "gelu")


@pytest.mark.parametrize("shape", [(160, 1, 1, 1024, 32), (150, 2, 2, 2048, 4), (100, 3, 3, 768, 768), (75, 7, 4, 1424, 356),
                                   (149, 1, 2, 1208, 151), (37, 7, 7, 1024, 32)])
def test_batches_of_few_pixels(eng, shape):
    """CTAs that take many units of channels, up to as many as they have threads for."""
    B, H, W, C, G = shape
    x, dy = nhwc(B, C, H, W, 1, torch.float16), nhwc(B, C, H, W, 2, torch.float16, offset=0.1)
    w, b = params(C, 3, torch.float16)
    out = eng.norm_ops.group_norm_act_forward(x, G, w, b, act="silu", checkpoint=True)
    check_forward(out, x, G, w, b, 1e-5, "silu")
    assert all(torch.equal(i, j) for i, j in zip(out[:3], eng.norm_ops.group_norm_act_forward(x, G, w, b, act="silu")))
    assert all(torch.equal(i, j) for i, j in zip(out[3:], eng.act8_encode(x)))
    mean, rstd = (t.float() for t in R.stats(x, G, 1e-5))
    for kept, values in ((x, x), (out[3:], R.act8_decode(*R.act8_encode(x)))):
        got = eng.norm_ops.group_norm_act_backward(dy, kept, mean, rstd, G, w, b, "silu")
        check_backward(got, dy, values, mean, rstd, G, w, b, "silu")
