"""Group norm, checkpoints and the weight gradient from a checkpoint at the ends of their ranges, on the GPU
against float64 (oracle/train_ref.py).

Bounds as in test_gpu_norm_act8.py: one rounding to the output's type, 64 e32 (e32 = 2^-24) of the terms'
magnitudes for what a value passes through in fp32.
"""
from __future__ import annotations

import math

import pytest
import torch

from oracle import train_ref as R

pytestmark = pytest.mark.gpu

E32 = 2.0**-24


@pytest.fixture(scope="module")
def eng():
    import depthwise_conv_b200 as d
    return d


def of_bias(eng, u, act, dtype, P=5, G=1):
    """act(u) through the norm: with a weight of 0 the activation's input is the bias.  [C] in float64.

    G = 1 and P = 5 run in the resident kernel."""
    C = u.numel()
    g = torch.Generator(device="cuda").manual_seed(C)
    x = torch.randn(1, P, 1, C, device="cuda", generator=g).to(dtype).permute(0, 3, 1, 2)
    y = eng.norm_ops.group_norm_act_forward(x, G, torch.zeros(C, device="cuda"), u.float().cuda(), act=act)[0]
    assert torch.equal(y.float().nan_to_num(7), y[:, :, :1].float().nan_to_num(7).expand_as(y)), "pixels differ"
    return y[0, :, 0, 0].double()


@pytest.mark.parametrize("act,ends", [("gelu", (math.inf, 0.0)), ("relu", (math.inf, 0.0)), ("none", (math.inf, -math.inf))])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("P", [5, 100000])
def test_infinite_activation_inputs(eng, act, ends, dtype, P):
    """An activation's input that is infinite (here the bias) gives the activation's limit, a NaN a NaN, and the
    channels beside it their own values; P = 5 in shared memory, 100000 in two passes."""
    u = torch.zeros(64, dtype=torch.float64)
    u[3], u[8], u[17], u[40] = math.inf, -math.inf, math.nan, 2.0
    y = of_bias(eng, u, act, dtype, P)
    assert y[3] == ends[0] and y[8] == ends[1] and torch.isnan(y[17])
    two = R.act_and_slope(u[40], act)[0].item()
    assert abs(y[40] - two) <= 2.0**-8 * two
    rest = torch.ones(64, dtype=torch.bool)
    rest[[3, 8, 17, 40]] = False
    assert (y[rest.cuda()] == 0).all()


@pytest.mark.parametrize("act", ["gelu", "silu"])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("P", [5, 5000])
def test_small_values_of_an_activation(eng, act, dtype, P):
    """Far below zero a value is small but still the activation's: little more than one rounding of the type.

    GELU's tail a Q(a) is off by at most 7.5e-8 < 1.3 e32, its ex2 and its product by 1 e32 more (a Q <= 0.17): 4 e32;
    and by at most 1.5e-3 < 2^-9 of itself up to |u| = 8.  The value's own fp32 operations, and SiLU's exponential,
    quotient and the exponent's argument (below 2^4, rounded at e32 of itself), are within 32 e32 of the value."""
    u = torch.linspace(-8, 8, 2048, dtype=torch.float64).float().double()
    y = of_bias(eng, u, act, dtype, P).cpu()
    ref = R.act_and_slope(u, act)[0]
    half = 2.0**-11 if dtype == torch.float16 else 2.0**-8
    finest = 2.0**-25 if dtype == torch.float16 else 0.0
    tail = torch.minimum(torch.full_like(ref, 4 * E32), 2.0**-9 * ref.abs())
    limit = half * ref.abs() + finest + tail + 32 * E32 * ref.abs()
    assert ((y - ref).abs() <= limit).all(), ((y - ref).abs() / limit).max()


@pytest.mark.parametrize("shape,kept", [((70000, 1, 2, 16, 2), "input"), ((70000, 1, 2, 16, 2), "checkpoint"),
                                        ((400000, 1, 2, 8, 1), "input")])
def test_parameter_gradients_of_many_samples(eng, shape, kept):
    """dweight and dbias where their sums over the samples are longest: gradients that are the same in every sample and
    fill a float's 24 bits, so that a chain of additions loses the same way again and again.

    In a sample (2 pixels at most) and over 32 partial sums fewer than 64 roundings, each at most e32 of the sum of the
    magnitudes; none from the number of samples.  x_hat's and the slope's roundings: 8 e32 of each term, and mean * rstd
    among x_hat's terms."""
    B, H, W, C, G = shape
    g = torch.Generator(device="cuda").manual_seed(B)
    x = torch.randn(B, H, W, C, device="cuda", generator=g).half().permute(0, 3, 1, 2)
    dy = torch.stack([torch.ones(C, device="cuda"), 1e-3 * (0.5 + torch.rand(C, device="cuda", generator=g))])
    dy = dy.half().expand(B, H, W, C).contiguous().permute(0, 3, 1, 2)
    w = torch.ones(C, device="cuda")
    mean, rstd = (t.float() for t in R.stats(x, G, 1e-5))
    saved = x if kept == "input" else eng.act8_encode(x)
    values = x if kept == "input" else R.act8_decode(*saved)
    _, dw, db = eng.norm_ops.group_norm_act_backward(dy, saved, mean, rstd, G, w, torch.zeros_like(w), "none")
    xh = R.normalised(values, mean, rstd)
    far = 1 + R._per_channel((mean.double() * rstd.double()).abs(), C)
    sums, size = (dy.double() * xh).sum(dim=(0, 2, 3)), (dy.double() * (xh.abs() + far)).sum(dim=(0, 2, 3))
    assert ((db.double() - dy.double().sum(dim=(0, 2, 3))).abs() <= 64 * E32 * dy.double().sum(dim=(0, 2, 3))).all()
    assert ((dw.double() - sums).abs() <= 64 * E32 * size).all()


def test_parameter_gradients_that_are_infinite(eng):
    """An infinite gradient gives an infinite sum (and a NaN where two of them cancel), in its own channel only."""
    x = torch.randn(40, 16, 3, 3, device="cuda").half().contiguous(memory_format=torch.channels_last)
    dy = torch.ones_like(x)
    dy[3, 4, 1, 1] = dy[30, 5, 0, 0] = math.inf
    dy[0, 6, 0, 0], dy[39, 6, 2, 2] = math.inf, -math.inf
    mean, rstd = (t.float() for t in R.stats(x, 2, 1e-5))
    db = eng.norm_ops.group_norm_act_backward(dy, x, mean, rstd, 2, None, torch.zeros(16, device="cuda"), "none")[2]
    assert db[4] == math.inf and db[5] == math.inf and torch.isnan(db[6])
    assert (db[[0, 1, 2, 3, *range(7, 16)]] == 360).all()


# ---- weight gradient: ranges of many steps ------------------------------------------------------------

def wgrad_chunks(B, H, W, C, K):
    """Ranges that the steps of a tile of columns are split into: each has a slice of the workspace."""
    import ctypes

    from depthwise_conv_b200 import _lib
    n = ctypes.c_int64(0)
    _lib.call("dwb_conv2d_nhwc_bwd_weight_act8_workspace", B, H, W, C, K, ctypes.byref(n))
    return n.value // (K * K * C * 4) // -(-W // 64)


def check_wgrad(eng, B, H, W, C, K, seed):
    """Bound: 128 products of 16 terms in a chain, each truncated at 2^-23 of the sum of the magnitudes at most, are
    2^-16 of it; as much again for the terms' alignment within a product and the additions of chains and slices."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn(B, H, W, C, device="cuda", generator=g) * (0.5 + torch.rand(C, device="cuda", generator=g))
    codes, scales = eng.act8_encode((x + 0.5).half().permute(0, 3, 1, 2))
    dy = (0.3 * torch.randn(B, H, W, C, device="cuda", generator=g) + 0.05).half().permute(0, 3, 1, 2)
    dw = eng.act8_ops.conv2d_nhwc_backward_weight_act8(codes, scales, dy, K)
    again = eng.act8_ops.conv2d_nhwc_backward_weight_act8(codes, scales, dy, K)
    assert torch.equal(dw, again)
    ref, size = R.dw_weight_grad(R.act8_decode(codes, scales), dy, K)
    assert ((dw.double() - ref).abs() <= 2.0**-15 * size).all(), ((dw.double() - ref).abs() / size).max()
    assert (dw.double() - ref).norm() <= 1e-5 * ref.norm()  # the bar of the 16-bit weight gradient
    return (dw.double() - ref).norm() / ref.norm()


# a width for each tile (16, 32, 48, 64 columns, two tiles), heights that end inside a step of 2 and 4 rows
@pytest.mark.parametrize("W,H", [(13, 41), (16, 42), (30, 43), (45, 39), (61, 41), (75, 38)])
@pytest.mark.parametrize("K", [1, 3, 5, 7, 9, 11, 13, 15, 17, 23, 25, 31])
def test_weight_gradient_of_one_long_range(eng, K, W, H):
    """So many channels that a CTA takes the images from the first row to the last: the ring of dy's rows goes round, x
    changes between its two buffers, images follow each other, and a chain ends in the middle of an image."""
    B, ctas = 3, 3 if K <= 7 else 2 if K <= 15 else 1
    C = 32 * 148 * ctas
    assert wgrad_chunks(B, H, W, C, K) <= 2
    check_wgrad(eng, B, H, W, C, K, 100 * K + W)


@pytest.mark.parametrize("W,H", [(13, 43), (16, 42), (30, 23), (45, 19), (61, 15), (75, 15)])
@pytest.mark.parametrize("K", [1, 3, 5, 7, 9, 11, 13, 15, 17, 23, 25, 31])
def test_weight_gradient_of_one_chain(eng, K, W, H):
    """The same with two images that make one chain at most: the kernel for ranges that end with their chain."""
    B, ctas = 2, 3 if K <= 7 else 2 if K <= 15 else 1
    C = 32 * 148 * ctas
    rows = 1 if K > 15 else 2  # of x that a set takes
    steps = 128 // (min(-(-W // 16), 4) if W <= 64 else 3) * rows
    assert wgrad_chunks(B, H, W, C, K) <= 2 and B * H <= steps
    check_wgrad(eng, B, H, W, C, K, 100 * K + W)


@pytest.mark.parametrize("B,H,W,C,K", [(2, 200, 64, 4736, 31), (40, 3, 15, 4736, 27), (1, 300, 33, 4736, 19), (64, 14, 14, 512, 27),
                                       (70, 7, 7, 9464, 13), (9, 56, 56, 2056, 7), (2, 180, 20, 9472, 9), (17, 1, 64, 14208, 5)])
def test_weight_gradient_of_long_ranges(eng, B, H, W, C, K):
    """Tall images, many small ones and a ragged last block of channels, each range several chains or images long."""
    assert wgrad_chunks(B, H, W, C, K) * 3 <= B * -(-H // 4)
    check_wgrad(eng, B, H, W, C, K, B + H)


# ---- no checkpoint where nothing reads it ------------------------------------------------------------

def test_evaluation_makes_no_checkpoint(eng):
    """A checkpointed block under no_grad: the same bits, and no more memory than the one without checkpoints."""
    from depthwise_conv_b200.convmixer import TrainableDWBlock
    torch.manual_seed(7)
    block = TrainableDWBlock(256, 7, 32, "gelu", checkpoint8=True).cuda()
    x = torch.randn(8, 32, 32, 256, device="cuda").half().permute(0, 3, 1, 2)
    want = block(x).detach()
    peak = []
    for block.checkpoint8 in (False, True):
        with torch.no_grad():
            block(x)
            torch.cuda.synchronize()
            torch.cuda.reset_peak_memory_stats()
            before = torch.cuda.memory_allocated()
            y = block(x)
            peak.append(torch.cuda.max_memory_allocated() - before)
            assert torch.equal(y, want)
            del y
    assert peak[0] == peak[1]


def test_a_frozen_weight_keeps_no_checkpoint(eng):
    x = torch.randn(4, 28, 28, 128, device="cuda").half().permute(0, 3, 1, 2).requires_grad_()
    w = (torch.randn(9, 9, 128, device="cuda") / 9).half()
    dy = torch.randn(4, 28, 28, 128, device="cuda").half().permute(0, 3, 1, 2)
    dx, = torch.autograd.grad(eng.conv2d_nhwc_act8(x, w.clone().requires_grad_()), x, dy)
    torch.cuda.synchronize()
    before = torch.cuda.memory_allocated()
    y = eng.conv2d_nhwc_act8(x, w)
    assert torch.cuda.memory_allocated() - before <= 2 * y.numel() + 4096
    assert torch.equal(torch.autograd.grad(y, x, dy)[0], dx)


@pytest.mark.parametrize("G", [65536, 32768, 1])
@pytest.mark.parametrize("H", [3, 150])
def test_the_most_channels(eng, G, H):
    """65536 channels, a group for each of them, for two, and one for all."""
    from test_gpu_norm_act8 import check_backward, check_forward
    B, W, C = 2, 3, 65536
    g = torch.Generator(device="cuda").manual_seed(H)
    x, dy = (torch.randn(B, H, W, C, device="cuda", generator=g).half().permute(0, 3, 1, 2) for _ in range(2))
    w, b = 1 + 0.3 * torch.randn(C, device="cuda", generator=g), 0.3 * torch.randn(C, device="cuda", generator=g)
    out = eng.norm_ops.group_norm_act_forward(x, G, w, b, 1e-5, "silu", checkpoint=True)
    check_forward(out, x, G, w, b, 1e-5, "silu")
    assert all(torch.equal(p, q) for p, q in zip(out[3:], eng.act8_encode(x)))
    mean, rstd = (t.float() for t in R.stats(x, G, 1e-5))
    for saved, values in ((x, x), (out[3:], R.act8_decode(*out[3:]))):
        got = eng.norm_ops.group_norm_act_backward(dy, saved, mean, rstd, G, w, b, "silu")
        check_backward(got, dy, values, mean, rstd, G, w, b, "silu")


# ---- group norm: plans that small tensors do not take ------------------------------------------------

def norm_workspace(B, H, W, C, G, backward):
    import ctypes

    from depthwise_conv_b200 import _lib
    n = ctypes.c_int64(0)
    _lib.call("dwb_group_norm_act_workspace", B, H, W, C, G, backward, ctypes.byref(n))
    return n.value


def whole_norm(eng, B, H, W, C, G, act, dtype, seed):
    """Forward with and without a checkpoint, the gradient from the input, from the checkpoint and into dy's buffer."""
    import ctypes

    from depthwise_conv_b200 import _lib
    from test_gpu_norm_act8 import check_backward, check_forward
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = (torch.randn(B, H, W, C, device="cuda", generator=g) + 0.5 * torch.randn(C, device="cuda", generator=g))
    x = x.to(dtype).permute(0, 3, 1, 2)
    dy = (0.3 * torch.randn(B, H, W, C, device="cuda", generator=g)).to(dtype).permute(0, 3, 1, 2)
    w, b = 1 + 0.3 * torch.randn(C, device="cuda", generator=g), 0.3 * torch.randn(C, device="cuda", generator=g)
    n = eng.norm_ops
    out = n.group_norm_act_forward(x, G, w, b, 1e-5, act, checkpoint=True)
    check_forward(out, x, G, w, b, 1e-5, act)
    assert all(torch.equal(p, q) for p, q in zip(out, n.group_norm_act_forward(x, G, w, b, 1e-5, act)))
    assert all(torch.equal(p, q) for p, q in zip(out[3:], eng.act8_encode(x)))
    codes, scales = out[3:]
    mean, rstd = (t.float() for t in R.stats(x, G, 1e-5))
    ws = torch.empty(max(16, norm_workspace(B, H, W, C, G, 1)), dtype=torch.uint8, device="cuda")
    for saved, values in ((x, x), ((codes, scales), R.act8_decode(codes, scales))):
        got = n.group_norm_act_backward(dy, saved, mean, rstd, G, w, b, act)
        check_backward(got, dy, values, mean, rstd, G, w, b, act)
        place = dy.clone(memory_format=torch.preserve_format)
        source = (x.data_ptr(), None, None) if saved is x else (None, codes.data_ptr(), scales.data_ptr())
        _lib.call("dwb_group_norm_act_nhwc_bwd", place.data_ptr(), *source, mean.data_ptr(), rstd.data_ptr(), w.data_ptr(),
                  b.data_ptr(), place.data_ptr(), None, None, ws.data_ptr(), ws.numel(), B, H, W, C, G,
                  {"none": 0, "relu": 1, "gelu": 2, "silu": 3}[act], 0 if dtype == torch.float16 else 1, 2,
                  torch.cuda.current_stream().cuda_stream)
        assert torch.equal(place, got[0])
        del got, values
    assert eng.device_error() == 0


@pytest.mark.parametrize("Cg,act,dtype", [(24, "gelu", torch.float16), (12, "silu", torch.bfloat16), (3, "gelu", torch.bfloat16),
                                          (876, "silu", torch.float16), (1752, "gelu", torch.float16)])
def test_batches_in_several_groups_of_samples(eng, Cg, act, dtype):
    """The two streaming passes over three groups of samples and more, the last one shorter: launches that do both
    passes, one after another, and load before the launch before them has ended.

    A group is 160 MB of what a pass reads: of 11 samples of 35 MB 4 + 4 + 3 forward, 2 x 5 + 1 in the gradient from the
    input (twice the bytes), 3 x 3 + 2 from a checkpoint.  Groups of whole vectors, of half vectors, of 3 channels, of
    more than a tile (an entry a channel) and of several tiles."""
    B, H, W, C = 11, 100, 100, 1752
    assert B * H * W * C * 2 > 2 * (160 << 20) and norm_workspace(B, H, W, C, C // Cg, 0) > 0  # streaming has a workspace
    whole_norm(eng, B, H, W, C, C // Cg, act, dtype, Cg)


@pytest.mark.parametrize("G", [128, 64, 512, 32])
@pytest.mark.parametrize("B,H,W", [(37, 27, 29), (19, 41, 37), (10, 53, 61)])
def test_many_units_in_small_ctas(eng, B, H, W, G):
    """The forward kernel's CTAs of 128 threads, from 8 an SM on, in clusters of 2, 4 and 8 (with 512 groups of a
    channel, whose entries take more of the shared memory, 4 and 8, and CTAs of 256 threads for the largest)."""
    assert norm_workspace(B, H, W, 512, G, 0) == 0
    whole_norm(eng, B, H, W, 512, G, "gelu" if G != 64 else "silu", torch.float16 if G != 32 else torch.bfloat16, B + G)


@pytest.mark.parametrize("shape", [(1, 3, 3, 2048, 1), (1, 3, 3, 1024, 1), (2, 3, 3, 1024, 2), (1, 1, 17, 2048, 1), (1, 1, 1, 1024, 1)])
def test_clusters_with_more_ctas_than_pixels_need(eng, shape):
    """Nine pixels over four CTAs of three: the last has none, and no say in the moments."""
    whole_norm(eng, *shape, "gelu", torch.float16, shape[2])


@pytest.mark.parametrize("act", ["none", "gelu", "silu", "relu"])
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("H,C,G", [(6, 64, 4), (6, 24, 8), (30000, 64, 2), (30000, 24, 1)])
def test_a_bad_value_takes_its_whole_group(eng, act, bad, H, C, G):
    """A NaN or an infinity in x makes all of its group's outputs NaN, for every activation, and no other group's;
    the gradient of its sample's group too, and the parameters' gradients in its channels."""
    g = torch.Generator(device="cuda").manual_seed(3)
    x = torch.randn(2, H, 3, C, device="cuda", generator=g).bfloat16().permute(0, 3, 1, 2)
    c = C // 2 + 1
    x[1, c, H // 2, 1] = bad
    lo, hi = c // (C // G) * (C // G), (c // (C // G) + 1) * (C // G)
    n = eng.norm_ops
    y, mean, rstd, codes, scales = n.group_norm_act_forward(x, G, act=act, checkpoint=True)
    inside = torch.zeros(2, C, dtype=torch.bool, device="cuda")
    inside[1, lo:hi] = True
    assert torch.equal(torch.isnan(y).amax(dim=(2, 3)), inside) and torch.equal(torch.isnan(y).all(dim=3).all(dim=2), inside)
    w = torch.ones(C, device="cuda")
    dx, dw, _ = n.group_norm_act_backward(torch.ones_like(x), x, mean, rstd, G, w, None, act)
    assert torch.equal(torch.isnan(dx).all(dim=3).all(dim=2), inside) and torch.equal(torch.isnan(dx).amax(dim=(2, 3)), inside)
    assert torch.equal(torch.isnan(dw), inside[1])
    assert (scales == 255).sum() == 1 and scales[1, H // 2, 1, c // 32] == 255


def test_compiled_forward_passes(eng):
    """Under torch.compile the functions trace without a break, with and without gradients asked for."""
    g = torch.Generator(device="cuda").manual_seed(5)
    x = torch.randn(2, 9, 11, 64, device="cuda", generator=g).half().permute(0, 3, 1, 2)
    w = (torch.randn(5, 5, 64, device="cuda", generator=g) / 5).half()
    v = torch.rand(64, device="cuda", generator=g)

    def run(x, w, v):
        return eng.group_norm_act(eng.conv2d_nhwc_act8(x, w), 8, v, v, act="gelu", checkpoint=True)

    with torch.no_grad():
        assert torch.equal(torch.compile(run, fullgraph=True)(x, w, v), run(x, w, v))


@pytest.mark.parametrize("shape,G,K", [((11, 100, 100, 1752), 73, 3), ((3, 61, 45, 4736), 32, 25), ((5, 40, 30, 9472), 1, 11)])
def test_long_calls_captured_and_replayed_beside_others(eng, shape, G, K):
    """Calls of many launches, and a weight gradient whose ranges have several chains, captured once and replayed on data
    that the capture has not seen, while the same calls run eagerly on another stream: the same bits as by themselves."""
    B, H, W, C = shape
    assert wgrad_chunks(B, H, W, C, K) * 4 <= B * -(-H // 4)
    g = torch.Generator(device="cuda").manual_seed(C)
    data = [[torch.randn(B, H, W, C, device="cuda", generator=g).half().permute(0, 3, 1, 2) for _ in range(2)] for _ in range(3)]
    w, b = 1 + 0.3 * torch.randn(C, device="cuda", generator=g), 0.3 * torch.randn(C, device="cuda", generator=g)

    def run(x, dy):
        y, mean, rstd, codes, scales = eng.norm_ops.group_norm_act_forward(x, G, w, b, 1e-5, "gelu", checkpoint=True)
        first = eng.norm_ops.group_norm_act_backward(dy, x, mean, rstd, G, w, b, "gelu")
        second = eng.norm_ops.group_norm_act_backward(dy, (codes, scales), mean, rstd, G, w, b, "gelu")
        return [y, mean, rstd, codes, *first, *second, eng.act8_ops.conv2d_nhwc_backward_weight_act8(codes, scales, dy, K)]

    want = [run(*d) for d in data]
    x, dy = (t.clone(memory_format=torch.preserve_format) for t in data[0])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = run(x, dy)
    side = torch.cuda.Stream()
    for i in (1, 0, 1):
        x.copy_(data[i][0])
        dy.copy_(data[i][1])
        side.wait_stream(torch.cuda.current_stream())
        graph.replay()
        with torch.cuda.stream(side):
            got = run(*data[2])
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(held, want[i])), i
        assert all(torch.equal(p, q) for p, q in zip(got, want[2])), i
    assert eng.device_error() == 0
