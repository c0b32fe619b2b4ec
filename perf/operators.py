"""The training operators that stand around the depthwise convolution, as cases to measure.

``norm``         group norm with its activation, channels last, forward: y, mean, rstd.
``norm_grad``    its backward pass from the 16-bit input: dx, dweight, dbias.
``norm_train8``  forward that writes an 8-bit checkpoint of its input, and the backward pass that reads it.
``codec``        an activation written as an 8-bit checkpoint and read back.
``wgrad8``       the depthwise weight gradient from the 8-bit checkpoint of the convolution's input.

A checkpoint holds, for every pixel and block of 32 channels, one exponent byte E and signed codes q of 8 bits; the
value is q * 2^(E - 127), and E = 255 marks a block that held an infinity or a NaN (all of it reads back as NaN).
``own`` chooses between the plain torch form and the framework's kernels.
"""
import math

import torch

own = False

_TYPES = {"float16": torch.float16, "bfloat16": torch.bfloat16}
_BLOCK = 32
# exponents a code may have: below the lowest one the type itself has no finer step, above the highest one 127 steps
# would leave its range
_EXPONENTS = {"float16": (-24, 9), "bfloat16": (-127, 121)}


def listed():
    return [
        # batch 1 of the 7x7 stage: launch latency is all of it
        dict(name="norm_7x7x1024_b1", op="norm", B=1, H=7, W=7, C=1024, G=32, act="gelu", dtype="float16", params="float16"),
        # a ConvMixer-1536 layer at a training batch
        dict(name="norm_32x32x1536_b16", op="norm", B=16, H=32, W=32, C=1536, G=32, act="gelu", dtype="float16", params="float16"),
        # the kernel-size sweep's layer: the largest activation
        dict(name="norm_56x56x1024_b32", op="norm", B=32, H=56, W=56, C=1024, G=64, act="silu", dtype="bfloat16", params="float32"),
        # one group over the whole image (a layer norm over C, H and W): the longest sums
        dict(name="norm_32x32x768_b8_onegroup", op="norm", B=8, H=32, W=32, C=768, G=1, act="relu", dtype="float16", params="float32"),
        # odd image, groups of 9 channels that no 16-byte vector respects
        dict(name="norm_grad_23x17x72_b3", op="norm_grad", B=3, H=23, W=17, C=72, G=8, act="silu", dtype="bfloat16", params="float32"),
        dict(name="norm_grad_32x32x1536_b16", op="norm_grad", B=16, H=32, W=32, C=1536, G=32, act="gelu", dtype="float16", params="float16"),
        # the 56x56 stage in training, groups of 4 channels
        dict(name="train8_56x56x128_b64", op="norm_train8", B=64, H=56, W=56, C=128, G=32, act="gelu", dtype="float16", params="float32"),
        dict(name="train8_32x32x768_b2", op="norm_train8", B=2, H=32, W=32, C=768, G=24, act="silu", dtype="bfloat16", params="bfloat16"),
        dict(name="codec_56x56x1024_b16", op="codec", B=16, H=56, W=56, C=1024, dtype="float16"),
        # channels that end inside a block
        dict(name="codec_13x11x200_b5", op="codec", B=5, H=13, W=11, C=200, dtype="bfloat16"),
        # a ConvMixer-768 layer at a training batch, and a small image under a large kernel
        dict(name="wgrad8_32x32x768_k7_b16", op="wgrad8", B=16, H=32, W=32, C=768, K=7, dtype="float16"),
        dict(name="wgrad8_14x14x512_k27_b2", op="wgrad8", B=2, H=14, W=14, C=512, K=27, dtype="float16"),
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["norm", "norm", "norm_grad", "norm_train8", "codec", "wgrad8"])
    H, W = _log_int(rng, 1, 112), _log_int(rng, 1, 112)
    if op == "wgrad8":
        K = rng.choice(range(3, 32, 2))
        C = 8 * _log_int(rng, 1, 192)
        most = 600_000_000 // (K * K)  # values: the plain form holds each of them K * K times
        H, W = min(H, 64), min(W, 64)
        while H * W * C > most:
            C = max(8, C // 16 * 8)
        B = _log_int(rng, 1, max(1, min(64, most // (H * W * C))))
        return dict(op=op, B=B, H=H, W=W, C=C, K=K, dtype="float16")
    C = 8 * _log_int(rng, 1, 256)
    values = 2 ** rng.uniform(13, 25.5)
    B = max(1, min(64, int(values / (H * W * C))))
    dtype = rng.choice(["float16", "bfloat16"])
    if op == "codec":
        return dict(op=op, B=B, H=H, W=W, C=C, dtype=dtype)
    # in a group of very few values the input gradient cancels to nothing but rounding
    G = rng.choice([g for g in range(1, C + 1) if C % g == 0 and (g == 1 or H * W * C // g >= 32)])
    # the backward pass at a ReLU's corner has two right answers: it is drawn for the forward pass alone
    act = rng.choice(["none", "relu", "gelu", "silu"] if op == "norm" else ["none", "gelu", "silu"])
    return dict(op=op, B=B, H=H, W=W, C=C, G=G, act=act, dtype=dtype, params=rng.choice([dtype, "float32"]))


def work(case):
    n = case["B"] * case["H"] * case["W"] * case["C"]
    saved = n + case["B"] * case["H"] * case["W"] * -(-case["C"] // _BLOCK)  # codes and exponent bytes
    op = case["op"]
    if op == "norm":
        return {"bytes": 4 * n, "flops": 12 * n}
    if op == "norm_grad":
        return {"bytes": 6 * n, "flops": 25 * n}
    if op == "norm_train8":
        return {"bytes": 4 * n + saved + saved + 4 * n, "flops": 45 * n}
    if op == "codec":
        return {"bytes": 4 * n + 2 * saved, "flops": 4 * n}
    taps = 1
    for size in (case["H"], case["W"]):  # pairs of an output and an input position that a tap joins
        taps *= sum(max(0, size - abs(k - case["K"] // 2)) for k in range(case["K"]))
    return {"bytes": 2 * n + saved + 4 * case["K"] ** 2 * case["C"], "flops": 2 * taps * case["B"] * case["C"]}


# ---- inputs --------------------------------------------------------------------------------------


def _nchw(t):
    """A [B, H, W, C] tensor as the channels_last [B, C, H, W] view that the framework takes."""
    return t.permute(0, 3, 1, 2)


def _activation(g, case):
    """What a convolution puts out: each channel with its own offset and spread, a few pixels far out."""
    B, H, W, C = case["B"], case["H"], case["W"], case["C"]
    x = torch.randn(B, H, W, C, device="cuda", generator=g)
    x = x * (0.5 + torch.rand(C, device="cuda", generator=g)) + 0.5 * torch.randn(C, device="cuda", generator=g)
    far = torch.rand(B, H, W, 1, device="cuda", generator=g) < 0.01
    return torch.where(far, x * 8, x).to(_TYPES[case["dtype"]])


def _gradient(g, case):
    shape = (case["B"], case["H"], case["W"], case["C"])
    return (0.1 * torch.randn(shape, device="cuda", generator=g)).to(_TYPES[case["dtype"]])


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    op = case["op"]
    s = dict(case=dict(case), x=_nchw(_activation(g, case)))
    if op == "codec":
        # rectified activations: whole blocks of zeros, and blocks of very small values
        x = s["x"].permute(0, 2, 3, 1)
        dead = torch.rand(x.shape[:3] + (1,), device="cuda", generator=g)
        x = torch.where(dead < 0.05, torch.zeros_like(x), torch.where(dead < 0.1, x * 1e-4, x.clamp(min=-0.25)))
        s["x"] = _nchw(x.contiguous())
    elif op == "wgrad8":
        s["codes"], s["scales"] = _encode(s["x"])
        del s["x"]
        s["dy"] = _nchw(_gradient(g, case))
    else:
        params = torch.float32 if case["params"] == "float32" else _TYPES[case["params"]]
        s["weight"] = (1 + 0.2 * torch.randn(case["C"], device="cuda", generator=g)).to(params)
        s["bias"] = (0.2 * torch.randn(case["C"], device="cuda", generator=g)).to(params)
        if op != "norm":
            s["dy"] = _nchw(_gradient(g, case))
        if op == "norm_grad":
            _, s["mean"], s["rstd"] = _norm(s["x"], s["weight"], s["bias"], case)
    return s


# ---- plain forms ---------------------------------------------------------------------------------


def _grouped(x, G):
    """[B, C, H, W] channels_last -> [B, P, G, C/G] in 32 bits."""
    B, C, H, W = x.shape
    return x.permute(0, 2, 3, 1).reshape(B, H * W, G, C // G).float()


def _ungrouped(v, like, dtype):
    B, C, H, W = like.shape
    return _nchw(v.reshape(B, H, W, C).to(dtype))


def _activate(u, act):
    if act == "relu":
        return u.clamp(min=0)
    if act == "gelu":
        return 0.5 * u * torch.erfc(u * -math.sqrt(0.5))
    if act == "silu":
        return u / (1 + torch.exp(-u))
    return u


def _slope(u, act):
    if act == "relu":
        return (u > 0).float()
    if act == "gelu":
        return 0.5 * torch.erfc(u * -math.sqrt(0.5)) + u * torch.exp(-0.5 * u * u) / math.sqrt(2 * math.pi)
    if act == "silu":
        s = 1 / (1 + torch.exp(-u))
        return s * (1 + u * (1 - s))
    return torch.ones_like(u)


_EPS = 1e-5


def _norm(x, weight, bias, case):
    G = case["G"]
    v = _grouped(x, G)
    mean = v.mean(dim=(1, 3), keepdim=True)
    centred = v - mean
    rstd = 1 / torch.sqrt((centred * centred).mean(dim=(1, 3), keepdim=True) + _EPS)
    u = centred * rstd * weight.float().view(G, -1) + bias.float().view(G, -1)
    y = _ungrouped(_activate(u, case["act"]), x, x.dtype)
    return y, mean.reshape(-1, G), rstd.reshape(-1, G)


def _norm_grad(dy, x, mean, rstd, weight, bias, case):
    G = case["G"]
    w, b = weight.float().view(G, -1), bias.float().view(G, -1)
    r = rstd.view(-1, 1, G, 1)
    xh = (_grouped(x, G) - mean.view(-1, 1, G, 1)) * r
    g = _grouped(dy, G) * _slope(xh * w + b, case["act"])
    gw = g * w
    m1 = gw.mean(dim=(1, 3), keepdim=True)
    m2 = (gw * xh).mean(dim=(1, 3), keepdim=True)
    dx = _ungrouped(r * (gw - m1 - xh * m2), dy, dy.dtype)
    return dx, (g * xh).sum(dim=(0, 1)).reshape(-1).to(weight.dtype), g.sum(dim=(0, 1)).reshape(-1).to(bias.dtype)


def _power_of_two(e):
    """2^e in 64 bits from its bits: exact, where pow and exp2 may be off in the last place."""
    return ((e.long() + 1023) << 52).view(torch.float64)


def _encode(x):
    """Codes [B, C, H, W] (channels_last) and exponent bytes [B, H, W, ceil(C / 32)] of a 16-bit activation."""
    low, high = _EXPONENTS[str(x.dtype).replace("torch.", "")]
    B, C, H, W = x.shape
    blocks = -(-C // _BLOCK)
    v = torch.zeros(B, H, W, blocks * _BLOCK, device=x.device)
    v[..., :C] = x.permute(0, 2, 3, 1)
    v = v.view(B, H, W, blocks, _BLOCK)
    top = v.abs().amax(dim=-1)
    m, e = torch.frexp(top)  # top = m 2^e, 0.5 <= m < 1
    e = e - 7 + (m > 127 / 128).int()
    e = torch.where(top > 0, e, low).clamp(low, high)
    fine = torch.isfinite(v).all(dim=-1)
    codes = torch.round(v.double() * _power_of_two(-e)[..., None]).clamp(-127, 127)
    codes = torch.where(fine[..., None], codes, 0).to(torch.int8)
    scales = torch.where(fine, e + 127, 255).to(torch.uint8)
    return _nchw(codes.view(B, H, W, -1)[..., :C].contiguous()), scales


def _decode(codes, scales, dtype):
    q = codes.permute(0, 2, 3, 1)
    step = torch.where(scales == 255, math.nan, _power_of_two(scales.int() - 127))
    v = q.double() * step.repeat_interleave(_BLOCK, dim=-1)[..., : q.shape[-1]]
    return _nchw(v.to(dtype))


def _wgrad8(codes, scales, dy, K):
    """dw[kh, kw, c]: every value times every value that a tap joins it with, summed."""
    B, C, H, W = dy.shape
    p = K // 2
    x = torch.zeros(B, H + 2 * p, W + 2 * p, C, device=dy.device)
    x[:, p : p + H, p : p + W] = _decode(codes, scales, torch.float32).permute(0, 2, 3, 1)
    windows = x.unfold(1, H, 1).unfold(2, W, 1)  # [B, K, K, C, H, W]: a view, no copy
    return (windows * dy.float()[:, None, None]).sum(dim=(0, 4, 5))


def run(state):
    s, case = state, state["case"]
    op = case["op"]
    if own:
        return _run_own(s, case, op)
    if op == "norm":
        return _norm(s["x"], s["weight"], s["bias"], case)
    if op == "norm_grad":
        return _norm_grad(s["dy"], s["x"], s["mean"], s["rstd"], s["weight"], s["bias"], case)
    if op == "norm_train8":
        y, mean, rstd = _norm(s["x"], s["weight"], s["bias"], case)
        kept = _decode(*_encode(s["x"]), torch.float32)
        return (y, mean, rstd) + _norm_grad(s["dy"], kept, mean, rstd, s["weight"], s["bias"], case)
    if op == "codec":
        return _decode(*_encode(s["x"]), s["x"].dtype)
    return _wgrad8(s["codes"], s["scales"], s["dy"], case["K"])


def _run_own(s, case, op):
    from depthwise_conv_b200 import act8_ops, norm_ops

    if op == "norm":
        return norm_ops.group_norm_act_forward(s["x"], case["G"], s["weight"], s["bias"], _EPS, case["act"])
    if op == "norm_grad":
        return norm_ops.group_norm_act_backward(s["dy"], s["x"], s["mean"], s["rstd"], case["G"], s["weight"], s["bias"], case["act"])
    if op == "norm_train8":
        y, mean, rstd, codes, scales = norm_ops.group_norm_act_forward(
            s["x"], case["G"], s["weight"], s["bias"], _EPS, case["act"], checkpoint=True)
        return (y, mean, rstd) + tuple(norm_ops.group_norm_act_backward(
            s["dy"], (codes, scales), mean, rstd, case["G"], s["weight"], s["bias"], case["act"]))
    if op == "codec":
        return act8_ops.act8_decode(*act8_ops.act8_encode(s["x"]), s["x"].dtype)
    return act8_ops.conv2d_nhwc_backward_weight_act8(s["codes"], s["scales"], s["dy"], case["K"])


# ---- the definitions in 64 bits ------------------------------------------------------------------


def _exact_kept(x):
    """The values that a checkpoint of x stands for, from its definition: the smallest step of which 127 reach."""
    low, high = _EXPONENTS[str(x.dtype).replace("torch.", "")]
    v = x.double()
    C = v.shape[1]
    kept = torch.empty_like(v)
    steps = torch.tensor([2.0**e for e in range(low, high + 1)], dtype=torch.float64, device=v.device)
    for at in range(0, C, _BLOCK):
        part = v[:, at : at + _BLOCK]
        top = part.abs().amax(dim=1, keepdim=True)
        step = steps[torch.searchsorted(127 * steps, top.contiguous()).clamp(max=len(steps) - 1)]
        kept[:, at : at + _BLOCK] = torch.round(part / step).clamp(-127, 127) * step
    return kept


def _exact_parts(x, mean, rstd, weight, bias, G):
    B, C, H, W = x.shape
    spread = lambda t: t.repeat_interleave(C // G, dim=1)[:, :, None, None]  # noqa: E731
    xh = (x - spread(mean)) * spread(rstd)
    return xh, xh * weight.double()[:, None, None] + bias.double()[:, None, None]


def _exact_cdf(u, act):
    return torch.special.ndtr(u) if act == "gelu" else torch.sigmoid(u)


def _exact_norm(x, weight, bias, case):
    G, act = case["G"], case["act"]
    flat = x.double().contiguous().view(x.shape[0], G, -1)
    var, mean = torch.var_mean(flat, dim=2, correction=0)
    rstd = (var + _EPS).rsqrt()
    _, u = _exact_parts(x.double(), mean, rstd, weight, bias, G)
    y = u if act == "none" else torch.maximum(u, torch.zeros_like(u)) if act == "relu" else u * _exact_cdf(u, act)
    return y, mean, rstd


def _exact_norm_grad(dy, x, mean, rstd, weight, bias, case):
    G, act = case["G"], case["act"]
    B, C, H, W = dy.shape
    n = H * W * (C // G)
    xh, u = _exact_parts(x.double(), mean.double(), rstd.double(), weight, bias, G)
    if act == "none":
        slope = torch.ones_like(u)
    elif act == "relu":
        slope = (u > 0).double()
    elif act == "gelu":
        slope = _exact_cdf(u, act) + u * torch.exp(-u * u / 2) / math.sqrt(2 * math.pi)
    else:
        slope = _exact_cdf(u, act) * (1 + u * _exact_cdf(-u, act))
    g = dy.double() * slope
    sum_g, sum_gx = g.sum(dim=(2, 3)), (g * xh).sum(dim=(2, 3))  # [B, C]
    w = weight.double()
    back = lambda t: ((t * w).view(B, G, -1).sum(dim=2) / n).repeat_interleave(C // G, dim=1)[:, :, None, None]  # noqa: E731
    dx = rstd.double().repeat_interleave(C // G, dim=1)[:, :, None, None] * (g * w[:, None, None] - back(sum_g) - xh * back(sum_gx))
    return dx, sum_gx.sum(dim=0), sum_g.sum(dim=0)


def _exact_wgrad8(s, case):
    B, C, H, W = s["dy"].shape
    K, p = case["K"], case["K"] // 2
    powers = torch.tensor([2.0 ** (e - 127) for e in range(256)], dtype=torch.float64, device=s["dy"].device)
    step = powers[s["scales"].long()].permute(0, 3, 1, 2).repeat_interleave(_BLOCK, dim=1)[:, :C]
    x = torch.nn.functional.pad(s["codes"].double() * step, (p, p, p, p)).contiguous()
    dy = s["dy"].double().contiguous()
    dw = torch.empty(K, K, C, dtype=torch.float64, device=dy.device)
    for kh in range(K):
        for kw in range(K):
            dw[kh, kw] = (x[:, :, kh : kh + H, kw : kw + W] * dy).sum(dim=(0, 2, 3))
    return dw


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "norm":
        return _exact_norm(s["x"], s["weight"], s["bias"], case)
    if op == "norm_grad":
        return _exact_norm_grad(s["dy"], s["x"], s["mean"], s["rstd"], s["weight"], s["bias"], case)
    if op == "norm_train8":
        y, mean, rstd = _exact_norm(s["x"], s["weight"], s["bias"], case)
        return (y, mean, rstd) + _exact_norm_grad(s["dy"], _exact_kept(s["x"]), mean, rstd, s["weight"], s["bias"], case)
    if op == "codec":
        return _exact_kept(s["x"])
    return _exact_wgrad8(s, case)
