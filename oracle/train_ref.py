"""Plain float64 restatements of the training operators (TEST INFRASTRUCTURE ONLY).

Group normalisation with an activation and its gradients, the 8-bit activation
checkpoint, and the depthwise weight gradient, each written from its definition
in torch float64 (any device).  Tensors are [B, C, H, W].
"""
from __future__ import annotations

import math

import torch

BLOCK = 32
EXPONENTS = {torch.float16: (-24, 9), torch.bfloat16: (-127, 121)}


def act_and_slope(u: torch.Tensor, act: str):
    if act == "relu":
        return torch.where(u < 0, torch.zeros_like(u), u), (u > 0).double()
    if act == "gelu":
        cdf = 0.5 * torch.special.erfc(-u / math.sqrt(2.0))
        return u * cdf, cdf + u * torch.exp(-0.5 * u * u) / math.sqrt(2 * math.pi)
    if act == "silu":
        s = torch.sigmoid(u)
        return u * s, s * (1 + u * torch.sigmoid(-u))
    return u, torch.ones_like(u)


def stats(x: torch.Tensor, G: int, eps: float):
    v = x.double().reshape(x.shape[0], G, -1)
    mean = v.mean(dim=2)
    var = ((v - mean[..., None]) ** 2).mean(dim=2)
    return mean, 1 / torch.sqrt(var + eps)


def _per_channel(t: torch.Tensor, C: int):
    return t.double().repeat_interleave(C // t.shape[1], dim=1)[:, :, None, None]


def _vec(p, C, otherwise, device):
    return (torch.full((C,), otherwise, dtype=torch.float64, device=device) if p is None else p.double())[:, None, None]


def normalised(x, mean, rstd):
    C = x.shape[1]
    return (x.double() - _per_channel(mean, C)) * _per_channel(rstd, C)


def group_norm_act(x, G, weight=None, bias=None, eps=1e-5, act="none"):
    """(y, mean, rstd, u)."""
    C = x.shape[1]
    mean, rstd = stats(x, G, eps)
    u = normalised(x, mean, rstd) * _vec(weight, C, 1.0, x.device) + _vec(bias, C, 0.0, x.device)
    return act_and_slope(u, act)[0], mean, rstd, u


def group_norm_act_grad(dy, x, mean, rstd, G, weight=None, bias=None, act="none"):
    """dict of dx, dweight, dbias, and the sizes of what is added up (for error bounds)."""
    B, C, H, W = dy.shape
    n = H * W * (C // G)
    w, b = _vec(weight, C, 1.0, dy.device), _vec(bias, C, 0.0, dy.device)
    xh = normalised(x, mean, rstd)
    g = dy.double() * act_and_slope(xh * w + b, act)[1]

    def group_mean(t):
        return _per_channel(t.reshape(B, G, -1).sum(dim=2) / n, C)

    r = _per_channel(rstd, C)
    dx = r * (g * w - group_mean(g * w) - xh * group_mean(g * w * xh))
    # magnitudes: each term of dx with its sums taken over absolute values (|dy| for |g|: |act'| < 1.13)
    a = 1.13 * dy.double().abs()
    size = r * (a * w.abs() + group_mean(a * w.abs()) + xh.abs() * group_mean(a * w.abs() * xh.abs()))
    return dict(dx=dx, dweight=(g * xh).sum(dim=(0, 2, 3)), dbias=g.sum(dim=(0, 2, 3)), dx_size=size,
                dweight_size=(a * xh.abs()).sum(dim=(0, 2, 3)), dbias_size=a.sum(dim=(0, 2, 3)), u=xh * w + b)


def act8_encode(x: torch.Tensor):
    """(codes int8 like x, exponent bytes uint8 [B, H, W, ceil(C / 32)]): every exponent tried in turn."""
    low, high = EXPONENTS[x.dtype]
    B, C, H, W = x.shape
    n = -(-C // BLOCK)
    v = torch.zeros(B, H, W, n * BLOCK, dtype=torch.float64, device=x.device)
    v[..., :C] = x.permute(0, 2, 3, 1)
    v = v.reshape(B, H, W, n, BLOCK)
    fine = torch.isfinite(v).all(dim=4)
    v = torch.where(fine[..., None], v, 0.0)
    amax = v.abs().amax(dim=4)
    exponent = torch.full(amax.shape, high, dtype=torch.int64, device=x.device)
    for e in range(high, low - 1, -1):
        exponent = torch.where(amax <= 127 * 2.0**e, e, exponent)
    step = torch.tensor([2.0**e for e in range(low, high + 1)], dtype=torch.float64, device=x.device)[exponent - low]
    q = torch.round(v / step[..., None]).clamp(-127, 127).to(torch.int8)
    codes = q.reshape(B, H, W, -1)[..., :C].permute(0, 3, 1, 2).contiguous(memory_format=torch.channels_last)
    return codes, torch.where(fine, exponent + 127, 255).to(torch.uint8)


def act8_decode(codes: torch.Tensor, scales: torch.Tensor):
    C = codes.shape[1]
    table = torch.tensor([2.0 ** (E - 127) for E in range(255)] + [math.nan], dtype=torch.float64, device=codes.device)
    step = table[scales.long()].repeat_interleave(BLOCK, dim=3)[..., :C].permute(0, 3, 1, 2)
    return codes.double() * step


def dw_weight_grad(x: torch.Tensor, dy: torch.Tensor, K: int):
    """(dw, sum of |terms|), both [K, K, C]."""
    B, C, H, W = dy.shape
    p = K // 2
    xp = torch.nn.functional.pad(x.double(), (p, p, p, p)).contiguous()
    g = dy.double().contiguous()
    dw = torch.empty(K, K, C, dtype=torch.float64, device=dy.device)
    size = torch.empty_like(dw)
    for kh in range(K):
        for kw in range(K):
            t = g * xp[:, :, kh:kh + H, kw:kw + W]
            dw[kh, kw] = t.sum(dim=(0, 2, 3))
            size[kh, kw] = t.abs().sum(dim=(0, 2, 3))
    return dw, size
