"""64-bit references of the 8-bit tensors, the linear layers on them and LayerNorm's training passes, from their
definitions (include/fvsr_lcsa.h), in torch on the tensors' own device."""
from __future__ import annotations

import math

import torch


def held(x, square=False):
    """(values in 64 bits, codes) that x (rows, cols) stands for in the 8-bit form: the smallest code >= 0 whose
    448 * 2^(code - 127) bounds the block, then e4m3 rounding by its step 2^(max(floor(log2 |v|), -6) - 3)."""
    x = x.double()
    rows, cols = x.shape
    bh = 128 if square else 1
    kb, rb = -(-cols // 128), -(-rows // bh)
    t = torch.zeros((rb * bh, kb * 128), dtype=torch.float64, device=x.device)
    t[:rows, :cols] = x
    t = t.view(rb, bh, kb, 128)
    top = t.abs().amax(dim=(1, 3), keepdim=True)
    bad = ~torch.isfinite(top)
    mant, exp = torch.frexp(torch.where(bad, torch.ones_like(top), top) / 448.0)  # top / 448 = mant * 2^exp, mant in [.5, 1)
    e = torch.where(mant == 0.5, exp - 1, exp).clamp(min=-127)
    e = torch.where(top == 0, torch.full_like(e, -127), e).double()
    v = t / torch.exp2(e)
    step = torch.exp2(torch.floor(torch.log2(v.abs().clamp(min=2.0 ** -30))).clamp(min=-6) - 3)
    out = torch.where(bad, torch.full_like(v, math.nan), torch.round(v / step) * step * torch.exp2(e))
    codes = torch.where(bad, torch.full_like(e, 255), e + 127).expand(rb, bh, kb, 1).reshape(rb * bh, kb)[:rows]
    return out.reshape(rb * bh, kb * 128)[:rows, :cols], codes.to(torch.uint8)


def linear(x, w, bias=None, epilogue=0, gate=None, resid=None):
    """(out, magnitude of what its sum adds up) in 64 bits of x (M, K), w (N, K) given by their 64-bit values."""
    y, size = x @ w.t(), x.abs() @ w.abs().t()
    if bias is not None:
        y, size = y + bias.double(), size + bias.double().abs()
    if epilogue == 1:
        y = y / (1.0 + torch.exp(-2.0 * math.sqrt(2.0 / math.pi) * (y + 0.044715 * y ** 3)))
    elif epilogue == 2:
        y = resid.double() + gate.double() * y
    return y, size


def norm(x, weight=None, bias=None, shift=None, scale=None, eps=1e-6):
    x = x.double()
    mean = x.mean(dim=1)
    rstd = 1.0 / torch.sqrt(((x - mean[:, None]) ** 2).mean(dim=1) + eps)
    y = (x - mean[:, None]) * rstd[:, None]
    if weight is not None:
        y = y * weight.double() + bias.double()
    if scale is not None:
        y = y * (1.0 + scale.double()) + shift.double()
    return y, mean, rstd


def norm_backward(dy, x, mean, rstd, weight=None, bias=None, scale=None):
    dy, x, mean, rstd = dy.double(), x.double(), mean.double()[:, None], rstd.double()[:, None]
    n = (x - mean) * rstd
    one = torch.ones(dy.shape[1], dtype=torch.float64, device=dy.device)
    w = weight.double() if weight is not None else one
    b = bias.double() if bias is not None else 0 * one
    s1 = 1.0 + scale.double() if scale is not None else one
    g = dy * s1 * w
    a, s = (dy * n).sum(0), dy.sum(0)
    dx = rstd * (g - g.mean(1, keepdim=True) - n * (g * n).mean(1, keepdim=True))
    return {"dx": dx, "dweight": s1 * a if weight is not None else None, "dbias": s1 * s if weight is not None else None,
            "dscale": w * a + b * s if scale is not None else None, "dshift": s if scale is not None else None}
