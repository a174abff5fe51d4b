"""Rows in 8-bit integers and their products, plainly and in 64 bits, on any device."""
import math

import torch


def quantised(u):
    """Codes (int64) and scales (float64) of rows given in 64 bits: 127 u / max |u| to the nearest, ties to even."""
    u = u.double()
    top = u.abs().amax(-1, keepdim=True) if u.shape[-1] else torch.zeros(*u.shape[:-1], 1, dtype=torch.float64, device=u.device)
    fine = torch.isfinite(top)
    codes = torch.where(fine & (top > 0), (127 * u / top).round(), torch.zeros_like(u))
    return codes.to(torch.int64), torch.where(fine, top / 127, torch.full_like(top, math.nan)).squeeze(-1)


def normed(t, weight):
    """What the codes of normed rows are made of: the stored sum times the weight, rounded to 32 bits once."""
    return t.float() * weight


def product(x_codes, x_scales, w_codes, w_scales, activation=None):
    """[rows, channels] (or half as many: gate and up in turns of eight) in 64 bits."""
    y = x_codes.double() @ w_codes.double().t() * x_scales.double()[:, None] * w_scales.double()
    if activation is None:
        return y
    pairs = y.view(y.shape[0], -1, 2, 8)
    g, u = pairs[:, :, 0].reshape(y.shape[0], -1), pairs[:, :, 1].reshape(y.shape[0], -1)
    if activation == "silu":
        return g * torch.sigmoid(g) * u, g, u
    return 0.5 * g * (1 + torch.tanh(math.sqrt(2 / math.pi) * (g + 0.044715 * g ** 3))) * u, g, u


def padded(rows, width, device="cuda", extra=0):
    """Room for codes whose rows begin at multiples of 16 bytes, full of a code of its own."""
    return torch.full((rows, -(-width // 16) * 16 + extra), 77, dtype=torch.int8, device=device)
