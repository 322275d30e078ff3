"""Plain restatements in 64 bits of ca_rms_norm, ca_linear_q8 and
ca_gated_linear for their tests."""
from __future__ import annotations

import math

import torch

from kv8_helpers import e4m3_round, need_exp

F8 = torch.float8_e4m3fn


def quantise_ref(y):
    """(e4m3 values, scales) of fp64 rows, by the rule of ca_rms_norm."""
    fin = torch.where(torch.isfinite(y), y.abs(), 0.0).amax(dim=1)
    s = torch.tensor([2.0 ** need_exp(float(a)) for a in fin], dtype=torch.float64)
    q = e4m3_round((y / s.unsqueeze(1)).clamp(-448, 448))
    return torch.where(torch.isnan(y), math.nan, q), s


def norm_ref(x, *, residual=None, w=None, eps=1e-6, norm=True):
    """(sum in the residual's type or None, y in 64 bits)."""
    h = x.double()
    s = None
    if residual is not None:
        s = (x.float() + residual.float()).to(residual.dtype)
        h = s.double()
    if norm:
        h = h / torch.sqrt((h * h).mean(dim=1, keepdim=True) + eps)
    if w is not None:
        h = h * w.double()
    return s, h


def operand(g, rows, cols, kind, loud=0.4):
    """A [rows, cols] operand and its fp32 scales (None for bf16)."""
    x = torch.randn(rows, cols, generator=g) * torch.exp(loud * torch.randn(1, cols, generator=g))
    if kind == "bf16":
        return x.to(torch.bfloat16), None
    s = torch.tensor([2.0 ** need_exp(float(a)) for a in x.abs().amax(dim=1)])
    return (x / s.unsqueeze(1)).to(F8), s


def values(x, s):
    return x.double() if s is None else x.float().double() * s.double().unsqueeze(1)


def product_ref(x, xs, w, ws):
    """The product in 64 bits, and the sum of its terms' magnitudes."""
    a, b = values(x, xs), values(w, ws)
    return a @ b.T, a.abs() @ b.abs().T


def activate_ref(g, kind):
    if kind == "silu":
        return g * torch.sigmoid(g)
    return 0.5 * g * (1 + torch.tanh(math.sqrt(2 / math.pi) * (g + 0.044715 * g ** 3)))
