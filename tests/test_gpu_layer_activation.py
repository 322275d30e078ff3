"""The gate's activation in fp32 outputs of ca_gated_linear, over gates that the
products give exactly: one column of 1 against the gates themselves.

Tolerances. silu: the exponential is off by 2^-22 (4 units of 2^-24) and two
roundings of its correction, its sum with 1 and the product with the other factor
round by a unit each, the quotient is off by 2 units of 2^-23: 12 * 2^-24
relative. gelu: x = 2 sqrt(2/pi) (g + 0.044715 g^3) takes at most seven roundings
of 2^-24 more, which change e^-x by |x| times as much and the result by e^-x /
(1 + e^-x) of that. Below 1e-36 the exponential runs to infinity."""
import math

import pytest
import torch

from canvas_attn import layer
from layer_helpers import F8, activate_ref

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


@pytest.mark.parametrize("kind", ["bf16", "e4m3"])
@pytest.mark.parametrize("n", [1, 20, 40, 200])
@pytest.mark.parametrize("act", ["silu", "gelu"])
def test_activation_of_exact_gates(act, n, kind):
    rows = 6000
    g = torch.linspace(-86, 86, rows) if act == "silu" else torch.linspace(-9.8, 9.8, rows)
    x = torch.zeros(n, 16)
    x[:, 0] = 1
    w, u = torch.zeros(rows, 16), torch.zeros(rows, 16)
    u[:, 0] = 1
    o = torch.empty(n, rows, device="cuda")
    if kind == "bf16":
        w[:, 0] = g
        w = w.to(torch.bfloat16)
        g = w[:, 0].float()
        layer.gated_linear(x.to(torch.bfloat16).cuda(), w.cuda(), u.to(torch.bfloat16).cuda(), o,
                           activation=act)
    else:
        w[:, 0] = 1
        layer.gated_linear(x.to(F8).cuda(), w.to(F8).cuda(), u.to(F8).cuda(), o, activation=act,
                           gate_scale=g.cuda())
    g = g.double()
    y = activate_ref(g, act)
    tol = 12 * U * y.abs()
    if act == "gelu":
        # 1 + tanh has no bits left at -9 in any type; g / (1 + e^-x) has.
        t = 2 * math.sqrt(2 / math.pi) * (g + 0.044715 * g ** 3)
        y = g / (1 + torch.exp(-t))
        tol = (12 + 7 * t.abs() * torch.sigmoid(-t)) * U * y.abs()
    err = (o.cpu().double() - y).abs()
    assert (err <= tol + 1e-36).all(), float((err / (tol + 1e-36)).max())


def test_unusual_gates():
    g = torch.tensor([0.0, -0.0, 1e-30, -1e-30, 100.0, -100.0, 3e38, -3e38, 1e15, -1e15])
    x, w = torch.ones(3, 16).to(F8), torch.zeros(10, 16)
    x[:, 1:] = 0
    w[:, 0] = 1
    for act in ("silu", "gelu"):
        o = torch.empty(3, 10, device="cuda")
        layer.gated_linear(x.cuda(), w.to(F8).cuda(), w.to(F8).cuda(), o, activation=act,
                           gate_scale=g.cuda())
        y = torch.where(g > 1, g, torch.where(g < -1, 0.0, g / 2))
        assert ((o.cpu() - y).abs() <= 2.0 ** -22 * y.abs() + 1e-36).all()
