"""Products whose scales lie far apart: results in range, of a sum that is out of
it with the larger scale alone."""
import pytest
import torch

from canvas_attn import layer
from layer_helpers import F8

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("sa,sw", [(2.0 ** 120, 2.0 ** -20), (2.0 ** -20, 2.0 ** 120),
                                   (2.0 ** 110, 2.0 ** -64), (2.0 ** -64, 2.0 ** -30),
                                   (-2.0 ** 120, 2.0 ** -24), (1.0, 1.0)])
@pytest.mark.parametrize("n,rows", [(1, 300), (20, 300), (64, 300), (300, 6000)])
def test_scales_far_apart(n, rows, sa, sw):
    # Whole numbers in steps of 32: sums of 64 products below 2^24 are exact in
    # fp32, and scales are powers of two, so that results are, too.
    g = torch.Generator().manual_seed(n)
    x = (torch.randint(-7, 8, (n, 64), generator=g) * 32.0).to(F8).cuda()
    w = (torch.randint(-7, 8, (rows, 64), generator=g) * 32.0).to(F8).cuda()
    xs, ws = torch.full((n,), sa, device="cuda"), torch.full((rows,), sw, device="cuda")
    b = torch.zeros(rows, device="cuda")
    want = (x.double() @ w.double().T) * (sa * sw)
    for bias in (None, b):
        o = torch.empty(n, rows, device="cuda")
        layer.linear_q8(x, xs, w, ws, o, bias=bias)
        assert torch.equal(o.double(), want)


@pytest.mark.parametrize("n,rows", [(1, 300), (20, 300), (64, 300), (300, 6000)])
def test_gated_scales_far_apart(n, rows):
    # Gates of 0 and of 100 and more (silu(g) is g to 2^-24 from there on), and the
    # other factor small, of scales 2^110 and 2^-110 or 2^-64: the quotient is off
    # by 2 units of 2^-23 and two roundings remain.
    g = torch.Generator().manual_seed(n)
    x = (torch.randint(0, 8, (n, 64), generator=g) * 32.0).to(F8).cuda()
    w = (torch.randint(0, 8, (rows, 64), generator=g) * 32.0).to(F8).cuda()
    xs = torch.full((n,), 2.0 ** 110, device="cuda")
    gs = torch.full((rows,), 2.0 ** -110, device="cuda")
    us = torch.full((rows,), 2.0 ** -64, device="cuda")
    o = torch.empty(n, rows, device="cuda")
    layer.gated_linear(x, w, w, o, act_scale=xs, gate_scale=gs, up_scale=us)
    a = x.double() @ w.double().T
    assert float(a[a > 0].min()) > 100
    want = a * a * 2.0 ** 46
    assert ((o.double() - want).abs() <= 8 * 2.0 ** -24 * want).all()


@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_scales_that_are_not_numbers(bad):
    x, w = torch.ones(30, 32).to(F8).cuda(), torch.ones(200, 32).to(F8).cuda()
    xs, ws = torch.ones(30, device="cuda"), torch.ones(200, device="cuda")
    xs[3], ws[7] = bad, bad
    o = torch.empty(30, 200, device="cuda")
    layer.linear_q8(x, xs, w, ws, o)
    want = 32 * xs.unsqueeze(1) * ws
    assert torch.equal(o.nan_to_num(), want.nan_to_num())
    assert torch.equal(torch.isnan(o), torch.isnan(want))
