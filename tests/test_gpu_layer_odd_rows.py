"""ca_rms_norm of rows whose width or stride is no multiple of 8, at widths that
take 4, 8 and 20 elements a thread (tolerances: test_gpu_layer.py)."""
import pytest

from test_gpu_layer import norm_case

import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("cols", [4095, 4097, 5001, 8191, 8193, 12289, 18943, 20479])
@pytest.mark.parametrize("x,res", [("bf16", None), ("bf16", "bf16"), ("bf16", "f32"),
                                   ("f32", None), ("f32", "bf16"), ("f32", "f32")])
@pytest.mark.parametrize("out", ["bf16", "f32", "e4m3"])
def test_odd_widths(out, x, res, cols):
    norm_case(6, cols, x=x, res=res, out=out)


@pytest.mark.parametrize("cols", [4097, 8193, 20479])
def test_odd_widths_of_many_rows(cols):
    # More rows than CTAs, so that each takes several.
    norm_case(1000, cols, res="bf16", out="e4m3")
    norm_case(700, cols, x="f32", out="bf16", pad=3)


@pytest.mark.parametrize("cols,pad", [(4096, 1), (8192, 3), (12288, 5), (20480, 1)])
def test_even_widths_of_odd_strides(cols, pad):
    for out in ("bf16", "f32", "e4m3"):
        norm_case(7, cols, x="bf16", res="f32", out=out, pad=pad)


@pytest.mark.parametrize("cols", [4097, 9001, 20479])
def test_quantisation_alone(cols):
    norm_case(9, cols, gain=False, norm=False, out="e4m3")
    norm_case(9, cols, x="f32", gain=False, norm=False, out="e4m3")


@pytest.mark.parametrize("cols", [5001, 9001])
def test_odd_rows_with_infinities(cols):
    from canvas_attn import layer
    from layer_helpers import F8, quantise_ref
    x = torch.randn(50, cols, generator=torch.Generator().manual_seed(cols))
    x[::2, 5] = float("inf")
    x[1::4, cols - 1] = float("nan")
    x[8] = -float("inf")
    sc = torch.zeros(50, device="cuda")
    out = torch.zeros(50, cols, device="cuda").to(F8)
    layer.quantize_rows(x.cuda(), out, sc)
    q, s = quantise_ref(x.double())
    assert torch.equal(sc.cpu().double(), s)
    assert torch.equal(out.cpu().float().double().nan_to_num(9), q.nan_to_num(9))
