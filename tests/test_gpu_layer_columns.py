"""Products of few tokens and many columns to fp32: more columns than eight
splits hold in accumulators of 1024 (bf16) or 4096 (e4m3).

Positive operands, where what the tensor core cuts off in its additions adds up.
An accumulator takes at most 64 additions of bf16 (16 pieces of 64 columns, four
each) or 128 of e4m3, each cutting off less than 2^-23 of what is there so far,
half the end's on average over a sum that grows evenly, to which 5% are given
for its unevenness; adding up at most 20 of them takes 20 * 2^-24."""
import pytest
import torch

from canvas_attn import layer
from test_gpu_layer import F8, TYPE, gated_case, linear_case

pytestmark = pytest.mark.gpu
ADDITIONS = {"bf16": 64, "e4m3": 128}


def one_sign(kind):
    return ADDITIONS[kind] / 2 * 1.05 * 2.0 ** -23 + 20 * 2.0 ** -24


@pytest.mark.parametrize("n", [1, 16, 17, 40, 64])
@pytest.mark.parametrize("cols", [32784, 262144])
def test_linear(n, cols):
    torch.manual_seed(n)
    x = torch.rand(n, cols, device="cuda").to(F8)
    w = torch.rand(200, cols, device="cuda").to(F8)
    o = torch.empty(n, 200, device="cuda")
    layer.linear_q8(x, None, w, None, o)
    y = x.double() @ w.double().T
    assert float(((o.double() - y).abs() / y).max()) < one_sign("e4m3")


@pytest.mark.parametrize("n", [1, 16, 17, 40, 64, 100])
@pytest.mark.parametrize("kind,cols", [("bf16", 8256), ("bf16", 18944), ("bf16", 65536),
                                       ("e4m3", 32784), ("e4m3", 262144)])
def test_gated(n, kind, cols):
    # Both factors are off by one_sign at most; the gates are above 100, where
    # silu(g) is g to less than 2^-24, and the three products round once each.
    torch.manual_seed(n)
    x = torch.rand(n, cols, device="cuda").to(TYPE[kind])
    g, u = (torch.rand(200, cols, device="cuda").to(x.dtype) for _ in range(2))
    o = torch.empty(n, 200, device="cuda")
    layer.gated_linear(x, g, u, o)
    a, b = x.double() @ g.double().T, x.double() @ u.double().T
    assert float(a.min()) > 100
    assert float(((o.double() - a * b).abs() / (a * b)).max()) < 2 * one_sign(kind) + 6 * 2.0 ** -24


@pytest.mark.parametrize("n", [1, 30, 64])
def test_both_signs(n):
    linear_case(n, 260, 33008, bias=True, res=True, out="f32", pad=1)
    for cols in (12288, 18944):
        gated_case(n, 300, cols, kind="bf16", act="gelu", out="f32", scale_w=0.01)
    gated_case(n, 140, 40000, kind="e4m3", out="f32", scale_w=0.01)
    gated_case(n, 140, 12288, kind="bf16")


def test_in_a_graph_and_on_two_streams_at_once():
    torch.manual_seed(5)
    x = torch.randn(50, 12288, device="cuda").to(torch.bfloat16)
    g, u = ((torch.randn(2000, 12288, device="cuda") * 0.01).to(x.dtype) for _ in range(2))
    y = torch.randn(40, 33008, device="cuda").to(F8)
    w = torch.randn(1500, 33008, device="cuda").to(F8)
    want = torch.empty(50, 2000, device="cuda"), torch.empty(40, 1500, device="cuda")
    layer.gated_linear(x, g, u, want[0])
    layer.linear_q8(y, None, w, None, want[1])
    got = [torch.zeros_like(o) for o in want]
    a = layer.make_gated_linear_args(x, g, u, got[0])
    b = layer.make_linear_q8_args(y, None, w, None, got[1])
    st = torch.cuda.Stream()
    torch.cuda.synchronize()
    gr = torch.cuda.CUDAGraph()
    with torch.cuda.graph(gr, stream=st):
        layer.gated_linear_args(a, st)
        layer.linear_q8_args(b, st)
    for _ in range(3):
        got[0].zero_()
        got[1].zero_()
        gr.replay()
    torch.cuda.synchronize()
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    for o in got:
        o.zero_()
    torch.cuda.synchronize()
    for i in range(10):
        layer.gated_linear_args(a, st if i % 2 else None)
        layer.linear_q8_args(b, None if i % 2 else st)
    torch.cuda.synchronize()
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
