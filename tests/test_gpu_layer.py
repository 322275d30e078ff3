"""ca_rms_norm, ca_linear_q8 and ca_gated_linear on the GPU against their
formulas in 64 bits.

Tolerances. A product of `cols` terms in fp32 is off by at most cols * 2^-23 of
the sum of its terms' magnitudes (each addition rounds or truncates once, by
2^-23 of a partial sum no larger than that); scales, bias and residual add four
roundings of 2^-24; the output type rounds once, by eps / 2. The activation's
slope is at most 1.13, and its exponential is off by 2 + 1.16 |x| units of
2^-23 (below 1e-5 relative for the arguments here).
The norm: a sum of squares of positive terms is off by at most (32 + 10) * 2^-24
relative (32 in a thread, a tree of ten), half of that in its root, and four
roundings more: 25 * 2^-24 < 2^-19 relative."""
import pytest
import torch

from canvas_attn import layer
from layer_helpers import (F8, activate_ref, norm_ref, operand, product_ref, quantise_ref)

pytestmark = pytest.mark.gpu
BF, F32 = torch.bfloat16, torch.float32
TYPE = {"bf16": BF, "f32": F32, "e4m3": F8}


def half(t):
    return torch.finfo(t).eps / 2


def gen(seed):
    return torch.Generator().manual_seed(seed)


# ------------------------------------------------------------------ the norm
def norm_case(rows, cols, x="bf16", res=None, out="bf16", gain=True, norm=True, seed=0, pad=0,
              eps=1e-5):
    g = gen(seed + rows * 7 + cols)
    xx = (torch.randn(rows, cols, generator=g) * 2).to(TYPE[x])
    rr = None if res is None else (torch.randn(rows, cols, generator=g) * 3).to(TYPE[res])
    w = torch.rand(cols, generator=g) + 0.5 if gain else None

    def dev(t):
        if t is None:
            return None
        d = torch.full((rows, cols + pad), 7.0, device="cuda").to(t.dtype)
        d[:, :cols] = t.cuda()
        return d[:, :cols]

    dx, dr = dev(xx), dev(rr)
    ds = None if rr is None else torch.zeros_like(dr)
    buf = torch.zeros(rows, cols + pad, device="cuda").to(TYPE[out])
    do, sc = buf[:, :cols], torch.zeros(rows, device="cuda") if out == "e4m3" else None
    layer.rms_norm(dx, do, w=None if w is None else w.cuda(), eps=eps, norm=norm, residual=dr,
                   sum_out=ds, out_scale=sc)
    torch.cuda.synchronize()
    if pad:
        assert (buf[:, cols:].float() == 0).all(), "columns behind the last one"
    s, y = norm_ref(xx, residual=rr, w=w, eps=eps, norm=norm)
    if rr is not None:
        assert torch.equal(ds.cpu(), s)
    rel = 2.0 ** -19
    if out != "e4m3":
        err = (do.cpu().double() - y).abs()
        assert (err <= (rel + half(TYPE[out])) * y.abs() + 1e-37).all(), float(err.max())
        return
    q, scale = quantise_ref(y)
    sc = sc.cpu().double()
    # A scale may differ where the largest magnitude is within `rel` of a border.
    near = torch.stack([quantise_ref(y * f)[1] for f in (1 - rel, 1 + rel)])
    assert ((sc == near[0]) | (sc == near[1])).all()
    got = do.cpu().float().double() * sc.unsqueeze(1)
    # Half a step of the value's binade; below 2^-6 of the scale steps are 2^-9.
    tol = (half(F8) + 2 * rel) * y.abs() + 2.0 ** -10 * sc.unsqueeze(1)
    assert ((got - y).abs() <= tol).all()
    if not norm and not gain and res is None:
        assert torch.equal(sc, scale) and torch.equal(do.cpu().float().double(), q)


@pytest.mark.parametrize("out", ["bf16", "f32", "e4m3"])
@pytest.mark.parametrize("res", [None, "bf16", "f32"])
@pytest.mark.parametrize("x", ["bf16", "f32"])
def test_norm_types(x, res, out):
    norm_case(5, 4096, x=x, res=res, out=out)
    norm_case(3, 1001, x=x, res=res, out=out)


@pytest.mark.parametrize("cols", [1, 7, 8, 100, 1024, 1032, 2048, 3584, 4104, 8192, 8200, 16384,
                                  16392, 18944, 20480, 20488, 32767, 32768, 40000])
@pytest.mark.parametrize("rows", [1, 700])
def test_norm_widths(rows, cols):
    norm_case(rows, cols, res="bf16", out="e4m3")


@pytest.mark.parametrize("pad", [1, 4, 8])
def test_norm_strides(pad):
    for out in ("bf16", "f32", "e4m3"):
        norm_case(9, 520, x="f32", res="f32", out=out, pad=pad)
        norm_case(9, 520, x="bf16", res="bf16", out=out, pad=pad)


def test_norm_without_gain_and_quantisation_alone():
    norm_case(64, 3584, gain=False, out="bf16")
    for cols in (3584, 77, 12288):
        norm_case(64, cols, gain=False, norm=False, out="e4m3")
        norm_case(64, cols, x="f32", gain=False, norm=False, out="e4m3")
    norm_case(64, 256, res="f32", gain=False, norm=False, out="f32")


def test_norm_in_place():
    g = gen(3)
    x, r = torch.randn(40, 512, generator=g).to(BF), torch.randn(40, 512, generator=g).to(BF)
    s, y = norm_ref(x, residual=r, eps=1e-6)
    dx, dr = x.cuda(), r.cuda()
    layer.rms_norm(dx, dx, residual=dr)  # the stream updated in place, the norm over x
    assert torch.equal(dr.cpu(), s)
    assert ((dx.cpu().double() - y).abs() <= (2.0 ** -19 + half(BF)) * y.abs()).all()


def test_norm_of_unusual_values():
    x = torch.randn(6, 300, generator=gen(4))
    x[0] = 0
    x[1, 3] = float("inf")
    x[2, 4] = float("nan")
    x[3] = 1e-30
    x[4] *= 1e18
    sc = torch.zeros(6, device="cuda")
    out = torch.zeros(6, 300, device="cuda").to(F8)
    layer.quantize_rows(x.cuda(), out, sc)
    q, s = quantise_ref(x.double())
    got = out.cpu().float().double()
    assert torch.equal(sc.cpu().double(), s)
    assert torch.equal(torch.isnan(got), torch.isnan(q))
    assert torch.equal(got.nan_to_num(), q.nan_to_num())
    y = torch.zeros(6, 300, device="cuda")
    layer.rms_norm(x.cuda(), y, eps=1e-6)
    y = y.cpu()
    assert (y[0] == 0).all() and torch.isnan(y[2]).all()
    assert torch.isnan(y[1, 3]) and (y[1, :3] == 0).all()


def test_quantisation_of_rows_with_infinities():
    # Every other row has infinities, at widths of one and of several warps.
    for cols in (64, 1000, 4096, 9000):
        x = torch.randn(50, cols, generator=gen(cols))
        x[::2, 5] = float("inf")
        x[::4, cols - 1] = -float("inf")
        x[8] = float("inf")
        sc = torch.zeros(50, device="cuda")
        out = torch.zeros(50, cols, device="cuda").to(F8)
        layer.quantize_rows(x.cuda(), out, sc)
        q, s = quantise_ref(x.double())
        assert torch.equal(sc.cpu().double(), s)
        assert torch.equal(out.cpu().float().double(), q)


def test_norm_of_no_rows():
    x = torch.zeros(0, 64, device="cuda")
    layer.rms_norm(x, torch.zeros(0, 64, device="cuda"))


# -------------------------------------------------------------- the products
def linear_case(n, rows, cols, bias=False, res=False, out="bf16", seed=0, scales=True, pad=0):
    g = gen(seed + n + rows * 3 + cols)
    x, xs = operand(g, n, cols, "e4m3")
    w, ws = operand(g, rows, cols, "e4m3")
    if not scales:
        xs = ws = None
    b = torch.randn(rows, generator=g) if bias else None
    t = TYPE[out]
    r = (torch.randn(n, rows, generator=g) * 2).to(t) if res else None
    buf = torch.full((n + 1, rows + pad), 5.0, device="cuda", dtype=t)
    o = buf[:n, :rows]
    act = torch.zeros(n, cols + 16 * pad, dtype=F8, device="cuda")[:, :cols]
    act.view(torch.uint8).copy_(x.view(torch.uint8).cuda())
    c = lambda v: None if v is None else v.cuda()  # noqa: E731
    st = torch.zeros(1, dtype=torch.int32, device="cuda")
    layer.linear_q8(act, c(xs), w.cuda(), c(ws), o, bias=c(b), residual=c(r), status=st)
    torch.cuda.synchronize()
    assert int(st) == 0
    assert (buf[n] == 5).all() and (buf[:, rows:] == 5).all(), "outside the output"
    y, mag = product_ref(x.cuda(), c(xs), w.cuda(), c(ws))
    big = mag.clone()
    if b is not None:
        y, big = y + b.cuda().double(), big + b.cuda().abs()
    if r is not None:
        y, big = y + r.cuda().double(), big + r.cuda().double().abs()
    tol = cols * 2.0 ** -23 * mag + 2.0 ** -22 * big + half(t) * y.abs()
    err = (o.double() - y).abs()
    assert (err <= tol).all(), float((err / tol).max())
    # Far inside that: errors of single roundings do not add up in one direction.
    assert float(err.norm() / y.norm()) < half(t) + 2e-6


@pytest.mark.parametrize("n", [1, 2, 15, 16, 17, 31, 33, 64, 65, 128, 129, 200, 257, 511])
def test_linear_tokens(n):
    linear_case(n, 384, 512, res=True)


@pytest.mark.parametrize("rows", [1, 2, 127, 128, 129, 255, 257, 1000])
@pytest.mark.parametrize("n", [1, 40, 300])
def test_linear_rows(n, rows):
    linear_case(n, rows, 272, bias=True)


@pytest.mark.parametrize("cols", [16, 32, 112, 128, 144, 1024, 4096, 4112, 18944])
@pytest.mark.parametrize("n", [1, 48, 300])
def test_linear_columns(n, cols):
    linear_case(n, 260, cols, out="f32")


@pytest.mark.parametrize("n", [3, 300])
def test_linear_types_and_strides(n):
    for out in ("bf16", "f32"):
        for bias in (False, True):
            for res in (False, True):
                linear_case(n, 264, 512, bias=bias, res=res, out=out, pad=3)
    linear_case(n, 264, 512, scales=False)


@pytest.mark.parametrize("n,rows,cols", [(1, 4096, 4096), (8, 18944, 1024), (443, 4608, 3584),
                                         (2048, 2304, 4096), (1000, 4100, 2048)])
def test_linear_sizes(n, rows, cols):
    linear_case(n, rows, cols, res=True)


def test_linear_residual_in_place():
    g = gen(21)
    x, xs = operand(g, 70, 256, "e4m3")
    w, ws = operand(g, 256, 256, "e4m3")
    r = torch.randn(70, 256, generator=g).to(BF).cuda()
    a, b = r.clone(), torch.empty_like(r)
    layer.linear_q8(x.cuda(), xs.cuda(), w.cuda(), ws.cuda(), b, residual=r)
    layer.linear_q8(x.cuda(), xs.cuda(), w.cuda(), ws.cuda(), a, residual=a)
    torch.cuda.synchronize()
    assert torch.equal(a, b)


def gated_case(n, rows, cols, kind="e4m3", act="silu", out="bf16", seed=0, pad=0, scale_w=0.05):
    g = gen(seed + n + rows * 3 + cols)
    x, xs = operand(g, n, cols, kind)
    ops = []
    for _ in range(2):
        w, ws = operand(g, rows, cols, kind)
        if kind == "bf16":
            w = (w.float() * scale_w).to(BF)
        else:
            ws = ws * scale_w
        ops.append((w, ws))
    (wg, gs), (wu, us) = ops
    t = TYPE[out]
    buf = torch.full((n + 1, rows + pad), 5.0, device="cuda", dtype=t)
    o = buf[:n, :rows]
    c = lambda v: None if v is None else v.cuda()  # noqa: E731
    st = torch.zeros(1, dtype=torch.int32, device="cuda")
    layer.gated_linear(c(x), c(wg), c(wu), o, activation=act, act_scale=c(xs), gate_scale=c(gs),
                       up_scale=c(us), status=st)
    torch.cuda.synchronize()
    assert int(st) == 0
    assert (buf[n] == 5).all() and (buf[:, rows:] == 5).all(), "outside the output"
    gv, gm = product_ref(c(x), c(xs), c(wg), c(gs))
    uv, um = product_ref(c(x), c(xs), c(wu), c(us))
    f = activate_ref(gv, act)
    y = f * uv
    e = cols * 2.0 ** -23 + 2.0 ** -22
    tol = (1.13 * e * gm * (uv.abs() + e * um) + e * um * f.abs()
           + (1e-5 + half(t)) * y.abs())
    err = (o.double() - y).abs()
    assert (err <= tol + 1e-30).all(), float((err / (tol + 1e-30)).max())
    assert float(err.norm() / y.norm()) < half(t) + 4e-6


@pytest.mark.parametrize("n", [1, 2, 16, 17, 33, 64, 65, 128, 130, 257, 500])
@pytest.mark.parametrize("kind", ["bf16", "e4m3"])
def test_gated_tokens(n, kind):
    gated_case(n, 384, 512, kind=kind)


@pytest.mark.parametrize("rows,cols", [(1, 16), (127, 144), (129, 1024), (1000, 80), (64, 4112),
                                       (2000, 2048)])
@pytest.mark.parametrize("n", [1, 40, 300])
@pytest.mark.parametrize("kind", ["bf16", "e4m3"])
def test_gated_shapes(n, rows, cols, kind):
    gated_case(n, rows, cols, kind=kind, act="gelu", out="f32", pad=1)


@pytest.mark.parametrize("act", ["silu", "gelu"])
@pytest.mark.parametrize("kind", ["bf16", "e4m3"])
def test_gated_wide_range(kind, act):
    # Gates of several hundred: the exponential runs to 0 and to infinity.
    gated_case(20, 300, 512, kind=kind, act=act, scale_w=8.0)
    gated_case(200, 300, 512, kind=kind, act=act, scale_w=8.0)


@pytest.mark.parametrize("n,rows,cols,kind", [(1, 18944, 3584, "e4m3"), (512, 2304, 4096, "bf16"),
                                              (1500, 1300, 4096, "e4m3")])
def test_gated_sizes(n, rows, cols, kind):
    gated_case(n, rows, cols, kind=kind)


# fp32 outputs of positive operands, where what the tensor core cuts off in its
# additions is cut off in one direction. An accumulator takes at most 128
# additions (32 pieces of 128 columns, four each), each cutting off less than
# 2^-23 of what is there so far, half the end's on average over a sum that grows
# evenly, to which 5% are given for its unevenness: 128 / 2 * 1.05 * 2^-23 =
# 8.0e-6 of an entry; joining up to ten of them and rounding takes 10 * 2^-24 =
# 6e-7.
ONE_SIGN = 67.2 * 2.0 ** -23 + 10 * 2.0 ** -24


@pytest.mark.parametrize("n,rows", [(1, 9600), (16, 640), (40, 9600), (100, 640), (600, 4000),
                                    (2048, 4096)])
@pytest.mark.parametrize("cols", [4112, 18944])
def test_linear_sums_of_one_sign(n, rows, cols):
    torch.manual_seed(n + cols)
    x = torch.rand(n, cols, device="cuda").to(F8)
    w = torch.rand(rows, cols, device="cuda").to(F8)
    o = torch.empty(n, rows, device="cuda")
    layer.linear_q8(x, None, w, None, o)
    y = x.double() @ w.double().T
    assert float(((o.double() - y).abs() / y).max()) < ONE_SIGN


@pytest.mark.parametrize("n", [1, 100, 300, 1100])
def test_linear_long_to_fp32(n):
    linear_case(n, 1300, 4368, bias=True, res=True, out="f32", pad=1)


@pytest.mark.parametrize("kind", ["bf16", "e4m3"])
@pytest.mark.parametrize("n", [16, 100, 2048])
def test_gated_sums_of_one_sign(n, kind):
    # Both factors are off by ONE_SIGN at most; the gates are above 100, where
    # silu(g) is g to less than 2^-24, and the three products round once each.
    torch.manual_seed(n)
    x = torch.rand(n, 8208, device="cuda").to(TYPE.get(kind, F8))
    g, u = (torch.rand(2000, 8208, device="cuda").to(x.dtype) for _ in range(2))
    o = torch.empty(n, 2000, device="cuda")
    layer.gated_linear(x, g, u, o)
    a, b = x.double() @ g.double().T, x.double() @ u.double().T
    assert float(a.min()) > 100
    assert float(((o.double() - a * b).abs() / (a * b)).max()) < 2 * ONE_SIGN + 6 * 2.0 ** -24


def test_products_in_a_graph_on_another_stream_twice():
    g = gen(31)
    x, xs = (t.cuda() for t in operand(g, 100, 1024, "e4m3"))
    w, ws = (t.cuda() for t in operand(g, 512, 1024, "e4m3"))
    u, us = (t.cuda() for t in operand(g, 512, 1024, "e4m3"))
    want = [torch.empty(100, 512, dtype=BF, device="cuda") for _ in range(2)]
    layer.linear_q8(x, xs, w, ws, want[0])
    layer.gated_linear(x, w, u, want[1], act_scale=xs, gate_scale=ws, up_scale=us)
    torch.cuda.synchronize()
    st = torch.cuda.Stream()
    got = [torch.empty(100, 512, dtype=BF, device="cuda") for _ in range(2)]
    a = layer.make_linear_q8_args(x, xs, w, ws, got[0])
    b = layer.make_gated_linear_args(x, w, u, got[1], act_scale=xs, gate_scale=ws, up_scale=us)
    gr = torch.cuda.CUDAGraph()
    with torch.cuda.graph(gr, stream=st):
        layer.linear_q8_args(a, st)
        layer.gated_linear_args(b, st)
    for _ in range(3):
        got[0].zero_()
        got[1].zero_()
        gr.replay()
    torch.cuda.synchronize()
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    # Calls of two streams at once.
    for i in range(10):
        layer.linear_q8_args(a, st if i % 2 else None)
        layer.gated_linear_args(b, None if i % 2 else st)
    torch.cuda.synchronize()
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
