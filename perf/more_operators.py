"""What a denoising step does between the attention's output and the tokens it
commits, in cases that can be measured.

  norm    residual addition and root-mean-square norm of rows, to bf16, fp32 or
          e4m3 with a scale for each row (a power of two: the smallest with
          amax <= 448 * scale); without the norm, the quantisation alone
  linear  act . W^T of e4m3 rows with their scales, with bias and residual
  gated   activation(x . Wg^T) * (x . Wu^T), operands in bf16 or in e4m3
  sample  a token for each candidate row of logits, with temperature, top-k,
          top-p and min-p, from a given random number

`own` false: plain torch. `own` true: the calls of canvas_attn.layer and
canvas_attn.denoise.
"""
import math
import os
import sys

import torch

own = False

E4M3 = torch.float8_e4m3fn
TYPES = {"bf16": torch.bfloat16, "f32": torch.float32, "e4m3": E4M3}
EPS = 1e-5


def listed():
    return [
        # One token of a 4096-wide model between attention and feed-forward: latency.
        dict(name="norm token 4096 q8", op="norm", rows=1, cols=4096, x="bf16", res="bf16", out="e4m3", norm=True),
        # A ragged batch's active rows of a 3584-wide model whose residual stream is kept in fp32.
        dict(name="norm canvas 1111x3584", op="norm", rows=1111, cols=3584, x="bf16", res="f32", out="bf16", norm=True),
        # Every row of a first full forward, for an 8-bit product behind it.
        dict(name="norm full 16384x4096 q8", op="norm", rows=16384, cols=4096, x="bf16", res="bf16", out="e4m3", norm=True),
        # The output projection of one token, added to the residual stream: the weights' bytes count.
        dict(name="linear token 4096x4096", op="linear", n=1, rows=4096, cols=4096, bias=False, res=True, out="bf16"),
        # Fused Q, K, V projection with bias (28 + 2 * 4 heads of 128) of a ragged batch of canvases.
        dict(name="linear canvas 443 3584-4608", op="linear", n=443, rows=4608, cols=3584, bias=True, res=False, out="bf16"),
        # The down projection of two full canvases.
        dict(name="linear full 8192 12288-4096", op="linear", n=8192, rows=4096, cols=12288, bias=False, res=True, out="bf16"),
        # Feed-forward of one token, 8-bit weights of a 3584-wide model.
        dict(name="gated token 3584-18944 q8", op="gated", n=1, rows=18944, cols=3584, kind="e4m3", act="silu", out="bf16"),
        # Sixteen sequences of 32 canvas rows, bf16 weights.
        dict(name="gated canvas 512 4096-12288", op="gated", n=512, rows=12288, cols=4096, kind="bf16", act="silu", out="bf16"),
        # Feed-forward of two full canvases in 8 bits.
        dict(name="gated full 8192 q8", op="gated", n=8192, rows=12288, cols=4096, kind="e4m3", act="gelu", out="bf16"),
        # The last masked position of one canvas, plain temperature.
        dict(name="sample one 32000", op="sample", cand=1, vocab=32000, kind="f32", temperature=0.7, top_k=0, top_p=1.0, min_p=0.0),
        # A block of 32 masked positions with every filter.
        dict(name="sample block 32x126464", op="sample", cand=32, vocab=126464, kind="f32", temperature=1.0, top_k=50, top_p=0.95, min_p=0.02),
        # Sixteen sequences of 32 candidates, a nucleus of bf16 logits.
        dict(name="sample batch 512x151936", op="sample", cand=512, vocab=151936, kind="bf16", temperature=0.8, top_k=0, top_p=0.9, min_p=0.0),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["norm", "linear", "gated", "sample"])
    if op == "norm":
        cols = rng.choice([_log(rng, 100, 18944), 8 * _log(rng, 32, 2368), 128 * _log(rng, 4, 148)])
        rows = _log(rng, 1, max(2, min(16384, (1 << 26) // cols)))
        return dict(op=op, rows=rows, cols=cols, x=rng.choice(["bf16", "bf16", "f32"]), res=rng.choice(["none", "bf16", "f32"]),
                    out=rng.choice(["bf16", "f32", "e4m3", "e4m3"]), norm=rng.random() < 0.8)
    if op == "sample":
        vocab = _log(rng, 1000, 262144)
        cand = _log(rng, 1, max(2, min(512, (1 << 26) // vocab)))
        return dict(op=op, cand=cand, vocab=vocab, kind=rng.choice(["f32", "f32", "bf16"]), temperature=rng.choice([0.0, 0.3, 0.7, 1.0, 1.5]),
                    top_k=rng.choice([0, 0, _log(rng, 1, 1000)]), top_p=rng.choice([1.0, 0.5, 0.9, 0.95]), min_p=rng.choice([0.0, 0.0, 0.05]))
    cols, rows = 16 * _log(rng, 16, 1184), _log(rng, 128, 18944)
    n = rng.choice([_log(rng, 1, 64), _log(rng, 32, 8192)])
    while n > 1 and n * rows * cols > 8192 * 4096 * 12288 // 2:
        n //= 2
    if op == "linear":
        return dict(op=op, n=n, rows=rows, cols=cols, bias=rng.random() < 0.5, res=rng.random() < 0.5, out=rng.choice(["bf16", "bf16", "f32"]))
    return dict(op=op, n=n, rows=rows, cols=cols, kind=rng.choice(["bf16", "e4m3"]), act=rng.choice(["silu", "gelu"]), out=rng.choice(["bf16", "bf16", "f32"]))


def _scale_of(amax):
    """2^k of the smallest k in [-64, 120] with amax <= 448 * 2^k (448 = 0.875 * 2^9)."""
    m, e = torch.frexp(amax)
    k = torch.where(amax > 0, torch.where(m <= 0.875, e - 9, e - 8).clamp(-64, 120), -64)
    return ((k.to(torch.int32) + 127) << 23).view(torch.float32)


def _quantised(x):
    """e4m3 rows and their scales."""
    s = _scale_of(x.abs().amax(dim=1))
    return (x / s.unsqueeze(1)).to(E4M3), s


def _loud(g, rows, cols, dev, spread):
    """Rows with a few loud channels and rows of different loudness, as a trained model's are."""
    x = torch.randn((rows, cols), generator=g, device=dev)
    x *= torch.exp(spread * torch.randn((1, cols), generator=g, device=dev))
    return x.mul_(torch.exp(0.3 * torch.randn((rows, 1), generator=g, device=dev)))


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(int(seed))
    s, op = dict(case=case), case["op"]
    new = lambda shape, kind: torch.empty(shape, dtype=TYPES[kind], device=dev)  # noqa: E731
    if op == "norm":
        shape = (case["rows"], case["cols"])
        s["x"] = _loud(g, *shape, dev, 0.5).to(TYPES[case["x"]])
        s["w"] = 0.5 + torch.rand(case["cols"], generator=g, device=dev)
        if case["res"] != "none":
            s["res"] = (4 * _loud(g, *shape, dev, 0.5)).to(TYPES[case["res"]])
            s["sum"] = new(shape, case["res"])
        s["out"] = new(shape, case["out"])
        s["scale"] = new((case["rows"],), "f32") if case["out"] == "e4m3" else None
        return s
    if op == "sample":
        n, v = case["cand"], case["vocab"]
        # Rows of different sharpness, with a few tokens that stand out. Two rows more than candidates: those of committed positions.
        x = torch.randn((n + 2, v), generator=g, device=dev) * (1 + 2 * torch.rand((n + 2, 1), generator=g, device=dev))
        at = torch.randint(0, v, (n + 2, 20), generator=g, device=dev)
        x.scatter_add_(1, at, 12 * torch.rand((n + 2, 20), generator=g, device=dev))
        s["logits"] = x.to(TYPES[case["kind"]])
        s["rows"] = torch.randperm(n + 2, generator=g, device=dev)[:n].sort().values.to(torch.int32)
        s["u"] = torch.rand(n, generator=g, device=dev)
        s["suppress"] = torch.tensor([0, 5, v // 2], dtype=torch.int32, device=dev)
        s["token"], s["prob"] = torch.empty(n, dtype=torch.int32, device=dev), new((n,), "f32")
        return s
    n, rows, cols = case["n"], case["rows"], case["cols"]
    kind = case.get("kind", "e4m3")
    for name in ("w",) if op == "linear" else ("w", "up"):
        w = _loud(g, rows, cols, dev, 0.2).mul_(cols ** -0.5)
        s[name], s[name + "_scale"] = _quantised(w) if kind == "e4m3" else (w.to(TYPES[kind]), None)
        del w
    x = _loud(g, n, cols, dev, 0.5)
    s["x"], s["x_scale"] = _quantised(x) if kind == "e4m3" else (x.to(TYPES[kind]), None)
    s["bias"] = torch.randn(rows, generator=g, device=dev) if case.get("bias") else None
    s["res"] = (2 * torch.randn((n, rows), generator=g, device=dev)).to(TYPES[case["out"]]) if case.get("res") else None
    s["out"] = new((n, rows), case["out"])
    return s


def _norm_plain(s):
    c = s["case"]
    h = s["x"].float()
    if c["res"] != "none":
        s["sum"].copy_(h + s["res"].float())
        h = s["sum"].float()
    if c["norm"]:
        h = h * torch.rsqrt(h.square().mean(dim=1, keepdim=True) + EPS) * s["w"]
    first = [s["sum"]] if c["res"] != "none" else []
    if c["out"] == "e4m3":
        return first + list(_quantised(h))
    return first + [h.to(TYPES[c["out"]])]


def _times(x, x_scale, w, w_scale):
    y = x.float() @ w.float().T
    return y if x_scale is None else y.mul_(x_scale.unsqueeze(1)).mul_(w_scale)


def _linear_plain(s):
    y = _times(s["x"], s["x_scale"], s["w"], s["w_scale"])
    if s["bias"] is not None:
        y = y + s["bias"]
    if s["res"] is not None:
        y = y + s["res"].float()
    return y.to(s["out"].dtype)


def _gated_plain(s):
    g = _times(s["x"], s["x_scale"], s["w"], s["w_scale"])
    u = _times(s["x"], s["x_scale"], s["up"], s["up_scale"])
    if s["case"]["act"] == "silu":
        g = g / (1 + torch.exp(-g))
    else:
        g = 0.5 * g * (1 + torch.tanh(math.sqrt(2 / math.pi) * (g + 0.044715 * g * g * g)))
    return (g * u).to(s["out"].dtype)


def _sample_plain(s):
    """In 64 bits: the drawn number falls next to borders between tokens."""
    c = s["case"]
    x = s["logits"][s["rows"].long()].float()
    x[:, s["suppress"].long()] = -math.inf
    x[:, c["vocab"] - 1] = -math.inf  # the mask token
    top = x.amax(dim=1, keepdim=True)
    if c["temperature"] == 0:
        token = x.argmax(dim=1)
    else:
        w = torch.exp((x.double() - top) / c["temperature"])
        order = x.sort(dim=1, descending=True, stable=True).indices
        ws = w.gather(1, order)
        if c["top_k"] > 0:
            ws[:, c["top_k"]:] = 0
        before = ws.cumsum(dim=1) - ws
        keep = (ws > 0) & (ws >= c["min_p"])
        if c["top_p"] < 1:
            keep &= before < c["top_p"] * ws.sum(dim=1, keepdim=True)
        keep[:, 0] = True
        w *= torch.zeros_like(keep).scatter_(1, order, keep)
        upto = w.cumsum(dim=1)
        token = (upto > s["u"].double().unsqueeze(1) * upto[:, -1:]).int().argmax(dim=1)
    prob = torch.exp(x.gather(1, token.unsqueeze(1)) - top) / torch.exp(x - top).sum(dim=1, keepdim=True)
    return [token.to(torch.int32), prob.squeeze(1)]


def _plan(s):
    """What a user's program builds once for buffers that it keeps: the argument block of its call."""
    root = os.path.join(os.getcwd(), "diffuse-rs_b200")
    if root not in sys.path:
        sys.path.insert(0, root)
    from canvas_attn import denoise, layer
    c = s["case"]
    if c["op"] == "norm":
        a = layer.make_rms_norm_args(s["x"], s["out"], w=s["w"] if c["norm"] else None, eps=EPS, norm=c["norm"], residual=s.get("res"), sum_out=s.get("sum"),
                                     out_scale=s["scale"])
        return layer.rms_norm_args, a, ([s["sum"]] if c["res"] != "none" else []) + [s["out"]] + ([s["scale"]] if c["out"] == "e4m3" else [])
    if c["op"] == "linear":
        a = layer.make_linear_q8_args(s["x"], s["x_scale"], s["w"], s["w_scale"], s["out"], bias=s["bias"], residual=s["res"])
        return layer.linear_q8_args, a, s["out"]
    if c["op"] == "gated":
        a = layer.make_gated_linear_args(s["x"], s["w"], s["up"], s["out"], act_scale=s["x_scale"], gate_scale=s["w_scale"], up_scale=s["up_scale"],
                                         activation=c["act"])
        return layer.gated_linear_args, a, s["out"]
    a = denoise.make_sample_args(s["logits"], s["rows"], s["u"], s["token"], s["prob"], n_vocab=c["vocab"], temperature=c["temperature"], top_k=c["top_k"],
                                 top_p=c["top_p"], min_p=c["min_p"], mask_id=c["vocab"] - 1, suppress=s["suppress"])
    return denoise.sample_args, a, [s["token"], s["prob"]]


def run(s):
    if not own:
        return {"norm": _norm_plain, "linear": _linear_plain, "gated": _gated_plain, "sample": _sample_plain}[s["case"]["op"]](s)
    if "plan" not in s:
        s["plan"] = _plan(s)
    call, a, out = s["plan"]
    call(a)
    return out


def work(case):
    size = {"bf16": 2, "f32": 4, "e4m3": 1, "none": 0}
    if case["op"] == "norm":
        n = case["rows"] * case["cols"]
        return {"bytes": n * (size[case["x"]] + 2 * size[case["res"]] + size[case["out"]]) + 4 * case["cols"] * case["norm"] + 4 * case["rows"] * (case["out"] == "e4m3"), "flops": 6 * n}
    if case["op"] == "sample":
        n = case["cand"] * case["vocab"]
        return {"bytes": n * size[case["kind"]] + 16 * case["cand"], "flops": 4 * n}
    n, rows, cols = case["n"], case["rows"], case["cols"]
    mats, kind = (1, "e4m3") if case["op"] == "linear" else (2, case["kind"])
    io = n * rows * size[case["out"]] * (2 if case.get("res") else 1) + 4 * rows * bool(case.get("bias"))
    scales = 4 * (n + mats * rows) if kind == "e4m3" else 0
    return {"bytes": (n + mats * rows) * cols * size[kind] + scales + io, "flops": 2 * mats * n * rows * cols}


def _two_to(k):
    """2^k in 64 bits, for whole k."""
    return ((k.long() + 1023) << 52).view(torch.float64)


def _e4m3_exact(x):
    """x to the nearest e4m3 value, ties to the even one, in 64 bits: steps of 2^(e - 3) for 2^e <= |x|, of 2^-9 below 2^-6, at most 448."""
    step = _two_to((torch.frexp(x)[1] - 1).clamp(min=-6) - 3)
    return (torch.round(x / step) * step).clamp(-448, 448)


def _norm_exact(s):
    c, out = s["case"], []
    h = s["x"].double()
    if c["res"] != "none":
        h = (h + s["res"].double()).to(TYPES[c["res"]]).double()  # the stream's own rounding
        out.append(h)
    if c["norm"]:
        h = h / torch.sqrt((h ** 2).sum(dim=1, keepdim=True) / c["cols"] + EPS) * s["w"].double()
    if c["out"] != "e4m3":
        return out + [h]
    amax = h.abs().amax(dim=1)
    k = (torch.ceil(torch.log2(amax.clamp(min=2.0 ** -50) / 448)) - 1).clamp(min=-64)
    for _ in range(3):
        k = torch.where(amax > 448 * _two_to(k), k + 1, k)
    return out + [_e4m3_exact(h / _two_to(k).unsqueeze(1)), _two_to(k)]


def _e4m3_values(x):
    b = x.view(torch.uint8).int()
    e, m = (b >> 3) & 15, (b & 7).double()
    v = torch.where(e == 0, m * 2.0 ** -9, (8 + m) * _two_to(e - 10))
    return torch.where(b >= 128, -v, v)


def _values(s, name):
    if s[name + "_scale"] is None:
        return s[name].double()
    return _e4m3_values(s[name]) * s[name + "_scale"].double().unsqueeze(1)


def _sample_exact(s):
    """Row by row: the kept set by its border in the sorted row, the token by a search in the kept tokens' sums; its probability in 64 bits."""
    c, prob = s["case"], []
    for r, u in zip(s["rows"].tolist(), s["u"].tolist()):
        x = s["logits"][r].double()
        dead = s["suppress"].tolist() + [c["vocab"] - 1]
        x[dead] = -math.inf
        if c["temperature"] == 0:
            token = int(torch.nonzero(x == x.max())[0])
        else:
            p = torch.softmax(x / c["temperature"], dim=0)
            v, at = torch.sort(x, descending=True, stable=True)
            sp = p[at]
            m = int((sp > 0).sum())
            if c["top_k"] > 0:
                m = min(m, c["top_k"])
            upto = torch.cumsum(sp[:m], dim=0)
            if c["top_p"] < 1:
                m = min(m, 1 + int((upto[:-1] < c["top_p"] * upto[-1]).sum()))
            m = max(1, min(m, int((sp >= c["min_p"] * sp[0]).sum())))
            kept = at[:m].sort().values
            sums = torch.cumsum(p[kept], dim=0)
            token = int(kept[min(m - 1, int(torch.searchsorted(sums, u * sums[-1:], right=True)))])
        prob.append(torch.softmax(x, dim=0)[token])
    return [None, torch.stack(prob)]


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "norm":
        return _norm_exact(s)
    if case["op"] == "sample":
        return _sample_exact(s)
    x = _values(s, "x")
    y = x @ _values(s, "w").T
    if case["op"] == "linear":
        y = y if s["bias"] is None else y + s["bias"].double()
        return y if s["res"] is None else y + s["res"].double()
    g = y * torch.sigmoid(y) if case["act"] == "silu" else torch.nn.functional.gelu(y, approximate="tanh")
    return g * (x @ _values(s, "up").T)
