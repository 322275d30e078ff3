"""One denoising step on the device, from a layer's attention block to the
drawn tokens: attention_block_dev, linear_q8 with the residual, rms_norm to
e4m3, gated_linear, quantize_rows, linear_q8, over two layers; the last norm,
the logits' product and the draw. Every call's output is checked against its
formula on the inputs that it was given, and the whole run, whose kernels may
overlap the ends of those before them, against the same run with a wait after
each call, bit by bit, also captured into a graph."""
import pytest
import torch

import canvas_attn as ca
from canvas_attn import denoise as dn
from canvas_attn import layer
from layer_helpers import F8, activate_ref, norm_ref, product_ref
from sample_helpers import STEP, sample_ref

pytestmark = pytest.mark.gpu
BF, F32 = torch.bfloat16, torch.float32
E, H, HKV, HD, FF, V, LAYERS = 256, 4, 2, 64, 720, 3001, 2


class Step:
    """Buffers and weights of a step over `n` rows of one sequence."""

    def __init__(self, n, seed):
        g = torch.Generator(device="cuda").manual_seed(seed)
        r = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
        self.n = n
        self.h0 = r(n, E).to(BF)
        self.pos = torch.arange(n, dtype=torch.int32, device="cuda").view(1, n)
        self.rope = torch.from_numpy(ca.build_rope_cache(max(n, 16), HD, 1e4)).cuda()
        self.q, self.k, self.v = (r(n, x, HD).to(BF) for x in (H, HKV, HKV))
        self.u = torch.rand(n, generator=g, device="cuda")
        self.gain = [0.5 + torch.rand(E, generator=g, device="cuda") for _ in range(LAYERS + 1)]
        self.w = []
        for _ in range(LAYERS):
            ws = []
            for rows, cols in ((E, H * HD), (FF, E), (FF, E), (E, FF)):
                q, s = self.new8(rows, cols)
                layer.quantize_rows(r(rows, cols) * cols ** -0.5, q, s)
                ws.append((q, s))
            self.w.append(ws)
        self.head = self.new8(V, E)
        layer.quantize_rows(r(V, E) * 0.2, *self.head)
        new = lambda *s: torch.empty(*s, dtype=BF, device="cuda")  # noqa: E731
        self.h, self.att, self.ff = new(n, E), new(1, n, H, HD), new(n, FF)
        self.ck, self.cv, self.qw = new(1, n, HKV, HD), new(1, n, HKV, HD), new(1, n, H, HD)
        self.a8, self.x8, self.f8 = self.new8(n, H * HD), self.new8(n, E), self.new8(n, FF)
        self.logits = torch.empty(n, V, device="cuda")
        self.token = torch.empty(n, dtype=torch.int32, device="cuda")
        self.prob = torch.empty(n, device="cuda")
        torch.cuda.synchronize()

    @staticmethod
    def new8(rows, cols):
        return (torch.zeros(rows, cols, device="cuda").to(F8), torch.zeros(rows, device="cuda"))

    def run(self, after, stream=None):
        """`after` is called behind each call with what it wrote and had."""
        kw = dict(stream=stream)
        self.h.copy_(self.h0)
        for i in range(LAYERS):
            (wo, so), (wg, sg), (wu, su), (wd, sd) = self.w[i]
            ca.attention_block_dev(
                self.q, self.k, self.v, batch=1, n_active=self.n, active_pos=self.pos,
                rope=self.rope, rope_len=self.rope.shape[0], rope_dim=HD, cache_k=self.ck,
                cache_v=self.cv, n_total=self.n, q_work=self.qw, out=self.att, n_head=H,
                n_head_kv=HKV, head_dim=HD, rms_eps=1e-5, scale=HD ** -0.5, **kw)
            layer.quantize_rows(self.att.view(self.n, H * HD), *self.a8, **kw)
            res = self.h.clone() if after is checked else None
            layer.linear_q8(*self.a8, wo, so, self.h, residual=self.h, **kw)
            after("linear", x=self.a8, w=(wo, so), res=res, out=self.h)
            layer.rms_norm(self.h, self.x8[0], w=self.gain[i], eps=1e-5, out_scale=self.x8[1], **kw)
            after("norm", x=self.h, w=self.gain[i], out=self.x8)
            layer.gated_linear(self.x8[0], wg, wu, self.ff, act_scale=self.x8[1], gate_scale=sg,
                               up_scale=su, **kw)
            after("gated", x=self.x8, w=(wg, sg), up=(wu, su), out=self.ff)
            layer.quantize_rows(self.ff, *self.f8, **kw)
            res = self.h.clone() if after is checked else None
            layer.linear_q8(*self.f8, wd, sd, self.h, residual=self.h, **kw)
            after("linear", x=self.f8, w=(wd, sd), res=res, out=self.h)
        layer.rms_norm(self.h, self.x8[0], w=self.gain[-1], eps=1e-5, out_scale=self.x8[1], **kw)
        layer.linear_q8(*self.x8, *self.head, self.logits, **kw)
        after("logits", x=self.x8, w=self.head, out=self.logits)
        dn.sample(self.logits, None, self.u, self.token, self.prob, temperature=0.9, top_p=0.95,
                  mask_id=V - 1, **kw)

    def outputs(self):
        return [t.clone() for t in (self.h, self.ff, self.logits, self.token, self.prob)]


def waiting(what, **inputs):
    torch.cuda.synchronize()


def plain(what, **inputs):
    pass


def checked(what, **t):
    torch.cuda.synchronize()
    if what == "norm":
        y = norm_ref(t["x"], w=t["w"], eps=1e-5)[1]
        got = t["out"][0].double() * t["out"][1].double().unsqueeze(1)
        assert ((got - y).abs() <= (2.0 ** -4 + 2.0 ** -18) * y.abs()
                + 2.0 ** -10 * t["out"][1].double().unsqueeze(1)).all()
        return
    y, mag = product_ref(*t["x"], *t["w"])
    cols = t["x"][0].shape[1]
    e = cols * 2.0 ** -23 + 2.0 ** -22
    half = torch.finfo(t["out"].dtype).eps / 2
    if what == "gated":
        u, um = product_ref(*t["x"], *t["up"])
        f = activate_ref(y, "silu")
        tol = 1.13 * e * mag * (u.abs() + e * um) + e * um * f.abs() + 1e-5 * (f * u).abs()
        y = f * u
    else:
        if t.get("res") is not None:
            y = y + t["res"].double()
            mag = mag + t["res"].double().abs()
        tol = e * mag
    assert ((t["out"].double() - y).abs() <= tol + half * y.abs()).all(), what


@pytest.mark.parametrize("n", [1, 13, 100, 300])
def test_a_step(n):
    s = Step(n, n)
    s.run(checked)
    torch.cuda.synchronize()
    for i in range(n):
        ref, p, slack = sample_ref(s.logits[i].cpu().numpy(), float(s.u[i]), temperature=0.9,
                                   top_p=0.95, dead=[V - 1])
        if slack > V * STEP:  # (the logits are the run's own, so a border may be too near)
            assert int(s.token[i]) == ref and abs(float(s.prob[i]) - p) <= 1e-5 * p
    s.run(waiting)
    want = s.outputs()
    for _ in range(3):
        s.run(plain)
        torch.cuda.synchronize()
        for a, b in zip(s.outputs(), want):
            assert torch.equal(a, b)
    st = torch.cuda.Stream()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=st):
        s.run(plain, stream=st)
    for _ in range(3):
        s.token.zero_()
        g.replay()
    torch.cuda.synchronize()
    for a, b in zip(s.outputs(), want):
        assert torch.equal(a, b)


def test_two_steps_on_two_streams():
    steps = [Step(100, 1), Step(33, 2)]
    want = []
    for s in steps:
        s.run(waiting)
        want.append(s.outputs())
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    for _ in range(3):
        for s, st in zip(steps, streams):
            with torch.cuda.stream(st):
                s.run(plain, stream=st)
    torch.cuda.synchronize()
    for s, w in zip(steps, want):
        for a, b in zip(s.outputs(), w):
            assert torch.equal(a, b)
