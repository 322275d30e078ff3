"""Denoising with the 8-bit inter-step cache: a stack of attention layers runs
the first step over every position, then block steps that recompute 32 canvas
rows of each sequence and read the rest from the cache, and picks tokens with
the candidate statistics. The same steps over the bf16 cache run beside it.

  python examples/kv8_denoise.py [--batch 4] [--total 1024] [--steps 8]

Random weights of a LLaDA-MoE-like layer (16 heads of 128, QK-norm). Prints
the caches' bytes, how far the two runs' outputs are apart, the time of a
block step over each, and how often the picked tokens agree.
"""
import argparse
import os
import sys

import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
sys.path.insert(0, os.path.join(ROOT, "diffuse-rs_b200"))

import canvas_attn as ca  # noqa: E402
from canvas_attn import denoise, kv8, projection  # noqa: E402

HEADS, KV, HD, VOCAB = 16, 16, 128, 4096


class Layer:
    def __init__(self, g, batch, n_total, dev):
        e = HEADS * HD
        w = lambda rows: (torch.randn(rows, e, generator=g, device=dev) * e ** -0.5).bfloat16()  # noqa: E731
        self.wqkv, self.wo = w(e + 2 * KV * HD), w(e)
        self.qn, self.kn = (torch.rand(HD, generator=g, device=dev) + 0.5 for _ in range(2))
        self.cache8 = kv8.Kv8Cache.alloc(batch, n_total, KV, HD, block_tokens=32, device=dev)
        self.k16 = torch.zeros(batch, n_total, KV, HD, dtype=torch.bfloat16, device=dev)
        self.v16 = torch.zeros_like(self.k16)
        self.kept = {}  # by rows of a sequence: q, k, v, out, positions, the step's arguments


def linear(x, w, residual=None, dtype=torch.bfloat16):
    """x w^T (+ residual) through the framework's projection."""
    n, cols = x.shape
    out = torch.empty(n, w.shape[0], dtype=dtype, device=x.device)
    projection.linear(x, w, out, n=n, rows=w.shape[0], cols=cols, residual=residual)
    return out


def forward(layers, x, pos, rope, n_total, eight):
    """Hidden states [batch, rows, e] of the rows at `pos` after every layer."""
    b, n, e = x.shape
    x = x.reshape(b * n, e)
    for ly in layers:
        h = (x.float() * torch.rsqrt(x.float().square().mean(-1, keepdim=True) + 1e-6)).bfloat16()
        kw = dict(rope=rope, rope_len=n_total, rope_dim=HD, q_norm_w=ly.qn, k_norm_w=ly.kn,
                  scale=HD ** -0.5)
        if n not in ly.kept:
            mk = lambda heads: torch.empty(b, n, heads, HD, dtype=x.dtype, device=x.device)  # noqa: E731
            q, k, v, out, at = mk(HEADS), mk(KV), mk(KV), mk(HEADS), torch.empty_like(pos)
            ly.kept[n] = (q, k, v, out, at, torch.empty_like(q),
                          kv8.make_block_args(q, k, v, ly.cache8, out, active_pos=at, **kw))
        q, k, v, out, at, q_work, step8 = ly.kept[n]
        for buf, y in zip((q, k, v), linear(h, ly.wqkv).split([HEADS * HD, KV * HD, KV * HD], -1)):
            buf.copy_(y.reshape(buf.shape))
        at.copy_(pos)
        if eight:
            kv8.block_args(step8)
        else:
            ca.attention_block_dev(q, k, v, batch=b, n_active=n, active_pos=at, cache_k=ly.k16,
                                   cache_v=ly.v16, n_total=n_total, q_work=q_work, out=out,
                                   n_head=HEADS, n_head_kv=KV, head_dim=HD, **kw)
        x = linear(out.view(b * n, e), ly.wo, residual=x)
    return x.view(b, n, e)


def main(argv=None):
    ap = argparse.ArgumentParser(description=__doc__)
    ap.add_argument("--batch", type=int, default=4)
    ap.add_argument("--total", type=int, default=1024)
    ap.add_argument("--steps", type=int, default=8)
    ap.add_argument("--layers", type=int, default=4)
    a = ap.parse_args(argv)
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(0)
    layers = [Layer(g, a.batch, a.total, dev) for _ in range(a.layers)]
    embed = torch.randn(VOCAB, HEADS * HD, generator=g, device=dev).bfloat16()
    rope = torch.from_numpy(ca.build_rope_cache(a.total, HD, 50000.0)).to(dev)
    tokens = torch.randint(0, VOCAB, (a.batch, a.total), generator=g, device=dev)
    everything = torch.arange(a.total, dtype=torch.int32, device=dev).repeat(a.batch, 1)
    far, same, ms = [], [], {True: [], False: []}
    for step in range(a.steps):
        if step == 0:
            pos = everything
        else:  # 32 canvas rows of the second half
            pos = (a.total // 2 + torch.rand(a.batch, a.total - a.total // 2, generator=g,
                                             device=dev).argsort(dim=1)[:, :32].sort(dim=1).values)
            pos = pos.to(torch.int32).contiguous()
        x = embed[tokens.gather(1, pos.long())]
        picked = {}
        for eight in (False, True):
            t0, t1 = (torch.cuda.Event(enable_timing=True) for _ in range(2))
            t0.record()
            y = forward(layers, x, pos, rope, a.total, eight)
            t1.record()
            logits = linear(y[:, -32:].reshape(-1, y.shape[-1]), embed, dtype=torch.float32)
            rows = torch.arange(logits.shape[0], dtype=torch.int32, device=dev)
            tok = torch.empty_like(rows)
            denoise.candidate_stats(logits, rows, tok, n_vocab=VOCAB, want_entropy=False)
            torch.cuda.synchronize()
            assert ca.device_status() == ca.CA_OK
            picked[eight] = (y.float(), tok)
            if step > 1:
                ms[eight].append(t0.elapsed_time(t1))
        (y16, t16), (y8, t8) = picked[False], picked[True]
        far.append(float((y8 - y16).norm() / y16.norm()))
        same.append(float((t8 == t16).float().mean()))
        tokens.scatter_(1, pos[:, -32:].long(), t16.view(a.batch, -1).long())
    c = layers[0].cache8
    bytes8 = sum(x.numel() * x.element_size() for x in (c.k, c.v, c.k_scale, c.v_scale))
    bytes16 = 2 * layers[0].k16.numel() * 2
    print(f"cache per layer: {bytes16 / 1e6:.1f} MB bf16, {bytes8 / 1e6:.1f} MB in 8 bits")
    print("outputs apart by (relative): " + " ".join(f"{f:.3f}" for f in far))
    print("tokens that agree:           " + " ".join(f"{f:.3f}" for f in same))
    if ms[True]:
        mid = lambda v: sorted(v)[len(v) // 2]  # noqa: E731
        print(f"block step: {mid(ms[False]):.3f} ms bf16, {mid(ms[True]):.3f} ms in 8 bits")
    return far, same


if __name__ == "__main__":
    main()
