"""The operators of the 8-bit inter-step cache, in cases that can be measured.

  store      bf16 K and V rows are quantised into the cache as they are written
  load       cache rows are read back as bf16
  attention  softmax(scale Q K^T) V over the cache, K and V taken as they are held

The cache holds K and V of every sequence position as e4m3 values [batch,
n_total, n_head_kv, head_dim] with one fp32 scale for each block of
`block` positions and kv head, [batch, ceil(n_total / block), n_head_kv]; the
value held is e4m3 * scale. Scales are powers of two: the smallest with
amax <= 448 * scale.

`own` false: plain torch in 32 bits. `own` true: the calls of canvas_attn.kv8.
"""
import math
import os
import sys

import torch

own = False

E4M3 = torch.float8_e4m3fn
K_MIN, K_MAX = -64, 120  # exponents a scale may have


def listed():
    return [
        # One committed token per sequence (Dream's 4 kv heads) joins caches whose last block is partly filled.
        dict(name="store token b4 h4", op="store", batch=4, n_total=1152, active=1, where="tail", kv=4, hd=128, block=32),
        # A denoising step of 16 sequences: 32 canvas rows scattered over the last 512 of 4128 positions.
        dict(name="store canvas b16 32of4128", op="store", batch=16, n_total=4128, active=32, where="canvas", kv=8, hd=128, block=32),
        # First full forward of a hybrid model's layer (head_dim 256): every position is written.
        dict(name="store full b4 8192 hd256", op="store", batch=4, n_total=8192, active=8192, where="all", kv=8, hd=256, block=64),
        # A few cached rows of one ragged sequence are gathered for inspection or a host copy (32 kv heads).
        dict(name="load gather 333of1111", op="load", batch=1, n_total=1111, rows=333, kv=32, hd=128, block=16),
        # A whole layer of 8 sequences is read back (a change of batch, an export).
        dict(name="load layer b8 4096", op="load", batch=8, n_total=4096, rows=4096, kv=16, hd=128, block=32),
        # The shortest call: one token over an odd 1001 positions, 28 query and 4 kv heads.
        dict(name="attn token b1 1001", op="attention", batch=1, sq=1, n_total=1024, lens=1001, ragged=False, heads=28, kv=4, hd=128, block=32, window=-1, prefix=-1, cap=0.0),
        # Single tokens of 16 ragged sequences.
        dict(name="attn token b16 4128", op="attention", batch=16, sq=1, n_total=4128, lens=4128, ragged=True, heads=32, kv=8, hd=128, block=32, window=-1, prefix=-1, cap=0.0),
        # A single token over a long cache.
        dict(name="attn token b1 131072", op="attention", batch=1, sq=1, n_total=131072, lens=131072, ragged=False, heads=32, kv=8, hd=128, block=64, window=-1, prefix=-1, cap=0.0),
        # Cached block step: 16 sequences, 32 masked canvas tokens over 4096 cached positions and themselves.
        dict(name="attn canvas b16 32x4128", op="attention", batch=16, sq=32, n_total=4128, lens=4128, ragged=False, heads=32, kv=8, hd=128, block=32, window=-1, prefix=-1, cap=0.0),
        # The same step without shared heads (32 kv heads, one query head each), a causal prompt of 700 tokens.
        dict(name="attn canvas b2 40x2100 mha", op="attention", batch=2, sq=40, n_total=2112, lens=2100, ragged=True, heads=32, kv=32, hd=128, block=16, window=-1, prefix=700, cap=0.0),
        # Full canvas of 2 sequences, 16 heads of their own: the step that recomputes every row.
        dict(name="attn full b2 4096", op="attention", batch=2, sq=4096, n_total=4096, lens=4096, ragged=False, heads=16, kv=16, hd=128, block=32, window=-1, prefix=-1, cap=0.0),
        # Sliding-window layer at head_dim 256 with a logit soft-cap: a 2048-token canvas of 8192 positions.
        dict(name="attn window b1 2048x8192 hd256", op="attention", batch=1, sq=2048, n_total=8192, lens=8192, ragged=False, heads=16, kv=8, hd=256, block=64, window=512, prefix=-1, cap=50.0),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["store", "load", "attention", "attention", "attention"])
    hd = rng.choice([64, 128, 128, 128, 256])
    block = rng.choice([16, 32, 64, 128])
    kv = rng.choice([2, 4, 8, 16])
    batch = _log(rng, 1, 16)
    n_total = _log(rng, 100, 8192)
    while batch * n_total * kv * hd > (1 << 25):
        batch, n_total = max(1, batch // 2), max(100, n_total * 3 // 4)
    if op == "store":
        where = rng.choice(["tail", "canvas", "all"])
        active = {"tail": _log(rng, 1, 16), "canvas": min(n_total, _log(rng, 4, 64)), "all": n_total}[where]
        return dict(op=op, batch=batch, n_total=n_total, active=active, where=where, kv=kv, hd=hd, block=block)
    if op == "load":
        return dict(op=op, batch=batch, n_total=n_total, rows=_log(rng, 20, n_total), kv=kv, hd=hd, block=block)
    heads = kv * rng.choice([1, 2, 4, 7, 8])
    sq = min(n_total, rng.choice([1, _log(rng, 2, 64), _log(rng, 64, 2048)]))
    while batch * heads * sq * n_total * hd > 2 * 16 * 4096 * 4096 * 128 // 2:
        sq = max(1, sq // 2)
    window = rng.choice([-1, -1, _log(rng, 16, 2048)])
    return dict(op=op, batch=batch, sq=sq, n_total=n_total, lens=max(sq, n_total - rng.randrange(0, 40)), ragged=rng.random() < 0.5, heads=heads, kv=kv, hd=hd,
                block=block, window=window, prefix=rng.choice([-1, -1, n_total // 3]), cap=rng.choice([0.0, 0.0, 50.0]))


def _blocks(case):
    return -(-case["n_total"] // case["block"])


def _scale_of(amax):
    """2^k of the smallest k with amax <= 448 * 2^k (448 = 0.875 * 2^9)."""
    m, e = torch.frexp(amax)
    k = torch.where(amax > 0, torch.where(m <= 0.875, e - 9, e - 8).clamp(K_MIN, K_MAX), K_MIN)
    return ((k.to(torch.int32) + 127) << 23).view(torch.float32)


def _per_row(scale, block, n):
    """A block's scale at each of its positions: [batch, n, kv, 1]."""
    return scale.repeat_interleave(block, dim=1)[:, :n].unsqueeze(-1)


def _by_block(x, block):
    """[batch, n, ...] as [batch, blocks, block, ...], the end filled with zeros."""
    n = x.shape[1]
    pad = -n % block
    if pad:
        x = torch.cat([x, x.new_zeros((x.shape[0], pad) + x.shape[2:])], dim=1)
    return x.reshape((x.shape[0], -1, block) + x.shape[2:])


def _filled(case, g, dev):
    """A cache of rows with a few loud channels and blocks of different loudness, as trained K and V have."""
    shape = (case["batch"], case["n_total"], case["kv"], case["hd"])
    x = torch.randn(shape, generator=g, device=dev)
    x *= torch.exp(0.4 * torch.randn((1, 1, case["kv"], case["hd"]), generator=g, device=dev))
    x *= torch.exp2(torch.randint(-1, 2, (case["batch"], _blocks(case), case["kv"]), generator=g, device=dev).float()).repeat_interleave(case["block"], dim=1)[:, : case["n_total"]].unsqueeze(-1)
    scale = _scale_of(_by_block(x, case["block"]).abs().amax(dim=(2, 4)))
    held = (x / _per_row(scale, case["block"], case["n_total"])).to(E4M3)
    return held.view(torch.uint8), scale


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(int(seed))
    k, ks = _filled(case, g, dev)
    v, vs = _filled(case, g, dev)
    b, n = case["batch"], case["n_total"]
    s = dict(case=case, k=k, v=v, ks=ks, vs=vs)
    bf = torch.bfloat16
    if case["op"] == "store":
        a = case["active"]
        if case["where"] == "tail":  # the next positions of sequences of different lengths
            s["kv_len"] = torch.randint(n // 2, n - a + 1, (b,), generator=g, device=dev, dtype=torch.int32)
            pos = s["kv_len"].unsqueeze(1) + torch.arange(a, device=dev, dtype=torch.int32)
        elif case["where"] == "canvas":  # masked positions of the last 512
            tail = min(n, max(512, a))
            order = torch.rand((b, tail), generator=g, device=dev).argsort(dim=1)[:, :a].sort(dim=1).values
            pos = n - tail + order
        else:
            pos = torch.arange(n, device=dev).expand(b, n)
        s["pos"] = pos.to(torch.int32).contiguous()
        for name in ("new_k", "new_v"):
            s[name] = (1.5 * torch.randn((b, a, case["kv"], case["hd"]), generator=g, device=dev)).to(bf)
    elif case["op"] == "load":
        rows = torch.rand((b, n), generator=g, device=dev).argsort(dim=1)[:, : case["rows"]].sort(dim=1).values
        s["pos"] = rows.to(torch.int32).contiguous()
        s["out"] = [torch.empty((b, case["rows"], case["kv"], case["hd"]), dtype=bf, device=dev) for _ in range(2)]
    else:
        sq, lens = case["sq"], case["lens"]
        s["q"] = torch.randn((b, sq, case["heads"], case["hd"]), generator=g, device=dev).to(bf)
        s["kv_len"] = torch.full((b,), lens, dtype=torch.int32, device=dev)
        if case["ragged"]:
            s["kv_len"] = torch.randint(max(sq, lens // 2), lens + 1, (b,), generator=g, device=dev, dtype=torch.int32)
        # The queries are the last rows of what each sequence holds.
        s["pos"] = (s["kv_len"].unsqueeze(1) - sq + torch.arange(sq, device=dev)).to(torch.int32).contiguous()
        s["out"] = torch.empty((b, sq, case["heads"], case["hd"]), dtype=bf, device=dev)
    return s


def _store_plain(s):
    c = s["case"]
    block, n, b = c["block"], c["n_total"], c["batch"]
    at = s["pos"].long()
    seq = torch.arange(b, device=at.device).unsqueeze(1)
    active = torch.zeros((b, n), dtype=torch.bool, device=at.device)
    active[seq, at] = True
    holds = torch.arange(n, device=at.device) < (s["kv_len"].unsqueeze(1) if "kv_len" in s else n)
    fresh = ~(_by_block(holds & ~active, block).any(dim=2))
    touched = _by_block(active, block).any(dim=2).unsqueeze(-1)
    out = []
    for held, scale, new in ((s["k"], s["ks"], s["new_k"]), (s["v"], s["vs"], s["new_v"])):
        x = torch.zeros((b, n) + new.shape[2:], dtype=torch.float32, device=at.device)
        x[seq, at] = new.float()
        need = _scale_of(_by_block(x, block).abs().amax(dim=(2, 4)))
        keep = ~fresh.unsqueeze(-1) & (scale > 0)
        now = torch.where(touched, torch.where(keep, torch.maximum(scale, need), need), scale)
        grown = touched & keep & (now > scale)
        row = _per_row(now, block, n)
        was = held.view(E4M3).float() * _per_row(torch.where(grown, scale / now, 1.0), block, n)
        y = torch.where(active.view(b, n, 1, 1), x / row, was).to(E4M3)
        held.copy_(y.view(torch.uint8))
        scale.copy_(now)
        out += [held.view(E4M3), scale]
    return out


def _load_plain(s):
    c = s["case"]
    at = s["pos"].long()
    seq = torch.arange(c["batch"], device=at.device).unsqueeze(1)
    return [(held[seq, at].view(E4M3).float() * scale[seq, at // c["block"]].unsqueeze(-1)).to(torch.bfloat16) for held, scale in ((s["k"], s["ks"]), (s["v"], s["vs"]))]


def _visible(c, pos, kv_len, n):
    """[batch, 1, sq, n]: what each query row sees."""
    q, k = pos.long().unsqueeze(-1), torch.arange(n, device=pos.device)
    see = k < kv_len.long().view(-1, 1, 1)
    if c["window"] >= 0:
        see = see & ((q - k).abs() < c["window"])
    if c["prefix"] >= 0:
        see = see & ((q >= c["prefix"]) | (k <= q))
    return see.unsqueeze(1)


def _attention_plain(s):
    c = s["case"]
    b, sq, h, kv, hd, n = c["batch"], c["sq"], c["heads"], c["kv"], c["hd"], c["n_total"]
    k = (s["k"].view(E4M3).float() * _per_row(s["ks"], c["block"], n)).permute(0, 2, 3, 1)
    v = (s["v"].view(E4M3).float() * _per_row(s["vs"], c["block"], n)).permute(0, 2, 1, 3)
    q = s["q"].float().view(b, sq, kv, h // kv, hd).permute(0, 2, 3, 1, 4).reshape(b, kv, -1, hd)
    t = (q @ k).mul_(hd ** -0.5).view(b, h, sq, n)
    if c["cap"] > 0:
        t = t.div_(c["cap"]).tanh_().mul_(c["cap"])
    t = t.masked_fill_(~_visible(c, s["pos"], s["kv_len"], n), -math.inf)
    t = t.sub_(t.amax(dim=-1, keepdim=True)).exp_()
    o = (t.view(b, kv, -1, n) @ v) / t.sum(dim=-1).view(b, kv, -1, 1)
    return o.view(b, h, sq, hd).transpose(1, 2).to(torch.bfloat16)


def _plan(s):
    """What a user's program builds once for buffers that it keeps: the cache's handle, the argument block of its call, the workspace."""
    root = os.path.join(os.getcwd(), "diffuse-rs_b200")
    if root not in sys.path:
        sys.path.insert(0, root)
    from canvas_attn import kv8
    c = s["case"]
    cache = kv8.Kv8Cache(s["k"], s["v"], s["ks"], s["vs"], c["block"])
    opt = lambda x: None if x < 0 else x  # noqa: E731
    if c["op"] == "store":
        a = kv8.make_store_args(cache, s["new_k"], s["new_v"], s["pos"], kv_len=s.get("kv_len"))
        return kv8, kv8.store_args, a
    if c["op"] == "load":
        return kv8, kv8.load_args, kv8.make_load_args(cache, s["out"][0], s["out"][1], s["pos"])
    a = kv8.make_attention_args(s["q"], cache, s["out"], q_pos=s["pos"], kv_len=s["kv_len"], sliding_window=opt(c["window"]), causal_prefix=opt(c["prefix"]),
                                scale=c["hd"] ** -0.5, softcap=c["cap"])
    return kv8, kv8.attention_args, a


def run(s):
    op = s["case"]["op"]
    if not own:
        return {"store": _store_plain, "load": _load_plain, "attention": _attention_plain}[op](s)
    if "plan" not in s:
        s["plan"] = _plan(s)
    _, call, a = s["plan"]
    call(a)
    if op == "store":
        return [s["k"].view(E4M3), s["ks"], s["v"].view(E4M3), s["vs"]]
    return s["out"]


def work(case):
    b, kv, hd, n = case["batch"], case["kv"], case["hd"], case["n_total"]
    if case["op"] == "store":
        # Rows in as bf16, out as e4m3; a scale read and written for each block that a row falls in (at most).
        rows = b * case["active"]
        blocks = b * min(case["active"], _blocks(case)) * kv
        return {"bytes": 2 * rows * kv * hd * 3 + 2 * blocks * 8 + rows * 4, "flops": 2 * 3 * rows * kv * hd}
    if case["op"] == "load":
        rows = b * case["rows"]
        return {"bytes": 2 * rows * kv * hd * 3 + 2 * b * min(case["rows"], _blocks(case)) * kv * 4 + rows * 4, "flops": 2 * rows * kv * hd}
    sq, h = case["sq"], case["heads"]
    length = case["lens"] if not case["ragged"] else (max(sq, case["lens"] // 2) + case["lens"]) // 2
    pairs, first = 0, length
    for i in range(sq):  # visible keys of the query at position length - sq + i
        q = length - sq + i
        lo, hi = 0, length
        if case["window"] >= 0:
            lo, hi = max(0, q - case["window"] + 1), min(length, q + case["window"])
        if case["prefix"] >= 0 and q < case["prefix"]:
            hi = min(hi, q + 1)
        pairs += max(0, hi - lo)
        first = min(first, lo)
    keys = length - first
    cache = 2 * b * kv * (keys * hd + -(-keys // case["block"]) * 4)
    return {"bytes": cache + 2 * b * sq * h * hd * 2 + b * sq * 4, "flops": 4 * b * h * pairs * hd}


def _two_to(k):
    """2^k in 64 bits, for whole k."""
    return ((k.long() + 1023) << 52).view(torch.float64)


def _e4m3_exact(x):
    """x to the nearest e4m3 value, ties to the even one, in 64 bits: steps of 2^(e - 3) for 2^e <= |x|, of 2^-9 below 2^-6, at most 448."""
    step = _two_to((torch.frexp(x)[1] - 1).clamp(min=-6) - 3)
    return (torch.round(x / step) * step).clamp(-448, 448)


def _store_exact(s):
    """Block by block from the definition: the rows that are written set what the scale has to reach; rows that stay keep what it was."""
    c = s["case"]
    block, n, b, n_blocks = c["block"], c["n_total"], c["batch"], _blocks(c)
    dev = s["k"].device
    place = torch.full((b, n_blocks * block), -1, dtype=torch.long, device=dev)
    place.scatter_(1, s["pos"].long(), torch.arange(c["active"], device=dev).expand(b, -1))
    place = place.view(b, n_blocks, block)
    index = torch.arange(n_blocks * block, device=dev).view(1, n_blocks, block)
    holds = index < torch.clamp(s["kv_len"].view(b, 1, 1) if "kv_len" in s else torch.full((b, 1, 1), n, device=dev), max=n)
    stays = (holds & (place < 0)).any(dim=2)
    out = []
    for held, scale, new in ((s["k"], s["ks"], s["new_k"]), (s["v"], s["vs"], s["new_v"])):
        old = torch.zeros((b, n_blocks * block, c["kv"], c["hd"]), dtype=torch.float64, device=dev)
        old[:, :n] = held.view(E4M3).double()
        old = old.view(b, n_blocks, block, c["kv"], c["hd"])
        rows = torch.gather(new.double(), 1, place.clamp(min=0).view(b, -1, 1, 1).expand(-1, -1, c["kv"], c["hd"])).view_as(old)
        is_new = (place >= 0).view(b, n_blocks, block, 1, 1)
        amax = torch.where(is_new, rows.abs(), 0.0).amax(dim=(2, 4))
        k = torch.ceil(torch.log2(amax.clamp(min=2.0 ** -50) / 448)) - 1
        for _ in range(3):  # the smallest k with amax <= 448 * 2^k
            k = torch.where(amax > 448 * _two_to(k), k + 1, k)
        need = torch.where(amax > 0, _two_to(k), 2.0 ** K_MIN)
        was = scale.double()
        any_new = (place >= 0).any(dim=2).unsqueeze(-1)
        now = torch.where(stays.unsqueeze(-1) & (was > 0), torch.maximum(was, need), need)
        now = torch.where(any_new, now, was)
        ratio = torch.where(any_new & stays.unsqueeze(-1) & (was > 0), was / now, 1.0).view(b, n_blocks, 1, c["kv"], 1)
        y = torch.where(is_new, _e4m3_exact(rows / now.view(b, n_blocks, 1, c["kv"], 1)), _e4m3_exact(old * ratio))
        out += [y.view(b, -1, c["kv"], c["hd"])[:, :n], now]
    return out


def _values(held, scale, block):
    """What the cache stands for, in 64 bits."""
    b = held.int()
    e, m = (b >> 3) & 15, (b & 7).double()
    x = torch.where(e == 0, m * 2.0 ** -9, (8 + m) * _two_to(e - 10))
    at = torch.arange(held.shape[1], device=held.device) // block
    return torch.where(b >= 128, -x, x) * scale.double()[:, at].unsqueeze(-1)


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "store":
        return _store_exact(s)
    if case["op"] == "load":
        seq = torch.arange(case["batch"], device=s["k"].device).unsqueeze(1)
        return [_values(s[x], s[x + "s"], case["block"])[seq, s["pos"].long()] for x in ("k", "v")]
    k, v = (_values(s[x], s[x + "s"], case["block"]) for x in ("k", "v"))
    group = case["heads"] // case["kv"]
    out = torch.empty(s["out"].shape, dtype=torch.float64, device=k.device)
    for b in range(case["batch"]):
        see = _visible(case, s["pos"][b : b + 1], s["kv_len"][b : b + 1], case["n_total"])[0, 0]
        for h in range(case["heads"]):
            t = s["q"][b, :, h].double() @ k[b, :, h // group].T / math.sqrt(case["hd"])
            if case["cap"] > 0:
                t = case["cap"] * torch.tanh(t / case["cap"])
            t = torch.where(see, t, -math.inf)
            out[b, :, h] = torch.softmax(t, dim=-1) @ v[b, :, h // group]
    return out
