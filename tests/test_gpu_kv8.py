"""The 8-bit cache on the GPU: store and load bit for bit, attention against
a 64-bit softmax over the held values.

Attention tolerance. Scores and sums are fp32, so against the 64-bit result
what counts is the f16 rounding of each weight, at most 2^-11 of it, hence at
most 2^-11 sum p |v| in an output; another 2^-11 of the same sum is left for
the scores, exponentials and fp32 sums (scores up to some tens with 24 bits:
errors of 2^-18 of a weight and less). bf16 outputs are held to the fp32
outputs of the same call, rounded, bit for bit.
"""
import ctypes

import pytest
import torch

import canvas_attn as ca
from canvas_attn import kv8
from kv8_helpers import F8, attention_ref, held_values, random_cache, store_ref

pytestmark = pytest.mark.gpu


def cache_of(g, b, n, h, d, T):
    k, ks = random_cache(g, b, n, h, d, T, "cuda")
    v, vs = random_cache(g, b, n, h, d, T, "cuda")
    return kv8.Kv8Cache(k, v, ks, vs, T)


def check_attention(q, cache, out, pos, lens, what="", **kw):
    """out against the 64-bit reference, sequence by sequence."""
    k = held_values(cache.k, cache.k_scale, cache.block_tokens)
    v = held_values(cache.v, cache.v_scale, cache.block_tokens)
    for b in range(len(lens)):
        ref, mag = attention_ref(q[b], k[b], v[b], pos[b], int(lens[b]), **kw)
        got = out[b].double()
        assert torch.equal(torch.isnan(got), torch.isnan(ref)), f"{what}: NaN pattern"
        err = torch.nan_to_num((got - ref).abs())
        tol = torch.nan_to_num(2.0 ** -10 * mag) + 1e-30
        assert bool((err <= tol).all()), \
            f"{what}: sequence {b}: {float((err / tol).max()):.2f} of the tolerance"


def run_attention(B, sq, H, Hkv, d, n, T, *, lens=None, window=None, prefix=None, cap=0.0,
                  seed=1, where="end", workspace=None, qscale=1.0, scale=None):
    g = torch.Generator().manual_seed(seed)
    cache = cache_of(g, B, n, Hkv, d, T)
    q = (qscale * torch.randn(B, sq, H, d, generator=g)).to(torch.bfloat16).cuda()
    lens = [n] * B if lens is None else lens
    if where == "end":
        pos = torch.stack([torch.arange(sq) + ln - sq for ln in lens])
    else:
        pos = torch.stack([torch.randperm(max(ln, sq), generator=g)[:sq].sort().values
                           for ln in lens])
    pos = pos.to(torch.int32).cuda()
    kv_len = torch.tensor(lens, dtype=torch.int32).cuda()
    out = torch.full((B, sq, H, d), 7.0, device="cuda")
    scale = d ** -0.5 if scale is None else scale
    kv8.attention(q, cache, out, q_pos=pos, kv_len=kv_len, sliding_window=window,
                  causal_prefix=prefix, scale=scale, softcap=cap, workspace=workspace)
    torch.cuda.synchronize()
    assert ca.device_status() == ca.CA_OK
    check_attention(q, cache, out, pos, lens, scale=scale, window=window, prefix=prefix, cap=cap)
    return q, cache, out, pos, kv_len


# Sizes on both sides of every tile: rows of 16 and 128, keys of 16, 64 and 128.
SHAPES = [
    # B, sq, H, Hkv, d, n, T
    (1, 1, 1, 1, 128, 1, 16), (2, 1, 8, 2, 128, 15, 16), (1, 1, 7, 1, 128, 17, 32),
    (3, 1, 32, 8, 128, 1001, 32), (1, 2, 16, 2, 128, 129, 64), (2, 5, 28, 4, 128, 127, 128),
    (1, 1, 8, 8, 64, 333, 16), (2, 3, 12, 4, 64, 200, 32), (1, 1, 16, 8, 256, 700, 64),
    (1, 4, 4, 2, 256, 97, 16), (1, 1, 4, 2, 512, 300, 32), (1, 9, 2, 1, 512, 70, 16),
    (1, 3, 4, 2, 96, 150, 32), (1, 2, 2, 1, 16, 40, 16), (1, 6, 4, 2, 192, 130, 64),
    (2, 32, 8, 2, 128, 260, 32), (1, 40, 4, 4, 128, 300, 16), (1, 33, 12, 4, 64, 513, 128),
    (1, 70, 6, 2, 256, 250, 32), (1, 200, 4, 2, 128, 400, 64), (2, 129, 2, 2, 128, 128, 32),
]


@pytest.mark.parametrize("B,sq,H,Hkv,d,n,T", SHAPES)
def test_attention_shapes(B, sq, H, Hkv, d, n, T):
    run_attention(B, sq, H, Hkv, d, max(n, sq), T)


@pytest.mark.parametrize("d,sq", [(128, 1), (128, 40), (64, 50), (256, 3), (256, 60), (512, 2)])
def test_attention_bf16_out(d, sq):
    q, cache, out, pos, kv_len = run_attention(2, sq, 8, 2, d, 300, 32)
    half = torch.full_like(out, 7.0, dtype=torch.bfloat16)
    kv8.attention(q, cache, half, q_pos=pos, kv_len=kv_len, scale=d ** -0.5)
    torch.cuda.synchronize()
    assert torch.equal(half, out.to(torch.bfloat16))


@pytest.mark.parametrize("d,sq,H,Hkv", [(128, 1, 8, 2), (128, 5, 4, 4), (128, 48, 8, 2),
                                        (64, 70, 4, 2), (256, 2, 4, 2), (256, 90, 2, 1)])
@pytest.mark.parametrize("kw", [
    dict(window=20), dict(window=1), dict(prefix=150), dict(prefix=1 << 30),
    dict(window=64, prefix=120), dict(cap=50.0), dict(cap=5.0, window=100),
    dict(scale=-0.1), dict(scale=-0.1, cap=20.0),
])
def test_attention_masks(d, sq, H, Hkv, kw):
    run_attention(2, sq, H, Hkv, d, 333, 32, lens=[333, 201], where="scattered", **kw)


@pytest.mark.parametrize("sq,H,Hkv", [(1, 4, 2), (48, 8, 2)])
def test_attention_rows_that_see_nothing(sq, H, Hkv):
    # Lengths of zero, and a window of zero: NaN, as the reference's 0 / 0.
    q, cache, out, pos, kv_len = run_attention(3, sq, H, Hkv, 128, 96, 32, lens=[96, 0, 48],
                                               where="scattered")
    assert bool(torch.isnan(out[1]).all()) and not bool(torch.isnan(out[0]).any())
    run_attention(1, sq, H, Hkv, 128, 96, 32, window=0, where="scattered")
    # Some rows of a tile see keys, others none (positions far past the end).
    pos = pos.clone()
    pos[0, ::2] = 4000
    kv8.attention(q, cache, out, q_pos=pos, kv_len=kv_len, sliding_window=30, scale=0.1)
    torch.cuda.synchronize()
    check_attention(q, cache, out, pos, [96, 0, 48], scale=0.1, window=30)


@pytest.mark.parametrize("sq", [1, 40])
def test_attention_ignores_what_lies_past_the_length(sq):
    # NaN codes, infinite and NaN scales past what is held, and other
    # sequences' rows, have no part in the result.
    g = torch.Generator().manual_seed(3)
    T, n, B = 32, 300, 2
    cache = cache_of(g, B, n, 2, 128, T)
    q = torch.randn(B, sq, 8, 128, generator=g).to(torch.bfloat16).cuda()
    lens = [170, 64]
    kv_len = torch.tensor(lens, dtype=torch.int32).cuda()
    for b, ln in enumerate(lens):
        cache.k[b, ln:] = 0x7f
        cache.v[b, ln:] = 0xff
        first = -(-ln // T)
        cache.k_scale[b, first:] = float("inf")
        cache.v_scale[b, first:] = float("nan")
    out = torch.empty(B, sq, 8, 128, device="cuda")
    kv8.attention(q, cache, out, kv_len=kv_len, scale=0.09)
    torch.cuda.synchronize()
    pos = torch.stack([torch.arange(sq) + ln - sq for ln in lens])
    check_attention(q, cache, out, pos, lens, scale=0.09)
    assert not bool(torch.isnan(out).any())


@pytest.mark.parametrize("sq,hd", [(1, 128), (1, 64), (2, 256), (48, 128)])
def test_attention_split_keys_join(sq, hd):
    # A long axis over one sequence: split over CTAs and joined; without a
    # workspace it is not split. Both against the reference, twice for the
    # tickets' return to zero, and bit for bit the same both times.
    q, cache, out, pos, kv_len = run_attention(1, sq, 4, 2, hd, 5000, 64, lens=[4987])
    a = kv8.make_attention_args(q, cache, out, q_pos=pos, kv_len=kv_len, scale=hd ** -0.5)
    assert kv8.workspace_bytes(a) > 0
    ws = a._keep[-1]
    first = None
    for _ in range(3):
        out.fill_(7.0)
        kv8.attention_args(a)
        torch.cuda.synchronize()
        assert int(ws[:kv8.TICKET_BYTES].sum()) == 0
        first = out.clone() if first is None else first
        assert torch.equal(out, first)
    run_attention(1, sq, 4, 2, hd, 5000, 64, lens=[4987], workspace=False)


def test_attention_scales_of_any_size():
    # V scales far apart from block to block ride in the exponent: a block of
    # tiny values with large weights, and the other way round. Scales that are
    # not powers of two are taken as they are.
    g = torch.Generator().manual_seed(9)
    for sq in (1, 40):
        cache = cache_of(g, 1, 256, 2, 128, 32)
        cache.v_scale *= torch.pow(2.0, torch.randint(-40, 40, cache.v_scale.shape,
                                                      generator=g).float()).cuda()
        cache.k_scale *= 0.7
        cache.v_scale *= 1.3
        q = (2 * torch.randn(1, sq, 4, 128, generator=g)).to(torch.bfloat16).cuda()
        out = torch.empty(1, sq, 4, 128, device="cuda")
        kv8.attention(q, cache, out, scale=0.1)
        torch.cuda.synchronize()
        check_attention(q, cache, out, torch.arange(sq).view(1, -1) + 256 - sq, [256], scale=0.1)


def test_attention_loud_and_quiet_queries():
    # Rows of Q of any magnitude: scaled by a power of two before f16.
    for sq in (1, 40):
        for qscale in (2.0 ** -30, 2.0 ** 20):
            run_attention(1, sq, 8, 2, 128, 200, 32, qscale=qscale, scale=0.1 / qscale)


def test_attention_nan_and_infinite_queries():
    # Such a row is NaN, its neighbours are not touched.
    g = torch.Generator().manual_seed(12)
    for sq, d in ((1, 128), (40, 128), (40, 256), (2, 512)):
        cache = cache_of(g, 1, 200, 2, d, 32)
        q = torch.randn(1, sq, 4, d, generator=g).to(torch.bfloat16).cuda()
        clean = torch.empty(1, sq, 4, d, device="cuda")
        kv8.attention(q, cache, clean, scale=0.1)
        for bad in (float("nan"), float("inf"), float("-inf")):
            q2, out = q.clone(), torch.empty_like(clean)
            q2[0, sq - 1, 1, 3] = bad
            kv8.attention(q2, cache, out, scale=0.1)
            torch.cuda.synchronize()
            assert ca.device_status() == ca.CA_OK
            assert bool(torch.isnan(out[0, sq - 1, 1]).all()), (sq, d, bad)
            out[0, sq - 1, 1] = clean[0, sq - 1, 1]
            assert torch.equal(out, clean), (sq, d, bad)


def test_attention_sink_and_flat_tail():
    # One key with nearly all the weight of a row, and thousands whose weights
    # are 2^-20 of it but add up.
    g = torch.Generator().manual_seed(4)
    n = 8192
    for sq in (1, 40):
        cache = cache_of(g, 1, n, 1, 128, 32)
        cache.k[:] = 0
        cache.k[0, 5, 0, 0] = 0x38 + 8 * 3  # 8.0
        cache.k_scale[:] = 1.0
        q = torch.zeros(1, sq, 2, 128, dtype=torch.bfloat16, device="cuda")
        q[..., 0] = 1.75
        out = torch.empty(1, sq, 2, 128, device="cuda")
        kv8.attention(q, cache, out, scale=1.0)
        torch.cuda.synchronize()
        check_attention(q, cache, out, torch.arange(sq).view(1, -1) + n - sq, [n], scale=1.0)


def test_attention_varlen_queries_and_strides():
    g = torch.Generator().manual_seed(5)
    B, n, H, Hkv, d, T = 4, 200, 8, 2, 128, 32
    lens, counts = [200, 131, 64, 1], [37, 0, 64, 1]
    wide = cache_of(g, B, n, 2 * Hkv, d, T)  # this cache's heads are the first half of wider rows
    cache = kv8.Kv8Cache(wide.k[:, :, :Hkv], wide.v[:, :, :Hkv],
                         wide.k_scale[:, :, :Hkv].contiguous(),
                         wide.v_scale[:, :, :Hkv].contiguous(), T)
    total = sum(counts)
    qkv = torch.randn(total, H + 3, d, generator=g).to(torch.bfloat16).cuda()
    q = qkv[:, :H]
    buf = torch.full((total, H + 2, d), 7.0, device="cuda")
    out = buf[:, :H]
    cu = torch.tensor([0] + list(torch.tensor(counts).cumsum(0)), dtype=torch.int32).cuda()
    kv_len = torch.tensor(lens, dtype=torch.int32).cuda()
    pos = torch.cat([torch.arange(c) + ln - c for c, ln in zip(counts, lens)]).to(torch.int32).cuda()
    prefix = torch.tensor([170, -1, 32, 5], dtype=torch.int32).cuda()
    kv8.attention(q, cache, out, cu_q=cu, max_sq=64, q_pos=pos, kv_len=kv_len, seq_prefix=prefix,
                  scale=d ** -0.5)
    torch.cuda.synchronize()
    k = held_values(cache.k.contiguous(), cache.k_scale, T)
    v = held_values(cache.v.contiguous(), cache.v_scale, T)
    at = 0
    for b in range(B):
        r = slice(at, at + counts[b])
        at += counts[b]
        if not counts[b]:
            continue
        pre = int(prefix[b])
        ref, mag = attention_ref(q[r], k[b], v[b], pos[r], lens[b], scale=d ** -0.5,
                                 prefix=None if pre < 0 else pre)
        assert bool(((out[r].double() - ref).abs() <= 2.0 ** -10 * mag + 1e-30).all()), b
    assert bool((buf[:, H:] == 7.0).all())


def test_attention_on_another_stream():
    g = torch.Generator().manual_seed(6)
    cache = cache_of(g, 1, 3000, 2, 128, 32)
    q = torch.randn(1, 1, 8, 128, generator=g).to(torch.bfloat16).cuda()
    out = torch.empty(1, 1, 8, 128, device="cuda")
    a = kv8.make_attention_args(q, cache, out, scale=0.1)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    kv8.attention_args(a, s)
    torch.cuda.current_stream().wait_stream(s)
    check_attention(q, cache, out, torch.tensor([[2999]]), [3000], scale=0.1)


def test_attention_in_a_graph():
    g = torch.Generator().manual_seed(7)
    cache = cache_of(g, 1, 3000, 2, 128, 32)
    q = torch.randn(1, 1, 8, 128, generator=g).to(torch.bfloat16).cuda()
    out = torch.empty(1, 1, 8, 128, device="cuda")
    a = kv8.make_attention_args(q, cache, out, scale=0.1)
    kv8.attention_args(a)
    torch.cuda.synchronize()
    want = out.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        kv8.attention_args(a, torch.cuda.current_stream())
    for _ in range(3):
        out.zero_()
        graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, want)


# ------------------------------------------------------------------ store
def store_case(B, n, Hkv, d, T, counts, lens, *, seed=1, loud=1.0, start=True, where="scattered",
               new=None):
    """Runs the store and its restatement; returns what they left."""
    g = torch.Generator().manual_seed(seed)
    cache = cache_of(g, B, n, Hkv, d, T)
    if not start:
        cache = kv8.Kv8Cache.alloc(B, n, Hkv, d, block_tokens=T)
    pos, rows, at = [], [], 0
    for b, c in enumerate(counts):
        if where == "scattered":
            p = torch.randperm(n, generator=g)[:c].sort().values
        else:
            p = torch.arange(c) + (lens[b] if lens is not None else n) - (0 if where == "tail" else c)
        pos.append(p)
        rows.append((at, at + c))
        at += c
    pos = torch.cat(pos).to(torch.int32)
    if new is None:
        new = [(loud * torch.randn(at, Hkv, d, generator=g)).to(torch.bfloat16) for _ in range(2)]
    held_len = lens if lens is not None else [n] * B
    kv_len = None if lens is None else torch.tensor(lens, dtype=torch.int32).cuda()
    want = []
    for held, scale, x in ((cache.k, cache.k_scale, new[0]), (cache.v, cache.v_scale, new[1])):
        h64, s64 = held.cpu().view(F8).double(), scale.cpu().double()
        store_ref(h64, s64, T, x.double(), rows, pos, n, held_len)
        want.append((h64, s64))
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    uniform = len(set(counts)) == 1
    cu = None if uniform else torch.tensor([0] + [r[1] for r in rows], dtype=torch.int32).cuda()
    kv8.store(cache, new[0].cuda(), new[1].cuda(), pos.cuda(), cu_active=cu, kv_len=kv_len,
              status=status)
    torch.cuda.synchronize()
    assert int(status) == 0
    for (h64, s64), held, scale in zip(want, (cache.k, cache.v), (cache.k_scale, cache.v_scale)):
        assert torch.equal(scale.cpu().double(), s64)
        assert torch.equal(held.cpu().view(F8).double(), h64)
    return cache


@pytest.mark.parametrize("B,n,Hkv,d,T,counts,lens,where", [
    (1, 1, 1, 16, 16, [1], None, "scattered"),
    (2, 40, 2, 128, 16, [5, 5], None, "scattered"),
    (2, 100, 3, 64, 32, [100, 100], None, "scattered"),       # every position
    (1, 131, 2, 256, 128, [130], None, "scattered"),          # all but one
    (3, 150, 2, 128, 64, [1, 1, 1], [0, 63, 149], "tail"),    # one token each
    (2, 300, 1, 80, 32, [70, 70], [0, 101], "tail"),
    (3, 90, 2, 128, 32, [0, 33, 90], None, "scattered"),      # ragged
    (2, 64, 2, 512, 128, [64, 3], None, "scattered"),
    (4, 1000, 4, 128, 32, [400] * 4, None, "scattered"),
])
@pytest.mark.parametrize("loud", [0.01, 1.0, 50.0])
def test_store_matches_definition(B, n, Hkv, d, T, counts, lens, where, loud):
    store_case(B, n, Hkv, d, T, counts, lens, where=where, loud=loud)


def test_store_many_rows_a_job():
    # More rows than warps of the GPU: a warp looks through up to 32 entries.
    store_case(2, 3000, 4, 16, 32, [3000, 3000], None, loud=2.0)
    store_case(2, 3000, 4, 16, 16, [2500, 2500], None, loud=2.0)


def test_store_into_an_empty_cache_then_grow():
    store_case(2, 96, 2, 128, 32, [9, 9], None, start=False)
    store_case(2, 96, 2, 128, 32, [9, 9], [0, 0], start=False)


def test_store_zeros_and_extremes():
    g = torch.Generator().manual_seed(8)
    z = torch.zeros(4, 1, 64, dtype=torch.bfloat16)
    store_case(1, 40, 1, 64, 16, [4], None, new=[z, z.clone()])
    x = torch.randn(4, 1, 64, generator=g)
    for f in (2.0 ** -80, 2.0 ** -60, 2.0 ** 100, 3e38 / 5):
        y = (x * f).clamp(-3.3e38, 3.3e38).to(torch.bfloat16)
        store_case(1, 40, 1, 64, 16, [4], [0], where="tail", new=[y, y.clone()])
    # The edge 448 * 2^k, one bf16 step past it, and ties of e4m3.
    y = torch.zeros(4, 1, 64)
    y[0, 0, 0], y[1, 0, 0] = 448.0, 450.0
    y[:, :, 1:] = torch.arange(4 * 63).view(4, 1, 63) * 0.5
    store_case(1, 64, 1, 64, 16, [4], [0], where="tail", new=[y.to(torch.bfloat16)] * 2)
    y[1, 0, 0] = 3.0
    store_case(1, 64, 1, 64, 16, [4], [0], where="tail", new=[y.to(torch.bfloat16)] * 2)


def test_store_infinities_and_nan():
    x = torch.ones(2, 1, 64, dtype=torch.bfloat16)
    x[0, 0, 3], x[1, 0, 5] = float("nan"), -2.0
    cache = kv8.Kv8Cache.alloc(1, 32, 1, 64, block_tokens=16)
    pos = torch.tensor([3, 7], dtype=torch.int32).cuda()
    kv8.store(cache, x.cuda(), x.cuda(), pos)
    k = held_values(cache.k, cache.k_scale, 16).cpu()
    assert bool(torch.isnan(k[0, 3, 0, 3])) and int(torch.isnan(k).sum()) == 1
    assert float(k[0, 7, 0, 5]) == -2.0 and float(k[0, 7, 0, 6]) == 1.0
    x[0, 0, 3] = float("inf")
    kv8.store(cache, x.cuda(), x.cuda(), pos)
    out = torch.empty(1, 32, 1, 64, device="cuda")
    kv8.load(cache, out, None)
    assert float(out[0, 3, 0, 3]) == float("inf")


def test_store_reports_bad_positions():
    cache = kv8.Kv8Cache.alloc(1, 32, 1, 64, block_tokens=16)
    x = torch.ones(3, 1, 64, dtype=torch.bfloat16, device="cuda")
    for bad in ([0, 5, 32], [-1, 3, 4], [4, 2, 20], [7, 7, 9]):
        status = torch.zeros(1, dtype=torch.int32, device="cuda")
        kv8.store(cache, x, x, torch.tensor(bad, dtype=torch.int32).cuda(), status=status)
        torch.cuda.synchronize()
        assert int(status) == ca.CA_ERR_INVALID, bad
    # Rows up to the first bad one of their block were written; no other position was.
    out = torch.empty(1, 32, 1, 64, device="cuda")
    kv8.load(cache, out, None)
    seen = set(torch.nonzero(out[0, :, 0, 0]).flatten().tolist())
    assert seen <= {0, 3, 4, 5, 7, 9, 20} and {0, 3, 4, 5, 7, 20} <= seen


def test_store_of_every_row_checks_its_positions():
    # As many rows as positions, but one of them elsewhere: its block is left
    # as it was and reported, the others are written.
    n, T = 100, 32
    cache = kv8.Kv8Cache.alloc(2, n, 3, 64, block_tokens=T)
    x = torch.ones(2, n, 3, 64, dtype=torch.bfloat16, device="cuda")
    pos = torch.arange(n, dtype=torch.int32).repeat(2, 1)
    pos[1, 40] = 39
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    kv8.store(cache, x, 2 * x, pos.cuda(), status=status)
    torch.cuda.synchronize()
    assert int(status) == ca.CA_ERR_INVALID
    for held, scale, want in ((cache.k, cache.k_scale, 1.0), (cache.v, cache.v_scale, 2.0)):
        y = held_values(held, scale, T)
        assert bool((y[0] == want).all()) and bool((y[1, 64:] == want).all())
        assert bool((y[1, :32] == want).all()) and bool((y[1, 32:64] == 0).all())


# ------------------------------------------------------------------ load
@pytest.mark.parametrize("B,n,Hkv,d,T,n_pos,dtype", [
    (1, 1, 1, 16, 16, 1, torch.bfloat16), (2, 100, 2, 128, 32, 100, torch.bfloat16),
    (3, 77, 4, 64, 16, 20, torch.float32), (2, 300, 3, 256, 128, 299, torch.bfloat16),
    (2, 50, 2, 80, 64, 50, torch.float32),
])
def test_load(B, n, Hkv, d, T, n_pos, dtype):
    g = torch.Generator().manual_seed(2)
    cache = cache_of(g, B, n, Hkv, d, T)
    pos = torch.stack([torch.randperm(n, generator=g)[:n_pos] for _ in range(B)])
    p32 = pos.to(torch.int32).cuda()
    for use in (p32, None):
        outs = [torch.full((B, n_pos, Hkv, d), 7.0, dtype=dtype, device="cuda") for _ in range(2)]
        kv8.load(cache, outs[0], outs[1], use)
        at = pos.cuda() if use is not None else torch.arange(n_pos, device="cuda").expand(B, -1)
        for held, scale, out in ((cache.k, cache.k_scale, outs[0]),
                                 (cache.v, cache.v_scale, outs[1])):
            want = held_values(held, scale, T)[torch.arange(B).view(-1, 1).cuda(), at]
            assert torch.equal(out.double(), want)
    only = torch.full((B, n_pos, Hkv, d), 7.0, dtype=dtype, device="cuda")
    kv8.load(cache, None, only, p32)
    assert torch.equal(only, only.clone()) and not bool((only == 7.0).all())


def test_load_reports_bad_positions():
    g = torch.Generator().manual_seed(2)
    cache = cache_of(g, 1, 20, 1, 64, 16)
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    out = torch.full((1, 3, 1, 64), 7.0, device="cuda")
    kv8.load(cache, out, None, torch.tensor([[1, 20, -1]], dtype=torch.int32).cuda(),
             status=status)
    assert int(status) == ca.CA_ERR_INVALID
    assert bool((out[0, 1:] == 7.0).all()) and not bool((out[0, 0] == 7.0).any())


# ------------------------------------------------------------------ block
@pytest.mark.parametrize("hd,rope_dim,ragged", [(64, 64, False), (128, 64, False), (128, 128, True),
                                                (256, 256, False), (80, 32, True)])
def test_block_is_its_parts(hd, rope_dim, ragged):
    # Norms and RoPE as the bf16 block leaves them (its cache and q_work), the
    # store and the attention of this cache: the same bits in one call.
    g = torch.Generator().manual_seed(hd)
    B, n, H, Hkv, T = 3, 300, 4, 2, 32
    counts = [50, 1, 23] if ragged else [40] * B
    total = sum(counts)
    bf = torch.bfloat16
    q, k, v = (torch.randn(total, h, hd, generator=g).to(bf).cuda() for h in (H, Hkv, Hkv))
    pos = torch.cat([torch.randperm(n, generator=g)[:c].sort().values for c in counts])
    pos = pos.to(torch.int32).cuda()
    wq, wk = (torch.rand(hd, generator=g).cuda() + 0.5 for _ in range(2))
    rope = torch.from_numpy(ca.build_rope_cache(n, rope_dim, 1e4)).cuda()
    kw = dict(active_pos=pos, rope=rope, rope_len=n, rope_dim=rope_dim, q_norm_w=wq, k_norm_w=wk,
              v_norm=True, rms_eps=1e-6, scale=hd ** -0.5)
    at = [0]
    for c in counts:
        at.append(at[-1] + c)
    cu = torch.tensor(at, dtype=torch.int32).cuda()
    k16 = torch.zeros(B * n, Hkv, hd, dtype=bf, device="cuda")
    v16 = torch.zeros_like(k16)
    q_work, out16 = torch.empty_like(q), torch.empty_like(q)
    ca.attention_block_dev(q, k, v, batch=B, n_active=0, cache_k=k16, cache_v=v16, n_total=0,
                           q_work=q_work, out=out16, n_head=H, n_head_kv=Hkv, head_dim=hd,
                           cu_active=cu, cu_total=(torch.arange(B + 1, dtype=torch.int32) * n).cuda(),
                           max_active=max(counts), total_active=total, total_cache=B * n, **kw)
    rows = torch.cat([pos[a:b].long() + i * n for i, (a, b) in enumerate(zip(at, at[1:]))])
    parts = cache_of(g, B, n, Hkv, hd, T)
    whole = kv8.Kv8Cache(parts.k.clone(), parts.v.clone(), parts.k_scale.clone(),
                         parts.v_scale.clone(), T)
    kv8.store(parts, k16[rows], v16[rows], pos, cu_active=cu)
    want = torch.full((total, H, hd), 7.0, device="cuda")
    kv8.attention(q_work, parts, want, cu_q=cu, max_sq=max(counts), q_pos=pos, scale=hd ** -0.5,
                  sliding_window=100)
    got = torch.full_like(want, 8.0)
    if ragged:
        kv8.attention_block(q, k, v, whole, got, cu_active=cu, max_active=max(counts),
                            sliding_window=100, **kw)
    else:
        four = lambda x: x.view((B, counts[0]) + x.shape[1:])  # noqa: E731
        kv8.attention_block(four(q), four(k), four(v), whole, four(got), sliding_window=100, **kw)
    torch.cuda.synchronize()
    for name in ("k", "v", "k_scale", "v_scale"):
        assert torch.equal(getattr(whole, name), getattr(parts, name)), name
    assert torch.equal(got, want)


def test_example_runs():
    import importlib.util
    import os
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    spec = importlib.util.spec_from_file_location(
        "kv8_denoise", os.path.join(root, "examples", "kv8_denoise.py"))
    m = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(m)
    far, same = m.main(["--batch", "2", "--total", "256", "--steps", "3", "--layers", "2"])
    # A value of 4 significant bits is within 2^-4 of what it stands for.
    assert max(far) < 2.0 ** -4 and min(same) > 0.5


def test_offsets_past_32_bits():
    # A cache of more than 2^32 bytes: the last sequence's rows.
    B, n, Hkv, d, T = 17, 131072, 16, 128, 128
    if torch.cuda.mem_get_info()[0] < 24 << 30:
        pytest.skip("needs 24 GB free")
    cache = kv8.Kv8Cache.alloc(B, n, Hkv, d, block_tokens=T)
    assert cache.k.numel() > 1 << 32
    g = torch.Generator().manual_seed(2)
    m = 200
    new = torch.randn(B * m, Hkv, d, generator=g).to(torch.bfloat16).cuda()
    pos = torch.arange(n - m, n, dtype=torch.int32).repeat(B).cuda()
    kv8.store(cache, new, new, pos)
    out = torch.empty(B, m, Hkv, d, dtype=torch.bfloat16, device="cuda")
    kv8.load(cache, out, None, pos)
    rel = (out.view_as(new).double() - new.double()).norm() / new.double().norm()
    assert float(rel) < 2.0 ** -4  # e4m3 keeps 4 bits: at most 2^-4 of each value
    for sq in (1, 40):
        q = torch.randn(B, sq, Hkv, d, generator=g).to(torch.bfloat16).cuda()
        res = torch.empty(B, sq, Hkv, d, device="cuda")
        qp = torch.full((B, sq), n - 1, dtype=torch.int32, device="cuda")
        kv8.attention(q, cache, res, q_pos=qp, sliding_window=m, scale=0.1)
        torch.cuda.synchronize()
        k = held_values(cache.k[B - 1:, n - 256:].contiguous(), cache.k_scale[B - 1:, -2:], T)[0]
        v = held_values(cache.v[B - 1:, n - 256:].contiguous(), cache.v_scale[B - 1:, -2:], T)[0]
        ref, mag = attention_ref(q[-1], k, v, qp[-1] - (n - 256), 256, scale=0.1, window=m)
        assert bool(((res[-1].double() - ref).abs() <= 2.0 ** -10 * mag + 1e-30).all())
