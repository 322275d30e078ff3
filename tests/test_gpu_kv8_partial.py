"""Attention over 8-bit caches of which only a part was stored: the blocks
past a sequence's length hold scale 0 (nothing written) or whatever an
allocation that was not zeroed holds, and have no part in the result. The
tolerance is that of test_gpu_kv8.py."""
import pytest
import torch

import canvas_attn as ca
from canvas_attn import kv8
from test_gpu_kv8 import cache_of, check_attention

pytestmark = pytest.mark.gpu


def partly_stored(g, lens, n, Hkv, d, T, fill=0.0):
    """A fresh cache with `lens` positions of each sequence stored; K scales
    of the blocks past them are `fill`."""
    B = len(lens)
    cache = kv8.Kv8Cache.alloc(B, n, Hkv, d, block_tokens=T)
    pos = torch.cat([torch.arange(ln) for ln in lens]).to(torch.int32).cuda()
    new = [torch.randn(sum(lens), Hkv, d, generator=g).to(torch.bfloat16).cuda() for _ in range(2)]
    cu = torch.tensor([0] + list(torch.tensor(lens).cumsum(0)), dtype=torch.int32).cuda()
    kv8.store(cache, new[0], new[1], pos, cu_active=cu,
              kv_len=torch.zeros(B, dtype=torch.int32, device="cuda"))
    for b, ln in enumerate(lens):
        cache.k_scale[b, -(-ln // T):] = fill
    return cache


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("sq", [1, 17, 200])
@pytest.mark.parametrize("fill", [0.0, float("nan"), -1.0, float("inf")])
def test_blocks_that_were_never_written(d, sq, fill):
    # Lengths that leave unwritten blocks in the last tile of 64 or 128 keys.
    g = torch.Generator().manual_seed(d + sq)
    lens = [300, 205]
    cache = partly_stored(g, lens, 512, 2, d, 16, fill)
    q = torch.randn(2, sq, 4, d, generator=g).to(torch.bfloat16).cuda()
    kv_len = torch.tensor(lens, dtype=torch.int32).cuda()
    pos = torch.stack([torch.arange(sq) + ln - sq for ln in lens]).to(torch.int32).cuda()
    for kw in (dict(), dict(window=50), dict(prefix=250), dict(cap=20.0)):
        out = torch.full((2, sq, 4, d), 7.0, device="cuda")
        names = dict(window="sliding_window", prefix="causal_prefix", cap="softcap")
        kv8.attention(q, cache, out, q_pos=pos, kv_len=kv_len, scale=d ** -0.5,
                      **{names[k]: v for k, v in kw.items()})
        torch.cuda.synchronize()
        assert ca.device_status() == ca.CA_OK
        check_attention(q, cache, out, pos, lens, what=str(kw), scale=d ** -0.5, **kw)
        assert not bool(torch.isnan(out).any())


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("fill", [0.0, float("nan")])
def test_unwritten_blocks_below_a_window(d, fill):
    # 40 rows see positions 311 on; blocks below 304 share their first tile.
    g = torch.Generator().manual_seed(d)
    n, sq, T = 400, 40, 16
    cache = cache_of(g, 1, n, 2, d, T)
    cache.k_scale[:, :19] = fill
    cache.v_scale[:, :19] = fill
    q = torch.randn(1, sq, 4, d, generator=g).to(torch.bfloat16).cuda()
    out = torch.full((1, sq, 4, d), 7.0, device="cuda")
    pos = torch.arange(n - sq, n, dtype=torch.int32, device="cuda").view(1, -1)
    kv8.attention(q, cache, out, q_pos=pos, sliding_window=50, scale=d ** -0.5)
    torch.cuda.synchronize()
    check_attention(q, cache, out, pos, [n], scale=d ** -0.5, window=50)
    assert not bool(torch.isnan(out).any())


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("sq", [1, 40])
def test_zero_queries_over_zero_keys(d, sq):
    # A row of zeros and a block of zeros (scale 2^-64): the product of their
    # scales is below what fp32 holds, beside keys that are masked.
    g = torch.Generator().manual_seed(d)
    n, T = 300, 32
    cache = cache_of(g, 1, n, 2, d, T)
    z = torch.zeros(T, 2, d, dtype=torch.bfloat16, device="cuda")
    at = torch.arange(256, 256 + T, dtype=torch.int32, device="cuda")
    keep = cache.v.clone(), cache.v_scale.clone()
    kv8.store(cache, z, z, at)
    cache.v, cache.v_scale = keep
    assert float(cache.k_scale[0, 8, 0]) == 2.0 ** -64
    q = torch.randn(1, sq, 4, d, generator=g).to(torch.bfloat16).cuda()
    q[0, -1, 1] = 0
    q[0, 0, 2] = 2.0 ** -100
    pos = torch.arange(n - sq, n, dtype=torch.int32, device="cuda").view(1, -1)
    for kw in (dict(), dict(window=100), dict(prefix=290)):
        out = torch.full((1, sq, 4, d), 7.0, device="cuda")
        kv8.attention(q, cache, out, q_pos=pos, scale=0.1, sliding_window=kw.get("window"),
                      causal_prefix=kw.get("prefix"))
        torch.cuda.synchronize()
        check_attention(q, cache, out, pos, [n], what=str(kw), scale=0.1, **kw)
        assert not bool(torch.isnan(out).any())


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("sq", [1, 40])
@pytest.mark.parametrize("cap", [0.0, 30.0])
def test_scale_of_zero_is_the_mean(d, sq, cap):
    g = torch.Generator().manual_seed(d)
    n = 300
    cache = cache_of(g, 1, n, 2, d, 32)
    q = torch.randn(1, sq, 4, d, generator=g).to(torch.bfloat16).cuda()
    pos = torch.arange(n - sq, n, dtype=torch.int32, device="cuda").view(1, -1)
    for window in (None, 70):
        out = torch.full((1, sq, 4, d), 7.0, device="cuda")
        kv8.attention(q, cache, out, q_pos=pos, scale=0.0, sliding_window=window, softcap=cap)
        torch.cuda.synchronize()
        check_attention(q, cache, out, pos, [n], scale=0.0, window=window, cap=cap)
        assert not bool(torch.isnan(out).any())


@pytest.mark.parametrize("d", [64, 128, 256])
def test_block_stores_and_attends_a_prompt_in_a_larger_cache(d):
    # The fused block over a fresh cache: a prompt, then a canvas after it.
    # Nothing is rotated or normed, so its queries are q itself.
    g = torch.Generator().manual_seed(d)
    B, n, T = 2, 4096, 32
    cache = kv8.Kv8Cache.alloc(B, n, 2, d, block_tokens=T)
    rope = torch.zeros(n, 2, device="cuda")
    held = 0
    for rows in (300, 32, 1):
        q, k, v = (torch.randn(B, rows, h, d, generator=g).to(torch.bfloat16).cuda()
                   for h in (4, 2, 2))
        pos = torch.arange(held, held + rows, dtype=torch.int32, device="cuda").repeat(B, 1)
        before = torch.full((B,), held, dtype=torch.int32, device="cuda")
        held += rows
        out = torch.full((B, rows, 4, d), 7.0, device="cuda")
        status = torch.zeros(1, dtype=torch.int32, device="cuda")
        kv8.attention_block(q, k, v, cache, out, active_pos=pos, rope=rope, rope_len=n, rope_dim=0,
                            held=before, kv_len=before + rows, scale=d ** -0.5, status=status)
        torch.cuda.synchronize()
        assert int(status) == 0 and ca.device_status() == ca.CA_OK
        check_attention(q, cache, out, pos, [held] * B, what=f"{rows} rows", scale=d ** -0.5)
        assert not bool(torch.isnan(out).any())
