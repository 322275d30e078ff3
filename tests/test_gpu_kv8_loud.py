"""Attention over the 8-bit cache with query rows that have loud channels.

Q enters the products as two e4m3 terms of a row scaled by 2^-e so that its
largest magnitude is in (224, 448]. The second term's step is at least 2^-9,
so an element is off by at most 2^-10 of 2^e, hence a score by at most
delta = scale 2^(e - 10) max_k |k|_1, a weight by a factor within e^(2 delta),
and an output by (e^(2 delta) - 1) sum p |v|, over the 2^-10 sum p |v| of
test_gpu_kv8.py."""
import pytest
import torch

import canvas_attn as ca
from canvas_attn import kv8
from kv8_helpers import attention_ref, held_values
from test_gpu_kv8 import cache_of

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("sq,d", [(1, 64), (40, 64), (1, 128), (40, 128), (2, 256), (40, 256),
                                  (3, 512)])
@pytest.mark.parametrize("loud", [2.0 ** 3, 2.0 ** 7, 2.0 ** 11])
def test_loud_channels(sq, d, loud):
    g = torch.Generator().manual_seed(d)
    n = 400
    cache = cache_of(g, 1, n, 2, d, 32)
    # K is quiet where Q is loud: a code of e4m3 has its exponent from bit 3.
    at = torch.randperm(d, generator=g)[:3].cuda()
    cache.k[..., at] = (cache.k[..., at] & 0x80) | 0x08
    q = torch.randn(1, sq, 4, d, generator=g)
    q[..., at.cpu()] *= loud
    q = q.to(torch.bfloat16).cuda()
    out = torch.full((1, sq, 4, d), 7.0, device="cuda")
    kv8.attention(q, cache, out, scale=d ** -0.5)
    torch.cuda.synchronize()
    assert ca.device_status() == ca.CA_OK
    k = held_values(cache.k, cache.k_scale, 32)[0]
    v = held_values(cache.v, cache.v_scale, 32)[0]
    pos = torch.arange(n - sq, n)
    ref, mag = attention_ref(q[0], k, v, pos, n, scale=d ** -0.5)
    amax = q[0].double().abs().amax(dim=-1, keepdim=True)
    two_e = torch.exp2(torch.ceil(torch.log2(amax / 448)))
    delta = d ** -0.5 * two_e * 2.0 ** -10 * k.abs().sum(dim=-1).max()
    tol = (2.0 ** -10 + torch.expm1(2 * delta)) * mag
    assert bool(((out[0].double() - ref).abs() <= tol).all())
