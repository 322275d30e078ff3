"""The fused block over the 8-bit cache with positions out of range: they are
reported, nothing is read or written outside the tables and the cache, and the
other rows are as if those were not there. Sizes for each form of the pre-ops
pass: scalar, token, bulk copies, pairs, ring."""
import pytest
import torch

import canvas_attn as ca
from canvas_attn import kv8
from test_gpu_kv8 import cache_of

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("hd,rope_dim,H,Hkv,rows,n", [
    (80, 32, 4, 2, 40, 200),       # one warp a row, scalar
    (128, 128, 4, 2, 40, 200),     # vectors, a token a warp
    (256, 256, 4, 2, 40, 200),     # bulk copies
    (256, 256, 56, 4, 20, 100),    # rotation pairs in a lane
    (64, 64, 16, 8, 8192, 9000),   # ring
])
def test_block_reports_positions_out_of_range(hd, rope_dim, H, Hkv, rows, n):
    g = torch.Generator().manual_seed(hd + H)
    T = 32
    q, k, v = (torch.randn(rows, h, hd, generator=g).to(torch.bfloat16).cuda()
               for h in (H, Hkv, Hkv))
    pos = torch.randperm(n, generator=g)[:rows].sort().values.to(torch.int32)
    pos[0], pos[-2], pos[-1] = -5, n, 1 << 30
    good = slice(1, rows - 2)
    rope = torch.from_numpy(ca.build_rope_cache(n, rope_dim, 1e4)).cuda()
    kw = dict(rope=rope, rope_len=n, rope_dim=rope_dim, scale=hd ** -0.5)
    clean = cache_of(g, 1, n, Hkv, hd, T)
    cache = kv8.Kv8Cache(clean.k.clone(), clean.v.clone(), clean.k_scale.clone(),
                         clean.v_scale.clone(), T)

    def block(c, part):
        out = torch.full((1,) + tuple(q[part].shape), 7.0, device="cuda")
        status = torch.zeros(1, dtype=torch.int32, device="cuda")
        kv8.attention_block(q[part].unsqueeze(0), k[part].unsqueeze(0), v[part].unsqueeze(0), c,
                            out, active_pos=pos[part].cuda(), status=status, **kw)
        torch.cuda.synchronize()
        return out[0], int(status)

    want, status = block(clean, good)
    assert status == 0
    out, status = block(cache, slice(0, rows))
    assert status == ca.CA_ERR_INVALID and ca.device_status() == ca.CA_OK
    for name in ("k", "v", "k_scale", "v_scale"):
        assert torch.equal(getattr(cache, name), getattr(clean, name)), name
    # The same rows in other tiles: fp32 sums of weights rounded to f16.
    assert float((out[good] - want).abs().max()) <= 2.0 ** -10 * 16
