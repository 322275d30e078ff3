"""The 8-bit cache's store where a block's rows are more than a job keeps in
registers (they are then read twice), and the read-back of one tensor alone:
bit for bit."""
import pytest
import torch

from canvas_attn import kv8
from kv8_helpers import held_values
from test_gpu_kv8 import cache_of, store_case

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("hd", [256, 512])
@pytest.mark.parametrize("n", [300, 256])
def test_store_of_every_row_in_wide_blocks(hd, n):
    # 128 rows of 16 or 32 units: two or four passes of four warps, and a last
    # block that is partly filled.
    store_case(2, n, 2, hd, 128, [n, n], None, loud=3.0)


@pytest.mark.parametrize("hd,Hkv,counts", [
    (256, 8, [2100]),             # nearly every row of one sequence
    (256, 16, [700, 0, 401]),     # ragged
    (512, 16, [600, 500]),
    (512, 16, [1100, 3]),
])
@pytest.mark.parametrize("loud", [0.02, 1.0, 60.0])
def test_store_of_many_rows_in_wide_blocks(hd, Hkv, counts, loud):
    # At least eight times as many (row, head) pairs as the GPU has warps at
    # half load: jobs of four warps. The rows that stay keep their bits (quiet
    # new rows) or are rounded again to the grown scale (loud ones).
    assert sum(counts) * 2 * Hkv > 7 * 148 * 32
    store_case(len(counts), max(counts) + 400, Hkv, hd, 128, counts, None, loud=loud)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("n_pos", [37, 300])
def test_load_of_one_tensor(dtype, n_pos):
    g = torch.Generator().manual_seed(4)
    B, n, Hkv, d, T = 3, 300, 5, 112, 32
    cache = cache_of(g, B, n, Hkv, d, T)
    pos = torch.stack([torch.randperm(n, generator=g)[:n_pos] for _ in range(B)])
    p32 = pos.to(torch.int32).cuda()
    rows = torch.arange(B).view(-1, 1).cuda(), pos.cuda()
    for held, scale, first in ((cache.k, cache.k_scale, True), (cache.v, cache.v_scale, False)):
        out = torch.full((B, n_pos, Hkv, d), 7.0, dtype=dtype, device="cuda")
        kv8.load(cache, out if first else None, None if first else out, p32)
        assert torch.equal(out.double(), held_values(held, scale, T)[rows])
