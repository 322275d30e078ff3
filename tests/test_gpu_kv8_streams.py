"""The 8-bit cache's Python calls on other streams than torch's current one:
scratch that a call makes itself is cleared before its kernels run and not
handed on while they do. The tolerance is that of test_gpu_kv8.py."""
import pytest
import torch

import canvas_attn as ca
from canvas_attn import kv8
from test_gpu_kv8 import cache_of, check_attention

pytestmark = pytest.mark.gpu

HOLD = 40_000_000  # clocks: some 20 ms


def setup(n=3000, sq=1):
    g = torch.Generator().manual_seed(21)
    cache = cache_of(g, 1, n, 2, 128, 32)
    q = torch.randn(1, sq, 8, 128, generator=g).to(torch.bfloat16).cuda()
    out = torch.full((1, sq, 8, 128), 7.0, device="cuda")
    pos = torch.arange(n - sq, n, dtype=torch.int32, device="cuda").view(1, -1)
    torch.cuda.synchronize()
    return cache, q, out, pos


def litter(n_bytes):
    """Leaves blocks of that size that are not zero to torch's allocator."""
    for _ in range(2):
        torch.full((n_bytes,), 0x55, dtype=torch.uint8, device="cuda")


def scratch_bytes(q, cache):
    return kv8.workspace_bytes(kv8.make_attention_args(q, cache, torch.empty_like(q),
                                                       workspace=False))


@pytest.mark.parametrize("sq", [1, 40])
def test_one_call_clears_its_workspace_on_its_stream(sq):
    cache, q, out, pos = setup(sq=sq)
    n = scratch_bytes(q, cache)
    assert n > kv8.TICKET_BYTES
    litter(n)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    torch.cuda._sleep(HOLD)  # what is asked of the current stream comes late
    kv8.attention(q, cache, out, scale=0.1, stream=s)
    s.synchronize()
    check_attention(q, cache, out, pos, [3000], scale=0.1)
    torch.cuda.synchronize()


@pytest.mark.parametrize("sq", [1, 40])
def test_one_call_keeps_its_workspace_until_it_has_run(sq):
    cache, q, out, pos = setup(sq=sq)
    n = scratch_bytes(q, cache)
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        torch.cuda._sleep(HOLD)
    kv8.attention(q, cache, out, scale=0.1, stream=s)
    litter(n)  # on the current stream, while the call waits for its turn
    torch.cuda.synchronize()
    check_attention(q, cache, out, pos, [3000], scale=0.1)


def test_one_call_on_the_default_stream_from_a_side_stream():
    cache, q, out, pos = setup()
    n = scratch_bytes(q, cache)
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        litter(n)
        torch.cuda._sleep(HOLD)
        kv8.attention(q, cache, out, scale=0.1)  # stream None: the legacy default stream
        litter(n)
    torch.cuda.default_stream().synchronize()
    check_attention(q, cache, out, pos, [3000], scale=0.1)
    torch.cuda.synchronize()


def test_kept_arguments_wait_for_their_workspace():
    cache, q, out, pos = setup()
    litter(scratch_bytes(q, cache))
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    torch.cuda._sleep(HOLD)
    a = kv8.make_attention_args(q, cache, out, scale=0.1)  # cleared after the sleep
    kv8.attention_args(a, s)
    kv8.attention_args(a, s.cuda_stream)
    s.synchronize()
    check_attention(q, cache, out, pos, [3000], scale=0.1)
    torch.cuda.synchronize()
    assert ca.device_status() == ca.CA_OK


def test_block_in_one_call_on_another_stream():
    # `work` and the workspace are the block's own: what the current stream
    # allocates and writes meanwhile must not be either.
    g = torch.Generator().manual_seed(5)
    n, hd = 3000, 128
    q, k, v = (torch.randn(1, 2, h, hd, generator=g).to(torch.bfloat16).cuda() for h in (8, 2, 2))
    pos = torch.tensor([[5, 2999]], dtype=torch.int32).cuda()
    rope = torch.zeros(n, 2, device="cuda")
    cache = cache_of(g, 1, n, 2, hd, 32)
    out = torch.full((1, 2, 8, hd), 7.0, device="cuda")
    work = 2 * 2 * (8 + 2 * 2) * hd
    n_bytes = scratch_bytes(q, cache)
    litter(n_bytes)
    litter(work)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        torch.cuda._sleep(HOLD)
    torch.cuda._sleep(2 * HOLD)
    # No norm and no rotation: the block's queries are q.
    kv8.attention_block(q, k, v, cache, out, active_pos=pos, rope=rope, rope_len=n, rope_dim=0,
                        scale=0.1, stream=s)
    keep = [torch.full((b,), 0x55, dtype=torch.uint8, device="cuda") for b in (work, n_bytes)]
    s.synchronize()
    check_attention(q, cache, out, pos, [n], scale=0.1)
    torch.cuda.synchronize()
    del keep


@pytest.mark.parametrize("sq", [1, 40])
def test_one_call_in_a_graph(sq):
    # The workspace is the graph's, cleared in each replay; arguments made
    # before the capture go into it as they are.
    cache, q, out, pos = setup(sq=sq)
    kept = torch.full_like(out, 7.0)
    a = kv8.make_attention_args(q, cache, kept, scale=0.1)
    kv8.attention(q, cache, out, scale=0.1)
    torch.cuda.synchronize()
    want = out.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        kv8.attention(q, cache, out, scale=0.1, stream=torch.cuda.current_stream())
        kv8.attention_args(a, torch.cuda.current_stream())
    for _ in range(3):
        out.zero_()
        kept.zero_()
        graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, want) and torch.equal(kept, want)
    check_attention(q, cache, out, pos, [3000], scale=0.1)
