"""ca_sample on the GPU against its definition in 64 bits.

The kernel rounds each weight to a multiple of 2^-44 and adds whole numbers, so
that a sum over a row of V entries is off by at most V * 2^-45 (a row's largest
weight is 1), and the product with u or top_p by a rounding more. Tokens are
required to be equal; that every deciding number is further from its border
than V * 2^-44 is a property of the inputs, asserted beside it. prob comes from
fp32 exponentials (2 units in the last place each) of an exact fp32 difference
rounded once (2^-24 of at most 100): 100 * 2^-24 + 2^-21 < 1e-5 relative."""
import numpy as np
import pytest
import torch

from canvas_attn import denoise as dn
from sample_helpers import STEP, sample_ref

pytestmark = pytest.mark.gpu


def logits_of(seed, rows, vocab, kind="f32", scale=3.0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(rows, vocab, generator=g) * scale
    return x.to(torch.bfloat16) if kind == "bf16" else x


def run(x, u, *, rows=None, stride=0, offset=0, dead=(), mask_id=-1, **kw):
    """Tokens and probabilities of a call on CPU logits x; `stride`, `offset`:
    a wider buffer, filled with what must not be read."""
    n_rows, v = x.shape
    wide = max(stride, v)
    buf = torch.full((n_rows * wide + offset,), 1e30, dtype=x.dtype, device="cuda")
    d = buf[offset:].view(n_rows, wide)
    d[:, :v] = x.cuda()
    keep = buf.clone()
    n = len(u)
    uu = torch.tensor(u, dtype=torch.float32, device="cuda")
    rr = None if rows is None else torch.tensor(rows, dtype=torch.int32, device="cuda")
    tok = torch.full((n,), -7, dtype=torch.int32, device="cuda")
    prob = torch.full((n,), float("nan"), device="cuda")
    sup = torch.tensor(list(dead), dtype=torch.int32, device="cuda") if dead else None
    dn.sample(d, rr, uu, tok, prob, n_vocab=v, mask_id=mask_id, suppress=sup, **kw)
    torch.cuda.synchronize()
    assert torch.equal(buf.view(torch.int16 if x.dtype == torch.bfloat16 else torch.int32),
                       keep.view(torch.int16 if x.dtype == torch.bfloat16 else torch.int32))
    return tok.cpu().tolist(), prob.cpu().tolist()


def check(x, u, *, rows=None, dead=(), mask_id=-1, stride=0, offset=0, **kw):
    tok, prob = run(x, u, rows=rows, dead=dead, mask_id=mask_id, stride=stride, offset=offset, **kw)
    xs = x.float().numpy()
    for i, ui in enumerate(u):
        ref, p, slack = sample_ref(xs[rows[i] if rows is not None else i], ui,
                                   dead=[mask_id, *dead], **kw)
        assert slack > x.shape[1] * STEP, "the inputs leave the token open"
        assert tok[i] == ref, (i, tok[i], ref)
        assert abs(prob[i] - p) <= 1e-5 * p + 1e-30, (i, prob[i], p)


def us(seed, n):
    return np.random.default_rng(seed).random(n, dtype=np.float32).tolist()


FILTERS = [dict(), dict(temperature=0.0), dict(temperature=0.3), dict(temperature=1.5),
           dict(top_k=1), dict(top_k=50), dict(top_p=0.9), dict(top_p=0.1), dict(min_p=0.05),
           dict(temperature=0.8, top_k=40, top_p=0.95, min_p=0.02),
           dict(temperature=1.2, top_k=700, top_p=0.5)]


@pytest.mark.parametrize("kw", FILTERS)
@pytest.mark.parametrize("vocab", [1, 2, 17, 1000, 4099, 32000])
def test_tokens_match_the_definition(vocab, kw):
    n = 5
    check(logits_of(vocab, n, vocab), us(vocab + 1, n), **kw)


@pytest.mark.parametrize("kind,vocab", [("f32", 126464), ("bf16", 151936), ("f32", 262144)])
@pytest.mark.parametrize("kw", [dict(temperature=0.7), dict(top_k=50, top_p=0.95),
                                dict(top_p=0.9), dict(temperature=0.9, top_p=0.97)])
def test_large_vocabularies(kind, vocab, kw):
    n = 4
    check(logits_of(vocab % 1000, n, vocab, kind), us(vocab % 1000 + 2, n), **kw)


@pytest.mark.parametrize("n", [1, 19, 37, 74, 75, 300])
def test_numbers_of_candidates(n):
    # Clusters of 8, 4, 2 and 1 CTAs.
    check(logits_of(n, n, 20011), us(n, n), top_p=0.8, temperature=0.9)


def test_rows_strides_and_alignment():
    x = logits_of(5, 9, 1003)
    rows = [8, 3, 3, 0, 5]
    check(x, us(6, 5), rows=rows, stride=1005, offset=1, top_k=30)
    check(x.to(torch.bfloat16), us(7, 5), rows=rows, stride=1007, offset=3, top_p=0.7)


def test_ties_go_to_the_lowest_index():
    x = torch.zeros(6, 5000)
    x[1, [4000, 70, 900]] = 2.0
    x[2] = (torch.arange(5000) % 7).float()
    check(x, [0.3, 0.7, 0.5, 0.9, 0.1, 0.0], rows=[0, 1, 2, 2, 1, 0], top_k=3)
    check(x, [0.31, 0.71, 0.51, 0.91, 0.11, 0.0], rows=[0, 1, 2, 2, 1, 0], top_p=0.50007)
    # bf16 logits tie often: 300 values at most among 30000.
    check(torch.round(logits_of(8, 4, 30000) * 8).div(8).to(torch.bfloat16), us(9, 4), top_k=77)
    check(torch.round(logits_of(8, 4, 30000) * 8).div(8).to(torch.bfloat16), us(10, 4),
          top_p=0.77)


def test_equal_rows_and_signed_zeros():
    x = torch.zeros(2, 60000)
    x[1, ::2] = -0.0
    for kw in (dict(top_p=0.5000071), dict(top_k=12345), dict()):
        check(x, [0.123457, 0.876543], **kw)


def test_suppressed_masked_and_unusual_entries():
    x = logits_of(11, 6, 3001)
    x[1, 5] = float("nan")
    x[2, :] = -float("inf")
    x[2, 2999] = -80.0
    x[3, 100:200] = -float("inf")
    x[4, [7, 8]] = float("inf")
    x[5] = -3e38
    x[5, 9] = 3e38
    u = [0.4, 0.6, 0.5, 0.2, 0.75, 0.9]
    for kw in (dict(), dict(top_k=20), dict(top_p=0.9), dict(temperature=0.0), dict(min_p=0.1)):
        check(x, u, dead=[0, 1, 2, 7, 2999 - 1, -4, 9999], mask_id=3000, **kw)


def test_rows_without_a_token():
    x = torch.full((2, 700), -float("inf"))
    x[1] = float("nan")
    for kw in (dict(), dict(top_k=3), dict(top_p=0.5), dict(temperature=0.0)):
        tok, prob = run(x, [0.5, 0.5], **kw)
        assert tok == [0, 0] and prob == [0.0, 0.0]


def test_unusual_numbers_and_settings():
    x = logits_of(12, 6, 2000)
    u = [0.0, 1.0, float("nan"), -1.0, 2.0, 0.99999994]
    check(x, u)
    check(x, u, top_p=0.6)
    check(x, us(1, 6), top_p=0.0)
    check(x, us(1, 6), min_p=2.0)
    check(x, us(1, 6), top_k=5000)
    check(x, us(1, 6), temperature=float("inf"))
    check(x, us(1, 6), temperature=1e-30)


def test_settings_of_each_candidate():
    x = logits_of(13, 5, 8000)
    u = us(14, 5)
    t, k = [0.0, 0.5, 1.0, 2.0, 1.0], [0, 3, 0, 400, 1]
    p, mp = [1.0, 0.9, 0.3, 0.95, 1.0], [0.0, 0.0, 0.2, 0.001, 0.0]
    f = lambda v, d: torch.tensor(v, dtype=d, device="cuda")  # noqa: E731
    tok, prob = run(x, u, temperature=f(t, torch.float32), top_k=f(k, torch.int32),
                    top_p=f(p, torch.float32), min_p=f(mp, torch.float32))
    for i in range(5):
        ref, pr, slack = sample_ref(x[i].numpy(), u[i], temperature=t[i], top_k=k[i], top_p=p[i],
                                    min_p=mp[i])
        assert slack > 8000 * STEP and tok[i] == ref and abs(prob[i] - pr) <= 1e-5 * pr


def test_row_out_of_range_and_missing_prob():
    x = logits_of(15, 3, 500).cuda()
    rows = torch.tensor([0, 3, -1, 2], dtype=torch.int32, device="cuda")
    u = torch.tensor([0.5] * 4, device="cuda")
    tok = torch.zeros(4, dtype=torch.int32, device="cuda")
    dn.sample(x, rows, u, tok)
    torch.cuda.synchronize()
    assert tok[1] == -1 and tok[2] == -1
    for i, r in ((0, 0), (3, 2)):
        assert tok[i] == sample_ref(x[r].cpu().numpy(), 0.5)[0]


def test_frequencies():
    # 4000 draws of one row of 8 entries: each count within 6 standard
    # deviations of n p (a chance of about 1e-8 for a right kernel; the numbers are fixed).
    x = torch.tensor([[0.0, 1.0, 2.0, -1.0, 0.5, 1.5, -2.0, 0.0]])
    n = 4000
    tok, _ = run(x, us(77, n), rows=[0] * n)
    p = torch.softmax(x[0].double(), 0).numpy()
    c = np.bincount(tok, minlength=8)
    assert (np.abs(c - n * p) <= 6 * np.sqrt(n * p * (1 - p))).all()


def test_same_bits_twice_and_in_a_graph_on_another_stream():
    x = logits_of(16, 40, 50000).cuda()
    u = torch.tensor(us(17, 40), device="cuda")
    outs = []
    st = torch.cuda.Stream()
    for _ in range(2):
        tok = torch.zeros(40, dtype=torch.int32, device="cuda")
        prob = torch.zeros(40, device="cuda")
        a = dn.make_sample_args(x, None, u, tok, prob, top_p=0.9)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=st):
            dn.sample_args(a, st)
        for _ in range(3):
            tok.zero_()
            g.replay()
        torch.cuda.synchronize()
        outs.append((tok, prob))
    assert torch.equal(outs[0][0], outs[1][0]) and torch.equal(outs[0][1], outs[1][1])
    tok = torch.zeros(40, dtype=torch.int32, device="cuda")
    dn.sample(x, None, u, tok, top_p=0.9)
    torch.cuda.synchronize()
    assert torch.equal(tok, outs[0][0])


def test_denoising_step_with_temperature():
    # process_logits at a temperature: the committed tokens are the
    # definition's for the numbers that the generator gives.
    L, P, vocab, mask_id = 48, 16, 5000, 4999
    x = logits_of(18, L, vocab)
    params = dn.StepParams(remasking=dn.CONFIDENCE, confidence_threshold=0.5, temperature=0.8,
                           top_k=60, top_p=0.9, suppress_ids=[3])
    st = dn.DenoiseState([1] * P + [mask_id] * (L - P), [False] * P + [True] * (L - P), mask_id)
    n = dn.process_logits(st, x.cuda(), vocab, range(P, L), 0, 2, 8, params,
                          shuffle_rng=np.random.default_rng(5))
    u = np.random.default_rng(5).random(L - P, dtype=np.float32)
    want = [sample_ref(x[P + i].numpy(), u[i], temperature=0.8, top_k=60, top_p=0.9,
                       dead=[3, mask_id]) for i in range(L - P)]
    assert n > 0 and all(w[2] > vocab * STEP for w in want)
    done = [i for i in range(L - P) if not st.is_masked[P + i]]
    assert len(done) == n
    for i in done:
        assert st.seq[P + i] == want[i][0]
    # The most confident draws are the ones committed.
    rest = [want[i][1] for i in range(L - P) if i not in done]
    assert min(want[i][1] for i in done) >= max(rest) * (1 - 2e-5)


@pytest.mark.parametrize("temperature", [0.0, 0.8])
def test_denoising_step_on_another_stream(temperature):
    # The results are read after the work of the stream that was given, which
    # is still busy when the call is made.
    L, vocab, mask_id = 24, 5000, 4999
    x = logits_of(31, L, vocab)
    params = dn.StepParams(remasking=dn.CONFIDENCE, temperature=temperature, top_k=60)
    host = x.cuda()
    u = np.random.default_rng(6).random(L, dtype=np.float32)
    want = [sample_ref(x[i].numpy(), u[i], temperature=temperature, top_k=60, dead=[mask_id])
            for i in range(L)]
    assert temperature == 0 or all(w[2] > vocab * STEP for w in want)
    side = torch.cuda.Stream()
    lg = torch.zeros_like(host)
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        torch.cuda._sleep(200_000_000)  # about a tenth of a second
        lg.copy_(host)
    st = dn.DenoiseState([mask_id] * L, [True] * L, mask_id)
    got = dn.collect_candidates(st, lg, vocab, range(L), 0, params, stream=side,
                                draw_rng=np.random.default_rng(6))
    torch.cuda.synchronize()
    assert [c.token for c in got] == [w[0] for w in want]


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("kw", [dict(top_p=0.9), dict(top_p=0.6, min_p=0.003),
                                dict(top_k=9000), dict(top_k=9000, min_p=0.01),
                                dict(top_k=40000, top_p=0.8), dict(top_k=59990)])
def test_wide_kept_sets(kind, kw):
    # Flat rows: tens of thousands of entries are kept, and the border falls
    # among hundreds of nearly equal ones.
    check(logits_of(19, 3, 60001, kind, scale=0.7), us(20, 3), **kw)


def test_wide_kept_sets_of_many_rows():
    # One CTA a row, and a vocabulary that leaves the last warps without entries.
    check(logits_of(21, 300, 12289, scale=0.5), us(22, 300), top_p=0.95)


@pytest.mark.parametrize("kw", [dict(top_p=0.9), dict(top_k=20003), dict(top_p=0.7, top_k=20003),
                                dict(top_p=0.50001, temperature=float("inf")),
                                dict(top_p=0.3, temperature=0.01), dict(top_k=5, temperature=50.0)])
def test_bf16_borders_next_to_zero(kw):
    # Entries within 2^-16 of the row's largest magnitude, zeros of both signs
    # among them, hold the border; and rows of small values alone.
    x = logits_of(23, 4, 30000)
    x[0] *= 1e-6
    x[0, :50] = 3.0
    x[1, 100:] = 0.0
    x[1, 101::3] = -0.0
    x[2] = x[2] * 1e-30
    x[3] = x[3] * 1e-3 + 200.0
    check(x.to(torch.bfloat16), us(24, 4), **kw)


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("k", [2, 7, 128, 129, 256, 257])
def test_small_top_k(kind, k):
    # Rows whose largest entries stand in one place, are equal, or are fewer
    # than k; and rows without any order.
    x = logits_of(25, 5, 40000, kind).float()
    x[0, 10000:10000 + k] += 30.0
    x[1] = 0.0
    x[1, 5::2000] = 9.0
    x[2, 3:] = -float("inf")
    x[3] = torch.arange(40000) * 1e-3
    x = x.to(torch.bfloat16) if kind == "bf16" else x
    check(x, us(26, 5), top_k=k)
    check(x, us(27, 5), top_k=k, top_p=0.8003, temperature=0.7)


@pytest.mark.parametrize("kw", [dict(top_p=0.9), dict(top_p=0.9, temperature=1.5),
                                dict(top_p=0.3, min_p=0.4), dict(top_k=5000),
                                dict(top_k=100000, min_p=0.31), dict(top_p=0.999),
                                dict(top_p=1e-4)])
def test_flat_rows_of_large_vocabularies(kw):
    # Thousands of entries in the border's bin of the first histogram.
    x = logits_of(28, 3, 250000, scale=0.2)
    x[1] *= 1e-3
    x[2, :1000] += 2.0
    check(x, us(29, 3), **kw)


def test_bf16_cuts_and_weights_next_to_zero():
    # top_k ends among tens of thousands of zeros, the nucleus of what it leaves
    # among the entries above them; and a temperature at which values next to
    # zero weigh although exp(l - m) of them is nothing.
    x = torch.zeros(2, 30000)
    x[0, 7:30000:300] = 3.0
    x[1, ::2] = 100.0
    x[1, 1::2] = torch.arange(15000) * 1e-7
    x = x.to(torch.bfloat16)
    check(x, [0.3141, 0.2718], top_k=15000, top_p=0.1003)
    check(x, [0.7141, 0.6718], temperature=50.0, top_p=0.9003)
    check(x, [0.9141, 0.8718], temperature=50.0, top_k=20000, top_p=0.97)
