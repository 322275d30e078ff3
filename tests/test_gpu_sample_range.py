"""ca_sample over its range of temperatures and logits, against the definition
in 64 bits (tolerances: test_gpu_sample.py).

Rows whose largest logit is far from 0 in units of the temperature, where an
exponent taken as a difference of two large products has no bits left."""
import numpy as np
import pytest
import torch

from sample_helpers import STEP, sample_ref
from test_gpu_sample import check, run, us

pytestmark = pytest.mark.gpu


def peaked(seed, rows, vocab, kind="f32"):
    """Rows whose maximum lies between 10 and 30, some 2 above the next entries
    (and, in every third row, twice)."""
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(rows, vocab, generator=g) * 2
    top = 10 + 20 * torch.rand(rows, generator=g)
    at = torch.randint(0, vocab, (rows, 2), generator=g)
    for i in range(rows):
        x[i, at[i, 0]] = top[i]
        x[i, at[i, 1]] = top[i] - (0 if i % 3 == 0 else 2)
    return x.to(torch.bfloat16) if kind == "bf16" else x


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("temperature", [1.0, 0.1, 0.05, 0.01, 1e-3])
@pytest.mark.parametrize("kw", [dict(), dict(top_k=40), dict(top_k=700), dict(top_p=0.9)])
def test_min_p_of_one_keeps_the_maximum(kw, temperature, kind):
    for rows, vocab in ((300, 1201), (30, 20011)):
        x = peaked(vocab, rows, vocab, kind)
        check(x, us(rows, rows), temperature=temperature, min_p=1.0, **kw)
    check(peaked(5, 100, 900, kind), us(6, 100), temperature=temperature, min_p=3.0, **kw)


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("exponent", [4, 8, 12, 16, 17, 18, 20, 22, 24, 26, 28])
@pytest.mark.parametrize("kw", [dict(), dict(top_k=40), dict(top_k=700), dict(top_p=0.9),
                                dict(min_p=0.3)])
def test_low_temperatures(kw, exponent, kind):
    t = 10.0 ** -exponent
    for rows, vocab in ((300, 1201), (30, 20011)):
        check(peaked(exponent + vocab, rows, vocab, kind), us(rows, rows), temperature=t, **kw)
    # Logits of the temperature's own size: many entries weigh.
    g = torch.Generator().manual_seed(exponent)
    x = torch.randn(40, 5003, generator=g) * 3 * t
    x = x.to(torch.bfloat16) if kind == "bf16" else x
    u = us(exponent + 1, 40)
    tok, _ = run(x, u, temperature=t, **kw)
    for i, ui in enumerate(u):
        ref, _, slack = sample_ref(x[i].float().numpy(), ui, temperature=t, **kw)
        assert slack > 5003 * STEP and tok[i] == ref


@pytest.mark.parametrize("kw", [dict(), dict(top_k=40), dict(top_k=700), dict(top_p=0.9),
                                dict(min_p=1.0)])
@pytest.mark.parametrize("base,temperature", [(-1e20, 0.7), (1e20, 0.7), (-1e20, 1e13),
                                              (3e7, 2.0), (-1e30, 1e-6)])
def test_logits_far_from_zero(base, temperature, kw):
    # Steps between neighbours of these are 2 at 3e7, 9e12 at 1e20.
    g = torch.Generator().manual_seed(7)
    step = float(np.spacing(np.float32(abs(base))))
    x = (base + step * torch.randint(-6, 7, (60, 2003), generator=g)).float()
    x[:, 100] = base + 8 * step
    x[::2, [300, 1500]] = base + 8 * step
    check(x, us(8, 60), temperature=temperature, **kw)
