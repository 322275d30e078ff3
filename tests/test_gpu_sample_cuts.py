"""ca_sample where top_k ends exactly between two groups of entries of different
weights, more of them than a list holds (tolerances: test_gpu_sample.py)."""
import numpy as np
import pytest
import torch

from test_gpu_sample import check, us

pytestmark = pytest.mark.gpu


def grouped(seed, rows, vocab, k, noise=0.0):
    """k entries of each row about 1 and the others about 0, or -1 in every other
    row, at random places."""
    g = torch.Generator().manual_seed(seed)
    x = noise * torch.rand(rows, vocab, generator=g)
    x[1::2] -= 1
    for i in range(rows):
        x[i, torch.randperm(vocab, generator=g)[:k]] += 1.0 if i % 2 == 0 else 2.0
    return x


@pytest.mark.parametrize("rows,vocab", [(3, 32000), (40, 32000), (200, 9000), (2, 150001)])
@pytest.mark.parametrize("k", [3073, 4000, 6007])
@pytest.mark.parametrize("noise", [0.0, 1e-3])
def test_top_k_ends_with_a_group(rows, vocab, k, noise):
    x = grouped(k + rows, rows, vocab, k, noise)
    check(x, us(rows + k, rows), top_k=k)
    check(x, us(rows + k + 1, rows), top_k=k, temperature=0.6)
    # The next ones on either side of the group's end.
    check(x, us(rows + k + 2, rows), top_k=k - 1)
    check(x, us(rows + k + 3, rows), top_k=k + 1)


def test_top_k_ends_with_a_group_and_min_p():
    x = grouped(1, 30, 32000, 4000)
    x[:, 77] = 3.0  # e^-2 = 0.135 of its weight for the group
    k = int((x[0] >= 1).sum())
    for min_p in (0.1, 0.2):
        check(x[::2], us(2, 15), top_k=k, min_p=min_p)
    check(x[::2], us(3, 15), top_k=k, top_p=0.7)
    check(x[::2].to(torch.bfloat16), us(4, 15), top_k=k, min_p=0.1)


def test_top_k_ends_among_bf16_values_next_to_zero():
    # Weights are told apart by steps of 1/32 in log2 from the maximum m: one whose
    # nearest step changes at 0 puts +1e-4 and -1e-4 on its two sides.
    m = torch.arange(1.0, 32.0, 2.0 ** -7).to(torch.bfloat16).unique()
    m = m[m < 16]
    place = m.double() * 1.4426950408889634 * 32
    m = m[((place - torch.floor(place) - 0.5).abs() < 2e-3)]
    assert len(m) > 0
    k = 4000
    for top in m[:4].tolist():
        x = torch.full((4, 20000), -1e-4)
        for i in range(4):
            x[i, torch.randperm(20000, generator=torch.Generator().manual_seed(i))[:k - 1]] = 1e-4
        x[:, 9] = top
        x = x.to(torch.bfloat16)
        n = int((x[0] > 0).sum())
        check(x[:1], [0.9999], top_k=n)
        check(x[:1], us(int(top * 100), 1), top_k=n, temperature=1.0)


@pytest.mark.parametrize("sigma,temperature", [(2.0, 1.0), (0.7, 0.9), (1.0, 0.5)])
def test_large_top_k_of_random_rows(sigma, temperature):
    g = torch.Generator().manual_seed(11)
    x = sigma * torch.randn(250, 30011, generator=g)
    # top_k counts up to the end of a bin of each row in turn.
    c = np.float32(1.4426950408889634 / np.float64(np.float32(temperature))) * np.float32(32)
    for i in range(0, 250, 50):
        row = x[i:i + 50]
        place = torch.round((row[0].max() - row[0]) * float(c))
        counts = torch.bincount(place.long()).cumsum(0)
        k = int(counts[counts > 3100][0])
        check(row, us(i, 50), top_k=k, temperature=temperature)
