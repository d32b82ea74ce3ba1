"""The draw of verify_drafts where sums of weights that are not exact meet chunks and threads that weigh nothing: a token of the row comes out, never -1."""
from fractions import Fraction

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"


def draw(kerns, weights, sample_u):
    """The next tokens of sequences of one token each."""
    n = weights.shape[0]
    tokens, out = torch.zeros(n, dtype=torch.int64, device=DEV), torch.full((n,), -77, dtype=torch.int64, device=DEV)
    kept = torch.full((n,), -77, dtype=torch.int32, device=DEV)
    kerns.verify_drafts(tokens, torch.arange(n + 1, dtype=torch.int32, device=DEV), weights.to(DEV), None, torch.zeros(n, device=DEV),
                        torch.as_tensor(sample_u, dtype=torch.float32).expand(n).contiguous().to(DEV), out, kept)
    assert kept.tolist() == [0] * n
    return out.tolist()


def test_a_mark_between_two_sums_of_the_same_weights(kerns):
    """0.5, 5e-17, 5e-17 and 0.5 in chunks of their own with empty ones between them: the sums up to the mark differ by half a unit in the last place, by their order."""
    w = torch.zeros(1, 10240)
    w[0, 0] = w[0, 8192] = 0.5
    w[0, 2048] = w[0, 4096] = 5e-17
    assert draw(kerns, w, 0.5)[0] in (4096, 8192)


@pytest.mark.parametrize("V", [900, 6000, 16000, 70000])
def test_empty_chunks_and_threads_beside_the_mark(kerns, V):
    """A row's halves with crumbs between them that are smaller than a sum's last place, most of the row empty."""
    n = 96
    g = torch.Generator().manual_seed(V)
    w = torch.zeros(n, V)
    for row in w:
        at = torch.randperm(V, generator=g)[:torch.randint(4, 40, (1,), generator=g)].sort().values
        row[at] = torch.rand(len(at), generator=g) * 2.0 ** -53
        row[at[0]] = row[at[-1]] = 0.5
    for mark in (0.5, 0.5 - 2.0 ** -25, 0.5 + 2.0 ** -24):
        for row, j in zip(w, draw(kerns, w, mark)):
            assert j >= 0 and row[j] > 0
            # sums of up to V numbers in 64 bits: each is off by less than V roundings of the total
            exact = {i: Fraction(float(row[i])) for i in row.nonzero().flatten().tolist()}
            total, front = sum(exact.values()), sum(x for i, x in exact.items() if i < j)
            slack = total * V / 2 ** 52
            assert front <= Fraction(mark) * total + slack and front + exact[j] >= Fraction(mark) * total - slack


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("V,tail", [(900, 300), (6000, 300), (16000, 300), (16000, 9000), (70000, 2049)])
def test_a_vocabulary_padded_with_zeros(kerns, V, tail, dtype):
    """No sum is larger than the whole: the last token that weighs something, which here is far more than what sums are off by."""
    n = 60
    w = torch.softmax(3.0 * torch.randn(n, V, generator=torch.Generator().manual_seed(tail)), -1)
    w[:, V - tail:] = 0
    w[:, V - tail - 1] = 1e-3
    assert draw(kerns, w.to(dtype), 1.0) == [V - tail - 1] * n
    # and a mark in front of the last token's weight by 2^-24 of the whole finds the same one
    assert draw(kerns, w.to(dtype), 1.0 - 2.0 ** -24) == [V - tail - 1] * n
