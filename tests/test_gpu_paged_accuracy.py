"""Attention over a paged cache within the bound of what its kernels round: the weights to the 16-bit type, the output, fp32 scores and sums.  A query that
is scaled and rounded in front of the product stays within paged_ref.attend's bound and not within this one."""
import math

import pytest
import torch

import paged_ref as ref
from test_gpu_paged import BATCHES, DEV, make_q, run_attend

pytestmark = pytest.mark.gpu


def definition(c, q, factor=None):
    """out [Hq, T, D] in float64 for q [Hq, T, D], and the bound of the error of each element.

    A weight is off by its rounding (eps / 2) and by its score's error ds: D exact products added up in fp32, a step of 2^-23 of sum |q k| at most for each, and
    four for the scale, the reference and the exponential (which adds 2^-21 by itself).  Numerator and denominator together: 2 R / (1 - R) of sum(w |v|), R =
    eps / 2 + exp(ds) - 1, and a step of 2^-23 for each of the keys that are added up (fewer rescalings than keys).  The output is rounded once.  With `factor`,
    the queries are multiplied by it and rounded to the 16-bit type first: a mistake, for this test's own test."""
    Hq, T, D = q.shape
    eps, n_rep = torch.finfo(q.dtype).eps, Hq // c.Hkv
    x_all = q.double().cpu() if factor is None else (q.double().cpu() * factor).to(q.dtype).double() / factor
    out, bound = torch.zeros(Hq, T, D, dtype=torch.float64), torch.zeros(Hq, T, D, dtype=torch.float64)
    for s, (n, past) in enumerate(c.seqs):
        lo, there = c.cu_list[s], c.row_there(s)
        for h in range(Hq if n else 0):
            k, v, x = c.k_dense[s][h // n_rep], c.v_dense[s][h // n_rep], x_all[h, lo:lo + n]
            seen = (torch.arange(n + past)[None, :] <= (past + torch.arange(n))[:, None]) & there[None, :]
            w = torch.softmax((x @ k.T / math.sqrt(D)).masked_fill(~seen, -math.inf), 1)
            size = ((x.abs() @ k.abs().T) / math.sqrt(D)).masked_fill(~seen, 0.0).amax(1, keepdim=True)
            R = eps / 2 + torch.expm1((D + 4) * 2.0 ** -23 * size + 2.0 ** -21)
            out[h, lo:lo + n] = w @ v
            bound[h, lo:lo + n] = (2 * R / (1 - R) + 2 * (n + past) * 2.0 ** -23) * (w @ v.abs())
    return out, bound * (1 + eps) + eps / 2 * out.abs() + 1e-12


@pytest.mark.parametrize("eight", [False, True], ids=["16", "e4m3"])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16], ids=["f16", "bf16"])
@pytest.mark.parametrize("batch", ["tokens of many", "drafts", "more drafts than columns", "chunks"])
def test_batches(kerns, batch, dtype, eight):
    c = ref.Paged(BATCHES[batch], 16, 2, 128, dtype, DEV, eight=eight)
    q = make_q(c.T, 8, 128, dtype)
    out = torch.full_like(q, 7.0)
    run_attend(kerns, c, q, out)
    want, bound = definition(c, q[0].transpose(0, 1))
    assert bool(((out[0].transpose(0, 1).double().cpu() - want).abs() <= bound).all())


def opposed(D, dtype, seed=1):
    """A query, and two keys of e4m3 numbers with scores of about 20 that are nearly alike; with the query multiplied by the softmax's scale in powers of two
    and rounded, one score goes up by nearly half a step of each of its terms and the other one goes down."""
    factor = math.log2(math.e) / math.sqrt(D)
    x = 1 + torch.rand(D, generator=torch.Generator().manual_seed(seed), dtype=torch.float64)
    x = x.to(dtype)
    off = (x.double() * factor).to(dtype).double() / factor / x.double() - 1
    order = off.argsort()
    keys, n = torch.zeros(2, D, dtype=torch.float64), D // 4
    size = next(a for a in (2.5, 3.0, 3.5, 4.0, 5.0, 6.0, 7.0, 8.0) if a * 1.5 * n / math.sqrt(D) >= 18)
    keys[0, order[-n:]] = size
    keys[1, order[:n]] = size
    # the lower score is brought to the higher one with the element of the least error
    scores = keys @ x.double() / math.sqrt(D)
    low, mid = int(scores[1] < scores[0]), order[D // 2]
    keys[low, mid] = ref.e4m3(((scores.max() - scores.min()) * math.sqrt(D) / x[mid].double()).clamp(max=448))
    return x, keys, factor


@pytest.mark.parametrize("eight", [False, True], ids=["16", "e4m3"])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16], ids=["f16", "bf16"])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("seqs", [[(1, 40)], [(3, 60)], [(40, 100)]], ids=["decode", "drafts", "chunks"])
def test_queries_are_not_rounded_again(kerns, seqs, D, dtype, eight):
    c = ref.Paged(seqs, 16, 1, D, dtype, DEV, eight=eight)
    x, keys, factor = opposed(D, dtype)
    rows = torch.zeros(16, D, dtype=torch.float64)
    rows[3], rows[9] = keys
    page = c.table_list[0][0]
    c.k_dense[0][0, :16] = rows
    if eight:
        c.k_scales.view(torch.uint8)[page] = 127
        c.k_pages.view(torch.uint8)[page, 0] = rows.to(torch.float8_e4m3fn).view(torch.uint8).to(DEV)
    else:
        c.k_pages[page, 0] = rows.to(dtype).to(DEV)
    q = x.expand(1, c.T, 4, D).contiguous().to(DEV)
    want, bound = definition(c, q[0].transpose(0, 1))
    wrong, _ = definition(c, q[0].transpose(0, 1), factor)
    assert bool(((wrong - want).abs() > 1.5 * bound).any(-1).all())   # every row would show it
    out = torch.full_like(q, 7.0)
    run_attend(kerns, c, q, out)
    assert bool(((out[0].transpose(0, 1).double().cpu() - want).abs() <= bound).all())
