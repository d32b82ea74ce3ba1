"""cu_seqlens that is no list of sequences from 0 to T: both appends and the attention take it for the same tokens at the same positions.

The rule: sequence s is the tokens cu[s] .. cu[s + 1] - 1, cut to those in [0, T); what is cut off moves no other token, so that token t stands at
positions[s] + t - cu[s], or, as one of the last before ctx_lens[s], at ctx_lens[s] - (cu[s + 1] - t)."""
import pytest
import torch

import paged_ref as ref
from test_gpu_paged import BASE, DEV, QT, bits, make_kv, make_q

pytestmark = pytest.mark.gpu


def cut(cu, T):
    """(sequence, first token, behind the last one) of those that have any."""
    parts = [(s, max(cu[s], 0), min(cu[s + 1], T)) for s in range(len(cu) - 1)]
    return [(s, lo, hi) for s, lo, hi in parts if hi > lo]


MANY = [(3 * i) // 2 for i in range(100)]   # 99 sequences of one or two tokens
CUS = {
    "starts in front": ([-2, 3, 9], 9),
    "ends behind": ([0, 5, 14], 9),
    "both": ([-4, 12], 9),
    "zeros behind": ([0, 5, 9, 0, 0], 9),
    "zeros behind, tokens of none": ([0, 4, 7, 0], 9),
    "out of order": ([6, 9, 0, 4], 9),
    "single tokens, zeros behind": ([0, 1, 2, 3, 0, 0], 5),
    "hundreds, zeros behind": (MANY + [0] * 250, MANY[-1] + 3),
    "hundreds, the first starts in front": ([-1] + MANY[1:], MANY[-1] - 1),
    "thousands, zeros behind": (MANY + [0] * 5000, MANY[-1]),
}


def build(name, eight, Hkv, D=64, **kw):
    """A cache of the whole sequences, and of what is cut off, with cu_seqlens and T of the case."""
    cu, T = CUS[name]
    c = ref.Paged([(max(b - a, 0), (20 + 13 * s) % 150 if b > a else 0) for s, (a, b) in enumerate(zip(cu, cu[1:]))], 16, Hkv, D, torch.float16, DEV, eight=eight, **kw)
    c.T, c.cu = T, torch.tensor(cu, dtype=torch.int32, device=DEV)
    return c, cu, T


@pytest.mark.parametrize("eight", [False, True], ids=["16", "e4m3"])
@pytest.mark.parametrize("name", list(CUS))
def test_append(kerns, name, eight):
    """q, the rows and the scales: those of a call for each sequence by itself, of the tokens that are left of it."""
    c, cu, T = build(name, eight, 2, held_only=True)
    q = make_q(T, 4, 64, torch.float16)
    k, v = make_kv(T, 2, 64, torch.float16)
    append = kerns.rope_kv_append_paged_fp8 if eight else kerns.rope_kv_append_paged
    want_q, want = q.clone(), [t.clone() for t in (c.k_pages, c.v_pages, *c.scales())]
    for s, lo, hi in cut(cu, T):
        part = [t[:, lo:hi].contiguous() for t in (want_q, k, v)]
        at = torch.tensor([c.seqs[s][1] + lo - cu[s]], dtype=torch.int32, device=DEV)
        append(1, 64, BASE, *part, torch.tensor([0, hi - lo], dtype=torch.int32, device=DEV), at, c.table[s:s + 1], *want)
        want_q[:, lo:hi] = part[0]
    append(1, 64, BASE, q, k, v, c.cu, c.past, c.table, c.k_pages, c.v_pages, *c.scales())
    torch.cuda.synchronize()
    assert torch.equal(bits(q), bits(want_q))
    for got, expected in zip((c.k_pages, c.v_pages, *c.scales()), want):
        assert torch.equal(got.view(torch.uint8), expected.view(torch.uint8))


@pytest.mark.parametrize("eight", [False, True], ids=["16", "e4m3"])
@pytest.mark.parametrize("Hq", [2, 24], ids=["few rows", "many rows"])
@pytest.mark.parametrize("name", list(CUS))
def test_attend(kerns, name, Hq, eight):
    """Against the definition over the tokens that are left; tokens of no sequence stay as they were."""
    c, cu, T = build(name, eight, 1)
    q = make_q(T, Hq, 64, torch.float16)
    out = torch.full_like(q, 7.0)
    call = kerns.flash_attn_paged_fp8 if eight else kerns.flash_attn_paged
    longest = max(hi - lo for _, lo, hi in cut(cu, T))
    call(*QT[q.dtype], q.transpose(1, 2), c.k_pages, c.v_pages, *c.scales(), c.table, c.cu, c.ctx, longest, out.transpose(1, 2))
    torch.cuda.synchronize()
    kept = cut(cu, T)
    left = ref.Paged([(1, 0)], 16, 1, 64, torch.float16, "cpu")
    left.seqs = [(hi - lo, c.seqs[s][1] + lo - cu[s]) for s, lo, hi in kept]
    left.cu_list, left.table_list = [lo for _, lo, _ in kept], [c.table_list[s] for s, _, _ in kept]
    left.k_dense, left.v_dense = ([d[s][:, :sum(n)] for (s, _, _), n in zip(kept, left.seqs)] for d in (c.k_dense, c.v_dense))
    want, bound = ref.attend(left, q[0].transpose(0, 1))
    belongs = torch.zeros(T, dtype=torch.bool)
    for _, lo, hi in kept:
        belongs[lo:hi] = True
    got = out[0].transpose(0, 1).double().cpu()
    assert ((got - want).abs() <= bound)[:, belongs].all()
    assert (got[:, ~belongs] == 7).all()
