"""Operators over a paged KV cache, in 16 bits and in e4m3: against float64 definitions (paged_ref.py), against the
operators over one-slab caches bit for bit, and at the edges (empty sequences, missing pages, NaN in rows that nothing was written to)."""
import ctypes

import pytest
import torch

import capi
import paged_ref as ref

pytestmark = pytest.mark.gpu
DEV = "cuda"
QT = {torch.float16: (1, 1, 2), torch.bfloat16: (30, 256, 512)}
BASE = 5e5


def make_q(T, Hq, D, dtype, seed=1):
    g = torch.Generator().manual_seed(seed)
    return torch.randn(1, T, Hq, D, generator=g).to(dtype).to(DEV)


def run_attend(kerns, c, q, out, max_q=None):
    """q, out [1, T, Hq, D]"""
    call = kerns.flash_attn_paged_fp8 if c.eight else kerns.flash_attn_paged
    call(*QT[q.dtype], q.transpose(1, 2), c.k_pages, c.v_pages, *c.scales(), c.table, c.cu, c.ctx,
         max([n for n, _ in c.seqs] + [1]) if max_q is None else max_q, out.transpose(1, 2))


def check_attend(kerns, c, Hq, max_q=None, seed=1):
    q = make_q(c.T, Hq, c.D, c.dtype, seed)
    out = torch.full_like(q, 7.0)
    run_attend(kerns, c, q, out, max_q)
    torch.cuda.synchronize()
    want, bound = ref.attend(c, q[0].transpose(0, 1))
    got = out[0].transpose(0, 1).double().cpu()
    err = (got - want).abs()
    assert torch.isfinite(got).all()
    assert (err <= bound).all(), f"max {float((err / bound).max()):.3f} of the bound, err {float(err.max()):.3g}"
    return out


# sequences of (new tokens, rows held before them)
BATCHES = {
    "first token": [(1, 0)],
    "one token": [(1, 37)],
    "one token, whole pages": [(1, 63), (1, 127), (1, 15), (1, 16)],
    "tokens of many": [(1, n) for n in (0, 1, 14, 15, 16, 17, 31, 63, 64, 65, 200, 333)],
    "longer than a share": [(1, 3000), (1, 5), (1, 1200)],
    "drafts": [(3, 100), (4, 0), (2, 64), (4, 517)],
    "more drafts than columns": [(9, 90), (7, 400)],
    "chunks": [(70, 0), (1, 130), (33, 200), (0, 50), (129, 3)],
    "prompt": [(300, 0)],
    "empty sequences": [(0, 0), (1, 5), (0, 100), (0, 0), (5, 5), (0, 3)],
}


@pytest.mark.parametrize("eight", [False, True], ids=["16", "e4m3"])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16], ids=["f16", "bf16"])
@pytest.mark.parametrize("batch", list(BATCHES))
def test_attend_batches(kerns, batch, dtype, eight):
    c = ref.Paged(BATCHES[batch], 16, 2, 128, dtype, DEV, eight=eight)
    check_attend(kerns, c, 8)


@pytest.mark.parametrize("eight", [False, True], ids=["16", "e4m3"])
@pytest.mark.parametrize("page,D,Hq,Hkv,order", [(16, 64, 8, 2, "heads"), (32, 128, 3, 3, "rows"), (64, 64, 6, 1, "rows"), (128, 128, 12, 2, "heads"),
                                                 (256, 128, 8, 8, "rows"), (1024, 64, 20, 1, "heads"), (16, 128, 48, 1, "rows"), (32, 128, 40, 8, "heads")])
def test_attend_heads_pages_strides(kerns, page, D, Hq, Hkv, order, eight):
    """Group sizes that are no power of two or above 16, every kind of page, both orders of a pool in memory, a table with a
    row stride of its own."""
    for seqs in ([(1, 300), (1, 2), (1, 77)], [(5, 140), (40, 0), (1, 9)]):
        check_attend(kerns, ref.Paged(seqs, page, Hkv, D, torch.float16, DEV, seed=page, order=order, eight=eight, gap=3), Hq)


@pytest.mark.parametrize("eight", [False, True], ids=["16", "e4m3"])
@pytest.mark.parametrize("page", [16, 64])
def test_attend_pages_that_are_not_there(kerns, page, eight):
    """The first pages given back, one in the middle, the last one, all of them: their rows take no part, the others keep their
    places, and a token without rows yields zeros."""
    n = [(300 + page - 1) // page, (301 + page - 1) // page, (99 + 17 + page - 1) // page, (40 + 70 + page - 1) // page]
    gone = {(0, i) for i in range(n[0] // 2)} | {(1, i) for i in range(n[1])} | {(2, 1 % n[2]), (2, n[2] - 1)} | {(3, 0)}
    c = ref.Paged([(1, 299), (1, 300), (17, 99), (70, 40)], page, 2, 128, torch.float16, DEV, gone=gone, eight=eight)
    out = check_attend(kerns, c, 4)
    assert (out[0, 1] == 0).all()
    c = ref.Paged([(1, 299), (1, 300)], page, 2, 128, torch.float16, DEV, gone={(0, i) for i in range(n[0] // 2)} | {(1, i) for i in range(n[1])}, eight=eight)
    check_attend(kerns, c, 4)


@pytest.mark.parametrize("eight", [False, True], ids=["16", "e4m3"])
@pytest.mark.parametrize("seqs", [[(1, 9), (1, 700)], [(4, 60), (2, 5)], [(65, 3), (20, 300)]], ids=["decode", "drafts", "chunks"])
def test_attend_bad_tables(kerns, seqs, eight):
    """Entries far outside the pool are pages that are not there."""
    c = ref.Paged(seqs, 16, 2, 64, torch.bfloat16, DEV, gone={(0, 0), (1, 0)}, eight=eight)
    for bad in (-2 ** 31, 2 ** 31 - 1, c.n_pages, -7):
        c.table[0, 0] = bad
        c.table[1, 0] = bad
        check_attend(kerns, c, 4)


@pytest.mark.parametrize("eight", [False, True], ids=["16", "e4m3"])
@pytest.mark.parametrize("seqs,Hq,Hkv,D,page,gone", [
    ([(20, 38000)], 4, 1, 64, 64, 0),                              # one block of rows in more pieces than lanes
    ([(60, 5000), (33, 90), (200, 0)], 4, 1, 128, 16, 0),          # pieces of long and short blocks together
    ([(60, 5000), (33, 3000)], 6, 2, 64, 32, 40),                  # their first pages given back
    ([(17 + i % 3, (37 * i) % 200) for i in range(150)], 2, 1, 64, 16, 0),   # more sequences than lanes
    ([(260, 2000)], 24, 8, 64, 16, 0),                             # more blocks than one round
    ([(700, 0), (300, 40)], 32, 8, 64, 16, 1),                     # blocks of two rounds
], ids=["many pieces", "long and short", "given back", "many sequences", "a round", "two rounds"])
def test_attend_pieces(kerns, seqs, Hq, Hkv, D, page, gone, eight):
    c = ref.Paged(seqs, page, Hkv, D, torch.float16, DEV, gone={(s, i) for s in range(len(seqs)) for i in range(gone)}, eight=eight)
    check_attend(kerns, c, Hq)


@pytest.mark.parametrize("eight", [False, True], ids=["16", "e4m3"])
@pytest.mark.parametrize("seqs,Hq,Hkv", [([(1, 9000), (1, 70), (1, 2500)], 8, 1), ([(1, (53 * i) % 700) for i in range(70)], 4, 1),
                                         ([(1, 3000 + 37 * i) for i in range(40)], 16, 8), ([(2, 5000), (4, 700), (0, 40)], 8, 2), ([(1, 20000)], 2, 1)],
                         ids=["uneven", "more than lanes", "the line", "drafts", "long"])
def test_attend_shares(kerns, seqs, Hq, Hkv, eight):
    """Chunks and shares: contexts that differ, more sequences than lanes, more pairs than units, many parts of a row; a table that is wider than the
    longest context needs."""
    for width in (None, 4000):
        c = ref.Paged(seqs, 16, Hkv, 64, torch.float16, DEV, eight=eight, width=width)
        check_attend(kerns, c, Hq)


@pytest.mark.parametrize("n_tokens", [1, 3, 50])
def test_attend_leaves_other_rows(kerns, n_tokens):
    """Rows of out behind the last sequence, and tokens past max_q_len, are left as they were."""
    c = ref.Paged([(n_tokens, 20), (n_tokens, 3)], 16, 2, 128, torch.float16, DEV)
    T = c.T + 5
    q = make_q(T, 4, 128, torch.float16)
    out = torch.full_like(q, 7.0)
    run_attend(kerns, c, q, out)
    want = torch.empty(1, c.T, 4, 128, dtype=q.dtype, device=DEV)
    run_attend(kerns, c, q[:, :c.T].contiguous(), want)
    assert (out[0, c.T:] == 7).all() and torch.equal(out[:, :c.T], want)
    if n_tokens > 1:
        out.fill_(7.0)
        run_attend(kerns, c, q, out, max_q=n_tokens - 1)
        for s in range(2):
            assert (out[0, (s + 1) * n_tokens - 1] == 7).all()
        bound = 1e-2
        err = (out[0, :n_tokens - 1] - want[0, :n_tokens - 1]).abs().max()
        assert float(err) <= bound


@pytest.mark.parametrize("eight", [False, True], ids=["16", "e4m3"])
def test_attend_bound_unknown(kerns, eight):
    """max_q_len 0: not known."""
    for seqs in ([(1, 100), (1, 3)], [(4, 30), (60, 0), (1, 200)]):
        c = ref.Paged(seqs, 32, 2, 128, torch.bfloat16, DEV, eight=eight)
        check_attend(kerns, c, 8, max_q=0)


@pytest.mark.parametrize("n,Hq", [(1, 4), (4, 4), (70, 4)], ids=["decode", "drafts", "chunks"])
@pytest.mark.parametrize("eight", [False, True], ids=["16", "e4m3"])
def test_attend_fewer_rows_than_tokens(kerns, n, Hq, eight):
    """A context shorter than the tokens: the first ones stand in front of row 0 and yield zeros, the others attend what is there."""
    c = ref.Paged([(n, 0), (n, 30)], 16, 2, 64, torch.float16, DEV, eight=eight)
    q = make_q(c.T, Hq, 64, torch.float16)
    held = n // 2
    c.ctx[0] = held
    out = torch.full_like(q, 7.0)
    run_attend(kerns, c, q, out)
    assert (out[0, :n - held] == 0).all()
    short = ref.Paged([(held, 0), (n, 30)], 16, 2, 64, torch.float16, DEV, eight=eight)
    short.k_dense = [c.k_dense[0][:, :held], c.k_dense[1]]
    short.v_dense = [c.v_dense[0][:, :held], c.v_dense[1]]
    want, bound = ref.attend(short, q[0, n - held:].transpose(0, 1))
    assert ((out[0, n - held:].transpose(0, 1).double().cpu() - want).abs() <= bound).all()


@pytest.mark.parametrize("seqs", [[(1, 40), (1, 900)], [(3, 40), (2, 1900)], [(80, 5), (3, 70)]], ids=["decode", "drafts", "chunks"])
def test_attend_malformed_index_tensors_stay_in_bounds(kerns, seqs):
    """cu_seqlens and ctx_lens that make no sense: q, out and the pools lie between guards that stay as they are (what such a call
    computes is not specified)."""
    c = ref.Paged(seqs, 16, 2, 64, torch.float16, DEV)
    whole = torch.full((1, c.T + 20, 4, 64), 5.0, dtype=torch.float16, device=DEV)
    out = whole[:, 10:10 + c.T]
    q = make_q(c.T, 4, 64, torch.float16)
    cus = [[0, c.T + 100, 2 * c.T], [-5, 3, c.T], [c.T, 1, 0], [2 ** 31 - 1, -2 ** 31, 7], [0, 0, 0]]
    ctxs = [[2 ** 31 - 1, 5], [-4, -2 ** 31], [0, 0], [1 << 20, 1]]
    for cu in cus:
        for ctx in ctxs:
            c.cu.copy_(torch.tensor(cu, dtype=torch.int32))
            c.ctx.copy_(torch.tensor(ctx, dtype=torch.int32))
            for max_q in (0, max(n for n, _ in seqs)):
                run_attend(kerns, c, q, out, max_q)
            torch.cuda.synchronize()
            assert (whole[:, :10] == 5).all() and (whole[:, 10 + c.T:] == 5).all()


def test_attend_empty_calls(kerns):
    """No sequences, no tokens, no pages."""
    c = ref.Paged([(1, 5)], 16, 2, 64, torch.float16, DEV)
    q = make_q(1, 4, 64, torch.float16)
    out = torch.full_like(q, 7.0)
    none = torch.zeros(0, dtype=torch.int32, device=DEV)
    kerns.flash_attn_paged(1, 1, 2, q.transpose(1, 2), c.k_pages, c.v_pages, c.table[:0], torch.zeros(1, dtype=torch.int32, device=DEV), none, 1, out.transpose(1, 2))
    assert (out == 7).all()
    kerns.flash_attn_paged(1, 1, 2, q[:, :0].transpose(1, 2), c.k_pages, c.v_pages, c.table, torch.zeros(2, dtype=torch.int32, device=DEV), c.ctx, 1, out[:, :0].transpose(1, 2))
    kerns.flash_attn_paged(1, 1, 2, q.transpose(1, 2), c.k_pages[:0], c.v_pages[:0], c.table, c.cu, c.ctx, 1, out.transpose(1, 2))
    assert (out == 0).all()
    out.fill_(7.0)
    kerns.flash_attn_paged(1, 1, 2, q.transpose(1, 2), c.k_pages, c.v_pages, c.table[:, :0], c.cu, c.ctx, 1, out.transpose(1, 2))
    assert (out == 0).all()


@pytest.mark.parametrize("seqs", [[(1, 2100), (1, 30)], [(2, 500), (1, 3)], [(100, 64), (1, 30)]], ids=["decode", "drafts", "chunks"])
def test_attend_nan_and_infinities_of_attended_rows(kerns, seqs):
    """A NaN in an attended row of V comes out, an infinite value too, and the other sequences stay as they were; a NaN in a row of K
    reaches the tokens that attend the row and no others."""
    c = ref.Paged(seqs, 16, 1, 64, torch.float16, DEV)
    n, past = seqs[0]
    q = make_q(c.T, 2, 64, torch.float16)
    clean = torch.empty_like(q)
    run_attend(kerns, c, q, clean)
    row = past + n - 1   # the last token's own row: attended by that token only
    page = c.table_list[0][row // 16]
    kept_k, kept_v = c.k_pages.clone(), c.v_pages.clone()
    out = torch.empty_like(q)
    for value in (float("nan"), float("inf")):
        c.v_pages[page, 0, row % 16, 3] = value
        run_attend(kerns, c, q, out)
        last = out[0, n - 1, :, 3].float()
        assert (torch.isnan(last) if value != value else last == value).all()
        assert torch.equal(out[0, n:], clean[0, n:])
    c.v_pages.copy_(kept_v)
    c.k_pages[page, 0, row % 16, 3] = float("nan")
    run_attend(kerns, c, q, out)
    assert torch.isnan(out[0, n - 1]).all()
    assert torch.equal(out[0, :n - 1], clean[0, :n - 1]) and torch.equal(out[0, n:], clean[0, n:])
    c.k_pages.copy_(kept_k)
    run_attend(kerns, c, q, out)
    assert torch.equal(out, clean)


@pytest.mark.parametrize("seqs,Hq,Hkv,D,max_q", [
    ([(4, 300), (3, 9)], 4, 1, 64, None), ([(2, 61), (3, 4)] + [(2, (41 * i) % 300) for i in range(70)], 6, 2, 128, None), ([(9, 130), (1, 7)], 8, 1, 128, 1),
    ([(90, 40), (70, 0)], 4, 2, 128, None), ([(50, 2100), (5, 5)], 12, 1, 64, None), ([(1030, 0), (1040, 9)], 48, 24, 128, None)],
    ids=["drafts", "drafts of many", "first tokens only", "chunks", "pieces", "prompts"])
@pytest.mark.parametrize("eight", [False, True], ids=["16", "e4m3"])
@pytest.mark.parametrize("dtype,value", [(torch.float16, float("inf")), (torch.bfloat16, float("nan"))], ids=["f16-inf", "bf16-nan"])
def test_attend_rows_that_are_not_finite_reach_who_attends_them(kerns, seqs, Hq, Hkv, D, max_q, eight, dtype, value):
    """V rows of some tokens hold an infinity (a NaN, which is all that e4m3 has): the tokens before them are as if they were not there,
    and those behind have it in its column and nowhere else."""
    c = ref.Paged(seqs, 16, Hkv, D, dtype, DEV, eight=eight)
    q = make_q(c.T, Hq, D, dtype)
    bad = {}   # sequence: first token that attends a bad row
    for s, (n, past) in enumerate(seqs[:2]):
        bad[s] = max(n // 2, 1) if n > 1 else n
        for i in range(bad[s], n, 3):
            page, row = c.table_list[s][(past + i) // 16], (past + i) % 16
            if eight:
                c.v_pages.view(torch.uint8)[page, :, row, 3] = 0x7f
            else:
                c.v_pages[page, :, row, 3] = value
    out = torch.full_like(q, 7.0)
    run_attend(kerns, c, q, out, max_q)
    want, bound = ref.attend(c, q[0].transpose(0, 1))
    got = out[0].transpose(0, 1).double().cpu()
    for s, (n, _) in enumerate(seqs):
        lo, done = c.cu_list[s], n if max_q is None else min(n, max_q)
        reached = torch.zeros(Hq, n, D, dtype=torch.bool)
        reached[:, bad.get(s, n):, 3] = True
        here = slice(lo, lo + done)
        reached = reached[:, :done]
        ok = (got[:, here] - want[:, here]).abs() <= bound[:, here]
        assert (ok | reached).all(), f"sequence {s}"
        x = got[:, here][reached]
        assert not torch.isfinite(x).any() and (value == value and not eight or torch.isnan(x).all()), f"sequence {s}"


@pytest.mark.parametrize("n", [3, 60], ids=["drafts", "chunks"])
def test_attend_a_page_whose_scale_is_no_number(kerns, n):
    """A scale of NaN makes NaN of the page's rows, for the tokens that attend one of them and no others."""
    c = ref.Paged([(n, 30), (2, 40)], 16, 1, 64, torch.bfloat16, DEV, eight=True)
    q = make_q(c.T, 4, 64, torch.bfloat16)
    c.v_scales.view(torch.uint8)[c.table_list[0][2]] = 255   # rows 32 .. 47: the tokens from the third on
    out = torch.full_like(q, 7.0)
    run_attend(kerns, c, q, out)
    want, bound = ref.attend(c, q[0].transpose(0, 1))
    got = out[0].transpose(0, 1).double().cpu()
    ok = (got - want).abs() <= bound
    assert ok[:, :2].all() and ok[:, n:].all() and torch.isnan(got[:, 2:n]).all()


@pytest.mark.parametrize("seqs", [[(1, 300), (1, 40)], [(3, 100), (4, 30)], [(70, 50), (9, 0)]], ids=["decode", "drafts", "chunks"])
@pytest.mark.parametrize("eight", [False, True], ids=["16", "e4m3"])
def test_pages_whose_offsets_pass_32_bits(kerns, seqs, eight):
    """Pages that lie 2^32 elements behind a pool's first one: the same bits as in a small pool, appended and attended."""
    c = ref.Paged(seqs, 64, 2, 128, torch.float16, DEV, eight=eight)
    n_big = 2 ** 32 // c.k_pages[0].numel() + 50 * c.n_pages
    pools = [torch.empty((n_big,) + c.k_pages.shape[1:], dtype=c.k_pages.dtype, device=DEV) for _ in range(2)]
    ids = n_big - 1 - 50 * torch.arange(c.n_pages, device=DEV)
    table = torch.where(c.table >= 0, ids.to(torch.int32)[c.table.long().clamp(min=0)], -1)
    scales = ()
    for pool, small in zip(pools, (c.k_pages, c.v_pages)):
        bits(pool)[ids] = bits(small)
    if eight:
        scales = tuple(torch.zeros(n_big, 2, dtype=torch.uint8, device=DEV) for _ in range(2))
        for big, small in zip(scales, c.scales()):
            big[ids] = small.view(torch.uint8)
        scales = tuple(x.view(torch.float8_e8m0fnu) for x in scales)
    q = make_q(c.T, 8, 128, torch.float16)
    k, v = make_q(c.T, 2, 128, torch.float16, 2), make_q(c.T, 2, 128, torch.float16, 3)
    outs = []
    for t, (kp, vp), sc in ((c.table, (c.k_pages, c.v_pages), c.scales()), (table, pools, scales)):
        mine, out = q.clone(), torch.empty_like(q)
        append, attend = (kerns.rope_kv_append_paged_fp8, kerns.flash_attn_paged_fp8) if eight else (kerns.rope_kv_append_paged, kerns.flash_attn_paged)
        append(1, 128, BASE, mine, k, v, c.cu, c.past, t, kp, vp, *sc)
        attend(*QT[q.dtype], mine.transpose(1, 2), kp, vp, *sc, t, c.cu, c.ctx, max(n for n, _ in seqs), out.transpose(1, 2))
        outs.append((mine, out))
    assert torch.equal(outs[0][0], outs[1][0]) and torch.equal(outs[0][1], outs[1][1]) and torch.isfinite(outs[0][1]).all()
    for pool, small in zip(pools, (c.k_pages, c.v_pages)):
        assert torch.equal(bits(pool)[ids], bits(small))


@pytest.mark.parametrize("n", [1, 3, 40], ids=["decode", "drafts", "chunks"])
@pytest.mark.parametrize("eight", [False, True], ids=["16", "e4m3"])
def test_attend_one_page_many_times(kerns, n, eight):
    """A table that names one page again and again, 2^17 rows, behind them one page of its own: a context is read by its table, however
    long; many times the same rows are the weights of one of them, many times.  Beside the bound of rounded weights, fp32 sums of up
    to 2^17 / 4 weights a lane and as many products are off by half a step a term."""
    c = ref.Paged([(n, 64)], 64, 1, 64, torch.float16, DEV, eight=eight)
    times = 2 ** 17 // 64
    table = torch.cat([c.table[:, :1].expand(1, times), c.table[:, 1:2]], 1).contiguous()
    ctx = torch.tensor([times * 64 + n], dtype=torch.int32, device=DEV)
    q = make_q(n, 4, 64, torch.float16)
    out = torch.full_like(q, 7.0)
    call = kerns.flash_attn_paged_fp8 if eight else kerns.flash_attn_paged
    call(*QT[q.dtype], q.transpose(1, 2), c.k_pages, c.v_pages, *c.scales(), table, c.cu, ctx, n, out.transpose(1, 2))
    big = ref.Paged([(n, 64)], 64, 1, 64, torch.float16, DEV, eight=eight)
    big.seqs, big.table_list = [(n, times * 64)], [[0] * (times + 1)]
    big.k_dense = [torch.cat([c.k_dense[0][:, :64].repeat(1, times, 1), c.k_dense[0][:, 64:]], 1)]
    big.v_dense = [torch.cat([c.v_dense[0][:, :64].repeat(1, times, 1), c.v_dense[0][:, 64:]], 1)]
    want, bound = ref.attend(big, q[0].transpose(0, 1))
    sums = 2 * 2.0 ** 15 * 2.0 ** -24 * float(big.v_dense[0].abs().max())
    assert ((out[0].transpose(0, 1).double().cpu() - want).abs() <= bound + sums).all()


@pytest.mark.parametrize("n", [1, 3, 80], ids=["decode", "drafts", "chunks"])
def test_attend_tokens_of_no_sequence(kerns, n):
    """Tokens that belong to no sequence, all of them empty, over a table wide enough for blocks to be cut: nothing is written, whatever the
    memory held that the call's workspace gets."""
    c = ref.Paged([(n, 40), (n, 90)], 16, 2, 64, torch.float16, DEV, width=300)
    q = make_q(c.T, 4, 64, torch.float16)
    out = torch.full_like(q, 7.0)
    for fill in (0x00, 0x7f):
        for cu in ([0, 0, 0], [c.T, c.T, c.T]):
            c.cu.copy_(torch.tensor(cu, dtype=torch.int32))
            before = [torch.full((size,), fill, dtype=torch.uint8, device=DEV) for size in (1 << 16, 1 << 20, 1 << 24, 1 << 26)]
            torch.cuda.synchronize()
            del before   # to the allocator, which hands it out again as it is
            run_attend(kerns, c, q, out, n)
            torch.cuda.synchronize()
            assert (out == 7).all()


@pytest.mark.parametrize("eight", [False, True], ids=["16", "e4m3"])
@pytest.mark.parametrize("n", [1, 5, 11], ids=["decode", "drafts", "chunks"])
def test_attend_hundreds_of_sequences(kerns, n, eight):
    """More sequences than are looked up at a time, some of them without tokens or without rows held."""
    seqs = [((i * 7) % (n + 1), (37 * i) % 90) for i in range(700)]
    c = ref.Paged(seqs, 16, 1, 64, torch.float16, DEV, eight=eight)
    check_attend(kerns, c, 2, max_q=n)


@pytest.mark.parametrize("eight", [False, True], ids=["16", "e4m3"])
def test_attend_pieces_of_two_rounds(kerns, eight):
    """A little more blocks than the chip holds at once: 73 of 128 rows, or 37 of 256, for each of eight KV heads."""
    c = ref.Paged([(2300, 0), (10, 1500)], 16, 8, 128, torch.bfloat16, DEV, eight=eight)
    check_attend(kerns, c, 32)


@pytest.mark.parametrize("seqs", [[(1, 4000), (1, 300)], [(3, 900), (2, 70)], [(50, 3000)]], ids=["decode", "drafts", "chunks"])
def test_attend_on_two_streams_at_once(kerns, seqs):
    """Calls in flight on the null stream and on another at the same time, of the same cache and of different ones: the bits of calls alone."""
    caches = [ref.Paged(seqs, 16, 2, 64, torch.float16, DEV, seed=s) for s in range(2)]
    qs = [make_q(c.T, 8, 64, torch.float16, 5 + i) for i, c in enumerate(caches)]
    alone = []
    for c, q in zip(caches, qs):
        out = torch.empty_like(q)
        run_attend(kerns, c, q, out)
        torch.cuda.synchronize()
        alone.append(out)
    side = torch.cuda.Stream()
    outs = [[torch.full_like(qs[0], 7.0) for _ in range(40)] for _ in range(2)]
    torch.cuda.synchronize()
    for i in range(40):
        run_attend(kerns, caches[i % 2], qs[i % 2], outs[0][i])
        with torch.cuda.stream(side):
            run_attend(kerns, caches[(i // 2) % 2], qs[(i // 2) % 2], outs[1][i])
    torch.cuda.synchronize()
    for i in range(40):
        assert torch.equal(outs[0][i], alone[i % 2]) and torch.equal(outs[1][i], alone[(i // 2) % 2])


@pytest.mark.parametrize("seqs,Hq", [([(1, 700), (1, 64)], 8), ([(4, 300), (3, 9)], 8), ([(90, 40)], 4)], ids=["decode", "drafts", "chunks"])
@pytest.mark.parametrize("eight", [False, True], ids=["16", "e4m3"])
def test_attend_repeats_and_streams(kerns, seqs, Hq, eight):
    """The same bits again, on the null stream as on another."""
    c = ref.Paged(seqs, 16, 2, 128, torch.float16, DEV, eight=eight)
    q = make_q(c.T, Hq, 128, torch.float16)
    first = torch.empty_like(q)
    run_attend(kerns, c, q, first)
    for _ in range(3):
        again = torch.empty_like(q)
        run_attend(kerns, c, q, again)
        assert torch.equal(first, again)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        other = torch.empty_like(q)
        run_attend(kerns, c, q, other)
    side.synchronize()
    assert torch.equal(first, other)


# ---- append --------------------------------------------------------------------------------------------------------------------
APPENDS = {
    "first token": [(1, 0)],
    "one token each": [(1, n) for n in (0, 5, 15, 16, 31, 32, 100, 70001)],
    "drafts": [(3, 14), (4, 0), (2, 31), (5, 100)],
    "chunks": [(40, 0), (1, 13), (0, 9), (130, 7), (64, 32), (0, 0), (33, 15)],
    "long chunk": [(600, 21)],
}


def make_kv(T, Hkv, D, dtype, seed=3):
    g = torch.Generator().manual_seed(seed)
    k, v = torch.randn(1, T, Hkv, D, generator=g), torch.randn(1, T, Hkv, D, generator=g) * 3
    k[..., 1] *= 9
    return k.to(dtype).to(DEV), v.to(dtype).to(DEV)


def slab_append(kerns, c, style, rd, q, k, v):
    """What rope_kv_append, one sequence at a time, makes of the new rows: q, and k and v as a 16-bit cache holds them [T, Hkv, D]."""
    q = q.clone()
    rows_k, rows_v = torch.empty_like(k[0]), torch.empty_like(v[0])
    for s, (n, past) in enumerate(c.seqs):
        if n == 0:
            continue
        lo = c.cu_list[s]
        kc = torch.zeros(1, c.Hkv, past + n, c.D, dtype=q.dtype, device=DEV)
        vc = torch.zeros_like(kc)
        part = q[:, lo:lo + n].contiguous()
        kerns.rope_kv_append(style, rd, BASE, part, k[:, lo:lo + n].contiguous(), v[:, lo:lo + n].contiguous(),
                             torch.tensor([past], dtype=torch.int32, device=DEV), kc, vc)
        q[:, lo:lo + n] = part
        rows_k[lo:lo + n] = kc[0, :, past:].transpose(0, 1)
        rows_v[lo:lo + n] = vc[0, :, past:].transpose(0, 1)
    return q, rows_k, rows_v


def bits(t):
    return t.contiguous().view(torch.uint8 if t.element_size() == 1 else torch.int16)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16], ids=["f16", "bf16"])
@pytest.mark.parametrize("batch", list(APPENDS))
@pytest.mark.parametrize("style,rd,D,page,order", [(0, 128, 128, 16, "heads"), (1, 128, 128, 32, "rows"), (1, 32, 64, 16, "heads"), (0, 64, 128, 64, "rows"), (1, 0, 64, 256, "heads")])
def test_append_bits(kerns, batch, dtype, style, rd, D, page, order):
    """q and the rows equal rope_kv_append's to the bit; every other byte of the pools stays."""
    seqs = [(n, p if page >= 32 or p < 1000 else p % 1000) for n, p in APPENDS[batch]] if page != 256 else APPENDS[batch]
    c = ref.Paged(seqs, page, 2, D, dtype, DEV, order=order, held_only=True, gap=2)
    q = make_q(c.T, 6, D, dtype)
    k, v = make_kv(c.T, 2, D, dtype)
    want_q, rows_k, rows_v = slab_append(kerns, c, style, rd, q, k, v)
    want = [c.k_pages.clone(), c.v_pages.clone()]
    for pool, rows in zip(want, (rows_k, rows_v)):
        for s, (n, past) in enumerate(c.seqs):
            for i in range(n):
                pool[c.table_list[s][(past + i) // page], :, (past + i) % page] = rows[c.cu_list[s] + i]
    k0, v0 = k.clone(), v.clone()
    kerns.rope_kv_append_paged(style, rd, BASE, q, k, v, c.cu, c.past, c.table, c.k_pages, c.v_pages)
    torch.cuda.synchronize()
    assert torch.equal(bits(q), bits(want_q))
    assert torch.equal(bits(c.k_pages), bits(want[0])) and torch.equal(bits(c.v_pages), bits(want[1]))
    assert torch.equal(k, k0) and torch.equal(v, v0)
    # and against the definition: half a step of the result plus the fp32 rotation's error
    for s, (n, past) in enumerate(c.seqs):
        if n and rd:
            lo = c.cu_list[s]
            y = ref.rotated(k0[0, lo:lo + n].double().cpu(), past, style, rd, BASE)
            x = rows_k[lo:lo + n].double().cpu()
            eps = torch.finfo(dtype).eps
            size = k0[0, lo:lo + n].double().cpu().abs().amax(-1, keepdim=True)
            assert ((x - y).abs() <= eps / 2 * (1 + 1e-3) * y.abs() + 2.0 ** -20 * size).all()


def expected_e4m3(c, rows, pool, scales, max_e):
    """Codes' values and exponents of a pool after rows [T, Hkv, D] (float64, what a 16-bit cache would hold) were appended."""
    values = pool.double().cpu() * torch.exp2(scales.view(torch.uint8).double().cpu() - 127)[:, :, None, None]
    exps = scales.view(torch.uint8).to(torch.int64).cpu() - 127
    raw = bits(pool).cpu().clone()
    for s, (n, past) in enumerate(c.seqs):
        if n == 0:
            continue
        for p in range(past // c.page, (past + n - 1) // c.page + 1):
            lo, hi = max(past, p * c.page), min(past + n, (p + 1) * c.page)
            at, old = c.table_list[s][p], lo - p * c.page
            if at < 0:
                continue
            for h in range(c.Hkv):
                new = rows[c.cu_list[s] + lo - past:c.cu_list[s] + hi - past, h]
                e = ref.needed_exponent(new, max_e)
                if old:
                    e = max(e, int(exps[at, h]))
                    if e > int(exps[at, h]):
                        raw[at, h, :old] = ref.e4m3(values[at, h, :old] / 2.0 ** e).to(torch.float8_e4m3fn).view(torch.uint8)
                exps[at, h] = e
                x = torch.where(torch.isfinite(new), new / 2.0 ** e, float("nan")).clamp(-448, 448)
                raw[at, h, old:hi - p * c.page] = ref.e4m3(x).to(torch.float8_e4m3fn).view(torch.uint8)
    return raw, exps


def same_codes(a, b):
    """Equal bytes; NaN codes (0x7f and 0xff) and the two zeros are one each."""
    a, b = a.to(torch.int16), b.to(torch.int16)
    for t in (a, b):
        t[(t & 0x7F) == 0x7F] = 0x7F
        t[t == 0x80] = 0
    return torch.equal(a, b)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16], ids=["f16", "bf16"])
@pytest.mark.parametrize("batch", list(APPENDS))
@pytest.mark.parametrize("style,rd,D,page,order,Hkv", [(0, 128, 128, 16, "heads", 8), (1, 128, 128, 32, "rows", 3), (1, 64, 64, 16, "heads", 1), (0, 64, 128, 64, "rows", 2),
                                                       (1, 32, 64, 256, "heads", 5), (1, 64, 128, 128, "heads", 8)])
def test_append_e4m3(kerns, batch, dtype, style, rd, D, page, order, Hkv):
    """Codes and scales from the definition, the rotated k rounded from 64 bits to the 16-bit type; every other byte stays.  q as
    rope_kv_append makes it."""
    c = ref.Paged([(n, p % 3000) for n, p in APPENDS[batch]], page, Hkv, D, dtype, DEV, order=order, held_only=True, eight=True)
    q = make_q(c.T, 2 * Hkv, D, dtype)
    k, v = make_kv(c.T, Hkv, D, dtype)
    want_q, _, rows_v = slab_append(kerns, c, style, rd, q, k, v)
    rows_k = torch.cat([ref.rotated(k[0, c.cu_list[s]:c.cu_list[s] + n].double().cpu(), past, style, rd, BASE).to(dtype) for s, (n, past) in enumerate(c.seqs)])
    max_e = 7 if dtype == torch.float16 else 119
    want = [expected_e4m3(c, r.double().cpu(), pool, sc, max_e) for r, pool, sc in ((rows_k, c.k_pages, c.k_scales), (rows_v, c.v_pages, c.v_scales))]
    kerns.rope_kv_append_paged_fp8(style, rd, BASE, q, k, v, c.cu, c.past, c.table, c.k_pages, c.v_pages, c.k_scales, c.v_scales)
    torch.cuda.synchronize()
    assert torch.equal(bits(q), bits(want_q))
    for pool, sc, (raw, exps) in zip((c.k_pages, c.v_pages), (c.k_scales, c.v_scales), want):
        assert torch.equal(sc.view(torch.uint8).cpu().to(torch.int64) - 127, exps)
        assert same_codes(bits(pool).cpu(), raw)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16], ids=["f16", "bf16"])
def test_append_e4m3_extremes(kerns, dtype):
    """Zeros, one value alone, amounts at the border of a scale, the type's largest and smallest, infinities and NaN; and a token whose
    large values move the codes in front of it out of the normal range."""
    page, D = 16, 64
    big, tiny = torch.finfo(dtype).max, torch.finfo(dtype).smallest_normal
    fills = [0.0, 448.0, 449.0 if dtype == torch.float16 else 450.0, 448.0 / 4, 1e-6, big, tiny, float("inf"), float("nan"), -1.0]
    c = ref.Paged([(1, 5)] * len(fills), page, 1, D, dtype, DEV, held_only=True, eight=True)
    k = torch.zeros(1, len(fills), 1, D, dtype=dtype)
    for i, f in enumerate(fills):
        k[0, i, 0, i] = f
        k[0, i, 0, 40] = 0.25 * (f if f == f and abs(f) < 1e30 else 1.0)
    k = k.to(DEV)
    v = (k * 1.0).contiguous()
    q = make_q(len(fills), 1, D, dtype)
    _, rows_k, rows_v = slab_append(kerns, c, 1, 0, q, k, v)
    max_e = 7 if dtype == torch.float16 else 119
    want = [expected_e4m3(c, r.double().cpu(), pool, sc, max_e) for r, pool, sc in ((rows_k, c.k_pages, c.k_scales), (rows_v, c.v_pages, c.v_scales))]
    kerns.rope_kv_append_paged_fp8(1, 0, BASE, q, k, v, c.cu, c.past, c.table, c.k_pages, c.v_pages, c.k_scales, c.v_scales)
    torch.cuda.synchronize()
    for pool, sc, (raw, exps) in zip((c.k_pages, c.v_pages), (c.k_scales, c.v_scales), want):
        assert torch.equal(sc.view(torch.uint8).cpu().to(torch.int64) - 127, exps)
        assert same_codes(bits(pool).cpu(), raw)


@pytest.mark.parametrize("eight", [False, True], ids=["16", "e4m3"])
def test_append_pages_that_are_not_there(kerns, eight):
    """Rows of such pages are dropped, negative positions too; q is rotated all the same.  Tokens of no sequence stay."""
    c = ref.Paged([(40, 10), (1, 33), (3, 2)], 16, 2, 64, torch.float16, DEV, held_only=True, eight=eight, gone={(0, 1), (1, 2)})
    c.past[2] = -2
    T = c.T + 4
    q = make_q(T, 4, 64, torch.float16)
    q0 = q.clone()
    k, v = make_kv(T, 2, 64, torch.float16)
    before = [bits(c.k_pages).clone(), bits(c.v_pages).clone()]
    call = kerns.rope_kv_append_paged_fp8 if eight else kerns.rope_kv_append_paged
    call(1, 64, BASE, q, k, v, c.cu, c.past, c.table, c.k_pages, c.v_pages, *c.scales())
    torch.cuda.synchronize()
    assert torch.equal(q[:, c.T:], q0[:, c.T:])
    y = ref.rotated(q0[0, :40].double().cpu(), 10, 1, 64, BASE)
    assert ((q[0, :40].double().cpu() - y).abs() <= 2.0 ** -11 * (1 + 1e-3) * y.abs() + 2.0 ** -20 * 8).all()
    for pool, old in zip((c.k_pages, c.v_pages), before):
        changed = (bits(pool) != old).flatten(3).any(-1).any(1).cpu()    # [page, row]
        want = torch.zeros_like(changed)
        for s, first, n in ((0, 10, 40), (2, 0, 1)):
            for r in range(first, first + n):
                p = c.table_list[s][r // 16]
                if p >= 0:
                    want[p, r % 16] = True
        if eight:
            assert not (changed & ~want).any(1)[[p for p in range(c.n_pages) if p not in (c.table_list[0][0], c.table_list[2][0])]].any()
        else:
            assert torch.equal(changed, want)


@pytest.mark.parametrize("eight", [False, True], ids=["16", "e4m3"])
def test_append_malformed_index_tensors_stay_in_bounds(kerns, eight):
    c = ref.Paged([(3, 4), (20, 9)], 16, 2, 64, torch.float16, DEV, held_only=True, eight=eight)
    k, v = make_kv(c.T, 2, 64, torch.float16)
    unused = [p for p in range(c.n_pages) if p not in sum(c.table_list, [])]
    before = bits(c.k_pages)[unused].clone()
    whole = torch.full((1, c.T + 20, 4, 64), 5.0, dtype=torch.float16, device=DEV)
    q = whole[:, 10:10 + c.T]
    call = kerns.rope_kv_append_paged_fp8 if eight else kerns.rope_kv_append_paged
    for cu in ([0, c.T + 100, 2 * c.T], [-5, 3, c.T], [c.T, 1, 0], [2 ** 31 - 1, -2 ** 31, 7], [0, 0, 0]):
        for past in ([2 ** 31 - 1, 5], [-4, -2 ** 31], [1 << 20, 1]):
            c.cu.copy_(torch.tensor(cu, dtype=torch.int32))
            c.past.copy_(torch.tensor(past, dtype=torch.int32))
            call(1, 64, BASE, q, k, v, c.cu, c.past, c.table, c.k_pages, c.v_pages, *c.scales())
            torch.cuda.synchronize()
            assert (whole[:, :10] == 5).all() and (whole[:, 10 + c.T:] == 5).all()
            assert torch.equal(bits(c.k_pages)[unused], before)


def test_append_many_sequences(kerns):
    """More sequences than lanes, thousands of them, empty ones between."""
    g = torch.Generator().manual_seed(5)
    seqs = [(int(n), int(p)) for n, p in zip(torch.randint(0, 3, (5000,), generator=g), torch.randint(0, 20, (5000,), generator=g))]
    for eight in (False, True):
        c = ref.Paged(seqs, 16, 1, 64, torch.float16, DEV, held_only=True, eight=False)
        if eight:
            c.eight = True
            c.k_pages, c.v_pages = (torch.zeros(c.n_pages, 1, 16, 64, dtype=torch.uint8, device=DEV).view(torch.float8_e4m3fn) for _ in range(2))
            c.k_scales, c.v_scales = (torch.full((c.n_pages, 1), 100, dtype=torch.uint8, device=DEV).view(torch.float8_e8m0fnu) for _ in range(2))
        q = make_q(c.T, 1, 64, torch.float16)
        k, v = make_kv(c.T, 1, 64, torch.float16)
        call = kerns.rope_kv_append_paged_fp8 if eight else kerns.rope_kv_append_paged
        call(1, 0, BASE, q, k, v, c.cu, c.past, c.table, c.k_pages, c.v_pages, *c.scales())
        torch.cuda.synchronize()
        page, row, tok = zip(*[(c.table_list[s][(p + i) // 16], (p + i) % 16, c.cu_list[s] + i) for s, (n, p) in enumerate(seqs) for i in range(n)])
        got = c.v_pages.float()[list(page), 0, list(row)]
        want = v[0, list(tok), 0].float()
        if eight:
            got = got * c.v_scales.float()[list(page)]
            assert ((got - want).abs() <= 2.0 ** -4 * want.abs() + 2.0 ** -5).all()
        else:
            assert torch.equal(got, want)
        if not eight:
            out = torch.empty_like(q)
            run_attend(kerns, c, q, out)
            tokens = [c.cu_list[s] for s, (n, p) in enumerate(seqs) if n > 0 and p == 0]   # attend their own row alone
            assert torch.equal(out[0, tokens], v[0, tokens])


# ---- together ------------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("eight", [False, True], ids=["16", "e4m3"])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16], ids=["f16", "bf16"])
def test_serving_run(kerns, dtype, eight):
    """Two prompts in chunks, then tokens one at a time, a page taken from the pool when one is needed: after every step the attention
    over the pages equals the attention over what they stand for, and, in 16 bits, the decode over one-slab caches."""
    Hq, Hkv, D, page = 8, 2, 128, 16
    n_pages, P = 40, 12
    if eight:
        k_pages, v_pages = (torch.full((n_pages, Hkv, page, D), 0x7F, dtype=torch.uint8, device=DEV).view(torch.float8_e4m3fn) for _ in range(2))
        scales = tuple(torch.zeros(n_pages, Hkv, dtype=torch.uint8, device=DEV).view(torch.float8_e8m0fnu) for _ in range(2))
    else:
        k_pages, v_pages = (torch.full((n_pages, Hkv, page, D), float("nan"), dtype=dtype, device=DEV) for _ in range(2))
        scales = ()
    free = torch.randperm(n_pages, generator=torch.Generator().manual_seed(9)).tolist()
    table = torch.full((2, P), -1, dtype=torch.int32)
    held = [0, 0]
    slab_k, slab_v = (torch.zeros(2, Hkv, P * page, D, dtype=dtype, device=DEV) for _ in range(2))
    g = torch.Generator().manual_seed(11)
    for step, lens in enumerate([(37, 20), (30, 0), (1, 50), (1, 1), (1, 1), (1, 1), (4, 3), (1, 1)]):
        for s in range(2):
            for i in range((held[s] + page - 1) // page, (held[s] + lens[s] + page - 1) // page):
                table[s, i] = free.pop()
        T = sum(lens)
        q, k, v = (torch.randn(1, T, h, D, generator=g).to(dtype).to(DEV) for h in (Hq, Hkv, Hkv))
        cu = torch.tensor([0, lens[0], T], dtype=torch.int32, device=DEV)
        pos = torch.tensor(held, dtype=torch.int32, device=DEV)
        ctx = torch.tensor([held[0] + lens[0], held[1] + lens[1]], dtype=torch.int32, device=DEV)
        bt = table.to(DEV)
        q_slab = q.clone()
        append = kerns.rope_kv_append_paged_fp8 if eight else kerns.rope_kv_append_paged
        append(1, D, BASE, q, k, v, cu, pos, bt, k_pages, v_pages, *scales)
        for s in range(2):
            if lens[s]:
                part = slice(cu[s].item(), cu[s + 1].item())
                x = q_slab[:, part].contiguous()
                kerns.rope_kv_append(1, D, BASE, x, k[:, part].contiguous(), v[:, part].contiguous(), pos[s:s + 1], slab_k[s:s + 1], slab_v[s:s + 1])
                q_slab[:, part] = x
        assert torch.equal(bits(q), bits(q_slab))
        out = torch.empty_like(q)
        attend = kerns.flash_attn_paged_fp8 if eight else kerns.flash_attn_paged
        attend(*QT[dtype], q.transpose(1, 2), k_pages, v_pages, *scales, bt, cu, ctx, max(lens), out.transpose(1, 2))
        held = [held[0] + lens[0], held[1] + lens[1]]
        # what the pages stand for, as dense rows
        c = ref.Paged([(n, h - n) for n, h in zip(lens, held)], page, Hkv, D, dtype, DEV)
        for name, pages, slab, i in (("k", k_pages, slab_k, 0), ("v", v_pages, slab_v, 1)):
            dense = []
            for s in range(2):
                ids = table[s, :(held[s] + page - 1) // page].long().to(DEV)
                x = pages.view(torch.uint8)[ids].view(torch.float8_e4m3fn).double() * scales[i].double()[ids][:, :, None, None] if eight else pages[ids].double()
                x = x.transpose(0, 1).flatten(1, 2)[:, :held[s]].cpu()
                dense.append(x)
                y = slab[s, :, :held[s]].double().cpu()
                if eight:   # half an e4m3 step, or half the smallest one under the page's scale, whose codes may have been moved a few times
                    assert ((x - y).abs() <= 2.0 ** -4 * y.abs() + 4 * 2.0 ** -10 * y.abs().max() / 224).all()
                else:
                    assert torch.equal(x, y)
            setattr(c, name + "_dense", dense)
        want, bound = ref.attend(c, q[0].transpose(0, 1))
        err = (out[0].transpose(0, 1).double().cpu() - want).abs()
        assert (err <= bound).all(), (step, float((err / bound).max()))


@pytest.mark.parametrize("eight", [False, True], ids=["16", "e4m3"])
@pytest.mark.parametrize("n", [1, 3, 40])
def test_graph(kerns, n, eight):
    """Append and attention captured once and replayed with other tokens, positions and pages, the program's own work between
    the replays: every replay equals the eager calls."""
    seqs = [(n, 100), (n, 31), (n, 700)]
    c = ref.Paged(seqs, 16, 2, 128, torch.bfloat16, DEV, held_only=True, eight=eight, width=64)
    k, v = make_kv(c.T, 2, 128, torch.bfloat16)
    q0 = make_q(c.T, 8, 128, torch.bfloat16)
    q, out = q0.clone(), torch.empty_like(q0)
    append = kerns.rope_kv_append_paged_fp8 if eight else kerns.rope_kv_append_paged

    def step(q, out, k_pages, v_pages, scales):
        append(1, 128, BASE, q, k, v, c.cu, c.past, c.table, k_pages, v_pages, *scales)
        call = kerns.flash_attn_paged_fp8 if eight else kerns.flash_attn_paged
        call(30, 256, 512, q.transpose(1, 2), k_pages, v_pages, *scales, c.table, c.cu, c.ctx, n, out.transpose(1, 2))

    fresh = [t.clone() for t in (c.k_pages, c.v_pages, *c.scales())]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(q, out, c.k_pages, c.v_pages, c.scales())
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(q, out, c.k_pages, c.v_pages, c.scales())
    for replay in range(4):
        g = torch.Generator().manual_seed(replay)
        k.copy_(torch.randn(k.shape, generator=g))
        q0.copy_(torch.randn(q0.shape, generator=g))
        past = [100 + replay, 31 - 7 * replay, 700 - 200 * replay]
        c.past.copy_(torch.tensor(past, dtype=torch.int32))
        c.ctx.copy_(torch.tensor([p + n for p in past], dtype=torch.int32))
        for t, f in zip((c.k_pages, c.v_pages, *c.scales()), fresh):
            bits(t).copy_(bits(f))
        state = [t.clone() for t in fresh]
        q.copy_(q0)
        graph.replay()
        torch.cuda.synchronize()
        q2, out2 = q0.clone(), torch.empty_like(out)
        step(q2, out2, state[0], state[1], tuple(state[2:]))
        torch.cuda.synchronize()
        assert torch.equal(q, q2) and torch.equal(bits(out), bits(out2))
        for t, f in zip((c.k_pages, c.v_pages, *c.scales()), state):
            assert torch.equal(bits(t), bits(f))


def test_opcheck(kerns):
    c = ref.Paged([(2, 5), (1, 20)], 16, 2, 64, torch.float16, DEV)
    c8 = ref.Paged([(2, 5), (1, 20)], 16, 2, 64, torch.float16, DEV, eight=True)
    q = make_q(c.T, 4, 64, torch.float16)
    k, v = make_kv(c.T, 2, 64, torch.float16)
    ops = torch.ops.minfer
    utils = ("test_schema", "test_faketensor")
    torch.library.opcheck(ops.rope_kv_append_paged.default, (1, 64, BASE, q.clone(), k, v, c.cu, c.past, c.table, c.k_pages.nan_to_num(0), c.v_pages.nan_to_num(0)), test_utils=utils)
    qt = q.transpose(1, 2)
    torch.library.opcheck(ops.flash_attn_paged.default, (1, 1, 2, qt, c.k_pages, c.v_pages, c.table, c.cu, c.ctx, 2, torch.zeros_like(q).transpose(1, 2)), test_utils=("test_faketensor",))
    torch.library.opcheck(ops.rope_kv_append_paged_fp8.default, (1, 64, BASE, q.clone(), k, v, c8.cu, c8.past, c8.table, c8.k_pages, c8.v_pages, *c8.scales()), test_utils=("test_faketensor",))
    torch.library.opcheck(ops.flash_attn_paged_fp8.default, (1, 1, 2, qt, c8.k_pages, c8.v_pages, *c8.scales(), c8.table, c8.cu, c8.ctx, 2, torch.zeros_like(q).transpose(1, 2)),
                          test_utils=("test_faketensor",))
