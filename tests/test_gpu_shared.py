"""Attention of groups that share a prefix, against float64 with a bound for every element, and against flash_attn_paged."""
import pytest
import torch

import paged_ref as ref

pytestmark = pytest.mark.gpu
DEV = "cuda"
QT = {torch.float16: (1, 1, 2), torch.bfloat16: (30, 256, 512)}


class Shared(ref.Paged):
    """A paged cache in which the sequences first .. last - 1 of every group (first, last, rows) name the first one's pages for those rows,
    rounded up to whole pages; a sequence that ends inside them has its last pages, and rows, from there."""

    # wide: the table has entries for so many rows that the call is one for the kernels that know of groups
    def __init__(self, seqs, groups, page, Hkv, D, dtype, told=None, wide=True, **kw):
        need = -(-max(sum(x) for x in seqs) // page) + 1
        width = max(need, 230000000 // (len(seqs) * Hkv * D * (2 if kw.get("eight") else 4) * page)) if wide else need
        super().__init__(seqs, page, Hkv, D, dtype, "cpu", width=width, **kw)
        self.k_dense, self.v_dense = list(self.k_dense), list(self.v_dense)
        for first, last, rows in groups:
            n = -(-rows // page)
            assert n * page <= sum(seqs[first])
            for s in range(first + 1, last):
                m = min(n, len(self.table_list[s]))
                self.table_list[s][:m] = self.table_list[first][:m]
                self.table[s, :m] = self.table[first, :m]
                for dense in (self.k_dense, self.v_dense):
                    have = min(m * page, sum(seqs[s]))
                    dense[s] = torch.cat((dense[first][:, :have], dense[s][:, have:]), 1)
        self.told = [r for _, _, r in groups] if told is None else told
        self.cu_groups = [first for first, _, _ in groups] + [groups[-1][1] if groups else 0]
        for name in ("table", "cu", "ctx", "k_pages", "v_pages", "k_scales", "v_scales"):
            x = getattr(self, name)
            setattr(self, name, None if x is None else x.to(DEV) if name[1:] != "_pages" or kw.get("order") != "rows" else x.transpose(1, 2).to(DEV).transpose(1, 2))

    def call(self, kerns, q, max_q=None, out=None, cu=None, groups=None, told=None):
        out = torch.full_like(q, float("nan")) if out is None else out
        f = kerns.flash_attn_paged_shared_fp8 if self.eight else kerns.flash_attn_paged_shared
        max_q = max([n for n, _ in self.seqs] + [1]) if max_q is None else max_q
        i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=DEV)
        f(*QT[q.dtype], q, self.k_pages, self.v_pages, *self.scales(), self.table, self.cu if cu is None else i32(cu), self.ctx,
          i32(self.cu_groups if groups is None else groups), i32(self.told if told is None else told), max_q, out)
        return out

    def unshared(self, kerns, q):
        out = torch.full_like(q, float("nan"))
        f = kerns.flash_attn_paged_fp8 if self.eight else kerns.flash_attn_paged
        f(*QT[q.dtype], q, self.k_pages, self.v_pages, *self.scales(), self.table, self.cu, self.ctx, max([n for n, _ in self.seqs] + [1]), out)
        return out


def queries(c, Hq, dtype, seed=0):
    g = torch.Generator().manual_seed(seed)
    return torch.randn(1, c.T, Hq, c.D, generator=g).to(dtype).to(DEV).transpose(1, 2)


def check(kerns, c, Hq, dtype, seed=0, **kw):
    q = queries(c, Hq, dtype, seed)
    out = c.call(kerns, q, **kw)
    want, bound = ref.attend(c, q[0].cpu())
    err = (out[0].cpu().double() - want).abs()
    assert not torch.isnan(err).any()
    assert (err <= bound).all(), float((err / bound).max())
    return out


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("eight", [False, True])
@pytest.mark.parametrize("Hq,Hkv,D", [(8, 2, 64), (8, 2, 128), (3, 3, 128), (32, 2, 64), (40, 2, 128), (16, 16, 64)])
def test_single_tokens(kerns, dtype, eight, Hq, Hkv, D):
    lens = [(1, 256 + p) for p in (0, 1, 15, 16, 40, 63, 200, 333)]
    check(kerns, Shared(lens, [(0, 8, 256)], 16, Hkv, D, dtype, eight=eight, seed=D), Hq, dtype)


@pytest.mark.parametrize("eight", [False, True])
def test_where_all_rows_fit_the_cache_it_is_flash_attn_paged(kerns, eight):
    c = Shared([(1, 256 + 9 * i) for i in range(6)], [(0, 6, 256)], 16, 2, 64, torch.float16, wide=False, eight=eight)
    q = queries(c, 8, torch.float16)
    assert torch.equal(c.call(kerns, q), c.unshared(kerns, q))


@pytest.mark.parametrize("eight", [False, True])
@pytest.mark.parametrize("page", [16, 64, 256])
@pytest.mark.parametrize("rows,told", [(256, 256), (512, 300), (256, 63), (256, 64), (512, 511), (768, 0), (256, -4)])
def test_prefixes_of_any_length(kerns, eight, page, rows, told):
    lens = [(1, rows + 10 * i) for i in range(5)]
    check(kerns, Shared(lens, [(0, 5, rows)], page, 2, 64, torch.float16, told=[told], eight=eight, seed=told + 9), 8, torch.float16)


@pytest.mark.parametrize("order", ["heads", "rows"])
@pytest.mark.parametrize("eight", [False, True])
def test_several_groups_and_sequences_without(kerns, order, eight):
    lens = [(1, 30), (1, 0)] + [(1, 200 + 7 * i) for i in range(6)] + [(1, 70 + i) for i in range(2)] + [(1, 640 + 90 * i) for i in range(5)] + [(1, 0), (1, 500)]
    c = Shared(lens, [(2, 8, 192), (8, 10, 64), (10, 15, 640)], 32, 4, 128, torch.bfloat16, order=order, eight=eight, gap=3)
    check(kerns, c, 12, torch.bfloat16)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("eight", [False, True])
@pytest.mark.parametrize("Hq,Hkv,D,most", [(8, 2, 128, 4), (8, 2, 64, 16), (4, 4, 128, 9), (12, 4, 64, 21), (32, 2, 128, 4)])
def test_drafts(kerns, dtype, eight, Hq, Hkv, D, most):
    lens = [(1 + (3 * i) % most, 320 + 13 * i) for i in range(9)] + [(2, 5)]
    check(kerns, Shared(lens, [(0, 9, 320)], 64, Hkv, D, dtype, eight=eight, seed=most), Hq, dtype)


@pytest.mark.parametrize("eight", [False, True])
@pytest.mark.parametrize("Hq,Hkv,D,most", [(24, 4, 128, 3), (8, 2, 128, 6), (16, 1, 64, 2), (8, 2, 64, 11), (48, 4, 128, 3), (40, 2, 64, 1), (13, 1, 128, 4), (96, 1, 64, 1), (101, 1, 128, 1)])
def test_more_than_16_columns(kerns, eight, Hq, Hkv, D, most):
    """17 to 101 (token, head) rows per KV head, in whole and partly filled pairs of 16; sequences that fill the first 16 alone; shares that end inside a sequence."""
    lens = [(1 + (5 * i) % most, 192 + (37 * i) % 900) for i in range(14)] + [(most, 3), (1, 200)]
    check(kerns, Shared(lens, [(0, 14, 192)], 32, Hkv, D, torch.bfloat16 if most == 3 else torch.float16, eight=eight, seed=Hq), Hq, torch.bfloat16 if most == 3 else torch.float16)


@pytest.mark.parametrize("eight", [False, True])
@pytest.mark.parametrize("D", [64, 128])
def test_a_row_that_some_of_a_pair_of_columns_attend(kerns, eight, D):
    """A NaN that the last drafts of a sequence attend and the first ones do not, at a border of 16 columns and on either side of it."""
    lens = [(7, 256 + 20 * i) for i in range(5)]
    clean = Shared(lens, [(0, 5, 256)], 16, 2, D, torch.float16, eight=eight)
    q = queries(clean, 8, torch.float16)
    want, bound = ref.attend(clean, q[0].cpu())
    for tok in (3, 4, 5):
        c = Shared(lens, [(0, 5, 256)], 16, 2, D, torch.float16, eight=eight)
        raw, row = c.v_pages.view(torch.uint8) if eight else c.v_pages, 276 + tok
        raw[c.table_list[1][row // 16], 1, row % 16, 9] = 0x7F if eight else float("nan")
        out = c.call(kerns, q)
        seen = torch.isnan(out[0]).any(-1)
        assert seen[4:].any(0).nonzero().flatten().tolist() == list(range(7 + tok, 14)) and not seen[:4].any()
        rest = [t for t in range(35) if not 7 + tok <= t < 14]
        assert ((out[0].cpu().double() - want).abs() <= bound)[:, rest].all()


def test_drafts_over_codes_in_a_table_just_wide_enough(kerns):
    """From 25 MB on the kernels for groups take what goes to flash_attn_paged below: both sides right, and 16 columns still the latter's."""
    lens = [(1 + 5 * (i % 2), 1100 + 10 * i) for i in range(8)]
    for Hkv, most in ((4, 6), (8, 6), (8, 4)):
        c = Shared([(min(n, most), past) for n, past in lens], [(0, 8, 512)], 512, Hkv, 128, torch.float16, wide=False, eight=True)
        q = queries(c, 4 * Hkv, torch.float16)
        out = check(kerns, c, 4 * Hkv, torch.float16)
        takes = most == 6 and 8 * c.width * 512 * 2 * Hkv * 128 >= 25000000
        assert takes == ((Hkv, most) == (8, 6))
        assert takes or torch.equal(out, c.unshared(kerns, q))


def test_longer_chunks_are_flash_attn_paged(kerns):
    c = Shared([(40, 128), (3, 140), (70, 200)], [(0, 3, 128)], 16, 2, 128, torch.float16)
    q = queries(c, 8, torch.float16)
    assert torch.equal(c.call(kerns, q), c.unshared(kerns, q))
    c = Shared([(1, 128), (1, 140)], [], 16, 2, 128, torch.float16)
    q = queries(c, 8, torch.float16)
    assert torch.equal(c.call(kerns, q), c.unshared(kerns, q))


@pytest.mark.parametrize("eight", [False, True])
def test_tokens_inside_the_prefix(kerns, eight):
    """Sequences that end in front of the prefix's end, or whose new tokens lie in it: each token attends the rows up to its own."""
    lens = [(1, 400), (3, 381), (4, 10), (1, 0), (2, 62), (4, 126), (1, 500), (4, 400)]
    check(kerns, Shared(lens, [(0, 8, 384)], 16, 2, 64, torch.float16, eight=eight), 8, torch.float16)
    lens = [(3, 300)] + [(1 + i % 4, 37 * i) for i in range(40)]
    check(kerns, Shared(lens, [(0, 41, 256)], 32, 2, 128, torch.bfloat16, eight=eight), 8, torch.bfloat16)


@pytest.mark.parametrize("n,groups", [(70, 1), (150, 3), (300, 100), (130, 65)])
def test_many_sequences_and_groups(kerns, n, groups):
    per = n // groups
    lens = [(1, 128 + (11 * s) % 50) for s in range(n)]
    check(kerns, Shared(lens, [(i * per, (i + 1) * per, 128) for i in range(groups)], 16, 2, 64, torch.float16), 8, torch.float16)


def test_more_sequences_than_are_looked_up_at_once(kerns):
    """More than 64 times 64 sequences, and as many groups of one and two behind each other."""
    lens = [(1, 64 + s % 3) for s in range(4300)]
    check(kerns, Shared(lens, [(10, 4290, 64)], 16, 1, 64, torch.float16, extra=1), 2, torch.float16)
    groups, at = [], 0
    while at < 4250:
        n = 1 + (at // 7) % 2
        groups.append((at, at + n, 64))
        at += n
    check(kerns, Shared(lens, groups[:4200], 16, 1, 64, torch.float16, extra=1), 2, torch.float16)


@pytest.mark.parametrize("D", [64, 128])
def test_missing_pages_beside_a_page_of_no_numbers(kerns, D):
    """Codes: pages that are missing in the prefix and among own rows, where nothing of the pool's first page, which is nobody's and holds codes and scales that are no numbers, is taken in their place."""
    lens = [(1 + i % 2, 300 + 30 * i) for i in range(5)]
    gone = {(s, i) for s in range(5) for i in (3, 8)} | {(1, 19), (3, 22)}
    c = Shared(lens, [(0, 5, 256)], 16, 2, D, torch.float16, gone=gone, eight=True)
    used = {x for row in c.table_list for x in row}
    free = next(i for i in range(1, c.n_pages) if i not in used)
    for pool in (c.k_pages, c.v_pages, c.k_scales, c.v_scales):
        x = pool.view(torch.uint8)
        x[free] = x[0]
        x[0] = 0x7F if pool.dim() == 4 else 0xFF
    c.table[c.table == 0] = free
    c.table_list = [[free if x == 0 else x for x in row] for row in c.table_list]
    check(kerns, c, 8, torch.float16)


def test_long_prefix_of_a_few(kerns):
    """More pieces than a merge takes of one row, were they as short as they may be."""
    lens = [(1, 20000 + 100 * i) for i in range(3)]
    check(kerns, Shared(lens, [(0, 3, 19968)], 256, 1, 64, torch.float16), 4, torch.float16)


def test_empty_sequences_and_padding(kerns):
    lens = [(0, 200), (1, 130), (0, 0), (2, 140), (0, 128), (1, 129), (0, 0), (0, 0)]
    c = Shared(lens, [(0, 6, 128)], 16, 2, 64, torch.float16)
    want = check(kerns, c, 8, torch.float16, max_q=2)
    q = queries(c, 8, torch.float16)
    for cu in (c.cu_list[:7] + [0, 0], c.cu_list[:7] + [9, 9]):
        assert torch.equal(c.call(kerns, q, max_q=2, cu=cu), want)
    # (an end in front of its start: the sixth sequence has no token, and the fourth token belongs to nobody)
    cut = c.call(kerns, q, max_q=2, cu=c.cu_list[:6] + [0, 0, 0])
    assert torch.equal(cut[:, :, :3], want[:, :, :3]) and torch.isnan(cut[:, :, 3]).all()
    # the group reaches over the sequences without tokens behind the last one
    for cu in (c.cu_list[:6] + [4, 0, 0], c.cu_list[:6] + [4, 4, 4], c.cu_list[:6] + [4, 2, 0], c.cu_list[:6] + [4, 3, 1], c.cu_list[:6] + [4, 9, 2]):
        assert torch.equal(c.call(kerns, q, max_q=2, cu=cu, groups=[0, 8]), want)
    # rows behind the last sequence stay as they were
    out = torch.full((1, 8, c.T + 3, 64), 7.0, dtype=torch.float16, device=DEV)
    q = torch.cat((q, torch.full((1, 8, 3, 64), float("nan"), dtype=torch.float16, device=DEV)), 2)
    c.call(kerns, q, max_q=2, out=out)
    assert torch.equal(out[:, :, :c.T], want) and (out[:, :, c.T:] == 7.0).all()


def test_a_group_of_empty_sequences_and_groups_of_one(kerns):
    lens = [(0, 70), (0, 80), (1, 200), (1, 90), (0, 64), (1, 300)]
    check(kerns, Shared(lens, [(0, 2, 64), (2, 3, 192), (3, 5, 64), (5, 6, 256)], 16, 2, 128, torch.bfloat16), 4, torch.bfloat16, max_q=1)


def test_pages_that_are_gone(kerns):
    """First pages of the prefix that a window gave back, a hole in it, and all of it."""
    lens = [(1, 520 + 9 * i) for i in range(6)]
    for gone in ([(s, i) for s in range(6) for i in range(7)], [(s, 9) for s in range(6)], [(s, i) for s in range(6) for i in range(32)], [(s, i) for s in range(6) for i in range(99)]):
        for eight in (False, True):
            check(kerns, Shared(lens, [(0, 6, 512)], 16, 2, 64, torch.float16, gone=gone, eight=eight), 8, torch.float16)


@pytest.mark.parametrize("eight", [False, True])
def test_rows_that_are_no_numbers(kerns, eight):
    """A NaN in the prefix reaches every token; one in a sequence's own rows that sequence's tokens from there on; one inside the prefix, behind a token, not it."""
    lens = [(2, 256 + 20 * i) for i in range(4)] + [(3, 100)]
    clean = Shared(lens, [(0, 5, 256)], 16, 2, 64, torch.float16, eight=eight)
    q = queries(clean, 8, torch.float16)
    base = clean.call(kerns, q)
    want, bound = ref.attend(clean, q[0].cpu())
    for s, row, hit in ((0, 30, list(range(11))), (1, 277, [3]), (0, 101, [0, 1, 2, 3, 4, 5, 6, 7, 9, 10]), (0, 250, list(range(8)))):
        c = Shared(lens, [(0, 5, 256)], 16, 2, 64, torch.float16, eight=eight)
        raw = c.v_pages.view(torch.uint8) if eight else c.v_pages
        raw[c.table_list[s][row // 16], 0, row % 16, 5] = 0x7F if eight else float("nan")
        out = c.call(kerns, q)
        seen = torch.isnan(out[0]).any(-1)
        assert seen[:4].any(0).nonzero().flatten().tolist() == hit
        assert not seen[4:].any() and torch.equal(out[:, 4:], base[:, 4:])
        # (keys from the row on are added one by one for the tokens in front of it, in another order)
        rest = [t for t in range(11) if t not in hit]
        assert ((out[0].cpu().double() - want).abs() <= bound)[:, rest].all()


def test_groups_that_nobody_checked(kerns):
    """Whatever cu_groups and prefix_lens hold: nothing out of bounds, and tokens of sequences that no group covers are right."""
    lens = [(1, 200 + i) for i in range(10)] + [(2, 100)]
    c = Shared(lens, [(0, 10, 192)], 16, 2, 64, torch.float16)
    q = queries(c, 8, torch.float16)
    want = c.unshared(kerns, q)
    for groups, told in (([0, 10, 3, 10], [192] * 3), ([5, 2, 9], [64, 192]), ([-7, 99], [1 << 30]), ([0, 11, 0, 11, 0, 11], [192] * 5), ([20, 30], [64]), ([0, 0, 0], [64, 64])):
        out = c.call(kerns, q, groups=groups, told=told)
        # (rows beyond those that are shared are read through the first sequence's table, where others' tokens may meet rows that nothing was written to)
        assert max(told) > 192 or not torch.isnan(out).any()
        if groups in ([20, 30], [0, 0, 0]):
            torch.testing.assert_close(out, want, atol=2e-3, rtol=2e-3)


def test_the_same_bits_again_on_another_stream_and_in_a_graph(kerns):
    lens = [(1 + i % 3, 700 + 31 * i) for i in range(20)]
    c = Shared(lens, [(0, 12, 640), (12, 18, 300)], 32, 2, 128, torch.bfloat16)
    q = queries(c, 8, torch.bfloat16)
    want = c.call(kerns, q)
    assert torch.equal(c.call(kerns, q), want)
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        assert torch.equal(c.call(kerns, q), want)
    torch.cuda.synchronize()
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=DEV)
    groups, told, out = i32(c.cu_groups), i32(c.told), torch.zeros_like(q)

    def step():
        kerns.flash_attn_paged_shared(*QT[q.dtype], q, c.k_pages, c.v_pages, c.table, c.cu, c.ctx, groups, told, 3, out)

    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        step()
    for k in range(3):
        told.copy_(i32([640, 300] if k != 1 else [128, 0]))
        out.zero_()
        g.replay()
        got = out.clone()
        step()
        assert torch.equal(got, out)
        if k != 1:
            assert torch.equal(got, want)


def test_calls_in_flight_on_two_streams(kerns):
    cases = [Shared([(1 + i % 2, 500 + 40 * i) for i in range(10)], [(0, 10, 448)], 16, 2, D, torch.float16, seed=D) for D in (64, 128)]
    qs = [queries(c, 8, torch.float16) for c in cases]
    wants = [c.call(kerns, q) for c, q in zip(cases, qs)]
    torch.cuda.synchronize()
    streams, outs = [torch.cuda.Stream(), torch.cuda.Stream()], [[], []]
    for _ in range(10):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                outs[i].append(cases[i].call(kerns, qs[i]))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(o, wants[i]) for o in outs[i])


def test_strides_and_large_offsets(kerns):
    """Views of q and out, and a pool whose pages lie past 2^32 bytes."""
    lens = [(1, 130 + i) for i in range(4)]
    c = Shared(lens, [(0, 4, 128)], 16, 1, 128, torch.float16)
    big = torch.empty((1 << 31) // (16 * 128) + 64, 1, 16, 128, dtype=torch.float16, device=DEV)   # 4 GiB
    far = big.shape[0] - c.n_pages
    want = check(kerns, c, 4, torch.float16)
    for name in ("k_pages", "v_pages"):
        big[far:] = getattr(c, name)
        if name == "k_pages":
            c.k_pages = big
            keep = big
            big = torch.empty_like(big)
        else:
            c.v_pages = big
    c.table = torch.where(c.table >= 0, c.table + far, -1).to(torch.int32)
    q = queries(c, 4, torch.float16)
    wide = torch.zeros(1, c.T, 9, 128 + 8, dtype=torch.float16, device=DEV)
    wide[:, :, 2:6, :128] = q.transpose(1, 2)
    out = torch.full((1, c.T, 8, 128 + 16), 5.0, dtype=torch.float16, device=DEV)
    c.call(kerns, wide[:, :, 2:6, :128].transpose(1, 2), out=out[:, :, 1:5, :128].transpose(1, 2))
    assert torch.equal(out[:, :, 1:5, :128].transpose(1, 2), want)
    out[:, :, 1:5, :128] = 5.0
    assert (out == 5.0).all()
    del keep


def test_refusals(kerns):
    c = Shared([(1, 130), (1, 140)], [(0, 2, 128)], 16, 2, 64, torch.float16)
    q = queries(c, 8, torch.float16)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=DEV)
    good = [*QT[q.dtype], q, c.k_pages, c.v_pages, c.table, c.cu, c.ctx, i32([0, 2]), i32([128]), 1, torch.empty_like(q)]
    for at, x, text in ((9, i32([0]), "prefix_lens"), (9, i32([[0, 2]]), "cu_groups"), (9, good[9].long(), "cu_groups"), (9, i32([0, 1, 2, 2]), "prefix_lens"), (10, good[10].float(), "prefix_lens"),
                        (3, q.float(), "float16 or bfloat16"), (4, c.k_pages.bfloat16(), "q's dtype"), (8, c.ctx[:1], "ctx_lens"), (11, -1, "negative"), (0, 8, "Q8_0")):
        with pytest.raises(RuntimeError, match=text):
            kerns.flash_attn_paged_shared(*good[:at], x, *good[at + 1:])
    with pytest.raises(RuntimeError, match="more groups"):
        kerns.flash_attn_paged_shared(*good[:9], i32([0, 1, 2, 2]), i32([64, 64, 64]), *good[11:])
