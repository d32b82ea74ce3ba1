"""Host side of the operators of a serving step, without a GPU: what they refuse (nothing is launched: the pointers are made up), their workspace
sizes, their place in the Python surface, and the definitions that the GPU tests compare with."""
import ctypes

import pytest
import torch

import capi
import capi_paged as cp
import capi_serving as cs
import serving_ref as ref
from test_paged_host import BAD_PAGES, pages

P = 0x100000   # made-up, 16-byte aligned addresses that do not overlap
A = [P + i * 0x10000 for i in range(16)]


def ring(**kw):
    d = dict(pages=A[0], state=A[1], state_after=A[2], n_pages=100)
    d.update(kw)
    return cs.PageRing(**d)


def tables(page=16, past=A[3], new=A[4], held=A[5], rg=None, table=A[6], stride=8, width=8, cu=A[7], ctx=A[8], slots=A[9], n_slots=10, after=A[10], n=4):
    rg = ring() if rg is None else rg
    return cs.lib().minfer_paged_tables(page, past, new, held, ctypes.byref(rg) if rg else None, table, stride, width, cu, ctx, slots, n_slots, after, n, None)


def release(page=16, keep=A[3], held=A[5], rg=None, table=A[6], stride=8, width=8, after=A[10], n=4, ws=A[11], ws_bytes=1 << 20):
    rg = ring() if rg is None else rg
    return cs.lib().minfer_paged_release(page, keep, held, ctypes.byref(rg) if rg else None, table, stride, width, after, n, ws, ws_bytes, None)


BAD_TABLES = [("page_size", dict(page=8)), ("page_size", dict(page=24)), ("page_size", dict(page=2048)), ("n_seqs", dict(n=-1)), ("n_seqs", dict(n=(1 << 24) + 1)),
              ("pages_per_seq", dict(width=-1)), ("pages_per_seq", dict(width=(1 << 26) + 1)), ("table_stride", dict(stride=7)), ("table_stride", dict(stride=-1)),
              ("number of pages", dict(rg=ring(n_pages=-1))), ("number of pages", dict(rg=ring(n_pages=1 << 31))), ("ring's pages", dict(rg=ring(pages=None))),
              ("ring's pages", dict(rg=ring(state=None))), ("ring's pages", dict(rg=ring(state_after=None))), ("must not be state", dict(rg=ring(state_after=A[1]))),
              ("must not be state", dict(rg=ring(state_after=A[1] + 8))), ("non-null", dict(held=None)), ("non-null", dict(table=None)), ("non-null", dict(after=None))]


@pytest.mark.parametrize("text,change", BAD_TABLES)
def test_tables_and_release_refuse(text, change):
    for call in (tables, release):
        assert call(**change) == capi.EINVAL
        assert text in capi.last_error()


@pytest.mark.parametrize("text,change", [
    ("n_slots", dict(n_slots=-1)), ("n_slots", dict(n_slots=1 << 31)), ("non-null", dict(cu=None)), ("non-null", dict(slots=None)), ("non-null", dict(past=None)),
    ("non-null", dict(new=None)), ("non-null", dict(ctx=None)), ("must not be inputs", dict(after=A[5])), ("must not be inputs", dict(ctx=A[3])), ("must not be inputs", dict(cu=A[4] + 12)),
    ("must not be inputs", dict(after=A[3] - 12))])
def test_tables_refuse(text, change):
    assert tables(**change) == capi.EINVAL
    assert text in capi.last_error()


def test_release_refuses():
    for change in (dict(after=A[5]), dict(after=A[3] + 4)):
        assert release(**change) == capi.EINVAL and "must not be inputs" in capi.last_error()
    assert release(keep=None) == capi.EINVAL
    need = cs.lib().minfer_paged_release_workspace_bytes(65)
    assert need >= 260 and cs.lib().minfer_paged_release_workspace_bytes(64) == 0   # (one launch does without)
    for ws, n in ((None, need), (A[11], need - 1), (A[11] + 2, need)):
        assert release(n=65, ws=ws, ws_bytes=n) == capi.EWORKSPACE and "workspace" in capi.last_error()
    null = cs.lib()
    assert null.minfer_paged_release(16, A[3], A[5], None, A[6], 8, 8, A[10], 4, A[11], 1 << 20, None) == capi.EINVAL and "ring is null" in capi.last_error()


def verify(dtype=capi.F32, bits=64, tokens=A[0], cu=A[1], target=A[2], draft=A[3], au=A[4], su=A[5], out=A[6], kept=A[7], n=3, T=9, V=100, ts=100, ds=100, ws=A[8], ws_bytes=1 << 30):
    return cs.lib().minfer_verify_drafts(dtype, bits, tokens, cu, target, draft, au, su, out, kept, n, T, V, ts, ds, ws, ws_bytes, None)


@pytest.mark.parametrize("text,change", [
    ("prob_dtype", dict(dtype=7)), ("prob_dtype", dict(dtype=capi.Q8_0)), ("token_bits", dict(bits=16)), ("n_seqs", dict(n=-1)), ("n_seqs", dict(n=65536)), ("T must", dict(T=-1)),
    ("T must", dict(T=(1 << 30) + 1)), ("V must", dict(V=0)), ("V must", dict(V=(1 << 28) + 1, ts=1 << 29, ds=1 << 29)), ("overlap", dict(ts=99)), ("overlap", dict(ds=99)),
    ("non-null", dict(cu=None)), ("non-null", dict(kept=None)), ("non-null", dict(su=None)), ("non-null", dict(tokens=None)), ("non-null", dict(target=None)),
    ("non-null", dict(au=None)), ("non-null", dict(out=None)), ("must not be tokens", dict(out=A[0])), ("must not be tokens", dict(out=A[0] + 64))])
def test_verify_refuses(text, change):
    assert verify(**change) == capi.EINVAL
    assert text in capi.last_error()


def test_verify_workspace():
    w = cs.lib().minfer_verify_drafts_workspace_bytes
    assert w(0, 100) == 0 and w(3, 0) == 0 and w(3, 2048) == 0       # a row of one chunk needs none
    need = w(3, 32000)
    assert need > 0 and verify(V=32000, ts=32000, ds=32000, ws_bytes=need - 1) == capi.EWORKSPACE
    assert verify(V=32000, ts=32000, ds=32000, ws=None) == capi.EWORKSPACE and verify(V=32000, ts=32000, ds=32000, ws=A[8] + 8) == capi.EWORKSPACE
    assert w(65535, 1 << 28) < 65535 * 256 * 8 + (1 << 20)           # 256 chunks of a row at most
    assert verify(n=0) == capi.OK


def shared(dtype=capi.F16, page_type=None, pg=None, q=P, cu=P, ctx=P, groups=P, prefix=P, out=P, n_seqs=4, n_groups=1, T=4, Hq=8, Hkv=2, D=128, max_q=1, st=None, ws=P, ws_bytes=1 << 40):
    st = st or capi.Strides(0, 128, 1024, 0, 0, 0, 0, 128, 1024)
    pg = wide() if pg is None else pg
    return cs.lib().minfer_flash_attn_paged_shared(dtype, dtype if page_type is None else page_type, q, ctypes.byref(pg) if pg else None, cu, ctx, groups, prefix, out, n_seqs,
                                                   n_groups, T, Hq, Hkv, D, max_q, ctypes.byref(st), ws, ws_bytes, None)


def wide(**kw):
    """Pages whose tables name more rows than fit the memory-side cache."""
    return pages(**{**dict(pages_per_seq=1 << 13, table_stride=1 << 13), **kw})


@pytest.mark.parametrize("text,change", BAD_PAGES)
def test_shared_refuses_bad_pages(text, change):
    for make in (pages, wide):
        assert shared(pg=make(**change)) == capi.EINVAL
        assert text in capi.last_error()


@pytest.mark.parametrize("text,change", [
    ("dtype", dict(dtype=capi.F32)), ("page_type", dict(page_type=capi.BF16)), ("head_dim", dict(D=96)), ("n_kv_heads", dict(Hkv=0)), ("multiple", dict(Hq=7)),
    ("n_heads > 65535", dict(Hq=131072)), ("negative", dict(n_seqs=-1)), ("negative", dict(T=-1)), ("negative", dict(max_q=-1)), ("negative", dict(n_groups=-1)), ("more groups", dict(n_groups=5)),
    ("non-null", dict(q=None)), ("non-null", dict(cu=None)), ("non-null", dict(ctx=None)), ("non-null", dict(out=None)), ("non-null", dict(groups=None)), ("non-null", dict(prefix=None)),
    ("aligned", dict(q=P + 4)), ("aligned", dict(out=P + 8)), ("strides", dict(st=capi.Strides(0, 4, 1024, 0, 0, 0, 0, 128, 1024))),
    ("strides", dict(st=capi.Strides(0, 128, 1024, 0, 0, 0, 0, 128, -8))), ("too large", dict(T=1 << 31)), ("too large", dict(n_seqs=1 << 20, T=1 << 20, pg=wide(pages_per_seq=1 << 20, table_stride=1 << 20)))])
def test_shared_refuses(text, change):
    assert shared(**change) == capi.EINVAL
    assert text in capi.last_error()


@pytest.mark.parametrize("D,max_q,rows", [(64, 4, (220000000 // 512, 150000000 // 256)), (64, 6, (70000000 // 512, 25000000 // 256)), (128, 4, (220000000 // 1024, 150000000 // 512)),
                                          (128, 6, (220000000 // 1024, 25000000 // 512))])
def test_shared_is_for_tables_of_many_rows(D, max_q, rows):
    """The workspace is that of flash_attn_paged below the first of the two kinds of pages' bounds, and larger from there on."""
    n, first = 16, -(-min(rows) // 16)
    f, plain = cs.lib().minfer_flash_attn_paged_shared_workspace_bytes, cs.lib().minfer_flash_attn_paged_workspace_bytes
    for context in (first - 1, first):
        args = (n * max_q, 8, 2, D, context, max_q)
        assert (f(n, 1, *args) > plain(n, *args)) == (context >= first)
        assert f(n, 0, *args) == plain(n, *args)


def test_shared_is_not_for_drafts_of_short_tables_or_small_groups():
    """More than 16 columns: 600 rows at least, 1000 and groups of three below 150 MB of codes; 16-bit rows, of which there are more bytes, 1200 or 2000 and groups of four."""
    f, plain = cs.lib().minfer_flash_attn_paged_shared_workspace_bytes, cs.lib().minfer_flash_attn_paged_workspace_bytes
    takes = lambda n, groups, context, max_q=6: f(n, groups, n * max_q, 32, 8, 128, context, max_q) > plain(n, n * max_q, 32, 8, 128, context, max_q)
    assert [takes(160, 1, c) for c in (592, 608)] == [False, True]
    assert [takes(40, 1, c) for c in (992, 1008)] == [False, True]
    assert [takes(40, g, 1500) for g in (14, 13)] == [False, True]
    assert [takes(160, g, 1500) for g in (81, 80)] == [False, True]
    assert takes(160, 160, 1500, max_q=1)


def test_shared_workspace_and_empty_calls():
    w = cs.lib().minfer_flash_attn_paged_shared_workspace_bytes
    for bad in ((0, 1, 1, 8, 2, 128, 1024, 1), (1, -1, 1, 8, 2, 128, 1024, 1), (1, 1, 0, 8, 2, 128, 1024, 1), (1, 1, 1, 7, 2, 128, 1024, 1)):
        assert w(*bad) == 0
    plain = cs.lib().minfer_flash_attn_paged_workspace_bytes
    # calls that know nothing of groups: short tables, long chunks, no groups
    for n, g, T, ctx, most in ((8, 1, 8, 2048, 1), (8, 1, 800, 1 << 17, 100), (8, 0, 8, 1 << 17, 1)):
        assert w(n, g, T, 32, 8, 128, ctx, most) == plain(n, T, 32, 8, 128, ctx, most)
    need = w(4, 1, 4, 8, 2, 128, (1 << 13) * 16, 1)
    assert need > 0
    for ws, n in ((None, need), (P, need - 1), (P + 8, need)):
        assert shared(ws=ws, ws_bytes=n) == capi.EWORKSPACE and "workspace" in capi.last_error()
    assert shared(n_seqs=0, n_groups=0) == capi.OK and shared(T=0) == capi.OK


def test_python_surface():
    import minfer.kernels.torch_ext  # noqa: F401
    from minfer.kernels import KernelBackend
    kerns = KernelBackend("torch_ext")
    for name in ("paged_tables", "paged_release", "verify_drafts", "flash_attn_paged_shared", "flash_attn_paged_shared_fp8"):
        assert callable(getattr(kerns, name)) and getattr(kerns, name).__doc__
        schema = str(getattr(torch.ops.minfer, name).default._schema)
        assert schema.startswith("minfer::" + name + "(") and schema.endswith("-> ()")
    # no CPU implementation
    i = torch.zeros(3, dtype=torch.int32)
    with pytest.raises(NotImplementedError):
        kerns.paged_tables(16, i[:2], i[:2], i[:2], i, i, i.view(1, 3)[:0], i, i[:2], i.long(), i[:2], i)
    with pytest.raises(NotImplementedError):
        kerns.verify_drafts(i, i, torch.zeros(3, 5), None, torch.zeros(3), torch.zeros(2), i, i[:2])


def test_fakes_check_what_the_operators_check():
    from torch._subclasses.fake_tensor import FakeTensorMode
    import minfer.kernels.torch_ext as ext
    with FakeTensorMode(allow_non_fake_inputs=True):
        dev = dict(device="cuda")
        i = lambda *s: torch.empty(*s, dtype=torch.int32, **dev)
        good = [16, i(4), i(4), i(4), i(9), i(3), i(4, 8), i(5), i(4), torch.empty(7, dtype=torch.int64, **dev), i(4), i(3)]
        ext.paged_tables(*good)
        with pytest.raises(RuntimeError):
            ext.paged_tables(*good[:9], i(7), *good[10:])
        probs, tok = torch.empty(7, 50, **dev), torch.empty(7, dtype=torch.int64, **dev)
        ext.verify_drafts(tok, i(4), probs, None, torch.empty(7, **dev), torch.empty(3, **dev), tok.clone(), i(3))
        with pytest.raises(RuntimeError):
            ext.verify_drafts(tok, i(4), probs, probs.half(), torch.empty(7, **dev), torch.empty(3, **dev), tok.clone(), i(3))
        q, pool = torch.empty(1, 8, 4, 64, dtype=torch.float16, **dev), torch.empty(6, 2, 16, 64, dtype=torch.float16, **dev)
        ext.flash_attn_paged_shared(1, 1, 2, q, pool, pool, i(4, 3), i(5), i(4), i(2), i(1), 1, q.clone())
        with pytest.raises(RuntimeError):
            ext.flash_attn_paged_shared(1, 1, 2, q, pool, pool, i(4, 3), i(5), i(4), i(3), i(1), 1, q.clone())


# ---- the definitions -------------------------------------------------------------------------------------------------------------
def test_tables_by_hand():
    # two sequences, pages of 16 rows: the first goes on in its page and needs one more, the second begins
    cu, ctx, slots, table, held, state = ref.tables(16, [15, 0], [3, 17], [1, 0], [6, 7, 3, 8, 9, 1, 2, 0, 3, 5], [9, 4, 0], [[4, -1, -1], [-1, -1, -1]], 20)
    assert cu == [0, 3, 20] and ctx == [18, 17] and held == [2, 2] and state == [2, 1, 0]
    assert table == [[4, 5, -1], [6, 7, -1]]
    assert slots == [4 * 16 + 15, 5 * 16, 5 * 16 + 1] + [6 * 16 + i for i in range(16)] + [7 * 16]


def test_release_by_hand():
    got, held, state = ref.release(16, [0, 20, 99], [3, 3, 1], [[4, -1, 2], [5, 6, 7], [0, -1, -1]], [9, 9, 9, 9, 9, 1, 9, 9, 3, 9], [7, 2, 0])
    assert held == [0, 2, 1] and state == [7, 5, 0]
    assert got == [2, 7, 9, 9, 9, 1, 9, 9, 3, 4]


def test_verify_keeps_the_targets_distribution():
    """Kept or drawn, the first token comes with the target's probabilities, whatever the drafter's are: counted over an even grid of random numbers."""
    p, q = torch.tensor([0.5, 0.25, 0.125, 0.125]), torch.tensor([0.125, 0.125, 0.5, 0.25])
    N = 64
    count = torch.zeros(4)
    for x in range(4):
        for u in range(N):
            for r in range(N):
                target = torch.stack((p, p))
                out, _ = ref.verify(torch.tensor([0, x]), [0, 2], target, torch.stack((q, q)), torch.tensor([(u + 0.5) / N, 0.0]), torch.tensor([(r + 0.5) / N]))
                count[out[0]] += float(q[x]) / (N * N)
    # a grid of N points meets each border (of the comparison and of the draw) within one cell, and there are at most four borders a token
    assert (count - p).abs().max() <= 4 / N
