"""Host side of the operators over a paged cache, without a GPU: what they refuse (nothing is launched: the pointers are made up),
their workspace sizes, their place in the Python surface, and the definitions that the GPU tests compare with."""
import ctypes

import pytest
import torch

import capi
import capi_paged as cp
import paged_ref as ref

P = 0x10000   # a made-up, 16-byte aligned address


def pages(**kw):
    d = dict(k=P, v=P, k_scales=P, v_scales=P, n_pages=8, page_size=16, stride_page=2 * 16 * 128, stride_head=16 * 128, stride_row=128,
             block_table=P, table_stride=4, pages_per_seq=4)
    d.update(kw)
    return cp.KvPages(**d)


def attend(dtype=capi.F16, page_type=None, pg=None, q=P, cu=P, ctx=P, out=P, n_seqs=2, T=2, Hq=8, Hkv=2, D=128, max_q=1, st=None, ws=P, ws_bytes=1 << 30):
    st = st or capi.Strides(0, 128, 1024, 0, 0, 0, 0, 128, 1024)
    pg = pages() if pg is None else pg
    return cp.lib().minfer_flash_attn_paged(dtype, dtype if page_type is None else page_type, q, ctypes.byref(pg) if pg else None, cu, ctx, out,
                                            n_seqs, T, Hq, Hkv, D, max_q, ctypes.byref(st), ws, ws_bytes, None)


def append(dtype=capi.F16, style=1, page_type=None, pg=None, q=P, k=P, v=P, cu=P, pos=P, n_seqs=2, T=2, Hq=8, Hkv=2, D=128, rd=128, base=1e4):
    pg = pages() if pg is None else pg
    return cp.lib().minfer_rope_kv_append_paged(dtype, style, dtype if page_type is None else page_type, q, k, v, cu, pos, ctypes.byref(pg) if pg else None,
                                                n_seqs, T, Hq, Hkv, D, rd, base, None)


BAD_PAGES = [("page_size", dict(page_size=8)), ("page_size", dict(page_size=48)), ("page_size", dict(page_size=2048)),
             ("number of pages", dict(n_pages=-1)), ("number of pages", dict(n_pages=1 << 31)), ("number of pages", dict(pages_per_seq=-1)),
             ("2^30", dict(pages_per_seq=(1 << 26) + 1)), ("table_stride", dict(table_stride=-1)), ("block_table is null", dict(block_table=None)),
             ("non-null", dict(k=None)), ("non-null", dict(v=None)), ("aligned", dict(k=P + 8)), ("aligned", dict(v=P + 2)),
             ("strides", dict(stride_page=-8)), ("strides", dict(stride_head=2044)), ("strides", dict(stride_row=132)),
             ("2^30", dict(stride_row=1 << 27))]


@pytest.mark.parametrize("text,change", BAD_PAGES)
def test_bad_pages_are_refused(text, change):
    for call in (attend, append):
        assert call(pg=pages(**change)) == capi.EINVAL
        assert text in capi.last_error()
    if text == "strides":
        return
    eight = {k: v for k, v in change.items()}
    for call in (attend, append):
        assert call(page_type=cp.FP8_E4M3, pg=pages(**eight)) == capi.EINVAL


def test_bad_8_bit_pages_are_refused():
    for change, text in ((dict(k_scales=None), "k_scales"), (dict(v_scales=None), "k_scales"), (dict(stride_row=136), "16 bytes"), (dict(stride_head=2056), "16 bytes")):
        for call in (attend, append):
            assert call(page_type=cp.FP8_E4M3, pg=pages(**change)) == capi.EINVAL
            assert text in capi.last_error()


def test_overlapping_pages_are_refused_by_the_append_only():
    for change in (dict(stride_page=0), dict(stride_head=0), dict(stride_row=120), dict(stride_row=0)):
        assert append(pg=pages(**change)) == capi.EINVAL
        assert "overlap" in capi.last_error()


@pytest.mark.parametrize("text,change", [
    ("dtype", dict(dtype=capi.F32)), ("page_type", dict(page_type=capi.BF16)), ("page_type", dict(page_type=capi.Q8_0)), ("head_dim", dict(D=96)), ("head_dim", dict(D=256)),
    ("n_kv_heads", dict(Hkv=0)), ("multiple", dict(Hq=7)), ("multiple", dict(Hq=0)), ("n_heads > 65535", dict(Hq=131072)), ("negative", dict(n_seqs=-1)), ("negative", dict(T=-1)),
    ("negative", dict(max_q=-1)), ("non-null", dict(q=None)), ("non-null", dict(cu=None)), ("non-null", dict(ctx=None)), ("non-null", dict(out=None)),
    ("aligned", dict(q=P + 4)), ("aligned", dict(out=P + 8)), ("strides", dict(st=capi.Strides(0, 4, 1024, 0, 0, 0, 0, 128, 1024))),
    ("strides", dict(st=capi.Strides(0, 128, 1024, 0, 0, 0, 0, 128, -8))), ("too large", dict(T=1 << 31, max_q=0)), ("too large", dict(T=1 << 29, Hq=64, Hkv=2))])
def test_attend_refusals(text, change):
    assert attend(**change) == capi.EINVAL
    assert text in capi.last_error()


def test_attend_null_pages_and_workspace():
    st = capi.Strides(0, 128, 1024, 0, 0, 0, 0, 128, 1024)
    assert cp.lib().minfer_flash_attn_paged(1, 1, P, None, P, P, P, 1, 1, 8, 2, 128, 1, ctypes.byref(st), P, 1 << 30, None) == capi.EINVAL
    assert "pages is null" in capi.last_error()
    pg = pages(pages_per_seq=1024, table_stride=1024)
    need = cp.lib().minfer_flash_attn_paged_workspace_bytes(2, 2, 8, 2, 128, 1024 * 16, 1)
    assert need > 0
    for ws, n in ((None, need), (P, need - 1), (P + 8, need)):
        assert attend(pg=pg, ws=ws, ws_bytes=n) == capi.EWORKSPACE
        assert "workspace" in capi.last_error()


@pytest.mark.parametrize("text,change", [
    ("dtype", dict(dtype=capi.F32)), ("page_type", dict(page_type=capi.BF16)), ("style", dict(style=2)), ("rotary_dim", dict(rd=130)), ("even", dict(rd=7)),
    ("multiple", dict(rd=8)), ("multiple", dict(style=0, rd=12)), ("freq_base", dict(base=0.0)), ("negative", dict(T=-1)), ("sequences", dict(n_seqs=-1)),
    ("null", dict(q=None)), ("null", dict(k=None)), ("null", dict(v=None)), ("null", dict(cu=None)), ("null", dict(pos=None)), ("aligned", dict(k=P + 4)),
    ("head_dim", dict(D=96, rd=64)), ("n_kv_heads", dict(Hkv=0))])
def test_append_refusals(text, change):
    for page_type in ((None,) if "page_type" in change or "dtype" in change else (None, cp.FP8_E4M3)):
        kw = dict(change)
        kw.setdefault("page_type", page_type)
        assert append(**kw) == capi.EINVAL
        assert text in capi.last_error()


def test_empty_calls_launch_nothing():
    assert attend(n_seqs=0) == capi.OK and attend(T=0) == capi.OK
    assert append(n_seqs=0) == capi.OK and append(T=0) == capi.OK


def test_workspace_sizes():
    w = cp.lib().minfer_flash_attn_paged_workspace_bytes
    for bad in ((0, 1, 8, 2, 128, 1024, 1), (1, 0, 8, 2, 128, 1024, 1), (1, 1, 7, 2, 128, 1024, 1)):
        assert w(*bad) == 0
    # many long prompts need none; single tokens of a long context do, and no more than 64 parts of a row each
    assert w(16, 16 * 4096, 32, 8, 128, 4096, 4096) == 0
    assert 0 < w(4, 4, 32, 8, 128, 1 << 17, 1) <= 4 * 32 * 64 * (128 + 2) * 4 + 4096


def test_python_surface():
    import minfer.kernels.torch_ext  # noqa: F401
    from minfer.kernels import KernelBackend
    kerns = KernelBackend("torch_ext")
    for name in ("rope_kv_append_paged", "rope_kv_append_paged_fp8", "flash_attn_paged", "flash_attn_paged_fp8"):
        assert callable(getattr(kerns, name))
        schema = str(getattr(torch.ops.minfer, name).default._schema)
        assert schema.startswith("minfer::" + name + "(int ") and schema.endswith("-> ()")
    # no CPU implementation
    q = torch.zeros(1, 2, 4, 64, dtype=torch.float16)
    k = torch.zeros(1, 2, 2, 64, dtype=torch.float16)
    pool = torch.zeros(3, 2, 16, 64, dtype=torch.float16)
    i = torch.zeros(2, dtype=torch.int32)
    with pytest.raises(NotImplementedError):
        kerns.rope_kv_append_paged(1, 64, 1e4, q, k, k, i, i[:1], i.view(1, 2), pool, pool)
    with pytest.raises(NotImplementedError):
        kerns.flash_attn_paged(1, 1, 2, q.transpose(1, 2), pool, pool, i.view(1, 2), i, i[:1], 1, q.transpose(1, 2))


# ---- the definitions -------------------------------------------------------------------------------------------------------------
def test_e4m3_rounding_is_torchs():
    x = torch.cat([torch.linspace(-448, 448, 40001), torch.randn(20000) * torch.exp2(torch.randint(-14, 8, (20000,)).float())]).double().clamp(-448, 448)
    assert torch.equal(ref.e4m3(x).float(), x.float().to(torch.float8_e4m3fn).float())


def test_needed_exponent():
    for e in (-20, -3, 0, 5):
        assert ref.needed_exponent(torch.tensor([448.0 * 2.0 ** e], dtype=torch.float64), 119) == e
        assert ref.needed_exponent(torch.tensor([-448.0 * 2.0 ** e * (1 + 1e-9)], dtype=torch.float64), 119) == e + 1
        assert ref.needed_exponent(torch.tensor([225.0 * 2.0 ** e], dtype=torch.float64), 119) == e
        assert ref.needed_exponent(torch.tensor([224.0 * 2.0 ** e], dtype=torch.float64), 119) == e - 1
    assert ref.needed_exponent(torch.zeros(3, dtype=torch.float64), 7) == -100
    assert ref.needed_exponent(torch.tensor([65504.0, float("inf")], dtype=torch.float64), 7) == 7


def test_attend_definition_against_torch():
    c = ref.Paged([(3, 20), (0, 4), (40, 0), (1, 0)], 16, 2, 64, torch.float32, "cpu")
    q = torch.randn(4, c.T, 64)
    out, _ = ref.attend(c, q)
    for s, (n, past) in enumerate(c.seqs):
        if n:
            lo = c.cu_list[s]
            mask = torch.arange(n + past)[None, :] <= past + torch.arange(n)[:, None]
            y = torch.nn.functional.scaled_dot_product_attention(q[:, lo:lo + n].double()[None], c.k_dense[s].repeat_interleave(2, 0)[None],
                                                                 c.v_dense[s].repeat_interleave(2, 0)[None], attn_mask=mask)
            assert torch.allclose(out[:, lo:lo + n], y[0], atol=1e-12)
