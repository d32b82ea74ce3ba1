"""Python wrappers and fake (meta) kernels of the attention ops and of the rotary-embedding step
before them, mirroring the reference's wrapper layer (reference:
src/minfer/kernels/torch_ext/ops.py:60-266): positional pass-through
to ``torch.ops.minfer.<op>.default``; the result is written into ``out``."""
from typing import Optional

import torch

_ACT_DTYPES = (torch.float16, torch.bfloat16)
_Q8_0 = 8   # GGML type number of the one block format built here: 32 values in 34 bytes


def dequant(qtype: int, qblock_size: int, qtype_size: int, x: torch.Tensor, y: torch.Tensor):
    """Dequantises the rows of x (uint8 [M, N/32*34], Q8_0 blocks) into y (float32 or float16 [M, N]);
    qblock_size is the number of values per block, qtype_size its bytes (reference: ops.py:8-21)."""
    return torch.ops.minfer.dequant.default(qtype, qblock_size, qtype_size, x, y)


@torch.library.register_fake("minfer::dequant")
def _(qtype, qblock_size, qtype_size, x, y):
    torch._check(x.dtype == torch.uint8)
    torch._check(y.dtype in (torch.float32, torch.float16))
    torch._check(x.device == y.device)
    torch._check(x.device.type == "cuda")
    torch._check(x.size(0) == y.size(0))


def quant(qtype: int, qblock_size: int, qtype_size: int, x: torch.Tensor, y: torch.Tensor):
    """Quantises the rows of x (float32 [M, N]; float16/bfloat16 also taken) into y (uint8 [M, N/32*34], Q8_0
    blocks), on the device (reference: ops.py:33-46, CPU only there)."""
    return torch.ops.minfer.quant.default(qtype, qblock_size, qtype_size, x, y)


@torch.library.register_fake("minfer::quant")
def _(qtype, qblock_size, qtype_size, x, y):
    torch._check(x.dtype in (torch.float32, torch.float16, torch.bfloat16))
    torch._check(y.dtype == torch.uint8)
    torch._check(x.device == y.device)
    torch._check(x.device.type == "cuda")
    torch._check(x.size(0) == y.size(0))


def flash_attn(
    qtype_int: int,
    qblock_size: int,
    qtype_size: int,
    q: torch.Tensor,
    k: torch.Tensor,
    v: torch.Tensor,
    mask: torch.Tensor,
    out: torch.Tensor,
):
    """Fused GQA attention under a dense bool mask [B,1,L,L] (True = attend).
    q/out [B,n_heads,L,D], k/v [B,n_kv_heads,L,D], any strides with unit stride on D.  With (qtype_int, qblock_size,
    qtype_size) = (8, 32, 34), k and v are Q8_0 blocks, uint8 [B,n_kv_heads,L,D/32*34], and q/out float16."""
    return torch.ops.minfer.flash_attn.default(qtype_int, qblock_size, qtype_size, q, k, v, mask, out)


@torch.library.register_fake("minfer::flash_attn")
def _(qtype_int, qblock_size, qtype_size, q, k, v, mask, out):
    torch._check(q.dtype in _ACT_DTYPES)
    kv_dtype = torch.uint8 if qtype_int == _Q8_0 else q.dtype
    torch._check(k.dtype == kv_dtype and v.dtype == kv_dtype and out.dtype == q.dtype)
    torch._check(mask.dtype == torch.bool)
    torch._check(q.device == k.device == v.device == out.device)
    torch._check(q.device.type == "cuda")
    torch._check(q.dim() == 4 and k.dim() == 4 and v.dim() == 4 and mask.dim() == 4 and out.dim() == 4)


def flash_attn_decode(
    qtype_int: int,
    qblock_size: int,
    qtype_size: int,
    q: torch.Tensor,
    k_cache: torch.Tensor,
    v_cache: torch.Tensor,
    ctx_lens: torch.Tensor,
    out: torch.Tensor,
):
    """Single-token decode: q/out [B,n_heads,1,D] against caches [B,n_kv_heads,Lmax,D]; query b
    attends cache rows 0..ctx_lens[b]-1 (ctx_lens int32 [B]).  With (qtype_int, qblock_size, qtype_size) =
    (8, 32, 34) the caches are Q8_0 blocks, uint8 [B,n_kv_heads,Lmax,D/32*34], and q/out float16."""
    return torch.ops.minfer.flash_attn_decode.default(qtype_int, qblock_size, qtype_size, q, k_cache, v_cache, ctx_lens, out)


@torch.library.register_fake("minfer::flash_attn_decode")
def _(qtype_int, qblock_size, qtype_size, q, k_cache, v_cache, ctx_lens, out):
    torch._check(q.dtype in _ACT_DTYPES and out.dtype == q.dtype)
    cache_dtype = torch.uint8 if qtype_int == _Q8_0 else q.dtype
    torch._check(k_cache.dtype == cache_dtype and v_cache.dtype == cache_dtype)
    torch._check(ctx_lens.dtype == torch.int32)
    torch._check(q.device == k_cache.device == v_cache.device == ctx_lens.device == out.device)
    torch._check(q.device.type == "cuda")
    torch._check(q.dim() == 4 and k_cache.dim() == 4 and v_cache.dim() == 4 and out.dim() == 4 and ctx_lens.dim() == 1)


def flash_attn_varlen(
    qtype_int: int,
    qblock_size: int,
    qtype_size: int,
    q: torch.Tensor,
    k: torch.Tensor,
    v: torch.Tensor,
    cu_seqlens: torch.Tensor,
    max_seqlen: int,
    out: torch.Tensor,
):
    """Packed ragged causal prefill: q/out [1,n_heads,T,D], k/v [1,n_kv_heads,T,D], cu_seqlens
    int32 [n_seqs+1]; rows cu_seqlens[s]..cu_seqlens[s+1]-1 attend causally among themselves."""
    return torch.ops.minfer.flash_attn_varlen.default(qtype_int, qblock_size, qtype_size, q, k, v, cu_seqlens, max_seqlen, out)


@torch.library.register_fake("minfer::flash_attn_varlen")
def _(qtype_int, qblock_size, qtype_size, q, k, v, cu_seqlens, max_seqlen, out):
    torch._check(q.dtype in _ACT_DTYPES)
    kv_dtype = torch.uint8 if qtype_int == _Q8_0 else q.dtype
    torch._check(k.dtype == kv_dtype and v.dtype == kv_dtype and out.dtype == q.dtype)
    torch._check(cu_seqlens.dtype == torch.int32)
    torch._check(q.device == k.device == v.device == cu_seqlens.device == out.device)
    torch._check(q.device.type == "cuda")
    torch._check(q.dim() == 4 and k.dim() == 4 and v.dim() == 4 and out.dim() == 4 and cu_seqlens.dim() == 1)



def il_rope(rotary_dim: int, start_pos: int, freq_base: float, x: torch.Tensor):
    """Interleaved rotary embedding, in place; x [B,L,n_heads,head_dim], token l at position start_pos + l."""
    return torch.ops.minfer.il_rope.default(rotary_dim, start_pos, freq_base, x)


@torch.library.register_fake("minfer::il_rope")
def _(rotary_dim, start_pos, freq_base, x):
    torch._check(x.dtype in _ACT_DTYPES)
    torch._check(x.dim() == 4)
    torch._check(x.device.type == "cuda")
    torch._check(rotary_dim <= x.size(3))


def neox_rope(rotary_dim: int, start_pos: int, freq_base: float, x: torch.Tensor):
    """NeoX (two-halves) rotary embedding, in place; x [B,L,n_heads,head_dim]."""
    return torch.ops.minfer.neox_rope.default(rotary_dim, start_pos, freq_base, x)


@torch.library.register_fake("minfer::neox_rope")
def _(rotary_dim, start_pos, freq_base, x):
    torch._check(x.dtype in _ACT_DTYPES)
    torch._check(x.dim() == 4)
    torch._check(x.device.type == "cuda")
    torch._check(rotary_dim <= x.size(3))


def rope_kv_append(
    style: int,
    rotary_dim: int,
    freq_base: float,
    q: torch.Tensor,
    k: torch.Tensor,
    v: torch.Tensor,
    positions: torch.Tensor,
    k_cache: torch.Tensor,
    v_cache: torch.Tensor,
):
    """Rotates q [B,L,n_heads,D] in place, writes the rotated k [B,L,n_kv_heads,D] and v into rows
    positions[b] + l of the caches [B,n_kv_heads,Lmax,D]; style 0 = interleaved, 1 = NeoX; positions
    int32 [B].  uint8 caches [B,n_kv_heads,Lmax,D/32*34] receive the rows as Q8_0 blocks."""
    return torch.ops.minfer.rope_kv_append.default(style, rotary_dim, freq_base, q, k, v, positions, k_cache, v_cache)


@torch.library.register_fake("minfer::rope_kv_append")
def _(style, rotary_dim, freq_base, q, k, v, positions, k_cache, v_cache):
    torch._check(q.dtype in _ACT_DTYPES)
    torch._check(k.dtype == q.dtype and v.dtype == q.dtype)
    torch._check(k_cache.dtype in (q.dtype, torch.uint8) and v_cache.dtype == k_cache.dtype)
    torch._check(positions.dtype == torch.int32)
    torch._check(q.device.type == "cuda")
    torch._check(q.dim() == 4 and k.dim() == 4 and v.dim() == 4 and k_cache.dim() == 4 and v_cache.dim() == 4)
    torch._check(rotary_dim <= q.size(3))


def rope_kv_append_norm(
    style: int,
    rotary_dim: int,
    freq_base: float,
    eps: float,
    q: torch.Tensor,
    k: torch.Tensor,
    v: torch.Tensor,
    wq_norm: torch.Tensor,
    wk_norm: torch.Tensor,
    positions: torch.Tensor,
    k_cache: torch.Tensor,
    v_cache: torch.Tensor,
):
    """rope_kv_append with the per-head RMS normalisation of q (weight wq_norm [D]) and k (wk_norm [D]) in front of
    the rotation: equals rmsnorm(q), rmsnorm(k), rope_kv_append in one pass (the reference model's optional q/k norm)."""
    return torch.ops.minfer.rope_kv_append_norm.default(style, rotary_dim, freq_base, eps, q, k, v, wq_norm, wk_norm,
                                                        positions, k_cache, v_cache)


@torch.library.register_fake("minfer::rope_kv_append_norm")
def _(style, rotary_dim, freq_base, eps, q, k, v, wq_norm, wk_norm, positions, k_cache, v_cache):
    torch._check(q.dtype in _ACT_DTYPES)
    torch._check(k.dtype == q.dtype and v.dtype == q.dtype and wq_norm.dtype == q.dtype and wk_norm.dtype == q.dtype)
    torch._check(k_cache.dtype in (q.dtype, torch.uint8) and v_cache.dtype == k_cache.dtype)
    torch._check(positions.dtype == torch.int32)
    torch._check(q.device.type == "cuda")
    torch._check(q.dim() == 4 and k.dim() == 4 and v.dim() == 4 and k_cache.dim() == 4 and v_cache.dim() == 4)
    torch._check(wq_norm.dim() == 1 and wk_norm.dim() == 1)
    torch._check(rotary_dim <= q.size(3))


def _check_pages(q, k_pages, v_pages, scales, block_table, cu_seqlens, lens):
    page_dtype = q.dtype if scales is None else torch.float8_e4m3fn
    torch._check(q.dtype in _ACT_DTYPES)
    torch._check(k_pages.dtype == page_dtype and v_pages.dtype == page_dtype)
    torch._check(all(t.dtype == torch.int32 for t in (block_table, cu_seqlens, lens)))
    torch._check(all(t.device == q.device for t in (k_pages, v_pages, block_table, cu_seqlens, lens)))
    torch._check(q.device.type == "cuda")
    torch._check(q.dim() == 4 and k_pages.dim() == 4 and v_pages.dim() == 4 and block_table.dim() == 2)
    torch._check(cu_seqlens.dim() == 1 and lens.dim() == 1)
    if scales is not None:
        torch._check(all(t.dtype == torch.float8_e8m0fnu and t.dim() == 2 and t.device == q.device for t in scales))


def rope_kv_append_paged(
    style: int,
    rotary_dim: int,
    freq_base: float,
    q: torch.Tensor,
    k: torch.Tensor,
    v: torch.Tensor,
    cu_seqlens: torch.Tensor,
    positions: torch.Tensor,
    block_table: torch.Tensor,
    k_pages: torch.Tensor,
    v_pages: torch.Tensor,
):
    """rope_kv_append into a paged cache, for packed tokens: rotates q [1,T,n_heads,D] in place and writes the rotated
    k [1,T,n_kv_heads,D] and v into k_pages/v_pages [n_pages,n_kv_heads,page_size,D].  Tokens cu_seqlens[s] ..
    cu_seqlens[s+1]-1 are sequence s's rows positions[s], positions[s]+1, ..; row r lies in page block_table[s, r // page_size]
    at row r % page_size.  All index tensors int32 (cu_seqlens [n_seqs+1], positions [n_seqs], block_table [n_seqs, pages]).
    A table entry outside the pool (-1) means no page: its rows are not written.  page_size is a power of two in 16..1024.
    Sequences that end at or in front of their start have no tokens (so cu_seqlens may end in zeros or in T), and what lies
    outside [0, T) is cut off without moving the other tokens; they must not overlap."""
    return torch.ops.minfer.rope_kv_append_paged.default(style, rotary_dim, freq_base, q, k, v, cu_seqlens, positions,
                                                         block_table, k_pages, v_pages)


@torch.library.register_fake("minfer::rope_kv_append_paged")
def _(style, rotary_dim, freq_base, q, k, v, cu_seqlens, positions, block_table, k_pages, v_pages):
    _check_pages(q, k_pages, v_pages, None, block_table, cu_seqlens, positions)
    torch._check(k.dtype == q.dtype and v.dtype == q.dtype and k.dim() == 4 and v.dim() == 4)
    torch._check(rotary_dim <= q.size(3))


def rope_kv_append_paged_fp8(
    style: int,
    rotary_dim: int,
    freq_base: float,
    q: torch.Tensor,
    k: torch.Tensor,
    v: torch.Tensor,
    cu_seqlens: torch.Tensor,
    positions: torch.Tensor,
    block_table: torch.Tensor,
    k_pages: torch.Tensor,
    v_pages: torch.Tensor,
    k_scales: torch.Tensor,
    v_scales: torch.Tensor,
):
    """rope_kv_append_paged into 8-bit pages: float8_e4m3fn codes with a power of two as the scale of each page and head
    (float8_e8m0fnu [n_pages,n_kv_heads]), the smallest with which the page's rows fit.  A page that gets its row 0 starts
    with the scale its new rows need; in a page that goes on, the scale grows if they need it, and the codes that are there
    move to it.  A page that a call writes to belongs to one sequence of that call."""
    return torch.ops.minfer.rope_kv_append_paged_fp8.default(style, rotary_dim, freq_base, q, k, v, cu_seqlens, positions,
                                                             block_table, k_pages, v_pages, k_scales, v_scales)


@torch.library.register_fake("minfer::rope_kv_append_paged_fp8")
def _(style, rotary_dim, freq_base, q, k, v, cu_seqlens, positions, block_table, k_pages, v_pages, k_scales, v_scales):
    _check_pages(q, k_pages, v_pages, (k_scales, v_scales), block_table, cu_seqlens, positions)
    torch._check(k.dtype == q.dtype and v.dtype == q.dtype and k.dim() == 4 and v.dim() == 4)
    torch._check(rotary_dim <= q.size(3))


def flash_attn_paged(
    qtype_int: int,
    qblock_size: int,
    qtype_size: int,
    q: torch.Tensor,
    k_pages: torch.Tensor,
    v_pages: torch.Tensor,
    block_table: torch.Tensor,
    cu_seqlens: torch.Tensor,
    ctx_lens: torch.Tensor,
    max_q_len: int,
    out: torch.Tensor,
):
    """Attention of packed tokens over a paged cache that holds their own rows already (rope_kv_append_paged): q/out
    [1,n_heads,T,D]; tokens cu_seqlens[s] .. cu_seqlens[s+1]-1 are the last ones of sequence s, which has ctx_lens[s] rows, and
    each attends the rows up to its own.  One token per sequence is a decode step, a few are drafts, many a chunk of a
    prompt; a call may mix them.  Rows of pages that are not there (table entry -1) are not attended; a token without any
    row yields zeros.  max_q_len bounds the tokens of a sequence (0 = not known); tokens past it are not computed."""
    return torch.ops.minfer.flash_attn_paged.default(qtype_int, qblock_size, qtype_size, q, k_pages, v_pages, block_table,
                                                     cu_seqlens, ctx_lens, max_q_len, out)


@torch.library.register_fake("minfer::flash_attn_paged")
def _(qtype_int, qblock_size, qtype_size, q, k_pages, v_pages, block_table, cu_seqlens, ctx_lens, max_q_len, out):
    _check_pages(q, k_pages, v_pages, None, block_table, cu_seqlens, ctx_lens)
    torch._check(out.dtype == q.dtype and out.shape == q.shape)


def flash_attn_paged_fp8(
    qtype_int: int,
    qblock_size: int,
    qtype_size: int,
    q: torch.Tensor,
    k_pages: torch.Tensor,
    v_pages: torch.Tensor,
    k_scales: torch.Tensor,
    v_scales: torch.Tensor,
    block_table: torch.Tensor,
    cu_seqlens: torch.Tensor,
    ctx_lens: torch.Tensor,
    max_q_len: int,
    out: torch.Tensor,
):
    """flash_attn_paged over 8-bit pages (rope_kv_append_paged_fp8): a row is its float8_e4m3fn codes times the page's and
    head's scale (float8_e8m0fnu [n_pages,n_kv_heads]), a number that q's dtype holds."""
    return torch.ops.minfer.flash_attn_paged_fp8.default(qtype_int, qblock_size, qtype_size, q, k_pages, v_pages, k_scales,
                                                         v_scales, block_table, cu_seqlens, ctx_lens, max_q_len, out)


@torch.library.register_fake("minfer::flash_attn_paged_fp8")
def _(qtype_int, qblock_size, qtype_size, q, k_pages, v_pages, k_scales, v_scales, block_table, cu_seqlens, ctx_lens, max_q_len, out):
    _check_pages(q, k_pages, v_pages, (k_scales, v_scales), block_table, cu_seqlens, ctx_lens)
    torch._check(out.dtype == q.dtype and out.shape == q.shape)


def flash_attn_paged_shared(
    qtype_int: int,
    qblock_size: int,
    qtype_size: int,
    q: torch.Tensor,
    k_pages: torch.Tensor,
    v_pages: torch.Tensor,
    block_table: torch.Tensor,
    cu_seqlens: torch.Tensor,
    ctx_lens: torch.Tensor,
    cu_groups: torch.Tensor,
    prefix_lens: torch.Tensor,
    max_q_len: int,
    out: torch.Tensor,
):
    """flash_attn_paged where groups of sequences share their first rows, a prompt that a whole batch stands behind: sequences
    cu_groups[i] .. cu_groups[i+1]-1 name the same pages for their first prefix_lens[i] rows, which are then read once for the group
    instead of once for each of them; sequences in front of the first group and behind the last share nothing, one between two groups is a group with a prefix of 0.  The result is
    flash_attn_paged's up to the order of the sums.  cu_groups int32 [n_groups+1] and prefix_lens int32 [n_groups] on the device.  Meant for single
    tokens and drafts: max_q_len, the bound of a sequence's tokens, times the query heads of a KV head up to 64; above that it is flash_attn_paged."""
    return torch.ops.minfer.flash_attn_paged_shared.default(qtype_int, qblock_size, qtype_size, q, k_pages, v_pages,
                                           block_table, cu_seqlens, ctx_lens, cu_groups, prefix_lens, max_q_len, out)


@torch.library.register_fake("minfer::flash_attn_paged_shared")
def _(qtype_int, qblock_size, qtype_size, q, k_pages, v_pages, block_table, cu_seqlens, ctx_lens, cu_groups, prefix_lens, max_q_len, out):
    _check_pages(q, k_pages, v_pages, None, block_table, cu_seqlens, ctx_lens)
    torch._check(all(t.dtype == torch.int32 and t.dim() == 1 and t.device == q.device for t in (cu_groups, prefix_lens)))
    torch._check(cu_groups.size(0) == prefix_lens.size(0) + 1)
    torch._check(out.dtype == q.dtype and out.shape == q.shape)


def flash_attn_paged_shared_fp8(
    qtype_int: int,
    qblock_size: int,
    qtype_size: int,
    q: torch.Tensor,
    k_pages: torch.Tensor,
    v_pages: torch.Tensor,
    k_scales: torch.Tensor,
    v_scales: torch.Tensor,
    block_table: torch.Tensor,
    cu_seqlens: torch.Tensor,
    ctx_lens: torch.Tensor,
    cu_groups: torch.Tensor,
    prefix_lens: torch.Tensor,
    max_q_len: int,
    out: torch.Tensor,
):
    """flash_attn_paged_shared over 8-bit pages, as flash_attn_paged_fp8 takes them."""
    return torch.ops.minfer.flash_attn_paged_shared_fp8.default(qtype_int, qblock_size, qtype_size, q, k_pages, v_pages, k_scales, v_scales,
                                           block_table, cu_seqlens, ctx_lens, cu_groups, prefix_lens, max_q_len, out)


@torch.library.register_fake("minfer::flash_attn_paged_shared_fp8")
def _(qtype_int, qblock_size, qtype_size, q, k_pages, v_pages, k_scales, v_scales, block_table, cu_seqlens, ctx_lens, cu_groups, prefix_lens, max_q_len, out):
    _check_pages(q, k_pages, v_pages, (k_scales, v_scales), block_table, cu_seqlens, ctx_lens)
    torch._check(all(t.dtype == torch.int32 and t.dim() == 1 and t.device == q.device for t in (cu_groups, prefix_lens)))
    torch._check(cu_groups.size(0) == prefix_lens.size(0) + 1)
    torch._check(out.dtype == q.dtype and out.shape == q.shape)


_IDS = (torch.int32, torch.int64)


def paged_tables(
    page_size: int,
    past_lens: torch.Tensor,
    new_lens: torch.Tensor,
    pages_held: torch.Tensor,
    free_ring: torch.Tensor,
    ring_state: torch.Tensor,
    block_table: torch.Tensor,
    cu_seqlens: torch.Tensor,
    ctx_lens: torch.Tensor,
    slots: torch.Tensor,
    held_after: torch.Tensor,
    state_after: torch.Tensor,
):
    """The index tensors of a step over a paged cache, made on the device from lengths.  Sequence s holds past_lens[s] rows in
    the first pages_held[s] pages of block_table[s] and gets new_lens[s] rows; the pages that it lacks are taken from the pool's free ones
    and written behind those (-1 where there are no more).  free_ring [n_pages] holds them as a ring whose ring_state is {first entry, free
    pages, unused}.  Written: cu_seqlens [n_seqs+1] and ctx_lens [n_seqs] as the paged operators take them (their `positions`
    are past_lens), slots [T] int64 (the row of the pool of every new token, page * page_size + row, or -1), held_after [n_seqs]
    and state_after [3] = {first entry, free pages, pages that were lacking}; these two go into the next call, in place of
    pages_held and ring_state, which must be other tensors.  Rows that got no page are held nowhere, and the next past_lens must not count them.  slots may be
    empty.  All other tensors int32."""
    return torch.ops.minfer.paged_tables.default(page_size, past_lens, new_lens, pages_held, free_ring, ring_state, block_table, cu_seqlens,
                                                 ctx_lens, slots, held_after, state_after)


@torch.library.register_fake("minfer::paged_tables")
def _(page_size, past_lens, new_lens, pages_held, free_ring, ring_state, block_table, cu_seqlens, ctx_lens, slots, held_after, state_after):
    ints = (past_lens, new_lens, pages_held, free_ring, ring_state, block_table, cu_seqlens, ctx_lens, held_after, state_after)
    torch._check(all(t.dtype == torch.int32 for t in ints) and slots.dtype == torch.int64)
    torch._check(past_lens.device.type == "cuda" and all(t.device == past_lens.device for t in (*ints, slots)))
    torch._check(block_table.dim() == 2 and all(t.dim() == 1 for t in (*ints[:5], *ints[6:], slots)))


def paged_release(
    page_size: int,
    keep_lens: torch.Tensor,
    pages_held: torch.Tensor,
    block_table: torch.Tensor,
    free_ring: torch.Tensor,
    ring_state: torch.Tensor,
    held_after: torch.Tensor,
    state_after: torch.Tensor,
):
    """Gives pages back to the ring that paged_tables takes them from: sequence s keeps the pages of its first keep_lens[s] rows
    (0: it ended; a large number: all of them), and those behind, up to pages_held[s], are added to free_ring in the order of sequences and
    pages; entries that name no page (a window that moved on) are left out.  held_after and state_after as in paged_tables; the
    table itself is not written.  A page that sequences share must be kept by all of them but one.  All tensors int32."""
    return torch.ops.minfer.paged_release.default(page_size, keep_lens, pages_held, block_table, free_ring, ring_state, held_after, state_after)


@torch.library.register_fake("minfer::paged_release")
def _(page_size, keep_lens, pages_held, block_table, free_ring, ring_state, held_after, state_after):
    ints = (keep_lens, pages_held, block_table, free_ring, ring_state, held_after, state_after)
    torch._check(all(t.dtype == torch.int32 for t in ints))
    torch._check(keep_lens.device.type == "cuda" and all(t.device == keep_lens.device for t in ints))
    torch._check(block_table.dim() == 2)


def verify_drafts(
    tokens: torch.Tensor,
    cu_seqlens: torch.Tensor,
    target_probs: torch.Tensor,
    draft_probs: Optional[torch.Tensor],
    accept_u: torch.Tensor,
    sample_u: torch.Tensor,
    out_tokens: torch.Tensor,
    n_accepted: torch.Tensor,
):
    """Checks drafted tokens against the target's probabilities, so that what is kept or drawn is distributed as the target says.
    tokens [T] (int32 or int64) are a step's: of sequence s, cu_seqlens[s] .. cu_seqlens[s+1]-1, the first is known, the others drafts.
    target_probs [T, V] row t is the target's distribution behind token t, draft_probs row t the one that the draft behind it was drawn
    from (None: drafts without probabilities, from a look-up).  The draft x behind token t is kept while accept_u[t] *
    draft_probs[t, x] < target_probs[t, x]; the next token is drawn with sample_u[s] from max(target - draft, 0) of the first row whose
    draft is not kept, or from the last row's target.  out_tokens [T]: kept drafts, the next token, -1 behind it;
    n_accepted [n_seqs] int32: the drafts kept.  Random numbers are float32 in [0, 1)."""
    return torch.ops.minfer.verify_drafts.default(tokens, cu_seqlens, target_probs, draft_probs, accept_u, sample_u, out_tokens, n_accepted)


@torch.library.register_fake("minfer::verify_drafts")
def _(tokens, cu_seqlens, target_probs, draft_probs, accept_u, sample_u, out_tokens, n_accepted):
    torch._check(tokens.dtype in _IDS and out_tokens.dtype == tokens.dtype and out_tokens.shape == tokens.shape)
    torch._check(target_probs.dtype in (torch.float32, *_ACT_DTYPES) and target_probs.dim() == 2)
    torch._check(draft_probs is None or (draft_probs.dtype == target_probs.dtype and draft_probs.shape == target_probs.shape))
    torch._check(accept_u.dtype == torch.float32 and sample_u.dtype == torch.float32)
    torch._check(cu_seqlens.dtype == torch.int32 and n_accepted.dtype == torch.int32)
    torch._check(tokens.device.type == "cuda")


def rmsnorm(eps: float, input: torch.Tensor, w: torch.Tensor, out: torch.Tensor):
    """RMS normalisation over vectors of length len(w) (the whole hidden dimension, or per head)."""
    return torch.ops.minfer.rmsnorm.default(eps, input, w, out)


@torch.library.register_fake("minfer::rmsnorm")
def _(eps, input, w, out):
    torch._check(input.dtype in _ACT_DTYPES)
    torch._check(w.dtype == input.dtype and out.dtype == input.dtype)
    torch._check(input.device == w.device == out.device)
    torch._check(input.device.type == "cuda")
    torch._check(input.shape == out.shape)
    torch._check(input.dim() in (3, 4))
    torch._check(input.size(-1) == w.size(0) or input.size(-1) % w.size(0) == 0)


def gemm(qtype_int: int, qblock_size: int, qtype_size: int, alpha: float, beta: float,
         A: torch.Tensor, B: torch.Tensor, C: torch.Tensor, D: torch.Tensor):
    """D = alpha * A B + beta * C; A [B,L,in_dim], weight B [in_dim,out_dim] (or [out_dim,in_dim]: A B^T), C and D
    [B,L,out_dim].  With (qtype_int, qblock_size, qtype_size) = (8, 32, 34) the weight is uint8 [out_dim, in_dim/32*34],
    rows of Q8_0 blocks, and the product is A B^T over the dequantised weight."""
    return torch.ops.minfer.gemm.default(qtype_int, qblock_size, qtype_size, alpha, beta, A, B, C, D)


@torch.library.register_fake("minfer::gemm")
def _(qtype_int, qblock_size, qtype_size, alpha, beta, A, B, C, D):
    torch._check(A.dtype in _ACT_DTYPES)
    torch._check(C.dtype == A.dtype and D.dtype == A.dtype)
    torch._check(B.dtype == (torch.uint8 if qtype_int == 8 else A.dtype))
    torch._check(A.device == B.device == C.device == D.device)
    torch._check(A.device.type == "cuda")
    torch._check(A.dim() == 3 and B.dim() == 2 and C.dim() == 3 and D.dim() == 3)
    torch._check(A.size(0) * A.size(1) == C.size(0) * C.size(1))
    torch._check(B.size(-1) == C.size(-1) or B.size(0) == C.size(-1))
    torch._check(C.shape == D.shape)
    torch._check(alpha != 0.0)


def qkv(q_qtype_int: int, k_qtype_int: int, v_qtype_int: int, q_qblock_size: int, k_qblock_size: int, v_qblock_size: int,
        q_qtype_size: int, k_qtype_size: int, v_qtype_size: int,
        x: torch.Tensor, wq: torch.Tensor, wk: torch.Tensor, wv: torch.Tensor,
        q_out: torch.Tensor, k_out: torch.Tensor, v_out: torch.Tensor):
    """The three projections q_out = x wq^T, k_out = x wk^T, v_out = x wv^T; x [B,L,hidden], weights [out,hidden]; a
    weight whose type triple is (8, 32, 34) is uint8 [out, hidden/32*34], rows of Q8_0 blocks."""
    return torch.ops.minfer.qkv.default(q_qtype_int, k_qtype_int, v_qtype_int, q_qblock_size, k_qblock_size, v_qblock_size,
                                        q_qtype_size, k_qtype_size, v_qtype_size, x, wq, wk, wv, q_out, k_out, v_out)


@torch.library.register_fake("minfer::qkv")
def _(q_qtype_int, k_qtype_int, v_qtype_int, q_qblock_size, k_qblock_size, v_qblock_size, q_qtype_size, k_qtype_size,
      v_qtype_size, x, wq, wk, wv, q_out, k_out, v_out):
    torch._check(x.dtype in _ACT_DTYPES)
    torch._check(all(t.dtype == x.dtype for t in (q_out, k_out, v_out)))
    torch._check(all(w.dtype == (torch.uint8 if qt == 8 else x.dtype) for w, qt in ((wq, q_qtype_int), (wk, k_qtype_int), (wv, v_qtype_int))))
    torch._check(x.device == wq.device == wk.device == wv.device == q_out.device == k_out.device == v_out.device)
    torch._check(x.device.type == "cuda")
    torch._check(x.dim() == 3 and q_out.dim() == 3 and k_out.dim() == 3 and v_out.dim() == 3)
    torch._check(wq.dim() == 2 and wk.dim() == 2 and wv.dim() == 2)
