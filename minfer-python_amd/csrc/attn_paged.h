// What the operators over a paged KV cache share: the cache as the kernels see it, and the checks of its description.
//
// A cache is a pool of pages, [n_pages, Hkv, page_size, D] for k and for v, and a table of pages per sequence: row r of sequence s
// lies in page block_table[s, r / page_size] at row r % page_size.  The table is device data that nobody has checked: an entry
// outside [0, n_pages) means that the page is not there (never mapped, or given back by a window that moved on); its rows are
// not attended and not written, and no address is made from it.  Pages are whole in memory, so any row of one may be read,
// but rows that nothing was written to may hold anything, NaN included.
//
// 8-bit pages hold e4m3 codes (four significant bits, exponents from 2^-6 to 2^8, 448 the largest) and one scale for each page, KV head
// and tensor, a power of two kept as its biased exponent (E8M0).  A power of two, because a page fills token by token: when a
// later token needs a larger scale the codes that are there move to it by a change of their exponents, exact unless they
// fall below the smallest normal code, where any other factor would round each of them once more.  And it makes code * scale a
// number of the 16-bit types, so that attention over 8-bit pages is attention over 16-bit rows, nothing rounded in between.
#pragma once

#include "attn_common.h"
#include "attn_host.h"

namespace minfer_attn {

struct PagedCache {
    void* k; void* v;
    uint8_t* k_scales; uint8_t* v_scales;   // 8-bit pages: [n_pages][Hkv]
    const int32_t* table;
    int64_t page_stride, head_stride, row_stride, table_stride;   // elements (bytes where the pages are 8-bit)
    int n_pages, page_log2, width;          // pages in the pool, log2 of a page's rows, table entries per sequence
};

// Input that no kernel of the launch writes, as constant memory: a load at a wave-uniform address is then a scalar one, and waiting
// for it does not wait for the vector loads in flight.
template <class V> MA_DEV V const_load(const V* p) {
    typedef const __attribute__((address_space(4))) V* const_ptr;
    return *(const_ptr)(uintptr_t)p;
}

// The same of a byte, through the aligned word that holds it (scalar loads are of words; a word never lies in two memory pages, so that
// one which holds a byte of a tensor may be read).
MA_DEV uint32_t const_byte(const uint8_t* p) {
    const uintptr_t at = (uintptr_t)p;
    return (const_load((const uint32_t*)(at & ~(uintptr_t)3)) >> (8 * (at & 3))) & 255u;
}

// Where a sequence's tokens of this call are, whatever cu_seqlens holds: those of lo .. hi - 1 that lie in [0, T), a start and a length.  What is
// cut off moves no other token: the first one's position is (lo cut) - lo further on, the last one's `behind` in front of the context's end.
struct TokenRange { int lo, len, behind; };
MA_DEV TokenRange token_range(int lo, int hi, int T) {
    lo = min(max(lo, 0), T);
    return TokenRange{lo, min(max(hi, lo), T) - lo, max(hi, T) - T};
}

// Rows of a sequence up to its last token that is there: ctx_lens' entry, cut to the table, without the rows of tokens behind T.
MA_DEV int context_of(const PagedCache& c, int ctx, const TokenRange& t) { return max(min(max(ctx, 0), c.width << c.page_log2) - t.behind, 0); }

// 2^(bits - 127) for a scale's byte; 255 is no number.  (2^-127 is a subnormal fp32.)
MA_DEV float scale_value(uint32_t bits) {
    return __builtin_bit_cast(float, bits == 0u ? 0x00400000u : bits == 255u ? 0x7fc00000u : bits << 23);
}

// Two e4m3 codes (the word's upper two with HI) times a scale as a pair of 16-bit values, one instruction: rounded once where the type cannot
// hold the product, which it can unless that is beyond its range; 2^-127 and NaN are scales like any other (checked for
// every code and scale).
template <class T, bool HI> MA_DEV uint32_t widen2(uint32_t codes, float scale) {
    if constexpr (std::is_same_v<T, F16>) return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(codes, scale, HI));
    else return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(codes, scale, HI));
}
MA_DEV void lds_write_b128(uint32_t addr, int imm, s16x8 x) {
    typedef __attribute__((address_space(3))) s16x8 lds_s16x8;
    *(lds_s16x8*)(uintptr_t)(addr + imm) = x;
}

// Four values of a cached row, from element `at` of a pool on.
template <class T, bool FP8> MA_DEV f32x4 row_values(const void* pool, int64_t at, uint32_t scale) {
    uint32_t lo, hi;
    if constexpr (FP8) {
        const uint32_t codes = *reinterpret_cast<const uint32_t*>((const char*)pool + at);
        lo = widen2<T, false>(codes, scale_value(scale));
        hi = widen2<T, true>(codes, scale_value(scale));
    } else {
        const uint2 x = *reinterpret_cast<const uint2*>((const short*)pool + at);
        lo = x.x; hi = x.y;
    }
    return f32x4{T::to_float((short)(lo & 0xffffu)), T::to_float((short)(lo >> 16)), T::to_float((short)(hi & 0xffffu)), T::to_float((short)(hi >> 16))};
}

// Keys first .. end - 1 of a sequence for NQ columns of a wave, key by key and without matrix products, in which a V row with an infinity or a NaN would
// meet the weights of zero of columns that do not attend it: for the few keys from the first such row on that some columns attend and others do not.
// Lane (l16, quad) holds column l16's O at d = 16db + 4 quad + 0..3 (o(db, i) of column i), its reference m (log2 units) and a
// share l of its sum; q[i] is its query row (null: no column), limit[i] the rows that it attends.  The test in front of it costs 0 to 2 % (prompt of 8192 f16 508 to
// 519 us, four drafts 27.7 to 28.2); a cache all of NaN makes three times the time of that prompt and twice that of the drafts.
template <class T, int D, bool FP8, int NQ, class Acc>
MA_DEV void attend_key_by_key(const PagedCache& c, int Hkv, int seq, int g, int first, int end, const short* const (&q)[NQ], const int (&limit)[NQ], float c2,
                              Acc o, float (&m)[NQ], float (&l)[NQ]) {
    const int quad = (threadIdx.x & 63) >> 4;
#pragma unroll 1
    for (int key = first; key < end; ++key) {
        const int id = const_load(c.table + (int64_t)seq * c.table_stride + min(key >> c.page_log2, c.width - 1));
        if ((unsigned)id >= (unsigned)c.n_pages) continue;
        const int64_t at = (int64_t)id * c.page_stride + (int64_t)g * c.head_stride + (int64_t)(key & ((1 << c.page_log2) - 1)) * c.row_stride + 4 * quad;
        const uint32_t ks = FP8 ? const_byte(c.k_scales + (int64_t)id * Hkv + g) : 0u, vs = FP8 ? const_byte(c.v_scales + (int64_t)id * Hkv + g) : 0u;
#pragma unroll
        for (int i = 0; i < NQ; ++i) {
            float score = 0.f;
#pragma unroll 1
            for (int d = 0; d < D; d += 16) {
                const f32x4 x = row_values<T, FP8>(c.k, at + d, ks), y = q[i] ? row_values<T, false>(q[i], 4 * quad + d, 0u) : f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int e = 0; e < 4; ++e) score = fmaf(x[e], y[e], score);
            }
            score = sum_across_quads(score) * c2;
            const bool on = q[i] && key < limit[i];
            const float m_new = on ? fmaxf(m[i], score) : m[i], base = m_new == -INFINITY ? 0.f : m_new;
            const float alpha = m[i] == -INFINITY ? (on ? 0.f : 1.f) : fast_exp2(m[i] - base);
            // (the weight as a product with V has it in front of these keys: rounded to the 16-bit type)
            const float w = T::to_float((short)(T::pack2(fast_exp2(score - base), 0.f) & 0xffffu));
            m[i] = m_new;
            l[i] = on ? l[i] * alpha + (quad == 0 ? w : 0.f) : l[i];
#pragma unroll
            for (int db = 0; db < D / 16; ++db) {
                const f32x4 x = row_values<T, FP8>(c.v, at + 16 * db, vs);
#pragma unroll
                for (int e = 0; e < 4; ++e) o(db, i)[e] = on ? fmaf(w, x[e], o(db, i)[e] * alpha) : o(db, i)[e];
            }
        }
    }
}

// Checks of a cache's description, for an operator called `op`; fills `c`.
inline int check_pages(const char* op, int dtype, int page_type, const minfer_kv_pages* pages, int64_t n_seqs, int64_t Hkv, int64_t D, PagedCache& c) {
    char msg[256];
    auto bad = [&](const char* what) { snprintf(msg, sizeof msg, "%s: %s", op, what); return fail(MINFER_ATTN_EINVAL, msg); };
    const bool eight = page_type == MINFER_FP8_E4M3;
    if (dtype != MINFER_ATTN_F16 && dtype != MINFER_ATTN_BF16) return bad("dtype must be MINFER_ATTN_F16 or MINFER_ATTN_BF16");
    if (!eight && page_type != dtype) return bad("page_type must be the activations' dtype or MINFER_FP8_E4M3");
    if (D != 64 && D != 128) return bad("head_dim must be 64 or 128");
    if (Hkv <= 0 || Hkv > 65535) return bad("n_kv_heads must be in 1..65535");
    if (!pages) return bad("pages is null");
    if (pages->page_size < 16 || pages->page_size > 1024 || (pages->page_size & (pages->page_size - 1)) != 0)
        return bad("page_size must be a power of two in 16..1024");
    if (pages->n_pages < 0 || pages->n_pages > 0x7fffffffLL || pages->pages_per_seq < 0) return bad("bad number of pages");
    const int64_t most = ((int64_t)1 << 30) / pages->page_size;   // (the products themselves need not fit 64 bits)
    if (pages->pages_per_seq > most) return bad("pages_per_seq * page_size > 2^30 unsupported");
    if (pages->table_stride < 0) return bad("table_stride must be non-negative");
    if (n_seqs > 0 && pages->pages_per_seq > 0 && !pages->block_table) return bad("block_table is null");
    if (pages->n_pages > 0) {
        if (!pages->k || !pages->v) return bad("k and v pages must be non-null");
        if (!aligned16(pages->k) || !aligned16(pages->v)) return bad("pages must be 16-byte aligned");
        if (eight && (!pages->k_scales || !pages->v_scales)) return bad("8-bit pages need k_scales and v_scales");
    }
    const int64_t unit = eight ? 16 : 8, s[3] = {pages->stride_page, pages->stride_head, pages->stride_row};
    for (int i = 0; i < 3; ++i)
        if (s[i] < 0 || s[i] % unit != 0) return bad(eight ? "page strides must be non-negative multiples of 16 bytes" : "page strides must be non-negative multiples of 8 elements");
    // (a lane's offset from a page's first row is 32 bits)
    if (pages->stride_row >= most) return bad("page_size * stride_row >= 2^30 unsupported");
    c.k = pages->k; c.v = pages->v;
    c.k_scales = (uint8_t*)pages->k_scales; c.v_scales = (uint8_t*)pages->v_scales;
    c.table = pages->block_table;
    c.page_stride = pages->stride_page; c.head_stride = pages->stride_head; c.row_stride = pages->stride_row;
    c.table_stride = pages->table_stride;
    c.n_pages = (int)pages->n_pages;
    c.page_log2 = __builtin_ctzll((unsigned long long)pages->page_size);
    c.width = (int)(pages->n_pages > 0 ? pages->pages_per_seq : 0);   // a pool without pages: nothing to attend or write, no table to read
    return MINFER_ATTN_OK;
}

// One call of the attention over a paged cache, as its kernels see it.
struct PagedParams {
    PagedCache c;
    const void* q; void* out;
    const int32_t* cu; const int32_t* ctx;
    float* part_o;     // partial results, un-normalised: decode [part][column][D], tiles [piece][KV head][row of the block][D] ...
    float* part_ml;    // ... with their reference (log2 units) and sum
    int64_t q1, q2, o1, o2;
    int n_seqs, T, Hq, Hkv, n_rep;
    int max_q;         // tokens of a sequence past this many are not computed
    int round;         // tiles: workgroups per KV head that the chip holds at once, which blocks of rows are cut up to fill; 0: none is cut
    int32_t* table;    // tiles: the number of pieces, and from the fourth entry on (sequence, block, part, parts) of each
    float scale_log2, inv_scale_log2;  // softmax scale * log2(e), and one over it
};

// Few query rows per KV head (csrc/attn_paged_decode.hip): whether a call with these sizes is one, its workspace, its launch.
bool paged_decode_takes(int64_t Hq, int64_t Hkv, int64_t max_q);
size_t paged_decode_workspace_bytes(int64_t n_seqs, int64_t Hq, int64_t Hkv, int64_t D, int64_t max_context, int64_t max_q);
int launch_paged_decode(PagedParams p, int dtype, int64_t D, bool eight, int64_t max_context, void* workspace, hipStream_t stream);

}  // namespace minfer_attn
