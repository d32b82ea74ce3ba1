// The streaming of cached rows through a wave, for few query rows per KV head over a paged cache for gfx950: the part that the attention of single tokens and
// drafts and that of groups which share a prefix have in common.
//
// A wave streams rows of one (sequence, KV head) on its own, with a ring of groups of rows in registers: 16 rows of 16-bit values,
// loaded as whole rows and turned into matrix operands in the wave's LDS; or 32 rows of e4m3 codes, K loaded straight in the
// operand's layout (the order of the contraction is free as long as q is loaded in the same) or as whole rows, V as whole rows, both widened on the way.
// A page holds at least 16 rows, so a group (or half of one) lies in one page, whose table entry is read as a scalar a group ahead.
// S^T[keys x 16 columns] = K Q^T, softmax per column with a lazy reference, O^T += V^T P^T.
#pragma once

#include "attn_paged.h"

namespace minfer_attn {

constexpr int kLineWaves = 4;          // waves per workgroup of the line
// Least rows of a wave's share of the line (us, 128 / 64 / 32, 32 heads on 8 of 128: 80 sequences of 6 to 100 21.2 / 16.3 / 13.9, of codes 17.1 / 13.2 / 12.9; 80 of
// 100 16.8 / 16.8 / 16.1; 4 heads on 1: 80 of up to 2000 15.8 / 14.8 / 17.5, one of 4000 with 69 of 6 22.6 / 19.3 / 19.3; where every wave has more nothing changes).
constexpr int kLeastShare = 64;
constexpr int kMaxParts = 64;          // partial results a column can have: a wave merges them, one to a lane

struct DecodeWork {
    PagedParams p;
    int32_t* seq_off;   // line: [n_seqs + 2] start of every sequence on the line, its length, the quota; written by workgroup 0
    int n_col;          // columns per KV head: max_q * n_rep
    int n_hg;           // groups of <= 16 columns per KV head
    int per_part;       // columns of a partial result: those of a group
    int n_wg;           // line: workgroups
    uint32_t* done;     // chunks: zeroed counters, one per pair, left zero; or null
};

template <bool FP8> constexpr int kRows = FP8 ? 32 : 16;   // rows of a group

// What a wave has to know about a sequence.
struct SeqInfo { int lo, len, ctx; };   // its first token, its number of tokens, the rows up to its last token
MA_DEV SeqInfo seq_info(const PagedParams& p, int s) {
    const TokenRange r = token_range(const_load(p.cu + s), const_load(p.cu + s + 1), p.T);
    return SeqInfo{r.lo, r.len, context_of(p.c, const_load(p.ctx + s), r)};
}

template <int D> struct ColumnAcc {
    f32x4 o[D / 16];   // lane (l16, quad): column l16, O at d = 16db + 4 quad + 0..3, un-normalised
    float m, l;        // the column's reference (log2 units) and sum
};

template <int D> struct DecodeGeom {
    static constexpr int RB = D * 2;
    static constexpr int G = RB / 16;
    static constexpr int RPI = 1024 / RB;              // 16-bit rows that one wave-wide load covers
    static constexpr int NI = 16 / RPI;                // such loads per 16 rows
    static constexpr int RPI8 = 1024 / D;              // the same for rows of codes
    static constexpr int NI8 = 16 / RPI8;
    static MA_DEV int swz_v(int row) { return D == 128 ? ((row & 7) << 1) : (((row >> 1) & 3) << 1); }
    static MA_DEV int swz_c(int row) { return D == 128 ? (row & 7) : ((row >> 1) & 3); }   // of codes
    static MA_DEV int swz_k(int row) { return D == 128 ? (row & 15) : ((row >> 1) & 7); }
};
template <int D, bool FP8> constexpr int kWaveLds = FP8 ? 32 * D * 2 : 2 * 16 * D * 2;   // V of 32 rows; or K and V of 16

// The columns of a group: what lane l16 needs of its own.
struct Column { const short* q; int limit; };   // its query row (null: no column), and the rows that it attends: 0 .. limit - 1
MA_DEV Column column_of(const DecodeWork& w, const SeqInfo& info, int g, int hg, int l16) {
    const PagedParams& p = w.p;
    const int col = hg * 16 + l16, tok = p.n_rep > 16 || p.max_q == 1 ? 0 : col / p.n_rep;
    Column c{nullptr, 0};
    if (col < w.n_col && tok < info.len) {
        c.q = (const short*)p.q + (int64_t)(info.lo + tok) * p.q2 + (int64_t)(g * p.n_rep + col - tok * p.n_rep) * p.q1;
        c.limit = info.ctx - info.len + tok + 1;
    }
    return c;
}

// Streams groups g0 .. g1 - 1 (at least one) of (sequence s, KV head g) for the columns of NC groups from hg on; `area` is the wave's own LDS.
// NS: groups on their way.  Three where nothing else runs; beside others' products two end sooner by up to 5 % (seven groups of sequences, 16-bit / codes, at head_dim 128 98 / 73 us with three,
// 97 / 71 with two, 99 / 76 with four; at 64 54 / 46, 51 / 44, 54 / 48).
// WHOLE_K: K's codes are loaded as whole rows as well and turned in the LDS.  Straight in the operand's layout a load's neighbouring lanes read 16 bytes of different rows, which the
// unit's address path takes in pieces: no matter where the memory bounds all units together (64 sequences to 8192 rows 100.8 us straight, 101.4 whole), but with a few
// units streaming beside others' products it does (attn_shared.hip, 192 sequences behind 16000 to 24000 rows 196 / 178; at head_dim 64, whose rows are 64 bytes, 129 / 132).
template <class T, int D, bool FP8, int NC, int NS, bool WHOLE_K>
MA_DEV void stream_columns(const DecodeWork& work, int s, const SeqInfo& info, int g, int hg, int g0, const int g1, char* area, ColumnAcc<D> (&acc)[NC]) {
    const PagedParams& p = work.p;
    using GEO = DecodeGeom<D>;
    constexpr int RB = GEO::RB, G = GEO::G, RPI = GEO::RPI, NI = GEO::NI, RPI8 = GEO::RPI8, NI8 = GEO::NI8;
    constexpr int KC = D / 32, DB = D / 16, GR = kRows<FP8>, NH = GR / 16;   // halves of 16 rows in a group
    const int lane = threadIdx.x & 63, l16 = lane & 15, quad = lane >> 4;
    const int ctx = info.ctx, page_mask = (1 << p.c.page_log2) - 1;
    const int32_t* const table = p.c.table + (int64_t)s * p.c.table_stride;
    Column col[NC];
#pragma unroll
    for (int n = 0; n < NC; ++n) col[n] = column_of(work, info, g, hg + n, l16);
    const int edge = ctx - info.len + 1;   // from this row on some columns attend what others do not
    int by_key = 0x7fffffff;               // the group from which on keys are taken one by one

    // Q^T fragments (B operand): column l16; contraction step c takes d = 32c + 8 quad + 0..7, or for codes, whose 16-byte pieces hold
    // two steps, d = 64 (c / 2) + 16 quad + 8 (c % 2) + 0..7
    s16x8 qf[NC][KC];
#pragma unroll
    for (int n = 0; n < NC; ++n)
#pragma unroll
        for (int c = 0; c < KC; ++c) {
            const int d = FP8 ? 64 * (c / 2) + 16 * quad + 8 * (c % 2) : 32 * c + 8 * quad;
            qf[n][c] = s16x8{0, 0, 0, 0, 0, 0, 0, 0};
            if (col[n].q) qf[n][c] = *reinterpret_cast<const s16x8*>(col[n].q + d);
        }

    // ---- pages ----
    struct Ids { int id[NH]; };
    auto ids_of = [&](int t) __attribute__((always_inline)) {
        Ids r;
#pragma unroll
        for (int h = 0; h < NH; ++h) r.id[h] = const_load(table + min((min(t, g1 - 1) * GR + 16 * h) >> p.c.page_log2, p.c.width - 1));
        return r;
    };
    auto is_there = [&](int id) __attribute__((always_inline)) { return (unsigned)id < (unsigned)p.c.n_pages; };
    const int64_t head_at = (int64_t)g * p.c.head_stride;
    auto half_at = [&](int id, int row) __attribute__((always_inline)) -> int64_t {
        return (int64_t)(is_there(id) ? id : 0) * p.c.page_stride + head_at + (int64_t)(row & page_mask) * p.c.row_stride;
    };

    // ---- a ring of groups on their way ----
    constexpr int NK = FP8 ? NH * D / 64 : NI, NV = FP8 ? NH * NI8 : NI;
    // (scales as the words that hold their bytes: to take them out is to wait for them.  there: bit h half h's page is, above bit 8 which bytes)
    struct Stage { u32x4 k[NK], v[NV]; uint32_t ks[NH], vs[NH]; int there; } ring[NS];
    // a lane's place inside the 16 rows: its row and chunk of load j, and its key's pieces of K's codes
    const int stride = (int)p.c.row_stride;
    constexpr int VPI = FP8 ? RPI8 : RPI, CPR = 64 / VPI;   // rows a load covers, 16-byte pieces per row
    const int v_row = lane / CPR, v_piece = (FP8 ? 16 : 8) * (lane % CPR), k_piece = 16 * quad;
    auto load_group = [&](int t, const Ids& ids, Stage& st) __attribute__((always_inline)) {
        // slots past the last group have every row of theirs be one row of that group, which costs a few cache lines
        const bool real = t < g1;
        const int step = real ? stride : 0, t_row = min(t, g1 - 1) * GR;
        st.there = 0;
#pragma unroll
        for (int h = 0; h < NH; ++h) {
            const int row0 = t_row + 16 * h, id = ids.id[h];
            st.there |= (is_there(id) && row0 < ctx) ? 1 << h : 0;
            const int64_t at = half_at(id, row0);
            if constexpr (FP8) {
                const char* kb = (const char*)p.c.k + at;
                const char* vb = (const char*)p.c.v + at;
#pragma unroll
                for (int j = 0; j < NI8; ++j)
                    st.k[h * NI8 + j] = stream_load(reinterpret_cast<const u32x4*>(kb + (uint32_t)(WHOLE_K ? (j * RPI8 + v_row) * step + v_piece : l16 * step + k_piece + 64 * j)));
#pragma unroll
                for (int j = 0; j < NI8; ++j) st.v[h * NI8 + j] = stream_load(reinterpret_cast<const u32x4*>(vb + (uint32_t)((j * RPI8 + v_row) * step + v_piece)));
                const int64_t sc = (int64_t)(is_there(id) ? id : 0) * p.Hkv + g;
                const uintptr_t ka = (uintptr_t)(p.c.k_scales + sc), va = (uintptr_t)(p.c.v_scales + sc);
                st.ks[h] = const_load((const uint32_t*)(ka & ~(uintptr_t)3));
                st.vs[h] = const_load((const uint32_t*)(va & ~(uintptr_t)3));
                st.there |= ((int)(ka & 3) | (int)(va & 3) << 2) << (8 + 4 * h);
            } else {
                const short* kb = (const short*)p.c.k + at;
                const short* vb = (const short*)p.c.v + at;
#pragma unroll
                for (int j = 0; j < NI; ++j) st.k[j] = stream_load(reinterpret_cast<const u32x4*>(kb + (uint32_t)((j * RPI + v_row) * step + v_piece)));
#pragma unroll
                for (int j = 0; j < NI; ++j) st.v[j] = stream_load(reinterpret_cast<const u32x4*>(vb + (uint32_t)((j * RPI + v_row) * step + v_piece)));
            }
        }
    };

    float m_ref[NC], l_sum[NC];
#pragma unroll
    for (int n = 0; n < NC; ++n) {
#pragma unroll
        for (int db = 0; db < DB; ++db) acc[n].o[db] = f32x4{0.f, 0.f, 0.f, 0.f};
        m_ref[n] = -INFINITY;
        l_sum[n] = 0.f;
    }
    const float c2 = p.scale_log2;
    constexpr float kLazyLog2 = 6.f;
    char* const my_v = area;
    char* const my_k = area + 16 * RB;   // 16-bit rows only

    auto consume = [&](int t, Stage& st) __attribute__((always_inline)) {
        int ln = threadIdx.x & 63;
        if ((FP8 || NC > 1) && D == 128) asm volatile("" : "+v"(ln));   // (places in LDS are worked out for every group: kept, they do not fit the registers of codes or of two columns a lane)
        const int lane = ln, l16 = ln & 15, quad = ln >> 4;
        f32x4 sc[NC][NH];
        // V rows behind the context may hold anything, NaN too, and their weight of zero would not take it out of the sums (of K only the
        // row's own scores are made, which are replaced)
        const int past = ctx - t * GR;
        if (past < GR) {
#pragma unroll
            for (int j = 0; j < NV; ++j) st.v[j] = j * VPI + v_row < past ? st.v[j] : u32x4{0u, 0u, 0u, 0u};
        }
        if constexpr (FP8) {
            static_assert(D / 64 == NI8, "as many loads either way");
            if (WHOLE_K) {   // (through the place where V's values go behind them)
#pragma unroll
                for (int i = 0; i < NK; ++i) {
                    const int row = i * RPI8 + lane / (D / 16);
                    *reinterpret_cast<u32x4*>(my_v + row * D + 16 * ((lane % (D / 16)) ^ GEO::swz_c(row))) = st.k[i];
                }
#pragma unroll
                for (int h = 0; h < NH; ++h)
#pragma unroll
                    for (int j = 0; j < NI8; ++j) st.k[h * NI8 + j] = *reinterpret_cast<const u32x4*>(my_v + (16 * h + l16) * D + 16 * ((4 * j + quad) ^ GEO::swz_c(l16)));
            }
#pragma unroll
            for (int h = 0; h < NH; ++h) {
#pragma unroll
                for (int n = 0; n < NC; ++n) sc[n][h] = f32x4{0.f, 0.f, 0.f, 0.f};
                const float ks = scale_value(st.ks[h] >> 8 * (st.there >> (8 + 4 * h) & 3) & 255u);
#pragma unroll
                for (int c = 0; c < KC; ++c) {
                    const u32x4 x = st.k[h * NI8 + c / 2];
                    const uint32_t lo = x[2 * (c % 2)], hi = x[2 * (c % 2) + 1];
                    const u32x4 a = {widen2<T, false>(lo, ks), widen2<T, true>(lo, ks), widen2<T, false>(hi, ks), widen2<T, true>(hi, ks)};
#pragma unroll
                    for (int n = 0; n < NC; ++n) sc[n][h] = T::mfma16(__builtin_bit_cast(s16x8, a), qf[n][c], sc[n][h]);
                }
            }
#pragma unroll
            for (int h = 0; h < NH; ++h) {
                const bool on = (st.there >> h & 1) != 0;   // (a page that is not there: what was loaded in its place is not multiplied)
                const float vs = on ? scale_value(st.vs[h] >> 8 * (st.there >> (10 + 4 * h) & 3) & 255u) : 1.f;
#pragma unroll
                for (int j = 0; j < NI8; ++j) {
                    const int row = 16 * h + j * RPI8 + lane / (D / 16), gr = 2 * (lane % (D / 16));
                    const u32x4 x = on ? st.v[h * NI8 + j] : u32x4{0u, 0u, 0u, 0u};
                    char* rowp = my_v + row * RB;
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        const u32x4 a = {widen2<T, false>(x[2 * i], vs), widen2<T, true>(x[2 * i], vs), widen2<T, false>(x[2 * i + 1], vs), widen2<T, true>(x[2 * i + 1], vs)};
                        *reinterpret_cast<u32x4*>(rowp + 16 * ((gr + i) ^ GEO::swz_v(row))) = a;
                    }
                }
            }
        } else {
#pragma unroll
            for (int j = 0; j < NI; ++j) {
                const int row = j * RPI + lane / G;
                *reinterpret_cast<u32x4*>(my_k + row * RB + 16 * ((lane % G) ^ GEO::swz_k(row))) = st.k[j];
            }
            const char* rowp = my_k + l16 * RB;
            const int sw = GEO::swz_k(l16);
#pragma unroll
            for (int n = 0; n < NC; ++n) sc[n][0] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int c = 0; c < KC; ++c) {
                const s16x8 a = *reinterpret_cast<const s16x8*>(rowp + 16 * ((4 * c + quad) ^ sw));
#pragma unroll
                for (int n = 0; n < NC; ++n) sc[n][0] = T::mfma16(a, qf[n][c], sc[n][0]);
            }
#pragma unroll
            for (int j = 0; j < NI; ++j) {
                const int row = j * RPI + lane / G;
                *reinterpret_cast<u32x4*>(my_v + row * RB + 16 * ((lane % G) ^ GEO::swz_v(row))) = st.v[j];
            }
        }
        const int row = 4 * quad + (l16 >> 2);
        const char* rowp_v = my_v + row * RB;
        const int sw_v = GEO::swz_v(row);   // rows 16 apart share a swizzle
        if (edge < min(t * GR + GR, ctx)) {
            // V rows that some columns attend and others do not: whether all are finite is what products with zero say
            f32x4 probe = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int db = 0; db < DB; ++db) {
                const int dcol = 16 * db + 4 * (l16 & 3), at = 16 * ((dcol >> 3) ^ sw_v) + 2 * (dcol & 7);
#pragma unroll
                for (int h = 0; h < NH; ++h) probe = T::mfma16k16(lds_read_tr16(rowp_v + 16 * h * RB + at), s16x4{0, 0, 0, 0}, probe);
            }
            if (__any(!(probe[0] + probe[1] + probe[2] + probe[3] == 0.f))) { by_key = t; return; }
        }
        uint32_t pk[NC][2 * NH];
#pragma unroll
        for (int n = 0; n < NC; ++n) {
            f32x4 (&x)[NH] = sc[n];
            // rows that the column does not attend
#pragma unroll
            for (int h = 0; h < NH; ++h) {
                const int left = (NH == 1 || (st.there >> h & 1)) ? col[n].limit - (t * GR + 16 * h + 4 * quad) : 0;
#pragma unroll
                for (int r = 0; r < 4; ++r) x[h][r] = r < left ? x[h][r] : -INFINITY;
            }
            float mx = fmaxf(fmaxf(x[0][0], x[0][1]), fmaxf(x[0][2], x[0][3]));
            if (NH == 2) mx = fmaxf(mx, fmaxf(fmaxf(x[NH - 1][0], x[NH - 1][1]), fmaxf(x[NH - 1][2], x[NH - 1][3])));
            auto grows = [&](float y) { return (y * c2 - m_ref[n]) > kLazyLog2 || (m_ref[n] == -INFINITY && y > -INFINITY); };
            if (__any(grows(mx))) {   // (one of the column's four lanes holds its largest score)
                mx = max_across_quads(mx);
                const float m_new = grows(mx) ? mx * c2 : m_ref[n];
                const float alpha = (m_ref[n] == -INFINITY) ? 0.f : fast_exp2(m_ref[n] - m_new);
                m_ref[n] = m_new;
                l_sum[n] *= alpha;
#pragma unroll
                for (int db = 0; db < DB; ++db) acc[n].o[db] *= alpha;
            }
            const float mc = (m_ref[n] == -INFINITY) ? 0.f : m_ref[n];
#pragma unroll
            for (int h = 0; h < NH; ++h) {
                pk[n][2 * h] = T::pack2(fast_exp2(fmaf(x[h][0], c2, -mc)), fast_exp2(fmaf(x[h][1], c2, -mc)));
                pk[n][2 * h + 1] = T::pack2(fast_exp2(fmaf(x[h][2], c2, -mc)), fast_exp2(fmaf(x[h][3], c2, -mc)));
                l_sum[n] = T::add_pair(pk[n][2 * h + 1], T::add_pair(pk[n][2 * h], l_sum[n]));   // sums the rounded weights that are multiplied (as in paged_tile_kernel)
            }
        }
        // O^T += V^T P^T: row d = 16db + l16, keys 4 quad + 0..3 (and 16 + 4 quad + 0..3)
#pragma unroll
        for (int db = 0; db < DB; ++db) {
            const int dcol = 16 * db + 4 * (l16 & 3), at = 16 * ((dcol >> 3) ^ sw_v) + 2 * (dcol & 7);
            const s16x4 a0 = lds_read_tr16(rowp_v + at);
            if constexpr (NH == 2) {
                const s16x4 a1 = lds_read_tr16(rowp_v + 16 * RB + at);
#pragma unroll
                for (int n = 0; n < NC; ++n)
                    acc[n].o[db] = T::mfma16(s16x8{a0[0], a0[1], a0[2], a0[3], a1[0], a1[1], a1[2], a1[3]},
                                             __builtin_bit_cast(s16x8, u32x4{pk[n][0], pk[n][1], pk[n][2 * NH - 2], pk[n][2 * NH - 1]}), acc[n].o[db]);
            } else {
#pragma unroll
                for (int n = 0; n < NC; ++n) {
                    uint2 pu; pu.x = pk[n][0]; pu.y = pk[n][1];
                    acc[n].o[db] = T::mfma16k16(a0, __builtin_bit_cast(s16x4, pu), acc[n].o[db]);
                }
            }
        }
    };

#pragma unroll
    for (int n = 0; n < NC; ++n) {
        acc[n].m = -INFINITY;
        acc[n].l = 0.f;
    }
    Ids first[NS + 1];   // requested together: one wait
#pragma unroll
    for (int i = 0; i <= NS; ++i) first[i] = ids_of(g0 + i);
    bool any = false;
#pragma unroll
    for (int h = 0; h < NH; ++h) any = any || is_there(first[0].id[h]);
    if (!any) {   // pages given back by a window that moved on: on to the first group that is there, 64 at a time (64 sequences to 8192 rows 183 us, the first half of them gone 116)
        int at = g1;
        for (int base = g0; base < g1; base += 64) {
            const Ids mine = ids_of(base + lane);
            bool on = false;
#pragma unroll
            for (int h = 0; h < NH; ++h) on = on || is_there(mine.id[h]);
            const uint64_t hit = __ballot(on && base + lane < g1);
            if (hit) { at = base + __builtin_amdgcn_readfirstlane(__ffsll((unsigned long long)hit) - 1); break; }
        }
        if (at >= g1) return;
        g0 = __builtin_amdgcn_readfirstlane(at);
#pragma unroll
        for (int i = 0; i <= NS; ++i) first[i] = ids_of(g0 + i);
    }
#pragma unroll
    for (int i = 0; i < NS; ++i) load_group(g0 + i, first[i], ring[i]);
    Ids next = first[NS];
    // the last round requests nothing: what a workgroup's barrier, or the next pair, would wait for (3 x 200 to 3000 rows of codes 11.9 us / 10.4, 64 x 50 to 300
    // 18.3 / 15.4, 64 x 512 to 8192 182.6 / 181.4)
    int t0 = g0;
    for (; t0 + NS < g1; t0 += NS) {
#pragma unroll
        for (int i = 0; i < NS; ++i) {
            if ((ring[i].there & 3) && t0 + i < by_key) consume(t0 + i, ring[i]);
            const Ids now = next;
            next = ids_of(t0 + i + NS + 1);
            load_group(t0 + i + NS, now, ring[i]);
        }
    }
#pragma unroll
    for (int i = 0; i < NS; ++i)
        if (t0 + i < g1 && (ring[i].there & 3) && t0 + i < by_key) consume(t0 + i, ring[i]);
    if (by_key < g1) {
        int l = l16;   // (worked out again: kept over the loop, the column's query row does not fit the registers of codes at D = 128)
        asm volatile("" : "+v"(l));
        const short* q[NC];
        int limit[NC];
#pragma unroll
        for (int n = 0; n < NC; ++n) {
            const Column again = column_of(work, info, g, hg + n, l);
            q[n] = again.q;
            limit[n] = again.limit;
        }
        attend_key_by_key<T, D, FP8, NC>(p.c, p.Hkv, s, g, by_key * GR, min(g1 * GR, ctx), q, limit, c2,
                                         [&](int db, int n) __attribute__((always_inline)) -> f32x4& { return acc[n].o[db]; }, m_ref, l_sum);
    }
#pragma unroll
    for (int n = 0; n < NC; ++n) {
        acc[n].m = m_ref[n];
        acc[n].l = sum_across_quads(l_sum[n]);
    }
}
// One group of columns.
template <class T, int D, bool FP8>
MA_DEV void stream_pages(const DecodeWork& work, int s, const SeqInfo& info, int g, int hg, int g0, const int g1, char* area, ColumnAcc<D>& acc) {
    stream_columns<T, D, FP8, 1, 3, false>(work, s, info, g, hg, g0, g1, area, reinterpret_cast<ColumnAcc<D> (&)[1]>(acc));
}

// Where column c of a column group's partial result `part` lies.  Partial results are numbered through the launch, those of a (sequence, KV head,
// column group) one after the other: there is room for as many as there can be of all of them together, not for the most that each could have
// (which for 256 sequences of 64 heads was 0.5 GiB, now 16 MiB; 4096 of 32 4 GiB, now 69 MiB).
MA_DEV int64_t part_row(const DecodeWork& w, int64_t part, int c) { return part * w.per_part + c; }

// A wave's partial result of every column of group hg, into the workspace, `first` columns behind the partial result's first.
template <int D> MA_DEV void store_part(const DecodeWork& w, int hg, int64_t part, const ColumnAcc<D>& acc, int first = 0) {
    const int lane = threadIdx.x & 63, l16 = lane & 15, quad = lane >> 4;
    if (hg * 16 + l16 >= w.n_col) return;
    const int64_t at = part_row(w, part, first + l16);
    float* dst = w.p.part_o + at * D + 4 * quad;
#pragma unroll
    for (int db = 0; db < D / 16; ++db) *reinterpret_cast<f32x4*>(dst + 16 * db) = acc.o[db];
    if (quad == 0) { w.p.part_ml[at * 2] = acc.m; w.p.part_ml[at * 2 + 1] = acc.l; }
}

// ---- the line ------------------------------------------------------------------------------------------------------
// Lengths in groups: every sequence's (zero without tokens) times its pairs, one after the other.  The quota: an equal share for
// every wave, kLeastShare rows at least, and as much as leaves no pair with more partial results than a merge takes.  Along the line either the share's
// number or the pair's, or both, go up by one from one partial result to the next: their sum numbers the partial results.
struct LineSeq { SeqInfo info; int groups; };
template <int GR> MA_DEV LineSeq line_seq(const DecodeWork& w, int s) {   // (per lane)
    const PagedParams& p = w.p;
    LineSeq r{{0, 0, 0}, 0};
    if (s < p.n_seqs) {
        const TokenRange t = token_range(p.cu[s], p.cu[s + 1], p.T);
        r.info = SeqInfo{t.lo, t.len, context_of(p.c, p.ctx[s], t)};
        r.groups = t.len > 0 ? (r.info.ctx + GR - 1) / GR : 0;
    }
    return r;
}

// Weights of a column's partial results, lane i holding part i's reference and sum (-inf and 0 in lanes without): w_i = 2^(m_i - max m), and the sum of
// l_i w_i.  A part whose scores are all NaN has a weight of zero and sums of NaN and is multiplied like any other.
struct PartWeights { float w, top, total; };
MA_DEV PartWeights part_weights(float m, float l) {
    PartWeights r;
    r.top = wave_max(m);
    r.w = m > -INFINITY ? fast_exp2(m - r.top) : 0.f;
    r.total = lane_sum<64>(l * r.w);
    return r;
}

}  // namespace minfer_attn
