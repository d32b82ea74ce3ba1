// Attention of few query rows per KV head over a paged cache for gfx950: single tokens of many sequences, drafts of a few tokens.
//
// HBM-bound: each cached row is used by at most 16 columns (a token and head each) at a time, so what counts is bytes in flight.  The columns of a
// KV head are its group's query heads for every new token of the sequence, token by token; up to 16 of them are the columns of one
// 16-wide matrix product, each with a limit of its own (the row of its token), so a few drafts read the cache once.
//
// A wave streams rows of one (sequence, KV head) on its own, with a ring of groups of rows in registers: 16 rows of 16-bit values,
// loaded as whole rows and turned into matrix operands in the wave's LDS; or 32 rows of e4m3 codes, K loaded straight in the
// operand's layout (the order of the contraction is free as long as q is loaded in the same), V as whole rows, both widened on the way.
// A page holds at least 16 rows, so a group (or half of one) lies in one page, whose table entry is read as a scalar a group ahead.
// S^T[keys x 16 columns] = K Q^T, softmax per column with a lazy reference, O^T += V^T P^T.
//
// Two ways to share the work out:
// * the line: all rows to be read, sequence by sequence, KV head by KV head, cut into as many equal shares as the launch has waves; a
//   wave's share covers parts of a few (sequence, KV head) pairs, each of which leaves a partial result that
//   paged_merge_kernel puts together.  Whatever the mix of contexts, all waves end together.  64 sequences of 512 to 8192 rows, 32 query
//   heads on 8 of 128: 179 us, 6.1 TB/s, of which the merge 5; over codes 98 us, 5.6 TB/s.
// * chunks, for few pairs: eight waves of a workgroup share one chunk of a pair and merge in LDS, and the last workgroup of a pair merges its
//   chunks (on the null stream; elsewhere paged_chunk_merge_kernel does).  A sequence is cut by its own context, which the host does not know.
//   12 sequences of 3 or 4 drafts, 28964 rows: 27 us, 4.4 TB/s; one token, 8 heads on 2 of 64, against 1501 rows 8 us, three against 5570 rows of
//   codes 10 us, which is latency: a launch, two dependent loads of tables, the first rows, the merge in LDS.
#include <algorithm>
#include <atomic>

#include "attn_paged.h"

namespace minfer_attn {

constexpr int kLineWaves = 4;          // waves per workgroup of the line
constexpr int kLineWgPerCu = 2;
constexpr int kChunkWaves = 8;
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

// Streams groups g0 .. g1 - 1 (at least one) of (sequence s, KV head g) for the columns of group hg; `area` is the wave's own LDS.
template <class T, int D, bool FP8>
MA_DEV void stream_pages(const DecodeWork& work, int s, const SeqInfo& info, int g, int hg, int g0, const int g1, char* area, ColumnAcc<D>& acc) {
    const PagedParams& p = work.p;
    using GEO = DecodeGeom<D>;
    constexpr int RB = GEO::RB, G = GEO::G, RPI = GEO::RPI, NI = GEO::NI, RPI8 = GEO::RPI8, NI8 = GEO::NI8;
    constexpr int KC = D / 32, DB = D / 16, GR = kRows<FP8>, NH = GR / 16;   // halves of 16 rows in a group
    constexpr int NS = 3;
    const int lane = threadIdx.x & 63, l16 = lane & 15, quad = lane >> 4;
    const int ctx = info.ctx, page_mask = (1 << p.c.page_log2) - 1;
    const int32_t* const table = p.c.table + (int64_t)s * p.c.table_stride;
    const Column col = column_of(work, info, g, hg, l16);
    const int edge = ctx - info.len + 1;   // from this row on some columns attend what others do not
    int by_key = 0x7fffffff;               // the group from which on keys are taken one by one

    // Q^T fragments (B operand): column l16; contraction step c takes d = 32c + 8 quad + 0..7, or for codes, whose 16-byte pieces hold
    // two steps, d = 64 (c / 2) + 16 quad + 8 (c % 2) + 0..7
    s16x8 qf[KC];
#pragma unroll
    for (int c = 0; c < KC; ++c) {
        const int d = FP8 ? 64 * (c / 2) + 16 * quad + 8 * (c % 2) : 32 * c + 8 * quad;
        qf[c] = s16x8{0, 0, 0, 0, 0, 0, 0, 0};
        if (col.q) qf[c] = *reinterpret_cast<const s16x8*>(col.q + d);
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
                for (int j = 0; j < D / 64; ++j) st.k[h * (D / 64) + j] = stream_load(reinterpret_cast<const u32x4*>(kb + (uint32_t)(l16 * step + k_piece + 64 * j)));
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

    f32x4 (&o_acc)[DB] = acc.o;
#pragma unroll
    for (int db = 0; db < DB; ++db) o_acc[db] = f32x4{0.f, 0.f, 0.f, 0.f};
    float m_ref = -INFINITY, l_sum = 0.f;
    const float c2 = p.scale_log2;
    constexpr float kLazyLog2 = 6.f;
    char* const my_v = area;
    char* const my_k = area + 16 * RB;   // 16-bit rows only

    auto consume = [&](int t, Stage& st) __attribute__((always_inline)) {
        int ln = threadIdx.x & 63;
        if (FP8 && D == 128) asm volatile("" : "+v"(ln));   // (places in LDS are worked out for every group: kept, they do not fit the registers of codes)
        const int lane = ln, l16 = ln & 15, quad = ln >> 4;
        f32x4 sc[NH];
        // V rows behind the context may hold anything, NaN too, and their weight of zero would not take it out of the sums (of K only the
        // row's own scores are made, which are replaced)
        const int past = ctx - t * GR;
        if (past < GR) {
#pragma unroll
            for (int j = 0; j < NV; ++j) st.v[j] = j * VPI + v_row < past ? st.v[j] : u32x4{0u, 0u, 0u, 0u};
        }
        if constexpr (FP8) {
#pragma unroll
            for (int h = 0; h < NH; ++h) {
                sc[h] = f32x4{0.f, 0.f, 0.f, 0.f};
                const float ks = scale_value(st.ks[h] >> 8 * (st.there >> (8 + 4 * h) & 3) & 255u);
#pragma unroll
                for (int c = 0; c < KC; ++c) {
                    const u32x4 x = st.k[h * (D / 64) + c / 2];
                    const uint32_t lo = x[2 * (c % 2)], hi = x[2 * (c % 2) + 1];
                    const u32x4 a = {widen2<T, false>(lo, ks), widen2<T, true>(lo, ks), widen2<T, false>(hi, ks), widen2<T, true>(hi, ks)};
                    sc[h] = T::mfma16(__builtin_bit_cast(s16x8, a), qf[c], sc[h]);
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
            sc[0] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int c = 0; c < KC; ++c) sc[0] = T::mfma16(*reinterpret_cast<const s16x8*>(rowp + 16 * ((4 * c + quad) ^ sw)), qf[c], sc[0]);
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
        // rows that the column does not attend
#pragma unroll
        for (int h = 0; h < NH; ++h) {
            const int left = (NH == 1 || (st.there >> h & 1)) ? col.limit - (t * GR + 16 * h + 4 * quad) : 0;
#pragma unroll
            for (int r = 0; r < 4; ++r) sc[h][r] = r < left ? sc[h][r] : -INFINITY;
        }
        float mx = fmaxf(fmaxf(sc[0][0], sc[0][1]), fmaxf(sc[0][2], sc[0][3]));
        if (NH == 2) mx = fmaxf(mx, fmaxf(fmaxf(sc[NH - 1][0], sc[NH - 1][1]), fmaxf(sc[NH - 1][2], sc[NH - 1][3])));
        auto grows = [&](float x) { return (x * c2 - m_ref) > kLazyLog2 || (m_ref == -INFINITY && x > -INFINITY); };
        if (__any(grows(mx))) {   // (one of the column's four lanes holds its largest score)
            mx = max_across_quads(mx);
            const float m_new = grows(mx) ? mx * c2 : m_ref;
            const float alpha = (m_ref == -INFINITY) ? 0.f : fast_exp2(m_ref - m_new);
            m_ref = m_new;
            l_sum *= alpha;
#pragma unroll
            for (int db = 0; db < DB; ++db) o_acc[db] *= alpha;
        }
        const float mc = (m_ref == -INFINITY) ? 0.f : m_ref;
        uint32_t pk[2 * NH];
#pragma unroll
        for (int h = 0; h < NH; ++h) {
            pk[2 * h] = T::pack2(fast_exp2(fmaf(sc[h][0], c2, -mc)), fast_exp2(fmaf(sc[h][1], c2, -mc)));
            pk[2 * h + 1] = T::pack2(fast_exp2(fmaf(sc[h][2], c2, -mc)), fast_exp2(fmaf(sc[h][3], c2, -mc)));
            l_sum = T::add_pair(pk[2 * h + 1], T::add_pair(pk[2 * h], l_sum));   // sums the rounded weights that are multiplied (as in paged_tile_kernel)
        }
        // O^T += V^T P^T: row d = 16db + l16, keys 4 quad + 0..3 (and 16 + 4 quad + 0..3)
#pragma unroll
        for (int db = 0; db < DB; ++db) {
            const int dcol = 16 * db + 4 * (l16 & 3), at = 16 * ((dcol >> 3) ^ sw_v) + 2 * (dcol & 7);
            const s16x4 a0 = lds_read_tr16(rowp_v + at);
            if constexpr (NH == 2) {
                const s16x4 a1 = lds_read_tr16(rowp_v + 16 * RB + at);
                o_acc[db] = T::mfma16(s16x8{a0[0], a0[1], a0[2], a0[3], a1[0], a1[1], a1[2], a1[3]},
                                      __builtin_bit_cast(s16x8, u32x4{pk[0], pk[1], pk[2 * NH - 2], pk[2 * NH - 1]}), o_acc[db]);
            } else {
                uint2 pu; pu.x = pk[0]; pu.y = pk[1];
                o_acc[db] = T::mfma16k16(a0, __builtin_bit_cast(s16x4, pu), o_acc[db]);
            }
        }
    };

    acc.m = -INFINITY;
    acc.l = 0.f;
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
        const Column again = column_of(work, info, g, hg, l);
        const short* const q[1] = {again.q};
        const int limit[1] = {again.limit};
        float m[1] = {m_ref}, sum[1] = {l_sum};
        attend_key_by_key<T, D, FP8, 1>(p.c, p.Hkv, s, g, by_key * GR, min(g1 * GR, ctx), q, limit, c2,
                                        [&](int db, int) __attribute__((always_inline)) -> f32x4& { return o_acc[db]; }, m, sum);
        m_ref = m[0];
        l_sum = sum[0];
    }
    acc.m = m_ref;
    acc.l = sum_across_quads(l_sum);
}

// Where column c of a column group's partial result `part` lies.  Partial results are numbered through the launch, those of a (sequence, KV head,
// column group) one after the other: there is room for as many as there can be of all of them together, not for the most that each could have
// (which for 256 sequences of 64 heads was 0.5 GiB, now 16 MiB; 4096 of 32 4 GiB, now 69 MiB).
MA_DEV int64_t part_row(const DecodeWork& w, int64_t part, int c) { return part * w.per_part + c; }

// A wave's partial result of every column, into the workspace.
template <int D> MA_DEV void store_part(const DecodeWork& w, int hg, int64_t part, const ColumnAcc<D>& acc) {
    const int lane = threadIdx.x & 63, l16 = lane & 15, quad = lane >> 4;
    if (hg * 16 + l16 >= w.n_col) return;
    const int64_t at = part_row(w, part, l16);
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

template <class T, int D, bool FP8>
__global__ __launch_bounds__(kLineWaves * 64, 2) void paged_line_kernel(const DecodeWork work) {
    __shared__ __attribute__((aligned(1024))) char lds[kLineWaves][kWaveLds<D, FP8>];
    constexpr int GR = kRows<FP8>;
    const PagedParams& p = work.p;
    const int lane = threadIdx.x & 63, w = wave_id();
    const int pairs = p.Hkv * work.n_hg, n_waves = work.n_wg * kLineWaves;
    const bool first = blockIdx.x == 0 && w == 0;   // the wave that leaves the sequences' places for the merge
    // 64 sequences at a time, 256 requested together; the first 64 are kept
    constexpr int UN = 4;
    LineSeq kept{{0, 0, 0}, 0};
    int total = 0, longest = 0;
    for (int base = 0; base < p.n_seqs; base += 64 * UN) {
        LineSeq q[UN];
#pragma unroll
        for (int u = 0; u < UN; ++u) q[u] = line_seq<GR>(work, base + 64 * u + lane);
        if (base == 0) kept = q[0];
#pragma unroll
        for (int u = 0; u < UN; ++u) {
            const int b = base + 64 * u;
            if (b >= p.n_seqs) break;
            const int incl = wave_inclusive_scan(q[u].groups * pairs);
            if (first && b + lane < p.n_seqs) work.seq_off[b + lane] = total + incl - q[u].groups * pairs;
            total += lane_value(incl, 63);
            longest = max(longest, q[u].groups);
        }
    }
    longest = (int)wave_max((float)longest);   // (below 2^24 exactly, and above rounded up or down by less than the parts to spare)
    const int quota = max(max((total + n_waves - 1) / n_waves, kLeastShare / GR), longest / (kMaxParts - 3) + 1);
    if (first && lane == 0) { work.seq_off[p.n_seqs] = total; work.seq_off[p.n_seqs + 1] = quota; }
    // shares to the waves of a workgroup in turn; where there are no more shares than workgroups, one to each
    // (the line's length and a share of it may together pass 31 bits)
    const int n_shares = total > 0 ? (total - 1) / quota + 1 : 0;
    const int wave = n_shares <= (int)gridDim.x ? w * (int)gridDim.x + (int)blockIdx.x : (int)blockIdx.x * kLineWaves + w;
    if (wave >= n_shares) return;
    int x = wave * quota;
    const int x_end = x + min(quota, total - x);
    // the sequence that holds position x
    int s = 0, off = 0, groups = 0;
    for (int base = 0, start = 0; base < p.n_seqs; base += 64) {
        const LineSeq q = base == 0 ? kept : line_seq<GR>(work, base + lane);
        const int incl = wave_inclusive_scan(q.groups * pairs), sum = lane_value(incl, 63);
        if (x < start + sum) {
            const int src = __builtin_amdgcn_readfirstlane(__ffsll((unsigned long long)__ballot(x < start + incl)) - 1);
            s = base + src;
            groups = lane_value(q.groups, src);
            off = start + lane_value(incl, src) - groups * pairs;
            break;
        }
        start += sum;
    }
    SeqInfo info = seq_info(p, s);
    while (x < x_end) {
        if (x >= off + pairs * groups) {   // the sequence is done: on to the next that has rows
            off += pairs * groups;
            do {
                info = seq_info(p, ++s);
                groups = info.len > 0 ? (info.ctx + GR - 1) / GR : 0;
            } while (groups == 0);
        }
        const int y = x - off, pair = y / groups, g0 = y - pair * groups, g1 = min(groups, g0 + (x_end - x));
        const int hg = work.n_hg == 1 ? 0 : pair / p.Hkv, g = pair - hg * p.Hkv;
        ColumnAcc<D> acc;
        stream_pages<T, D, FP8>(work, s, info, g, hg, g0, g1, lds[w], acc);
        store_part<D>(work, hg, (int64_t)s * pairs + pair + wave, acc);
        x += g1 - g0;
    }
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

// out = sum_i O_i w_i / sum_i l_i w_i, w_i = 2^(m_i - max m), over the parts of a row; a wave per row (sequence, token, head), lane i holding part i's
// reference and sum.
template <class T, int D, int GR>
__global__ __launch_bounds__(256) void paged_merge_kernel(const DecodeWork work) {
    const PagedParams& p = work.p;
    constexpr int EPL = D / 64;
    const int lane = threadIdx.x & 63;
    const int64_t row = (int64_t)blockIdx.x * 4 + wave_id();
    const int per_seq = p.Hkv * work.n_col;
    if (row >= (int64_t)p.n_seqs * per_seq) return;
    const int s = (int)(row / per_seq), in = (int)(row - (int64_t)s * per_seq), g = in / work.n_col, col = in - g * work.n_col;
    const SeqInfo info = seq_info(p, s);
    const int tok = col / p.n_rep;
    if (tok >= info.len) return;
    const int groups = (info.ctx + GR - 1) / GR, quota = const_load(work.seq_off + p.n_seqs + 1), pair = (col / 16) * p.Hkv + g;
    const int start = const_load(work.seq_off + s) + pair * groups, first = start / quota;   // the pair's first group and its share
    const int ns = groups > 0 ? min((start + groups - 1) / quota - first + 1, kMaxParts) : 0;
    const int64_t at0 = part_row(work, (int64_t)s * p.Hkv * work.n_hg + pair + first, col % 16);
    const float* src = p.part_o + at0 * D + EPL * lane;
    auto load_o = [&](int part, float (&x)[EPL]) __attribute__((always_inline)) {
        const float* at = src + (int64_t)part * work.per_part * D;
        if (EPL == 2) { const f32x2 v = *reinterpret_cast<const f32x2*>(at); x[0] = v[0]; x[EPL - 1] = v[1]; }
        else x[0] = at[0];
    };
    // the first parts' rows beside their references and sums
    f32x2 ml = {-INFINITY, 0.f};
    if (lane < ns) ml = *reinterpret_cast<const f32x2*>(p.part_ml + (at0 + (int64_t)lane * work.per_part) * 2);
    constexpr int kEarly = 4;
    float x[8][EPL];
#pragma unroll
    for (int u = 0; u < kEarly; ++u) {
#pragma unroll
        for (int e = 0; e < EPL; ++e) x[u][e] = 0.f;
        if (ns > 0) load_o(min(u, ns - 1), x[u]);
    }
    const PartWeights pw = part_weights(ml[0], ml[1]);
    float acc[EPL];
#pragma unroll
    for (int e = 0; e < EPL; ++e) acc[e] = 0.f;
    for (int s0 = 0; s0 < ns; s0 += 8) {
#pragma unroll
        for (int u = 0; u < 8; ++u)
            if (s0 > 0 || u >= kEarly) load_o(min(s0 + u, ns - 1), x[u]);
#pragma unroll
        for (int u = 0; u < 8; ++u) {
            const float wi = lane_value(pw.w, min(s0 + u, 63));
#pragma unroll
            for (int e = 0; e < EPL; ++e) acc[e] += s0 + u < ns ? x[u][e] * wi : 0.f;
        }
    }
    const float inv = pw.total > 0.f ? 1.f / pw.total : 0.f;
    uint16_t* dst = reinterpret_cast<uint16_t*>(p.out) + (int64_t)(info.lo + tok) * p.o2 + (int64_t)(g * p.n_rep + col - tok * p.n_rep) * p.o1 + EPL * lane;
    if (EPL == 2) *reinterpret_cast<uint32_t*>(dst) = T::pack2(acc[0] * inv, acc[EPL - 1] * inv);
    else dst[0] = (uint16_t)(T::pack2(acc[0] * inv, 0.f) & 0xffffu);
}

// ---- chunks ----------------------------------------------------------------------------------------------------------
// What the line costs a small problem is latency: a wave streams its rows one group after the other, and a second launch merges.  Here the eight waves of
// a workgroup share a chunk and merge in LDS.  A pair that is one chunk long is done with that; otherwise the chunk's result goes to
// the workspace, and the workgroup that comes last (a counter per pair) merges the pair's.  Results cross from one XCD's L2 to
// another's: they are written and read with device-scope accesses, which go past the L2s on both sides, and a workgroup counts itself
// only when its own have arrived; the reader's loads stand behind a barrier that thread 0 reaches with the count's value in hand.
MA_DEV void store_shared(float* p, float x) { __hip_atomic_store(p, x, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); }
MA_DEV float load_shared(const float* p) { return __hip_atomic_load(const_cast<float*>(p), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); }
MA_DEV void store_shared2(float* p, f32x2 x) {
    __hip_atomic_store(reinterpret_cast<uint64_t*>(p), __builtin_bit_cast(uint64_t, x), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
MA_DEV f32x2 load_shared2(const float* p) {
    return __builtin_bit_cast(f32x2, __hip_atomic_load(reinterpret_cast<uint64_t*>(const_cast<float*>(p)), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT));
}

// Every pair of a sequence is cut into the same number of chunks, equal to within a group; the chunk's size, the same for all sequences, is the
// smallest (256 rows at least) that leaves no more chunks than workgroups.  Up to 64 sequences, one to a lane; all waves
// work it out for themselves.
template <int GR> struct ChunkPlan {
    LineSeq q;        // per lane: the sequence
    int each, incl;   // per lane: chunks of each of its pairs; chunks of the sequences up to and with it
    int total;
    MA_DEV ChunkPlan(const DecodeWork& w, int n_wg) {
        const int lane = threadIdx.x & 63, pairs = w.p.Hkv * w.n_hg;
        q = line_seq<GR>(w, lane);
        const bool on = lane < w.p.n_seqs && q.info.len > 0;
        const int sum = lane_value(wave_inclusive_scan(q.groups * pairs), 63), active = __popcll(__ballot(on));
        const int longest = (int)wave_max((float)q.groups);
        // a pair's last chunk is half full on average: that many workgroups are as good as not there
        int size = max(max((sum + n_wg - 1) / max(n_wg - active * pairs / 2, 1), 256 / GR), longest / kMaxParts + 1);
        for (;; size += 1 + size / 16) {   // (ends: with the longest context as the size there is one chunk a pair, and no more pairs than workgroups)
            each = on ? max((q.groups + size - 1) / size, 1) : 0;
            incl = wave_inclusive_scan(each * pairs);
            total = lane_value(incl, 63);
            if (total <= n_wg) break;
        }
    }
};

// Merges the n chunks, from number `first` of the launch on, of the columns of (s, g, hg) from the workspace and stores the output rows; all threads of the workgroup, a wave 64
// elements of a column at a time, without LDS and barriers (with the weights made by 16 threads in LDS it took twice the time).  The order of
// the sums depends on nothing but n.
template <class T, int D>
MA_DEV void merge_chunks(const DecodeWork& w, const SeqInfo& info, int g, int hg, int first, int n) {
    const PagedParams& p = w.p;
    const int lane = threadIdx.x & 63, wave = wave_id(), cols = min(16, w.n_col - hg * 16);
    const int64_t at0 = part_row(w, first, 0), step = (int64_t)w.per_part * D;
    constexpr int PER = 16 * D / (kChunkWaves * 64);
    float x[PER][8];
    f32x2 ml[PER];
#pragma unroll
    for (int e = 0; e < PER; ++e) {
        const int idx = (wave + e * kChunkWaves) * 64;
        if (idx < cols * D) {
            const int64_t at = at0 + idx / D;
            ml[e] = load_shared2(p.part_ml + (at + (int64_t)min(lane, n - 1) * w.per_part) * 2);
            const float* src = p.part_o + at * D + idx % D + lane;
#pragma unroll
            for (int u = 0; u < 8; ++u) x[e][u] = load_shared(src + min(u, n - 1) * step);
        }
    }
#pragma unroll
    for (int e = 0; e < PER; ++e) {
        const int idx = (wave + e * kChunkWaves) * 64;
        if (idx >= cols * D) break;
        const int c = idx / D, d = idx % D + lane, col = hg * 16 + c, tok = col / p.n_rep;
        const PartWeights pw = part_weights(lane < n ? ml[e][0] : -INFINITY, lane < n ? ml[e][1] : 0.f);
        const float* src = p.part_o + (at0 + c) * D + d;
        float sum = 0.f;
        for (int s0 = 0; s0 < n; s0 += 8) {
            if (s0 > 0) {
#pragma unroll
                for (int u = 0; u < 8; ++u) x[e][u] = load_shared(src + min(s0 + u, n - 1) * step);
            }
#pragma unroll
            for (int u = 0; u < 8; ++u) {
                const float wi = lane_value(pw.w, min(s0 + u, 63));
                sum += s0 + u < n ? x[e][u] * wi : 0.f;
            }
        }
        if (tok < info.len)
            reinterpret_cast<uint16_t*>(p.out)[(int64_t)(info.lo + tok) * p.o2 + (int64_t)(g * p.n_rep + col - tok * p.n_rep) * p.o1 + d] = (uint16_t)(T::pack2(sum * (pw.total > 0.f ? 1.f / pw.total : 0.f), 0.f) & 0xffffu);
    }
}

template <class T, int D, bool FP8>
__global__ __launch_bounds__(kChunkWaves * 64, 2) void paged_chunk_kernel(const DecodeWork work) {
    const PagedParams& p = work.p;
    constexpr int NW = kChunkWaves, DB = D / 16, GR = kRows<FP8>, WAVE_LDS = kWaveLds<D, FP8>;
    constexpr int ORS = D + 4;   // floats between two columns of a wave's result: their 16-byte pieces start in different banks
    constexpr int LDS = NW * WAVE_LDS > NW * 16 * ORS * 4 ? NW * WAVE_LDS : NW * 16 * ORS * 4;
    __shared__ __attribute__((aligned(1024))) char lds[LDS];   // the waves' row areas, then their results
    __shared__ float ml_s[2 * NW * 16];
    __shared__ int last_s;
    const int tid = threadIdx.x, lane = tid & 63, w = wave_id(), l16 = lane & 15, quad = lane >> 4;
    const int pairs = p.Hkv * work.n_hg;
    const ChunkPlan<GR> plan(work, (int)gridDim.x);
    const int x = (int)blockIdx.x;
    if (x >= plan.total) return;
    const int s = __builtin_amdgcn_readfirstlane(__ffsll((unsigned long long)__ballot(x < plan.incl)) - 1);
    const SeqInfo info{lane_value(plan.q.info.lo, s), lane_value(plan.q.info.len, s), lane_value(plan.q.info.ctx, s)};
    const int n = lane_value(plan.each, s), all = lane_value(plan.q.groups, s);   // chunks and groups of the pair
    const int local = x - (lane_value(plan.incl, s) - n * pairs), pair = local / n, split = local - pair * n;
    const int hg = work.n_hg == 1 ? 0 : pair / p.Hkv, g = pair - hg * p.Hkv;
    const int size = all / n, longer = all - size * n;   // the first `longer` chunks are a group longer
    const int first = split * size + min(split, longer), groups = size + (split < longer ? 1 : 0);
    const int per = (groups + NW - 1) / NW;
    const int g_lo = min(w * per, groups), g_hi = min(g_lo + per, groups);
    ColumnAcc<D> acc;
    acc.m = -INFINITY; acc.l = 0.f;
#pragma unroll
    for (int db = 0; db < DB; ++db) acc.o[db] = f32x4{0.f, 0.f, 0.f, 0.f};
    if (g_hi > g_lo) stream_pages<T, D, FP8>(work, s, info, g, hg, first + g_lo, first + g_hi, lds + w * WAVE_LDS, acc);
    __syncthreads();   // every wave is done with its row area
    const int cols = min(16, work.n_col - hg * 16);
    float* o_s = reinterpret_cast<float*>(lds);   // [wave][column][ORS]
    if (l16 < cols) {
        float* dst = o_s + (w * 16 + l16) * ORS + 4 * quad;
#pragma unroll
        for (int db = 0; db < DB; ++db) *reinterpret_cast<f32x4*>(dst + 16 * db) = acc.o[db];
        if (quad == 0) { ml_s[w * 16 + l16] = acc.m; ml_s[(NW + w) * 16 + l16] = acc.l; }
    }
    __syncthreads();
    const bool whole = n <= 1;   // the chunk is the whole context: its result is the output
    const int64_t at0 = part_row(work, x, 0);
    for (int idx = w * 64; idx < cols * D; idx += NW * 64) {   // a wave 64 elements of a column
        const int c = idx / D, d = idx % D + lane;
        const PartWeights pw = part_weights(lane < NW ? ml_s[lane * 16 + c] : -INFINITY, lane < NW ? ml_s[(NW + lane) * 16 + c] : 0.f);
        float sum = 0.f;
#pragma unroll
        for (int i = 0; i < NW; ++i) sum += o_s[(i * 16 + c) * ORS + d] * lane_value(pw.w, i);
        if (whole) {
            const int col = hg * 16 + c, tok = col / p.n_rep;
            if (tok < info.len)
                reinterpret_cast<uint16_t*>(p.out)[(int64_t)(info.lo + tok) * p.o2 + (int64_t)(g * p.n_rep + col - tok * p.n_rep) * p.o1 + d] = (uint16_t)(T::pack2(sum * (pw.total > 0.f ? 1.f / pw.total : 0.f), 0.f) & 0xffffu);
        } else {
            store_shared(p.part_o + (at0 + c) * D + d, sum);
            if (idx % D == 0 && lane == 0) store_shared2(p.part_ml + (at0 + c) * 2, f32x2{pw.top, pw.total});
        }
    }
    if (whole || !work.done) return;
    wait_vmcnt<0>();   // the thread's stores have arrived
    __syncthreads();
    if (tid == 0) {
        uint32_t* done = work.done + s * pairs + pair;
        const uint32_t before = __hip_atomic_fetch_add(done, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        last_s = before == (uint32_t)(n - 1);
        if (last_s) __hip_atomic_store(done, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
    __syncthreads();
    if (last_s) merge_chunks<T, D>(work, info, g, hg, x - split, n);
}

// (where there are no counters) grid (column groups x KV heads, sequences)
template <class T, int D, int GR>
__global__ __launch_bounds__(kChunkWaves * 64) void paged_chunk_merge_kernel(const DecodeWork work, int n_wg) {
    const PagedParams& p = work.p;
    const int s = blockIdx.y, hg = (int)blockIdx.x / p.Hkv, g = (int)blockIdx.x - hg * p.Hkv;
    const ChunkPlan<GR> plan(work, n_wg);
    const int n = lane_value(plan.each, s), pairs = p.Hkv * work.n_hg;
    if (n > 1) merge_chunks<T, D>(work, seq_info(p, s), g, hg, lane_value(plan.incl, s) - n * (pairs - (int)blockIdx.x), n);
}

// Workgroups of the line: as many as the chip holds at once.
static int compute_units() {
    static std::atomic<int> cached[64];
    int dev = 0;
    if (hipGetDevice(&dev) != hipSuccess || dev < 0 || dev >= 64) dev = 0;
    int n = cached[dev].load(std::memory_order_relaxed);
    if (n == 0) {
        if (hipDeviceGetAttribute(&n, hipDeviceAttributeMultiprocessorCount, dev) != hipSuccess || n <= 0) n = 256;
        cached[dev].store(n, std::memory_order_relaxed);
    }
    return n;
}

bool paged_decode_takes(int64_t Hq, int64_t Hkv, int64_t max_q) { return max_q == 1 || max_q * (Hq / Hkv) <= 16; }

template <class T, int D, bool FP8> static int launch_line(DecodeWork w, hipStream_t stream) {
    hipLaunchKernelGGL((paged_line_kernel<T, D, FP8>), dim3((unsigned)w.n_wg), dim3(kLineWaves * 64), 0, stream, w);
    if (int rc = check_launch("paged_line_kernel")) return rc;
    const int64_t rows = (int64_t)w.p.n_seqs * w.p.Hkv * w.n_col;
    hipLaunchKernelGGL((paged_merge_kernel<T, D, kRows<FP8>>), dim3((unsigned)((rows + 3) / 4)), dim3(256), 0, stream, w);
    return check_launch("paged_merge_kernel");
}
// Whether a call is one for chunks.  Up to a pair for every unit always (us, chunks / line, contexts alike and from a sixteenth up, 32 heads on 8 of 128: one of 4000
// 10.0 / 14.0, 8.2 / 10.6; 4 of 30000 78 / 87, 43 / 62; 16 of 4000 44 / 48, 26 / 31, of 20000 e4m3 109 / 114, 87 / 76; 32 of 300 8.4 / 15.9, 7.2 / 12.3, of 1500
// e4m3 21 / 28, 18 / 21; where every unit has one long context, contexts that differ leave units idle: 32 of 6000 123 / 131, 79 / 72, e4m3 66 / 73, 55 / 45).
// Two rounds of whole contexts where the table has no room for long ones: 64 of 100 11.5 / 13.2, 10.7 / 14.0, of 400 23.0 / 24.6, 17.0 / 17.6, of 1000
// 44.5 / 48.8, 30.2 / 30.4, of 2000 82 / 88, 55 / 53, of 6000 242 / 251, 148 / 141; e4m3 of 100 11.4 / 11.4, 10.9 / 12.5, of 400 18.1 / 21.1, 16.8 / 15.6, of 700 23.4 /
// 27.1, 20.7 / 20.8, of 1000 32.0 / 31.0, 27.9 / 24.4.
static int chunk_rounds(int64_t n_seqs, int64_t pairs, int64_t max_context, bool eight) {
    const int64_t units = compute_units();
    if (n_seqs > 64 || pairs > kStreamCounters) return 0;
    return pairs <= units ? 1 : pairs <= 2 * units && max_context <= (eight ? 768 : 2048) ? 2 : 0;
}

// How a call is laid out, from its sizes alone.
struct DecodePlan {
    int64_t n_col, n_hg, per_part;   // as in DecodeWork
    int rounds;                      // chunk_rounds
    int64_t parts;                   // partial results: chunks, a workgroup each; of the line, shares and pairs
    size_t o_bytes, ml_bytes, bytes;
};
static size_t whole_lines(int64_t bytes) { return ((size_t)bytes + 255) / 256 * 256; }
static DecodePlan plan_decode(bool eight, int64_t n_seqs, int64_t Hq, int64_t Hkv, int64_t D, int64_t max_context, int64_t max_q) {
    DecodePlan r{};
    r.n_col = max_q * (Hq / Hkv);
    r.n_hg = (r.n_col + 15) / 16;
    r.per_part = std::min<int64_t>(r.n_col, 16);
    const int64_t pairs = n_seqs * Hkv * r.n_hg, units = compute_units();
    r.rounds = chunk_rounds(n_seqs, pairs, max_context, eight);
    r.parts = r.rounds > 0 ? r.rounds * units : units * kLineWgPerCu * kLineWaves + pairs;
    r.o_bytes = whole_lines(r.parts * r.per_part * D * 4);
    r.ml_bytes = whole_lines(r.parts * r.per_part * 2 * 4);
    r.bytes = r.o_bytes + r.ml_bytes + (r.rounds > 0 ? 0 : whole_lines((n_seqs + 2) * 4));
    return r;
}
size_t paged_decode_workspace_bytes(int64_t n_seqs, int64_t Hq, int64_t Hkv, int64_t D, int64_t max_context, int64_t max_q) {
    return std::max(plan_decode(false, n_seqs, Hq, Hkv, D, max_context, max_q).bytes, plan_decode(true, n_seqs, Hq, Hkv, D, max_context, max_q).bytes);
}

template <class T, int D, bool FP8> static int launch_chunks(DecodeWork w, int rounds, hipStream_t stream) {
    const int n_wg = rounds * compute_units();
    w.done = stream_counters(stream);
    hipLaunchKernelGGL((paged_chunk_kernel<T, D, FP8>), dim3((unsigned)n_wg), dim3(kChunkWaves * 64), 0, stream, w);
    if (int rc = check_launch("paged_chunk_kernel")) return rc;
    if (w.done) return MINFER_ATTN_OK;
    hipLaunchKernelGGL((paged_chunk_merge_kernel<T, D, kRows<FP8>>), dim3((unsigned)(w.p.Hkv * w.n_hg), (unsigned)w.p.n_seqs), dim3(kChunkWaves * 64), 0, stream, w, n_wg);
    return check_launch("paged_chunk_merge_kernel");
}
template <class T, int D, bool FP8> static int launch_rows(const DecodeWork& w, int rounds, hipStream_t stream) {
    return rounds > 0 ? launch_chunks<T, D, FP8>(w, rounds, stream) : launch_line<T, D, FP8>(w, stream);
}
template <class T> static int launch_decode_as(const DecodeWork& w, int64_t D, bool eight, int rounds, hipStream_t stream) {
    if (eight) return D == 128 ? launch_rows<T, 128, true>(w, rounds, stream) : launch_rows<T, 64, true>(w, rounds, stream);
    return D == 128 ? launch_rows<T, 128, false>(w, rounds, stream) : launch_rows<T, 64, false>(w, rounds, stream);
}

int launch_paged_decode(PagedParams p, int dtype, int64_t D, bool eight, int64_t max_context, void* workspace, hipStream_t stream) {
    DecodeWork w{};
    const DecodePlan plan = plan_decode(eight, p.n_seqs, p.Hq, p.Hkv, D, max_context, p.max_q);
    w.n_col = (int)plan.n_col;
    w.n_hg = (int)plan.n_hg;
    w.per_part = (int)plan.per_part;
    w.n_wg = compute_units() * kLineWgPerCu;
    const int64_t rows = (int64_t)p.n_seqs * p.Hkv * w.n_col;
    if (rows > 0x7fffffffLL || (int64_t)p.n_seqs * p.Hkv * w.n_hg * ((max_context + 15) / 16 + 1) > 0x7fffffffLL - 65536)
        return fail(MINFER_ATTN_EINVAL, "flash_attn_paged: problem too large for one launch");
    p.part_o = (float*)workspace;
    p.part_ml = (float*)((char*)workspace + plan.o_bytes);
    w.seq_off = plan.rounds > 0 ? nullptr : (int32_t*)((char*)p.part_ml + plan.ml_bytes);
    w.p = p;
    return dtype == MINFER_ATTN_F16 ? launch_decode_as<F16>(w, D, eight, plan.rounds, stream) : launch_decode_as<BF16>(w, D, eight, plan.rounds, stream);
}

}  // namespace minfer_attn
