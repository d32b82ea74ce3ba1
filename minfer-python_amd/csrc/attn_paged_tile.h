// The walk of a block of rows over the 64-key tiles of a paged cache for gfx950, the part that the attention of packed tokens and that of groups which share
// a prefix have in common.
//
// Per tile a wave computes S^T = K Q^T and O^T += V^T P^T with v_mfma_f32_16x16x32, the scores staying in registers as the second
// product's operand; tiles are double-buffered in LDS, 16-bit rows copied there directly, 8-bit codes through registers, in which
// they become 16-bit values (exactly: a scale is a power of two).  A tile's rows come from up to four pages, looked up a tile ahead
// as scalars: pages have at least 16 rows, so a copy instruction's rows lie in one.
//
// Rows that nothing was written to, behind the context in its last page, and rows of pages that are not there may hold NaN, which a weight of zero would
// not take out of a sum: their scores are replaced, and their V rows are cleared in LDS, in the few tiles that have any.  A row with an infinity or a NaN
// that a sequence's later tokens attend is kept from its earlier ones as well (attend_key_by_key).
#pragma once

#include "attn_paged.h"

namespace minfer_attn {

template <int D, int NW> struct PagedGeom {
    static constexpr int RB = D * 2;                 // bytes per 16-bit row
    static constexpr int G = RB / 16;                // 16-byte granules per row
    static constexpr int RPI = 1024 / RB;            // rows one wave-wide copy instruction covers
    static constexpr int NLD = 64 / (NW * RPI);      // copy instructions per wave, tile and tensor
    static constexpr int RPI8 = 1024 / D;            // the same for rows of codes
    static constexpr int NLD8 = 64 / (NW * RPI8);
    static constexpr int TILE_BYTES = 64 * RB;
    // granule swizzles that make the 16-row reads of K and the transpose reads of V free of bank conflicts
    static MA_DEV int swz_k(int row) { return (row / (256 / RB)) & (G - 1); }
    static MA_DEV int swz_v(int row) { return D == 128 ? ((row & 7) << 1) : (((row >> 1) & 3) << 1); }
};

// Sixteen e4m3 codes times a scale.
template <class T> MA_DEV void widen16(u32x4 codes, float scale, s16x8 (&to)[2]) {
    uint32_t w[8];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        w[2 * i] = widen2<T, false>(codes[i], scale);
        w[2 * i + 1] = widen2<T, true>(codes[i], scale);
    }
#pragma unroll
    for (int h = 0; h < 2; ++h) to[h] = __builtin_bit_cast(s16x8, u32x4{w[4 * h], w[4 * h + 1], w[4 * h + 2], w[4 * h + 3]});
}

// The first row of a sequence in a page that is there (its context if there is none): a window that moved on has given the pages
// in front of it back.  Looked for only where the first page is missing, 64 pages at a time; the whole wave.
MA_DEV int first_row(const PagedCache& c, int seq, int ctx) {
    const int32_t* table = c.table + (int64_t)seq * c.table_stride;
    const int lane = threadIdx.x & 63, n = (ctx + (1 << c.page_log2) - 1) >> c.page_log2;
    for (int base = 0; base < n; base += 64) {
        const int i = base + lane;
        const uint64_t hit = __ballot(i < n && (unsigned)table[min(i, n - 1)] < (unsigned)c.n_pages);
        if (hit) return (base + __ffsll((unsigned long long)hit) - 1) << c.page_log2;
    }
    return ctx + 63;   // behind the last tile
}

// LDS of a workgroup: its stages, the rows' area where it has one of its own, the codes' areas.  A block of one sequence's rows meets tiles that blocks beside
// it have just read, and two stages do: a tile is on its way for the time of one.  The rows of a group that shares a prefix are few and read tiles
// nobody has (SHARED): three tiles are on their way, into four stages of 16-bit rows, or into four areas of codes in front of two stages.
template <int D, bool FP8, int NW, bool SHARED> struct TileLds {
    using GEO = PagedGeom<D, NW>;
    static constexpr int STAGE_BYTES = 2 * GEO::TILE_BYTES;   // the K tile followed by the V tile
    static constexpr int ROWS_BYTES = 32 * GEO::RB;
    static constexpr int RING = 4;                            // SHARED: stages, or areas of codes
    static constexpr int STAGES = SHARED && !FP8 ? RING : 2;
    // The waves' query rows on their way in and output rows on their way out: with four waves inside a stage (the query rows in stage 1, which no
    // tile touches before the barrier of tile 0; the output rows in the stage that the last tile did not use), with eight beside them.
    // SHARED: the query rows in the last two stages.
    static constexpr bool kAliasRows = SHARED || NW * ROWS_BYTES <= STAGE_BYTES;
    static constexpr int ROWS_AT = SHARED ? (STAGES - 2) * STAGE_BYTES : kAliasRows ? STAGE_BYTES : 2 * STAGE_BYTES;
    static_assert(!SHARED || NW * ROWS_BYTES <= 2 * STAGE_BYTES, "query rows in two stages");
    static constexpr int NR = FP8 ? GEO::NLD8 : 1;            // loads of codes per wave, tile and tensor
    static constexpr int RAW_BYTES = FP8 ? 2 * NR * 1024 : 0, RAW_AT = STAGES * STAGE_BYTES + (kAliasRows ? 0 : NW * ROWS_BYTES);
    static constexpr int BYTES = RAW_AT + NW * RAW_BYTES * (SHARED ? RING : 1);
};

// What a workgroup walks: the tiles of a block of rows of KV head g, the `part`-th of `parts` equal pieces of them; or (SHARED) n_own of them, from tile t_lo on.
// The rows are (token, head) pairs from token `lo` on, `rows` in all, of which the workgroup's are row0 .. row_end - 1: those of a sequence, whose table row and
// context these are and whose token 0 stands at pos0; or (`prefix`) those of the sequences first .. last - 1 that share one, ctx being its rows, whole tiles, all
// of which every row attends, but for tokens that stand inside them (`inside`: there are some).
// Its partial results: the `slot`-th of all pieces, or (SHARED) from row `slot` of them on.
struct TileJob { int g, seq, lo, ctx, pos0, rows, row0, row_end, part, parts, slot, t_lo, n_own, first, last; bool prefix, inside; };

MA_DEV int tiles_of(int pos0, int rows, int n_rep, int block, int BR) { return (max(pos0 + min(block * BR + BR - 1, rows - 1) / n_rep + 1, 0) + 63) >> 6; }

// Position of packed token t, which is one of the sequences first .. last - 1 (cu_seqlens' entries do not fall up to the last one's end); -1 if it is not.  A search by halves: 4000 sequences behind 1024 rows,
// one of them inside, 138 us (131 with none; 2034 along the sequences), 192 behind 6400 74 (67; 134).
MA_DEV int position_of(const PagedParams& p, int first, int last, int t) {
    int s = first, end = last - 1;   // the last sequence that does not begin behind t
    while (s < end) {
        const int mid = (s + end + 1) >> 1;
        if (p.cu[mid] <= t) s = mid; else end = mid - 1;
    }
    if (s >= last) return -1;
    const TokenRange r = token_range(p.cu[s], p.cu[s + 1], p.T);
    return t >= r.lo && t < r.lo + r.len ? context_of(p.c, p.ctx[s], r) - r.len + t - r.lo : -1;
}

template <class T, int D, bool FP8, int NW, bool SHARED> MA_DEV void attend_tiles(const PagedParams& p, const TileJob& job, char* const lds) {
    using LDS = TileLds<D, FP8, NW, SHARED>;
    using GEO = typename LDS::GEO;
    constexpr int KEYS = 64, NB = KEYS / 16;   // of a tile: keys, blocks of 16
    constexpr int RB = GEO::RB, G = GEO::G, RPI = GEO::RPI, NLD = GEO::NLD;
    constexpr int KC = D / 32;   // 32-wide contraction chunks of Q K^T
    constexpr int DB = D / 16;   // 16-row blocks of O^T
    constexpr int BR = NW * 32;  // rows of a workgroup
    constexpr int STAGE_BYTES = LDS::STAGE_BYTES, ROWS_BYTES = LDS::ROWS_BYTES;
    constexpr bool kAliasRows = LDS::kAliasRows;

    const int lane = threadIdx.x & 63, w = wave_id();
    const int l16 = lane & 15, quad = lane >> 4;
    const int g = job.g, seq = job.seq, ctx = job.ctx;
    const int last_row = (SHARED ? job.row_end : job.rows) - 1;
    const int row0 = job.row0 + w * 32;                                  // the wave's first row
    const bool wave_on = row0 <= last_row;

    // ---- the wave's query rows, copied global->LDS as whole rows ----
    char* const q_stage = lds + LDS::ROWS_AT + w * ROWS_BYTES;
#pragma unroll
    for (int j = 0; j < 32 / RPI; ++j) {
        const int row = j * RPI + lane / G, r = min(row0 + row, last_row), t = r / p.n_rep;
        const short* src = (const short*)p.q + (int64_t)(job.lo + t) * p.q2 + (int64_t)(g * p.n_rep + r - t * p.n_rep) * p.q1 + 8 * ((lane % G) ^ GEO::swz_k(row));
        copy16_global_to_lds(src, q_stage + j * RPI * RB);
    }

    // ---- pages: the 16-row blocks of a tile -----------------------------------------------------------------
    const int32_t* const table = p.c.table + (int64_t)seq * p.c.table_stride;
    struct Pages { int id[NB]; };
    auto pages_of = [&](int kt) __attribute__((always_inline)) {
        Pages r;
#pragma unroll
        for (int b = 0; b < NB; ++b) r.id[b] = const_load(table + min((kt * KEYS + 16 * b) >> p.c.page_log2, p.c.width - 1));
        return r;
    };
    int t_lo, n_own;
    Pages next3[3];
    if constexpr (SHARED) {
        t_lo = job.t_lo;
        n_own = job.n_own;
        next3[0] = pages_of(t_lo);   // asked for together with the table's first entry
        next3[1] = pages_of(t_lo + 1);
        next3[2] = pages_of(t_lo + 2);
        // (tiles in front of the first page that is there)
        if (n_own > 0 && (unsigned)const_load(p.c.table + (int64_t)seq * p.c.table_stride) >= (unsigned)p.c.n_pages) {
            const int t_first = min(max(__builtin_amdgcn_readfirstlane(first_row(p.c, seq, ctx)) / KEYS, t_lo), t_lo + n_own);
            n_own -= t_first - t_lo;
            t_lo = t_first;
#pragma unroll
            for (int i = 0; i < 3; ++i) next3[i] = pages_of(t_lo + i);
        }
    } else {
        const int tiles = tiles_of(job.pos0, job.rows, p.n_rep, job.row0 / BR, BR);
        int t_first = 0;
        if (tiles > 0 && (unsigned)const_load(p.c.table + (int64_t)seq * p.c.table_stride) >= (unsigned)p.c.n_pages)
            t_first = __builtin_amdgcn_readfirstlane(first_row(p.c, seq, ctx)) / KEYS;
        const int n_tiles = max(tiles - t_first, 0), each = n_tiles / job.parts, longer = n_tiles - each * job.parts;
        t_lo = t_first + job.part * each + min(job.part, longer);
        n_own = each + (job.part < longer ? 1 : 0);
    }

    // positions of the lane's two rows (one per block of 16), cut to the last key, and the wave's least and greatest
    int pos[2] = {job.pos0 + min(row0 + l16, last_row) / p.n_rep, job.pos0 + min(row0 + 16 + l16, last_row) / p.n_rep};
    int wave_first = job.pos0 + min(row0, last_row) / p.n_rep, wave_last = job.pos0 + min(row0 + 31, last_row) / p.n_rep;
    if (SHARED && job.prefix) {
        pos[0] = pos[1] = wave_first = wave_last = ctx - 1;
        if (job.inside) {
#pragma unroll
            for (int qb = 0; qb < 2; ++qb) pos[qb] = min(ctx - 1, position_of(p, job.first, job.last, job.lo + min(row0 + 16 * qb + l16, last_row) / p.n_rep));
            wave_first = __builtin_amdgcn_readfirstlane(-(int)wave_max((float)-min(pos[0], pos[1]))) - 64;   // (as a float it is off by less than a tile)
        }
    }

    auto is_there = [&](int id) __attribute__((always_inline)) { return (unsigned)id < (unsigned)p.c.n_pages; };
    // bit b: the page of the tile's block b is there
    auto there_of = [&](const Pages& pg) __attribute__((always_inline)) {
        int r = 0;
#pragma unroll
        for (int b = 0; b < NB; ++b) r |= is_there(pg.id[b]) ? 1 << b : 0;
        return r;
    };
    // whether all rows of a tile exist and hold what was written to them
    auto whole = [&](int kt, int there) __attribute__((always_inline)) { return kt * KEYS + KEYS <= ctx && there == (1 << NB) - 1; };
    const int page_mask = (1 << p.c.page_log2) - 1;
    // rows first .. of tile kt, which lie in page `id`: their offset in a pool, in elements (a page that is not there: page 0, whose
    // rows are there to be read)
    auto rows_at = [&](int id, int key) __attribute__((always_inline)) -> int64_t {
        return (int64_t)(is_there(id) ? id : 0) * p.c.page_stride + (int64_t)g * p.c.head_stride + (int64_t)(key & page_mask) * p.c.row_stride;
    };

    const uint32_t dst0 = (uint32_t)__builtin_amdgcn_readfirstlane((int)(lds_addr(lds) + w * 1024));
    // ---- 16-bit rows: global -> LDS.  Instruction j of the wave covers rows (j * NW + w) * RPI .. of the tile, all in one block of 16.
    uint32_t k_off = 0, v_off = 0;
    if (!FP8) {
        const int row_in = lane / G, row = w * RPI + row_in, gr = lane % G;
        k_off = (uint32_t)(row_in * (int)p.c.row_stride + 8 * (gr ^ GEO::swz_k(row))) * 2u;
        v_off = (uint32_t)(row_in * (int)p.c.row_stride + 8 * (gr ^ GEO::swz_v(row))) * 2u;
    }
    auto copy_tile = [&](int kt, const Pages& pg, auto stage_tag, uint32_t dst) __attribute__((always_inline)) {
        for_range<0, NLD>([&](auto j_tag) __attribute__((always_inline)) {
            constexpr int j = decltype(j_tag)::value, b0 = j * NW * RPI / 16;
            constexpr int AT = decltype(stage_tag)::value * STAGE_BYTES + j * NW * 1024;
            const int id = NW * RPI == 16 ? pg.id[b0] : (w * RPI < 16 ? pg.id[b0] : pg.id[(b0 + 1) % NB]);
            static_assert(NW * RPI == 16 || NW * RPI == 32, "a round of copies covers one or two blocks of 16 rows");
            const int64_t at = rows_at(id, kt * KEYS + (j * NW + w) * RPI);
            copy16_global_to_lds_at<AT, true>((const short*)p.c.k + at, k_off, dst);
            copy16_global_to_lds_at<AT + GEO::TILE_BYTES, true>((const short*)p.c.v + at, v_off, dst);
        });
    };
    // V rows of a tile that nothing may be multiplied with: the wave clears those that it copied itself
    auto clear_rows = [&](int kt, int there, int stage) __attribute__((always_inline)) {
        for_range<0, NLD>([&](auto j_tag) __attribute__((always_inline)) {
            constexpr int j = decltype(j_tag)::value;
            const int row = (j * NW + w) * RPI + lane / G;
            if (kt * KEYS + row >= ctx || !(there >> (row >> 4) & 1))
                *reinterpret_cast<u32x4*>(lds + stage * STAGE_BYTES + GEO::TILE_BYTES + (j * NW + w) * 1024 + 16 * lane) = u32x4{0u, 0u, 0u, 0u};
        });
    };
    // ---- 8-bit rows: global -> the wave's own LDS area as they are, and from there through registers into a stage.  Load j of the wave covers
    // rows (j * NW + w) * RPI8 .., 8 or 16 of one block, 16 codes a lane, which the lane itself reads back.
    constexpr int NR = LDS::NR, RPI8 = GEO::RPI8;
    const uint32_t raw0 = (uint32_t)__builtin_amdgcn_readfirstlane((int)lds_addr(lds + (FP8 ? LDS::RAW_AT + w * LDS::RAW_BYTES * (SHARED ? LDS::RING : 1) : 0)));
    struct Scales { uint32_t k[NR], v[NR]; } scales{};   // of the tile in the raw area, as their bytes
    const uint32_t c_off = (uint32_t)((lane / (D / 16)) * (int)p.c.row_stride + 16 * (lane % (D / 16)));
    auto block_of = [&](int j) __attribute__((always_inline)) { return ((j * NW + w) * RPI8) >> 4; };
    auto page_of = [&](const Pages& pg, int b) __attribute__((always_inline)) {
        return NB == 2 ? (b == 0 ? pg.id[0] : pg.id[1]) : b == 0 ? pg.id[0] : b == 1 ? pg.id[1] : b == 2 ? pg.id[NB / 2] : pg.id[NB - 1];
    };
    auto request_codes = [&](int kt, const Pages& pg, uint32_t raw) __attribute__((always_inline)) {
        for_range<0, NR>([&](auto j_tag) __attribute__((always_inline)) {
            constexpr int j = decltype(j_tag)::value;
            const int id = page_of(pg, block_of(j));
            const int64_t at = rows_at(id, kt * KEYS + (j * NW + w) * RPI8);
            copy16_global_to_lds_at<2 * j * 1024, true>((const char*)p.c.k + at, c_off, raw);
            copy16_global_to_lds_at<(2 * j + 1) * 1024, true>((const char*)p.c.v + at, c_off, raw);
        });
    };
    auto scales_of = [&](const Pages& pg) __attribute__((always_inline)) {
        Scales r;
#pragma unroll
        for (int j = 0; j < NR; ++j) {
            const int id = page_of(pg, block_of(j));
            const int64_t sc = (int64_t)(is_there(id) ? id : 0) * p.Hkv + g;
            r.k[j] = const_byte(p.c.k_scales + sc);
            r.v[j] = const_byte(p.c.v_scales + sc);
        }
        return r;
    };
    // The words that hold a tile's scales and, two bits each, which byte of them: to take the bytes out is to wait for the words.
    struct ScaleWords { uint32_t k[NR], v[NR]; int bytes; };
    auto words_of = [&](const Pages& pg) __attribute__((always_inline)) {
        ScaleWords r{};
#pragma unroll
        for (int j = 0; j < NR; ++j) {
            const int id = page_of(pg, block_of(j));
            const int64_t sc = (int64_t)(is_there(id) ? id : 0) * p.Hkv + g;
            const uintptr_t ka = (uintptr_t)(p.c.k_scales + sc), va = (uintptr_t)(p.c.v_scales + sc);
            r.k[j] = const_load((const uint32_t*)(ka & ~(uintptr_t)3));
            r.v[j] = const_load((const uint32_t*)(va & ~(uintptr_t)3));
            r.bytes |= ((int)(ka & 3) | (int)(va & 3) << 2) << 4 * j;
        }
        return r;
    };
    auto bytes_of = [&](const ScaleWords& x) __attribute__((always_inline)) {
        Scales r;
#pragma unroll
        for (int j = 0; j < NR; ++j) {
            r.k[j] = x.k[j] >> 8 * (x.bytes >> 4 * j & 3) & 255u;
            r.v[j] = x.v[j] >> 8 * (x.bytes >> (4 * j + 2) & 3) & 255u;
        }
        return r;
    };
    // The same (SHARED) of K (kv 0) or V (1) alone, read and stored at different places.
    struct Half { u32x4 x[NR]; };
    auto read_half = [&](uint32_t raw, int kv, Half& r) __attribute__((always_inline)) {
        for_range<0, NR>([&](auto j_tag) __attribute__((always_inline)) {
            constexpr int j = decltype(j_tag)::value;
            r.x[j] = __builtin_bit_cast(u32x4, kv == 0 ? lds_read_b128(raw + 16 * lane, 2 * j * 1024) : lds_read_b128(raw + 16 * lane, (2 * j + 1) * 1024));
        });
    };
    auto store_half = [&](int kt, int there, int stage, int kv, Half& from) __attribute__((always_inline)) {
        int ln = lane;
        asm volatile("" : "+v"(ln));   // (as below)
        const int row_in = ln / (D / 16), gr = 2 * (ln % (D / 16)), row_w = w * RPI8 + row_in;
        const uint32_t base = lds_addr(lds) + stage * STAGE_BYTES + row_w * RB;
        const uint32_t to = kv == 0 ? base + 16 * (gr ^ GEO::swz_k(row_w)) : base + GEO::TILE_BYTES + 16 * (gr ^ GEO::swz_v(row_w));
        for_range<0, NR>([&](auto j_tag) __attribute__((always_inline)) {
            constexpr int j = decltype(j_tag)::value, AT = j * NW * RPI8 * RB;
            s16x8 x[2];
            float scale = scale_value(kv == 0 ? scales.k[j] : scales.v[j]);
            if (kv == 1) {   // (V of no row, and the scale of no page, are not multiplied)
                const bool on = (there >> block_of(j) & 1) && kt * KEYS + j * NW * RPI8 + row_w < ctx;
                scale = on ? scale : 1.f;
#pragma unroll
                for (int e = 0; e < 4; ++e) from.x[j][e] = on ? from.x[j][e] : 0u;
            }
            widen16<T>(from.x[j], scale, x);
            lds_write_b128(to, AT, x[0]);
            lds_write_b128(to ^ 16u, AT, x[1]);
        });
    };
    auto widen_tile = [&](int kt, int there, int stage, uint32_t raw) __attribute__((always_inline)) {
        // (the lane's places are worked out for every tile: ten instructions; kept across tiles they do not fit the registers at D = 128)
        int ln = lane;
        asm volatile("" : "+v"(ln));
        const int row_in = ln / (D / 16), gr = 2 * (ln % (D / 16)), row_w = w * RPI8 + row_in;   // row of load 0; the swizzles repeat every 16 rows
        const uint32_t base = lds_addr(lds) + stage * STAGE_BYTES + row_w * RB;
        const uint32_t k_to = base + 16 * (gr ^ GEO::swz_k(row_w)), v_to = base + GEO::TILE_BYTES + 16 * (gr ^ GEO::swz_v(row_w));
        static_assert((NW * RPI8) % 16 == 0 && GEO::TILE_BYTES % 32 == 0, "granule gr + 1 is at the address of gr with bit 4 turned");
        for_range<0, NR>([&](auto j_tag) __attribute__((always_inline)) {
            constexpr int j = decltype(j_tag)::value, AT = j * NW * RPI8 * RB;
            const bool on = (there >> block_of(j) & 1) && kt * KEYS + j * NW * RPI8 + row_w < ctx;
            s16x8 x[2];
            widen16<T>(__builtin_bit_cast(u32x4, lds_read_b128(raw + 16 * ln, 2 * j * 1024)), scale_value(scales.k[j]), x);
            lds_write_b128(k_to, AT, x[0]);
            lds_write_b128(k_to ^ 16u, AT, x[1]);
            widen16<T>(__builtin_bit_cast(u32x4, lds_read_b128(raw + 16 * ln, (2 * j + 1) * 1024)), scale_value(scales.v[j]), x);
            lds_write_b128(v_to, AT, on ? x[0] : s16x8{0, 0, 0, 0, 0, 0, 0, 0});
            lds_write_b128(v_to ^ 16u, AT, on ? x[1] : s16x8{0, 0, 0, 0, 0, 0, 0, 0});
        });
        // the area's reads have returned before the next codes are sent there
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    };

    // ---- per-lane LDS read addresses (stage 0; the other stage and the row blocks are immediates) ----
    uint32_t k_rd[KC], v_rd[DB];
    {
        const int sw = GEO::swz_k(l16);
#pragma unroll
        for (int c = 0; c < KC; ++c) k_rd[c] = lds_addr(lds) + l16 * RB + 16 * ((4 * c + quad) ^ sw);
        const int vrow = 4 * quad + (l16 >> 2), swv = GEO::swz_v(vrow);
#pragma unroll
        for (int db = 0; db < DB; ++db) {
            const int dcol = 16 * db + 4 * (l16 & 3);
            v_rd[db] = lds_addr(lds + GEO::TILE_BYTES) + vrow * RB + 16 * ((dcol >> 3) ^ swv) + 2 * (dcol & 7);
        }
    }

    f32x4 o_acc[DB][2];
#pragma unroll
    for (int db = 0; db < DB; ++db)
#pragma unroll
        for (int qb = 0; qb < 2; ++qb) o_acc[db][qb] = f32x4{0.f, 0.f, 0.f, 0.f};
    // reference exponent of the lane's two rows (log2 units, -inf until a key has been seen), moved only when an exponent exceeds it by
    // more than kLazyLog2, so that weights stay below 2^kLazyLog2; its negative (0 while there is none), the score from which
    // on it moves, and the lane's share of the denominators
    float m_ref[2] = {-INFINITY, -INFINITY}, neg_ref[2] = {0.f, 0.f}, grow_at[2] = {-INFINITY, -INFINITY}, l_sum[2] = {0.f, 0.f};
    constexpr float kLazyLog2 = 8.f;
    const float c2 = p.scale_log2, inv_c2 = p.inv_scale_log2;
    s16x8 qf[2][KC];
    int by_key = 0x7fffffff;   // the tile from which on the wave's keys are taken one by one

    // `beside(i)`, i = 0, 1, 2: what is done between the products with V
    auto process_tile = [&](auto stage_tag, int kt, int there, auto beside) __attribute__((always_inline)) {
        constexpr int SOFF = decltype(stage_tag)::value * STAGE_BYTES;
        const int key0 = kt * KEYS;
        auto pin = [&]() __attribute__((always_inline)) { __builtin_amdgcn_sched_barrier(0); };
        auto read_v = [&](int ck, int db) __attribute__((always_inline)) -> s16x8 {
            const s16x4 t0 = lds_read_tr16(v_rd[db], SOFF + (32 * ck) * RB), t1 = lds_read_tr16(v_rd[db], SOFF + (32 * ck + 16) * RB);
            return s16x8{t0[0], t0[1], t0[2], t0[3], t1[0], t1[1], t1[2], t1[3]};
        };
        s16x8 va[DB];
        // S^T = K Q^T: register e of block [kb][qb] is key 16kb + 4 quad + e of row 16qb + l16
        f32x4 e_acc[NB][2];
        {
            s16x8 kf[2][NB];
#pragma unroll
            for (int c = 0; c < 2 && c < KC; ++c)
#pragma unroll
                for (int kb = 0; kb < NB; ++kb) kf[c][kb] = lds_read_b128(k_rd[c], SOFF + 16 * kb * RB);
            pin();
            for_range<0, KC * NB>([&](auto i_tag) __attribute__((always_inline)) {
                constexpr int i = decltype(i_tag)::value, c = i / NB, kb = i % NB;
#pragma unroll
                for (int qb = 0; qb < 2; ++qb) e_acc[kb][qb] = T::mfma16(kf[c & 1][kb], qf[qb][c], c == 0 ? f32x4{0.f, 0.f, 0.f, 0.f} : e_acc[kb][qb]);
                pin();
                if (c + 2 < KC) {
                    kf[c & 1][kb] = lds_read_b128(k_rd[c + 2], SOFF + 16 * kb * RB);
                } else if (c + 1 == KC) {
#pragma unroll
                    for (int db = kb * (DB / NB); db < (kb + 1) * (DB / NB); ++db) va[db] = read_v(0, db);
                }
                pin();
            });
        }
        if (key0 + KEYS - 1 > wave_first) {
            // V rows that some of the wave's tokens attend and others do not: whether all are finite is what products with zero say
            f32x4 probe = {0.f, 0.f, 0.f, 0.f};
            const s16x8 zero = {0, 0, 0, 0, 0, 0, 0, 0};
#pragma unroll
            for (int db = 0; db < DB; ++db) {
                probe = T::mfma16(va[db], zero, probe);
                if (NB == 4) probe = T::mfma16(read_v(1, db), zero, probe);
            }
            if (__any(!(probe[0] + probe[1] + probe[2] + probe[3] == 0.f))) {
                by_key = kt;
#pragma unroll
                for (int i = 0; i < 3; ++i) beside(i);
                return;
            }
        }
        if (key0 + KEYS - 1 > wave_first || !whole(kt, there)) {
#pragma unroll
            for (int qb = 0; qb < 2; ++qb) {
                const int lim = pos[qb] - key0 - 4 * quad;   // largest kept 16kb + e
#pragma unroll
                for (int kb = 0; kb < NB; ++kb) {
                    const int lim_kb = there >> kb & 1 ? lim : -1;
#pragma unroll
                    for (int e = 0; e < 4; ++e) e_acc[kb][qb][e] = 16 * kb + e <= lim_kb ? e_acc[kb][qb][e] : -INFINITY;
                }
            }
        }
        {
            float mx[2];
#pragma unroll
            for (int qb = 0; qb < 2; ++qb) {
                float m = max3(e_acc[0][qb][0], e_acc[0][qb][1], e_acc[0][qb][2]);
                m = max3(m, e_acc[0][qb][3], e_acc[1][qb][0]);
#pragma unroll
                for (int kb = 1; kb < NB; ++kb) {
                    m = max3(m, e_acc[kb][qb][1], e_acc[kb][qb][2]);
                    m = kb < NB - 1 ? max3(m, e_acc[kb][qb][3], e_acc[(kb + 1) % NB][qb][0]) : max2(m, e_acc[kb][qb][3]);
                }
                mx[qb] = m;
            }
            if (__any(mx[0] > grow_at[0] || mx[1] > grow_at[1])) {
                mx[0] = max_across_quads(mx[0]);
                mx[1] = max_across_quads(mx[1]);
#pragma unroll
                for (int qb = 0; qb < 2; ++qb) {
                    const float m_new = mx[qb] > grow_at[qb] ? mx[qb] * c2 : m_ref[qb];
                    const float alpha = (m_ref[qb] == -INFINITY) ? 0.f : fast_exp2(m_ref[qb] - m_new);
                    m_ref[qb] = m_new;
                    neg_ref[qb] = (m_new == -INFINITY) ? 0.f : -m_new;
                    grow_at[qb] = (m_new + kLazyLog2) * inv_c2;
                    l_sum[qb] *= alpha;
#pragma unroll
                    for (int db = 0; db < DB; ++db)
#pragma unroll
                        for (int e = 0; e < 4; ++e) o_acc[db][qb][e] *= alpha;
                }
            }
        }
        // P = 2^E and O^T += V^T P^T, 32 keys and 16 rows at a time, the next weights made between the MFMAs of the current ones.  The weights are rounded to the
        // 16-bit type, since an MFMA takes both operands in one type and V is there in that: error against 64 bits 2.5e-4 (f16) and 2.2e-3 (bf16) of the output's scale, of
        // which the output's own rounding makes 2.0e-4 and 1.7e-3.  What the rounding leaves as a second operand would be half as many MFMAs again.
        float ls[2] = {0.f, 0.f};
        auto weights_quarter = [&](int ck, int qb, int i) __attribute__((always_inline)) -> uint32_t {
            const int kb = 2 * ck + (i >> 1), r = 2 * (i & 1);
            const uint32_t pk = T::pack2(fast_exp2(__builtin_fmaf(e_acc[kb][qb][r], c2, neg_ref[qb])), fast_exp2(__builtin_fmaf(e_acc[kb][qb][r + 1], c2, neg_ref[qb])));
            ls[qb] = T::add_pair(pk, ls[qb]);   // the denominator sums the rounded weights the MFMA uses
            asm volatile("" : "+v"(ls[qb]));
            return pk;
        };
        uint32_t pw[2][4];
#pragma unroll
        for (int i = 0; i < 4; ++i) pw[0][i] = weights_quarter(0, 0, i);
        pin();
#pragma unroll
        for (int s = 0; s < NB; ++s) {
            const int ck = s >> 1, qb = s & 1;
            const s16x8 pcur = __builtin_bit_cast(s16x8, u32x4{pw[s & 1][0], pw[s & 1][1], pw[s & 1][2], pw[s & 1][3]});
#pragma unroll
            for (int db = 0; db < DB; ++db) {
                o_acc[db][qb] = T::mfma16(va[db], pcur, o_acc[db][qb]);
                pin();
                if (qb == 1 && ck + 1 < NB / 2) va[db] = read_v(1, db);
                if (s + 1 < NB && db < 4) pw[(s + 1) & 1][db] = weights_quarter((s + 1) >> 1, (s + 1) & 1, db);
                pin();
            }
            if (s < 3) beside(s);
        }
        l_sum[0] += ls[0];
        l_sum[1] += ls[1];
    };

    // ---- main loop: one barrier per tile, the rows of the next ones on their way under it ----
    auto read_queries = [&]() __attribute__((always_inline)) {
        const uint32_t qa = lds_addr(q_stage) + l16 * RB;
        const int sw = GEO::swz_k(l16);
#pragma unroll
        for (int qb = 0; qb < 2; ++qb)
#pragma unroll
            for (int c = 0; c < KC; ++c) qf[qb][c] = lds_read_b128(qa + 16 * ((4 * c + quad) ^ sw), 16 * qb * RB);
    };
    auto pin_pages = [&](Pages& x) __attribute__((always_inline)) {
#pragma unroll
        for (int b = 0; b < NB; ++b) asm volatile("" : "+s"(x.id[b]));
    };
    if constexpr (!SHARED) {
        Pages pg{};                   // of the next tile to be requested
        int there = 0, there_1 = 0;   // pages of the tile at work and of the one behind it
        if (n_own > 0) {
            pg = pages_of(t_lo);
            there = there_of(pg);
            if (FP8) { request_codes(t_lo, pg, raw0); scales = scales_of(pg); }
            else copy_tile(t_lo, pg, std::integral_constant<int, 0>{}, dst0);
            pg = pages_of(t_lo + 1);
        }
        // the query rows were requested first
        if (!FP8 && n_own > 0) wait_vmcnt<2 * NLD>(); else wait_vmcnt<0>();
        read_queries();
        if (FP8 && n_own > 0) {
            widen_tile(t_lo, there, 0, raw0);
            if (n_own > 1) { request_codes(t_lo + 1, pg, raw0); scales = scales_of(pg); }
            there_1 = there_of(pg);
            pg = pages_of(t_lo + 2);
        }
        auto iteration = [&](auto stage_tag, int it) {
            constexpr int STAGE = decltype(stage_tag)::value;
            const int kt = t_lo + it;
            int there_2 = 0;
            // The table's entries, and the scales of codes about to be sent for, are asked for here and waited for in front of the barrier, where the wave
            // waits anyway: scalar loads return in no order, so that with one on its way every wait for an LDS read is one for all of them.
            Pages after = pages_of(FP8 ? kt + 3 : kt + 2);
            Scales scales_2{};
            if (FP8) scales_2 = scales_of(pg);
            if (!FP8) {
                wait_vmcnt<0>();       // this wave's share of the tile has landed
                if (!whole(kt, there)) clear_rows(kt, there, STAGE);
            }
            pin_pages(after);
            if (FP8) {
    #pragma unroll
                for (int j = 0; j < NR; ++j) asm volatile("" : "+s"(scales_2.k[j]), "+s"(scales_2.v[j]));
            }
            __syncthreads();           // everyone's has; the other stage is no longer being read
            if (it + 1 < n_own) {
                if (FP8) {
                    wait_vmcnt<0>();   // the wave's codes of the next tile have
                    widen_tile(kt + 1, there_1, STAGE ^ 1, raw0);
                    if (it + 2 < n_own) request_codes(kt + 2, pg, raw0);
                    there_2 = there_of(pg);
                    scales = scales_2;
                } else {
                    copy_tile(kt + 1, pg, std::integral_constant<int, STAGE ^ 1>{}, dst0);
                    there_1 = there_of(pg);
                }
                pg = after;
            }
            if (wave_on && there && kt * KEYS <= wave_last && kt < by_key) process_tile(stage_tag, kt, there, [](int) {});
            there = there_1;
            there_1 = there_2;
        };
        for (int it = 0; it < n_own; it += 2) {
            iteration(std::integral_constant<int, 0>{}, it);
            if (it + 1 < n_own) iteration(std::integral_constant<int, 1>{}, it + 1);
        }
    } else {
        constexpr int RING = LDS::RING, STAGES = LDS::STAGES, LOADS = FP8 ? 2 * NR : 2 * NLD;   // a wave's copies of a tile
        // until all but the last `tiles` tiles of those that the wave asked for are there
        auto wait_but = [&](int tiles) __attribute__((always_inline)) {
            static_assert(3 * LOADS < 64, "counted by six bits");
            if (tiles >= 3) wait_vmcnt<3 * LOADS>(); else if (tiles == 2) wait_vmcnt<2 * LOADS>(); else if (tiles == 1) wait_vmcnt<LOADS>(); else wait_vmcnt<0>();
        };
        // (on to the next stage: the addresses, not the code, go round the ring)
        auto next_stage = [&](int it) __attribute__((always_inline)) {
            const uint32_t step = (it & (STAGES - 1)) == STAGES - 1 ? (uint32_t)(-(STAGES - 1) * STAGE_BYTES) : (uint32_t)STAGE_BYTES;
#pragma unroll
            for (int c = 0; c < KC; ++c) k_rd[c] += step;
#pragma unroll
            for (int db = 0; db < DB; ++db) v_rd[db] += step;
        };
        const std::integral_constant<int, 0> zero{};
        Pages pg = next3[0], pg1 = next3[1];
        const Pages pg2 = next3[2];
        int theres = there_of(pg) | there_of(pg1) << NB;   // pages that are there, NB bits a tile: of the tile at work and those behind it
        if constexpr (!FP8) {
            if (n_own > 0) copy_tile(t_lo, pg, zero, dst0);
            if (n_own > 1) copy_tile(t_lo + 1, pg1, zero, dst0 + STAGE_BYTES);
            wait_but(min(n_own, 2));   // the query rows were requested first
            read_queries();
            __syncthreads();           // everyone's are read, out of the stages of the next tiles
            if (n_own > 2) copy_tile(t_lo + 2, pg2, zero, dst0 + 2 * STAGE_BYTES);
            theres |= there_of(pg2) << 2 * NB;
            pg = pages_of(t_lo + 3);
            for (int it = 0; it < n_own; ++it) {
                const int kt = t_lo + it, there = theres & ((1 << NB) - 1);
                Pages after = pages_of(kt + 4);
                wait_but(min(n_own - 1 - it, 2));   // this wave's share of the tile has landed
                if (!whole(kt, there)) clear_rows(kt, there, it & (STAGES - 1));
                pin_pages(after);
                __syncthreads();                    // everyone's has; the stage of the tile in front is no longer being read
                if (it + 3 < n_own) copy_tile(kt + 3, pg, zero, dst0 + ((it + 3) & (STAGES - 1)) * STAGE_BYTES);
                theres = theres >> NB | there_of(pg) << 2 * NB;
                pg = after;
                if (wave_on && there && kt * KEYS <= wave_last && kt < by_key) process_tile(zero, kt, there, [](int) {});
                next_stage(it);
            }
        } else {
            constexpr int AREA = LDS::RAW_BYTES;
            if (n_own > 0) request_codes(t_lo, pg, raw0);
            if (n_own > 1) request_codes(t_lo + 1, pg1, raw0 + AREA);
            if (n_own > 2) request_codes(t_lo + 2, pg2, raw0 + 2 * AREA);
            scales = scales_of(pg);
            Scales scales_1 = scales_of(pg1);
            pg = pages_of(t_lo + 3);
            pg1 = pg2;                 // of the tile whose scales are asked for next
            wait_but(min(n_own, 3));
            read_queries();
            __syncthreads();
            if (n_own > 3) request_codes(t_lo + 3, pg, raw0 + 3 * AREA);
            if (n_own > 0) {
                wait_but(min(n_own - 1, 3));
#pragma unroll
                for (int kv = 0; kv < 2; ++kv) {
                    Half half;
                    read_half(raw0, kv, half);
                    store_half(t_lo, theres & ((1 << NB) - 1), 0, kv, half);
                }
            }
            scales = scales_1;
            pg = pages_of(t_lo + 4);
            for (int it = 0; it < n_own; ++it) {
                const int kt = t_lo + it, there = theres & ((1 << NB) - 1);
                // the table's entries, the scales and the codes are asked for together: one wait
                Pages after = pages_of(kt + 5), after_1 = pages_of(kt + 3);
                ScaleWords words = words_of(pg1);
                __builtin_amdgcn_sched_barrier(0);
                pin_pages(after);
                pin_pages(after_1);
#pragma unroll
                for (int j = 0; j < NR; ++j) asm volatile("" : "+s"(words.k[j]), "+s"(words.v[j]));
                scales_1 = bytes_of(words);
                __syncthreads();       // everyone's share of the tile is widened; the other stage is no longer being read
                theres = theres >> NB | there_of(pg1) << NB;
                if (it + 4 < n_own) request_codes(kt + 4, pg, raw0 + (it & (RING - 1)) * AREA);
                // the next tile's codes, K's and V's one after the other (behind the last tile: what the area holds, into a stage that nobody reads)
                const uint32_t area = raw0 + ((it + 1) & (RING - 1)) * AREA;
                Half half;
                auto next_tile = [&](int i) __attribute__((always_inline)) {
                    if (i == 0) {
                        wait_but(min(n_own - 2 - it, 3));   // the wave's codes of the next tile have landed
                        read_half(area, 0, half);
                    } else {
                        store_half(kt + 1, theres & ((1 << NB) - 1), (it + 1) & 1, i - 1, half);
                        if (i == 1) read_half(area, 1, half);
                    }
                };
                if (wave_on && there && kt * KEYS <= wave_last && kt < by_key) process_tile(zero, kt, there, next_tile);
                else
                    for (int i = 0; i < 3; ++i) next_tile(i);
                scales = scales_1;
                pg = after;
                pg1 = after_1;
                next_stage(it);
            }
        }
    }

    if (!wave_on) return;
    if (by_key < t_lo + n_own) {
        const short* q[2];
        const int limit[2] = {pos[0] + 1, pos[1] + 1};
#pragma unroll
        for (int qb = 0; qb < 2; ++qb) {
            const int r = min(row0 + 16 * qb + l16, last_row), t = r / p.n_rep;
            q[qb] = (const short*)p.q + (int64_t)(job.lo + t) * p.q2 + (int64_t)(g * p.n_rep + r - t * p.n_rep) * p.q1;
        }
        attend_key_by_key<T, D, FP8, 2>(p.c, p.Hkv, seq, g, by_key * KEYS, min(wave_last + 1, (t_lo + n_own) * KEYS), q, limit, c2,
                                        [&](int db, int qb) __attribute__((always_inline)) -> f32x4& { return o_acc[db][qb]; }, m_ref, l_sum);
    }
    float l_all[2];
#pragma unroll
    for (int qb = 0; qb < 2; ++qb) l_all[qb] = sum_across_quads(l_sum[qb]);
    if (SHARED || job.parts > 1) {
        const int64_t part = SHARED ? (int64_t)job.slot : ((int64_t)job.slot * p.Hkv + g) * BR;
#pragma unroll
        for (int qb = 0; qb < 2; ++qb) {
            if (row0 + 16 * qb + l16 > last_row) continue;
            const int64_t slot = part + w * 32 + 16 * qb + l16;
            float* dst = p.part_o + slot * D + 4 * quad;
#pragma unroll
            for (int db = 0; db < DB; ++db) *reinterpret_cast<f32x4*>(dst + 16 * db) = o_acc[db][qb];
            if (quad == 0) { p.part_ml[slot * 2] = m_ref[qb]; p.part_ml[slot * 2 + 1] = l_all[qb]; }
        }
        return;
    }
    // normalised rows through LDS, so that a store instruction writes whole rows
    const uint32_t so = kAliasRows ? lds_addr(lds) + (n_own & 1) * STAGE_BYTES + w * ROWS_BYTES : lds_addr(q_stage);
    typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
    typedef __attribute__((address_space(3))) u32x2 lds_u32x2;
    wave_lds_order();
#pragma unroll
    for (int qb = 0; qb < 2; ++qb) {
        const float inv = l_all[qb] > 0.f ? 1.f / l_all[qb] : 0.f;
#pragma unroll
        for (int db = 0; db < DB; ++db) {
            u32x2 pk;
            pk.x = T::pack2(o_acc[db][qb][0] * inv, o_acc[db][qb][1] * inv);
            pk.y = T::pack2(o_acc[db][qb][2] * inv, o_acc[db][qb][3] * inv);
            const int row = 16 * qb + l16, gi = 2 * db + (quad >> 1);
            *(lds_u32x2*)(uintptr_t)(so + row * RB + 16 * (gi ^ (row & (G - 1))) + 8 * (quad & 1)) = pk;
        }
    }
    wave_lds_order();
#pragma unroll
    for (int i = 0; i < 32 / RPI; ++i) {
        const int row = i * RPI + lane / G, r = row0 + row, gi = lane % G;
        const s16x8 val = lds_read_b128(so + row * RB + 16 * (gi ^ (row & (G - 1))), 0);
        if (r <= last_row) {
            const int t = r / p.n_rep;
            *reinterpret_cast<s16x8*>((short*)p.out + (int64_t)(job.lo + t) * p.o2 + (int64_t)(g * p.n_rep + r - t * p.n_rep) * p.o1 + 8 * gi) = val;
        }
    }
}

}  // namespace minfer_attn
