// Attention of packed tokens over a paged KV cache for gfx950: chunks of prompts, drafts and single tokens.
//
// Rows.  The new tokens of a sequence and the query heads of a KV head's group are one list of rows, token by token, heads innermost
// (row = token * n_rep + head): whatever the group's size, 32 rows of a wave attend one KV head, and a sequence of a few tokens
// fills its rows with heads.  A workgroup takes NW * 32 rows and walks the sequence's 64-key tiles up to its last row's position;
// where that makes few workgroups the tiles of a long sequence's blocks are cut into pieces with a workgroup each (find_piece), which
// leave un-normalised sums in the workspace for paged_combine_kernel.
//
// Per tile a wave computes S^T = K Q^T and O^T += V^T P^T with v_mfma_f32_16x16x32, the scores staying in registers as the second
// product's operand; tiles are double-buffered in LDS, 16-bit rows copied there directly, 8-bit codes through registers, in which
// they become 16-bit values (exactly: a scale is a power of two).  A tile's rows come from up to four pages, looked up a tile ahead
// as scalars: pages have at least 16 rows, so a copy instruction's rows lie in one.
//
// Rows that nothing was written to, behind the context in its last page, and rows of pages that are not there may hold NaN, which a weight of zero would
// not take out of a sum: their scores are replaced, and their V rows are cleared in LDS, in the few tiles that have any.  A row with an infinity or a NaN
// that a sequence's later tokens attend is kept from its earlier ones as well (attend_key_by_key).
#include <algorithm>

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

// The first 64-key tile of a sequence with a page that is there (its number of tiles if there is none): a window that moved on has given the pages
// in front of it back.  Looked for only where the first page is missing, 64 pages at a time; the whole wave.
MA_DEV int first_tile(const PagedCache& c, int seq, int ctx) {
    const int32_t* table = c.table + (int64_t)seq * c.table_stride;
    const int lane = threadIdx.x & 63, n = (ctx + (1 << c.page_log2) - 1) >> c.page_log2;
    for (int base = 0; base < n; base += 64) {
        const int i = base + lane;
        const uint64_t hit = __ballot(i < n && (unsigned)table[min(i, n - 1)] < (unsigned)c.n_pages);
        if (hit) return ((base + __ffsll((unsigned long long)hit) - 1) << c.page_log2) >> 6;
    }
    return (ctx + 63) >> 6;
}

MA_DEV int tiles_of(int pos0, int rows, int n_rep, int block, int BR) { return (max(pos0 + min(block * BR + BR - 1, rows - 1) / n_rep + 1, 0) + 63) >> 6; }

// What a workgroup does: the `part`-th of `parts` equal pieces of the tiles of a block of rows (NW * 32 of them); piece `x` of the launch.
struct Piece { int seq, block, part, parts; };

// The x-th piece (seq < 0: there is none) and, with it, how many there are.  The blocks of a sequence are cut into the same number of pieces, its last
// block's tiles over a size that is the same for all sequences: the smallest that leaves no more pieces than workgroups which the chip
// holds at once (p.round, or a multiple of it where the blocks alone are more).  Every wave works it out for itself, a sequence to a lane: with sums over
// all blocks in LDS it took 14 us in front of a launch's first tile, this 1.
template <int BR> MA_DEV Piece find_piece(const PagedParams& p, int x, int& all) {
    const int lane = threadIdx.x & 63;
    Piece r{-1, 0, 0, 1};
    if (p.round == 0) {   // whole blocks, of any number of sequences
        all = 0;
        for (int base = 0; base < p.n_seqs; base += 64) {
            TokenRange t{0, 0, 0};
            if (base + lane < p.n_seqs) t = token_range(p.cu[base + lane], p.cu[base + lane + 1], p.T);
            const int n = (min(t.len, p.max_q) * p.n_rep + BR - 1) / BR;
            const int incl = wave_inclusive_scan(n), total = lane_value(incl, 63);
            if (x < total) {
                const int s = __builtin_amdgcn_readfirstlane(__ffsll((unsigned long long)__ballot(x < incl)) - 1);
                r.seq = base + s;
                r.block = lane_value(n, s) - 1 - (x - lane_value(incl - n, s));   // most keys first
                return r;
            }
            x -= total;
        }
        return r;
    }
    int n = 0, tiles = 0;   // the lane's sequence: blocks, tiles of the last one
    if (lane < p.n_seqs) {
        const TokenRange t = token_range(p.cu[lane], p.cu[lane + 1], p.T);
        const int ctx = context_of(p.c, p.ctx[lane], t), rows = min(t.len, p.max_q) * p.n_rep;
        n = (rows + BR - 1) / BR;
        tiles = n > 0 ? max(tiles_of(ctx - t.len, rows, p.n_rep, n - 1, BR), 1) : 0;
        // (a window that moved on: half of the pages, a guess, which only the number of pieces goes by)
        if (n > 0 && ctx > 0 && (unsigned)p.c.table[(int64_t)lane * p.c.table_stride] >= (unsigned)p.c.n_pages) tiles = (tiles + 1) / 2;
    }
    const int blocks = lane_value(wave_inclusive_scan(n), 63), most = (blocks + p.round - 1) / p.round * p.round;
    const float sum = lane_sum<64>((float)n * (float)tiles);
    constexpr int kLeastTiles = 4;
    int size = max((int)(sum / (float)max(most, 1)), kLeastTiles), parts, incl;
    for (;; size += 1 + size / 8) {   // (ends: with the most tiles of a sequence as the size there is a piece for every block, and `most` is no less)
        parts = (tiles + size - 1) / size;
        incl = wave_inclusive_scan(n * parts);
        all = lane_value(incl, 63);
        if (all <= most) break;
    }
    if (x >= all) return r;
    r.seq = __builtin_amdgcn_readfirstlane(__ffsll((unsigned long long)__ballot(x < incl)) - 1);
    r.parts = lane_value(parts, r.seq);
    const int blocks_of = lane_value(n, r.seq), local = x - (lane_value(incl, r.seq) - blocks_of * r.parts);
    r.block = blocks_of - 1 - local / r.parts;
    r.part = local % r.parts;
    return r;
}

// Bound by the matrix unit with the exponentials and, over codes, the widening between its instructions.  A prompt of 8192, 32 query heads on 8 of 128, f16:
// 515 us, 1067 TFLOP/s, nine tenths of what a library product of 8192^3 reaches; 4 chunks, 1257 tokens to 13795 rows, 24 heads on 8, bf16: 66 us, 774; 2 chunks,
// 1778 tokens to 12315 rows of codes, 64 heads on 8, a window that moved on: 226 us, 804.  Prompts of 512 and 1024 take 17 and 28: 5 us and 1.4 a tile.
template <class T, int D, bool FP8, int NW>
__global__ __launch_bounds__(NW * 64, 2) void paged_tile_kernel(const PagedParams p) {
    using GEO = PagedGeom<D, NW>;
    constexpr int RB = GEO::RB, G = GEO::G, RPI = GEO::RPI, NLD = GEO::NLD;
    constexpr int KC = D / 32;   // 32-wide contraction chunks of Q K^T
    constexpr int DB = D / 16;   // 16-row blocks of O^T
    constexpr int BR = NW * 32;  // rows of a workgroup
    constexpr int STAGE_BYTES = 2 * GEO::TILE_BYTES;   // the K tile followed by the V tile
    constexpr int ROWS_BYTES = 32 * RB;
    // The waves' query rows on their way in and output rows on their way out: with four waves inside a stage (the query rows in stage 1, which no
    // tile touches before the barrier of tile 0; the output rows in the stage that the last tile did not use), with eight beside them.
    constexpr bool kAliasRows = NW * ROWS_BYTES <= STAGE_BYTES;
    __shared__ __attribute__((aligned(1024))) char kv_lds[2][STAGE_BYTES];
    __shared__ __attribute__((aligned(1024))) char rows_lds[kAliasRows ? 1 : NW][kAliasRows ? 16 : ROWS_BYTES];

    const int lane = threadIdx.x & 63, w = wave_id();
    const int l16 = lane & 15, quad = lane >> 4;

    // ---- which KV head, range of tiles and block of rows; a KV head's workgroups on one XCD (ids go round-robin) ----
    int g, rank;
    if ((p.Hkv & 7) == 0) {
        const int per = p.Hkv >> 3, m = (int)blockIdx.x >> 3;
        g = (m % per) * 8 + ((int)blockIdx.x & 7);
        rank = m / per;
    } else {
        g = (int)blockIdx.x % p.Hkv;
        rank = (int)blockIdx.x / p.Hkv;
    }
    int all;
    const Piece me = find_piece<BR>(p, rank, all);
    if (p.round > 0 && blockIdx.x == 0 && threadIdx.x == 0) p.table[0] = all;   // for the combine kernel (of no sequences, too)
    if (me.seq < 0) return;
    const int seq = me.seq, block = me.block;
    if (p.round > 0 && g == 0 && threadIdx.x == 0) reinterpret_cast<int4*>(p.table)[1 + rank] = make_int4(me.seq, me.block, me.part, me.parts);
    const TokenRange range = token_range(const_load(p.cu + seq), const_load(p.cu + seq + 1), p.T);
    const int seq_lo = range.lo, seq_len = range.len;
    const int ctx = context_of(p.c, const_load(p.ctx + seq), range);
    const int pos0 = ctx - seq_len;                                      // position of the sequence's token 0
    const int rows = min(seq_len, p.max_q) * p.n_rep, last_row = rows - 1;
    const int row0 = block * BR + w * 32;                                // the wave's first row
    const bool wave_on = row0 < rows;
    const int tiles = tiles_of(pos0, rows, p.n_rep, block, BR);
    int t_first = 0;
    if (tiles > 0 && (unsigned)const_load(p.c.table + (int64_t)seq * p.c.table_stride) >= (unsigned)p.c.n_pages)
        t_first = __builtin_amdgcn_readfirstlane(first_tile(p.c, seq, ctx));
    const int n_tiles = max(tiles - t_first, 0), each = n_tiles / me.parts, longer = n_tiles - each * me.parts;
    const int t_lo = t_first + me.part * each + min(me.part, longer), n_own = each + (me.part < longer ? 1 : 0);
    const int wave_first = pos0 + min(row0, last_row) / p.n_rep, wave_last = pos0 + min(row0 + 31, last_row) / p.n_rep;

    // positions of the lane's two rows (one per block of 16)
    const int pos[2] = {pos0 + min(row0 + l16, last_row) / p.n_rep, pos0 + min(row0 + 16 + l16, last_row) / p.n_rep};

    // ---- the wave's query rows, copied global->LDS as whole rows ----
    char* const q_stage = kAliasRows ? &kv_lds[1][w * ROWS_BYTES] : &rows_lds[kAliasRows ? 0 : w][0];
#pragma unroll
    for (int j = 0; j < 32 / RPI; ++j) {
        const int row = j * RPI + lane / G, r = min(row0 + row, last_row), t = r / p.n_rep;
        const short* src = (const short*)p.q + (int64_t)(seq_lo + t) * p.q2 + (int64_t)(g * p.n_rep + r - t * p.n_rep) * p.q1 + 8 * ((lane % G) ^ GEO::swz_k(row));
        copy16_global_to_lds(src, q_stage + j * RPI * RB);
    }

    // ---- pages: the four 16-row blocks of a tile -----------------------------------------------------------------
    const int32_t* const table = p.c.table + (int64_t)seq * p.c.table_stride;
    struct Pages { int id[4]; };
    auto pages_of = [&](int kt) __attribute__((always_inline)) {
        Pages r;
#pragma unroll
        for (int b = 0; b < 4; ++b) r.id[b] = const_load(table + min((kt * 64 + 16 * b) >> p.c.page_log2, p.c.width - 1));
        return r;
    };
    auto is_there = [&](int id) __attribute__((always_inline)) { return (unsigned)id < (unsigned)p.c.n_pages; };
    // bit b: the page of the tile's block b is there
    auto there_of = [&](const Pages& pg) __attribute__((always_inline)) {
        return (is_there(pg.id[0]) ? 1 : 0) | (is_there(pg.id[1]) ? 2 : 0) | (is_there(pg.id[2]) ? 4 : 0) | (is_there(pg.id[3]) ? 8 : 0);
    };
    // whether all 64 rows of a tile exist and hold what was written to them
    auto whole = [&](int kt, int there) __attribute__((always_inline)) { return kt * 64 + 64 <= ctx && there == 15; };
    const int page_mask = (1 << p.c.page_log2) - 1;
    // rows first .. of tile kt, which lie in page `id`: their offset in a pool, in elements (a page that is not there: page 0, whose
    // rows are there to be read)
    auto rows_at = [&](int id, int key) __attribute__((always_inline)) -> int64_t {
        return (int64_t)(is_there(id) ? id : 0) * p.c.page_stride + (int64_t)g * p.c.head_stride + (int64_t)(key & page_mask) * p.c.row_stride;
    };

    const uint32_t dst0 = (uint32_t)__builtin_amdgcn_readfirstlane((int)(lds_addr(&kv_lds[0][0]) + w * 1024));
    // ---- 16-bit rows: global -> LDS.  Instruction j of the wave covers rows (j * NW + w) * RPI .. of the tile, all in one block of 16.
    uint32_t k_off = 0, v_off = 0;
    if (!FP8) {
        const int row_in = lane / G, row = w * RPI + row_in, gr = lane % G;
        k_off = (uint32_t)(row_in * (int)p.c.row_stride + 8 * (gr ^ GEO::swz_k(row))) * 2u;
        v_off = (uint32_t)(row_in * (int)p.c.row_stride + 8 * (gr ^ GEO::swz_v(row))) * 2u;
    }
    auto copy_tile = [&](int kt, const Pages& pg, auto stage_tag) __attribute__((always_inline)) {
        for_range<0, NLD>([&](auto j_tag) __attribute__((always_inline)) {
            constexpr int j = decltype(j_tag)::value, b0 = j * NW * RPI / 16;
            constexpr int AT = decltype(stage_tag)::value * STAGE_BYTES + j * NW * 1024;
            const int id = NW * RPI == 16 ? pg.id[b0] : (w * RPI < 16 ? pg.id[b0] : pg.id[(b0 + 1) & 3]);
            static_assert(NW * RPI == 16 || NW * RPI == 32, "a round of copies covers one or two blocks of 16 rows");
            const int64_t at = rows_at(id, kt * 64 + (j * NW + w) * RPI);
            copy16_global_to_lds_at<AT, true>((const short*)p.c.k + at, k_off, dst0);
            copy16_global_to_lds_at<AT + GEO::TILE_BYTES, true>((const short*)p.c.v + at, v_off, dst0);
        });
    };
    // V rows of a tile that nothing may be multiplied with: the wave clears those that it copied itself
    auto clear_rows = [&](int kt, int there, int stage) __attribute__((always_inline)) {
        for_range<0, NLD>([&](auto j_tag) __attribute__((always_inline)) {
            constexpr int j = decltype(j_tag)::value;
            const int row = (j * NW + w) * RPI + lane / G;
            if (kt * 64 + row >= ctx || !(there >> (row >> 4) & 1))
                *reinterpret_cast<u32x4*>(&kv_lds[stage][GEO::TILE_BYTES + (j * NW + w) * 1024 + 16 * lane]) = u32x4{0u, 0u, 0u, 0u};
        });
    };
    // ---- 8-bit rows: global -> the wave's own LDS area as they are, and from there through registers into a stage.  Load j of the wave covers
    // rows (j * NW + w) * RPI8 .., 8 or 16 of one block, 16 codes a lane, which the lane itself reads back.
    constexpr int NR = FP8 ? GEO::NLD8 : 1, RPI8 = GEO::RPI8;
    __shared__ __attribute__((aligned(1024))) char raw_lds[FP8 ? NW : 1][FP8 ? 2 * NR * 1024 : 16];
    const uint32_t raw0 = (uint32_t)__builtin_amdgcn_readfirstlane((int)lds_addr(&raw_lds[FP8 ? w : 0][0]));
    struct Scales { uint32_t k[NR], v[NR]; } scales{};   // of the tile in the raw area, as their bytes
    const uint32_t c_off = (uint32_t)((lane / (D / 16)) * (int)p.c.row_stride + 16 * (lane % (D / 16)));
    auto block_of = [&](int j) __attribute__((always_inline)) { return ((j * NW + w) * RPI8) >> 4; };
    auto request_codes = [&](int kt, const Pages& pg) __attribute__((always_inline)) {
        for_range<0, NR>([&](auto j_tag) __attribute__((always_inline)) {
            constexpr int j = decltype(j_tag)::value;
            const int b = block_of(j), id = b == 0 ? pg.id[0] : b == 1 ? pg.id[1] : b == 2 ? pg.id[2] : pg.id[3];
            const int64_t at = rows_at(id, kt * 64 + (j * NW + w) * RPI8);
            copy16_global_to_lds_at<2 * j * 1024, true>((const char*)p.c.k + at, c_off, raw0);
            copy16_global_to_lds_at<(2 * j + 1) * 1024, true>((const char*)p.c.v + at, c_off, raw0);
        });
    };
    auto scales_of = [&](const Pages& pg) __attribute__((always_inline)) {
        Scales r;
#pragma unroll
        for (int j = 0; j < NR; ++j) {
            const int b = block_of(j), id = b == 0 ? pg.id[0] : b == 1 ? pg.id[1] : b == 2 ? pg.id[2] : pg.id[3];
            const int64_t sc = (int64_t)(is_there(id) ? id : 0) * p.Hkv + g;
            r.k[j] = const_byte(p.c.k_scales + sc);
            r.v[j] = const_byte(p.c.v_scales + sc);
        }
        return r;
    };
    auto widen_tile = [&](int kt, int there, int stage) __attribute__((always_inline)) {
        // (the lane's places are worked out for every tile: ten instructions; kept across tiles they do not fit the registers at D = 128)
        int ln = lane;
        asm volatile("" : "+v"(ln));
        const int row_in = ln / (D / 16), gr = 2 * (ln % (D / 16)), row_w = w * RPI8 + row_in;   // row of load 0; the swizzles repeat every 16 rows
        const uint32_t base = lds_addr(&kv_lds[0][0]) + stage * STAGE_BYTES + row_w * RB;
        const uint32_t k_to = base + 16 * (gr ^ GEO::swz_k(row_w)), v_to = base + GEO::TILE_BYTES + 16 * (gr ^ GEO::swz_v(row_w));
        static_assert((NW * RPI8) % 16 == 0 && GEO::TILE_BYTES % 32 == 0, "granule gr + 1 is at the address of gr with bit 4 turned");
        for_range<0, NR>([&](auto j_tag) __attribute__((always_inline)) {
            constexpr int j = decltype(j_tag)::value, AT = j * NW * RPI8 * RB;
            const bool on = (there >> block_of(j) & 1) && kt * 64 + j * NW * RPI8 + row_w < ctx;
            s16x8 x[2];
            widen16<T>(__builtin_bit_cast(u32x4, lds_read_b128(raw0 + 16 * ln, 2 * j * 1024)), scale_value(scales.k[j]), x);
            lds_write_b128(k_to, AT, x[0]);
            lds_write_b128(k_to ^ 16u, AT, x[1]);
            widen16<T>(__builtin_bit_cast(u32x4, lds_read_b128(raw0 + 16 * ln, (2 * j + 1) * 1024)), scale_value(scales.v[j]), x);
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
        for (int c = 0; c < KC; ++c) k_rd[c] = lds_addr(&kv_lds[0][0]) + l16 * RB + 16 * ((4 * c + quad) ^ sw);
        const int vrow = 4 * quad + (l16 >> 2), swv = GEO::swz_v(vrow);
#pragma unroll
        for (int db = 0; db < DB; ++db) {
            const int dcol = 16 * db + 4 * (l16 & 3);
            v_rd[db] = lds_addr(&kv_lds[0][GEO::TILE_BYTES]) + vrow * RB + 16 * ((dcol >> 3) ^ swv) + 2 * (dcol & 7);
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

    auto process_tile = [&](auto stage_tag, int kt, int there) __attribute__((always_inline)) {
        constexpr int SOFF = decltype(stage_tag)::value * STAGE_BYTES;
        const int key0 = kt * 64;
        auto pin = [&]() __attribute__((always_inline)) { __builtin_amdgcn_sched_barrier(0); };
        auto read_v = [&](int ck, int db) __attribute__((always_inline)) -> s16x8 {
            const s16x4 t0 = lds_read_tr16(v_rd[db], SOFF + (32 * ck) * RB), t1 = lds_read_tr16(v_rd[db], SOFF + (32 * ck + 16) * RB);
            return s16x8{t0[0], t0[1], t0[2], t0[3], t1[0], t1[1], t1[2], t1[3]};
        };
        s16x8 va[DB];
        // S^T = K Q^T: register e of block [kb][qb] is key 16kb + 4 quad + e of row 16qb + l16
        f32x4 e_acc[4][2];
        {
            s16x8 kf[2][4];
#pragma unroll
            for (int c = 0; c < 2 && c < KC; ++c)
#pragma unroll
                for (int kb = 0; kb < 4; ++kb) kf[c][kb] = lds_read_b128(k_rd[c], SOFF + 16 * kb * RB);
            pin();
            for_range<0, KC * 4>([&](auto i_tag) __attribute__((always_inline)) {
                constexpr int i = decltype(i_tag)::value, c = i / 4, kb = i % 4;
#pragma unroll
                for (int qb = 0; qb < 2; ++qb) e_acc[kb][qb] = T::mfma16(kf[c & 1][kb], qf[qb][c], c == 0 ? f32x4{0.f, 0.f, 0.f, 0.f} : e_acc[kb][qb]);
                pin();
                if (c + 2 < KC) {
                    kf[c & 1][kb] = lds_read_b128(k_rd[c + 2], SOFF + 16 * kb * RB);
                } else if (c + 1 == KC) {
#pragma unroll
                    for (int db = kb * (DB / 4); db < (kb + 1) * (DB / 4); ++db) va[db] = read_v(0, db);
                }
                pin();
            });
        }
        if (key0 + 63 > wave_first) {
            // V rows that some of the wave's tokens attend and others do not: whether all are finite is what products with zero say
            f32x4 probe = {0.f, 0.f, 0.f, 0.f};
            const s16x8 zero = {0, 0, 0, 0, 0, 0, 0, 0};
#pragma unroll
            for (int db = 0; db < DB; ++db) probe = T::mfma16(read_v(1, db), zero, T::mfma16(va[db], zero, probe));
            if (__any(!(probe[0] + probe[1] + probe[2] + probe[3] == 0.f))) { by_key = kt; return; }
        }
        if (key0 + 63 > wave_first || !whole(kt, there)) {
#pragma unroll
            for (int qb = 0; qb < 2; ++qb) {
                const int lim = pos[qb] - key0 - 4 * quad;   // largest kept 16kb + e
#pragma unroll
                for (int kb = 0; kb < 4; ++kb) {
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
                for (int kb = 1; kb < 4; ++kb) {
                    m = max3(m, e_acc[kb][qb][1], e_acc[kb][qb][2]);
                    m = kb < 3 ? max3(m, e_acc[kb][qb][3], e_acc[kb + 1][qb][0]) : max2(m, e_acc[kb][qb][3]);
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
        for (int s = 0; s < 4; ++s) {
            const int ck = s >> 1, qb = s & 1;
            const s16x8 pcur = __builtin_bit_cast(s16x8, u32x4{pw[s & 1][0], pw[s & 1][1], pw[s & 1][2], pw[s & 1][3]});
#pragma unroll
            for (int db = 0; db < DB; ++db) {
                o_acc[db][qb] = T::mfma16(va[db], pcur, o_acc[db][qb]);
                pin();
                if (qb == 1 && ck == 0) va[db] = read_v(1, db);
                if (s + 1 < 4 && db < 4) pw[(s + 1) & 1][db] = weights_quarter((s + 1) >> 1, (s + 1) & 1, db);
                pin();
            }
        }
        l_sum[0] += ls[0];
        l_sum[1] += ls[1];
    };

    // ---- main loop: one barrier per tile, the next tile's rows on their way under it ----
    Pages pg{};                   // of the next tile to be requested
    int there = 0, there_1 = 0;   // pages of the tile at work and of the one behind it
    if (n_own > 0) {
        pg = pages_of(t_lo);
        there = there_of(pg);
        if (FP8) { request_codes(t_lo, pg); scales = scales_of(pg); }
        else copy_tile(t_lo, pg, std::integral_constant<int, 0>{});
        pg = pages_of(t_lo + 1);
    }
    // the query rows were requested first
    if (!FP8 && n_own > 0) wait_vmcnt<2 * NLD>(); else wait_vmcnt<0>();
    {
        const uint32_t qa = lds_addr(q_stage) + l16 * RB;
        const int sw = GEO::swz_k(l16);
#pragma unroll
        for (int qb = 0; qb < 2; ++qb)
#pragma unroll
            for (int c = 0; c < KC; ++c) qf[qb][c] = lds_read_b128(qa + 16 * ((4 * c + quad) ^ sw), 16 * qb * RB);
    }
    if (FP8 && n_own > 0) {
        widen_tile(t_lo, there, 0);
        if (n_own > 1) { request_codes(t_lo + 1, pg); scales = scales_of(pg); }
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
        asm volatile("" : "+s"(after.id[0]), "+s"(after.id[1]), "+s"(after.id[2]), "+s"(after.id[3]));
        if (FP8) {
#pragma unroll
            for (int j = 0; j < NR; ++j) asm volatile("" : "+s"(scales_2.k[j]), "+s"(scales_2.v[j]));
        }
        __syncthreads();           // everyone's has; the other stage is no longer being read
        if (it + 1 < n_own) {
            if (FP8) {
                wait_vmcnt<0>();   // the wave's codes of the next tile have
                widen_tile(kt + 1, there_1, STAGE ^ 1);
                if (it + 2 < n_own) request_codes(kt + 2, pg);
                there_2 = there_of(pg);
                scales = scales_2;
            } else {
                copy_tile(kt + 1, pg, std::integral_constant<int, STAGE ^ 1>{});
                there_1 = there_of(pg);
            }
            pg = after;
        }
        if (wave_on && there && kt * 64 <= wave_last && kt < by_key) process_tile(stage_tag, kt, there);
        there = there_1;
        there_1 = there_2;
    };
    for (int it = 0; it < n_own; it += 2) {
        iteration(std::integral_constant<int, 0>{}, it);
        if (it + 1 < n_own) iteration(std::integral_constant<int, 1>{}, it + 1);
    }

    if (!wave_on) return;
    if (by_key < t_lo + n_own) {
        const short* q[2];
        const int limit[2] = {pos[0] + 1, pos[1] + 1};
#pragma unroll
        for (int qb = 0; qb < 2; ++qb) {
            const int r = min(row0 + 16 * qb + l16, last_row), t = r / p.n_rep;
            q[qb] = (const short*)p.q + (int64_t)(seq_lo + t) * p.q2 + (int64_t)(g * p.n_rep + r - t * p.n_rep) * p.q1;
        }
        attend_key_by_key<T, D, FP8, 2>(p.c, p.Hkv, seq, g, by_key * 64, min(wave_last + 1, (t_lo + n_own) * 64), q, limit, c2,
                                        [&](int db, int qb) __attribute__((always_inline)) -> f32x4& { return o_acc[db][qb]; }, m_ref, l_sum);
    }
    float l_all[2];
#pragma unroll
    for (int qb = 0; qb < 2; ++qb) l_all[qb] = sum_across_quads(l_sum[qb]);
    if (me.parts > 1) {
        const int64_t part = (int64_t)(rank * p.Hkv + g) * BR;
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
    const uint32_t so = kAliasRows ? lds_addr(&kv_lds[0][0]) + (n_own & 1) * STAGE_BYTES + w * ROWS_BYTES : lds_addr(q_stage);
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
            *reinterpret_cast<s16x8*>((short*)p.out + (int64_t)(seq_lo + t) * p.o2 + (int64_t)(g * p.n_rep + r - t * p.n_rep) * p.o1 + 8 * gi) = val;
        }
    }
}

// out = sum_i O_i w_i / sum_i l_i w_i with w_i = 2^(m_i - max m) over the pieces of a block that was cut; D/4 lanes per row, four pieces requested at a
// time, references and sums with them.  A piece without keys has a sum of zero and is left out; one whose scores are all NaN has sums of NaN and
// is multiplied like any other.  grid (rows of a block / rows of a workgroup, KV heads, pieces): a block's first piece does it.  Bound by
// memory: 7 us after the 4 chunks above.
template <class T, int D, int BR>
__global__ __launch_bounds__(256) void paged_combine_kernel(const PagedParams p) {
    constexpr int LPR = D / 4, RPW = 256 / LPR;   // lanes per row, rows per workgroup
    const int row = (int)blockIdx.x * RPW + (int)threadIdx.x / LPR, d = 4 * ((int)threadIdx.x % LPR), g = blockIdx.y, first = blockIdx.z;
    if (first >= const_load(p.table)) return;
    const int32_t* me = p.table + 4 * (1 + first);
    // (sequences that overlap, which no valid call has, could have more pieces than there is room for)
    const int seq = const_load(me), block = const_load(me + 1), n = min(const_load(me + 3), (int)gridDim.z - first);
    if (n <= 1 || const_load(me + 2) != 0) return;
    const TokenRange range = token_range(const_load(p.cu + seq), const_load(p.cu + seq + 1), p.T);
    const int r = block * BR + row;
    if (r >= min(range.len, p.max_q) * p.n_rep) return;
    const int64_t step = (int64_t)p.Hkv * BR, at0 = ((int64_t)first * p.Hkv + g) * BR + row;
    float top = -INFINITY, total = 0.f;
    f32x4 acc = {0.f, 0.f, 0.f, 0.f};
    for (int i0 = 0; i0 < n; i0 += 4) {
        f32x2 ml[4];
        f32x4 o[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            const int64_t at = at0 + min(i0 + u, n - 1) * step;
            ml[u] = *reinterpret_cast<const f32x2*>(p.part_ml + at * 2);
            o[u] = *reinterpret_cast<const f32x4*>(p.part_o + at * D + d);
        }
        float now = top;
#pragma unroll
        for (int u = 0; u < 4; ++u) now = fmaxf(now, ml[u][0]);
        const float was = top > -INFINITY ? fast_exp2(top - now) : (now > -INFINITY ? 0.f : 1.f);
        total *= was;
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[e] *= was;
        top = now;
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            const bool on = i0 + u < n && !(ml[u][1] == 0.f);
            const float w = ml[u][0] > -INFINITY ? fast_exp2(ml[u][0] - now) : 0.f;
            total += on ? ml[u][1] * w : 0.f;
#pragma unroll
            for (int e = 0; e < 4; ++e) acc[e] += on ? o[u][e] * w : 0.f;
        }
    }
    const float inv = total > 0.f ? 1.f / total : 0.f;
    const int t = r / p.n_rep;
    uint2 pk;
    pk.x = T::pack2(acc[0] * inv, acc[1] * inv);
    pk.y = T::pack2(acc[2] * inv, acc[3] * inv);
    *reinterpret_cast<uint2*>((uint16_t*)p.out + (int64_t)(range.lo + t) * p.o2 + (int64_t)(g * p.n_rep + r - t * p.n_rep) * p.o1 + d) = pk;
}

static int64_t bounded_tokens(int64_t T, int64_t max_q_len) { return max_q_len > 0 && max_q_len < T ? max_q_len : T; }

// How a call is laid out, from its sizes alone (contexts and lengths are on the device).
struct PagedPlan {
    int waves;         // per workgroup
    int64_t blocks;    // bound of the blocks of rows of all sequences
    int64_t round;     // workgroups per KV head that the chip holds at once where blocks may be cut, 0 where none is
    int64_t pieces;    // bound of the pieces, per KV head
    size_t o_bytes, ml_bytes, table_bytes;
};
// Waves of a workgroup, 32 rows each (times in us, four / eight; 32 heads on 8 of 128, bf16).  16-bit rows: four, and two workgroups to a unit (three at head_dim
// 64), eight being one to a unit: 2 x 700 tokens behind 8000 224 / 244, a prompt of 512 16.6 / 21.0, of 2048 53.5 / 62.9, of 8192 492 / 494, of 16384 1925 / 1911.  Codes
// at head_dim 128: eight where a sequence can fill them, which widen a tile for twice as many rows: 2 x 700 behind 8000 338 / 295, 2048 behind 20000 827 / 725, a
// prompt of 4096 184 / 158, of 512 21.8 / 24.5; where it cannot, 60 x 20 behind 2000 to 8000, 277 / 361.
constexpr int kWavesBig = 8, kWavesSmall = 4;
constexpr int64_t kUnits = 256;
static int64_t blocks_of(int64_t n_seqs, int64_t T, int64_t n_rep, int64_t max_q, int waves) {
    const int64_t rows = waves * 32;
    return std::min(n_seqs * ((max_q * n_rep + rows - 1) / rows), T * n_rep / rows + n_seqs);
}
// Blocks of rows are cut where whole ones would leave more than a quarter of the chip's rounds of workgroups empty, of two rounds at most: the combine's
// launch and the sums' way through memory cost 4 to 8 us where that gains nothing (us, whole / cut, heads as above: 350 tokens behind 8000, a sixth of a round 179 / 63, 700
// behind 8000, a third, 185 / 122, of codes 289 / 159; 8 x 330 behind 250 to 16000, 1.5 rounds 425 / 360, of codes 616 / 499, but 4 x 700 behind 8000, 1.4 rounds of equal
// contexts 444 / 451; 60 x 20 behind 2000 to 8000, one round, 258 / 262), and not where contexts are short (a prompt of 512 16.6 / 21.2, of 1024 27.7 / 31.3, of codes 24.5
// / 27.0 and 41.8 / 38.7).  The host knows sizes, not contexts: where the blocks fill the chip and one context is far longer than the others, its
// blocks end alone (64 x 20 tokens, 63 behind 2000 and one behind 60000: 1270, behind 2000 all of them 102; 2048 tokens with 60 single ones, one of them at 60000 rows, 1298, in two
// calls 110 and 133).  So it is with more than 64 sequences, which are not cut (64 x 5 tokens of 16 heads on 2 behind 8000 106, 65 of them 168).
static bool cuts_blocks(bool eight, int64_t wgs, int64_t round, int64_t n_seqs, int64_t max_context) {
    const int64_t rounds = (wgs + round - 1) / round;
    return rounds <= 2 && 4 * wgs <= 3 * rounds * round && n_seqs <= 64 && max_context > (eight ? 512 : 1024);
}
static PagedPlan plan_paged(bool eight, int64_t n_seqs, int64_t T, int64_t Hq, int64_t Hkv, int64_t D, int64_t max_q, int64_t max_context) {
    PagedPlan r{};
    const int64_t n_rep = Hq / Hkv;
    r.waves = eight && D == 128 && max_q * n_rep > kWavesSmall * 32 ? kWavesBig : kWavesSmall;
    r.blocks = blocks_of(n_seqs, T, n_rep, max_q, r.waves);
    const int64_t wgs = r.blocks * Hkv, round = r.waves == kWavesBig ? kUnits : 2 * kUnits;   // workgroups that the chip holds at once
    r.pieces = r.blocks;
    if (cuts_blocks(eight, wgs, round, n_seqs, max_context)) {
        r.round = std::max<int64_t>(round / Hkv, 1);
        r.pieces = (r.blocks + r.round - 1) / r.round * r.round;
        r.o_bytes = (size_t)(r.pieces * Hkv * r.waves * 32 * D * 4);
        r.ml_bytes = (size_t)(r.pieces * Hkv * r.waves * 32 * 2 * 4);
        r.table_bytes = (size_t)(r.pieces + 1) * 16;
    }
    return r;
}

template <class T, int D, bool FP8, int NW>
static int launch_paged(const PagedParams& p, const PagedPlan& plan, hipStream_t stream) {
    const int64_t wgs = plan.pieces * p.Hkv;
    hipLaunchKernelGGL((paged_tile_kernel<T, D, FP8, NW>), dim3((unsigned)wgs), dim3(NW * 64), 0, stream, p);
    if (int rc = check_launch("paged_tile_kernel")) return rc;
    if (plan.round == 0) return MINFER_ATTN_OK;
    constexpr int BR = NW * 32;
    hipLaunchKernelGGL((paged_combine_kernel<T, D, BR>), dim3(BR * (D / 4) / 256, (unsigned)p.Hkv, (unsigned)plan.pieces), dim3(256), 0, stream, p);
    return check_launch("paged_combine_kernel");
}
template <class T, bool FP8> static int launch_paged_as(const PagedParams& p, const PagedPlan& plan, int64_t D, hipStream_t stream) {
    if (D == 64) return launch_paged<T, 64, FP8, kWavesSmall>(p, plan, stream);
    if constexpr (FP8)
        if (plan.waves == kWavesBig) return launch_paged<T, 128, FP8, kWavesBig>(p, plan, stream);
    return launch_paged<T, 128, FP8, kWavesSmall>(p, plan, stream);
}

}  // namespace minfer_attn

using namespace minfer_attn;

MINFER_ATTN_EXPORT size_t minfer_flash_attn_paged_workspace_bytes(int64_t n_seqs, int64_t T, int64_t Hq, int64_t Hkv, int64_t D, int64_t max_context,
                                                                  int64_t max_q_len) {
    if (n_seqs <= 0 || T <= 0 || Hq <= 0 || Hkv <= 0 || D <= 0 || max_context < 0 || Hq % Hkv != 0) return 0;
    const int64_t max_q = bounded_tokens(T, max_q_len);
    if (paged_decode_takes(Hq, Hkv, max_q)) return paged_decode_workspace_bytes(n_seqs, Hq, Hkv, D, max_context, max_q);
    size_t most = 0;   // of both kinds of pages
    for (const bool eight : {false, true}) {
        const PagedPlan r = plan_paged(eight, n_seqs, T, Hq, Hkv, D, max_q, max_context);
        most = std::max(most, r.o_bytes + r.ml_bytes + r.table_bytes);
    }
    return most;
}

MINFER_ATTN_EXPORT int minfer_flash_attn_paged(int dtype, int page_type, const void* q, const minfer_kv_pages* pages, const int32_t* cu_seqlens,
                                               const int32_t* ctx_lens, void* out, int64_t n_seqs, int64_t T, int64_t Hq, int64_t Hkv, int64_t D,
                                               int64_t max_q_len, const minfer_attn_strides* st, void* workspace, size_t workspace_bytes,
                                               void* stream_v) {
    clear_error();
    PagedParams p{};
    if (int rc = check_pages("flash_attn_paged", dtype, page_type, pages, n_seqs, Hkv, D, p.c)) return rc;
    auto bad = [&](const char* what) { return fail(MINFER_ATTN_EINVAL, what); };
    if (Hq <= 0 || Hq % Hkv != 0) return bad("flash_attn_paged: n_heads must be a positive multiple of n_kv_heads");
    if (Hq > 65535) return bad("flash_attn_paged: n_heads > 65535 unsupported");
    if (!st) return bad("flash_attn_paged: strides is null");
    if (n_seqs < 0 || T < 0 || max_q_len < 0) return bad("flash_attn_paged: negative size");
    if (n_seqs == 0 || T == 0) return MINFER_ATTN_OK;
    if (!q || !out || !cu_seqlens || !ctx_lens) return bad("flash_attn_paged: q, out, cu_seqlens and ctx_lens must be non-null");
    if (!aligned16(q) || !aligned16(out)) return bad("flash_attn_paged: q and out must be 16-byte aligned");
    const int64_t s[4] = {st->q1, st->q2, st->o1, st->o2};
    for (int i = 0; i < 4; ++i)
        if (s[i] < 0 || s[i] % 8 != 0) return bad("flash_attn_paged: strides of q and out must be non-negative multiples of 8 elements");
    const int64_t max_context = (int64_t)p.c.width << p.c.page_log2;
    p.q = q; p.out = out; p.cu = cu_seqlens; p.ctx = ctx_lens;
    p.q1 = st->q1; p.q2 = st->q2; p.o1 = st->o1; p.o2 = st->o2;
    p.n_seqs = (int)n_seqs; p.T = (int)T; p.Hq = (int)Hq; p.Hkv = (int)Hkv; p.n_rep = (int)(Hq / Hkv);
    p.scale_log2 = (float)(1.4426950408889634 / sqrt((double)D));
    p.inv_scale_log2 = (float)(sqrt((double)D) / 1.4426950408889634);
    const bool eight = page_type == MINFER_FP8_E4M3;
    const int64_t max_q = bounded_tokens(T, max_q_len);
    if (T > (1 << 30) || T * Hq > 0x7fffffffLL - 4096 || n_seqs > (1 << 24)) return bad("flash_attn_paged: problem too large for one launch");
    p.max_q = (int)max_q;
    if (paged_decode_takes(Hq, Hkv, max_q)) {
        const size_t need = paged_decode_workspace_bytes(n_seqs, Hq, Hkv, D, max_context, max_q);
        if (!workspace || !aligned16(workspace) || workspace_bytes < need)
            return fail(MINFER_ATTN_EWORKSPACE, "flash_attn_paged: workspace too small or misaligned (see minfer_flash_attn_paged_workspace_bytes)");
        return launch_paged_decode(p, dtype, D, eight, max_context, workspace, (hipStream_t)stream_v);
    }
    const PagedPlan plan = plan_paged(eight, n_seqs, T, Hq, Hkv, D, max_q, max_context);
    // (workgroups and their ids are 32-bit numbers)
    if (plan.pieces * Hkv > 0x7fffffffLL) return bad("flash_attn_paged: problem too large for one launch");
    if (plan.round > 0 && (!workspace || !aligned16(workspace) || workspace_bytes < plan.o_bytes + plan.ml_bytes + plan.table_bytes))
        return fail(MINFER_ATTN_EWORKSPACE, "flash_attn_paged: workspace too small or misaligned (see minfer_flash_attn_paged_workspace_bytes)");
    p.round = (int)plan.round;
    p.part_o = (float*)workspace;
    p.part_ml = (float*)((char*)workspace + plan.o_bytes);
    p.table = (int32_t*)((char*)workspace + plan.o_bytes + plan.ml_bytes);
    hipStream_t stream = (hipStream_t)stream_v;
    if (dtype == MINFER_ATTN_F16) return eight ? launch_paged_as<F16, true>(p, plan, D, stream) : launch_paged_as<F16, false>(p, plan, D, stream);
    return eight ? launch_paged_as<BF16, true>(p, plan, D, stream) : launch_paged_as<BF16, false>(p, plan, D, stream);
}
