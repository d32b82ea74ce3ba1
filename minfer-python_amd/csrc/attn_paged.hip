// Attention of packed tokens over a paged KV cache for gfx950: chunks of prompts, drafts and single tokens.
//
// Rows.  The new tokens of a sequence and the query heads of a KV head's group are one list of rows, token by token, heads innermost
// (row = token * n_rep + head): whatever the group's size, 32 rows of a wave attend one KV head, and a sequence of a few tokens
// fills its rows with heads.  A workgroup takes NW * 32 rows and walks the sequence's 64-key tiles up to its last row's position;
// where that makes few workgroups the tiles of a long sequence's blocks are cut into pieces with a workgroup each (find_piece), which
// leave un-normalised sums in the workspace for paged_combine_kernel.
//
// The walk over the tiles is csrc/attn_paged_tile.h's.
#include <algorithm>

#include "attn_paged_tile.h"

namespace minfer_attn {

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
    __shared__ __attribute__((aligned(1024))) char lds[TileLds<D, FP8, NW, false>::BYTES];
    constexpr int BR = NW * 32;
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
    if (p.round > 0 && g == 0 && threadIdx.x == 0) reinterpret_cast<int4*>(p.table)[1 + rank] = make_int4(me.seq, me.block, me.part, me.parts);
    const TokenRange range = token_range(const_load(p.cu + me.seq), const_load(p.cu + me.seq + 1), p.T);
    const int ctx = context_of(p.c, const_load(p.ctx + me.seq), range);
    const TileJob job{g, me.seq, range.lo, ctx, ctx - range.len, min(range.len, p.max_q) * p.n_rep, me.block * BR, 0, me.part, me.parts, rank, 0, 0, 0, 0, false, false};
    attend_tiles<T, D, FP8, NW, false>(p, job, lds);
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
