// Attention of few query rows per sequence over a paged cache where groups of sequences share their first pages, for gfx950: a batch behind one instruction or
// document, whose pages every table names.  The prefix's rows are read once for all of a group's tokens instead of once for each sequence.
//
// out = softmax over [prefix, own rows] is made of two softmaxes with references and sums of their own:
// * the prefix: the tokens of a group times the query heads of a KV head are a list of rows, up to 256 of which (128 at head_dim 64) walk the prefix's 64-key tiles
//   together (attend_tiles): matrix work, 2.05 us a tile of 256 rows, 1.07 PFLOP/s (codes 2.5), the rate of the prompts' kernel;
// * the own rows: streamed by single waves (stream_columns), for up to 32 (token, head) columns together: bound by memory.
// Both are lines of places, cut into equal shares, and one launch, whose workgroups are divided between them so that both end together (tile_ranks).  Everything
// is a partial result, and shared_merge_kernel puts a row's together.  32 heads on 8 of 128: 64 tokens behind 6000 rows and 50 to 1500 of their own 52 us, 4.5 TB/s of
// what has to be read once (flash_attn_paged 233); 192 behind 16000 to 24000 rows of codes 176, bound by products and widening (1316); 24 sequences of 3 to 6 tokens behind
// 12000 rows 54 (145).  Of that the start is 7 us (lengths and groups looked up 2.2, the first rows 4), the merge 5 to 9.
//
// How the work is cut follows from device data (lengths, contexts, groups) that every wave looks up for itself, a sequence or a group to a lane.
#include <algorithm>

#include "attn_paged_stream.h"
#include "attn_paged_tile.h"

namespace minfer_attn {

typedef int i32x4 __attribute__((ext_vector_type(4)));

// Waves of a workgroup, up to 32 rows of a block each, and workgroups of the launch, as many as the chip holds at once: four tiles of 32 KiB leave room for one on a
// compute unit, of 16 KiB (head_dim 64) for two.
constexpr int shared_waves(int64_t D) { return D == 128 ? 8 : 4; }
constexpr int shared_wgs(int64_t D) { return 256 * 8 / shared_waves(D); }
template <int D> constexpr int kSharedWaves = shared_waves(D);
template <int D> constexpr int kBlockRows = shared_waves(D) * 32;
// Of all rows that the tables may name (shared_takes): from here on; where there are more than 16 columns, at head_dim 64 and over codes.
constexpr int64_t kSharedBytes = 220000000, kSharedBytesCodes = 150000000, kSharedBytesPairs = 70000000, kSharedBytesPairsCodes = 25000000, kSharedBytesLong = 600000000;
constexpr int kMaxSharedHeads = 128;                               // KV heads: each has workgroups of its own for the prefix

struct SharedWork {
    DecodeWork d;                    // of the own rows; part_o / part_ml of d.p are theirs
    const int32_t* cu_groups; const int32_t* prefix;
    int n_groups;
    float* tile_o; float* tile_ml;   // partial results of the tiles: [KV head][part_rows][D] and their references and sums (tile_row)
    int part_rows;                   // that there is room for, per KV head
    i32x4* seq_tab;                  // [n_seqs]: a sequence's place on its line, its group (-1: none); then the quotas of both lines
    i32x4* group_tab;                // [n_groups]: first token, (token, head) rows, place of its first block on the line of tiles, rows of the groups in front
};

// Rows of group i's prefix that are computed for all its tokens together: whole tiles.
MA_DEV int shared_rows(const SharedWork& w, int i) { return min(max(w.prefix[i], 0), w.d.p.c.width << w.d.p.c.page_log2) & ~63; }

struct Group { int first, last, lo, rows, tiles; };   // sequences (up to the last one with tokens), first token, (token, head) rows, tiles of the prefix
// The whole wave, a group to a lane.
MA_DEV Group group_at(const SharedWork& w, int i) {
    const PagedParams& p = w.d.p;
    Group r{0, 0, 0, 0, 0};
    int hi = 0;
    bool ends_empty = false;
    if (i < w.n_groups) {
        r.first = min(max(w.cu_groups[i], 0), p.n_seqs);
        r.last = min(max(w.cu_groups[i + 1], r.first), p.n_seqs);
        r.tiles = shared_rows(w, i) >> 6;
        const int begin = p.cu[max(r.last - 1, 0)], end = p.cu[r.last];
        r.lo = min(max(p.cu[r.first], 0), p.T);
        hi = min(max(end, 0), p.T);
        ends_empty = r.last > r.first && r.tiles > 0 && token_range(begin, end, p.T).len == 0;
    }
    // (a group whose last sequence has no tokens: where its entries fall, as behind the last sequence of a padded batch, they say nothing of the group's end, which is that of
    // its last sequence with tokens, looked for 64 at a time)
    uint64_t odd = __ballot(ends_empty);
    while (odd) {
        const int lane = threadIdx.x & 63, at = __ffsll((unsigned long long)odd) - 1, first = lane_value(r.first, at);
        int found = lane_value(r.lo, at), found_last = first;
        for (int end = lane_value(r.last, at); end > first; end -= 64) {
            const int s = end - 1 - lane;
            TokenRange t{0, 0, 0};
            if (s >= first) t = token_range(p.cu[s], p.cu[s + 1], p.T);
            const uint64_t some = __ballot(t.len > 0);
            if (some) {
                const int src = __ffsll((unsigned long long)some) - 1;
                found = lane_value(t.lo + t.len, src);
                found_last = end - src;
                break;
            }
        }
        if (lane == at) { hi = found; r.last = found_last; }
        odd &= odd - 1;
    }
    r.rows = r.last > r.first ? max(hi - r.lo, 0) * p.n_rep : 0;
    return r;
}

// What the waves of a workgroup have looked up (all of them the same, each for itself): the first 64 groups, and of the first 64 times 64 what lies on the line of tiles
// in front of them.
struct SharedLds { Group groups[64]; int tiles_before[64], rows_before[64]; };

// The group of sequence s (-1: none): cu_groups is a list of increasing starts.
MA_DEV int group_of(const SharedWork& w, const SharedLds& l, int s) {
    if (w.n_groups <= 64) {
        int lo = 0, hi = w.n_groups - 1;
        while (lo < hi) {
            const int mid = (lo + hi + 1) >> 1;
            if (l.groups[mid].first <= s) lo = mid; else hi = mid - 1;
        }
        return l.groups[lo].first <= s && s < l.groups[lo].last ? lo : -1;
    }
    int lo = 0, hi = w.n_groups;   // the last entry that is <= s, of n_groups + 1
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (w.cu_groups[mid] <= s) lo = mid; else hi = mid - 1;
    }
    return lo < w.n_groups && w.cu_groups[lo] <= s ? lo : -1;
}

// What a sequence has behind the prefix: the first group of rows and how many there are.
struct OwnSeq { SeqInfo info; int group, g0, groups; };
template <int GR> MA_DEV OwnSeq own_of(const SharedWork& w, const SharedLds& l, int s, const SeqInfo& info) {   // (per lane)
    OwnSeq r{info, s < w.d.p.n_seqs ? group_of(w, l, s) : -1, 0, 0};
    if (r.group >= 0) r.g0 = (w.n_groups <= 64 ? l.groups[r.group].tiles * 64 : shared_rows(w, r.group)) / GR;
    r.groups = info.len > 0 ? max((info.ctx + GR - 1) / GR - r.g0, 0) : 0;
    return r;
}
template <int GR> MA_DEV OwnSeq own_seq(const SharedWork& w, const SharedLds& l, int s) { return own_of<GR>(w, l, s, line_seq<GR>(w.d, s).info); }

// Blocks of a group's rows, equal to within a wave's: every row of a block attends all tiles of the prefix.
template <int D> MA_DEV int blocks_of(const Group& g) { return g.tiles > 0 ? (g.rows + kBlockRows<D> - 1) / kBlockRows<D> : 0; }
MA_DEV int rows_of_block(int rows, int blocks) { return ((rows + blocks - 1) / blocks + 31) & ~31; }
MA_DEV int prefix_rows(const Group& g) { return g.tiles > 0 ? g.rows : 0; }   // that have partial results of tiles

// Where the partial results of a share's part of a block lie, `row` rows of all groups in front of the block's first.  From one to the next along the line either the share's
// number goes up by one, and with it a whole block's rows, or the rows in front by the block's, or both: they do not meet, and all rows and a block for
// every share are room enough, however many groups there are.  (With room for a whole block of each group 4096 of them, 32 heads on 8 of 128, were 4.2 GiB, now 0.1.)
template <int D> MA_DEV uint32_t tile_row(int row, int share) { return (uint32_t)row + (uint32_t)(share * kBlockRows<D>); }

// What it costs to begin with a block, or with a (sequence, KV head, group of columns), inside a share (looking it up, requesting its first rows and waiting for
// them), in tiles and in groups of rows: that many places of the line in front of it are its, where nothing is.
// (Groups of rows, us without / with: 90 sequences in 7 groups 97.4 / 93.2, 64 of one token over head_dim 64 36.2 / 34.3, over codes 35.2 / 33.5.)
constexpr int kTileLead = 2, kPairLead = 2;

// How the launch is laid out, worked out by every wave.  Both kinds of work are lines, cut into equal shares: the tiles of all blocks of the
// groups' rows, for every KV head; and the groups of the sequences' own rows, for every KV head and group of columns.
struct SharedPlan {
    int n_tile;                   // workgroups for tiles, the launch's first ones
    int tiles, tile_quota;        // of the line of tiles, per KV head
    int total, quota;             // of the other
    int inside_first, inside_last;   // sequences, the first and the last one with a token inside its group's prefix (none: the first is behind the last)
    int starts;                   // lane i: what lies on that line in front of sequence 64 i
};

// Time of the own rows in tiles (what a workgroup takes for one whose waves all have rows: 2.05 us at head_dim 128, 2.5 over codes, 1.2 and 1.6 at head_dim 64, and 3 us before its first): `own`
// of them a group for one workgroup, less with more of them, but never less than `chip` / workgroups of the launch a group, the memory's share.  Fitted to the times of 48
// calls of one group of columns and 24 of two at every division of the workgroups, over all of which the division that comes of it is 0.8 % slower than the best, at most 7 %; us at it / at
// the best: 64 sequences behind 6000 rows 52.1 / 52.1, over codes 41.1 / 41.1, 90 in seven groups 89.8 / 89.5, 24 with drafts 54.0 / 53.6, 192 behind 16000 to 24000 rows 217 / 217, of codes 175 / 175.
struct OwnCost { float own, chip; };
template <int D, int GR, int NC> constexpr OwnCost kOwnCost =
    NC == 1 ? (D == 128 ? (GR == 16 ? OwnCost{0.08f, 0.068f} : OwnCost{0.0912f, 0.017f}) : (GR == 16 ? OwnCost{0.139f, 0.053f} : OwnCost{0.157f, 0.074f}))
            : (D == 128 ? (GR == 16 ? OwnCost{0.104f, 0.035f} : OwnCost{0.1f, 0.04f}) : (GR == 16 ? OwnCost{0.21f, 0.045f} : OwnCost{0.113f, 0.336f}));

// A tile's time where some waves have no rows: 1.6 us with two of eight.
template <int D> MA_DEV float tile_time(int rows) { return 0.73f + 0.27f * (float)((rows + 31) >> 5) / (float)kSharedWaves<D>; }

// Workgroups per KV head for the tiles, of G in all: those with which both kinds of work take the same time, tiles W / n and own rows A / (G - n) + B / G, or one or
// two more where whole tiles to a share make that the shorter.  `each`: a tile's time on average.
template <int D, int GR, int NC> MA_DEV int tile_ranks(int tiles, float each, int total, int Hkv, int G) {
    const float W = (float)tiles * each * (float)Hkv, A = kOwnCost<D, GR, NC>.own * (float)total, B = kOwnCost<D, GR, NC>.chip * (float)total, S = W + A + B;
    const int most = (G - (total > 0 ? G / 16 : 0)) / Hkv;   // (own rows of a token or two: 192 sequences behind 16000 to 24000 rows of codes 127 us with a sixteenth for them, 133 with an eighth)
    const int first = min(max((int)(2.f * W * (float)G / (S + sqrtf(fmaxf(S * S - 4.f * B * W, 0.f))) / (float)Hkv), 1), most);
    int best = first;
    float least = 3.0e38f;
#pragma unroll
    for (int i = 0; i < 3; ++i) {
        const int r = min(first + i, most);
        const float t = fmaxf((float)((tiles + r - 1) / r) * each + 1.5f, A / (float)max(G - r * Hkv, 1) + B / (float)G);
        if (t < least) { least = t; best = r; }
    }
    return __builtin_amdgcn_readfirstlane(best);
}

MA_DEV int own_length(int groups) { return groups > 0 ? groups + kPairLead : 0; }

template <int D, int GR, int NC> MA_DEV SharedPlan plan_shared(const SharedWork& w, bool writes, SharedLds& l) {
    const PagedParams& p = w.d.p;
    const int lane = threadIdx.x & 63, pairs = p.Hkv * w.d.n_hg;
    SharedPlan r{};
    r.inside_first = 0x7fffffff;
    r.inside_last = -1;
    int rows = 0, longest = 0, longest_own = 0;
    float work = 0.f;
    for (int base = 0; base < w.n_groups; base += 64) {
        const Group q = group_at(w, base + lane);
        if (base == 0) l.groups[lane] = q;   // (all waves write the same, and each reads what it wrote)
        if (base < 64 * 64 && lane == 0) {
            l.tiles_before[base >> 6] = r.tiles;
            l.rows_before[base >> 6] = rows;
        }
        const int n = blocks_of<D>(q), length = n * (q.tiles + kTileLead), incl = wave_inclusive_scan(length), in_front = wave_inclusive_scan(prefix_rows(q));
        if (writes && base + lane < w.n_groups) w.group_tab[base + lane] = i32x4{q.lo, q.rows, r.tiles + incl - length, rows + in_front - prefix_rows(q)};
        work += lane_sum<64>(n > 0 ? (float)length * tile_time<D>(rows_of_block(q.rows, n)) : 0.f);
        r.tiles += lane_value(incl, 63);
        rows += lane_value(in_front, 63);
        longest = max(longest, q.tiles);
    }
    wave_lds_order();
    constexpr int UN = 4;   // times 64 sequences requested together
    for (int base = 0; base < p.n_seqs; base += 64 * UN) {
        SeqInfo info[UN];
#pragma unroll
        for (int u = 0; u < UN; ++u) info[u] = line_seq<GR>(w.d, base + 64 * u + lane).info;
#pragma unroll
        for (int u = 0; u < UN; ++u) {
            const int from = base + 64 * u;
            if (from >= p.n_seqs) break;
            const OwnSeq q = own_of<GR>(w, l, from + lane, info[u]);
            const int length = own_length(q.groups) * pairs, incl = wave_inclusive_scan(length);
            if (writes && from + lane < p.n_seqs) w.seq_tab[from + lane] = i32x4{r.total + incl - length, q.group, 0, 0};
            if (lane == from >> 6) r.starts = r.total;
            r.total += lane_value(incl, 63);
            longest_own = max(longest_own, q.groups);
            const uint64_t in = __ballot(q.info.len > 0 && q.info.ctx - q.info.len < q.g0 * GR - 1);
            if (in) {
                r.inside_first = min(r.inside_first, from + __ffsll((unsigned long long)in) - 1);
                r.inside_last = from + 63 - __clzll((long long)in);
            }
        }
    }
    const int G = (int)gridDim.x, ranks = r.tiles > 0 ? tile_ranks<D, GR, NC>(r.tiles, work / (float)r.tiles, r.total, p.Hkv, G) : 0;
    r.n_tile = ranks * p.Hkv;
    longest = __builtin_amdgcn_readfirstlane((int)wave_max((float)longest));
    longest_own = __builtin_amdgcn_readfirstlane((int)wave_max((float)longest_own));
    constexpr int kLeastTiles = 2;
    r.tile_quota = max(max((r.tiles + ranks - 1) / max(ranks, 1), kLeastTiles), longest / (kMaxParts - 3) + 1);
    const int n_waves = (G - r.n_tile) * kSharedWaves<D>;
    r.quota = max(max((r.total + n_waves - 1) / max(n_waves, 1), kLeastShare / GR), longest_own / (kMaxParts - 3) + 1);
    if (writes && lane == 0) w.seq_tab[p.n_seqs] = i32x4{r.quota, r.tile_quota, 0, 0};
    return r;
}

// The block that holds place x of the line of tiles: its job (n_own: its tiles from there on; 0: there is no such block).
template <int D> MA_DEV TileJob shared_job(const SharedWork& w, int x, const SharedPlan& plan, const SharedLds& l) {
    const int lane = threadIdx.x & 63;
    TileJob job{};
    // the 64 groups that it lies in
    const uint64_t in_front = __ballot(lane == 0 || (lane * 64 < w.n_groups && l.tiles_before[lane] <= x));
    const int strip = 63 - __builtin_amdgcn_readfirstlane(__clzll((long long)in_front));
    int before = strip > 0 ? __builtin_amdgcn_readfirstlane(l.rows_before[strip]) : 0;   // rows
    x -= strip > 0 ? __builtin_amdgcn_readfirstlane(l.tiles_before[strip]) : 0;
    for (int base = strip * 64; base < w.n_groups; base += 64) {
        const Group q = base == 0 ? l.groups[lane] : group_at(w, base + lane);
        const int blocks = blocks_of<D>(q), n = blocks * (q.tiles + kTileLead), incl = wave_inclusive_scan(n), sum = lane_value(incl, 63), rows = wave_inclusive_scan(prefix_rows(q));
        if (x >= sum) {
            x -= sum;
            before += lane_value(rows, 63);
            continue;
        }
        const int src = __builtin_amdgcn_readfirstlane(__ffsll((unsigned long long)__ballot(x < incl)) - 1);
        const int tiles = lane_value(q.tiles, src), n_blocks = lane_value(blocks, src);
        job.seq = job.first = lane_value(q.first, src);
        job.last = lane_value(q.last, src);
        job.lo = lane_value(q.lo, src);
        job.rows = lane_value(q.rows, src);
        job.ctx = tiles * 64;
        x -= lane_value(incl - n, src);
        if (x < 0 || tiles <= 0 || x >= lane_value(n, src)) return job;   // (groups that overlap: sums past 31 bits)
        const int length = tiles + kTileLead, block = x / length, per = rows_of_block(job.rows, n_blocks);
        job.row0 = block * per;
        job.row_end = min(job.row0 + per, job.rows);
        job.t_lo = x - block * length - kTileLead;   // (below zero: places in front of the first tile)
        job.n_own = tiles - job.t_lo;
        job.slot = before + lane_value(rows - prefix_rows(q), src) + job.row0;
        job.prefix = true;
        job.inside = plan.inside_first < job.last && plan.inside_last >= job.first;   // (of a group between two that have such tokens: looked for in vain)
        return job;
    }
    return job;
}

// A share of the tiles of a KV head.
template <class T, int D, bool FP8> MA_DEV void shared_tiles(const SharedWork& w, const SharedPlan& plan, PagedParams p, char* lds, const SharedLds& l) {
    int g, rank;
    if ((p.Hkv & 7) == 0) {   // a KV head's workgroups on one XCD (ids go round-robin)
        const int per = p.Hkv >> 3, m = (int)blockIdx.x >> 3;
        g = (m % per) * 8 + ((int)blockIdx.x & 7);
        rank = m / per;
    } else {
        g = (int)blockIdx.x % p.Hkv;
        rank = (int)blockIdx.x / p.Hkv;
    }
    p.part_o = w.tile_o;
    p.part_ml = w.tile_ml;
    if (rank > (plan.tiles - 1) / plan.tile_quota) return;   // (fewer shares than workgroups)
    const int x0 = rank * plan.tile_quota, x1 = x0 + min(plan.tile_quota, plan.tiles - x0);
    bool busy = false;
    for (int x = x0; x < x1;) {
        TileJob job = shared_job<D>(w, x, plan, l);
        job.n_own = min(job.n_own, x1 - x);
        const uint32_t slot = tile_row<D>(job.slot, rank);
        if (job.n_own <= 0 || slot > (uint32_t)(w.part_rows - kBlockRows<D>)) break;   // (groups that overlap, which no valid call has: more rows than there is room for)
        job.slot = g * w.part_rows + (int)slot;
        x += job.n_own;
        job.n_own += min(job.t_lo, 0);
        job.t_lo = max(job.t_lo, 0);
        if (job.n_own <= 0) continue;   // (the share ends in front of the block's first tile)
        job.g = g;
        if (busy) {   // every wave is done with the stages, and its results are on their way no more
            wait_vmcnt<0>();
            __syncthreads();
        }
        busy = true;
        attend_tiles<T, D, FP8, kSharedWaves<D>, true>(p, job, lds);
    }
}

// The line, as in paged_line_kernel, of the rows behind the prefixes.
template <class T, int D, bool FP8, int NC> MA_DEV void shared_line(const SharedWork& w, const SharedPlan& plan, char* lds, const SharedLds& l) {
    constexpr int GR = kRows<FP8>;
    const DecodeWork& d = w.d;
    const PagedParams& p = d.p;
    const int lane = threadIdx.x & 63, wid = wave_id(), pairs = p.Hkv * d.n_hg;
    const int n_wg = (int)gridDim.x - plan.n_tile, wg = (int)blockIdx.x - plan.n_tile, quota = plan.quota, total = plan.total;
    const int n_shares = total > 0 ? (total - 1) / quota + 1 : 0;
    const int wave = n_shares <= n_wg ? wid * n_wg + wg : wg * kSharedWaves<D> + wid;
    if (wave >= n_shares) return;
    int x = wave * quota;
    const int x_end = x + min(quota, total - x);
    int s = 0, off = 0, groups = 0, first = 0;
    const int strip = 63 - __builtin_amdgcn_readfirstlane(__clzll((long long)__ballot(lane == 0 || (lane * 64 < p.n_seqs && plan.starts <= x))));
    for (int base = strip * 64, start = lane_value(plan.starts, strip); base < p.n_seqs; base += 64) {
        const OwnSeq q = own_seq<GR>(w, l, base + lane);
        const int incl = wave_inclusive_scan(own_length(q.groups) * pairs), sum = lane_value(incl, 63);
        if (x < start + sum) {
            const int src = __builtin_amdgcn_readfirstlane(__ffsll((unsigned long long)__ballot(x < start + incl)) - 1);
            s = base + src;
            groups = lane_value(q.groups, src);
            first = lane_value(q.g0, src);
            off = start + lane_value(incl, src) - own_length(groups) * pairs;
            break;
        }
        start += sum;
    }
    SeqInfo info = seq_info(p, s);
    while (x < x_end) {
        if (x >= off + pairs * own_length(groups)) {   // the sequence is done: on to the next that has rows
            off += pairs * own_length(groups);
            do {
                info = seq_info(p, ++s);
                const OwnSeq q = own_of<GR>(w, l, s, info);
                first = __builtin_amdgcn_readfirstlane(q.g0);
                groups = __builtin_amdgcn_readfirstlane(q.groups);
            } while (groups == 0);
        }
        const int length = own_length(groups), pair = (x - off) / length, y = x - off - pair * length;   // y: the first pair_lead places are empty
        const int n = min(length - y, x_end - x), g1 = y + n - kPairLead, g0 = max(y - kPairLead, 0);
        x += n;
        if (g1 <= g0) continue;
        const int g = d.n_hg == 1 ? pair : pair / d.n_hg, hg = pair - g * d.n_hg;   // (a KV head's groups of columns read the same rows one after the other)
        ColumnAcc<D> acc[NC];
        stream_columns<T, D, FP8, NC, 2, FP8 && D == 128>(d, s, info, g, hg * NC, first + g0, first + g1, lds + wid * kWaveLds<D, FP8>, acc);
#pragma unroll
        for (int n = 0; n < NC; ++n) store_part<D>(d, hg * NC + n, (int64_t)s * pairs + pair + wave, acc[n], 16 * n);
    }
}

template <class T, int D, bool FP8, int NC>
__global__ __launch_bounds__(kSharedWaves<D> * 64, 2) void shared_kernel(const SharedWork w) {
    using LDS = TileLds<D, FP8, kSharedWaves<D>, true>;
    static_assert(kSharedWaves<D> * kWaveLds<D, FP8> <= LDS::BYTES, "one area for both");
    __shared__ __attribute__((aligned(1024))) char lds[LDS::BYTES];
    __shared__ SharedLds looked_up;
    const SharedPlan plan = plan_shared<D, kRows<FP8>, NC>(w, blockIdx.x == 0 && wave_id() == 0, looked_up);
    if ((int)blockIdx.x < plan.n_tile) shared_tiles<T, D, FP8>(w, plan, w.d.p, lds, looked_up);
    else shared_line<T, D, FP8, NC>(w, plan, lds, looked_up);
}

// out = sum_i O_i w_i / sum_i l_i w_i, w_i = 2^(m_i - max m), over the parts of a row, those of the line and those of its group's prefix; a wave per row (sequence,
// token, head), lane i holding the references and sums of both parts i.
template <class T, int D, int GR, int NC>
__global__ __launch_bounds__(256) void shared_merge_kernel(const SharedWork w) {
    const DecodeWork& work = w.d;
    const PagedParams& p = work.p;
    constexpr int EPL = D / 64;
    const int lane = threadIdx.x & 63;
    const int64_t row = (int64_t)blockIdx.x * 4 + wave_id();
    const int per_seq = p.Hkv * work.n_col;
    if (row >= (int64_t)p.n_seqs * per_seq) return;
    const int s = (int)(row / per_seq), in = (int)(row - (int64_t)s * per_seq), g = in / work.n_col, col = in - g * work.n_col;
    const SeqInfo info = seq_info(p, s);
    const int tok = col / p.n_rep, head = col - tok * p.n_rep;
    if (tok >= info.len) return;
    const i32x4 own = const_load(w.seq_tab + s);   // as written by plan_shared
    const int group = own[1];
    const i32x4 quotas = const_load(w.seq_tab + p.n_seqs);
    constexpr int BR = kBlockRows<D>;
    // partial results of an item's tiles, which are n from place x of the line on: their number, and the first one's
    struct Span { int n; int64_t first; };
    auto span_of = [&](int x, int n, int quota) {
        const int share = x / quota;
        return Span{n > 0 ? min((x + n - 1) / quota - share + 1, kMaxParts) : 0, share};
    };
    // the parts of the group's prefix
    int n_pre = 0, skip = 0;
    int64_t pre0 = 0;
    if (group >= 0) {
        skip = shared_rows(w, group);
        const i32x4 t = const_load(w.group_tab + group);
        const int r = (info.lo + tok - t[0]) * p.n_rep + head;
        if (skip > 0 && r >= 0 && r < t[1]) {
            const int blocks = (t[1] + BR - 1) / BR, per = rows_of_block(t[1], blocks), block = r / per;
            const int x = t[2] + block * ((skip >> 6) + kTileLead) + kTileLead, at = t[3] + r;
            const Span a = span_of(x, skip >> 6, quotas[1]);
            const int64_t end = (int64_t)at + (a.first + a.n - 1) * BR;
            n_pre = x >= 0 && at >= 0 && end < w.part_rows ? a.n : 0;   // (what groups that overlap have no room for)
            pre0 = n_pre > 0 ? (int64_t)g * w.part_rows + at + a.first * BR : 0;
        }
    }
    // those of the sequence's own rows
    const int groups = max((info.ctx + GR - 1) / GR - skip / GR, 0), pair = g * work.n_hg + col / (16 * NC);
    const Span own_span = span_of(own[0] + pair * own_length(groups) + kPairLead, groups, quotas[0]);
    const int ns = own_span.n;
    const int64_t at0 = part_row(work, (int64_t)s * p.Hkv * work.n_hg + pair + own_span.first, col % (16 * NC));
    const float* const pre_o = w.tile_o + pre0 * D + EPL * lane;
    const float* const own_o = p.part_o + at0 * D + EPL * lane;
    const int64_t pre_step = (int64_t)BR * D, own_step = (int64_t)work.per_part * D;
    auto load_o = [&](const float* at, float (&x)[EPL]) __attribute__((always_inline)) {
        if (EPL == 2) { const f32x2 v = *reinterpret_cast<const f32x2*>(at); x[0] = v[0]; x[EPL - 1] = v[1]; }
        else x[0] = at[0];
    };
    // the first parts' rows behind the requests of their references and sums (each behind a branch, of which the built code waits in front of some for what is on its way)
    f32x2 ml = {-INFINITY, 0.f}, pre = {-INFINITY, 0.f};
    if (lane < ns) ml = *reinterpret_cast<const f32x2*>(p.part_ml + (at0 + (int64_t)lane * work.per_part) * 2);
    if (lane < n_pre) pre = *reinterpret_cast<const f32x2*>(w.tile_ml + (pre0 + (int64_t)lane * BR) * 2);
    constexpr int kEarly = 4;
    float x_pre[8][EPL], x_own[8][EPL];
#pragma unroll
    for (int u = 0; u < kEarly; ++u) {
        if (n_pre > 0) load_o(pre_o + min(u, n_pre - 1) * pre_step, x_pre[u]);
        if (ns > 0) load_o(own_o + min(u, ns - 1) * own_step, x_own[u]);
    }
    const float top = wave_max(max2(ml[0], pre[0]));
    const float w_own = ml[0] > -INFINITY ? fast_exp2(ml[0] - top) : 0.f, w_pre = pre[0] > -INFINITY ? fast_exp2(pre[0] - top) : 0.f;
    const float all = lane_sum<64>(ml[1] * w_own + pre[1] * w_pre);
    float acc[EPL];
#pragma unroll
    for (int e = 0; e < EPL; ++e) acc[e] = 0.f;
    auto add = [&](const float* src, int64_t step, int n, float weight, float (&x)[8][EPL]) __attribute__((always_inline)) {
        for (int i0 = 0; i0 < n; i0 += 8) {
#pragma unroll
            for (int u = 0; u < 8; ++u)
                if (i0 > 0 || u >= kEarly) load_o(src + min(i0 + u, n - 1) * step, x[u]);
#pragma unroll
            for (int u = 0; u < 8; ++u) {
                const float wi = lane_value(weight, min(i0 + u, 63));
#pragma unroll
                for (int e = 0; e < EPL; ++e) acc[e] += i0 + u < n ? x[u][e] * wi : 0.f;
            }
        }
    };
    add(pre_o, pre_step, n_pre, w_pre, x_pre);
    add(own_o, own_step, ns, w_own, x_own);
    const float inv = all > 0.f ? 1.f / all : 0.f;
    uint16_t* dst = reinterpret_cast<uint16_t*>(p.out) + (int64_t)(info.lo + tok) * p.o2 + (int64_t)(g * p.n_rep + head) * p.o1 + EPL * lane;
    if (EPL == 2) *reinterpret_cast<uint32_t*>(dst) = T::pack2(acc[0] * inv, acc[EPL - 1] * inv);
    else dst[0] = (uint16_t)(T::pack2(acc[0] * inv, 0.f) & 0xffffu);
}

// Groups of 16 columns that a wave streams a sequence's own rows for together: two where there are more than one.  (us, one at a time / two, each at the best division of the workgroups;
// 32 heads on 8 of 128, sequences of 3 to 6 tokens behind 12000 rows: 24 with 10 to 900 own rows 54.7 / 53.7, of codes 60.1 / 58.9; 40 with 1000 to 6000 225 / 141, of codes 165 / 116;
// 64 heads, 24 with 10 to 3000 125 / 107; at head_dim 64, 60 with 1000 to 6000 175 / 114, of codes 146 / 112.)
static int64_t column_groups(int64_t n_col) { return n_col > 16 ? 2 : 1; }

// How a call is laid out, from its sizes alone.
struct SharedSizes { int64_t n_col, n_hg, per_part, parts, blocks, part_rows; size_t o_bytes, ml_bytes, tile_o_bytes, tile_ml_bytes, seq_bytes, bytes; };
static size_t lines(int64_t bytes) { return ((size_t)bytes + 255) / 256 * 256; }
static SharedSizes shared_sizes(int64_t n_seqs, int64_t n_groups, int64_t T, int64_t Hq, int64_t Hkv, int64_t D, int64_t max_q) {
    SharedSizes r{};
    const int64_t n_rep = Hq / Hkv;
    r.n_col = max_q * n_rep;
    const int64_t cols = 16 * column_groups(r.n_col);
    r.n_hg = (r.n_col + cols - 1) / cols;
    r.per_part = std::min<int64_t>(r.n_col, cols);
    const int64_t wgs = shared_wgs(D), block_rows = shared_waves(D) * 32;
    // shares and pairs; rows and shares (tile_row), those of groups that do not overlap
    r.parts = wgs * shared_waves(D) + n_seqs * Hkv * r.n_hg;
    r.blocks = T * n_rep / block_rows + n_groups;
    r.part_rows = T * n_rep + wgs / Hkv * block_rows;
    r.o_bytes = lines(r.parts * r.per_part * D * 4);
    r.ml_bytes = lines(r.parts * r.per_part * 2 * 4);
    r.tile_o_bytes = lines(r.part_rows * Hkv * D * 4);
    r.tile_ml_bytes = lines(r.part_rows * Hkv * 2 * 4);
    r.seq_bytes = lines((n_seqs + 1) * 16);
    r.bytes = r.o_bytes + r.ml_bytes + r.tile_o_bytes + r.tile_ml_bytes + r.seq_bytes + lines(n_groups * 16);
    return r;
}

// Whether the lines and the merge's rows are 32-bit numbers, were all contexts as long as the tables: of several thousand sequences with tables of a million rows they are not.
static bool fits_a_launch(int64_t n_seqs, int64_t n_groups, int64_t T, int64_t Hq, int64_t Hkv, int64_t D, int64_t max_context, int64_t max_q) {
    constexpr int64_t kMost = 0x7fffffffLL;
    if (T > (1 << 30) || T * Hq > kMost - 4096 || n_seqs > (1 << 24) || max_context > (1 << 30)) return false;
    const SharedSizes z = shared_sizes(n_seqs, n_groups, T, Hq, Hkv, D, max_q);
    return z.blocks * (max_context / 64 + kTileLead) <= kMost - 65536 && z.part_rows * Hkv <= kMost && n_seqs * Hkv * z.n_col <= kMost && n_seqs * Hkv * z.n_hg * ((max_context + 15) / 16 + 4) <= kMost - 65536;
}

// Whether a call is one for these kernels; others go to flash_attn_paged.  Longer chunks fill its blocks of rows with a single sequence's tokens.  And where all
// sequences' rows together are no more than the memory-side cache holds, a prefix that is read once for each of them comes from there, and one launch or two
// that know nothing of groups end sooner.  (us, shared / not, 400 own rows at most; 32 heads on 8 of 128: 8 sequences behind 4000 rows, 144 MB, 20.8 / 17.7, 4 behind
// 16000, 269 MB, 29.4 / 33.2, 16 behind 4000, 288 MB, 23.1 / 27.3, 64 behind 256, 172 MB, 24.9 / 23.1; 8 on 2 of 64: 64 behind 4000, 144 MB, 20.3 / 17.4, 32 behind 16000,
// 269 MB, 22.8 / 26.5; of codes: 8 behind 4000, 72 MB, 24.3 / 17.7, 16 behind 4000, 144 MB, 25.3 / 24.4, 64 behind 1000, 183 MB, 27.6 / 36.6.)  More than 16 columns
// are read once here and twice or more often there, which matters over codes and at head_dim 64 (3 to 6 tokens, 32 heads on 8 of 128, codes: 8 sequences behind 1000, 22 MB, 24.0 / 23.8, 8 behind
// 2000, 38 MB, 27.1 / 28.3, 8 behind 8000, 139 MB, 36.8 / 54.6; 16-bit 16 behind 2000, 154 MB, 30.4 / 29.3; 8 on 2 of 64: 32 behind 4000, 72 MB, 24.3 / 23.7, 32 behind 8000, 139 MB, 27.0 / 31.7;
// of codes 32 behind 2000, 19 MB, 20.2 / 22.5, 64 behind 8000, 139 MB, 34.1 / 59.4).  But every row of theirs makes partial results, whose way through memory short contexts do not pay for (64
// sequences of 3 to 6 tokens, 32 heads on 8 of 128, codes: behind 384 36.6 / 24.2, 768 38.9 / 36.6, 1536 45.3 / 60.9; 160 behind 768, 294 MB, 67.6 / 96.4; 16-bit 64 behind 768 38.5 / 26.8, behind 1536 42.3 / 44.1,
// 64 heads 59.0 / 48.7; 160 behind 1536, 1.1 GB, 118 / 131), nor does a prefix of two (60 sequences in groups of 2 / 3 / 4 behind 2000 with 1000 of their own, codes 84.5, 65.8, 56.8 / 65; with
// drafts 104, 84, 80 / 105; 16-bit 92, 75, 63 / 111; with drafts 114, 91, 81 / 86).  Of more columns there are more partial results, and past 32 of them own rows are read twice, so that what pays for them goes by
// their number (kSharedRowsPerColumn; 8 to 2000 sequences of 17 to 64 columns in tables no wider than contexts, 1208 calls: against the better one a call loses 14, 4.5, 16 and 11 % on average without this line, 3, 2, 4 and 5 with it (codes at
// head_dim 64 and 128, 16 bits at 64 and 128); 555 of 48 columns of codes behind 256 with 441 of their own at head_dim 64 343 / 139, 342 at 128 behind 320 with 248 225 / 144, 16-bit 508 of 64 behind 512 with 2627 221 / 114; 305 of 24 behind 5312 259 / 476).  The host knows the table's width, not the contexts: a table far wider than they are costs a short
// call 8 us.
constexpr int64_t kSharedRowsPerColumn[2][2] = {{100, 70}, {70, 25}};   // [codes][head_dim 128]
static bool shared_takes(bool eight, int64_t n_seqs, int64_t n_groups, int64_t T, int64_t Hq, int64_t Hkv, int64_t D, int64_t max_context, int64_t max_q) {
    const int64_t n_rep = Hq / Hkv, bytes = 2 * Hkv * D * (eight ? 1 : 2);   // of a row of all heads, k and v
    if (n_groups == 0 || Hkv > kMaxSharedHeads || (max_q > 1 && (n_rep > 16 || max_q * n_rep > 64))) return false;
    if (!fits_a_launch(n_seqs, n_groups, T, Hq, Hkv, D, max_context, max_q)) return false;
    const bool pairs = max_q * n_rep > 16;
    if (pairs && max_context < max_q * n_rep * kSharedRowsPerColumn[eight][D == 128]) return false;
    const int64_t rows = n_seqs * max_context;
    auto most = [&](int64_t total) { return rows >= total / bytes; };
    if (!pairs) return most(eight ? kSharedBytesCodes : kSharedBytes) && (!eight || n_seqs >= 3 * n_groups);
    if (eight) return most(kSharedBytesCodes) ? max_context >= 600 && n_seqs >= 2 * n_groups : most(kSharedBytesPairsCodes) && max_context >= 1000 && n_seqs >= 3 * n_groups;
    return most(D == 64 ? kSharedBytesPairs : kSharedBytes) && max_context >= (most(kSharedBytesLong) ? 1200 : 2000) && n_seqs >= 4 * n_groups;
}

template <class T, int D, bool FP8, int NC> static int launch_shared(const SharedWork& w, hipStream_t stream) {
    hipLaunchKernelGGL((shared_kernel<T, D, FP8, NC>), dim3(shared_wgs(D)), dim3(kSharedWaves<D> * 64), 0, stream, w);
    if (int rc = check_launch("shared_kernel")) return rc;
    const int64_t rows = (int64_t)w.d.p.n_seqs * w.d.p.Hkv * w.d.n_col;
    hipLaunchKernelGGL((shared_merge_kernel<T, D, kRows<FP8>, NC>), dim3((unsigned)((rows + 3) / 4)), dim3(256), 0, stream, w);
    return check_launch("shared_merge_kernel");
}
template <class T, int D, bool FP8> static int launch_columns(const SharedWork& w, hipStream_t stream) {
    return column_groups(w.d.n_col) == 1 ? launch_shared<T, D, FP8, 1>(w, stream) : launch_shared<T, D, FP8, 2>(w, stream);
}
template <class T> static int launch_shared_as(const SharedWork& w, int64_t D, bool eight, hipStream_t stream) {
    if (eight) return D == 128 ? launch_columns<T, 128, true>(w, stream) : launch_columns<T, 64, true>(w, stream);
    return D == 128 ? launch_columns<T, 128, false>(w, stream) : launch_columns<T, 64, false>(w, stream);
}

static int64_t bounded_tokens(int64_t T, int64_t max_q_len) { return max_q_len > 0 && max_q_len < T ? max_q_len : T; }

}  // namespace minfer_attn

using namespace minfer_attn;

MINFER_ATTN_EXPORT size_t minfer_flash_attn_paged_shared_workspace_bytes(int64_t n_seqs, int64_t n_groups, int64_t T, int64_t Hq, int64_t Hkv, int64_t D,
                                                                         int64_t max_context, int64_t max_q_len) {
    if (n_seqs <= 0 || n_groups < 0 || T <= 0 || Hq <= 0 || Hkv <= 0 || D <= 0 || max_context < 0 || Hq % Hkv != 0) return 0;
    const int64_t max_q = bounded_tokens(T, max_q_len);
    const size_t plain = minfer_flash_attn_paged_workspace_bytes(n_seqs, T, Hq, Hkv, D, max_context, max_q_len);
    size_t most = 0;   // of both kinds of pages
    for (const bool eight : {false, true})
        most = std::max(most, shared_takes(eight, n_seqs, n_groups, T, Hq, Hkv, D, max_context, max_q) ? shared_sizes(n_seqs, n_groups, T, Hq, Hkv, D, max_q).bytes : plain);
    return most;
}

MINFER_ATTN_EXPORT int minfer_flash_attn_paged_shared(int dtype, int page_type, const void* q, const minfer_kv_pages* pages, const int32_t* cu_seqlens,
                                                      const int32_t* ctx_lens, const int32_t* cu_groups, const int32_t* prefix_lens, void* out, int64_t n_seqs,
                                                      int64_t n_groups, int64_t T, int64_t Hq, int64_t Hkv, int64_t D, int64_t max_q_len,
                                                      const minfer_attn_strides* st, void* workspace, size_t workspace_bytes, void* stream_v) {
    clear_error();
    SharedWork w{};
    PagedParams& p = w.d.p;
    if (int rc = check_pages("flash_attn_paged_shared", dtype, page_type, pages, n_seqs, Hkv, D, p.c)) return rc;
    auto bad = [&](const char* what) { return fail(MINFER_ATTN_EINVAL, what); };
    if (Hq <= 0 || Hq % Hkv != 0) return bad("flash_attn_paged_shared: n_heads must be a positive multiple of n_kv_heads");
    if (Hq > 65535) return bad("flash_attn_paged_shared: n_heads > 65535 unsupported");
    if (!st) return bad("flash_attn_paged_shared: strides is null");
    if (n_seqs < 0 || T < 0 || max_q_len < 0 || n_groups < 0) return bad("flash_attn_paged_shared: negative size");
    if (n_groups > n_seqs) return bad("flash_attn_paged_shared: more groups than sequences");
    if (n_seqs == 0 || T == 0) return MINFER_ATTN_OK;
    if (!q || !out || !cu_seqlens || !ctx_lens) return bad("flash_attn_paged_shared: q, out, cu_seqlens and ctx_lens must be non-null");
    if (n_groups > 0 && (!cu_groups || !prefix_lens)) return bad("flash_attn_paged_shared: cu_groups and prefix_lens must be non-null");
    const int64_t max_q = bounded_tokens(T, max_q_len), max_context = (int64_t)p.c.width << p.c.page_log2;
    const bool eight = page_type == MINFER_FP8_E4M3;
    if (!shared_takes(eight, n_seqs, n_groups, T, Hq, Hkv, D, max_context, max_q))
        return minfer_flash_attn_paged(dtype, page_type, q, pages, cu_seqlens, ctx_lens, out, n_seqs, T, Hq, Hkv, D, max_q_len, st, workspace, workspace_bytes, stream_v);
    if (!aligned16(q) || !aligned16(out)) return bad("flash_attn_paged_shared: q and out must be 16-byte aligned");
    const int64_t s[4] = {st->q1, st->q2, st->o1, st->o2};
    for (int i = 0; i < 4; ++i)
        if (s[i] < 0 || s[i] % 8 != 0) return bad("flash_attn_paged_shared: strides of q and out must be non-negative multiples of 8 elements");
    const SharedSizes z = shared_sizes(n_seqs, n_groups, T, Hq, Hkv, D, max_q);
    if (!workspace || !aligned16(workspace) || workspace_bytes < z.bytes)
        return fail(MINFER_ATTN_EWORKSPACE, "flash_attn_paged_shared: workspace too small or misaligned (see minfer_flash_attn_paged_shared_workspace_bytes)");
    p.q = q; p.out = out; p.cu = cu_seqlens; p.ctx = ctx_lens;
    p.q1 = st->q1; p.q2 = st->q2; p.o1 = st->o1; p.o2 = st->o2;
    p.n_seqs = (int)n_seqs; p.T = (int)T; p.Hq = (int)Hq; p.Hkv = (int)Hkv; p.n_rep = (int)(Hq / Hkv);
    p.max_q = (int)max_q;
    p.scale_log2 = (float)(1.4426950408889634 / sqrt((double)D));
    p.inv_scale_log2 = (float)(sqrt((double)D) / 1.4426950408889634);
    char* at = (char*)workspace;
    p.part_o = (float*)at; at += z.o_bytes;
    p.part_ml = (float*)at; at += z.ml_bytes;
    w.tile_o = (float*)at; at += z.tile_o_bytes;
    w.tile_ml = (float*)at; at += z.tile_ml_bytes;
    w.seq_tab = (i32x4*)at; at += z.seq_bytes;
    w.group_tab = (i32x4*)at;
    w.d.n_col = (int)z.n_col; w.d.n_hg = (int)z.n_hg; w.d.per_part = (int)z.per_part;
    w.cu_groups = cu_groups; w.prefix = prefix_lens; w.n_groups = (int)n_groups;
    w.part_rows = (int)z.part_rows;
    return dtype == MINFER_ATTN_F16 ? launch_shared_as<F16>(w, D, eight, (hipStream_t)stream_v) : launch_shared_as<BF16>(w, D, eight, (hipStream_t)stream_v);
}
