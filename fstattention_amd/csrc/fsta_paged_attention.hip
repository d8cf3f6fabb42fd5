// Attention of a batch's new tokens (single tokens, prompt chunks, draft trees) over each sequence's pages, for gfx950.
//
// Rows of a sequence's work are (new token, query head of the group that shares a K/V head), token by token: a tile of 32 R
// rows sees one K/V head, so every key is read once for the whole group.  A wave owns 32 rows as the columns of
//     S^T = K_tile . Q^T      and      O^T += V_tile^T . P^T        (32x32x16 matrix instructions, 32 keys a tile)
// with a float32 base-2 online softmax in between; P stays in the registers the scores came in.  R waves share a tile of keys
// (row groups), S tiles are worked on at a time (key shares, joined at the end through LDS): (R, S) = (1, 4), (2, 2), (4, 1), (8, 1).
// Keys and values come page by page straight into an LDS ring (global -> LDS transfers of 1 KiB) through a buffer resource per 16
// rows; rows past the sequence's end read as zeros, pages outside the cache from a row of zeros, so that what lies in unused rows of
// a page can not turn a weight of zero into a NaN.
// 8-bit rows are widened to the type of Q and V to bfloat16; where Q is float16 the keys' powers of two go to the scores.
// What bounds it: few rows, reading keys once (64 sequences of 16 to 8192 keys, 8 K/V heads of 128, 251 MB: 50.8 us with
// the join, 4.9 TB/s; 8-bit, 16 of 8192 to 32768 keys, 607 MB: 119 us with the join, 5.1 TB/s); many rows, the matrix
// cores, whose products wait for the exponentials in between (4096 tokens after 16384, 32 heads: 1.24e12 operations in 1180 us, 1050
// TFLOP/s, where a large matrix product reaches 1200 to 1300); one short sequence, one launch and four round trips (9.8 us).
#include "fsta_paged_attention.h"

#include <algorithm>

namespace fsta {
namespace {

using namespace paged;

constexpr int kDecodeLeast = 16, kChunkLeast = 8;          // tiles of a run, at least

// ---- who does what --------------------------------------------------------------------------------------------------------
// Every sequence's rows are cut into tiles of tile_rows and, where that is faster, its keys into runs of at most `longest` tiles.
// The cut is a function of the lengths alone; every wave works it out for itself from the arrays (64 sequences at a time, a lane
// each: one round trip and a few prefix sums), so that no launch has to come before this one and the host never waits for a length.
// Of four cuts (none, and runs for 1, 2 or 3 rounds' worth of units) the one is taken whose units would be done first: rounds of
// workgroups times what a unit lasts, its start included, and joining the runs.  (Measured with every cut forced, us whole / for one,
// two, three rounds, 8 K/V heads of 128, a token each: 64 sequences of 16 to 8192 keys 153 / 55 / 57 / 51, 32 of 4096 keys 96 / 97 / 90 /
// 98, 40 of them 111 / 112 / 133 / 114, one of 16384 287 / 22 / 21 / 21; 2 sequences of 256 tokens on 1256 to 1500 keys, 32 heads: 45 /
// 35 / 38 / 50, 4 of them 47 / 61 / 61 / 63.  The estimate takes three, whole, three, one; two, whole: up to a tenth from the best.)
// From 65 sequences on, whose lengths a wave does not hold all at once, runs are for two rounds,
// in which few keys stay whole: 70 sequences of 16 to 8192 keys 178 / 102 / 95 / 86, 128 of 2048 to 4096 266 / 268 / 268 / 282, 256 of 16 to
// 2048 103 / 113 / 106 / 101.
struct Cut {
    uint32_t longest;              // tiles of keys in a run
    // (a batch has fewer than 2^30 rows; tile_rows is a power of two)
    __device__ __forceinline__ static int row_tiles(const SeqLens& s, const PagedAttnParams& p) {
        return (s.fresh * p.group + p.tile_rows - 1) >> p.row_shift;
    }
    __device__ __forceinline__ static int key_tiles(const SeqLens& s) { return max((s.keys + kTileN - 1) / kTileN, 1); }
    __device__ __forceinline__ uint32_t runs(const SeqLens& s) const { return ((uint32_t)key_tiles(s) + longest - 1) / longest; }
};

// Largest of the lanes up to and including this one
__device__ __forceinline__ uint32_t wave_prefix_max(uint32_t x) {
    auto from = [](uint32_t v, auto ctrl, auto rows) {
        return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, decltype(ctrl)::value, decltype(rows)::value, 0xf, false);
    };
    x = max(x, from(x, std::integral_constant<int, 0x111>{}, std::integral_constant<int, 0xf>{}));   // row_shr:1, 2, 4, 8
    x = max(x, from(x, std::integral_constant<int, 0x112>{}, std::integral_constant<int, 0xf>{}));
    x = max(x, from(x, std::integral_constant<int, 0x114>{}, std::integral_constant<int, 0xf>{}));
    x = max(x, from(x, std::integral_constant<int, 0x118>{}, std::integral_constant<int, 0xf>{}));
    x = max(x, from(x, std::integral_constant<int, 0x142>{}, std::integral_constant<int, 0xa>{}));   // row_bcast:15, :31
    x = max(x, from(x, std::integral_constant<int, 0x143>{}, std::integral_constant<int, 0xc>{}));
    return x;
}

struct Place {
    SeqLens s;
    int seq, row_tile, run, runs, part;      // part: of the tile's first run, -1 where the keys are not cut
};

// Tiles of keys in a run.  (In float: a rounding of 2^-24 moves a cut by nothing that counts.)
__device__ __forceinline__ uint32_t choose(const PagedAttnParams& p, const SeqLens& first, float work) {
    auto run_of = [&](int units) { return (uint32_t)fminf(fmaxf(ceilf(work / (float)units), (float)p.least_tiles), 1073741824.f); };
    if (p.batch.batch > 64) return run_of(p.run_units[1]);
    const uint32_t tiles = (uint32_t)Cut::row_tiles(first, p);
    const float keys = tiles ? (float)Cut::key_tiles(first) : 0.f;
    const float most = (float)lane_of(wave_prefix_max((uint32_t)keys), 63);
    float best = INFINITY;
    uint32_t longest = 1u << 30;
#pragma unroll
    for (int i = -1; i < 3; ++i) {
        const uint32_t run = i < 0 ? 1u << 30 : run_of(p.run_units[i < 0 ? 0 : i]);
        const float runs = ceilf(keys * __builtin_amdgcn_rcpf((float)run));
        const float units = (float)lane_of(wave_prefix_sum(tiles * (uint32_t)runs), 63) * (float)p.batch.kv_heads;
        const float lasts = fminf(most, (float)run) + p.unit_cost;
        const float done = (ceilf(units / p.slots) - 1.f) * (work / fmaxf(units, 1.f) + p.unit_cost) + lasts + (most > (float)run ? p.cut_cost + units * p.cut_unit_cost : 0.f);
        if (done < best) {
            best = done;
            longest = run;
        }
    }
    return longest;
}

// The first 64 sequences' lengths, and the cut
__device__ __forceinline__ SeqLens make_cut(const PagedAttnParams& p, int lane, Cut* cut) {
    const SeqLens first = seq_lens(p.batch, lane);       // (the first 64 sequences' lengths are loaded once)
    uint64_t cost = 0;
    for (int c = 0; c < p.batch.batch; c += 64) {
        const SeqLens s = c ? seq_lens(p.batch, c + lane) : first;
        // (summed in two pieces; from 2^49 on, where nothing is cut, it may be too small)
        const uint64_t mine = (uint64_t)Cut::row_tiles(s, p) * (uint64_t)Cut::key_tiles(s);
        const uint32_t low = (uint32_t)mine & 0xffffffu, high = (uint32_t)min(mine >> 24, (uint64_t)1 << 25);
        cost += lane_of(wave_prefix_sum(low), 63);
        cost += (uint64_t)lane_of(wave_prefix_sum(high), 63) << 24;
    }
    cut->longest = choose(p, first, (float)cost * (float)p.batch.kv_heads);
    return first;
}

// The item-th (tile of rows, run of keys) of the batch, or with JOINS the item-th tile whose keys are cut; the tiles of a
// sequence last ones first (causal: they have most keys).  False: there is no such item.
template <bool JOINS> __device__ __forceinline__ bool find_item(const PagedAttnParams& p, const SeqLens& first, const Cut& cut, uint32_t item, int lane, Place* out) {
    uint32_t parts = 0;
    for (int c = 0; c < p.batch.batch; c += 64) {
        const SeqLens s = c ? seq_lens(p.batch, c + lane) : first;
        const uint32_t tiles = (uint32_t)Cut::row_tiles(s, p), runs = cut.runs(s);
        const uint32_t cut_items = runs > 1 ? tiles * runs : 0u;
        const uint32_t mine = !JOINS ? tiles * runs : runs > 1 ? tiles : 0u;
        const uint32_t upto = wave_prefix_sum(mine), parts_upto = wave_prefix_sum(cut_items);
        const uint32_t all = lane_of(upto, 63);
        if (item < all) {
            const int who = __builtin_ctzll(__ballot(upto > item));
            out->seq = c + who;
            out->s.start = (int)lane_of((uint32_t)s.start, who);
            out->s.fresh = (int)lane_of((uint32_t)s.fresh, who);
            out->s.keys = (int)lane_of((uint32_t)s.keys, who);
            const uint32_t n_tiles = lane_of(tiles, who), n_runs = lane_of(runs, who);
            const uint32_t in_seq = item - (lane_of(upto, who) - lane_of(mine, who));
            const uint32_t t = JOINS ? in_seq : in_seq / n_runs;
            out->row_tile = (int)(n_tiles - 1 - t);
            out->run = JOINS ? 0 : (int)(in_seq - t * n_runs);
            out->runs = (int)n_runs;
            out->part = n_runs > 1 ? (int)(parts + lane_of(parts_upto, who) - lane_of(cut_items, who) + t * n_runs) : -1;
            return true;
        }
        item -= all;
        parts += lane_of(parts_upto, 63);
    }
    return false;
}

// ---- the kernel -----------------------------------------------------------------------------------------------------------

// 8-bit tiles: up to two row groups read them as they are and widen in registers; four share a widened copy.
template <int D, int R, int S, bool FP8> struct Shape {
    static constexpr bool kWiden = FP8 && R > 2;
    static constexpr int kStep = R >= 4 && !FP8 ? 2 : 1;                   // tiles worked on between barriers
    static constexpr int kStages = R == 8 ? 9 : R == 4 ? 5 : FP8 && R == 2 ? 4 : 2;
    using Raw = Fetch<D, R, FP8, kWiden>;
    static constexpr int kWideBytes = 2 * kTileN * D * 2;
    static constexpr int kPowerBytes = kTileN * 4;                          // behind a widened tile: its keys' powers of two
    static constexpr int kShareBytes = kStages * Raw::kBytes + (kWiden ? kWideBytes + kPowerBytes : 0);
    static_assert(!kWiden || kStep == 1, "one widened tile");
    static constexpr size_t kJoin = S > 1 ? (size_t)S * R * (32 * D + 64) * 4 : 0;
    static constexpr size_t kLds = (size_t)S * kShareBytes > kJoin ? (size_t)S * kShareBytes : kJoin;
};

// SPLIT: weights go to the matrix cores as pairs of bfloat16, hi + lo.  ONCE: no sequence has more rows than a tile, so nobody else
// reads a workgroup's keys.  Up to 64 rows that is asked for every sequence on its own, whatever the host knows; asked at every
// tile of 128 rows and more it costs 1 to 4 % (4096 tokens after 16384 1257 -> 1289 us, head_dim 64 460 -> 477).
template <bool BF16, int D, int R, int S, bool FP8, bool SPLIT, bool ONCE>
__global__ __launch_bounds__(R * S * 64, 2) void paged_attn_kernel(PagedAttnParams p) {
    using SH = Shape<D, R, S, FP8>;
    using F = typename SH::Raw;
    using G = RowGroup<BF16, D, FP8, FP8 && !SH::kWiden, SPLIT>;
    constexpr int kStages = SH::kStages, kStep = SH::kStep, kDTiles = G::kDTiles;
    extern __shared__ __attribute__((aligned(16))) unsigned char smem[];

    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int share = wave / R, group_of_rows = wave % R;

    // unit -> (item, K/V head): the heads of an item follow each other, so with 8 heads (or a divisor) the tiles of a head are
    // on one XCD (unit % 8) and share its L2
    const uint32_t item = blockIdx.x / (uint32_t)p.batch.kv_heads;
    const int head = (int)(blockIdx.x - item * (uint32_t)p.batch.kv_heads);
    Place at;
    Cut cut;
    const SeqLens lens = make_cut(p, lane, &cut);
    if (blockIdx.x == 0 && tid == 0) *p.run_length = cut.longest;        // (the join reads it)
    if (!find_item<false>(p, lens, cut, item, lane, &at)) return;
    const SeqLens s = at.s;

    // this unit's tiles of keys
    const int tile_keys = keys_of_tile(p, s, at.row_tile);
    const int tiles = (tile_keys + kTileN - 1) / kTileN;
    const int tile0 = (int)((int64_t)tiles * at.run / at.runs), tile1 = (int)((int64_t)tiles * (at.run + 1) / at.runs);
    const int my_tiles = (tile1 - tile0 - share + S - 1) / S;       // of this share (tile0 + share, + S, ...)
    const int steps = (tile1 - tile0 + S * kStep - 1) / (S * kStep);

    // this wave's rows
    const int row0 = at.row_tile << p.row_shift;                    // of the tile, among (token, head of the group)
    const int rows_left = min(s.fresh * p.group - row0, p.tile_rows);
    G rows(lane);
    const int half = rows.half, ql = rows.ql;
    const int my_row = group_of_rows * 32 + ql;                     // in the tile
    const bool has_rows = group_of_rows * 32 < rows_left;
    Rows mine = rows_of(p, s, head, row0, rows_left, group_of_rows * 32, ql);
    mine.sight.keep(p);
    rows.load_q(static_cast<const uint16_t*>(p.q) + (int64_t)(s.start + mine.token) * p.q_token_stride + (int64_t)mine.q_head * p.q_head_stride);
    rows.reset();

    // ---- ring of tiles ----------------------------------------------------------------------------------------------------
    unsigned char* ring = smem + share * SH::kShareBytes;
    const F fetch(p, head, group_of_rows, lane);
    const auto once = [&] {
        if constexpr (R < 4) return s.fresh * p.group <= p.tile_rows;
        else return std::bool_constant<ONCE>{};
    }();
    const const_i32 table = table_of(p, at.seq);
    int next_p0 = 0, next_p1 = 0;             // pages of the share's tile that is fetched next
    auto look_up = [&](int i) {
        if (i < my_tiles) {
            const int first = (tile0 + share + i * S) * kTileN;
            next_p0 = page_at(p, table, s.keys, first);
            next_p1 = p.batch.page_shift > 4 ? next_p0 : page_at(p, table, s.keys, first + 16);     // (tiles lie at multiples of 32)
        }
    };
    uint32_t bad_halves = 0;                  // two bits per slot: halves of its tile on pages outside the cache
    auto issue = [&](int i) {                 // the share's i-th tile into slot i % kStages
        const int slot = (int)((uint32_t)i % kStages), p0 = next_p0, p1 = next_p1;
        look_up(i + 1);
        const uint32_t bad = fetch.tile(p, s.keys, head, (tile0 + share + i * S) * kTileN, p0, p1, ring + slot * F::kBytes, lane, once);
        bad_halves = (bad_halves & ~(3u << (2 * slot))) | (bad << (2 * slot));
    };
    look_up(0);
    int issued = 0;
    if (my_tiles > 0) { issue(0); issued = 1; }
    rows.await_q();
    mine.sight.await_kept();
    // A wave that has a ring of its own refills a slot as soon as it is done with it; waves that share one, behind the next barrier.
    constexpr int kFill = R == 1 ? kStages : kStages - kStep;
    for (; issued < my_tiles && issued < kFill; ++issued) issue(issued);

    const uint32_t ring_lds = lds_addr(ring), wide_lds = ring_lds + kStages * F::kBytes;
    auto bad_of = [&](int i) { return (bad_halves >> (2 * (int)((uint32_t)i % kStages))) & 3u; };
    auto lies_at = [&](int i) { return SH::kWiden ? wide_lds : ring_lds + ((uint32_t)i % kStages) * F::kBytes; };
    auto first_of = [&](int i) { return (tile0 + share + i * S) * kTileN; };
    auto compute = [&](int i) {
        const int first = first_of(i);
        if (first > mine.sight.high_limit) return;
        const uint32_t bad = bad_of(i);
        rows.tile(lies_at(i), lies_at(i) + (SH::kWiden ? SH::kWideBytes : F::kDma * 1024), p.scale_log2e, bad || !mine.sight.whole(p, first), [&] { return mine.sight.word(p, first, bad); });
    };
    // 8-bit rows: the share's waves widen the landed tile into the 16-bit layout, once for all row groups: values times their powers
    // of two in bfloat16, keys in the type of Q (in float16 without their powers, which are laid down as floats)
    auto widen = [&](int i) {
        const uint32_t raw = ring_lds + ((uint32_t)i % kStages) * F::kBytes, wide = lies_at(i);
        constexpr int kPieces = 2 * kTileN * D / 16 / 64 / R;          // 16-byte pieces per lane
        u32x4 bytes[kPieces];
        uint32_t E[kPieces];
#pragma unroll
        for (int j = 0; j < kPieces; ++j) {
            const int piece = (group_of_rows * kPieces + j) * 64 + lane;
            bytes[j] = lds_read_b128(raw + piece * 16);
            asm volatile("ds_read_u8 %0, %1" : "=v"(E[j]) : "v"(raw + F::kDma * 1024 + piece / (D / 16)) : "memory");
        }
        lds_wait();
#pragma unroll
        for (int j = 0; j < kPieces; ++j) {
            const int piece = (group_of_rows * kPieces + j) * 64 + lane;
            const int r = piece / (D / 16), c = piece % (D / 16);      // r: 0..31 keys, 32..63 values
            const bool is_v = group_of_rows * kPieces + j >= kTileN * D / 16 / 64;      // (r >= kTileN, said for the whole wave)
            lds_tie(bytes[j]);
            lds_tie(E[j]);
            const uint32_t power = min(E[j], 254u) << 23;              // (exponents of unused rows may be anything)
            const float scale = __builtin_bit_cast(float, power);
            if constexpr (G::kScaleScores)
                if (!is_v && c == 0) lds_write_b32(wide + SH::kWideBytes + 4 * r, power);
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const uint32_t lo = bytes[j][2 * h], hi = bytes[j][2 * h + 1];
                const u32x4 w = is_v || BF16 ? widen8<true>(lo, hi, scale) : widen8<false>(lo, hi, 1.f);
                const int rr = r & (kTileN - 1);
                const int chunk = is_v ? v_chunk<D>(rr, 2 * c + h) : k_chunk<D>(rr, 2 * c + h);
                lds_write_b128(wide + (uint32_t)((is_v ? kTileN * D * 2 : 0) + rr * D * 2 + chunk * 16), w);
            }
        }
    };
    // A step's tiles have landed for everyone who reads them, and everyone is done with those before: their slots are refilled.
    auto arrive = [&](int step) {
        const int i = step * kStep;
        wait_tiles<F::kPerTile, kFill - kStep>(max(issued - min(i + kStep, my_tiles), 0));
        if constexpr (R > 1) {
            ring_barrier();
#pragma unroll
            for (int k = 0; k < kStep; ++k)
                if (issued < my_tiles) { issue(issued); ++issued; }
        }
    };
    int step = 0;
    bool arrived = false;
    if constexpr (kStep == 2) {               // steps of two tiles that all rows see whole, up to the first that is none (a loop of its
                                              // own: in one with the others the accumulators are copied at every step)
        const int whole_keys = has_rows ? min(mine.sight.low_limit + 1, p.mask == kTree ? mine.sight.old : s.keys) : 0;
        const int whole_steps = min(my_tiles / 2, (whole_keys / kTileN - tile0) / 2);
        for (; step < whole_steps; ++step) {
            arrive(step);
            if ((bad_of(2 * step) | bad_of(2 * step + 1)) != 0) {
                arrived = true;
                break;
            }
            rows.two_tiles(lies_at(2 * step), lies_at(2 * step + 1), p.scale_log2e);
        }
    }
    for (; step < steps; ++step) {
        if (!arrived) arrive(step);
        arrived = false;
        const int i = step * kStep, here = min(my_tiles - i, kStep);
        if constexpr (SH::kWiden) {
            for (int k = 0; k < here; ++k) widen(i + k);
            ring_barrier();
        }
        if (has_rows)
#pragma unroll 1
            for (int k = 0; k < here; ++k) compute(i + k);
        if constexpr (R == 1) {
            lds_wait();
            if (issued < my_tiles) { issue(issued); ++issued; }
        }
    }

    // ---- rows out: a lane has O[row][32 dt + 8 j + 4 half .. + 3], quad 4 dt + j ----------------------------------------------
    // (a row's first element for this lane: in o or in the workspace; null: nowhere)
    auto open_row = [&](float m_i, float l_tot, bool first) -> unsigned char* {
        const float lse = l_tot == 0.f ? -INFINITY : m_i + log2f(l_tot);
        if (at.part < 0) {
            // (worked out again: kept over the loop they cost registers that it needs)
            const int token = (int)((uint32_t)(row0 + my_row) / (uint32_t)p.group);
            const int64_t row = (int64_t)(s.start + token) * (p.batch.kv_heads * p.group) + head * p.group + (row0 + my_row) - token * p.group;
            if (p.lse && first && half == 0) p.lse[row] = lse;
            return reinterpret_cast<unsigned char*>(static_cast<uint16_t*>(p.o) + row * D + 4 * half);
        }
        if ((at.part + at.run + 1) * p.batch.kv_heads <= p.parts) {
            const int64_t row = ((int64_t)(at.part + at.run) * p.batch.kv_heads + head) * p.tile_rows + my_row;
            if (first && half == 0) p.part_lse[row] = lse;
            return reinterpret_cast<unsigned char*>(p.part_o + row * D + 4 * half);
        }
        return nullptr;
    };
    auto put = [&](unsigned char* to, int quad, f32x4 x) {
        if (at.part < 0) store_row<BF16>(reinterpret_cast<uint16_t*>(to) + 8 * quad, x[0], x[1], x[2], x[3]);
        else if (to) *reinterpret_cast<f32x4*>(reinterpret_cast<float*>(to) + 8 * quad) = x;
    };
    auto inverse = [](float l) { return l > 0.f ? 1.f / l : l == 0.f ? 0.f : l; };      // (NaN stays)
    auto& o = rows.o;
    auto quad_of = [&](int quad) {
        const int dt = quad / 4, j = quad % 4;
        return f32x4{o[dt][4 * j], o[dt][4 * j + 1], o[dt][4 * j + 2], o[dt][4 * j + 3]};
    };
    if constexpr (S > 1) {
        // The shares' sums meet in LDS, in the order of the shares; every wave joins and writes its part of the head dims, 16 bytes a
        // lane at a time.  (One wave joining all of it: 64 tokens on 256 keys 9.3 us instead of 8.4, 64 sequences of a token 59.5
        // instead of 57.3.)
        constexpr int kQuads = 4 * kDTiles, kPer = kQuads / S, kWaveFloats = 32 * D + 64;
        float* area = reinterpret_cast<float*>(smem) + (size_t)group_of_rows * kWaveFloats;
        float* mine_at = area + (size_t)share * R * kWaveFloats;
        const float l_mine = rows.row_sum();
        __syncthreads();
#pragma unroll
        for (int quad = 0; quad < kQuads; ++quad) reinterpret_cast<f32x4*>(mine_at)[quad * 64 + lane] = quad_of(quad);
        if (half == 0) {
            mine_at[32 * D + ql] = rows.m_i;
            mine_at[32 * D + 32 + ql] = l_mine;
        }
        __syncthreads();
        if (my_row >= rows_left) return;
        float m[S], f[S];
#pragma unroll
        for (int i = 0; i < S; ++i) m[i] = area[(size_t)i * R * kWaveFloats + 32 * D + ql];
        float m_i = m[0], l_tot = 0.f;
#pragma unroll
        for (int i = 1; i < S; ++i) m_i = fmaxf(m_i, m[i]);
#pragma unroll
        for (int i = 0; i < S; ++i) {
            f[i] = m[i] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m[i] - m_i);
            l_tot += area[(size_t)i * R * kWaveFloats + 32 * D + 32 + ql] * f[i];
        }
        unsigned char* to = open_row(m_i, l_tot, share == 0);
        const float inv = inverse(l_tot);
#pragma unroll
        for (int k = 0; k < kPer; ++k) {
            const int quad = share * kPer + k;
            f32x4 x = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int i = 0; i < S; ++i) x += reinterpret_cast<const f32x4*>(area + (size_t)i * R * kWaveFloats)[quad * 64 + lane] * f[i];
            put(to, quad, x * inv);
        }
    } else {
        if (my_row >= rows_left) return;
        const float l_tot = rows.row_sum(), inv = inverse(l_tot);
        unsigned char* to = open_row(rows.m_i, l_tot, true);
#pragma unroll
        for (int quad = 0; quad < 4 * kDTiles; ++quad) put(to, quad, quad_of(quad) * inv);
    }
}

// Joins the runs of a tile's keys, in an order that the run count alone decides: D / 4 lanes take a row and every SUBS-th run of
// it, four runs' loads in flight at a time; what they have is joined through LDS (tiles of 128 rows and more are in few runs: one
// share).  A workgroup takes ROWS rows at a time of a (tile whose keys are cut, K/V head).
template <bool BF16, int D, int ROWS>
__global__ __launch_bounds__(256) void paged_join_kernel(PagedAttnParams p) {
    constexpr int kLanes = D / 4, kSubs = 256 / kLanes / ROWS;
    __shared__ float shared_o[kSubs > 1 ? 256 : 1][5];
    __shared__ float shared_l[kSubs > 1 ? 256 : 1];
    const int tid = threadIdx.x, lane = tid & 63;
    const uint32_t item = blockIdx.x / (uint32_t)p.batch.kv_heads;
    const int head = (int)(blockIdx.x - item * (uint32_t)p.batch.kv_heads);
    Place at;
    if (!find_item<true>(p, seq_lens(p.batch, lane), Cut{*p.run_length}, item, lane, &at)) return;
    const int rows = min(at.s.fresh * p.group - (at.row_tile << p.row_shift), p.tile_rows);
    const int runs = max(min(at.runs, p.parts / p.batch.kv_heads - at.part), 0);
    const int my = tid / kLanes, sub = my / ROWS, col = 4 * (tid % kLanes);
    for (int r0 = blockIdx.y * ROWS; r0 < rows; r0 += gridDim.y * ROWS) {
        const int r = r0 + my % ROWS;
        float m = -INFINITY, sum = 0.f;
        f32x4 acc = {0.f, 0.f, 0.f, 0.f};
        if (r < rows) {
            const int64_t row0 = ((int64_t)at.part * p.batch.kv_heads + head) * p.tile_rows + r, step = (int64_t)p.batch.kv_heads * p.tile_rows;
            for (int i0 = sub; i0 < runs; i0 += 4 * kSubs) {
                float l[4];
                f32x4 x[4];
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const int64_t row = row0 + (int64_t)min(i0 + j * kSubs, runs - 1) * step;
                    l[j] = p.part_lse[row];
                    x[j] = *reinterpret_cast<const f32x4*>(p.part_o + row * D + col);
                }
                float top = m;
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    if (i0 + j * kSubs >= runs) l[j] = -INFINITY;
                    top = fmaxf(top, l[j]);
                }
                if (top == -INFINITY && !(l[0] != l[0] || l[1] != l[1] || l[2] != l[2] || l[3] != l[3])) continue;    // nothing seen so far
                const float back = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m - top);
                m = top;
                sum *= back;
                acc *= back;
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    if (l[j] == -INFINITY) continue;
                    const float w = __builtin_amdgcn_exp2f(l[j] - top);      // (a NaN stays one)
                    sum += w;
                    acc += x[j] * w;
                }
            }
        }
        if constexpr (kSubs > 1) {
            shared_l[tid] = m;
#pragma unroll
            for (int e = 0; e < 4; ++e) shared_o[tid][e] = acc[e];
            shared_o[tid][4] = sum;
            __syncthreads();
            if (sub == 0)
                for (int other = 1; other < kSubs; ++other) {
                    const int t = tid + other * ROWS * kLanes;
                    const float m_b = shared_l[t], sum_b = shared_o[t][4];
                    if (m_b == -INFINITY && sum_b == 0.f) continue;
                    const float top = fmaxf(m, m_b);
                    const float fa = m == -INFINITY && sum == 0.f ? 0.f : __builtin_amdgcn_exp2f(m - top);
                    const float fb = __builtin_amdgcn_exp2f(m_b - top);
                    m = top;
                    sum = sum * fa + sum_b * fb;
#pragma unroll
                    for (int e = 0; e < 4; ++e) acc[e] = acc[e] * fa + shared_o[t][e] * fb;
                }
            __syncthreads();
        }
        if (sub > 0 || r >= rows) continue;
        const float inv = sum == 0.f ? 0.f : 1.f / sum;
        const int flat = (at.row_tile << p.row_shift) + r;
        const int token = (int)((uint32_t)flat / (uint32_t)p.group);
        const int64_t out_row = (int64_t)(at.s.start + token) * (p.batch.kv_heads * p.group) + head * p.group + (flat - token * p.group);
        if (p.lse && col == 0) p.lse[out_row] = sum == 0.f ? -INFINITY : m + log2f(sum);
        const u32x2 w = {Mma<BF16>::pack_out(acc[0] * inv, acc[1] * inv), Mma<BF16>::pack_out(acc[2] * inv, acc[3] * inv)};
        *reinterpret_cast<u32x2*>(static_cast<uint16_t*>(p.o) + out_row * D + col) = w;
    }
}

// ---- host -----------------------------------------------------------------------------------------------------------------

// Rows of a workgroup's tile where there is much to do.  Up to 64 rows a sequence the keys are all there is to read, and pairs of waves
// share them out, at two workgroups per CU, so that one's start lies under the other's keys.  (Up to 32 rows tiles of 32, whose four
// waves have a ring each, fill the CU's LDS with one workgroup where rows are of 128 in 16 bits: 64 sequences of a token and 16 to 8192
// keys 57.9 us, by pairs 51.9; 200 of 64 to 128 keys 57.4 and 35.3; 124 of up to 40 keys, 16 K/V heads, 49.6 and 27.5; only a CU that
// has one unit misses the longer ring, 32 sequences of 4096 keys 92.3 and 97.2.  Of 64 or 8 bits two of them fit, and they are faster:
// 40.0 and 45.6 for 32 sequences of 500 to 8192 keys of 64.)  From 128 rows on every wave has rows of its own.  256 rows where there are two rounds of such
// tiles (4096 after 16384: 1221 -> 1189 us; with one round the last tiles of a causal chunk are waited for: 2048 tokens 63 -> 71 us).
// 8-bit tiles are widened by all waves together, behind a barrier more, which two workgroups per CU hide and one does not (2048
// tokens on 8192 keys, 32 query on 8 K/V heads, 348 -> 384 us; 343 now, with float16 queries and pairs of weights 461); head_dim 64 fits three workgroups of 128 rows on a CU.
int rows_for_rate(int64_t most_rows, int64_t all_rows, int32_t kv_heads, int32_t head_dim, bool fp8) {
    if (most_rows <= 32 && (head_dim == 64 || fp8)) return 32;
    if (most_rows <= 64) return 64;
    return head_dim == 128 && !fp8 && all_rows / 256 * kv_heads >= 2 * kCus ? 256 : 128;
}

// Where there is little, a call lasts as long as one workgroup, and smaller tiles, whose waves share out the keys, are done sooner
// as long as they are not much more than a card's worth.  (32 query on 8 K/V heads of 128, rows 128 / 64 / 32: 64 tokens on 256 keys
// 12.5 / 10.5 / 9.3 us, of 8 bits 16.0 / 11.4 / 9.6; 256 tokens on 256 keys 12.6 / 10.8 / 13.2, on 1024 keys 19.8 / 23.1 / 22.3; 5 x 38
// tokens of 4 K/V heads on 362 keys 17.5 / 15.8 / 13.9; 16 x 64 tokens on 250 keys 15.0 / 17.5 / 41; 32 tokens on 16384 keys 42 / 32 /
// 34; 64 tokens on 16384 keys 42 / 48 / 50.)  What the host knows of the keys is that the page table's rows hold no more.
int rows_of_tile(int rate, int64_t seqs, int64_t all_rows, int64_t most_keys, int32_t kv_heads) {
    const int64_t units32 = std::max((all_rows + 31) / 32, seqs) * kv_heads, units64 = std::max((all_rows + 63) / 64, seqs) * kv_heads;
    if (rate > 32 && most_keys <= kDecodeLeast * kTileN && units32 <= kCus * 3 / 4) return 32;
    if (rate > 64 && (units64 <= kCus / 16 || (units64 <= kCus / 2 && units64 * most_keys < kCus * kDecodeLeast * kTileN))) return 64;
    return rate;
}

// What choose weighs (slots: workgroups at a time, one per CU up to 64 rows, as tiles of 32 rows of 128 in 16 bits have it; two of 64 rows
// or of smaller tiles fit, and three of 128 rows at head_dim 64, which the estimate does not know), in the time a workgroup takes
// for a tile of keys (0.66 us alone on its CU with up to 64 rows; with 128 rows
// 0.9 us alone, and two share a CU at 1.05 us): a unit's start and end 4 to 5 us, with few rows
// half hidden under another's keys (2 tiles; 7: 16 sequences of 4 tokens 47.5 us instead of 45.7), the join's launch 5 us; with many rows it is the
// results of the runs, which go to memory and back, 64 KB a unit (4 sequences of 256 tokens, 32 K/V heads, 1256 to 1500 keys: cut
// 65 us, whole 49; the same 18 tiles for any number of units: 4 sequences of 256 tokens, 8 heads, 1500 keys 28.1 us instead of 24.5,
// 6 sequences of 1 to 130 tokens on up to 700 keys, 40 heads of 64, 20.7 instead of 15.2; 30 tiles: 256 tokens on 1024 keys 31 instead of 20).
struct Costs { float slots, unit, cut, cut_unit; };
Costs costs_of(int tile_rows) { return tile_rows >= 128 ? Costs{(tile_rows == 256 ? 1.f : 2.f) * kCus, 6.f, 0.f, 18.f / 512.f} : Costs{kCus, 2.f, 8.f, 0.f}; }

struct Sizes {
    int tile_rows;
    int64_t most_rows;          // of a sequence, as far as the host can guess
    int64_t sure_rows;          // .. and as it knows
    int64_t row_tiles;          // at most, over the batch
    int64_t items, parts;       // of all heads: parts
    int64_t cut_tiles;          // a head's
    int64_t floats;             // of workspace
    int run_units[3], least_tiles;
};
// Most rows of a sequence: by max_q_len, else as if every sequence had new tokens, where that can be
int64_t most_rows_of(int32_t batch, int32_t tokens, int32_t max_q_len, int group) {
    const int32_t most = max_q_len > 0 ? max_q_len : tokens >= batch ? tokens - batch + 1 : tokens;
    return (int64_t)std::min(most, tokens) * group;
}
Sizes sizes_of(int tile_rows, int32_t batch, int32_t tokens, int32_t max_q_len, int32_t heads, int32_t kv_heads, int32_t head_dim) {
    Sizes z;
    const int group = heads / kv_heads;
    z.most_rows = most_rows_of(batch, tokens, max_q_len, group);
    z.sure_rows = max_q_len > 0 ? z.most_rows : (int64_t)tokens * group;
    z.tile_rows = tile_rows;
    z.row_tiles = ((int64_t)tokens * group + (int64_t)(batch < tokens ? batch : tokens) * (z.tile_rows - 1)) / z.tile_rows;
    for (int i = 0; i < 3; ++i) z.run_units[i] = z.tile_rows == 256 ? kCus / 2 << i : (i + 1) * kCus;
    z.least_tiles = z.tile_rows == 32 ? kDecodeLeast : kChunkLeast;
    // a run has at least cost / run_units tiles (rounded: 2^-20 more), a tile of rows at most one run more than whole ones, and
    // no more tiles of rows are cut than there are, or than units were wanted
    const int64_t most = z.run_units[2], runs = (most + most / 256 + kv_heads) / kv_heads;
    z.items = z.row_tiles + runs;
    z.cut_tiles = z.row_tiles < runs ? z.row_tiles : runs;
    z.parts = (runs + z.cut_tiles) * kv_heads;
    z.floats = z.parts * z.tile_rows * (head_dim + 1) + 4;
    return z;
}

template <bool BF16, int D, int R, int S, bool FP8, bool ONCE>
int launch_units_of(const PagedAttnParams& p, int64_t units, hipStream_t stream) {
    // bfloat16 weights as pairs where the matrix cores wait for keys anyway, and where queries and results are float16: over 8-bit
    // values, which only bfloat16 holds whatever their scale
    constexpr bool kSplit = FP8 ? R < 4 || !BF16 : R < 4 && BF16;
    constexpr auto kernel = &paged_attn_kernel<BF16, D, R, S, FP8, kSplit, ONCE>;
    constexpr size_t lds = Shape<D, R, S, FP8>::kLds;
    if (units * R * S * 64 >= (int64_t)1 << 32) return fail(FSTA_EUNSUPPORTED, "fsta_paged_attention: %d tokens", p.batch.tokens);
    if constexpr (lds > 64 * 1024) {
        const int rc = allow_full_lds<kernel>();
        if (rc != FSTA_OK) return rc;
    }
    hipLaunchKernelGGL((paged_attn_kernel<BF16, D, R, S, FP8, kSplit, ONCE>), dim3((unsigned)units), dim3(R * S * 64), lds, stream, p);
    FSTA_HIP_OK(hipGetLastError());
    return FSTA_OK;
}

template <bool BF16, int D, int R, int S, bool FP8> int launch_units(const PagedAttnParams& p, int64_t units, const Sizes& z, hipStream_t stream) {
    if constexpr (R >= 4)
        if (z.sure_rows <= z.tile_rows) return launch_units_of<BF16, D, R, S, FP8, true>(p, units, stream);
    return launch_units_of<BF16, D, R, S, FP8, false>(p, units, stream);
}

template <bool BF16, int D, int ROWS> int launch_join(const PagedAttnParams& p, const Sizes& z, hipStream_t stream) {
    const int64_t items = z.cut_tiles;
    const int64_t rows = z.most_rows < z.tile_rows ? z.most_rows : z.tile_rows;
    // Most of them find that there is nothing to do, and one that has rows waits for two round trips: as many as are on the card
    // at a time.  (Half as many: 17 sequences of 28 heads, chunks and single tokens, 55.1 -> 53.5 us with the attention; 16
    // sequences of 4 tokens 55.1 -> 52.5; twice as many 53.0 and 53.2.)
    const int64_t wanted = (rows + ROWS - 1) / ROWS, room = 8 * kCus / (items * p.batch.kv_heads) + 1;
    const dim3 grid((unsigned)(items * p.batch.kv_heads), (unsigned)(wanted < room ? wanted : room));
    hipLaunchKernelGGL((paged_join_kernel<BF16, D, ROWS>), grid, dim3(256), 0, stream, p);
    FSTA_HIP_OK(hipGetLastError());
    return FSTA_OK;
}

template <bool BF16, int D, bool FP8> int launch_attention(const PagedAttnParams& p, const Sizes& z, hipStream_t stream) {
    const int64_t units = z.items * p.batch.kv_heads;
    int rc;
    if (z.tile_rows == 32) rc = launch_units<BF16, D, 1, 4, FP8>(p, units, z, stream);
    else if (z.tile_rows == 64) rc = launch_units<BF16, D, 2, 2, FP8>(p, units, z, stream);
    else if (z.tile_rows == 128) rc = launch_units<BF16, D, 4, 1, FP8>(p, units, z, stream);
    else if constexpr (D == 128 && !FP8) rc = launch_units<BF16, D, 8, 1, FP8>(p, units, z, stream);
    else rc = FSTA_EUNSUPPORTED;
    if (rc != FSTA_OK) return rc;
    // nothing is cut where no sequence can have more tiles than the shortest run has
    const int64_t most_tiles = (((int64_t)p.batch.width << p.batch.page_shift) + kTileN - 1) / kTileN;
    if (most_tiles <= z.least_tiles) return FSTA_OK;
    if (z.tile_rows == 32) return launch_join<BF16, D, 1>(p, z, stream);
    if (z.tile_rows == 64) return launch_join<BF16, D, 2>(p, z, stream);
    return launch_join<BF16, D, 1024 / D>(p, z, stream);
}

int check_heads(const char* who, int32_t batch, int32_t tokens, int32_t heads, int32_t kv_heads) {
    if (heads <= 0 || kv_heads <= 0 || heads % kv_heads) return fail(FSTA_EINVAL, "%s: heads=%d kv_heads=%d", who, heads, kv_heads);
    if ((int64_t)tokens * heads > 0x3fffffff) return fail(FSTA_EUNSUPPORTED, "%s: %d tokens of %d heads", who, tokens, heads);
    if (batch > 65536) return fail(FSTA_EUNSUPPORTED, "%s: batch=%d (at most 65536)", who, batch);
    return FSTA_OK;
}

}  // namespace
}  // namespace fsta

using namespace fsta;

extern "C" size_t fsta_paged_attention_workspace_bytes(int32_t batch, int32_t tokens, int32_t max_q_len, int32_t heads, int32_t kv_heads,
                                                       int32_t head_dim, int32_t cache_dtype) {
    if (batch <= 0 || tokens <= 0 || kv_heads <= 0 || heads <= 0 || heads % kv_heads || head_dim <= 0) return 0;
    // (whichever of its answers rows_of_tile gives)
    const int group = heads / kv_heads;
    const int rate = rows_for_rate(most_rows_of(batch, tokens, max_q_len, group), (int64_t)tokens * group, kv_heads, head_dim, cache_dtype == FSTA_FP8);
    int64_t floats = 0;
    for (const int rows : {32, 64, rate})
        if (rows <= rate) floats = std::max(floats, sizes_of(rows, batch, tokens, max_q_len, heads, kv_heads, head_dim).floats);
    return (size_t)floats * sizeof(float);
}

extern "C" int fsta_paged_attention(const void* q, int64_t q_token_stride, int64_t q_head_stride, const void* k_cache,
                                    const void* v_cache, const uint8_t* k_exponent, const uint8_t* v_exponent,
                                    const int32_t* page_table, const int32_t* kv_lens, const int32_t* q_starts,
                                    const uint32_t* tree_bits, int32_t tree_words, void* o, float* lse, int32_t batch, int32_t width,
                                    int32_t tokens, int32_t max_q_len, int32_t num_pages, int32_t page_size, int32_t heads,
                                    int32_t kv_heads, int32_t head_dim, int32_t dtype, int32_t cache_dtype, int32_t mask,
                                    float sm_scale, void* workspace, size_t workspace_bytes, void* stream) {
    const char* who = "fsta_paged_attention";
    PagedAttnParams p = {};
    p.batch = PagedBatch{page_table, kv_lens, q_starts, batch, width, num_pages, 0, kv_heads, tokens};
    int rc = check_paged_batch(who, p.batch, page_size, head_dim, cache_dtype, true);
    if (rc == FSTA_OK) rc = check_heads(who, batch, tokens, heads, kv_heads);
    if (rc != FSTA_OK) return rc;
    if (dtype != FSTA_F16 && dtype != FSTA_BF16) return fail(FSTA_EINVAL, "%s: dtype=%d", who, dtype);
    if (cache_dtype != FSTA_FP8 && cache_dtype != dtype) return fail(FSTA_EINVAL, "%s: cache_dtype=%d for dtype=%d", who, cache_dtype, dtype);
    if (mask != FSTA_PAGED_ALL && mask != FSTA_PAGED_CAUSAL && mask != FSTA_PAGED_TREE) return fail(FSTA_EINVAL, "%s: mask=%d", who, mask);
    if (!(sm_scale > 0.f) || !(sm_scale < INFINITY)) return fail(FSTA_EINVAL, "%s: sm_scale=%g (must be positive)", who, (double)sm_scale);
    if (tree_words < 0 || (mask == FSTA_PAGED_TREE && tree_words > 0 && !tree_bits)) return fail(FSTA_EINVAL, "%s: tree_words=%d without tree_bits", who, tree_words);
    if (tokens == 0) return FSTA_OK;
    if (batch == 0) return fail(FSTA_EINVAL, "%s: %d tokens of no sequence", who, tokens);
    if (width == 0 || num_pages == 0) return fail(FSTA_EINVAL, "%s: a cache without pages", who);
    if (!q || !o || !k_cache || !v_cache || (cache_dtype == FSTA_FP8 && (!k_exponent || !v_exponent))) return fail(FSTA_EINVAL, "%s: null pointer", who);
    if (misaligned(q, 16) || misaligned(o, 16) || misaligned(k_cache, 16) || misaligned(v_cache, 16) || ((q_token_stride | q_head_stride) & 7))
        return fail(FSTA_EINVAL, "%s: rows of q, o and the cache must be 16-byte aligned", who);
    if (misaligned(k_exponent, 4) || misaligned(v_exponent, 4) || misaligned(lse, 4) || misaligned(tree_bits, 4))
        return fail(FSTA_EINVAL, "%s: exponents, lse and tree_bits must be 4-byte aligned", who);
    const int64_t all_rows = (int64_t)tokens * (heads / kv_heads);
    const int rate = rows_for_rate(most_rows_of(batch, tokens, max_q_len, heads / kv_heads), all_rows, kv_heads, head_dim, cache_dtype == FSTA_FP8);
    const Sizes z = sizes_of(rows_of_tile(rate, batch < tokens ? batch : tokens, all_rows, (int64_t)width * page_size, kv_heads), batch, tokens, max_q_len, heads, kv_heads, head_dim);
    const size_t need = (size_t)z.floats * sizeof(float);
    if (!workspace || workspace_bytes < need) return fail(FSTA_EINVAL, "%s: needs %zu bytes of workspace, got %zu", who, need, workspace_bytes);
    if (misaligned(workspace, 16)) return fail(FSTA_EINVAL, "%s: the workspace must be 16-byte aligned", who);
    while ((1 << p.batch.page_shift) < page_size) ++p.batch.page_shift;
    p.q = q; p.q_token_stride = q_token_stride; p.q_head_stride = q_head_stride;
    p.k = k_cache; p.v = v_cache; p.k_exponent = k_exponent; p.v_exponent = v_exponent;
    p.o = o; p.lse = lse;
    p.tree_bits = tree_bits; p.tree_words = mask == FSTA_PAGED_TREE ? tree_words : 0; p.mask = mask;
    p.group = heads / kv_heads; p.tile_rows = z.tile_rows; p.row_shift = z.tile_rows == 32 ? 5 : z.tile_rows == 64 ? 6 : z.tile_rows == 128 ? 7 : 8; p.parts = (int32_t)z.parts; p.least_tiles = z.least_tiles;
    for (int i = 0; i < 3; ++i) p.run_units[i] = z.run_units[i];
    const Costs costs = costs_of(z.tile_rows);
    p.slots = costs.slots; p.unit_cost = costs.unit; p.cut_cost = costs.cut; p.cut_unit_cost = costs.cut_unit;
    p.scale_log2e = sm_scale * kLog2e;
    p.part_o = static_cast<float*>(workspace);
    p.part_lse = p.part_o + (size_t)z.parts * z.tile_rows * head_dim;
    p.run_length = reinterpret_cast<uint32_t*>(p.part_lse + (size_t)z.parts * z.tile_rows);
    hipStream_t st = static_cast<hipStream_t>(stream);
    const bool fp8 = cache_dtype == FSTA_FP8;
    if (dtype == FSTA_BF16) {
        if (head_dim == 128) return fp8 ? launch_attention<true, 128, true>(p, z, st) : launch_attention<true, 128, false>(p, z, st);
        return fp8 ? launch_attention<true, 64, true>(p, z, st) : launch_attention<true, 64, false>(p, z, st);
    }
    if (head_dim == 128) return fp8 ? launch_attention<false, 128, true>(p, z, st) : launch_attention<false, 128, false>(p, z, st);
    return fp8 ? launch_attention<false, 64, true>(p, z, st) : launch_attention<false, 64, false>(p, z, st);
}
