// Attention of a batch's new tokens (single tokens, prompt chunks, draft trees) over each sequence's pages, for gfx950.
//
// Rows of a sequence's work are (new token, query head of the group that shares a K/V head), token by token: a tile of 32 R
// rows sees one K/V head, so every key is read once for the whole group.  A wave owns 32 rows as the columns of
//     S^T = K_tile . Q^T      and      O^T += V_tile^T . P^T        (32x32x16 matrix instructions, 32 keys a tile)
// with a float32 base-2 online softmax in between; P stays in the registers the scores came in.  R waves share a tile of keys
// (row groups), S tiles are worked on at a time (key shares, joined at the end through LDS): (R, S) = (1, 4), (1, 1), (2, 2), (4, 1).
// Keys and values come page by page straight into an LDS ring (global -> LDS transfers of 1 KiB); rows that do not exist (past
// the sequence's end, on a page outside the cache) come from a row of zeros, so that what lies in unused rows of a page can not
// turn a weight of zero into a NaN.
#include "fsta_mfma_common.h"
#include "fsta_paged.h"

namespace fsta {
namespace {

using namespace mfma;


constexpr int kDecodeShares = 4, kDecodeUnits = 512, kMiddleUnits = 512, kChunkUnits = 256;
constexpr int kDecodeLeast = 16, kChunkLeast = 8;

enum Mask { kAll = 0, kCausal = 1, kTree = 2 };

struct PagedAttnParams {
    PagedBatch batch;
    const void* q;
    int64_t q_token_stride, q_head_stride;
    const void* k;
    const void* v;
    const uint8_t* k_exponent;
    const uint8_t* v_exponent;
    void* o;                       // [tokens, heads, D]
    float* lse;                    // [tokens, heads] or null
    const uint32_t* tree_bits;     // [tokens, tree_words]
    float* part_o;                 // [part][kv_heads][rows][D]
    float* part_lse;               // [part][kv_heads][rows]
    int32_t tree_words, mask, group, tile_rows, row_shift, parts;
    int32_t run_units, least_tiles; // units the launch is cut into where it has fewer, and the least tiles of a run
    float scale_log2e;
};

__device__ const uint32_t kZeroRow[4] = {0u, 0u, 0u, 0u};

// ---- who does what --------------------------------------------------------------------------------------------------------
// Every sequence's rows are cut into tiles of tile_rows and, where the launch would otherwise not fill the GPU, its keys into
// runs.  The cut is a function of the lengths alone; every wave works it out for itself from the arrays (64 sequences at a
// time, a lane each: one round trip and a prefix sum), so that no launch has to come before this one and the host never waits
// for a length.  A run has cost / run_units tiles, cost = all (tile of rows, tile of keys) pairs of the batch.
struct Cut {
    uint32_t longest;              // tiles of keys in a run
    // (a batch has fewer than 2^30 rows; tile_rows is a power of two)
    __device__ __forceinline__ static int row_tiles(const SeqLens& s, const PagedAttnParams& p) {
        return (s.fresh * p.group + p.tile_rows - 1) >> p.row_shift;
    }
    __device__ __forceinline__ static int key_tiles(const SeqLens& s) { return max((s.keys + kTileN - 1) / kTileN, 1); }
    __device__ __forceinline__ uint32_t runs(const SeqLens& s) const { return ((uint32_t)key_tiles(s) + longest - 1) / longest; }
};

struct Place {
    SeqLens s;
    int seq, row_tile, run, runs, part;      // part: of the tile's first run, -1 where the keys are not cut
};

__device__ __forceinline__ uint32_t lane_of(uint32_t x, int lane) { return (uint32_t)__builtin_amdgcn_readlane((int)x, lane); }

// The item-th (tile of rows, run of keys) of the batch, or with JOINS the item-th tile whose keys are cut; the tiles of a
// sequence last ones first (causal: they have most keys).  False: there is no such item.
template <bool JOINS> __device__ __forceinline__ bool find_item(const PagedAttnParams& p, uint32_t item, int lane, Place* out) {
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
    // (rounded up, in float: a rounding of 2^-24 moves the cut by nothing that counts, and both kernels round alike)
    const float longest = ceilf((float)cost * (float)p.batch.kv_heads / (float)p.run_units);
    const Cut cut{(uint32_t)fminf(fmaxf(longest, (float)p.least_tiles), 1073741824.f)};
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

// Number of keys that any row of a tile may see (its rows are tokens first .. last of the sequence's new ones)
__device__ __forceinline__ int keys_of_tile(const PagedAttnParams& p, const SeqLens& s, int row_tile) {
    if (p.mask != kCausal) return s.keys;
    const uint32_t last_row = (uint32_t)min((row_tile + 1) << p.row_shift, s.fresh * p.group) - 1u;
    return max(s.keys - s.fresh + (int)(last_row / (uint32_t)p.group) + 1, 0);
}

// ---- the kernel -----------------------------------------------------------------------------------------------------------

// 8-bit tiles: up to two row groups read them as they are and widen in registers; four share a widened copy.
template <int D, int R, int S, bool FP8> struct Shape {
    static constexpr bool kWiden = FP8 && R > 2;
    static constexpr int kStages = R == 4 ? 4 : FP8 ? 4 : 2;
    static constexpr int kRowBytes = FP8 ? D : 2 * D;             // a key's or a value's row in the cache
    static constexpr int kDma = 2 * kTileN * kRowBytes / 1024;    // transfers of a tile's K and V
    static constexpr int kPer = kDma / R;                         // of them a wave's
    static constexpr int kPerTile = kPer + (FP8 ? 1 : 0);         // (and one of the exponents)
    static constexpr int kRawBytes = kDma * 1024 + (FP8 ? 256 : 0);
    static constexpr int kWideBytes = 2 * kTileN * D * 2;
    static constexpr int kShareBytes = kStages * kRawBytes + (kWiden ? kWideBytes : 0);
    static constexpr size_t kJoin = (size_t)(S - 1) * R * (32 * D + 64) * 4;
    static constexpr size_t kLds = (size_t)S * kShareBytes > kJoin ? (size_t)S * kShareBytes : kJoin;
    static_assert(kDma % R == 0, "a wave has whole transfers");
};

// Positions of 16-byte chunks in rows of an 8-bit tile: keys are read 8 bytes from each of 32 rows, values 32 bytes from each
// of 16 (by the transposing read)
template <int D> __device__ __forceinline__ int k8_chunk(int row, int c) { return D == 128 ? c ^ ((row >> 1) & 7) : c ^ ((row >> 2) & 3); }
template <int D> __device__ __forceinline__ int v8_chunk(int row, int c) { return D == 128 ? c ^ (2 * ((row >> 1) & 3)) : c ^ (2 * ((row >> 2) & 1)); }

// 8 e4m3 bytes times a power of two, in the 16-bit type
template <bool BF16> __device__ __forceinline__ u32x4 widen8(uint32_t lo, uint32_t hi, float scale) {
    u32x4 w;
    if constexpr (BF16) {
        w[0] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, scale, false));
        w[1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, scale, true));
        w[2] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, scale, false));
        w[3] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, scale, true));
    } else {
        w[0] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(lo, scale, false));
        w[1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(lo, scale, true));
        w[2] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(hi, scale, false));
        w[3] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(hi, scale, true));
    }
    return w;
}

template <int N, typename F> __device__ __forceinline__ void static_for(F f) {
    if constexpr (N > 0) {
        static_for<N - 1>(f);
        f(std::integral_constant<int, N - 1>{});
    }
}
// Waits until at most N of this wave's LDS accesses are outstanding (they finish in order; scalar loads in between can only make
// it wait longer).
template <int N> __device__ __forceinline__ void wait_lds() { asm volatile("s_waitcnt lgkmcnt(%0)" : : "n"(N) : "memory"); }

template <bool DIRECT> struct VRaw { VPair x[2]; };        // values of 32 head dims x 32 keys as they come out of LDS
template <> struct VRaw<true> { u32x2 x[2]; };

// SPLIT: weights go to the matrix cores as pairs of bfloat16, hi + lo.  ONCE: every key is read by one workgroup only, past the
// caches.
template <bool BF16, int D, int R, int S, bool FP8, bool SPLIT, bool ONCE>
__global__ __launch_bounds__(R * S * 64, 2) void paged_attn_kernel(PagedAttnParams p) {
    using SH = Shape<D, R, S, FP8>;
    constexpr bool kDirect = FP8 && !SH::kWiden;
    using MM = Mma<BF16>;
    using PV = Mma<BF16 || kDirect>;          // weights times values: 8-bit values are exact in bfloat16 whatever their scale
    using Frag = typename MM::frag;
    using PFrag = typename PV::frag;
    constexpr int kStages = SH::kStages;
    constexpr int kSteps = D / 16;            // matrix instructions of a tile's scores
    constexpr int kDTiles = D / 32;           // 32-row tiles of O^T
    constexpr float kTrustedSum = BF16 ? 16777216.f : 32768.f;
    extern __shared__ __attribute__((aligned(16))) unsigned char smem[];

    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int share = wave / R, group_of_rows = wave % R;
    const int ql = lane & 31, half = lane >> 5;

    // unit -> (item, K/V head): the heads of an item follow each other, so with 8 heads (or a divisor) the tiles of a head are
    // on one XCD (unit % 8) and share its L2
    const uint32_t item = blockIdx.x / (uint32_t)p.batch.kv_heads;
    const int head = (int)(blockIdx.x - item * (uint32_t)p.batch.kv_heads);
    Place at;
    if (!find_item<false>(p, item, lane, &at)) return;
    const SeqLens s = at.s;
    const int old = s.keys - s.fresh;         // keys in front of the new tokens (negative: the first new ones have no place)

    // this unit's tiles of keys
    const int tile_keys = keys_of_tile(p, s, at.row_tile);
    const int tiles = (tile_keys + kTileN - 1) / kTileN;
    const int tile0 = (int)((int64_t)tiles * at.run / at.runs), tile1 = (int)((int64_t)tiles * (at.run + 1) / at.runs);
    const int my_tiles = (tile1 - tile0 - share + S - 1) / S;       // of this share (tile0 + share, + S, ...)
    const int steps = (tile1 - tile0 + S - 1) / S;

    // this wave's rows
    const int row0 = at.row_tile << p.row_shift;                    // of the tile, among (token, head of the group)
    const int rows_left = min(s.fresh * p.group - row0, p.tile_rows);
    const int my_row = group_of_rows * 32 + ql;                     // in the tile
    const bool has_rows = group_of_rows * 32 < rows_left;
    const uint32_t group = (uint32_t)p.group;
    const int token = (int)((uint32_t)(row0 + min(my_row, rows_left - 1)) / group);
    const int q_head = head * p.group + (row0 + min(my_row, rows_left - 1)) - token * p.group;
    const int first_token = (int)((uint32_t)(row0 + group_of_rows * 32) / group);
    const int last_token = (int)((uint32_t)(row0 + min(group_of_rows * 32 + 31, rows_left - 1)) / group);
    const int limit = p.mask == kCausal ? old + token : s.keys - 1;                  // this row's last key
    const int low_limit = p.mask == kCausal ? old + first_token : s.keys - 1;        // of the wave's rows, the least and
    const int high_limit = p.mask == kCausal ? old + last_token : s.keys - 1;        // the greatest

    // ---- Q: B operand of S^T, lane holds Q[row][16 ks + 8 half .. + 7] -----------------------------------------------------
    Frag qf[kSteps];
    {
        const uint16_t* src = static_cast<const uint16_t*>(p.q) + (int64_t)(s.start + token) * p.q_token_stride + (int64_t)q_head * p.q_head_stride;
#pragma unroll
        for (int ks = 0; ks < kSteps; ++ks) {
            const u32x4 raw = *reinterpret_cast<const u32x4*>(src + 16 * ks + 8 * half);
            qf[ks] = __builtin_bit_cast(Frag, raw);
        }
    }

    // ---- ring of tiles ----------------------------------------------------------------------------------------------------
    unsigned char* ring = smem + share * SH::kShareBytes;
    constexpr int kLanesPerRow = SH::kRowBytes / 16, kRowsPerDma = 64 / kLanesPerRow;
    const int page_rows = 1 << p.batch.page_shift;
    uint32_t dma_off[SH::kPer];               // this lane's piece, from the start of its 16 rows
    int dma_row[SH::kPer];
    bool dma_is_v[SH::kPer];
#pragma unroll
    for (int i = 0; i < SH::kPer; ++i) {
        const int u = group_of_rows * SH::kPer + i;
        dma_is_v[i] = u >= SH::kDma / 2;
        const int r = (u % (SH::kDma / 2)) * kRowsPerDma + lane / kLanesPerRow;
        const int slot = lane % kLanesPerRow;
        const int chunk = SH::kWiden ? slot : FP8 ? (dma_is_v[i] ? v8_chunk<D>(r, slot) : k8_chunk<D>(r, slot)) : dma_is_v[i] ? v_chunk<D>(r, slot) : k_chunk<D>(r, slot);
        dma_row[i] = r;
        dma_off[i] = (uint32_t)((r & 15) * SH::kRowBytes + chunk * 16);
    }
    // Pages of a tile's two 16-key halves, by scalar loads (through the constant address space: a load the compiler takes for a
    // vector one it would wait for with vmcnt(0), i.e. for the whole ring), one tile ahead of their use.
    typedef const int32_t __attribute__((address_space(4))) * const_i32;
    const const_i32 table = (const_i32)(uintptr_t)(p.batch.page_table + (size_t)at.seq * p.batch.width);
    auto page_of = [&](int tile, int g) {
        return table[__builtin_amdgcn_readfirstlane(min(tile * kTileN + 16 * g, s.keys - 1) >> p.batch.page_shift)];
    };
    int next_p0 = 0, next_p1 = 0;             // of the share's tile that is issued next
    auto look_up = [&](int i) {
        if (i < my_tiles) {
            next_p0 = page_of(tile0 + share + i * S, 0);
            next_p1 = page_of(tile0 + share + i * S, 1);
        }
    };
    typedef const void __attribute__((address_space(1))) * global_ptr;
    typedef void __attribute__((address_space(3))) * lds_ptr;
    uint32_t bad_halves = 0;                  // two bits per slot: halves of its tile on pages outside the cache
    auto issue = [&](int i) {                 // the share's i-th tile into slot i % kStages
        const int tile = tile0 + share + i * S, slot = i % kStages;
        const int first = tile * kTileN;
        const bool ok0 = (unsigned)next_p0 < (unsigned)p.batch.num_pages, ok1 = (unsigned)next_p1 < (unsigned)p.batch.num_pages;
        const int64_t row_0 = (((int64_t)(ok0 ? next_p0 : 0) * p.batch.kv_heads + head) << p.batch.page_shift) + (first & (page_rows - 1));
        const int64_t row_1 = (((int64_t)(ok1 ? next_p1 : 0) * p.batch.kv_heads + head) << p.batch.page_shift) + ((first + 16) & (page_rows - 1));
        look_up(i + 1);
        bad_halves = (bad_halves & ~(3u << (2 * slot))) | ((ok0 ? 0u : 1u) << (2 * slot)) | ((ok1 ? 0u : 2u) << (2 * slot));
        unsigned char* dst = ring + slot * SH::kRawBytes;
        auto half_of = [&](int j) { return (((group_of_rows * SH::kPer + j) % (SH::kDma / 2)) * kRowsPerDma) / 16; };
        auto base_of = [&](int j) { return static_cast<const unsigned char*>(dma_is_v[j] ? p.v : p.k) + (half_of(j) ? row_1 : row_0) * SH::kRowBytes; };
        if (first + kTileN <= s.keys && ok0 && ok1) {
#pragma unroll
            for (int j = 0; j < SH::kPer; ++j)
                __builtin_amdgcn_global_load_lds((global_ptr)(base_of(j) + dma_off[j]), (lds_ptr)(dst + (group_of_rows * SH::kPer + j) * 1024), 16, 0, ONCE ? 2 : 0);
        } else {
#pragma unroll
            for (int j = 0; j < SH::kPer; ++j) {
                const bool here = first + dma_row[j] < s.keys && (half_of(j) ? ok1 : ok0);
                const unsigned char* src = here ? base_of(j) + dma_off[j] : reinterpret_cast<const unsigned char*>(kZeroRow);
                __builtin_amdgcn_global_load_lds((global_ptr)src, (lds_ptr)(dst + (group_of_rows * SH::kPer + j) * 1024), 16, 0, 0);
            }
        }
        if constexpr (FP8) {                  // exponents of the 32 keys, then of the 32 values, four to a lane
            const int l = lane & 15, g = (l >> 2) & 1;
            const uint8_t* src = ((l & 8) ? p.v_exponent : p.k_exponent) + (g ? row_1 : row_0) + 4 * (l & 3);
            const bool here = first + 16 * g < s.keys && (g ? ok1 : ok0);
            src = here ? src : reinterpret_cast<const uint8_t*>(kZeroRow);
            __builtin_amdgcn_global_load_lds((global_ptr)src, (lds_ptr)(dst + SH::kDma * 1024), 4, 0, 0);
        }
    };
    look_up(0);
    // A wave that has a ring of its own refills a slot as soon as it is done with it; waves that share one, behind the next barrier.
    // (The Q rows are waited for here, behind the first tile's requests: left to their first use inside the loop, the wait would be
    // one for every transfer on its way, at every tile.)
    int issued = 0;
    if (my_tiles > 0) { issue(0); issued = 1; }
#pragma unroll
    for (int ks = 0; ks < kSteps; ++ks) lds_tie(qf[ks]);
    for (; issued < my_tiles && issued < (R == 1 ? kStages : kStages - 1); ++issued) issue(issued);

    float m_i = -INFINITY, l_i = 0.f;
    f32x16 o[kDTiles];
#pragma unroll
    for (int dt = 0; dt < kDTiles; ++dt)
#pragma unroll
        for (int i = 0; i < 16; ++i) o[dt][i] = 0.f;

    const uint32_t k_lane0 = (uint32_t)(ql * D + k_chunk<D>(ql, half) * 8) * 2;
    const int tr_row = 4 * half + ((lane & 15) >> 2), tr_col = 16 * ((lane >> 4) & 1) + 4 * (lane & 3);
    const uint32_t v_lane0 = (uint32_t)(tr_row * D + v_chunk<D>(tr_row, tr_col >> 3) * 8 + (tr_col & 7)) * 2;
    // (8-bit tiles: rows of D bytes; the transposing read hands a lane 8 keys, four from either 8-key half)
    const uint32_t k8_lane0 = (uint32_t)(ql * D + k8_chunk<D>(ql, 0) * 16 + 8 * half);
    const int tr8_row = 4 * half + ((lane & 15) >> 1) + ((lane & 8) ? 4 : 0);
    const uint32_t v8_lane0 = (uint32_t)(tr8_row * D + v8_chunk<D>(tr8_row, (lane >> 4) & 1) * 16 + 8 * (lane & 1));
    const float sc = p.scale_log2e;

    auto compute = [&](int i, const unsigned char* tile_lds) {
        const int tile = tile0 + share + i * S, first = tile * kTileN;
        if (!has_rows || first > high_limit) return;
        // S^T
        f32x16 sv;
#pragma unroll
        for (int e = 0; e < 16; ++e) sv[e] = 0.f;
        // (K fragments: all requested, then used as they arrive; LDS reads come back in order)
        const uint32_t exps = lds_addr(tile_lds) + SH::kDma * 1024;      // (8-bit tiles read as they are)
        uint32_t v_exp[4];
        if constexpr (kDirect) {
            const uint32_t k_addr0 = lds_addr(tile_lds) + k8_lane0;
            uint32_t E;
            asm volatile("ds_read_u8 %0, %1" : "=v"(E) : "v"(exps + ql) : "memory");
            u32x2 raw[kSteps];
#pragma unroll
            for (int ks = 0; ks < kSteps; ++ks) raw[ks] = lds_read_b64(k_addr0 ^ (uint32_t)(ks << 4));
#pragma unroll
            for (int j = 0; j < 4; ++j) v_exp[j] = lds_read_b32(exps + kTileN + 8 * j + 4 * half);
            wait_lds<kSteps + 4>();
            lds_tie(E);
            const float scale = __builtin_bit_cast(float, min(E, 254u) << 23);     // (exponents of unused rows may be anything)
            static_for<kSteps>([&](auto ks) {
                constexpr int k = decltype(ks)::value;
                wait_lds<kSteps + 3 - k>();
                lds_tie(raw[k]);
                sv = MM::mfma(__builtin_bit_cast(Frag, widen8<BF16>(raw[k][0], raw[k][1], scale)), qf[k], sv);
            });
            lds_wait();
#pragma unroll
            for (int j = 0; j < 4; ++j) lds_tie(v_exp[j]);
        } else {
            const uint32_t k_addr0 = lds_addr(tile_lds) + k_lane0;
            u32x4 raw[kSteps];
#pragma unroll
            for (int ks = 0; ks < kSteps; ++ks) raw[ks] = lds_read_b128(k_addr0 ^ (uint32_t)(ks << 5));
            static_for<kSteps>([&](auto ks) {
                constexpr int k = decltype(ks)::value;
                wait_lds<kSteps - 1 - k>();
                lds_tie(raw[k]);
                sv = MM::mfma(__builtin_bit_cast(Frag, raw[k]), qf[k], sv);
            });
        }
        // which of the tile's keys this lane's row sees
        const uint32_t bad = (bad_halves >> (2 * (i % kStages))) & 3u;
        const bool tree = p.mask == kTree && first + kTileN > old;
        if (bad || tree || first + kTileN - 1 > low_limit) {
            const int rel = limit - first;
            uint32_t word = rel >= 31 ? ~0u : rel < 0 ? 0u : (2u << rel) - 1u;
            if (bad & 1u) word &= 0xffff0000u;
            if (bad & 2u) word &= 0x0000ffffu;
            if (tree) {                       // keys in front of the new tokens are seen by all, the others by their bit
                const int number = first - old;
                const int wi = number >> 5, sh = number & 31;
                const uint32_t* bits = p.tree_bits + (int64_t)(s.start + token) * p.tree_words;
                const uint32_t lo = wi < 0 ? ~0u : wi < p.tree_words ? bits[wi] : 0u;
                const uint32_t hi = wi + 1 < 0 ? ~0u : wi + 1 < p.tree_words ? bits[wi + 1] : 0u;
                word &= sh ? (lo >> sh) | (hi << (32 - sh)) : lo;
            }
            const uint32_t mine = word >> (4 * half);
#pragma unroll
            for (int e = 0; e < 16; ++e)
                if (!((mine >> (8 * (e / 4) + e % 4)) & 1u)) sv[e] = -INFINITY;
        }
        // Weights against the running maximum as it stands (a power of two on a row's weights cancels in O / l); the tile's
        // own maximum is only looked for when a sum gets large, or at the first tile.
        float pw[16], sum = 0.f;
        const float neg_m = m_i == -INFINITY ? 0.f : -m_i;
#pragma unroll
        for (int e = 0; e < 16; ++e) {
            pw[e] = __builtin_amdgcn_exp2f(__builtin_fmaf(sv[e], sc, neg_m));
            sum += pw[e];
        }
        const bool redo = !(sum <= kTrustedSum) || m_i == -INFINITY;
        if (__ballot(redo) != 0ull) {
            float mx = -INFINITY;
#pragma unroll
            for (int e = 0; e < 16; ++e) mx = fmaxf(mx, sv[e]);
            float a, b;
            swap_halves(mx, false, a, b);
            mx = fmaxf(a, b) * sc;
            const bool raise = mx > m_i + kRescaleSlack || (m_i == -INFINITY && mx > -INFINITY);
            const float alpha = raise ? __builtin_amdgcn_exp2f(m_i - mx) : 1.f;
            if (raise) m_i = mx;
            l_i *= alpha;
#pragma unroll
            for (int dt = 0; dt < kDTiles; ++dt)
#pragma unroll
                for (int e = 0; e < 16; ++e) o[dt][e] *= alpha;
            const float neg = m_i == -INFINITY ? 0.f : -m_i;
            sum = 0.f;
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                pw[e] = __builtin_amdgcn_exp2f(__builtin_fmaf(sv[e], sc, neg));
                sum += pw[e];
            }
        }
        l_i += sum;
        if constexpr (kDirect) {              // the values' powers of two go to the weights (exponents of unused rows may be anything)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const uint32_t four = v_exp[j];
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    pw[4 * j + e] *= __builtin_bit_cast(float, min((four >> (8 * e)) & 255u, 254u) << 23);
            }
        }
        PFrag ph[2], pl[2];
#pragma unroll
        for (int k2 = 0; k2 < 2; ++k2) {
            u32x4 hi4, lo4;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const float a = pw[8 * k2 + 2 * e], b = pw[8 * k2 + 2 * e + 1];
                const uint32_t hi = PV::pack(a, b);
                hi4[e] = hi;
                if (SPLIT) lo4[e] = PV::pack(a - PV::low(hi), b - PV::high(hi));
            }
            ph[k2] = __builtin_bit_cast(PFrag, hi4);
            if (SPLIT) pl[k2] = __builtin_bit_cast(PFrag, lo4);
        }
        // O^T (the fragments of the next 32 head dims are requested before the products of these)
        auto read_v = [&](int dt, VRaw<kDirect>& f) {
            if constexpr (kDirect) {
                const uint32_t addr = (lds_addr(tile_lds) + (uint32_t)(kTileN * D) + v8_lane0) ^ (uint32_t)(dt << 5);
                asm volatile("ds_read_b64_tr_b8 %0, %1" : "=v"(f.x[0]) : "v"(addr) : "memory");
                asm volatile("ds_read_b64_tr_b8 %0, %1 offset:%2" : "=v"(f.x[1]) : "v"(addr), "n"(16 * D) : "memory");
            } else {
                const uint32_t addr = (lds_addr(tile_lds) + (uint32_t)(kTileN * D * 2) + v_lane0) ^ (uint32_t)(dt << 6);
                f.x[0].a = lds_read_tr16(addr);
                f.x[0].b = lds_read_tr16_at<8 * D * 2>(addr);
                f.x[1].a = lds_read_tr16_at<16 * D * 2>(addr);
                f.x[1].b = lds_read_tr16_at<24 * D * 2>(addr);
            }
        };
        VRaw<kDirect> raw_v[kDTiles];
        read_v(0, raw_v[0]);
        static_for<kDTiles>([&](auto t) {
            constexpr int dt = decltype(t)::value;
            if constexpr (dt + 1 < kDTiles) {
                read_v(dt + 1, raw_v[dt + 1]);
                wait_lds<kDirect ? 2 : 4>();
            } else {
                lds_wait();
            }
            PFrag f[2];
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                if constexpr (kDirect) {
                    lds_tie(raw_v[dt].x[h]);
                    f[h] = __builtin_bit_cast(PFrag, widen8<true>(raw_v[dt].x[h][0], raw_v[dt].x[h][1], 1.f));
                } else {
                    lds_tie(raw_v[dt].x[h].a);
                    lds_tie(raw_v[dt].x[h].b);
                    f[h] = __builtin_bit_cast(PFrag, raw_v[dt].x[h]);
                }
            }
            o[dt] = PV::mfma(f[0], ph[0], o[dt]);
            o[dt] = PV::mfma(f[1], ph[1], o[dt]);
            if (SPLIT) {
                o[dt] = PV::mfma(f[0], pl[0], o[dt]);
                o[dt] = PV::mfma(f[1], pl[1], o[dt]);
            }
        });
    };

    // 8-bit rows: the share's waves widen the landed tile into the 16-bit layout, once for all row groups
    auto widen = [&](int i) {
        const uint32_t raw = lds_addr(ring + (i % kStages) * SH::kRawBytes);
        const uint32_t wide = lds_addr(ring + kStages * SH::kRawBytes);
        constexpr int kPieces = 2 * kTileN * D / 16 / 64 / R;          // 16-byte pieces per lane
#pragma unroll
        for (int j = 0; j < kPieces; ++j) {
            const int piece = (group_of_rows * kPieces + j) * 64 + lane;
            const int r = piece / (D / 16), c = piece % (D / 16);      // r: 0..31 keys, 32..63 values
            const bool is_v = r >= kTileN;
            u32x4 bytes = lds_read_b128(raw + piece * 16);
            uint32_t E;
            asm volatile("ds_read_u8 %0, %1" : "=v"(E) : "v"(raw + SH::kDma * 1024 + r) : "memory");
            lds_wait();
            lds_tie(bytes);
            lds_tie(E);
            const float scale = __builtin_bit_cast(float, min(E, 254u) << 23);     // (exponents of unused rows may be anything)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const u32x4 w = widen8<BF16>(bytes[2 * h], bytes[2 * h + 1], scale);
                const int rr = r & (kTileN - 1);
                const int chunk = is_v ? v_chunk<D>(rr, 2 * c + h) : k_chunk<D>(rr, 2 * c + h);
                lds_write_b128(wide + (uint32_t)((is_v ? kTileN * D * 2 : 0) + rr * D * 2 + chunk * 16), w);
            }
        }
    };

    constexpr int kAhead = R == 1 ? kStages - 1 : kStages - 2;     // tiles that may be on their way behind the one that is waited for
    for (int i = 0; i < steps; ++i) {
        // tile i has landed for everyone who reads it, and everyone is done with the tile before it: its slot is refilled
        if (issued - i - 1 >= kAhead) wait_vmcnt<kAhead * SH::kPerTile>();
        else wait_tiles_outstanding<SH::kPerTile>(max(issued - i - 1, 0));
        auto refill = [&]() { if (issued < my_tiles) { issue(issued); ++issued; } };
        if constexpr (R > 1) { ring_barrier(); refill(); }
        if constexpr (SH::kWiden) {
            if (i < my_tiles) widen(i);
            ring_barrier();
            if (i < my_tiles) compute(i, ring + kStages * SH::kRawBytes);
        } else {
            if (i < my_tiles) compute(i, ring + (i % kStages) * SH::kRawBytes);
        }
        if constexpr (R == 1) { lds_wait(); refill(); }
    }

    // ---- join of the shares: through LDS, in the order of the shares --------------------------------------------------------
    float l_tot;
    {
        float a, b;
        swap_halves(l_i, false, a, b);
        l_tot = a + b;
    }
    if constexpr (S > 1) {
        float* area = reinterpret_cast<float*>(smem);
        constexpr int kWaveFloats = 32 * D + 64;
        __syncthreads();
        if (share > 0) {
            float* mine = area + (size_t)((share - 1) * R + group_of_rows) * kWaveFloats;
#pragma unroll
            for (int dt = 0; dt < kDTiles; ++dt)
#pragma unroll
                for (int e = 0; e < 16; ++e) mine[(dt * 16 + e) * 64 + lane] = o[dt][e];
            if (half == 0) {
                mine[32 * D + ql] = m_i;
                mine[32 * D + 32 + ql] = l_tot;
            }
        }
        __syncthreads();
        if (share > 0) return;
#pragma unroll 1
        for (int other = 1; other < S; ++other) {
            const float* theirs = area + (size_t)((other - 1) * R + group_of_rows) * kWaveFloats;
            const float m_b = theirs[32 * D + ql], l_b = theirs[32 * D + 32 + ql];
            const float m = fmaxf(m_i, m_b);
            const float fa = m_i == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m_i - m);
            const float fb = m_b == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m_b - m);
            m_i = m;
            l_tot = l_tot * fa + l_b * fb;
#pragma unroll
            for (int dt = 0; dt < kDTiles; ++dt)
#pragma unroll
                for (int e = 0; e < 16; ++e) o[dt][e] = o[dt][e] * fa + theirs[(dt * 16 + e) * 64 + lane] * fb;
        }
    }
    if (my_row >= rows_left) return;

    // ---- rows out: lane has O[row][32 dt + 8 j + 4 half .. + 3] -------------------------------------------------------------
    const float inv = l_tot > 0.f ? 1.f / l_tot : l_tot == 0.f ? 0.f : l_tot;      // (NaN stays)
    const float lse = l_tot == 0.f ? -INFINITY : m_i + log2f(l_tot);
    if (at.part < 0) {
        const int64_t out_row = (int64_t)(s.start + token) * (p.batch.kv_heads * p.group) + q_head;
        if (p.lse && half == 0) p.lse[out_row] = lse;
        uint16_t* dst = static_cast<uint16_t*>(p.o) + out_row * D + 4 * half;
#pragma unroll
        for (int dt = 0; dt < kDTiles; ++dt)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const u32x2 w = {MM::pack_out(o[dt][4 * j] * inv, o[dt][4 * j + 1] * inv), MM::pack_out(o[dt][4 * j + 2] * inv, o[dt][4 * j + 3] * inv)};
                *reinterpret_cast<u32x2*>(dst + 32 * dt + 8 * j) = w;
            }
    } else if (at.part + at.run < p.parts) {
        const int64_t part_row = ((int64_t)(at.part + at.run) * p.batch.kv_heads + head) * p.tile_rows + my_row;
        if (half == 0) p.part_lse[part_row] = lse;
        float* dst = p.part_o + part_row * D + 4 * half;
#pragma unroll
        for (int dt = 0; dt < kDTiles; ++dt)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const f32x4 w = {o[dt][4 * j] * inv, o[dt][4 * j + 1] * inv, o[dt][4 * j + 2] * inv, o[dt][4 * j + 3] * inv};
                *reinterpret_cast<f32x4*>(dst + 32 * dt + 8 * j) = w;
            }
    }
}

// Joins the runs of a tile's keys, in an order that the run count alone decides: D / 4 lanes take a row and every SUBS-th run of
// it, four runs' loads in flight at a time; what they have is joined through LDS.  A workgroup takes ROWS rows at a time of a
// (tile whose keys are cut, K/V head).
template <bool BF16, int D, int ROWS>
__global__ __launch_bounds__(256) void paged_join_kernel(PagedAttnParams p) {
    constexpr int kLanes = D / 4, kSubs = 256 / kLanes / ROWS;
    __shared__ float shared_o[kSubs > 1 ? 256 : 1][5];
    __shared__ float shared_l[kSubs > 1 ? 256 : 1];
    const int tid = threadIdx.x, lane = tid & 63;
    const uint32_t item = blockIdx.x / (uint32_t)p.batch.kv_heads;
    const int head = (int)(blockIdx.x - item * (uint32_t)p.batch.kv_heads);
    Place at;
    if (!find_item<true>(p, item, lane, &at)) return;
    const int rows = min(at.s.fresh * p.group - (at.row_tile << p.row_shift), p.tile_rows);
    const int runs = max(min(at.runs, p.parts - at.part), 0);
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

// Rows of a workgroup's tile by the most rows a sequence can have: up to 32 rows the keys are all there is to read and its
// waves share them out; from 128 rows on every wave has rows of its own.
int rows_of_tile(int64_t most_rows) { return most_rows <= 32 ? 32 : most_rows <= 64 ? 64 : 128; }

struct Sizes {
    int tile_rows, shares;
    int64_t most_rows;          // of a sequence, as far as the host knows
    int64_t row_tiles;          // at most, over the batch
    int64_t items, parts;
    int run_units, least_tiles;
};
Sizes sizes_of(int32_t batch, int32_t tokens, int32_t max_q_len, int32_t heads, int32_t kv_heads) {
    Sizes z;
    const int group = heads / kv_heads;
    z.most_rows = (int64_t)(max_q_len > 0 && max_q_len < tokens ? max_q_len : tokens) * group;
    z.tile_rows = rows_of_tile(z.most_rows);
    z.row_tiles = ((int64_t)tokens * group + (int64_t)(batch < tokens ? batch : tokens) * (z.tile_rows - 1)) / z.tile_rows;
    z.shares = z.tile_rows == 32 ? kDecodeShares : z.tile_rows == 64 ? 2 : 1;
    z.run_units = z.tile_rows == 32 ? kDecodeUnits : z.tile_rows == 64 ? kMiddleUnits : kChunkUnits;
    z.least_tiles = z.tile_rows == 32 ? kDecodeLeast : kChunkLeast;
    // a run has at least cost / run_units tiles (rounded: 2^-20 more), and a tile of rows one run more than whole ones
    const int64_t runs = (z.run_units + z.run_units / 1024 + kv_heads) / kv_heads;
    z.items = z.row_tiles + runs;
    z.parts = 2 * runs;         // a cut tile of t key tiles has fewer than 2 t / longest runs
    return z;
}

template <bool BF16, int D, int R, int S, bool FP8, bool ONCE>
int launch_units_of(const PagedAttnParams& p, int64_t units, hipStream_t stream) {
    // bfloat16 weights as pairs where the matrix cores wait for keys anyway
    constexpr bool kSplit = R < 4 && (BF16 || FP8);
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

// (a sequence whose rows fit one tile has its keys read once)
template <bool BF16, int D, int R, int S, bool FP8> int launch_units(const PagedAttnParams& p, int64_t units, const Sizes& z, hipStream_t stream) {
    return z.most_rows <= z.tile_rows ? launch_units_of<BF16, D, R, S, FP8, true>(p, units, stream)
                                      : launch_units_of<BF16, D, R, S, FP8, false>(p, units, stream);
}

template <bool BF16, int D, int ROWS> int launch_join(const PagedAttnParams& p, const Sizes& z, hipStream_t stream) {
    const int64_t items = (z.run_units + z.run_units / 1024 + p.batch.kv_heads) / p.batch.kv_heads;      // more than there are cut tiles
    const int64_t rows = z.most_rows < z.tile_rows ? z.most_rows : z.tile_rows;
    const dim3 grid((unsigned)(items * p.batch.kv_heads), (unsigned)((rows + ROWS - 1) / ROWS));
    hipLaunchKernelGGL((paged_join_kernel<BF16, D, ROWS>), grid, dim3(256), 0, stream, p);
    FSTA_HIP_OK(hipGetLastError());
    return FSTA_OK;
}

template <bool BF16, int D, bool FP8> int launch_attention(const PagedAttnParams& p, const Sizes& z, hipStream_t stream) {
    const int64_t units = z.items * p.batch.kv_heads;
    int rc;
    if (z.tile_rows == 32) rc = launch_units<BF16, D, 1, kDecodeShares, FP8>(p, units, z, stream);
    else if (z.tile_rows == 64) rc = launch_units<BF16, D, 2, 2, FP8>(p, units, z, stream);
    else rc = launch_units<BF16, D, 4, 1, FP8>(p, units, z, stream);
    if (rc != FSTA_OK) return rc;
    // nothing is cut where no sequence can have more tiles than the shortest run has
    const int64_t most_tiles = (((int64_t)p.batch.width << p.batch.page_shift) + kTileN - 1) / kTileN;
    if (most_tiles <= z.least_tiles) return FSTA_OK;
    if (z.tile_rows == 32) return launch_join<BF16, D, 1>(p, z, stream);
    if (z.tile_rows == 64) return launch_join<BF16, D, 2>(p, z, stream);
    return launch_join<BF16, D, 8>(p, z, stream);
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
                                                       int32_t head_dim) {
    if (batch <= 0 || tokens <= 0 || kv_heads <= 0 || heads <= 0 || heads % kv_heads || head_dim <= 0) return 0;
    const Sizes z = sizes_of(batch, tokens, max_q_len, heads, kv_heads);
    return (size_t)z.parts * (size_t)kv_heads * (size_t)z.tile_rows * (size_t)(head_dim + 1) * sizeof(float);
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
    const Sizes z = sizes_of(batch, tokens, max_q_len, heads, kv_heads);
    const size_t need = fsta_paged_attention_workspace_bytes(batch, tokens, max_q_len, heads, kv_heads, head_dim);
    if (!workspace || workspace_bytes < need) return fail(FSTA_EINVAL, "%s: needs %zu bytes of workspace, got %zu", who, need, workspace_bytes);
    if (misaligned(workspace, 16)) return fail(FSTA_EINVAL, "%s: the workspace must be 16-byte aligned", who);
    while ((1 << p.batch.page_shift) < page_size) ++p.batch.page_shift;
    p.q = q; p.q_token_stride = q_token_stride; p.q_head_stride = q_head_stride;
    p.k = k_cache; p.v = v_cache; p.k_exponent = k_exponent; p.v_exponent = v_exponent;
    p.o = o; p.lse = lse;
    p.tree_bits = tree_bits; p.tree_words = mask == FSTA_PAGED_TREE ? tree_words : 0; p.mask = mask;
    p.group = heads / kv_heads; p.tile_rows = z.tile_rows; p.row_shift = z.tile_rows == 32 ? 5 : z.tile_rows == 64 ? 6 : 7; p.parts = (int32_t)z.parts; p.run_units = z.run_units; p.least_tiles = z.least_tiles;
    p.scale_log2e = sm_scale * kLog2e;
    p.part_o = static_cast<float*>(workspace);
    p.part_lse = p.part_o + (size_t)z.parts * kv_heads * z.tile_rows * head_dim;
    hipStream_t st = static_cast<hipStream_t>(stream);
    const bool fp8 = cache_dtype == FSTA_FP8;
    if (dtype == FSTA_BF16) {
        if (head_dim == 128) return fp8 ? launch_attention<true, 128, true>(p, z, st) : launch_attention<true, 128, false>(p, z, st);
        return fp8 ? launch_attention<true, 64, true>(p, z, st) : launch_attention<true, 64, false>(p, z, st);
    }
    if (head_dim == 128) return fp8 ? launch_attention<false, 128, true>(p, z, st) : launch_attention<false, 128, false>(p, z, st);
    return fp8 ? launch_attention<false, 64, true>(p, z, st) : launch_attention<false, 64, false>(p, z, st);
}
