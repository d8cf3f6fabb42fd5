// What the kernels of the attention over pages share: their arguments, and what a wave does with a tile of 32 keys.
#pragma once

#include "fsta_mfma_common.h"
#include "fsta_paged.h"

namespace fsta {
namespace paged {

using namespace mfma;

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
    float* part_o;                 // parts of rows whose keys several workgroups take: [part][rows][D] float32, normalised
    float* part_lse;               // [part][rows], base 2
    uint32_t* run_length;          // the cut's, behind the parts
    int32_t tree_words, mask, group, tile_rows, row_shift, parts;
    int32_t run_units[3], least_tiles;   // units that a launch may be cut into, the least tiles of a run
    float slots, unit_cost;              // workgroups that run at once; what a unit costs, in tiles
    float cut_cost, cut_unit_cost;       // .. the joining, and per unit
    float scale_log2e;
};

__device__ static const uint32_t kZeroRow[4] = {0u, 0u, 0u, 0u};

__device__ __forceinline__ uint32_t lane_of(uint32_t x, int lane) { return (uint32_t)__builtin_amdgcn_readlane((int)x, lane); }

// Number of keys that any row of a tile may see (its rows are tokens first .. last of the sequence's new ones)
__device__ __forceinline__ int keys_of_tile(const PagedAttnParams& p, const SeqLens& s, int row_tile) {
    if (p.mask != kCausal) return s.keys;
    const uint32_t last_row = (uint32_t)min((row_tile + 1) << p.row_shift, s.fresh * p.group) - 1u;
    return max(s.keys - s.fresh + (int)(last_row / (uint32_t)p.group) + 1, 0);
}

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


// 32 rows (token, query head) of a wave against tiles of 32 keys, all in registers:
//     S^T = K_tile . Q^T      O^T += V_tile^T . P^T        (32x32x16 matrix instructions)
// A lane holds 16 scores of row lane & 31: keys 8 (e / 4) + 4 (lane >> 5) + e % 4, which is also how the transposing reads hand
// it the values' rows, so that the weights go to the second product from the registers they are in.
// FP8: the cache is 8-bit.  DIRECT: so are the tiles, widened here.  SPLIT: weights go to the matrix cores as pairs of bfloat16, hi + lo.
template <bool BF16, int D, bool FP8, bool DIRECT, bool SPLIT> struct RowGroup {
    using MM = Mma<BF16>;
    using PV = Mma<BF16 || FP8>;              // weights times values: 8-bit values are exact in bfloat16 whatever their scale
    using Frag = typename MM::frag;
    using PFrag = typename PV::frag;
    static constexpr int kSteps = D / 16;     // matrix instructions of a tile's scores
    static constexpr int kDTiles = D / 32;    // 32-row tiles of O^T
    static constexpr float kTrustedSum = BF16 || FP8 ? 16777216.f : 32768.f;
    static constexpr uint32_t kVBytes = kTileN * D * (DIRECT ? 1 : 2);      // values behind keys
    static constexpr uint32_t kExps = 2 * kTileN * D;                       // 8-bit tiles: exponents of the keys, of the values
    // float16 holds bytes, but not every byte times its power of two: the keys' powers go to the scores
    static constexpr bool kScaleScores = FP8 && !BF16;

    int ql, half;
    uint32_t k_lane0, v_lane0;                // this lane's addresses in a tile
    Frag qf[kSteps];                          // B operand: Q[row][16 ks + 8 half .. + 7]
    float m_i, l_i;                           // running maximum (base 2), this lane's sum
    f32x16 o[kDTiles];                        // O[row][32 dt + 8 (e / 4) + 4 half + e % 4]

    __device__ __forceinline__ explicit RowGroup(int lane) : ql(lane & 31), half(lane >> 5) {
        if constexpr (DIRECT) {               // (the transposing read hands a lane 8 keys, four from either 8-key half)
            const int row = 4 * half + ((lane & 15) >> 1) + ((lane & 8) ? 4 : 0);
            k_lane0 = (uint32_t)(ql * D + k8_chunk<D>(ql, 0) * 16 + 8 * half);
            v_lane0 = (uint32_t)(row * D + v8_chunk<D>(row, (lane >> 4) & 1) * 16 + 8 * (lane & 1));
        } else {
            const int row = 4 * half + ((lane & 15) >> 2), col = 16 * ((lane >> 4) & 1) + 4 * (lane & 3);
            k_lane0 = (uint32_t)(ql * D + k_chunk<D>(ql, half) * 8) * 2;
            v_lane0 = (uint32_t)(row * D + v_chunk<D>(row, col >> 3) * 8 + (col & 7)) * 2;
        }
    }
    __device__ __forceinline__ void load_q(const uint16_t* row) {
#pragma unroll
        for (int ks = 0; ks < kSteps; ++ks) {
            const u32x4 raw = *reinterpret_cast<const u32x4*>(row + 16 * ks + 8 * half);
            qf[ks] = __builtin_bit_cast(Frag, raw);
        }
    }
    // The loads are waited for here: left to their first use inside the loop over the tiles, that wait would be one for every
    // transfer on its way, at every tile.
    __device__ __forceinline__ void await_q() {
#pragma unroll
        for (int ks = 0; ks < kSteps; ++ks) lds_tie(qf[ks]);
    }
    __device__ __forceinline__ void reset() {
        m_i = -INFINITY;
        l_i = 0.f;
#pragma unroll
        for (int dt = 0; dt < kDTiles; ++dt)
#pragma unroll
            for (int e = 0; e < 16; ++e) o[dt][e] = 0.f;
    }
    // Sign bits of the halves whose exponent is all ones (adding the exponent's lowest bit carries into the sign's place)
    __device__ __forceinline__ static uint32_t not_finite(PFrag a, PFrag b) {
        constexpr uint32_t kTop = BF16 || FP8 ? 0x7f807f80u : 0x7c007c00u, kLow = BF16 || FP8 ? 0x00800080u : 0x04000400u;
        const u32x4 x = __builtin_bit_cast(u32x4, a), y = __builtin_bit_cast(u32x4, b);
        uint32_t bits = 0u;
#pragma unroll
        for (int e = 0; e < 4; ++e) bits |= ((x[e] & kTop) + kLow) | ((y[e] & kTop) + kLow);
        return bits & 0x80008000u;
    }
    // The values' fragment with what is not finite replaced by 0
    __device__ __forceinline__ static PFrag only_finite(PFrag f) {
        constexpr uint32_t kTop = BF16 || FP8 ? 0x7f80u : 0x7c00u;
        u32x4 w = __builtin_bit_cast(u32x4, f);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            if ((w[e] & kTop) == kTop) w[e] &= 0xffff0000u;
            if ((w[e] & (kTop << 16)) == kTop << 16) w[e] &= 0xffffu;
        }
        return __builtin_bit_cast(PFrag, w);
    }
    // 1 where it is +inf (sign 0) / -inf (sign 1) or NaN, 0 elsewhere
    __device__ __forceinline__ static PFrag infinite(PFrag f, uint32_t sign) {
        constexpr uint32_t kTop = BF16 || FP8 ? 0x7f80u : 0x7c00u, kOne = BF16 || FP8 ? 0x3f80u : 0x3c00u;
        u32x4 w = __builtin_bit_cast(u32x4, f);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const uint32_t x = w[e] ^ (sign << 15 | sign << 31);
            const uint32_t lo = x & 0xffffu, hi = x >> 16;
            w[e] = ((lo & 0x7fffu) > kTop || lo == kTop ? kOne : 0u) | ((hi & 0x7fffu) > kTop || hi == kTop ? kOne << 16 : 0u);
        }
        return __builtin_bit_cast(PFrag, w);
    }

    // One tile at LDS address `at` (keys, values), 8-bit ones' exponents at `exps` (widened ones': the keys' powers of two).  masked
    // (uniform): word() is the row's bits of the keys it sees.
    template <typename Word> __device__ __forceinline__ void tile(uint32_t at, uint32_t exps, float sc, bool masked, Word word) {
        // S^T (K fragments: all requested, then used as they arrive; LDS reads come back in order)
        f32x16 sv;
#pragma unroll
        for (int e = 0; e < 16; ++e) sv[e] = 0.f;
        uint32_t v_exp[4], k_exp[4];
        u32x4 k_power[4];
        if constexpr (kScaleScores) {
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if constexpr (DIRECT) k_exp[j] = lds_read_b32(exps + 8 * j + 4 * half);
                else k_power[j] = lds_read_b128(exps + 4 * (8 * j + 4 * half));
        }
        if constexpr (DIRECT) {
            uint32_t E = 127u;
            if constexpr (!kScaleScores) asm volatile("ds_read_u8 %0, %1" : "=v"(E) : "v"(exps + ql) : "memory");
            u32x2 raw[kSteps];
#pragma unroll
            for (int ks = 0; ks < kSteps; ++ks) raw[ks] = lds_read_b64((at + k_lane0) ^ (uint32_t)(ks << 4));
            if constexpr (kScaleScores) wait_lds<kSteps>();                        // (the counter of LDS accesses goes up to 15)
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
            u32x4 raw[kSteps];
#pragma unroll
            for (int ks = 0; ks < kSteps; ++ks) raw[ks] = lds_read_b128((at + k_lane0) ^ (uint32_t)(ks << 5));
            static_for<kSteps>([&](auto ks) {
                constexpr int k = decltype(ks)::value;
                wait_lds<kSteps - 1 - k>();
                lds_tie(raw[k]);
                sv = MM::mfma(__builtin_bit_cast(Frag, raw[k]), qf[k], sv);
            });
        }
        if constexpr (kScaleScores) {         // (requested in front of the keys: they are here)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                if constexpr (DIRECT) lds_tie(k_exp[j]);
                else lds_tie(k_power[j]);
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    if constexpr (DIRECT) k_power[j][e] = min((k_exp[j] >> (8 * e)) & 255u, 254u) << 23;
                    sv[4 * j + e] *= __builtin_bit_cast(float, (uint32_t)k_power[j][e]);
                }
            }
        }
        uint32_t mine = ~0u;                  // bit 8 (e / 4) + e % 4: this lane's score e counts
        if (masked) {
            mine = word() >> (4 * half);
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
        if constexpr (DIRECT) {               // the values' powers of two go to the weights
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
                // A pair's high part is cut off, not rounded, and 2^-23 of the weight is added to the low one: it is greater than
                // zero where the weight is, and both parts' products with an infinity have the same sign.
                if (SPLIT) {
                    hi4[e] = __builtin_amdgcn_perm(__builtin_bit_cast(uint32_t, b), __builtin_bit_cast(uint32_t, a), 0x07060302u);
                    lo4[e] = PV::pack(__builtin_fmaf(a, 1.f + 0x1p-23f, -PV::low(hi4[e])), __builtin_fmaf(b, 1.f + 0x1p-23f, -PV::high(hi4[e])));
                } else {
                    hi4[e] = PV::pack(a, b);
                }
            }
            ph[k2] = __builtin_bit_cast(PFrag, hi4);
            if (SPLIT) pl[k2] = __builtin_bit_cast(PFrag, lo4);
        }
        // O^T (the fragments of the next 32 head dims are requested before the products of these)
        auto read_v = [&](int dt, VRaw<DIRECT>& f) {
            const uint32_t addr = (at + kVBytes + v_lane0) ^ (uint32_t)(dt << (DIRECT ? 5 : 6));
            if constexpr (DIRECT) {
                asm volatile("ds_read_b64_tr_b8 %0, %1" : "=v"(f.x[0]) : "v"(addr) : "memory");
                asm volatile("ds_read_b64_tr_b8 %0, %1 offset:%2" : "=v"(f.x[1]) : "v"(addr), "n"(16 * D) : "memory");
            } else {
                f.x[0].a = lds_read_tr16(addr);
                f.x[0].b = lds_read_tr16_at<8 * D * 2>(addr);
                f.x[1].a = lds_read_tr16_at<16 * D * 2>(addr);
                f.x[1].b = lds_read_tr16_at<24 * D * 2>(addr);
            }
        };
        VRaw<DIRECT> raw_v[kDTiles];
        read_v(0, raw_v[0]);
        static_for<kDTiles>([&](auto t) {
            constexpr int dt = decltype(t)::value;
            if constexpr (dt + 1 < kDTiles) {
                read_v(dt + 1, raw_v[dt + 1]);
                wait_lds<DIRECT ? 2 : 4>();
            } else {
                lds_wait();
            }
            PFrag f[2];
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                if constexpr (DIRECT) {
                    lds_tie(raw_v[dt].x[h]);
                    f[h] = __builtin_bit_cast(PFrag, widen8<true>(raw_v[dt].x[h][0], raw_v[dt].x[h][1], 1.f));
                } else {
                    lds_tie(raw_v[dt].x[h].a);
                    lds_tie(raw_v[dt].x[h].b);
                    f[h] = __builtin_bit_cast(PFrag, raw_v[dt].x[h]);
                }
            }
            // A value that is not finite must reach the rows that see its key and no other, although a weight of zero times it
            // is a NaN: where the tile is masked, such values are taken out and put back row by row, by their signs.
            if (masked && __ballot(not_finite(f[0], f[1]) != 0u) != 0ull) {
                constexpr uint32_t kOne = BF16 || FP8 ? 0x3f80u : 0x3c00u;
#pragma unroll 1
                for (uint32_t sign = 0; sign < 2; ++sign) {
                    f32x16 touched;
#pragma unroll
                    for (int e = 0; e < 16; ++e) touched[e] = 0.f;
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        u32x4 seen;
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            const int bit = 8 * (2 * h + e / 2) + 2 * (e % 2);
                            seen[e] = ((mine >> bit) & 1u ? kOne : 0u) | ((mine >> (bit + 1)) & 1u ? kOne << 16 : 0u);
                        }
                        touched = PV::mfma(infinite(f[h], sign), __builtin_bit_cast(PFrag, seen), touched);
                    }
#pragma unroll
                    for (int e = 0; e < 16; ++e)
                        if (touched[e] > 0.f) o[dt][e] += sign ? -INFINITY : INFINITY;
                }
                f[0] = only_finite(f[0]);
                f[1] = only_finite(f[1]);
            }
            o[dt] = PV::mfma(f[0], ph[0], o[dt]);
            o[dt] = PV::mfma(f[1], ph[1], o[dt]);
            if (SPLIT) {
                o[dt] = PV::mfma(f[0], pl[0], o[dt]);
                o[dt] = PV::mfma(f[1], pl[1], o[dt]);
            }
        });
    }

    // Weights 2 i and 2 i + 1 against the maximum -neg_m, packed; adds them to the sum
    __device__ __forceinline__ static uint32_t two_weights(const f32x16& sv, int i, float sc, float neg_m, float& sum) {
        const float a = __builtin_amdgcn_exp2f(__builtin_fmaf(sv[2 * i], sc, neg_m));
        const float b = __builtin_amdgcn_exp2f(__builtin_fmaf(sv[2 * i + 1], sc, neg_m));
        sum += a;
        sum += b;
        return PV::pack(a, b);
    }
    __device__ __forceinline__ bool doubtful(float sum) const { return __ballot(!(sum <= kTrustedSum) || m_i == -INFINITY) != 0ull; }
    // Where the maximum as it stands is not good enough (a first tile, a large sum): raises it and weighs again
    __device__ __forceinline__ void raise(const f32x16& sv, float sc, uint32_t (&w)[8], float& sum) {
        float mx = -INFINITY;
#pragma unroll
        for (int e = 0; e < 16; ++e) mx = fmaxf(mx, sv[e]);
        float a, b;
        swap_halves(mx, false, a, b);
        mx = fmaxf(a, b) * sc;
        const bool up = mx > m_i + kRescaleSlack || (m_i == -INFINITY && mx > -INFINITY);
        const float alpha = up ? __builtin_amdgcn_exp2f(m_i - mx) : 1.f;
        if (up) m_i = mx;
        l_i *= alpha;
#pragma unroll
        for (int dt = 0; dt < kDTiles; ++dt)
#pragma unroll
            for (int e = 0; e < 16; ++e) o[dt][e] *= alpha;
        const float neg_m = m_i == -INFINITY ? 0.f : -m_i;
        sum = 0.f;
#pragma unroll
        for (int i = 0; i < 8; ++i) w[i] = two_weights(sv, i, sc, neg_m, sum);
    }
    __device__ __forceinline__ static PFrag fragment(const uint32_t (&w)[8], int h) {
        const u32x4 x = {w[4 * h], w[4 * h + 1], w[4 * h + 2], w[4 * h + 3]};
        return __builtin_bit_cast(PFrag, x);
    }
    // Two 16-bit tiles that every row sees whole.  Instructions are issued in this order: the scores of both tiles take turns, so
    // that none waits for the one in front of it; the weights of the second tile are worked out between the products of the first
    // tile's values.
    __device__ __forceinline__ void two_tiles(uint32_t at_a, uint32_t at_b, float sc) {
        static_assert(!DIRECT && !SPLIT, "16-bit tiles, weights rounded once");
        constexpr int kFirst = 3;                 // fragments of either tile that are requested ahead
        u32x4 ka[kSteps], kb[kSteps];
        auto read_k = [&](int ks) {
            ka[ks] = lds_read_b128((at_a + k_lane0) ^ (uint32_t)(ks << 5));
            kb[ks] = lds_read_b128((at_b + k_lane0) ^ (uint32_t)(ks << 5));
        };
        VPair va[kDTiles][2], vb[kDTiles][2];
        auto read_v = [&](uint32_t at, int dt, VPair (&v)[2]) {
            const uint32_t addr = (at + kVBytes + v_lane0) ^ (uint32_t)(dt << 6);
            v[0].a = lds_read_tr16(addr);
            v[0].b = lds_read_tr16_at<8 * D * 2>(addr);
            v[1].a = lds_read_tr16_at<16 * D * 2>(addr);
            v[1].b = lds_read_tr16_at<24 * D * 2>(addr);
        };
        auto tie_v = [&](VPair (&v)[2]) {
            lds_tie(v[0].a); lds_tie(v[0].b); lds_tie(v[1].a); lds_tie(v[1].b);
        };
        f32x16 sa, sb;
#pragma unroll
        for (int e = 0; e < 16; ++e) sa[e] = sb[e] = 0.f;
#pragma unroll
        for (int ks = 0; ks < kFirst; ++ks) read_k(ks);
        static_for<kSteps>([&](auto step) {
            constexpr int ks = decltype(step)::value;
            if constexpr (ks + kFirst < kSteps) read_k(ks + kFirst);
            wait_lds<2 * (kSteps - 1 - ks < kFirst ? kSteps - 1 - ks : kFirst)>();
            lds_tie(ka[ks]);
            lds_tie(kb[ks]);
            sa = MM::mfma(__builtin_bit_cast(Frag, ka[ks]), qf[ks], sa);
            sb = MM::mfma(__builtin_bit_cast(Frag, kb[ks]), qf[ks], sb);
            asm volatile("" : "+v"(sa), "+v"(sb));     // (products in this place: left alone, the compiler puts them behind all reads)
        });
        // values: half of the head dims requested ahead of the weights, the others behind them
        constexpr int kHalf = kDTiles / 2;
#pragma unroll
        for (int dt = 0; dt < kHalf; ++dt) read_v(at_a, dt, va[dt]);
        uint32_t wa[8], wb[8];
        float sum_a = 0.f, sum_b = 0.f, neg_m = m_i == -INFINITY ? 0.f : -m_i;
#pragma unroll
        for (int i = 0; i < 8; ++i) wa[i] = two_weights(sa, i, sc, neg_m, sum_a);
        if (doubtful(sum_a)) raise(sa, sc, wa, sum_a);
        l_i += sum_a;
#pragma unroll
        for (int dt = kHalf; dt < kDTiles; ++dt) read_v(at_a, dt, va[dt]);
        wait_lds<4 * (kDTiles - kHalf)>();
#pragma unroll
        for (int dt = 0; dt < kHalf; ++dt) tie_v(va[dt]);
        neg_m = m_i == -INFINITY ? 0.f : -m_i;
        constexpr int kPer = 8 / (2 * kDTiles);        // pairs of weights between two products
        auto product = [&](auto step) {
            constexpr int i = decltype(step)::value, dt = (i / (2 * kHalf)) * kHalf + i % kHalf, h = (i / kHalf) % 2;
            o[dt] = PV::mfma(__builtin_bit_cast(PFrag, va[dt][h]), fragment(wa, h), o[dt]);
#pragma unroll
            for (int k = i * kPer; k < (i + 1) * kPer; ++k) {
                wb[k] = two_weights(sb, k, sc, neg_m, sum_b);
                asm volatile("" : "+v"(wb[k]), "+v"(o[dt]));
            }
        };
        static_for<kDTiles>(product);
        lds_wait();
#pragma unroll
        for (int dt = kHalf; dt < kDTiles; ++dt) tie_v(va[dt]);
        static_for<kDTiles>([&](auto step) { product(std::integral_constant<int, kDTiles + decltype(step)::value>{}); });
#pragma unroll
        for (int dt = 0; dt < kHalf; ++dt) read_v(at_b, dt, vb[dt]);
        if (doubtful(sum_b)) raise(sb, sc, wb, sum_b);
        l_i += sum_b;
#pragma unroll
        for (int dt = kHalf; dt < kDTiles; ++dt) read_v(at_b, dt, vb[dt]);
        wait_lds<4 * (kDTiles - kHalf)>();
#pragma unroll
        for (int dt = 0; dt < kHalf; ++dt) tie_v(vb[dt]);
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int dt = 0; dt < kHalf; ++dt) o[dt] = PV::mfma(__builtin_bit_cast(PFrag, vb[dt][h]), fragment(wb, h), o[dt]);
        lds_wait();
#pragma unroll
        for (int dt = kHalf; dt < kDTiles; ++dt) tie_v(vb[dt]);
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int dt = kHalf; dt < kDTiles; ++dt) o[dt] = PV::mfma(__builtin_bit_cast(PFrag, vb[dt][h]), fragment(wb, h), o[dt]);
    }

    // Sum over both halves of the lanes that share a row
    __device__ __forceinline__ float row_sum() const {
        float a, b;
        swap_halves(l_i, false, a, b);
        return a + b;
    }
};

// What a wave's rows see of the keys, besides what the tiles themselves say
struct Sight {
    int limit, low_limit, high_limit;         // last key of this lane's row; the least and greatest of the wave's rows
    int old;                                  // keys in front of the new tokens (negative: the first new ones have no place)
    const uint32_t* bits;                     // this row's mask (trees)
    // .. and its first words: a load in front of a tile's weights would wait for every transfer on its way
    static constexpr int kKept = 8;
    uint32_t kept[kKept];

    __device__ __forceinline__ void keep(const PagedAttnParams& p) {
#pragma unroll
        for (int i = 0; i < kKept; ++i) kept[i] = 0u;
        if (p.mask == kTree) {
#pragma unroll
            for (int i = 0; i < kKept; ++i)
                if (i < p.tree_words) kept[i] = bits[i];
        }
    }
    __device__ __forceinline__ void await_kept() {
#pragma unroll
        for (int i = 0; i < kKept; ++i) lds_tie(kept[i]);
    }
    // Word i (uniform); all ones in front of the first: keys in front of the new tokens are seen by all
    __device__ __forceinline__ uint32_t word_of(const PagedAttnParams& p, int i) const {
        if (i < 0) return ~0u;
        if (i >= p.tree_words) return 0u;
        if (i >= kKept) return bits[i];       // (2 trees on 2000 keys, 32 heads of 128: 512 nodes 72 us, unmasked 58; 256 nodes on 1500 keys 42 and 35)
        uint32_t w = 0u;                      // (by masks: a choice among them would put them into memory)
#pragma unroll
        for (int k = 0; k < kKept; ++k) w |= kept[k] & (0u - (uint32_t)(i == k));
        return w;
    }

    __device__ __forceinline__ bool whole(const PagedAttnParams& p, int first) const {      // every row sees every key of the tile
        return first + kTileN - 1 <= low_limit && !(p.mask == kTree && first + kTileN > old);
    }
    // bits of the tile's keys; bad: halves of it on pages outside the cache
    __device__ __forceinline__ uint32_t word(const PagedAttnParams& p, int first, uint32_t bad) const {
        const int rel = limit - first;
        uint32_t w = rel >= 31 ? ~0u : rel < 0 ? 0u : (2u << rel) - 1u;
        if (bad & 1u) w &= 0xffff0000u;
        if (bad & 2u) w &= 0x0000ffffu;
        if (p.mask == kTree && first + kTileN > old) {
            const int number = first - old, wi = number >> 5, sh = number & 31;
            const uint32_t lo = word_of(p, wi);
            w &= sh ? (lo >> sh) | (word_of(p, wi + 1) << (32 - sh)) : lo;
        }
        return w;
    }
};
// Rows first_row .. first_row + 31 of a tile (rows_left of them exist), this lane's `my_row`
struct Rows { int token, q_head; Sight sight; };
__device__ __forceinline__ Rows rows_of(const PagedAttnParams& p, const SeqLens& s, int head, int row0, int rows_left, int first_row, int ql) {
    Rows r;
    const uint32_t group = (uint32_t)p.group;
    const int mine = row0 + min(first_row + ql, rows_left - 1);
    r.token = (int)((uint32_t)mine / group);
    r.q_head = head * p.group + mine - r.token * p.group;
    r.sight.old = s.keys - s.fresh;
    const bool causal = p.mask == kCausal;
    r.sight.limit = causal ? r.sight.old + r.token : s.keys - 1;
    r.sight.low_limit = causal ? r.sight.old + (int)((uint32_t)(row0 + first_row) / group) : s.keys - 1;
    r.sight.high_limit = causal ? r.sight.old + (int)((uint32_t)(row0 + min(first_row + 31, rows_left - 1)) / group) : s.keys - 1;
    r.sight.bits = p.tree_bits + (int64_t)(s.start + r.token) * p.tree_words;
    return r;
}

// Pages by scalar loads, through the constant address space (a load the compiler takes for a vector one it waits for with
// vmcnt(0), i.e. for the whole ring)
typedef const int32_t __attribute__((address_space(4))) * const_i32;
__device__ __forceinline__ const_i32 table_of(const PagedAttnParams& p, int seq) {
    return (const_i32)(uintptr_t)(p.batch.page_table + (size_t)seq * p.batch.width);
}
__device__ __forceinline__ int page_at(const PagedAttnParams& p, const_i32 table, int keys, int pos) {
    return table[__builtin_amdgcn_readfirstlane(min(pos, keys - 1) >> p.batch.page_shift)];
}

// Transfers of a tile's keys and values (and exponents) from its pages to a ring slot, as wave `part` of PARTS.
// WIDENED: an 8-bit tile that is copied into the 16-bit layout afterwards lies in LDS as it does in memory.
constexpr int kRawBuffer = 0x00020000;        // buffer resource, word 3: raw 32-bit data

template <int D, int PARTS, bool FP8, bool WIDENED> struct Fetch {
    static constexpr int kRowBytes = FP8 ? D : 2 * D;             // a key's or a value's row in the cache
    static constexpr int kDma = 2 * kTileN * kRowBytes / 1024;    // transfers of 1 KiB
    static constexpr int kPer = kDma / PARTS;                     // of them this wave's
    static constexpr int kPerTile = kPer + (FP8 ? 1 : 0);         // (and one of the exponents)
    static constexpr int kBytes = kDma * 1024 + (FP8 ? 256 : 0);
    static_assert(kDma % PARTS == 0, "a wave has whole transfers");
    static constexpr int kLanesPerRow = kRowBytes / 16, kRowsPerDma = 64 / kLanesPerRow;

    static constexpr int kPerHalf = 16 / kRowsPerDma;             // transfers of 16 rows
    static constexpr int kRun = kPer < kPerHalf ? kPer : kPerHalf;   // of them this wave's, one behind the other
    static_assert(kPer % kRun == 0 && kPerHalf % kRun == 0, "a wave has whole halves, or a part of one");

    int first_unit;
    // This lane's piece of the wave's first transfer of a half.  The next ones lie 1 KiB further each, in memory and in LDS; the keys' swizzle
    // changes by a constant from one to the next, the values' not at all.
    uint32_t k_off, v_off;
    // A wave whose transfers are all keys' or all values', of one 16-key half, has one address a tile.
    static constexpr bool kOneSide = PARTS >= 2, kOneHalf = PARTS >= 4;
    const unsigned char* side;                // the head's rows of page 0 in the tensor that it fetches from
    const unsigned char* v_side;              // .. and in v, where it fetches both
    uint64_t page_bytes;
    uint32_t turn;                            // what the keys' swizzle changes by
    __device__ __forceinline__ Fetch(const PagedAttnParams& p, int head, int part, int lane) : first_unit(part * kPer) {
        const int64_t at = ((int64_t)head << p.batch.page_shift) * kRowBytes;
        const unsigned char* k = static_cast<const unsigned char*>(p.k) + at;
        v_side = static_cast<const unsigned char*>(p.v) + at;
        side = kOneSide && part >= PARTS / 2 ? v_side : k;
        page_bytes = ((uint64_t)p.batch.kv_heads << p.batch.page_shift) * kRowBytes;
        const int r = lane / kLanesPerRow, slot = lane % kLanesPerRow;
        k_off = (uint32_t)(r * kRowBytes + (WIDENED ? slot : FP8 ? k8_chunk<D>(r, slot) : k_chunk<D>(r, slot)) * 16);
        v_off = (uint32_t)(r * kRowBytes + (WIDENED ? slot : FP8 ? v8_chunk<D>(r, slot) : v_chunk<D>(r, slot)) * 16);
        if (kOneSide && part >= PARTS / 2) k_off = v_off;
        turn = WIDENED || (kOneSide && part >= PARTS / 2) ? 0u : 64u;
        const uint32_t skip = (uint32_t)(first_unit % kPerHalf);
        k_off = (k_off ^ (skip * turn)) + skip * 1024u;
    }
    __device__ __forceinline__ bool is_v(int j) const { return first_unit + j >= kDma / 2; }
    __device__ __forceinline__ int half_of(int j) const { return ((first_unit + j) % (kDma / 2)) / kPerHalf; }

    // p0, p1: pages of the tile's 16-key halves; returns the halves that are on none.  A half's rows are a buffer of as many bytes
    // as there are rows: what a lane asks for behind its end the hardware answers with zeros, and no lane needs an address.
    // once (a bool, or one known to the compiler): nobody else reads these keys, past the caches.
    template <typename Once>
    __device__ __forceinline__ uint32_t tile(const PagedAttnParams& p, int keys, int head, int first, int p0, int p1, unsigned char* dst, int lane, Once once) const {
        typedef const void __attribute__((address_space(1))) * global_ptr;
        typedef void __attribute__((address_space(3))) * lds_ptr;
        const uint32_t page_mask = (1u << p.batch.page_shift) - 1u;
        const bool ok0 = (unsigned)p0 < (unsigned)p.batch.num_pages, ok1 = (unsigned)p1 < (unsigned)p.batch.num_pages;
#if defined(__HIP_DEVICE_COMPILE__)           // (the host pass knows no buffer resources)
        auto rows_at = [&](const unsigned char* tensor, int half) {
            const bool ok = half ? ok1 : ok0;
            const uint32_t page = (uint32_t)(ok ? (half ? p1 : p0) : 0), in_page = ((uint32_t)first + 16u * half) & page_mask;
            // (said to be uniform: a resource in vector registers is tried lane by lane)
            const int rows = __builtin_amdgcn_readfirstlane(ok ? max(min(keys - first - 16 * half, 16), 0) : 0);
            const uint64_t from = (uint64_t)tensor + page * page_bytes + in_page * (uint32_t)kRowBytes;
            const uint64_t base = (uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)from) |
                                  ((uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)(from >> 32)) << 32);
            return __builtin_amdgcn_make_buffer_rsrc((void*)base, 0, rows * kRowBytes, kRawBuffer);
        };
        const unsigned char* v_from = kOneSide ? side : v_side;
        const auto k0 = rows_at(side, kOneHalf ? half_of(0) : 0), k1 = kOneHalf ? k0 : rows_at(side, 1);
        const auto v0 = kOneSide ? k0 : rows_at(v_from, 0), v1 = kOneSide ? k1 : rows_at(v_from, 1);
        auto transfers = [&](auto policy) {
            constexpr int kPolicy = decltype(policy)::value;
            static_for<kPer>([&](auto index) {
                constexpr int j = decltype(index)::value, in_half = j % kRun;
                constexpr bool v = !kOneSide && j >= kDma / 2;
                constexpr int half = kOneHalf ? 0 : j % (kDma / 2) / kPerHalf;
                const uint32_t off = v ? v_off : k_off ^ (in_half * turn);
                lds_ptr to = (lds_ptr)(dst + (first_unit + j - in_half) * 1024);
                if constexpr (v && half) __builtin_amdgcn_raw_ptr_buffer_load_lds(v1, to, 16, off, 0, in_half * 1024, kPolicy);
                else if constexpr (v) __builtin_amdgcn_raw_ptr_buffer_load_lds(v0, to, 16, off, 0, in_half * 1024, kPolicy);
                else if constexpr (half) __builtin_amdgcn_raw_ptr_buffer_load_lds(k1, to, 16, off, 0, in_half * 1024, kPolicy);
                else __builtin_amdgcn_raw_ptr_buffer_load_lds(k0, to, 16, off, 0, in_half * 1024, kPolicy);
            });
        };
        if constexpr (!std::is_same_v<Once, bool>) transfers(std::integral_constant<int, Once::value ? 2 : 0>{});
        else if (once) transfers(std::integral_constant<int, 2>{});
        else transfers(std::integral_constant<int, 0>{});
#endif
        if constexpr (FP8) {                  // exponents of the 32 keys, then of the 32 values, four to a lane
            const int l = lane & 15, g = (l >> 2) & 1;
            const int64_t row = ((((int64_t)(g ? (ok1 ? p1 : 0) : (ok0 ? p0 : 0)) * p.batch.kv_heads + head) << p.batch.page_shift)) +
                                (int64_t)(((uint32_t)first + 16u * g) & page_mask);
            const uint8_t* src = ((l & 8) ? p.v_exponent : p.k_exponent) + row + 4 * (l & 3);
            const bool here = first + 16 * g < keys && (g ? ok1 : ok0);
            src = here ? src : reinterpret_cast<const uint8_t*>(kZeroRow);
            __builtin_amdgcn_global_load_lds((global_ptr)src, (lds_ptr)(dst + kDma * 1024), 4, 0, 0);
        }
        return (ok0 ? 0u : 1u) | (ok1 ? 0u : 2u);
    }
};

// At most `tiles` (0 .. MOST) tiles' worth of this wave's transfers outstanding, PER instructions each
template <int PER, int MOST> __device__ __forceinline__ void wait_tiles(int tiles) {
    static_assert(MOST * PER < 64, "vmcnt has 6 bits");
    if (tiles >= MOST) {
        wait_vmcnt<MOST * PER>();
    } else {
        if constexpr (MOST > 0) wait_tiles<PER, MOST - 1>(tiles);
    }
}

// A row's 4 consecutive values to the output
template <bool BF16> __device__ __forceinline__ void store_row(uint16_t* dst, float a, float b, float c, float d) {
    const u32x2 w = {Mma<BF16>::pack_out(a, b), Mma<BF16>::pack_out(c, d)};
    *reinterpret_cast<u32x2*>(dst) = w;
}

}  // namespace paged
}  // namespace fsta
