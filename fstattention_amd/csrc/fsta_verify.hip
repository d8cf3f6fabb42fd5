// Which tokens of a batch of draft trees stand against the model's logits, and the token behind each accepted path.
//
// At an accepted node the children are asked one after the other; what the model has left after each that fell is
//   W = max(P - s q, 0) over the tokens not asked yet:
// speculative sampling replaces p by norm max(p - q', 0) each time, with q' = q / r the draft's probabilities over the tokens not
// drawn before; with p = W / Z that is max(W / Z - q / r, 0) = max(P - (s + Z / r) q, 0) / Z, so s grows by Z / r and nothing else has to be
// kept per token.  Without the draft's probabilities a child is its own proposal: W loses the token, nothing else.
//
// Decisions compare sums over the vocabulary with a random number, and the next token is the place where a running sum passes
// one: in 32 bits a sum of 10^5 terms is off by more than many of them are large, so weights and sums are of 64 bits.  Only a first
// sum (of P) without draft probabilities may be one of 32 bits with a bound of its error (kDoubt): a decision inside the bound is taken once more
// by 64, and the token is always picked by 64.
//
// A row is summed in parts of 2048 tokens, a wave each.  What depends on a sum comes in a later launch.  Where the rows of all nodes
// are few enough (chains(), kAllGiven):
//   stats_kernel   the parts of the rows of all nodes with children;
//   stands_kernel  which child stands at each node by these sums: walks only follow;
//   step_kernel    with draft probabilities: sums of W where a child fell, one of every sequence's a launch;
//   last_kernel    without: the row at each walk's end in 64 bits;
// and where they are not
//   step_kernel    one step of all sequences: each workgroup takes the decisions that the sums so far allow (all workgroups of a
//                  sequence the same ones), and its parts of the sum that is wanted next.  Only the rows on accepted paths are read;
//   last_kernel    as above.  In both cases then
//   walk_kernel    a workgroup per sequence goes on alone from wherever a sequence is to its end, and picks its next token.
// What bounds it: few rows, the chain of launches and of loads that need each other (8 to 20 us before the first sum and behind the last);
// many, the exponentials: 95 cycles of a SIMD for 64 of 64 bits, some 35 for 64 of 32.
#include "fsta_common.h"

namespace fsta {
namespace {

typedef unsigned int u32x2 __attribute__((ext_vector_type(2)));
typedef unsigned int u32x4 __attribute__((ext_vector_type(4)));

constexpr int kChildren = FSTA_VERIFY_MAX_CHILDREN;
constexpr int kRun = 512;                 // tokens that a wave looks at at once, eight a lane
constexpr int kPart = 4 * kRun;
constexpr int kMaxParts = 256;            // of a row: longer rows have longer parts
constexpr int kTree = 512;                // nodes of a tree that are kept in LDS
constexpr int kStepThreads = 256, kWalkThreads = 256;

// Of a part of a row: its largest logit (and, where the temperature is 0, the first place that has it), and the sum of the weights,
// against that logit, or in a sum of W against the row's
struct Part {
    double sum;
    float top;
    int32_t best;
};

// Where a sequence is, between launches
struct State {
    int32_t node, count;                  // the accepted node in question, how many before and with it
    int32_t child, asked, summed;         // as in Walk
    int32_t phase;                        // kFirst, kAgain: what the parts of this step are; kDone: no child stands
    int32_t held, where;                  // kDone: what the last parts were, and whose: of the steps' buffers 0 and 1, or kOfNode
    int32_t ready, exact;                 // whether the parts are there; whether they have to be 64 bits
    double shift, left;                   // s, r
    float top;                            // of the node's row, in kAgain
    int32_t pad;
};
enum { kFirst = 0, kAgain = 1, kDone = 2, kQuick = 3 };
enum { kOfNode = 2 };

struct VerifyArgs {
    const void *logits, *draft;
    int64_t logits_stride, draft_stride;
    const int64_t *tokens, *parent;
    const int32_t* q_starts;
    const float *u_accept, *u_next, *temperatures;
    float temperature;
    int32_t *path, *counts;
    int64_t* next;
    int32_t batch, nodes, vocabulary, max_path;
    int32_t parts_per_row, part_length;
    const Part* all_parts;                // of every node with children, or null ..
    int32_t* stands;                      // .. and the child that stands there, -1: none, or sums of W have to be asked
    Part *parts_out;                      // stats_kernel
    Part* parts[2];                       // of every sequence, by steps in turn
    State* states[2];
    int32_t turn, fresh;                  // which of them a step writes (walk_kernel: the last one wrote); fresh: no step was before
};

struct Half { unsigned short bits; };
struct Brain { unsigned short bits; };
__device__ __forceinline__ float value(float x) { return x; }
__device__ __forceinline__ float value(Half x) { return (float)__builtin_bit_cast(_Float16, x.bits); }
__device__ __forceinline__ float value(Brain x) { return __builtin_bit_cast(float, (uint32_t)x.bits << 16); }

// Eight values of a row at any address that the type allows (a row of odd length starts anywhere), as they come: taking them apart
// is what waits for them
template <typename T> struct Eight {
    u32x4 w[sizeof(T) / 2];
};
__device__ __forceinline__ float value(const Eight<float>& x, int e) {
    const uint32_t word = x.w[e / 4][e % 4];
    return __builtin_bit_cast(float, word);
}
__device__ __forceinline__ float value(const Eight<Half>& x, int e) { return value(Half{(unsigned short)(x.w[0][e / 2] >> (e & 1) * 16)}); }
__device__ __forceinline__ float value(const Eight<Brain>& x, int e) {
    return __builtin_bit_cast(float, e & 1 ? x.w[0][e / 2] & 0xffff0000u : x.w[0][e / 2] << 16);
}

// 2^d for -1000 <= d <= 0, exactly 1 for 0.  2^f = 1 + f g(f) over |f| <= 1/2, g the polynomial of degree 9 that meets (2^f - 1) / f at
// the Chebyshev points: off by 6e-16 at most.  Rounding to a whole number and scaling by its power of two go through the bits of the
// sum with 1.5 2^52: sums, products and their fusions run at full rate in 64 bits, conversions and ldexp do not.  A wave takes 90 to 100
// cycles for its 64, alone on its SIMD or not.
template <int N> __device__ __forceinline__ void powers(double (&d)[N]) {
    constexpr double kRound = 6755399441055744.0;
    constexpr double kG[10] = {7.070977866508138e-09, 1.0205905413765595e-07, 1.3215451633221434e-06, 1.5252672924850737e-05, 0.00015403530424776529,
                               0.0013333558200794592, 0.009618129107618665, 0.05550410866465167, 0.24022650695910075, 0.6931471805599462};
    double k[N], f[N], p[N];
#pragma unroll
    for (int i = 0; i < N; ++i) k[i] = d[i] + kRound;
#pragma unroll
    for (int i = 0; i < N; ++i) f[i] = d[i] - (k[i] - kRound);
#pragma unroll
    for (int i = 0; i < N; ++i) p[i] = kG[0];
#pragma unroll
    for (int c = 1; c < 10; ++c) {
#pragma unroll
        for (int i = 0; i < N; ++i) p[i] = fma(p[i], f[i], kG[c]);
    }
#pragma unroll
    for (int i = 0; i < N; ++i) {
        u32x2 bits = __builtin_bit_cast(u32x2, fma(p[i], f[i], 1.0));
        bits[1] += __builtin_bit_cast(u32x2, k[i])[0] << 20;
        d[i] = __builtin_bit_cast(double, bits);
    }
}
// exp((l - against) / T), the logit `against` being the largest: any l (NaN: as -inf); infinite ones share all weight
__device__ __forceinline__ double weight_of(float l, float against, double rate) {
    if (against == INFINITY) return l == INFINITY ? 1.0 : 0.0;
    const double d = ((double)l - (double)against) * rate;
    const bool far = d < -1000.0;         // (scaled in two steps: the result may have fewer bits)
    double p[1] = {far ? fmax(d, -1200.0) + 200.0 : d};
    powers(p);
    return d > -1200.0 ? (far ? p[0] * 0x1p-200 : p[0]) : 0.0;
}
// .. of eight logits
__device__ __forceinline__ void weights_of(const float (&l)[8], float against, double rate, double (&w)[8]) {
    const bool infinite = against == INFINITY;
    const double top = infinite ? 0.0 : (double)against;
    float least = INFINITY;
#pragma unroll
    for (int e = 0; e < 8; ++e) least = fminf(least, fmaxf(l[e], -INFINITY));       // (fmaxf takes the number of the two)
    const bool far = infinite || !(((double)least - top) * rate >= -1000.0);
#pragma unroll
    for (int h = 0; h < 8; h += 4) {
        double d[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) d[e] = ((double)l[h + e] - top) * rate;
        powers(d);
#pragma unroll
        for (int e = 0; e < 4; ++e) w[h + e] = d[e];
        __builtin_amdgcn_sched_barrier(0);
    }
    if (!far) return;
#pragma unroll
    for (int h = 0; h < 8; h += 2) {
        double d[2];
#pragma unroll
        for (int e = 0; e < 2; ++e) d[e] = fmax(fmin(((double)l[h + e] - top) * rate, 0.0), -1200.0) + 200.0;
        powers(d);
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            const float x = l[h + e];
            w[h + e] = infinite ? (x == INFINITY ? 1.0 : 0.0) : ((double)x - top) * rate > -1200.0 ? d[e] * 0x1p-200 : 0.0;
        }
        __builtin_amdgcn_sched_barrier(0);
    }
}

// log2(e) / T of a sequence; 0: greedy
__device__ __forceinline__ double rate_of(const VerifyArgs& a, int b) {
    const float tau = a.temperatures ? a.temperatures[b] : a.temperature;
    return tau > 0.f ? fmax(1.4426950408889634074 / (double)tau, 1e-300) : 0.0;
}

// The weights of one row: P against its largest logit, W with the draft's row
template <typename L, typename Q> struct Row {
    const L* logits;
    const Q* draft;                       // or null
    double rate;                          // log2(e) / T; 0: the largest logit's first place has all mass
    float top;
    int best;
    double shift;                         // s
    int n;                                // the vocabulary
    // of eight tokens as they were loaded
    __device__ __forceinline__ void eight(const Eight<L>& l, const Eight<Q>& q, double (&w)[8]) const {
        float x[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = value(l, e);
        weights_of(x, top, rate, w);
        if (!draft || !(shift > 0.0)) return;
#pragma unroll
        for (int e = 0; e < 8; ++e) w[e] = fmax(w[e] - shift * fmax((double)value(q, e), 0.0), 0.0);
    }
    __device__ __forceinline__ double weight(float l, double q) const {
        const double p = weight_of(l, top, rate);
        return shift > 0.0 ? fmax(p - shift * q, 0.0) : p;
    }
    __device__ __forceinline__ double proposed(int x) const { return draft ? fmax((double)value(draft[x]), 0.0) : 0.0; }
};

struct Shared {
    double sum[kMaxParts];                // parts' sums against the row's largest logit
    Part part[kMaxParts];                 // walk_kernel's own
    int32_t parent[kTree], token[kTree];  // -1: none
    int32_t stands[kTree];
    uint32_t fell[kWalkThreads / 64][kPart / 32];     // a wave's part: which tokens fell
    int32_t fallen[kChildren];            // tokens that left P at this node
    double lost[kChildren];               // .. and their weights
    double wave_sum[kWalkThreads / 64];
    int32_t best[kWalkThreads / 64], last[kWalkThreads / 64];
};

// Steps of a sum (or least, or largest) over the lanes up to each: from 1, 2, 4 and 8 lanes below within rows of 16, then the rows'
// last lanes to the rows behind them.  Register moves: a shuffle through LDS takes ten times as long, and decisions wait for these.
template <int STEP> __device__ __forceinline__ uint32_t from_below(uint32_t none, uint32_t x) {
    constexpr int kControl[6] = {0x111, 0x112, 0x114, 0x118, 0x142, 0x143}, kRows[6] = {0xf, 0xf, 0xf, 0xf, 0xa, 0xc};
    return (uint32_t)__builtin_amdgcn_update_dpp((int)none, (int)x, kControl[STEP], kRows[STEP], 0xf, false);
}
template <int STEP> __device__ __forceinline__ double from_below(double x) {
    const uint64_t bits = __builtin_bit_cast(uint64_t, x);
    return __builtin_bit_cast(double, (uint64_t)from_below<STEP>(0u, (uint32_t)(bits >> 32)) << 32 | from_below<STEP>(0u, (uint32_t)bits));
}
template <typename F> __device__ __forceinline__ void six_steps(F f) {
    f(std::integral_constant<int, 0>{});
    f(std::integral_constant<int, 1>{});
    f(std::integral_constant<int, 2>{});
    f(std::integral_constant<int, 3>{});
    f(std::integral_constant<int, 4>{});
    f(std::integral_constant<int, 5>{});
}
// The value of lane l, the same l in all lanes
__device__ __forceinline__ int of_lane(int x, int l) { return __builtin_amdgcn_readlane(x, l); }
__device__ __forceinline__ double of_lane(double x, int l) {
    const uint64_t bits = __builtin_bit_cast(uint64_t, x);
    return __builtin_bit_cast(double, (uint64_t)(uint32_t)of_lane((int)(bits >> 32), l) << 32 | (uint32_t)of_lane((int)bits, l));
}
__device__ __forceinline__ double sum_up_to(double x) {
    six_steps([&](auto step) { x += from_below<decltype(step)::value>(x); });
    return x;
}
__device__ __forceinline__ double sum_of(double x) { return of_lane(sum_up_to(x), 63); }
__device__ __forceinline__ float max_of(float x) {
    six_steps([&](auto step) {
        x = fmaxf(x, __builtin_bit_cast(float, from_below<decltype(step)::value>(0xff800000u, __builtin_bit_cast(uint32_t, x))));
    });
    return __builtin_bit_cast(float, of_lane(__builtin_bit_cast(int, x), 63));
}
__device__ __forceinline__ int min_of(int x) {
    six_steps([&](auto step) { x = min(x, (int)from_below<decltype(step)::value>((uint32_t)INT32_MAX, (uint32_t)x)); });
    return of_lane(x, 63);
}
__device__ __forceinline__ int max_of(int x) {
    six_steps([&](auto step) { x = max(x, (int)from_below<decltype(step)::value>((uint32_t)INT32_MIN, (uint32_t)x)); });
    return of_lane(x, 63);
}
__device__ __forceinline__ void first_best(float& top, int& best) {
    const float most = max_of(top);
    best = min_of(top == most ? best : INT32_MAX);
    top = most;
}

// Eight values of a row of n >= 8 from place first_of(i, n) on: i, or the last at which there are eight
__device__ __forceinline__ int first_of(int i, int n) { return min(i, n - 8); }
template <typename T> __device__ __forceinline__ Eight<T> load_eight(const T* row, int i, int n) {
    Eight<T> x;
    __builtin_memcpy(&x, row + first_of(i, n), sizeof(x));
    return x;
}

// Which of the eight places from `at` on lie outside [i, end), as bits
__device__ __forceinline__ uint32_t outside(int at, int i, int end) {
    const int skip = min(i - at, 8), stop = min(max(end - at, 0), 8);
    return ((1u << skip) - 1u) | ~((1u << stop) - 1u);
}
template <typename T> __device__ __forceinline__ void leave_out(uint32_t out, T none, T (&x)[8]) {
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = out >> e & 1u ? none : x[e];
}

// A sum in 32 bits is off by less than kDoubt of itself: a weight 2^-t by three roundings of its exponent, 1.3e-7 t of itself, and a step
// of the exponential, 1.2e-7; the mean of t over the weights is at most log2 of the vocabulary (it is the entropy of W / Z less log2 Z, and
// Z is 1 at least), 31, so 4.1e-6 in all; eight weights at a time are added in 32 bits, 2e-7, the rest in 64.
constexpr double kDoubt = 0x1p-17;
constexpr double kQuickRate = 1e6;        // log2(e) / T at most: (l - top) log2(e) / T is a number then

// Parts [p, p_end) of a row by one wave: their largest logits and the sums against them, in one pass: what is summed so far is
// scaled when a larger logit comes.  The next part's runs are on their way while one's are looked at.  QUICK: weights in 32 bits.
template <bool QUICK, typename L>
__device__ __forceinline__ void first_sums(const L* row, double rate, int vocabulary, int part_length, int p, int p_end, Part* out) {
    const int lane = threadIdx.x & 63;
    if (p >= p_end) return;
    if (vocabulary < 8) {                 // a token per lane
        const float x = lane < vocabulary ? value(row[lane]) : -INFINITY;
        Part part{1.0, x == x ? x : -INFINITY, lane};
        first_best(part.top, part.best);
        if (rate != 0.0) part.sum = sum_of(part.top > -INFINITY ? weight_of(x, part.top, rate) : 0.0);
        if (lane == 0) out[p] = part;
        return;
    }
    constexpr int kRing = kPart / kRun;
    const int last = (int)min((int64_t)p_end * part_length, (int64_t)vocabulary);
    const auto load = [&](int i) { return load_eight(row, i + lane * 8, vocabulary); };
    Eight<L> ring[kRing];
#pragma unroll
    for (int r = 0; r < kRing; ++r) {
        ring[r] = load(p * part_length + r * kRun);
        __builtin_amdgcn_sched_barrier(0);                       // (in this order: the loop waits for one at a time)
    }
    float top = -INFINITY;
    int best = INT32_MAX, end = (int)min((int64_t)p * part_length + part_length, (int64_t)last);
    double sum = 0.0;
#pragma unroll 1
    for (int i1 = p * part_length; i1 < last; i1 += kPart) {
        if (QUICK && rate != 0.0) {
            // one largest logit for four runs, and the next four on their way as soon as these are taken apart
            float x[kRing][8], m = -INFINITY;
#pragma unroll
            for (int r = 0; r < kRing; ++r) {
                const int i0 = i1 + r * kRun, i = i0 + lane * 8;
#pragma unroll
                for (int e = 0; e < 8; ++e) x[r][e] = value(ring[r], e);
                if (i0 + kRun > vocabulary) leave_out(outside(first_of(i, vocabulary), i, vocabulary), -INFINITY, x[r]);
#pragma unroll
                for (int e = 0; e < 8; ++e) m = fmaxf(m, x[r][e]);
                ring[r] = load(min(i0 + kPart, last));
                __builtin_amdgcn_sched_barrier(0);
            }
            m = max_of(m);
            if (m > top) {
                if (sum > 0.0) sum *= weight_of(top, m, rate);
                top = m;
            }
            const float by = fmaxf((float)rate, 1e-30f);         // (times -inf: -inf)
            if (top < INFINITY) {
#pragma unroll
                for (int r = 0; r < kRing; ++r) {
                    float w[8];
#pragma unroll
                    for (int e = 0; e < 8; ++e) w[e] = __builtin_amdgcn_exp2f(fmaxf(x[r][e] - top, -INFINITY) * by);
                    sum += (double)(((w[0] + w[1]) + (w[2] + w[3])) + ((w[4] + w[5]) + (w[6] + w[7])));
                }
            } else {
#pragma unroll
                for (int r = 0; r < kRing; ++r) {
#pragma unroll
                    for (int e = 0; e < 8; ++e) sum += x[r][e] == top ? 1.0 : 0.0;
                }
            }
        } else {
#pragma unroll
            for (int r = 0; r < kRing; ++r) {
                const int i0 = i1 + r * kRun, i = i0 + lane * 8, at = first_of(i, vocabulary);
                if (i0 < last) {
                    float x[8], m = -INFINITY;                       // (fmaxf passes over a NaN)
#pragma unroll
                    for (int e = 0; e < 8; ++e) x[e] = value(ring[r], e);
                    if (i0 + kRun > vocabulary) leave_out(outside(at, i, vocabulary), -INFINITY, x);
#pragma unroll
                    for (int e = 0; e < 8; ++e) m = fmaxf(m, x[e]);
                    if (rate == 0.0) {
                        if (m > top) {
                            top = m;
#pragma unroll
                            for (int e = 7; e >= 0; --e)
                                if (x[e] == m) best = at + e;
                        }
                    } else {
                        m = max_of(m);
                        if (m > top) {
                            if (sum > 0.0) sum *= weight_of(top, m, rate);
                            top = m;
                        }
                        if (!QUICK && top > -INFINITY) {
                            double w[8];
                            weights_of(x, top, rate, w);
#pragma unroll
                            for (int e = 0; e < 8; ++e) sum += w[e];
                        }
                    }
                }
                // (behind the last use of what it replaces, so that it comes to the same registers)
                ring[r] = load(min(i0 + kPart, last));
                __builtin_amdgcn_sched_barrier(0);
            }
        }
        if (i1 + kPart < end) continue;
        Part part{1.0, top, best};
        if (rate == 0.0) first_best(part.top, part.best);
        else part.sum = sum_of(sum);
        if (lane == 0) out[p] = part;
        ++p;
        end = (int)min((int64_t)end + part_length, (int64_t)last);
        top = -INFINITY;
        best = INT32_MAX;
        sum = 0.0;
    }
}

// Sum of a row's weights over [from, to) without the tokens that fell, by one wave; `fell`: room for kPart bits
template <typename L, typename Q>
__device__ __forceinline__ double sum_again(const Row<L, Q>& row, int from, int to, const int32_t* fallen, int n_fallen, uint32_t* fell) {
    const int lane = threadIdx.x & 63;
    const bool drafted = row.draft && row.shift > 0.0;
    double sum = 0.0;
    if (row.n < 8) {                      // a token per lane
        const int i = from + lane;
        if (i < to) sum = row.weight(value(row.logits[i]), row.proposed(i));
        for (int k = 0; k < n_fallen; ++k)
            if (fallen[k] == i) sum = 0.0;
        return sum_of(sum);
    }
    for (int i0 = from; i0 < to; i0 += kPart) {
        bool any = false;
        for (int k0 = 0; k0 < n_fallen; k0 += 64) {
            const int x = k0 + lane < n_fallen ? fallen[k0 + lane] - i0 : -1;
            const bool here = x >= 0 && x < min(kPart, to - i0);
            if (!__ballot(here)) continue;
            if (!any) {
                fell[lane] = 0u;
                __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            }
            any = true;
            if (here) atomicOr(&fell[x >> 5], 1u << (x & 31));
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        const int end = min(i0 + kPart, to);
        const auto logits = [&](int i) { return load_eight(row.logits, i + lane * 8, row.n); };
        const auto drafts = [&](int i) { return drafted ? load_eight(row.draft, i + lane * 8, row.n) : Eight<Q>{}; };
        constexpr int kAtOnce = 2;
        Eight<L> ring[kAtOnce];
        Eight<Q> draft_ring[kAtOnce];
#pragma unroll
        for (int r = 0; r < kAtOnce; ++r) {
            ring[r] = logits(i0 + r * kRun);
            draft_ring[r] = drafts(i0 + r * kRun);
            __builtin_amdgcn_sched_barrier(0);
        }
#pragma unroll 1
        for (int i2 = i0; i2 < end; i2 += kAtOnce * kRun) {
#pragma unroll
            for (int r = 0; r < kAtOnce; ++r) {
                const int i1 = i2 + r * kRun, i = i1 + lane * 8, at = first_of(i, row.n);
                double w[8];
                row.eight(ring[r], draft_ring[r], w);
                if (any || i1 + kRun > end) {
                    uint32_t out = outside(at, i, end);
                    if (any) {
                        const int bit = at - i0, word = min(max(bit, 0) >> 5, kPart / 32 - 2);
                        const uint64_t bits = (uint64_t)fell[word + 1] << 32 | fell[word];
                        out |= (uint32_t)(bit < 0 ? bits << min(-bit, 8) : bits >> (bit - 32 * word));
                    }
                    leave_out(out, 0.0, w);
                }
#pragma unroll
                for (int e = 0; e < 8; ++e) sum += w[e];
                ring[r] = logits(i1 + kAtOnce * kRun);
                draft_ring[r] = drafts(i1 + kAtOnce * kRun);
                __builtin_amdgcn_sched_barrier(0);
            }
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    }
    return sum_of(sum);
}

// One sequence's walk, by a workgroup.  Every wave takes all decisions itself, from the same numbers.  Of a wave that looks at one
// node only (THREADS 64) there is no Shared.
template <typename L, typename Q, int THREADS> struct Walk {
    static constexpr int kWaves = THREADS / 64;
    static constexpr bool kOneNode = THREADS == 64;
    const VerifyArgs& a;
    Shared* const sh;
    const bool notes;                     // this workgroup writes the path
    int b, start, nodes;
    bool greedy;
    Row<L, Q> row;
    int node, count, child, asked;        // children below `child` have fallen, `asked` of them
    int summed, fallen;                   // children below `summed` were left out of the sum; entries of sh->fallen
    int held, where;                      // the last sum: kFirst, kAgain or kQuick; as in State
    bool exact, always_exact;             // the node's first sum has to be 64 bits
    double all, whole, left;              // Z, Z when the sum was taken, r
    // the strip of 64 nodes whose children are asked next: a child per lane, and which lanes
    int strip = 0, token = -1;
    uint64_t kids = 0, all_kids = 0;      // .. are left, were there
    float logit = 0.f, draft = 0.f, u = 0.f;
    int early_parent, early_token, early_stands;      // of node threadIdx.x, on their way

    __device__ __forceinline__ Walk(const VerifyArgs& args, Shared* shared, int sequence, bool writes) : a(args), sh(shared), notes(writes), b(sequence) {
        start = min(max(a.q_starts[b], 0), a.nodes);
        nodes = max(min(a.q_starts[b + 1], a.nodes) - start, 0);
        const float tau = a.temperatures ? a.temperatures[b] : a.temperature;
        greedy = !(tau > 0.f);
        row.rate = greedy ? 0.0 : fmax(1.4426950408889634074 / (double)tau, 1e-300);
        all = whole = left = 1.0;
        node = child = asked = summed = fallen = held = where = 0;
        count = 1;
        row.shift = 0.0;
        row.top = -INFINITY;
        row.best = -1;
        row.n = a.vocabulary;
        always_exact = exact = !a.draft && row.rate > kQuickRate;
        const bool mine = !kOneNode && (int)threadIdx.x < min(nodes, kTree);
        early_parent = mine ? parent_in_memory(threadIdx.x) : -1;
        early_token = mine ? token_in_memory(threadIdx.x) : -1;
        early_stands = mine && a.all_parts ? a.stands[start + threadIdx.x] : -1;
    }
    // The tree is in LDS from here on
    __device__ __forceinline__ void read_tree() {
        if ((int)threadIdx.x < min(nodes, kTree)) {
            sh->parent[threadIdx.x] = early_parent;
            sh->token[threadIdx.x] = early_token;
            sh->stands[threadIdx.x] = early_stands;
        }
        for (int j = threadIdx.x + THREADS; j < min(nodes, kTree); j += THREADS) {
            sh->parent[j] = parent_in_memory(j);
            sh->token[j] = token_in_memory(j);
            sh->stands[j] = a.all_parts ? a.stands[start + j] : -1;
        }
        __syncthreads();
    }
    __device__ __forceinline__ int parent_in_memory(int j) const {
        const int64_t p = a.parent[start + j];
        return p >= 0 && p < j ? (int)p : -1;
    }
    __device__ __forceinline__ int token_in_memory(int j) const {
        const int64_t x = a.tokens[start + j];
        return x >= 0 && x < a.vocabulary ? (int)x : -1;
    }
    __device__ __forceinline__ bool is_child(int j) const {
        if (j >= nodes) return false;
        if constexpr (kOneNode) return parent_in_memory(j) == node;
        else return (j < kTree ? sh->parent[j] : parent_in_memory(j)) == node;
    }
    __device__ __forceinline__ int token_of(int j) const {
        if constexpr (kOneNode) return token_in_memory(j);
        else return j < kTree ? sh->token[j] : token_in_memory(j);
    }
    // (trees that overlap leave entries that nobody wrote: a child comes behind its parent, whatever is there)
    __device__ __forceinline__ int stands_at(int j) const {
        const int child = j < kTree ? sh->stands[j] : a.stands[start + j];
        return child > j && child < nodes ? child : -1;
    }

    // To the next strip with children of the node, from node `from` on: what they are asked with
    __device__ __forceinline__ void look(int from) {
        const int lane = threadIdx.x & 63;
        kids = 0;
        for (strip = from; strip < nodes && !kids; strip += kids ? 0 : 64) kids = __ballot(is_child(strip + lane));
        all_kids = kids;
        const bool mine = kids >> lane & 1;
        if (!kids) return;
        // (loads of all lanes, the others' from a place that there is: a branch around them would wait for each)
        token = mine ? token_of(strip + lane) : -1;
        const int x = max(token, 0);
        const L l = row.logits[x];
        Q q{};
        if (row.draft) q = row.draft[x];
        u = a.u_accept[start + min(strip + lane, nodes - 1)];
        logit = value(l);
        draft = value(q);
    }
    __device__ __forceinline__ void stand_on(int at, int how_many) {
        node = at;
        count = how_many;
        child = summed = at + 1;
        fallen = asked = 0;
        left = 1.0;
        exact = always_exact;
        row.logits = static_cast<const L*>(a.logits) + (start + (int64_t)node) * a.logits_stride;
        row.draft = a.draft && !greedy ? static_cast<const Q*>(a.draft) + (start + (int64_t)node) * a.draft_stride : nullptr;
        row.shift = 0.0;
        row.top = -INFINITY;
        row.best = -1;
    }
    // .. from where on it goes on through children that are known to stand
    __device__ __forceinline__ void stand_at(int at, int how_many) {
        if constexpr (kOneNode) {
            node = at;
            return;
        }
        note(at, how_many);
        if (a.all_parts) {
            for (int j = stands_at(at); j >= 0 && how_many < a.max_path; j = stands_at(j)) note(at = j, ++how_many);
        }
        stand_on(at, how_many);
        look(at + 1);
        exact |= !a.draft && !kids;       // nothing to ask: its sum is the one that the next token is picked from
    }
    __device__ __forceinline__ const Part* parts_of(const Part* all, int64_t which) const { return all + which * a.parts_per_row; }
    __device__ __forceinline__ const Part* parts_of_node() const { return parts_of(a.all_parts, start + (int64_t)node); }
    __device__ __forceinline__ const Part* parts_of_step(int turn) const { return parts_of(a.parts[turn], b); }
    __device__ __forceinline__ void take(int what, const Part* parts) {
        if (what == kAgain) take_again(parts);
        else take_first(parts);
        held = what;
    }
    // Where the state is, with the sum that it waits for (or the last one, at a walk's end); the tree is in LDS behind it
    __device__ __forceinline__ void resume(const State& s, const Part* parts) {
        stand_on(s.node, s.count);
        exact |= s.exact != 0;
        if (s.phase != kFirst) {
            child = s.child;
            asked = s.asked;
            left = s.left;
            row.shift = s.shift;
            row.top = s.top;
        }
        if (parts) take(s.phase == kDone ? s.held : s.phase == kFirst && !exact && !a.draft ? kQuick : s.phase, parts);
        read_tree();
        if (s.phase == kFirst && !parts) {
            stand_at(s.node, s.count);
            exact |= s.exact != 0;
        } else if (s.phase != kDone) {
            look(child);
        }
        if (s.phase == kFirst) exact |= !a.draft && !kids;
    }
    __device__ __forceinline__ void part_range(int p, int* from, int* to) const {
        *from = (int)min((int64_t)p * a.part_length, (int64_t)a.vocabulary);
        *to = (int)min((int64_t)*from + a.part_length, (int64_t)a.vocabulary);
    }

    // The parts of the first sum of the row: its largest logit, Z.  (Every wave writes the same to sh->sum.)
    __device__ __forceinline__ void take_first(const Part* parts) {
        const int lane = threadIdx.x & 63;
        Part mine = parts[min(lane, a.parts_per_row - 1)];
        if (lane >= a.parts_per_row) mine = Part{0.0, -INFINITY, INT32_MAX};
        float top = mine.top;
        int best = mine.best;
        for (int p = lane + 64; p < a.parts_per_row; p += 64)
            if (parts[p].top > top) top = parts[p].top, best = parts[p].best;
        first_best(top, best);
        row.top = top;
        row.best = top > -INFINITY ? best : -1;
        double sum = 0.0;
        if (!greedy) {
            for (int p = lane; p < a.parts_per_row; p += 64) {
                const Part part = p == lane ? mine : parts[p];
                const double s = part.sum > 0.0 ? part.sum * weight_of(part.top, top, row.rate) : 0.0;
                sum += s;
                if constexpr (!kOneNode) sh->sum[p] = s;
            }
        }
        whole = all = sum_of(sum);
        summed = child;
    }
    // .. of a sum of W
    __device__ __forceinline__ void take_again(const Part* parts) {
        double sum = 0.0;
        for (int p = threadIdx.x & 63; p < a.parts_per_row; p += 64) {
            const double s = parts[p].sum;
            sum += s;
            sh->sum[p] = s;
        }
        whole = all = sum_of(sum);
        summed = child;
    }

    // Whether a child before child j has its token x
    __device__ __forceinline__ bool fell_before(int j, int x) const {
        for (int i0 = node + 1; i0 < j; i0 += 64) {
            const int i = i0 + (threadIdx.x & 63);
            if (__ballot(i < j && is_child(i) && token_of(i) == x)) return true;
        }
        return false;
    }

    // .. of the strip's child of lane l
    __device__ __forceinline__ bool fell_before_in_strip(int l, int x) const {
        return __ballot((all_kids >> (threadIdx.x & 63) & 1) && (int)(threadIdx.x & 63) < l && token == x) || fell_before(strip, x);
    }

    // Asks children until one stands (kFirst: `node` is that one now), a sum of W is wanted (kAgain) or there are no more (kDone)
    __device__ __forceinline__ int ask() {
        if (row.top == -INFINITY) return kDone;                  // nothing to choose: all children fall
        while (kids && count < a.max_path && asked < kChildren) {
            const double q = row.draft ? fmax((double)draft, 0.0) : 0.0, w = row.weight(logit, q);
            for (; kids && asked < kChildren; kids &= kids - 1) {
                const int l = __ffsll((unsigned long long)kids) - 1, x = of_lane(token, l), j = strip + l;
                ++asked;
                child = j + 1;
                if (x < 0) continue;
                if (greedy) {
                    if (x != row.best) continue;
                    stand_at(j, count + 1);
                    return kFirst;
                }
                if (fell_before_in_strip(l, x)) continue;
                const double wx = of_lane(w, l), qx = of_lane(q, l), ux = of_lane((double)u, l);
                const bool drawn = qx > 0.0 && left > 0.0;
                // Too near to tell by a sum in 32 bits: once more, in 64
                if (held == kQuick && fabs(ux * all - wx) <= kDoubt * whole) {
                    stand_at(node, count);
                    exact = true;
                    return kFirst;
                }
                // (W is at most Z: with u at 1 or more only the rounding of Z could let a given child stand)
                if (drawn ? ux * all * qx < wx * left : ux < 1.0 && ux * all < wx) {
                    stand_at(j, count + 1);
                    return kFirst;
                }
                if (drawn) {
                    row.shift += all / left;
                    left -= qx;
                } else {
                    // the sum loses one term; where little is left of it, it is taken again
                    all -= wx;
                    if (wx == 0.0 || all > whole * 0x1p-10) continue;
                }
                kids = 0;
                return kAgain;
            }
            if (asked < kChildren) look(strip + 64);
        }
        return kDone;
    }

    // The tokens that fell, in sh->fallen; behind those that the sum leaves out (returned: how many) each comes once
    __device__ __forceinline__ int collect() {
        const int lane = threadIdx.x & 63;
        __syncthreads();
        fallen = 0;
        for (int i0 = node + 1; i0 < summed; i0 += 64) {
            const int i = i0 + lane, x = i < summed && is_child(i) ? token_of(i) : -1;
            const uint64_t those = __ballot(x >= 0);
            if (x >= 0 && threadIdx.x < 64) sh->fallen[fallen + __popcll(those & ((1ull << lane) - 1))] = x;
            fallen += __popcll(those);
        }
        const int before = fallen;
        for (int i0 = summed; i0 < child; i0 += 64) {
            const int i = i0 + lane, mine = i < child && is_child(i) ? token_of(i) : -1;
            for (uint64_t those = __ballot(mine >= 0); those; those &= those - 1) {
                const int l = __ffsll((unsigned long long)those) - 1, x = of_lane(mine, l);
                if (fell_before(i0 + l, x)) continue;
                if (threadIdx.x == 0) sh->fallen[fallen] = x;
                ++fallen;
            }
        }
        __syncthreads();
        return before;
    }

    __device__ __forceinline__ int share(int which, int waves) const { return (int)((int64_t)a.parts_per_row * which / waves); }
    // The share of wave `which` of `waves` in the row's sums: into out[part]
    template <bool QUICK> __device__ __forceinline__ void sum_parts(bool first, int which, int waves, Part* out) {
        const int p0 = share(which, waves), p1 = share(which + 1, waves);
        if (first) {
            first_sums<QUICK>(row.logits, row.rate, a.vocabulary, a.part_length, p0, p1, out);
            return;
        }
        for (int p = p0; p < p1; ++p) {
            int from, to;
            part_range(p, &from, &to);
            const double sum = sum_again(row, from, to, sh->fallen, fallen, sh->fell[threadIdx.x >> 6]);
            if ((threadIdx.x & 63) == 0) out[p] = Part{sum, row.top, 0};
        }
    }
    // Sums over the whole row by this workgroup alone, a part a wave: into sh->part
    __device__ __forceinline__ void sum_alone(bool first) {
        const int wave = threadIdx.x >> 6;
        __syncthreads();
        sum_parts<false>(first, wave, kWaves, sh->part);
        __syncthreads();
    }

    // The smallest token at which the running sum of the weights passes u of all of it, the last one with any weight where rounding
    // (or u >= 1) lets none; -1 where there is no weight
    __device__ __forceinline__ int pick(double u) {
        const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
        __syncthreads();                  // sh->sum
        if (child > summed) {
            // a part loses the terms that fell since its sum was taken; where little is left of it, its sum is taken again
            const int old = collect();
            for (int k = old + tid; k < fallen; k += THREADS) {
                const int x = sh->fallen[k];
                sh->lost[k] = row.weight(value(row.logits[x]), row.proposed(x));
            }
            __syncthreads();
            for (int p = tid; p < a.parts_per_row; p += THREADS) {
                double lost = 0.0;
                for (int k = old; k < fallen; ++k)
                    if (sh->fallen[k] / a.part_length == p) lost += sh->lost[k];
                const double s = sh->sum[p];
                if (lost > 0.0) sh->sum[p] = s - lost > s * 0x1p-10 ? s - lost : -1.0;
            }
            __syncthreads();
        } else {
            collect();
        }
        double sum;
        for (int resort = 0;; ++resort) {
            for (int p = wave; p < a.parts_per_row; p += kWaves) {
                if (sh->sum[p] >= 0.0) continue;
                int from, to;
                part_range(p, &from, &to);
                const double s = sum_again(row, from, to, sh->fallen, fallen, sh->fell[wave]);
                if (lane == 0) sh->sum[p] = s;
            }
            __syncthreads();
            sum = 0.0;
            for (int p = lane; p < a.parts_per_row; p += 64) sum += sh->sum[p];
            sum = sum_of(sum);
            if (sum > 0.0) break;
            if (resort == 2) return -1;                          // rounding left nothing: P without what fell, then P
            row.shift = 0.0;
            if (resort == 1) fallen = 0;
            __syncthreads();
            for (int p = tid; p < a.parts_per_row; p += THREADS) sh->sum[p] = -1.0;
            __syncthreads();
        }
        double target = u < 1.0 ? u * sum : INFINITY;
        int chosen = -1, last = -1;
        double before = 0.0, at_chosen = 0.0;
        for (int p0 = 0; p0 < a.parts_per_row && chosen < 0; p0 += 64) {
            const double s = p0 + lane < a.parts_per_row ? sh->sum[p0 + lane] : 0.0;
            const double up_to = sum_up_to(s);
            const uint64_t weighs = __ballot(s > 0.0), passes = __ballot(s > 0.0 && before + up_to > target);
            if (weighs) last = p0 + 63 - __builtin_clzll(weighs);
            if (passes) {
                const int l = __ffsll((unsigned long long)passes) - 1;
                chosen = p0 + l;
                at_chosen = before + (of_lane(up_to, l) - of_lane(s, l));
            }
            before += of_lane(up_to, 63);
        }
        if (chosen < 0) {
            chosen = last;
            at_chosen = 0.0;
            target = INFINITY;
        }
        target -= at_chosen;
        int from, to;
        part_range(chosen, &from, &to);
        int found = -1;
        for (; from < to; from += THREADS * 8) {
            // eight tokens a thread: threads' sums, then the tokens of each thread
            double w[8], mine = 0.0;
            int i = from + tid * 8, at = i;
            if (row.n < 8) {              // a token per thread
                at = i = from + tid;
#pragma unroll
                for (int e = 0; e < 8; ++e) w[e] = 0.0;
                if (i < to) w[0] = row.weight(value(row.logits[i]), row.proposed(i));
            } else {
                at = first_of(i, row.n);
                Eight<Q> draft = {};
                if (row.draft && row.shift > 0.0) draft = load_eight(row.draft, i, row.n);
                row.eight(load_eight(row.logits, i, row.n), draft, w);
                leave_out(outside(at, i, to), 0.0, w);
            }
            for (int k = 0; k < fallen; ++k) {
                const int f = sh->fallen[k] - at;
                if (f >= 0 && f < 8) leave_out(1u << f, 0.0, w);
            }
#pragma unroll
            for (int e = 0; e < 8; ++e) mine += w[e];
            const double up_to = sum_up_to(mine);
            __syncthreads();
            if (lane == 63) sh->wave_sum[wave] = up_to;
            __syncthreads();
            double run = up_to - mine, here = 0.0;
            for (int k = 0; k < kWaves; ++k) {
                if (k < wave) run += sh->wave_sum[k];
                here += sh->wave_sum[k];
            }
            // Every thread names its first token that passes the target; the smallest counts.  None: the largest with any weight.
            int passes = INT32_MAX, weighs = -1;
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                run += w[e];
                if (w[e] > 0.0) {
                    weighs = at + e;
                    if (run > target && passes == INT32_MAX) passes = at + e;
                }
            }
            passes = min_of(passes);
            weighs = max_of(weighs);
            if (lane == 0) sh->best[wave] = passes, sh->last[wave] = weighs;
            __syncthreads();
            for (int k = 0; k < kWaves; ++k) {
                passes = min(passes, sh->best[k]);
                weighs = max(weighs, sh->last[k]);
            }
            if (weighs >= 0) found = weighs;
            if (passes != INT32_MAX) return passes;
            target -= here;
        }
        return found;
    }

    // The end of a sequence's walk
    __device__ __forceinline__ void answer() {
        int next = -1;
        if (nodes == 0) count = 0;
        else if (row.top > -INFINITY) next = greedy ? row.best : pick(a.u_next[b]);
        if (threadIdx.x == 0) {
            a.counts[b] = count;
            a.next[b] = next;
        }
        for (int i = count + threadIdx.x; i < a.max_path; i += THREADS) a.path[(int64_t)b * a.max_path + i] = -1;
    }
    __device__ __forceinline__ void note(int at, int how_many) const {
        if (notes && threadIdx.x == 0) a.path[(int64_t)b * a.max_path + how_many - 1] = at;
    }

    // Takes decisions for as long as the sums are there; `taken`: the state's is
    __device__ __forceinline__ int go_on(int phase, bool taken) {
        for (;;) {
            if (!taken) {
                if (phase != kFirst || !a.all_parts || !kids || exact) return phase;
                take(a.draft ? kFirst : kQuick, parts_of_node());
                where = kOfNode;
            }
            taken = false;
            phase = ask();
            if (phase == kDone) return phase;
        }
    }
};

// A node's sequence: how many start at or before it (less one), by 64 places at a time
__device__ __forceinline__ int sequence_of(const VerifyArgs& a, int64_t t) {
    const int lane = threadIdx.x & 63;
    int first = 0, count = a.batch;
    while (count > 64) {
        const int step = (count + 63) / 64, at = lane * step;
        const int before = __popcll(__ballot(at < count && a.q_starts[first + min(at, count - 1)] <= t));
        if (before == 0) return -1;
        first += (before - 1) * step;
        count = min(step, count - (before - 1) * step);
    }
    return first - 1 + __popcll(__ballot(lane < count && a.q_starts[first + min(lane, count - 1)] <= t));
}

// The first sums of all rows, largest logit and sum in one pass.  blockIdx.x: parts of a row, .y: node.  250 rows of 32000 float32 (16 trees of
// 64 nodes) 18 us in sums of 32 bits, 32 MB; 32 trees' of 50021 float16 with draft probabilities 22.5 us in 64.  2048 workgroups for all rows: 1024 56
// us instead of 53.5 for 8 x 64 rows of 131072 tokens, 4096 52 there and 52 instead of 50 for 16 x 64 of 32000.
template <typename L, bool QUICK> __global__ __launch_bounds__(kStepThreads, QUICK && sizeof(L) == 2 ? 4 : 3) void stats_kernel(VerifyArgs a) {
    constexpr int kWaves = kStepThreads / 64;
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    for (int64_t t = blockIdx.y; t < a.nodes; t += gridDim.y) {
        const int b = sequence_of(a, t);
        if (b < 0) continue;
        const int start = max(a.q_starts[b], 0), end = min(a.q_starts[b + 1], a.nodes), node = (int)(t - start);
        uint64_t any = 0;
        for (int64_t j = t + 1; j < end && !any; j += 64) any = __ballot(j + lane < end && a.parent[j + lane] == node);
        if (!any) continue;
        const double rate = rate_of(a, b);
        const int which = blockIdx.x * kWaves + wave, waves = gridDim.x * kWaves;
        first_sums<QUICK>(static_cast<const L*>(a.logits) + t * a.logits_stride, rate, a.vocabulary, a.part_length,
                   (int)((int64_t)a.parts_per_row * which / waves), (int)((int64_t)a.parts_per_row * (which + 1) / waves), a.parts_out + t * a.parts_per_row);
    }
}

// Which child stands at each node, by the first sums of all rows, a wave per node: a walk does not wait for one decision after the
// other (2 us each: parts, largest, sum, the children's logits).  4.4 us for a chain of 6, 7.3 for 16 trees of 64; the calls without it 38 instead
// of 29 us, and 55 instead of 53.
template <typename L, typename Q> __global__ __launch_bounds__(kStepThreads) void stands_kernel(VerifyArgs a) {
    const int lane = threadIdx.x & 63;
    for (int64_t t = (int64_t)blockIdx.x * (kStepThreads / 64) + (threadIdx.x >> 6); t < a.nodes; t += (int64_t)gridDim.x * (kStepThreads / 64)) {
        const int b = sequence_of(a, t);
        if (b < 0) continue;
        Walk<L, Q, 64> w(a, nullptr, b, false);
        const int node = (int)(t - w.start);
        if (node < 0 || node >= w.nodes) continue;
        w.stand_on(node, 1);
        w.look(node + 1);
        int phase = kDone;
        if (w.kids && !w.exact) {
            w.take(a.draft ? kFirst : kQuick, w.parts_of_node());
            phase = w.ask();
        }
        if (lane == 0) a.stands[t] = phase == kFirst && !w.exact ? w.node : -1;
    }
}

// blockIdx.x: parts of a row, .y: sequence.  DRAWN: there are the draft's probabilities, and sums are 64 bits.  Without them a first
// sum of 32 bits is enough for almost every decision; rows whose sum has to be 64 bits wait for last_kernel, sums without what fell for
// walk_kernel.  128 sequences, 131072 bfloat16: 11 us the roots' step (33 MB), 15 to 10 the next ones while ever fewer go on; 5 to 6 of them pass
// before the first load of a row (state, tree, the parts so far, the children's logits).  32 sequences of 50021, drawn: 10 us.
template <typename L, typename Q, bool DRAWN> __global__ __launch_bounds__(kStepThreads, DRAWN ? 2 : 3) void step_kernel(VerifyArgs a) {
    constexpr int kWaves = kStepThreads / 64;
    __shared__ Shared sh;
    const int wave = threadIdx.x >> 6;
    const bool speaks = blockIdx.x == 0;
    for (int b = blockIdx.y; b < a.batch; b += gridDim.y) {
        State s{0, 1, 1, 0, 1, kFirst, kFirst, 0, 0, 0, 0.0, 1.0, 0.f, 0};
        if (!a.fresh) s = a.states[a.turn ^ 1][b];
        if (!a.fresh && (s.phase == kDone || !s.ready)) {
            if (speaks && threadIdx.x == 0) a.states[a.turn][b] = s;
            continue;
        }
        __syncthreads();
        Walk<L, Q, kStepThreads> w(a, &sh, b, speaks);
        if (w.nodes == 0) {
            s.phase = kDone;
        } else if (a.fresh && !a.all_parts) {         // the roots' sums wait for nothing
            w.stand_on(0, 1);
            w.note(0, 1);
        } else {
            w.where = a.turn ^ 1;
            w.resume(s, a.fresh ? nullptr : w.parts_of_step(a.turn ^ 1));
            s.phase = w.go_on(s.phase, !a.fresh);
        }
        const bool sums = s.phase != kDone && (DRAWN || (s.phase == kFirst && !w.exact));
        if (speaks && threadIdx.x == 0)
            a.states[a.turn][b] = State{w.node, w.count, w.child, w.asked, w.summed, s.phase, w.held, w.where, sums, w.exact, w.row.shift, w.left, w.row.top, 0};
        if (!sums) continue;
        if (DRAWN && s.phase == kAgain) {
            w.summed = w.child;
            w.collect();
        }
        Part* out = a.parts[a.turn] + (int64_t)b * a.parts_per_row;
        const int which = blockIdx.x * kWaves + wave, waves = gridDim.x * kWaves;
        if constexpr (DRAWN) w.template sum_parts<false>(s.phase == kFirst, which, waves, out);
        else first_sums<true>(w.row.logits, w.row.rate, a.vocabulary, a.part_length, w.share(which, waves), w.share(which + 1, waves), out);
    }
}

// Sums of 64 bits where there are none: of the row that a sequence's next token is picked from, and of rows whose children's fate
// sums of 32 bits do not tell.  They go to the buffer that the last step did not write.  Without steps that is the row of the last child that
// is known to stand.  blockIdx.x: parts of a row, .y: sequence.  128 rows of 131072 bfloat16 23 us, of which the exponentials take half; 16 of
// 32000 float32 7 us.
__device__ __forceinline__ bool wants_last(const VerifyArgs& a, const State& s, double rate) {
    if (a.fresh) return a.all_parts && rate != 0.0;
    return s.phase == kDone ? s.held == kQuick && rate != 0.0 : s.phase == kFirst && !s.ready;
}
template <typename L> __global__ __launch_bounds__(kStepThreads, 3) void last_kernel(VerifyArgs a) {
    constexpr int kWaves = kStepThreads / 64;
    __shared__ int32_t stands[kTree];
    const int which = blockIdx.x * kWaves + (threadIdx.x >> 6), waves = gridDim.x * kWaves;
    for (int b = blockIdx.y; b < a.batch; b += gridDim.y) {
        State s = {};
        if (!a.fresh) s = a.states[a.turn][b];
        const int start = min(max(a.q_starts[b], 0), a.nodes), nodes = min(a.q_starts[b + 1], a.nodes) - start;
        const double rate = rate_of(a, b);
        if (nodes <= 0 || !wants_last(a, s, rate)) continue;
        if (a.fresh) {
            __syncthreads();
            for (int j = threadIdx.x; j < min(nodes, kTree); j += kStepThreads) stands[j] = a.stands[start + j];
            __syncthreads();
            for (int count = 1; count < a.max_path; ++count) {
                const int child = s.node < kTree ? stands[s.node] : a.stands[start + s.node];
                if (child <= s.node || child >= nodes) break;
                s.node = child;
            }
        }
        first_sums<false>(static_cast<const L*>(a.logits) + (start + (int64_t)s.node) * a.logits_stride, rate, a.vocabulary, a.part_length,
                          (int)((int64_t)a.parts_per_row * which / waves), (int)((int64_t)a.parts_per_row * (which + 1) / waves),
                          a.parts[a.turn ^ 1] + (int64_t)b * a.parts_per_row);
    }
}

// What is left of every walk, and the next tokens, a workgroup per sequence: sums here are one workgroup's work, so that launches before it
// leave few.  8 us where nothing is left but to pick, 14 for 128 sequences of 131072 tokens, 17 where the decisions at the last node come first
// (16 trees): loads that need each other, and ten barriers.  256 threads look at a part at once, and two workgroups fit a CU: with 512 the call for
// 500 trees of 32000 tokens takes 110 us instead of 100, for 2000 of 8000 173 instead of 137, for few the same; with 128 one to two more up to
// 500, 131 for 2000.
template <typename L, typename Q> __global__ __launch_bounds__(kWalkThreads, 2) void walk_kernel(VerifyArgs a) {
    __shared__ Shared sh;
    for (int b = blockIdx.x; b < a.batch; b += gridDim.x) {
        __syncthreads();
        State s{0, 1, 1, 0, 1, kFirst, kFirst, 0, 0, 0, 0.0, 1.0, 0.f, 0};
        if (!a.fresh) s = a.states[a.turn][b];
        Walk<L, Q, kWalkThreads> w(a, &sh, b, true);
        const bool last = w.nodes > 0 && !a.draft && wants_last(a, s, w.row.rate);
        if (w.nodes > 0 && s.phase == kDone) {
            if (last) s.held = kFirst;
            w.resume(s, last ? w.parts_of_step(a.turn ^ 1) : s.where == kOfNode ? w.parts_of(a.all_parts, w.start + s.node) : w.parts_of_step(s.where));
            w.summed = s.summed;
        } else if (w.nodes > 0) {
            if (last) s.exact = 1;
            bool taken = last || (!a.fresh && s.ready);
            w.where = a.turn;
            w.resume(s, taken && !a.fresh ? w.parts_of_step(last ? a.turn ^ 1 : a.turn) : nullptr);
            if (taken && a.fresh) w.take(kFirst, w.parts_of_step(a.turn ^ 1));
            while ((s.phase = w.go_on(s.phase, taken)) != kDone) {
                if (s.phase == kAgain) {
                    w.summed = w.child;
                    w.collect();
                }
                w.sum_alone(s.phase == kFirst);
                w.take(s.phase, sh.part);
                if (s.phase == kAgain) w.look(w.child);
                taken = true;
            }
            if (w.held == kQuick && !w.greedy && w.row.top > -INFINITY) {       // the sum that the next token is picked from
                w.sum_alone(true);
                w.take(kFirst, sh.part);
                w.summed = w.node + 1;
            }
        }
        w.answer();
    }
}

// ---- host --------------------------------------------------------------------------------------------------------------

struct Plan {
    int32_t parts, part_length;
    bool all;                             // the sums of all nodes with children first
    int32_t steps;
    size_t bytes;
};
size_t rounded(size_t bytes) { return (bytes + 15) / 16 * 16; }

// Chains: no more nodes than paths have places, and not because those are given generously
bool chains(int64_t batch, int64_t nodes, int32_t max_path) { return max_path <= 16 && nodes <= batch * max_path; }

// Sums of all rows first, or only of the rows that walks come to, a launch each?  The first costs with all nodes' tokens, the second a launch
// (and what comes before its first sum) per node of the longest path.  Measured, all rows / steps, us:
//   no draft probabilities  16 x 64 nodes of 32000 tokens 53 / 68, 32 x 64 68 / 71, 8 x 64 of 131072 65 / 66, 64 x 23 of 50021 60 / 76, 16 x 64 of 131072 96 / 67
//                           (both ways have gained since: 54 the third, 60 the last)
//   with them               4 x 64 of 50021 73 / 90, 8 x 23 of 131072 76 / 77, 32 x 23 of 32000 79 / 80, 8 x 64 of 50021 105 / 91
//   chains                  256 x 6 of 131072 152 / 170, with draft probabilities 128 x 6 133 / 171
constexpr double kAllGiven = 80e6, kAllDrawn = 20e6, kAllChains = 200e6;
constexpr int64_t kLargeTree = 1 << 17;   // (a node looks for its children through all behind it: walks do that at a few nodes, all rows at each)
// Steps: one per node of a path, and of each child that falls for draft probabilities some more; behind ten the walks go on alone (a workgroup
// instead of a row's share of them all, but a launch less).  With all sums there a step is one that falls: a chain has one, trees
// of four children 105 us with four steps, 112 with three, 100 with six; of three 84, 82 and 90.
constexpr int kMostSteps = 10, kDrawnSteps = 4;
// Workgroups that share the rows of a launch.  Steps without draft probabilities: 128 sequences of 131072 tokens 116 us with 512 and twice as many
// behind the third step, when fewer sequences are left (117 with 512 throughout, 124 with 384, 122 with 768, 131 with 1024); with them
// 182 with 512, 235 with 384, 229 with 768; last rows 121 with 512, 768 and 1024.
constexpr int kStatsGroups = 2048, kDrawnGroups = 512, kGivenGroups = 512, kLastGroups = 768;

Plan plan_of(int64_t batch, int64_t nodes, int64_t vocabulary, bool draft, int32_t max_path) {
    Plan p;
    p.part_length = (int32_t)((vocabulary + (int64_t)kPart * kMaxParts - 1) / ((int64_t)kPart * kMaxParts) * kPart);
    p.parts = (int32_t)((vocabulary + p.part_length - 1) / p.part_length);
    p.all = (double)nodes * vocabulary <= (chains(batch, nodes, max_path) ? kAllChains : draft ? kAllDrawn : kAllGiven);
    p.all = p.all && (nodes <= kLargeTree || nodes <= 16 * batch);
    p.steps = max_path + (draft ? 3 : 0) < kMostSteps ? max_path + (draft ? 3 : 0) : kMostSteps;
    if (p.all) p.steps = draft ? (chains(batch, nodes, max_path) ? 1 : kDrawnSteps) : 0;
    p.bytes = 2 * (rounded(sizeof(Part) * (size_t)(batch * p.parts)) + rounded(sizeof(State) * (size_t)batch));
    if (p.all) p.bytes += rounded(sizeof(Part) * (size_t)(nodes * p.parts)) + rounded(sizeof(int32_t) * (size_t)nodes);
    return p;
}

template <typename L, typename Q> int launch(VerifyArgs a, const Plan& plan, void* workspace, hipStream_t stream) {
    uint8_t* work = static_cast<uint8_t*>(workspace);
    // as many workgroups as the GPU holds, and no more: what comes before a workgroup's first sum takes as long as one
    const auto groups = [&](int64_t rows, int64_t most) {
        const int64_t needed = (a.parts_per_row + kStepThreads / 64 - 1) / (kStepThreads / 64), fit = (most + rows - 1) / rows;
        return dim3((unsigned)(needed < fit ? needed : fit), (unsigned)(rows < 65535 ? rows : 65535));
    };
    if (plan.all && a.nodes > 0) {
        a.parts_out = reinterpret_cast<Part*>(work);
        a.all_parts = a.parts_out;
        work += rounded(sizeof(Part) * (size_t)a.nodes * a.parts_per_row);
        a.stands = reinterpret_cast<int32_t*>(work);
        work += rounded(sizeof(int32_t) * (size_t)a.nodes);
        if (a.draft) hipLaunchKernelGGL((stats_kernel<L, false>), groups(a.nodes, kStatsGroups), dim3(kStepThreads), 0, stream, a);
        else hipLaunchKernelGGL((stats_kernel<L, true>), groups(a.nodes, kStatsGroups), dim3(kStepThreads), 0, stream, a);
        const unsigned waves = kStepThreads / 64, of_nodes = ((unsigned)a.nodes + waves - 1) / waves;
        hipLaunchKernelGGL((stands_kernel<L, Q>), dim3(of_nodes < 65536 ? of_nodes : 65536), dim3(kStepThreads), 0, stream, a);
    }
    for (int i = 0; i < 2; ++i) {
        a.parts[i] = reinterpret_cast<Part*>(work);
        work += rounded(sizeof(Part) * (size_t)a.batch * a.parts_per_row);
        a.states[i] = reinterpret_cast<State*>(work);
        work += rounded(sizeof(State) * (size_t)a.batch);
    }
    a.fresh = 1;
    for (int i = 0; i < plan.steps; ++i) {
        a.turn = i & 1;
        if (a.draft) hipLaunchKernelGGL((step_kernel<L, Q, true>), groups(a.batch, kDrawnGroups), dim3(kStepThreads), 0, stream, a);
        else hipLaunchKernelGGL((step_kernel<L, float, false>), groups(a.batch, i < 3 ? kGivenGroups : 2 * kGivenGroups), dim3(kStepThreads), 0, stream, a);
        a.fresh = 0;
    }
    if (!a.draft) hipLaunchKernelGGL((last_kernel<L>), groups(a.batch, kLastGroups), dim3(kStepThreads), 0, stream, a);
    hipLaunchKernelGGL((walk_kernel<L, Q>), dim3((unsigned)(a.batch < 65536 ? a.batch : 65536)), dim3(kWalkThreads), 0, stream, a);
    FSTA_HIP_OK(hipGetLastError());
    return FSTA_OK;
}

template <typename L> int launch(const VerifyArgs& a, int32_t draft_dtype, const Plan& plan, void* workspace, hipStream_t stream) {
    if (!a.draft || draft_dtype == FSTA_F32) return launch<L, float>(a, plan, workspace, stream);
    return draft_dtype == FSTA_F16 ? launch<L, Half>(a, plan, workspace, stream) : launch<L, Brain>(a, plan, workspace, stream);
}

bool is_float(int32_t dtype) { return dtype == FSTA_F32 || dtype == FSTA_F16 || dtype == FSTA_BF16; }

}  // namespace
}  // namespace fsta

using namespace fsta;

extern "C" size_t fsta_verify_workspace_bytes(int32_t batch, int32_t nodes, int32_t vocabulary, int32_t max_path, int32_t draft) {
    if (batch <= 0 || nodes < 0 || vocabulary < 1 || max_path < 1) return 0;
    return plan_of(batch, nodes, vocabulary, draft != 0, max_path).bytes;
}

extern "C" int fsta_verify_drafts(const void* logits, int64_t logits_stride, int32_t logits_dtype, const void* draft, int64_t draft_stride,
                                  int32_t draft_dtype, const int64_t* tokens, const int64_t* parent, const int32_t* q_starts, const float* u_accept,
                                  const float* u_next, const float* temperatures, float temperature, int32_t* path, int32_t* counts,
                                  int64_t* next_tokens, int32_t batch, int32_t nodes, int32_t vocabulary, int32_t max_path, void* workspace,
                                  size_t workspace_bytes, void* stream) {
    const char* who = "fsta_verify_drafts";
    if (batch < 0 || nodes < 0 || vocabulary < 1 || max_path < 1)
        return fail(FSTA_EINVAL, "%s: batch=%d nodes=%d vocabulary=%d max_path=%d", who, batch, nodes, vocabulary, max_path);
    if (!is_float(logits_dtype)) return fail(FSTA_EINVAL, "%s: logits_dtype=%d", who, logits_dtype);
    if (draft && !is_float(draft_dtype)) return fail(FSTA_EINVAL, "%s: draft_dtype=%d", who, draft_dtype);
    if (!temperatures && (temperature < 0.f || temperature != temperature || temperature == INFINITY))
        return fail(FSTA_EINVAL, "%s: temperature=%g", who, (double)temperature);
    if (logits_stride < 0 || (draft && draft_stride < 0)) return fail(FSTA_EINVAL, "%s: negative stride", who);
    if (vocabulary > INT32_MAX - 65536 || batch > INT32_MAX - 65536) return fail(FSTA_EUNSUPPORTED, "%s: batch=%d vocabulary=%d", who, batch, vocabulary);
    if (batch == 0) return FSTA_OK;
    if (!q_starts || !u_next || !path || !counts || !next_tokens || (nodes > 0 && (!logits || !tokens || !parent || !u_accept)))
        return fail(FSTA_EINVAL, "%s: null pointer", who);
    const unsigned size = logits_dtype == FSTA_F32 ? 4 : 2, draft_size = draft_dtype == FSTA_F32 ? 4 : 2;
    if (misaligned(logits, size) || (draft && misaligned(draft, draft_size)) || misaligned(tokens, 8) || misaligned(parent, 8) || misaligned(next_tokens, 8) ||
        misaligned(q_starts, 4) || misaligned(u_accept, 4) || misaligned(u_next, 4) || misaligned(temperatures, 4) || misaligned(path, 4) || misaligned(counts, 4))
        return fail(FSTA_EINVAL, "%s: a tensor is not aligned to its elements", who);
    const Plan plan = plan_of(batch, nodes, vocabulary, draft != nullptr, max_path);
    if (plan.bytes && (!workspace || misaligned(workspace, 16) || workspace_bytes < plan.bytes))
        return fail(FSTA_EINVAL, "%s: workspace of %zu bytes (%zu needed, 16-byte aligned)", who, workspace_bytes, plan.bytes);
    VerifyArgs a = {};
    a.logits = logits;
    a.draft = draft;
    a.logits_stride = logits_stride;
    a.draft_stride = draft_stride;
    a.tokens = tokens;
    a.parent = parent;
    a.q_starts = q_starts;
    a.u_accept = u_accept;
    a.u_next = u_next;
    a.temperatures = temperatures;
    a.temperature = temperature;
    a.path = path;
    a.counts = counts;
    a.next = next_tokens;
    a.batch = batch;
    a.nodes = nodes;
    a.vocabulary = vocabulary;
    a.max_path = max_path;
    a.parts_per_row = plan.parts;
    a.part_length = plan.part_length;
    hipStream_t s = static_cast<hipStream_t>(stream);
    if (logits_dtype == FSTA_F32) return launch<float>(a, draft_dtype, plan, workspace, s);
    return logits_dtype == FSTA_F16 ? launch<Half>(a, draft_dtype, plan, workspace, s) : launch<Brain>(a, draft_dtype, plan, workspace, s);
}
