// Which tokens of a batch of draft trees stand against the model's logits, and the token behind each accepted path.
//
// At an accepted node the children are asked one after the other; what the model has left after each that fell is
//   W = max(P - s q, 0) over the tokens not asked yet:
// speculative sampling replaces p by norm max(p - q', 0) each time, with q' = q / r the draft's probabilities over the tokens not
// drawn before; with p = W / Z that is max(W / Z - q / r, 0) = max(P - (s + Z / r) q, 0) / Z, so s grows by Z / r and nothing else has to be
// kept per token.  Without the draft's probabilities a child is its own proposal: W loses the token, nothing else.
//
// Decisions compare sums over the vocabulary with a random number, and the next token is the place where a running sum passes
// one: in 32 bits a sum of 10^5 terms is off by more than many of them are large, so weights and sums are 64 bits here.
//
// A row is summed in parts of 2048 tokens, a wave each.  What depends on a sum comes in a later launch:
//   stats_kernel  the parts of the rows of all nodes with children (few rows: the walks behind it do not wait for sums);
//   step_kernel   one step of all sequences: each workgroup takes the decisions that the sums so far allow (all workgroups of a
//                 sequence the same ones), and its parts of the sum that is wanted next.  Only the rows on accepted paths are read;
//   walk_kernel   a workgroup per sequence goes on alone from wherever a sequence is to its end, and picks its next token.
#include "fsta_common.h"

namespace fsta {
namespace {

constexpr int kChildren = FSTA_VERIFY_MAX_CHILDREN;
constexpr int kRun = 512;                 // tokens that a wave looks at at once, eight a lane
constexpr int kPart = 4 * kRun;
constexpr int kMaxParts = 256;            // of a row: longer rows have longer parts
constexpr int kTree = 512;                // nodes of a tree that are kept in LDS
constexpr int kStepThreads = 256, kWalkThreads = 512;

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
    double shift, left;                   // s, r
    float top;                            // of the node's row, in kAgain
    int32_t pad;
};
enum { kFirst = 0, kAgain = 1, kDone = 2 };
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
    const Part* all_parts;                // of every node with children, or null
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

// Eight values of a row at any address that the type allows (a row of odd length starts anywhere)
template <typename T> struct Eight {
    T v[8];
};

// 2^d for d <= 0, exactly 1 for 0; 0 for NaN, -inf and all below -1000.  2^f = 1 + f g(f) over |f| <= 1/2, g the polynomial of degree 9
// that meets (2^f - 1) / f at the Chebyshev points: off by 6e-16 at most.  Rounding to a whole number and scaling by its power of
// two go through the bits of the sum with 1.5 2^52: sums, products and their fusions run at full rate in 64 bits, conversions and
// ldexp do not (by those the exponentials took twice as long).
__device__ __forceinline__ double power(double d) {
    constexpr double kRound = 6755399441055744.0;
    const double k = d + kRound, f = d - (k - kRound);
    double p = 7.070977866508138e-09;
    p = fma(p, f, 1.0205905413765595e-07);
    p = fma(p, f, 1.3215451633221434e-06);
    p = fma(p, f, 1.5252672924850737e-05);
    p = fma(p, f, 0.00015403530424776529);
    p = fma(p, f, 0.0013333558200794592);
    p = fma(p, f, 0.009618129107618665);
    p = fma(p, f, 0.05550410866465167);
    p = fma(p, f, 0.24022650695910075);
    p = fma(p, f, 0.6931471805599462);
    p = fma(p, f, 1.0);
    const uint64_t bits = __builtin_bit_cast(uint64_t, p);
    const uint32_t high = (uint32_t)(bits >> 32) + ((uint32_t)__builtin_bit_cast(uint64_t, k) << 20);
    p = __builtin_bit_cast(double, (uint64_t)high << 32 | (uint32_t)bits);
    return d > -1000.0 ? p : 0.0;
}
// exp((l - against) / T), the logit `against` being the largest; infinite ones share all weight
__device__ __forceinline__ double weight_of(float l, float against, double rate) {
    return against == INFINITY ? (l == INFINITY ? 1.0 : 0.0) : power(((double)l - (double)against) * rate);
}

// The weights of one row: P against its largest logit, W with the draft's row
template <typename L, typename Q> struct Row {
    const L* logits;
    const Q* draft;                       // or null
    double rate;                          // log2(e) / T; 0: the largest logit's first place has all mass
    float top;
    int best;
    double shift;                         // s
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
    uint32_t fell[kWalkThreads / 64][kPart / 32];     // a wave's part: which tokens fell
    int32_t fallen[kChildren];            // tokens that left P at this node
    double wave_sum[kWalkThreads / 64];
    int32_t best[kWalkThreads / 64], last[kWalkThreads / 64];
};

__device__ __forceinline__ double sum_of(double x) {
#pragma unroll
    for (int d = 32; d; d >>= 1) x += __shfl_xor(x, d);
    return x;
}
__device__ __forceinline__ double sum_up_to(double x) {
    const int lane = threadIdx.x & 63;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const double y = __shfl_up(x, d);
        if (lane >= d) x += y;
    }
    return x;
}
__device__ __forceinline__ float max_of(float x) {
#pragma unroll
    for (int d = 32; d; d >>= 1) x = fmaxf(x, __shfl_xor(x, d));
    return x;
}
__device__ __forceinline__ void first_best(float& top, int& best) {
#pragma unroll
    for (int d = 32; d; d >>= 1) {
        const float other = __shfl_xor(top, d);
        const int at = __shfl_xor(best, d);
        if (other > top || (other == top && at < best)) top = other, best = at;
    }
}

// Eight values from token i on, `none` at and behind token `to`
template <typename T> __device__ __forceinline__ void load_eight(const T* row, int i, int to, float none, float (&x)[8]) {
    if (i + 8 <= to) {
        Eight<T> w;
        __builtin_memcpy(&w, row + i, sizeof(w));
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = value(w.v[e]);
    } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = i + e < to ? value(row[i + e]) : none;
    }
}

// Tokens [from, to) of a row by one wave: the largest logit and the sum against it, in one pass: what is summed so far is
// scaled when a larger logit comes.  All lanes have the result.
template <typename L> __device__ Part first_sum(const L* row, double rate, int from, int to) {
    constexpr int kAtOnce = kPart / kRun;
    const int lane = threadIdx.x & 63;
    float top = -INFINITY;
    int best = INT32_MAX;
    double sum = 0.0;
    for (int i0 = from; i0 < to; i0 += kPart) {
        float x[kAtOnce][8];
#pragma unroll
        for (int r = 0; r < kAtOnce; ++r) load_eight(row, i0 + r * kRun + lane * 8, to, -INFINITY, x[r]);
        float m = -INFINITY;              // (fmaxf passes over a NaN)
#pragma unroll
        for (int r = 0; r < kAtOnce; ++r)
#pragma unroll
            for (int e = 0; e < 8; ++e) m = fmaxf(m, x[r][e]);
        if (rate == 0.0) {
            if (m > top) {
                top = m;
#pragma unroll
                for (int r = kAtOnce - 1; r >= 0; --r)
#pragma unroll
                    for (int e = 7; e >= 0; --e)
                        if (x[r][e] == m) best = i0 + r * kRun + lane * 8 + e;
            }
            continue;
        }
        m = max_of(m);
        if (m > top) {
            if (sum > 0.0) sum *= weight_of(top, m, rate);
            top = m;
        }
        if (top == INFINITY) {
#pragma unroll
            for (int r = 0; r < kAtOnce; ++r)
#pragma unroll
                for (int e = 0; e < 8; ++e) sum += x[r][e] == INFINITY ? 1.0 : 0.0;
        } else if (top > -INFINITY) {
            const double against = top;
#pragma unroll
            for (int r = 0; r < kAtOnce; ++r) {
#pragma unroll
                for (int e = 0; e < 8; ++e) sum += power(((double)x[r][e] - against) * rate);
                __builtin_amdgcn_sched_barrier(0);               // (eight at a time: all at once they need twice the registers)
            }
        }
    }
    if (rate == 0.0) {
        first_best(top, best);
        return Part{1.0, top, best};
    }
    return Part{sum_of(sum), top, 0};
}

// Sum of a row's weights over [from, to) without the tokens that fell, by one wave; `fell`: room for kPart bits
template <typename L, typename Q>
__device__ double sum_again(const Row<L, Q>& row, int from, int to, const int32_t* fallen, int n_fallen, uint32_t* fell) {
    const int lane = threadIdx.x & 63;
    const bool drafted = row.draft && row.shift > 0.0;
    double sum = 0.0;
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
        const auto add = [&](const float (&x)[8], const float (&q)[8], uint32_t out) {
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                double w = weight_of(x[e], row.top, row.rate);
                if (drafted) w = fmax(w - row.shift * fmax((double)q[e], 0.0), 0.0);
                sum += out >> e & 1 ? 0.0 : w;
            }
        };
        const auto left_out = [&](int i) { return any ? fell[(i - i0) >> 5] >> ((i - i0) & 31) : 0u; };
        for (int i = i0 + lane * 8; i < min(i0 + kPart, to); i += 2 * kRun) {
            float x[8], y[8], q[8] = {}, p[8] = {};
            load_eight(row.logits, i, to, -INFINITY, x);
            load_eight(row.logits, min(i + kRun, to), to, -INFINITY, y);
            if (drafted) {
                load_eight(row.draft, i, to, 0.f, q);
                load_eight(row.draft, min(i + kRun, to), to, 0.f, p);
            }
            add(x, q, left_out(i));
            __builtin_amdgcn_sched_barrier(0);
            add(y, p, left_out(i + kRun));
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    }
    return sum_of(sum);
}

// One sequence's walk, by a workgroup.  Every wave takes all decisions itself, from the same numbers.
template <typename L, typename Q, int THREADS> struct Walk {
    static constexpr int kWaves = THREADS / 64;
    const VerifyArgs& a;
    Shared& sh;
    int b, start, nodes;
    bool greedy;
    Row<L, Q> row;
    int node, count, child, asked;        // children below `child` have fallen, `asked` of them
    int summed, fallen;                   // children below `summed` were left out of the sum; entries of sh.fallen
    int held, where;                      // the last sum, as in State
    double all, whole, left;              // Z, Z when the sum was taken, r
    // the strip of 64 nodes whose children are asked next: a child per lane, and which lanes
    int strip, token;
    uint64_t kids;
    float logit;
    double q, u;

    __device__ Walk(const VerifyArgs& args, Shared& shared, int sequence) : a(args), sh(shared), b(sequence) {
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
        for (int j = threadIdx.x; j < min(nodes, kTree); j += THREADS) {
            sh.parent[j] = parent_in_memory(j);
            sh.token[j] = token_in_memory(j);
        }
        __syncthreads();
    }
    __device__ int parent_in_memory(int j) const {
        const int64_t p = a.parent[start + j];
        return p >= 0 && p < j ? (int)p : -1;
    }
    __device__ int token_in_memory(int j) const {
        const int64_t x = a.tokens[start + j];
        return x >= 0 && x < a.vocabulary ? (int)x : -1;
    }
    __device__ bool is_child(int j) const { return j < nodes && (j < kTree ? sh.parent[j] : parent_in_memory(j)) == node; }
    __device__ int token_of(int j) const { return j < kTree ? sh.token[j] : token_in_memory(j); }

    // To the next strip with children of the node, from node `from` on: what they are asked with
    __device__ void look(int from) {
        const int lane = threadIdx.x & 63;
        kids = 0;
        for (strip = from; strip < nodes && !kids; strip += kids ? 0 : 64) kids = __ballot(is_child(strip + lane));
        const bool mine = kids >> lane & 1;
        token = mine ? token_of(strip + lane) : -1;
        logit = token >= 0 ? value(row.logits[token]) : -INFINITY;
        q = token >= 0 ? row.proposed(token) : 0.0;
        u = mine ? (double)a.u_accept[start + strip + lane] : 0.0;
    }
    __device__ void stand_at(int at, int how_many) {
        node = at;
        count = how_many;
        child = summed = at + 1;
        fallen = asked = 0;
        left = 1.0;
        row.logits = static_cast<const L*>(a.logits) + (start + (int64_t)node) * a.logits_stride;
        row.draft = a.draft && !greedy ? static_cast<const Q*>(a.draft) + (start + (int64_t)node) * a.draft_stride : nullptr;
        row.shift = 0.0;
        row.top = -INFINITY;
        row.best = -1;
        look(at + 1);
    }
    __device__ void resume(const State& s) {
        stand_at(s.node, s.count);
        if (s.phase == kFirst) return;
        child = s.child;
        asked = s.asked;
        left = s.left;
        row.shift = s.shift;
        row.top = s.top;
        look(child);
    }
    __device__ void part_range(int p, int* from, int* to) const {
        *from = (int)min((int64_t)p * a.part_length, (int64_t)a.vocabulary);
        *to = (int)min((int64_t)*from + a.part_length, (int64_t)a.vocabulary);
    }

    // The parts of the first sum of the row: its largest logit, Z.  (Every wave writes the same to sh.sum.)
    __device__ void take_first(const Part* parts) {
        const int lane = threadIdx.x & 63;
        float top = -INFINITY;
        int best = INT32_MAX;
        for (int p = lane; p < a.parts_per_row; p += 64) {
            const Part part = parts[p];
            if (part.top > top) top = part.top, best = part.best;
        }
        first_best(top, best);
        row.top = top;
        row.best = top > -INFINITY ? best : -1;
        double sum = 0.0;
        if (!greedy) {
            for (int p = lane; p < a.parts_per_row; p += 64) {
                const Part part = parts[p];
                const double s = part.sum > 0.0 ? part.sum * weight_of(part.top, top, row.rate) : 0.0;
                sum += s;
                sh.sum[p] = s;
            }
        }
        whole = all = sum_of(sum);
        summed = child;
        held = kFirst;
    }
    // .. of a sum of W
    __device__ void take_again(const Part* parts) {
        double sum = 0.0;
        for (int p = threadIdx.x & 63; p < a.parts_per_row; p += 64) {
            const double s = parts[p].sum;
            sum += s;
            sh.sum[p] = s;
        }
        whole = all = sum_of(sum);
        summed = child;
        held = kAgain;
    }

    // Whether a child before child j has its token x
    __device__ bool fell_before(int j, int x) const {
        for (int i0 = node + 1; i0 < j; i0 += 64) {
            const int i = i0 + (threadIdx.x & 63);
            if (__ballot(i < j && is_child(i) && token_of(i) == x)) return true;
        }
        return false;
    }

    // Asks children until one stands (kFirst: `node` is that one now), a sum of W is wanted (kAgain) or there are no more (kDone)
    __device__ int ask() {
        if (row.top == -INFINITY) return kDone;                  // nothing to choose: all children fall
        while (kids && count < a.max_path && asked < kChildren) {
            const double w = row.weight(logit, q);
            for (; kids && asked < kChildren; kids &= kids - 1) {
                const int l = __ffsll((unsigned long long)kids) - 1, x = __shfl(token, l), j = strip + l;
                ++asked;
                child = j + 1;
                if (x < 0) continue;
                if (greedy) {
                    if (x != row.best) continue;
                    stand_at(j, count + 1);
                    return kFirst;
                }
                if (fell_before(j, x)) continue;
                const double wx = __shfl(w, l), qx = __shfl(q, l), ux = __shfl(u, l);
                const bool drawn = qx > 0.0 && left > 0.0;
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

    // The tokens that fell, in sh.fallen; behind those that the sum leaves out (returned: how many) each comes once
    __device__ int collect() {
        const int lane = threadIdx.x & 63;
        __syncthreads();
        fallen = 0;
        for (int i0 = node + 1; i0 < summed; i0 += 64) {
            const int i = i0 + lane, x = i < summed && is_child(i) ? token_of(i) : -1;
            const uint64_t those = __ballot(x >= 0);
            if (x >= 0 && threadIdx.x < 64) sh.fallen[fallen + __popcll(those & ((1ull << lane) - 1))] = x;
            fallen += __popcll(those);
        }
        const int before = fallen;
        for (int i0 = summed; i0 < child; i0 += 64) {
            const int i = i0 + lane, mine = i < child && is_child(i) ? token_of(i) : -1;
            for (uint64_t those = __ballot(mine >= 0); those; those &= those - 1) {
                const int l = __ffsll((unsigned long long)those) - 1, x = __shfl(mine, l);
                if (fell_before(i0 + l, x)) continue;
                if (threadIdx.x == 0) sh.fallen[fallen] = x;
                ++fallen;
            }
        }
        __syncthreads();
        return before;
    }

    // Sums over the whole row by this workgroup alone, a part a wave: into sh.part
    __device__ void sum_alone(bool first) {
        const int wave = threadIdx.x >> 6;
        __syncthreads();
        for (int p = wave; p < a.parts_per_row; p += kWaves) {
            int from, to;
            part_range(p, &from, &to);
            const Part part = first ? first_sum(row.logits, row.rate, from, to) : Part{sum_again(row, from, to, sh.fallen, fallen, sh.fell[wave]), row.top, 0};
            if ((threadIdx.x & 63) == 0) sh.part[p] = part;
        }
        __syncthreads();
    }

    // The smallest token at which the running sum of the weights passes u of all of it, the last one with any weight where rounding
    // (or u >= 1) lets none; -1 where there is no weight
    __device__ int pick(double u) {
        const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
        __syncthreads();                  // sh.sum
        if (child > summed) {
            // a part loses the terms that fell since its sum was taken; where little is left of it, its sum is taken again
            const int old = collect();
            for (int p = wave; p < a.parts_per_row; p += kWaves) {
                int from, to;
                part_range(p, &from, &to);
                double lost = 0.0;
                for (int k = old + lane; k < fallen; k += 64) {
                    const int x = sh.fallen[k];
                    if (x >= from && x < to) lost += row.weight(value(row.logits[x]), row.proposed(x));
                }
                lost = sum_of(lost);
                double s = sh.sum[p];
                if (lost > 0.0) s = s - lost > s * 0x1p-10 ? s - lost : sum_again(row, from, to, sh.fallen, fallen, sh.fell[wave]);
                if (lane == 0) sh.sum[p] = s;
            }
            __syncthreads();
        } else {
            collect();
        }
        // the part that holds it: the first whose end passes the target, or the last with weight
        const auto total = [&] {
            double sum = 0.0;
            for (int p = lane; p < a.parts_per_row; p += 64) sum += sh.sum[p];
            return sum_of(sum);
        };
        double sum = total();
        for (int resort = 0; !(sum > 0.0); ++resort) {           // rounding left nothing: P without what fell, then P
            if (resort == 2) return -1;
            row.shift = 0.0;
            if (resort == 1) fallen = 0;
            sum_alone(false);
            for (int p = tid; p < a.parts_per_row; p += THREADS) sh.sum[p] = sh.part[p].sum;
            __syncthreads();
            sum = total();
        }
        double target = u * sum;
        int chosen = -1, last = -1;
        double before = 0.0, at_chosen = 0.0;
        for (int p0 = 0; p0 < a.parts_per_row && chosen < 0; p0 += 64) {
            const double s = p0 + lane < a.parts_per_row ? sh.sum[p0 + lane] : 0.0;
            const double up_to = sum_up_to(s);
            const uint64_t weighs = __ballot(s > 0.0), passes = __ballot(s > 0.0 && before + up_to > target);
            if (weighs) last = p0 + 63 - __builtin_clzll(weighs);
            if (passes) {
                const int l = __ffsll((unsigned long long)passes) - 1;
                chosen = p0 + l;
                at_chosen = before + (__shfl(up_to, l) - __shfl(s, l));
            }
            before += __shfl(up_to, 63);
        }
        if (chosen < 0) chosen = last, at_chosen = 0.0, target = INFINITY;
        target -= at_chosen;
        int from, to;
        part_range(chosen, &from, &to);
        // the same among the waves' shares of it, until a thread has eight tokens
        while (to - from > THREADS * 8) {
            const int each = ((to - from + kWaves - 1) / kWaves + 7) & ~7;
            int lo = (int)min((int64_t)from + (int64_t)wave * each, (int64_t)to);
            const double mine = sum_again(row, lo, min(lo + each, to), sh.fallen, fallen, sh.fell[wave]);
            __syncthreads();
            if (lane == 0) sh.wave_sum[wave] = mine;
            __syncthreads();
            before = 0.0;
            chosen = last = -1;
            for (int w = 0; w < kWaves && chosen < 0; ++w) {
                const double s = sh.wave_sum[w];
                if (s > 0.0) {
                    last = w;
                    if (before + s > target) chosen = w, at_chosen = before;
                }
                before += s;
            }
            if (chosen < 0) {
                if (last < 0) return -1;
                chosen = last;
                at_chosen = 0.0;
                target = INFINITY;
            }
            target -= at_chosen;
            from = (int)min((int64_t)from + (int64_t)chosen * each, (int64_t)to);
            to = min(from + each, to);
        }
        double w[8], mine = 0.0;
        const int i = min(from + tid * 8, to);
        float x[8], qs[8];
        load_eight(row.logits, i, to, -INFINITY, x);
        const bool drafted = row.draft && row.shift > 0.0;
        if (drafted) load_eight(row.draft, i, to, 0.f, qs);
#pragma unroll
        for (int e = 0; e < 8; ++e) w[e] = i + e < to ? row.weight(x[e], drafted ? fmax((double)qs[e], 0.0) : 0.0) : 0.0;
        for (int k = 0; k < fallen; ++k) {
            const int f = sh.fallen[k] - i;
#pragma unroll
            for (int e = 0; e < 8; ++e)
                if (f == e) w[e] = 0.0;
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) mine += w[e];
        const double up_to = sum_up_to(mine);
        __syncthreads();
        if (lane == 63) sh.wave_sum[wave] = up_to;
        __syncthreads();
        double run = up_to - mine;
        for (int k = 0; k < wave; ++k) run += sh.wave_sum[k];
        // Every thread names its first token that passes the target; the smallest counts.  None: the largest with any weight.
        int passes = INT32_MAX, weighs = -1;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            run += w[e];
            if (w[e] > 0.0) {
                weighs = i + e;
                if (run > target && passes == INT32_MAX) passes = i + e;
            }
        }
#pragma unroll
        for (int d = 32; d; d >>= 1) {
            passes = min(passes, __shfl_xor(passes, d));
            weighs = max(weighs, __shfl_xor(weighs, d));
        }
        if (lane == 0) sh.best[wave] = passes, sh.last[wave] = weighs;
        __syncthreads();
        for (int k = 0; k < kWaves; ++k) {
            passes = min(passes, sh.best[k]);
            weighs = max(weighs, sh.last[k]);
        }
        return passes != INT32_MAX ? passes : weighs;
    }

    // The end of a sequence's walk
    __device__ void answer() {
        int next = -1;
        if (nodes == 0) count = 0;
        else if (row.top > -INFINITY) next = greedy ? row.best : pick(a.u_next[b]);
        if (threadIdx.x == 0) {
            a.counts[b] = count;
            a.next[b] = next;
        }
        for (int i = count + threadIdx.x; i < a.max_path; i += THREADS) a.path[(int64_t)b * a.max_path + i] = -1;
    }
    __device__ void note() const {
        if (threadIdx.x == 0) a.path[(int64_t)b * a.max_path + count - 1] = node;
    }

    __device__ const Part* parts_of_node() const { return a.all_parts + (start + (int64_t)node) * a.parts_per_row; }
    __device__ const Part* parts_of_step(int turn) const { return a.parts[turn] + (int64_t)b * a.parts_per_row; }
    __device__ void take(int what, const Part* parts) {
        if (what == kFirst) take_first(parts);
        else take_again(parts);
    }
    // Takes decisions for as long as the sums are there; `parts`: the one that the state waits for, or null
    __device__ int go_on(int phase, const Part* parts, bool noting) {
        for (;;) {
            if (phase == kFirst && !parts && a.all_parts && kids) {
                parts = parts_of_node();
                where = kOfNode;
            }
            if (!parts) return phase;
            take(phase, parts);
            parts = nullptr;
            phase = ask();
            if (phase == kFirst && noting) note();
            if (phase != kFirst) return phase;
        }
    }
};

// blockIdx.x: parts in fours, .y: node
template <typename L> __global__ __launch_bounds__(kStepThreads, 4) void stats_kernel(VerifyArgs a) {
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    for (int64_t t = blockIdx.y; t < a.nodes; t += gridDim.y) {
        // the node's sequence: how many start at or before it
        int b = -1;
        for (int c = 0; c < a.batch; c += 64) b += __popcll(__ballot(c + lane < a.batch && a.q_starts[c + lane] <= t));
        if (b < 0) continue;
        const int start = max(a.q_starts[b], 0), end = min(a.q_starts[b + 1], a.nodes), node = (int)(t - start);
        uint64_t any = 0;
        for (int64_t j = t + 1; j < end && !any; j += 64) any = __ballot(j + lane < end && a.parent[j + lane] == node);
        if (!any) continue;
        const float tau = a.temperatures ? a.temperatures[b] : a.temperature;
        const double rate = tau > 0.f ? fmax(1.4426950408889634074 / (double)tau, 1e-300) : 0.0;
        const int p = blockIdx.x * (kStepThreads / 64) + wave;
        if (p >= a.parts_per_row) continue;
        const int from = (int)min((int64_t)p * a.part_length, (int64_t)a.vocabulary), to = (int)min((int64_t)from + a.part_length, (int64_t)a.vocabulary);
        const Part part = first_sum(static_cast<const L*>(a.logits) + t * a.logits_stride, rate, from, to);
        if (lane == 0) a.parts_out[t * a.parts_per_row + p] = part;
    }
}

// blockIdx.x: parts in fours, .y: sequence
template <typename L, typename Q> __global__ __launch_bounds__(kStepThreads, 3) void step_kernel(VerifyArgs a) {
    __shared__ Shared sh;
    const int wave = threadIdx.x >> 6;
    const bool speaks = blockIdx.x == 0;
    for (int b = blockIdx.y; b < a.batch; b += gridDim.y) {
        State s{0, 1, 1, 0, 1, kFirst, kFirst, 0, 0.0, 1.0, 0.f, 0};
        if (!a.fresh) s = a.states[a.turn ^ 1][b];
        if (s.phase == kDone) {
            if (speaks && threadIdx.x == 0) a.states[a.turn][b] = s;
            continue;
        }
        __syncthreads();
        Walk<L, Q, kStepThreads> w(a, sh, b);
        if (w.nodes == 0) {
            s.phase = kDone;
        } else {
            w.resume(s);
            w.where = a.turn ^ 1;
            if (a.fresh && speaks) w.note();
            s.phase = w.go_on(s.phase, a.fresh ? nullptr : w.parts_of_step(a.turn ^ 1), speaks);
        }
        if (speaks && threadIdx.x == 0)
            a.states[a.turn][b] = State{w.node, w.count, w.child, w.asked, w.summed, s.phase, w.held, w.where, w.row.shift, w.left, w.row.top, 0};
        if (s.phase == kDone) continue;
        if (s.phase == kAgain) {
            w.summed = w.child;
            w.collect();
        }
        const int p = blockIdx.x * (kStepThreads / 64) + wave;
        if (p >= a.parts_per_row) continue;
        int from, to;
        w.part_range(p, &from, &to);
        const Part part = s.phase == kFirst ? first_sum(w.row.logits, w.row.rate, from, to)
                                            : Part{sum_again(w.row, from, to, sh.fallen, w.fallen, sh.fell[wave]), w.row.top, 0};
        if ((threadIdx.x & 63) == 0) a.parts[a.turn][(int64_t)b * a.parts_per_row + p] = part;
    }
}

template <typename L, typename Q> __global__ __launch_bounds__(kWalkThreads, 2) void walk_kernel(VerifyArgs a) {
    __shared__ Shared sh;
    for (int b = blockIdx.x; b < a.batch; b += gridDim.x) {
        __syncthreads();
        Walk<L, Q, kWalkThreads> w(a, sh, b);
        if (w.nodes > 0) {
            State s{0, 1, 1, 0, 1, kFirst, kFirst, 0, 0.0, 1.0, 0.f, 0};
            if (!a.fresh) s = a.states[a.turn][b];
            w.resume(s);
            if (s.phase == kDone) {
                w.take(s.held, s.where == kOfNode ? w.parts_of_node() : w.parts_of_step(s.where));
                w.summed = s.summed;
            } else {
                if (a.fresh) w.note();
                const Part* parts = a.fresh ? nullptr : w.parts_of_step(a.turn);
                while ((s.phase = w.go_on(s.phase, parts, true)) != kDone) {
                    if (s.phase == kAgain) {
                        w.summed = w.child;
                        w.collect();
                    }
                    w.sum_alone(s.phase == kFirst);
                    parts = sh.part;
                }
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

constexpr int kMostSteps = 10;
constexpr double kAllBytes = 128e6;

Plan plan_of(int64_t batch, int64_t nodes, int64_t vocabulary, int size, bool draft, int32_t max_path) {
    Plan p;
    p.part_length = (int32_t)((vocabulary + (int64_t)kPart * kMaxParts - 1) / ((int64_t)kPart * kMaxParts) * kPart);
    p.parts = (int32_t)((vocabulary + p.part_length - 1) / p.part_length);
    p.all = (double)nodes * vocabulary * size <= kAllBytes;
    p.steps = max_path + (draft ? 3 : 0) < kMostSteps ? max_path + (draft ? 3 : 0) : kMostSteps;
    if (p.all) p.steps = draft ? 4 : 1;
    p.bytes = (p.all ? rounded(sizeof(Part) * (size_t)(nodes * p.parts)) : 0) + 2 * (rounded(sizeof(Part) * (size_t)(batch * p.parts)) + rounded(sizeof(State) * (size_t)batch));
    return p;
}

template <typename L, typename Q> int launch(VerifyArgs a, const Plan& plan, void* workspace, hipStream_t stream) {
    uint8_t* work = static_cast<uint8_t*>(workspace);
    const unsigned groups = (unsigned)((a.parts_per_row + kStepThreads / 64 - 1) / (kStepThreads / 64));
    if (plan.all && a.nodes > 0) {
        a.parts_out = reinterpret_cast<Part*>(work);
        a.all_parts = a.parts_out;
        work += rounded(sizeof(Part) * (size_t)a.nodes * a.parts_per_row);
        hipLaunchKernelGGL((stats_kernel<L>), dim3(groups, (unsigned)(a.nodes < 65535 ? a.nodes : 65535)), dim3(kStepThreads), 0, stream, a);
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
        hipLaunchKernelGGL((step_kernel<L, Q>), dim3(groups, (unsigned)(a.batch < 65535 ? a.batch : 65535)), dim3(kStepThreads), 0, stream, a);
        a.fresh = 0;
    }
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

extern "C" size_t fsta_verify_workspace_bytes(int32_t batch, int32_t nodes, int32_t vocabulary, int32_t logits_dtype, int32_t draft) {
    if (batch <= 0 || nodes < 0 || vocabulary < 1) return 0;
    return plan_of(batch, nodes, vocabulary, logits_dtype == FSTA_F32 ? 4 : 2, draft != 0, 1).bytes;
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
    if (vocabulary > INT32_MAX - 65536) return fail(FSTA_EUNSUPPORTED, "%s: vocabulary=%d", who, vocabulary);
    if (batch == 0) return FSTA_OK;
    if (!q_starts || !u_next || !path || !counts || !next_tokens || (nodes > 0 && (!logits || !tokens || !parent || !u_accept)))
        return fail(FSTA_EINVAL, "%s: null pointer", who);
    const unsigned size = logits_dtype == FSTA_F32 ? 4 : 2, draft_size = draft_dtype == FSTA_F32 ? 4 : 2;
    if (misaligned(logits, size) || (draft && misaligned(draft, draft_size)) || misaligned(tokens, 8) || misaligned(parent, 8) || misaligned(next_tokens, 8) ||
        misaligned(q_starts, 4) || misaligned(u_accept, 4) || misaligned(u_next, 4) || misaligned(temperatures, 4) || misaligned(path, 4) || misaligned(counts, 4))
        return fail(FSTA_EINVAL, "%s: a tensor is not aligned to its elements", who);
    const Plan plan = plan_of(batch, nodes, vocabulary, (int)size, draft != nullptr, max_path);
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
