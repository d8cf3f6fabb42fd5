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
#include "fsta_common.h"

namespace fsta {
namespace {

constexpr int kThreads = 1024, kWaves = kThreads / 64;
constexpr int kChildren = FSTA_VERIFY_MAX_CHILDREN;

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

// 2^d for d <= 0 (NaN and -inf: 0), to some 1e-14 of it: e^y over |y| <= ln 2 / 2 by its series, y^12 / 12! < 1e-14
__device__ __forceinline__ double power(double d) {
    d = fmax(d, -1100.0);
    const double n = rint(d), y = (d - n) * 0.69314718055994530942;
    double p = 1.0 / 39916800.0;
    p = fma(p, y, 1.0 / 3628800.0);
    p = fma(p, y, 1.0 / 362880.0);
    p = fma(p, y, 1.0 / 40320.0);
    p = fma(p, y, 1.0 / 5040.0);
    p = fma(p, y, 1.0 / 720.0);
    p = fma(p, y, 1.0 / 120.0);
    p = fma(p, y, 1.0 / 24.0);
    p = fma(p, y, 1.0 / 6.0);
    p = fma(p, y, 0.5);
    p = fma(p, y, 1.0);
    p = fma(p, y, 1.0);
    return ldexp(p, (int)n);
}

// The weights of one row: P against its largest logit, W with the draft's row
template <typename L, typename Q> struct Row {
    const L* logits;
    const Q* draft;
    double rate;                          // log2(e) / T; 0: the largest logit's place has all mass
    float top;
    int best;
    double shift;                         // s
    __device__ double probability(int x) const {
        if (rate == 0.0) return x == best ? 1.0 : 0.0;
        const float l = value(logits[x]);
        return l == top ? 1.0 : power(((double)l - (double)top) * rate);
    }
    __device__ double proposed(int x) const { return draft ? fmax((double)value(draft[x]), 0.0) : 0.0; }
    __device__ double weight(int x) const {
        const double p = probability(x);
        return draft && shift > 0.0 ? fmax(p - shift * proposed(x), 0.0) : p;
    }
};

struct Shared {
    double sum[kWaves];
    float top[kWaves];
    int best[kWaves];
    int fallen[kChildren];                // tokens that left P at this node
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

// Largest logit of a row and the first place that has it (NaN: -inf)
template <typename L> __device__ void find_top(const L* row, int n, Shared& sh, float* top, int* best) {
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    float m = -INFINITY;
    int at = INT32_MAX;
    for (int i = tid * 8; i < n; i += kThreads * 8) {
        if (i + 8 <= n) {
            Eight<L> w;
            __builtin_memcpy(&w, row + i, sizeof(w));
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const float x = value(w.v[e]);
                if (x > m) m = x, at = i + e;
            }
        } else {
            for (int e = i; e < n; ++e) {
                const float x = value(row[e]);
                if (x > m) m = x, at = e;
            }
        }
    }
#pragma unroll
    for (int d = 32; d; d >>= 1) {
        const float om = __shfl_xor(m, d);
        const int oa = __shfl_xor(at, d);
        if (om > m || (om == m && oa < at)) m = om, at = oa;
    }
    __syncthreads();
    if (lane == 0) sh.top[wave] = m, sh.best[wave] = at;
    __syncthreads();
    m = sh.top[0], at = sh.best[0];
    for (int w = 1; w < kWaves; ++w)
        if (sh.top[w] > m || (sh.top[w] == m && sh.best[w] < at)) m = sh.top[w], at = sh.best[w];
    *top = m;
    *best = m > -INFINITY ? at : -1;
}

// A wave's share of [first, first + count): its own run of whole eights
__device__ __forceinline__ void share(int first, int count, int wave, int* from, int* to) {
    const int each = ((count + kWaves - 1) / kWaves + 7) & ~7;
    *from = min(first + min(wave * (int64_t)each, (int64_t)count), (int64_t)first + count);
    *to = (int)min((int64_t)*from + each, (int64_t)first + count);
}

// Sum of a row's weights over [from, to) without the tokens that fell: one wave, the sum in all lanes
template <typename L, typename Q> __device__ double sum_run(const Row<L, Q>& row, int from, int to, const int* fallen, int n_fallen) {
    const int lane = threadIdx.x & 63;
    double sum = 0.0;
    for (int i = from + lane * 8; i < to; i += 64 * 8) {
        double w[8];
        if (i + 8 <= to) {
            Eight<L> l;
            __builtin_memcpy(&l, row.logits + i, sizeof(l));
            Eight<Q> q;
            if (row.draft) __builtin_memcpy(&q, row.draft + i, sizeof(q));
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const float x = value(l.v[e]);
                w[e] = row.rate == 0.0 ? (i + e == row.best ? 1.0 : 0.0) : x == row.top ? 1.0 : power(((double)x - (double)row.top) * row.rate);
                if (row.draft && row.shift > 0.0) w[e] = fmax(w[e] - row.shift * fmax((double)value(q.v[e]), 0.0), 0.0);
            }
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e) w[e] = i + e < to ? row.weight(i + e) : 0.0;
        }
        for (int k = 0; k < n_fallen; ++k) {
            const int x = fallen[k];
            if (x >= i && x < i + 8) {
#pragma unroll
                for (int e = 0; e < 8; ++e)
                    if (x == i + e) w[e] = 0.0;
            }
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) sum += w[e];
    }
    return sum_of(sum);
}

// Sums of the waves' shares of [first, first + count) in sh.sum; returns all of them together
template <typename L, typename Q> __device__ double sum_all(const Row<L, Q>& row, int first, int count, int n_fallen, Shared& sh) {
    int from, to;
    share(first, count, threadIdx.x >> 6, &from, &to);
    const double mine = sum_run(row, from, to, sh.fallen, n_fallen);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) sh.sum[threadIdx.x >> 6] = mine;
    __syncthreads();
    double sum = 0.0;
    for (int w = 0; w < kWaves; ++w) sum += sh.sum[w];
    return sum;
}

// The smallest token at which the running sum of the weights passes u of all of it, the last one with any weight where rounding
// (or u >= 1) lets none; -1 where there is no weight.  sh.sum holds the waves' shares of the whole row.
template <typename L, typename Q> __device__ int pick(const Row<L, Q>& row, int vocabulary, double u, double all, int n_fallen, Shared& sh) {
    if (!(all > 0.0)) return -1;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    double target = u * all;
    int first = 0, count = vocabulary;
    for (;;) {
        // the share that holds it: the first whose end passes the target, or the last with weight
        int chosen = -1, last = -1;
        double before = 0.0, at = 0.0, at_last = 0.0;
        for (int w = 0; w < kWaves && chosen < 0; ++w) {
            const double s = sh.sum[w];
            if (s > 0.0) last = w, at_last = before;
            if (before + s > target && s > 0.0) chosen = w, at = before;
            before += s;
        }
        if (chosen < 0) chosen = last, at = at_last, target = INFINITY;
        int from, to;
        share(first, count, chosen, &from, &to);
        target -= at;
        first = from;
        count = to - from;
        if (count <= kThreads * 8) break;
        sum_all(row, first, count, n_fallen, sh);
    }
    // a run of up to eight tokens a thread: threads' sums, then the tokens of the thread that holds it
    double w[8], mine = 0.0;
    const int i = first + tid * 8;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        w[e] = tid * 8 + e < count ? row.weight(i + e) : 0.0;
        for (int k = 0; k < n_fallen; ++k)
            if (sh.fallen[k] == i + e) w[e] = 0.0;
        mine += w[e];
    }
    const double up_to = sum_up_to(mine);
    __syncthreads();
    if (lane == 63) sh.sum[wave] = up_to;
    __syncthreads();
    double before = 0.0;
    for (int k = 0; k < wave; ++k) before += sh.sum[k];
    // Every thread names its first token that passes the target; the smallest counts.  None: the largest with any weight.
    int passes = INT32_MAX, last = -1;
    double run = before + (up_to - mine);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        run += w[e];
        if (w[e] > 0.0) {
            last = i + e;
            if (run > target && passes == INT32_MAX) passes = i + e;
        }
    }
#pragma unroll
    for (int d = 32; d; d >>= 1) {
        passes = min(passes, __shfl_xor(passes, d));
        last = max(last, __shfl_xor(last, d));
    }
    __syncthreads();
    if (lane == 0) sh.best[wave] = passes, sh.fallen[wave] = last;
    __syncthreads();
    for (int k = 0; k < kWaves; ++k) {
        passes = min(passes, sh.best[k]);
        last = max(last, sh.fallen[k]);
    }
    return passes != INT32_MAX ? passes : last;
}

// A workgroup per sequence walks its tree.  Every wave takes all decisions itself, from the same numbers; the workgroup shares
// the sums over the vocabulary.
template <typename L, typename Q> __global__ __launch_bounds__(kThreads) void verify_kernel(VerifyArgs a) {
    __shared__ Shared sh;
    const int tid = threadIdx.x, lane = tid & 63;
    for (int b = blockIdx.x; b < a.batch; b += gridDim.x) {
        const int start = min(max(a.q_starts[b], 0), a.nodes), nodes = max(min(a.q_starts[b + 1], a.nodes) - start, 0);
        const float tau = a.temperatures ? a.temperatures[b] : a.temperature;
        const bool greedy = !(tau > 0.f);
        const int64_t *tokens = a.tokens + start, *parent = a.parent + start;
        int32_t* path = a.path + (int64_t)b * a.max_path;
        int node = 0, count = 0, next = -1;
        while (count < nodes) {
            if (tid == 0) path[count] = node;
            ++count;
            Row<L, Q> row{static_cast<const L*>(a.logits) + (start + (int64_t)node) * a.logits_stride,
                          a.draft && !greedy ? static_cast<const Q*>(a.draft) + (start + (int64_t)node) * a.draft_stride : nullptr,
                          greedy ? 0.0 : fmax(1.4426950408889634074 / (double)tau, 1e-300), 0.f, 0, 0.0};
            find_top(row.logits, a.vocabulary, sh, &row.top, &row.best);
            if (row.best < 0) break;                                     // nothing to choose: all children fall
            double all = greedy ? 1.0 : sum_all(row, 0, a.vocabulary, 0, sh), left = 1.0;
            int fallen = 0, after = -1, asked = 0;
            for (int j0 = node + 1; j0 < nodes && after < 0 && asked < kChildren && count < a.max_path; j0 += 64) {
                uint64_t children = __ballot(j0 + lane < nodes && parent[min(j0 + lane, nodes - 1)] == node);
                for (; children && after < 0 && asked < kChildren; children &= children - 1) {
                    const int child = j0 + __ffsll((unsigned long long)children) - 1;
                    ++asked;
                    const int64_t token = tokens[child];
                    if (token < 0 || token >= a.vocabulary) continue;
                    const int x = (int)token;
                    if (greedy) {
                        if (x == row.best) after = child;
                        continue;
                    }
                    bool gone = false;
                    for (int k = lane; k < fallen; k += 64) gone |= sh.fallen[k] == x;
                    if (__ballot(gone)) continue;
                    const double u = a.u_accept[start + child], w = row.weight(x), q = row.proposed(x);
                    const bool drawn = q > 0.0 && left > 0.0;
                    if (drawn ? u * all * q < w * left : u * all < w) {
                        after = child;
                        continue;
                    }
                    if (drawn) {
                        row.shift += all / left;
                        left -= q;
                    }
                    __syncthreads();
                    if (tid == 0) sh.fallen[fallen] = x;
                    ++fallen;
                    __syncthreads();
                    all = sum_all(row, 0, a.vocabulary, fallen, sh);
                }
            }
            if (after >= 0) {
                node = after;
                continue;
            }
            if (greedy) {
                next = row.best;
                break;
            }
            const double u = a.u_next[b];
            if (!(all > 0.0)) {                // rounding left nothing: P without what fell, then P
                row.shift = 0.0;
                all = sum_all(row, 0, a.vocabulary, fallen, sh);
            }
            if (!(all > 0.0)) {
                fallen = 0;
                all = sum_all(row, 0, a.vocabulary, 0, sh);
            }
            next = pick(row, a.vocabulary, u, all, fallen, sh);
            break;
        }
        if (tid == 0) {
            a.counts[b] = count;
            a.next[b] = next;
        }
        for (int i = count + tid; i < a.max_path; i += kThreads) path[i] = -1;
        __syncthreads();
    }
}

template <typename L, typename Q> int launch(const VerifyArgs& a, hipStream_t stream) {
    hipLaunchKernelGGL((verify_kernel<L, Q>), dim3((unsigned)(a.batch < 65536 ? a.batch : 65536)), dim3(kThreads), 0, stream, a);
    FSTA_HIP_OK(hipGetLastError());
    return FSTA_OK;
}

template <typename L> int launch(const VerifyArgs& a, int32_t draft_dtype, hipStream_t stream) {
    if (!a.draft || draft_dtype == FSTA_F32) return launch<L, float>(a, stream);
    return draft_dtype == FSTA_F16 ? launch<L, Half>(a, stream) : launch<L, Brain>(a, stream);
}

bool is_float(int32_t dtype) { return dtype == FSTA_F32 || dtype == FSTA_F16 || dtype == FSTA_BF16; }

}  // namespace
}  // namespace fsta

using namespace fsta;

extern "C" size_t fsta_verify_workspace_bytes(int32_t, int32_t, int32_t, int32_t, int32_t) { return 0; }

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
    const VerifyArgs a{logits, draft, logits_stride, draft_stride, tokens, parent, q_starts, u_accept, u_next, temperatures, temperature, path, counts,
                       next_tokens, batch, nodes, vocabulary, max_path};
    hipStream_t s = static_cast<hipStream_t>(stream);
    if (logits_dtype == FSTA_F32) return launch<float>(a, draft_dtype, s);
    return logits_dtype == FSTA_F16 ? launch<Half>(a, draft_dtype, s) : launch<Brain>(a, draft_dtype, s);
}
