// The paged KV cache: rows of new tokens into their pages (16-bit as they are, or as e4m3 bytes with a power of two per row),
// pages back to dense tensors, and the masks of draft trees in the form the attention over pages reads.
//
// Memory-bound, element-wise.  An 8-bit row x of head_dim values is kept as bytes b and one exponent byte E: x ~ b 2^(E - 127)
// with the smallest power under which max |x| <= 448.  A power of two and not max |x| / 448: e4m3 is a floating-point format,
// so where in a binade its largest value falls costs nothing but the last subnormal bit, and b 2^(E - 127) is exact in bfloat16, to
// which the conversion instruction itself widens it (it takes a scale).  float16 holds every b, but not every b 2^(E - 127): above
// 65504 it is infinite, below 2^-14 it loses bits (rows read as float16; the attention keeps the powers apart).
#include "fsta_paged.h"

namespace fsta {
namespace {

typedef unsigned int u32x4 __attribute__((ext_vector_type(4)));
typedef unsigned int u32x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef unsigned short u16x2 __attribute__((ext_vector_type(2)));

constexpr int kThreads = 256;
constexpr int kTreeRows = 64;             // rows of a tree's masks per workgroup
constexpr int kTreeNodes = 8192;          // nodes of a tree in LDS at most (64 KB)
constexpr int kUnits = 4;                 // 16-byte pieces of 16-bit rows per thread

struct RowArgs {
    PagedBatch batch;
    const void* src[2];                   // k, v of the new tokens (write)
    int64_t token_stride[2], head_stride[2];
    void* pool[2];                        // cache k, v
    uint8_t* exponent[2];                 // 8-bit rows only
    void* out[2];                         // dense k, v (read)
    int32_t max_len;
};

template <bool BF16> __device__ __forceinline__ float half_of(uint32_t word, int hi) {
    if constexpr (BF16) return __builtin_bit_cast(float, hi ? word & 0xffff0000u : word << 16);
    else return (float)__builtin_bit_cast(_Float16, (unsigned short)(hi ? word >> 16 : word & 0xffffu));
}

// Largest finite magnitude of a lane's 8 values (infinities and NaNs have no say in the scale)
template <bool BF16> __device__ __forceinline__ float finite_max(u32x4 w) {
    float mx = 0.f;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        const uint32_t word = w[e / 2];
        const float a = fabsf(half_of<BF16>(word, e & 1));
        mx = fmaxf(mx, a < INFINITY ? a : 0.f);
    }
    return mx;
}

// Largest magnitude of a lane's 8 values as its 16 bits without the sign (they order like the values; infinities and NaN on top)
__device__ __forceinline__ uint32_t top_bits(u32x4 w) {
    u16x2 m = {0, 0};
#pragma unroll
    for (int e = 0; e < 4; ++e) m = __builtin_elementwise_max(m, __builtin_bit_cast(u16x2, w[e] & 0x7fff7fffu));
    return max((uint32_t)m[0], (uint32_t)m[1]);
}
// Largest over the LANES (8 or 16) lanes of a row: neighbours, pairs, and the row's quads and halves mirrored
template <int LANES> __device__ __forceinline__ uint32_t row_max(uint32_t x) {
    x = max(x, (uint32_t)__builtin_amdgcn_mov_dpp((int)x, 0xb1, 0xf, 0xf, true));
    x = max(x, (uint32_t)__builtin_amdgcn_mov_dpp((int)x, 0x4e, 0xf, 0xf, true));
    x = max(x, (uint32_t)__builtin_amdgcn_mov_dpp((int)x, 0x141, 0xf, 0xf, true));
    if constexpr (LANES == 16) x = max(x, (uint32_t)__builtin_amdgcn_mov_dpp((int)x, 0x140, 0xf, 0xf, true));
    return x;
}

// E of a row: mantissa and exponent of max |x| = m 2^(x), m in [1, 2): 448 = 1.75 * 2^8
__device__ __forceinline__ int row_exponent(float amax) {
    if (!(amax > 0.f)) return 127;
    const uint32_t bits = __builtin_bit_cast(uint32_t, amax);
    const int e = (int)(bits >> 23) - 127 - 8 + ((bits & 0x7fffffu) > 0x600000u ? 1 : 0);   // (denormal: far below the clamp)
    return 127 + min(max(e, -110), 120);
}

// 8 values times 2^-(E - 127), rounded to e4m3 (nearest even; at most 448 by the choice of E); FINITE: all of them are; infinities
// and NaN: NaN
template <bool BF16, bool FINITE> __device__ __forceinline__ u32x2 to_bytes(u32x4 w, int E) {
    const float inv = __builtin_bit_cast(float, (uint32_t)(254 - E) << 23);
    u32x2 out;
#pragma unroll
    for (int half = 0; half < 2; ++half) {
        float x[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const float y = half_of<BF16>(w[2 * half + e / 2], e & 1) * inv;
            x[e] = FINITE || fabsf(y) <= 448.f ? y : __builtin_nanf("");
        }
        int pk = __builtin_amdgcn_cvt_pk_fp8_f32(x[0], x[1], 0, false);
        pk = __builtin_amdgcn_cvt_pk_fp8_f32(x[2], x[3], pk, true);
        out[half] = (uint32_t)pk;
    }
    return out;
}

// 8 bytes times 2^(E - 127) in the 16-bit type
template <bool BF16> __device__ __forceinline__ u32x4 to_halves(u32x2 b, int E) {
    const float scale = __builtin_bit_cast(float, (uint32_t)E << 23);
    u32x4 out;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const uint32_t word = b[i];
        if constexpr (BF16) {
            out[2 * i] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(word, scale, false));
            out[2 * i + 1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(word, scale, true));
        } else {
            out[2 * i] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(word, scale, false));
            out[2 * i + 1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(word, scale, true));
        }
    }
    return out;
}

// Rows [token][k, v][head]; a workgroup takes a run of them, D / 8 lanes a row.  The values are requested first; meanwhile
// each wave finds the places of some of the run's tokens (sequence: how many sequences start at or before the token).
// Bound by the copy: 8192 tokens of 16 heads of 128, 16 bits, 134 MB in 26.7 us, 5.0 TB/s, as a large copy on this card; 61 tokens 3.8
// us, a launch and two round trips.  Four rows' loads a thread are on their way before a place is known; the source is read past the
// caches, since nothing reads it again, and the rows written stay in them for the attention that follows.  8-bit rows: 80 MB in 20.5
// us; the largest magnitude is found among the 16-bit patterns, packed, and between lanes without LDS (one value at a time through
// float and LDS: 23 us); a wave that meets an infinity or a NaN looks again, value by value.
template <bool BF16, int D, bool FP8>
__global__ __launch_bounds__(kThreads) void paged_write_kernel(RowArgs a) {
    constexpr int kLanes = D / 8, kRowsPerPass = kThreads / kLanes, kRows = kRowsPerPass * kUnits;
    __shared__ int64_t place[kRows / 2 + 2];       // row of the token's key in a pool of one head, or -1; a token has two rows at least
    const PagedBatch& p = a.batch;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int sub = tid % kLanes;
    const uint32_t rows_per_token = 2u * (uint32_t)p.kv_heads;
    const uint64_t rows = (uint64_t)p.tokens * rows_per_token;
    const uint64_t row0 = (uint64_t)blockIdx.x * kRows;
    const int first_token = (int)(row0 / rows_per_token);
    const int last_token = (int)min((row0 + kRows - 1) / rows_per_token, (uint64_t)p.tokens - 1);

    u32x4 w[kUnits];
    int token[kUnits], tensor[kUnits], head[kUnits];
#pragma unroll
    for (int i = 0; i < kUnits; ++i) {
        const uint64_t row = row0 + i * kRowsPerPass + tid / kLanes;
        token[i] = -1;
        if (row < rows) {
            const uint32_t in_run = (uint32_t)(row - (uint64_t)first_token * rows_per_token);
            token[i] = first_token + (int)(in_run / rows_per_token);
            const uint32_t r = in_run % rows_per_token;
            tensor[i] = r >= (uint32_t)p.kv_heads;
            head[i] = (int)(r - (tensor[i] ? p.kv_heads : 0));
            const int64_t at = tensor[i] ? token[i] * a.token_stride[1] + head[i] * a.head_stride[1]
                                         : token[i] * a.token_stride[0] + head[i] * a.head_stride[0];
            const uint16_t* src = static_cast<const uint16_t*>(tensor[i] ? a.src[1] : a.src[0]) + at;
            w[i] = __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(src) + sub);
        }
    }
    for (int t = first_token + wave; t <= last_token; t += kThreads / 64) {
        int b = -1;
        for (int c = 0; c < p.batch; c += 64)
            b += __popcll(__ballot(c + lane < p.batch && p.q_starts[c + lane] <= t));
        int64_t at = -1;
        if (b >= 0) {
            const SeqLens s = seq_lens(p, b);
            const int i = t - s.start, pos = s.keys - s.fresh + i;
            if (i < s.fresh && pos >= 0 && pos < s.keys) {
                const int page = p.page_table[(size_t)b * p.width + (pos >> p.page_shift)];
                if (page >= 0 && page < p.num_pages)
                    at = (((int64_t)page * p.kv_heads) << p.page_shift) + (pos & ((1 << p.page_shift) - 1));
            }
        }
        if (lane == 0) place[t - first_token] = at;
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kUnits; ++i) {
        int E = 0;
        bool all_finite = true;
        if constexpr (FP8) {               // (all lanes take part; those without a row look at what is in the register)
            const uint32_t top = row_max<kLanes>(top_bits(w[i]));
            float amax = half_of<BF16>(top, 0);
            all_finite = __ballot(top >= (BF16 ? 0x7f80u : 0x7c00u)) == 0ull;
            if (!all_finite) {
                amax = finite_max<BF16>(w[i]);
#pragma unroll
                for (int d = 1; d < kLanes; d <<= 1) amax = fmaxf(amax, __shfl_xor(amax, d));
            }
            E = row_exponent(amax);
        }
        const int64_t at = token[i] >= 0 ? place[token[i] - first_token] : -1;
        if (at < 0) continue;
        const int64_t row = at + ((int64_t)head[i] << p.page_shift);
        if constexpr (FP8) {
            reinterpret_cast<u32x2*>(static_cast<uint8_t*>(tensor[i] ? a.pool[1] : a.pool[0]) + row * D)[sub] = all_finite ? to_bytes<BF16, true>(w[i], E) : to_bytes<BF16, false>(w[i], E);
            if (sub == 0) (tensor[i] ? a.exponent[1] : a.exponent[0])[row] = (uint8_t)E;
        } else {
            reinterpret_cast<u32x4*>(static_cast<uint16_t*>(tensor[i] ? a.pool[1] : a.pool[0]) + row * D)[sub] = w[i];
        }
    }
}

// Output rows [tensor][sequence][head][position]; blockIdx.x: the run of positions, .y: head and tensor, .z: sequence.
// Bound by the copy: 8 sequences of 100 to 8192 keys, 8 heads of 128, 362 MB with the zeros behind them in 66.7 us, 5.4 TB/s; the 8-bit
// rows of 12948 keys back to 16 bits in 15 us.
template <bool BF16, int D, bool FP8>
__global__ __launch_bounds__(kThreads) void paged_read_kernel(RowArgs a) {
    constexpr int kLanes = D / 8, kRowsPerPass = kThreads / kLanes, kRows = kRowsPerPass * kUnits;
    const PagedBatch& p = a.batch;
    const int tid = threadIdx.x, sub = tid % kLanes;
    const int tensor = blockIdx.y >= (unsigned)p.kv_heads, head = (int)blockIdx.y - (tensor ? p.kv_heads : 0);
    for (int b = blockIdx.z; b < p.batch; b += gridDim.z) {
        const int keys = (int)min((int64_t)max(p.kv_lens[b], 0), (int64_t)p.width << p.page_shift);
        u32x4 w[kUnits];
#pragma unroll
        for (int i = 0; i < kUnits; ++i) {
            const int pos = (int)blockIdx.x * kRows + i * kRowsPerPass + tid / kLanes;
            w[i] = u32x4{0u, 0u, 0u, 0u};
            if (pos >= min(keys, a.max_len)) continue;
            const int page = p.page_table[(size_t)b * p.width + (pos >> p.page_shift)];
            if (page < 0 || page >= p.num_pages) continue;
            const int64_t row = (((int64_t)page * p.kv_heads + head) << p.page_shift) + (pos & ((1 << p.page_shift) - 1));
            if constexpr (FP8) {
                const u32x2 bytes = reinterpret_cast<const u32x2*>(static_cast<const uint8_t*>(tensor ? a.pool[1] : a.pool[0]) + row * D)[sub];
                w[i] = to_halves<BF16>(bytes, (tensor ? a.exponent[1] : a.exponent[0])[row]);
            } else {
                w[i] = reinterpret_cast<const u32x4*>(static_cast<const uint16_t*>(tensor ? a.pool[1] : a.pool[0]) + row * D)[sub];
            }
        }
        uint16_t* out = static_cast<uint16_t*>(tensor ? a.out[1] : a.out[0]) + ((int64_t)b * p.kv_heads + head) * a.max_len * D;
#pragma unroll
        for (int i = 0; i < kUnits; ++i) {
            const int pos = (int)blockIdx.x * kRows + i * kRowsPerPass + tid / kLanes;
            if (pos < a.max_len) __builtin_nontemporal_store(w[i], reinterpret_cast<u32x4*>(out + (int64_t)pos * D) + sub);
        }
    }
}

// Draft trees to masks: bit j of a node's row is set where j is the node itself or one of its ancestors (numbers within its
// tree).  A parent is a smaller number (anything else counts as a root), so a walk to the root meets the words of a row from the
// node's own downwards, and what one node of a word contributes to it is the same for every walk that enters the word there: the
// bits of its ancestors among the word's 32 nodes, and the number at which the walk leaves them.  Both come from five rounds of
// doubling between the lanes of half a wave, for all nodes up to the workgroup's own; they stay in LDS, and a row is then a walk
// over words, one LDS read each, instead of one dependent read of global memory per ancestor.  Rows are cleared first, 16 bytes
// a lane, since most words of a deep tree's rows are empty.  Nodes that LDS has no room for (their numbers are the largest ones)
// are walked in global memory until the walk reaches those that it holds.  Bound by latency: 16 trees of up to 256 nodes 4.8 us, of
// which a launch is about 3; 4 trees of up to 2048 nodes, 85 ancestors each and 2 MB of rows, 9.8 us (28 us by the walk over nodes).
// 64 rows a workgroup, and not 256: the doubling is done by more workgroups then, but on CUs that would have nothing to do.
struct TreeNode { uint32_t bits; int32_t exit; };

__global__ __launch_bounds__(kThreads) void tree_bits_kernel(const int64_t* parent, const int32_t* q_starts, int32_t batch,
                                                             int32_t tokens, int32_t words, int32_t room, uint32_t* bits) {
    extern __shared__ TreeNode nodes[];
    const int tid = threadIdx.x, lane = tid & 63;
    {   // tokens of no tree
        const int first = min(max(q_starts[0], 0), tokens), end = min(max(q_starts[batch], 0), tokens);
        const int64_t none = (int64_t)(first + max(tokens - max(first, end), 0)) * words;
        for (int64_t i = (int64_t)blockIdx.x * kThreads + tid; i < none; i += (int64_t)gridDim.x * kThreads)
            bits[i < (int64_t)first * words ? i : i + (int64_t)(max(first, end) - first) * words] = 0u;
    }
    const int chunks = (words * 32 + kTreeRows - 1) / kTreeRows;
    for (int64_t item = blockIdx.x; item < (int64_t)chunks * batch; item += gridDim.x) {
        const int b = (int)(item / chunks), start = min(max(q_starts[b], 0), tokens);
        const int count = min(max(q_starts[b + 1], 0), tokens) - start;
        // The last chunk of a tree takes what a tree of more nodes than the rows have bits has over
        const int chunk = (int)(item % chunks);
        for (int64_t node0 = (int64_t)chunk * kTreeRows; node0 < count && (node0 / kTreeRows == chunk || chunk == chunks - 1); node0 += kTreeRows) {
            const int own = (int)min((int64_t)count - node0, (int64_t)kTreeRows);
            const int known = ((int)min(node0 + own, (int64_t)room) + 31) & ~31;
            const int64_t* up = parent + start;
            uint32_t* rows = bits + (start + node0) * words;
            const auto parent_of = [&](int n) {
                const int64_t p = up[n];
                return p >= 0 && p < n ? (int)p : -1;
            };
            for (int n = tid; n < known; n += kThreads) {   // whole half waves: known is a multiple of 32
                const int p = n < count ? parent_of(n) : -1;
                const int base = n & ~31, inside = p >= base;
                uint32_t mask = 1u << (n & 31);
                int link = inside ? (lane & 32) + (p & 31) : lane;
#pragma unroll
                for (int round = 0; round < 5; ++round) {
                    mask |= (uint32_t)__shfl((int)mask, link);
                    link = __shfl(link, link);
                }
                nodes[n] = {mask, __shfl(p, link)};
            }
            const int64_t total = (int64_t)own * words;         // (64 rows of 2^25 words are accepted)
            if ((reinterpret_cast<uintptr_t>(rows) & 15) == 0) {
                for (int64_t i = tid; i < total / 4; i += kThreads) reinterpret_cast<u32x4*>(rows)[i] = u32x4{0u, 0u, 0u, 0u};
                for (int64_t i = (total & ~(int64_t)3) + tid; i < total; i += kThreads) rows[i] = 0u;
            } else {
                for (int64_t i = tid; i < total; i += kThreads) rows[i] = 0u;
            }
            __syncthreads();
            if (tid < own) {
                uint32_t* row = rows + (int64_t)tid * words;
                int node = (int)node0 + tid;
                uint32_t word = 0u;
                while (node >= known) {
                    word |= 1u << (node & 31);
                    const int next = parent_of(node);
                    if (next < (node & ~31)) {
                        if (node / 32 < words) row[node / 32] = word;
                        word = 0u;
                    }
                    node = next;
                }
                while (node >= 0) {
                    const TreeNode at = nodes[node];
                    if (node / 32 < words) row[node / 32] = at.bits;
                    node = at.exit;
                }
            }
            __syncthreads();
        }
    }
}

template <bool BF16, int D> int launch_write(const RowArgs& a, bool fp8, hipStream_t stream) {
    constexpr uint64_t kRows = (uint64_t)kThreads / (D / 8) * kUnits;
    const uint64_t groups = ((uint64_t)a.batch.tokens * 2u * (uint64_t)a.batch.kv_heads + kRows - 1) / kRows;
    if (groups * kThreads >= (uint64_t)1 << 32) return fail(FSTA_EUNSUPPORTED, "fsta_paged_write: %d tokens of %d heads", a.batch.tokens, a.batch.kv_heads);
    if (fp8) hipLaunchKernelGGL((paged_write_kernel<BF16, D, true>), dim3((unsigned)groups), dim3(kThreads), 0, stream, a);
    else hipLaunchKernelGGL((paged_write_kernel<BF16, D, false>), dim3((unsigned)groups), dim3(kThreads), 0, stream, a);
    FSTA_HIP_OK(hipGetLastError());
    return FSTA_OK;
}

template <bool BF16, int D> int launch_read(const RowArgs& a, bool fp8, hipStream_t stream) {
    constexpr int kRows = kThreads / (D / 8) * kUnits;
    const int64_t runs = ((int64_t)a.max_len + kRows - 1) / kRows;
    const int64_t heads = 2 * (int64_t)a.batch.kv_heads;
    // (more sequences than a grid of 2^32 threads holds are walked by the workgroups)
    int64_t seqs = a.batch.batch < 65535 ? a.batch.batch : 65535;
    while (seqs > 1 && (double)runs * (double)heads * (double)seqs * kThreads >= 4294967296.0) seqs = (seqs + 1) / 2;
    if ((double)runs * (double)heads * (double)seqs * kThreads >= 4294967296.0)
        return fail(FSTA_EUNSUPPORTED, "fsta_paged_read: %d positions of %d heads", a.max_len, a.batch.kv_heads);
    const dim3 grid((unsigned)runs, (unsigned)heads, (unsigned)seqs);
    if (fp8) hipLaunchKernelGGL((paged_read_kernel<BF16, D, true>), grid, dim3(kThreads), 0, stream, a);
    else hipLaunchKernelGGL((paged_read_kernel<BF16, D, false>), grid, dim3(kThreads), 0, stream, a);
    FSTA_HIP_OK(hipGetLastError());
    return FSTA_OK;
}

int check_pool(const char* who, const void* k, const void* v, const uint8_t* ke, const uint8_t* ve, bool fp8) {
    if (!k || !v || (fp8 && (!ke || !ve))) return fail(FSTA_EINVAL, "%s: null pointer", who);
    if (misaligned(k, 16) || misaligned(v, 16)) return fail(FSTA_EINVAL, "%s: the cache must be 16-byte aligned", who);
    if (misaligned(ke, 4) || misaligned(ve, 4)) return fail(FSTA_EINVAL, "%s: exponents must be 4-byte aligned", who);
    return FSTA_OK;
}

int shift_of(int32_t page_size) {
    int s = 0;
    while ((1 << s) < page_size) ++s;
    return s;
}

}  // namespace

int check_paged_batch(const char* who, const PagedBatch& p, int32_t page_size, int32_t head_dim, int32_t cache_dtype, bool new_tokens) {
    if (p.batch < 0 || p.tokens < 0 || p.width < 0 || p.num_pages < 0 || p.kv_heads <= 0)
        return fail(FSTA_EINVAL, "%s: batch=%d tokens=%d width=%d num_pages=%d kv_heads=%d", who, p.batch, p.tokens, p.width, p.num_pages, p.kv_heads);
    if (page_size < 16 || page_size > 4096 || (page_size & (page_size - 1)))
        return fail(FSTA_EUNSUPPORTED, "%s: page_size=%d (a power of two from 16 to 4096)", who, page_size);
    if (head_dim != 64 && head_dim != 128) return fail(FSTA_EUNSUPPORTED, "%s: head_dim=%d (64 or 128)", who, head_dim);
    if (cache_dtype != FSTA_F16 && cache_dtype != FSTA_BF16 && cache_dtype != FSTA_FP8)
        return fail(FSTA_EINVAL, "%s: cache_dtype=%d", who, cache_dtype);
    if (p.kv_heads > 16384) return fail(FSTA_EUNSUPPORTED, "%s: kv_heads=%d (at most 16384)", who, p.kv_heads);
    if ((int64_t)p.width * page_size > 0x7fffffc0ll) return fail(FSTA_EUNSUPPORTED, "%s: %d pages of %d keys in a sequence", who, p.width, page_size);
    if (p.batch > 0 && ((p.width > 0 && !p.page_table) || !p.kv_lens || (new_tokens && !p.q_starts))) return fail(FSTA_EINVAL, "%s: null pointer", who);
    if (misaligned(p.page_table, 4) || misaligned(p.kv_lens, 4) || misaligned(p.q_starts, 4))
        return fail(FSTA_EINVAL, "%s: page_table, kv_lens and q_starts must be 4-byte aligned", who);
    return FSTA_OK;
}

}  // namespace fsta

using namespace fsta;

extern "C" int fsta_paged_write(const void* k, const void* v, int64_t k_token_stride, int64_t k_head_stride, int64_t v_token_stride,
                                int64_t v_head_stride, void* k_cache, void* v_cache, uint8_t* k_exponent, uint8_t* v_exponent,
                                const int32_t* page_table, const int32_t* kv_lens, const int32_t* q_starts, int32_t batch,
                                int32_t width, int32_t tokens, int32_t num_pages, int32_t page_size, int32_t kv_heads,
                                int32_t head_dim, int32_t dtype, int32_t cache_dtype, void* stream) {
    const char* who = "fsta_paged_write";
    RowArgs a = {};
    a.batch = PagedBatch{page_table, kv_lens, q_starts, batch, width, num_pages, 0, kv_heads, tokens};
    int rc = check_paged_batch(who, a.batch, page_size, head_dim, cache_dtype, true);
    if (rc != FSTA_OK) return rc;
    if (dtype != FSTA_F16 && dtype != FSTA_BF16) return fail(FSTA_EINVAL, "%s: dtype=%d", who, dtype);
    if (cache_dtype != FSTA_FP8 && cache_dtype != dtype) return fail(FSTA_EINVAL, "%s: cache_dtype=%d for dtype=%d", who, cache_dtype, dtype);
    if (batch == 0 || tokens == 0 || width == 0 || num_pages == 0) return FSTA_OK;
    const bool fp8 = cache_dtype == FSTA_FP8;
    if (!k || !v) return fail(FSTA_EINVAL, "%s: null pointer", who);
    rc = check_pool(who, k_cache, v_cache, k_exponent, v_exponent, fp8);
    if (rc != FSTA_OK) return rc;
    if (misaligned(k, 16) || misaligned(v, 16) || ((k_token_stride | k_head_stride | v_token_stride | v_head_stride) & 7))
        return fail(FSTA_EINVAL, "%s: rows of k and v must be 16-byte aligned", who);
    a.batch.page_shift = shift_of(page_size);
    a.src[0] = k; a.src[1] = v;
    a.token_stride[0] = k_token_stride; a.token_stride[1] = v_token_stride;
    a.head_stride[0] = k_head_stride; a.head_stride[1] = v_head_stride;
    a.pool[0] = k_cache; a.pool[1] = v_cache;
    a.exponent[0] = k_exponent; a.exponent[1] = v_exponent;
    hipStream_t s = static_cast<hipStream_t>(stream);
    if (dtype == FSTA_BF16) return head_dim == 128 ? launch_write<true, 128>(a, fp8, s) : launch_write<true, 64>(a, fp8, s);
    return head_dim == 128 ? launch_write<false, 128>(a, fp8, s) : launch_write<false, 64>(a, fp8, s);
}

extern "C" int fsta_paged_read(const void* k_cache, const void* v_cache, const uint8_t* k_exponent, const uint8_t* v_exponent,
                               const int32_t* page_table, const int32_t* kv_lens, void* k, void* v, int32_t batch, int32_t width,
                               int32_t max_len, int32_t num_pages, int32_t page_size, int32_t kv_heads, int32_t head_dim,
                               int32_t dtype, int32_t cache_dtype, void* stream) {
    const char* who = "fsta_paged_read";
    RowArgs a = {};
    a.batch = PagedBatch{page_table, kv_lens, nullptr, batch, width, num_pages, 0, kv_heads, 0};
    int rc = check_paged_batch(who, a.batch, page_size, head_dim, cache_dtype, false);
    if (rc != FSTA_OK) return rc;
    if (max_len < 0) return fail(FSTA_EINVAL, "%s: max_len=%d", who, max_len);
    if (dtype != FSTA_F16 && dtype != FSTA_BF16) return fail(FSTA_EINVAL, "%s: dtype=%d", who, dtype);
    if (cache_dtype != FSTA_FP8 && cache_dtype != dtype) return fail(FSTA_EINVAL, "%s: cache_dtype=%d for dtype=%d", who, cache_dtype, dtype);
    if (batch == 0 || max_len == 0) return FSTA_OK;
    const bool fp8 = cache_dtype == FSTA_FP8;
    if (!k || !v) return fail(FSTA_EINVAL, "%s: null pointer", who);
    if (num_pages > 0) {                 // (an empty pool may have no memory: no page is looked at)
        rc = check_pool(who, k_cache, v_cache, k_exponent, v_exponent, fp8);
        if (rc != FSTA_OK) return rc;
    }
    if (misaligned(k, 16) || misaligned(v, 16)) return fail(FSTA_EINVAL, "%s: k and v must be 16-byte aligned", who);
    a.batch.page_shift = shift_of(page_size);
    a.pool[0] = const_cast<void*>(k_cache); a.pool[1] = const_cast<void*>(v_cache);
    a.exponent[0] = const_cast<uint8_t*>(k_exponent); a.exponent[1] = const_cast<uint8_t*>(v_exponent);
    a.out[0] = k; a.out[1] = v;
    a.max_len = max_len;
    hipStream_t s = static_cast<hipStream_t>(stream);
    if (dtype == FSTA_BF16) return head_dim == 128 ? launch_read<true, 128>(a, fp8, s) : launch_read<true, 64>(a, fp8, s);
    return head_dim == 128 ? launch_read<false, 128>(a, fp8, s) : launch_read<false, 64>(a, fp8, s);
}

extern "C" int fsta_tree_bits(const int64_t* parent, const int32_t* q_starts, int32_t batch, int32_t tokens, int32_t words,
                              uint32_t* bits, void* stream) {
    const char* who = "fsta_tree_bits";
    if (batch < 0 || tokens < 0 || words < 0) return fail(FSTA_EINVAL, "%s: batch=%d tokens=%d words=%d", who, batch, tokens, words);
    if (tokens == 0 || words == 0) return FSTA_OK;
    if (batch == 0) return fail(FSTA_EINVAL, "%s: %d tokens of no sequence", who, tokens);
    if (!parent || !q_starts || !bits) return fail(FSTA_EINVAL, "%s: null pointer", who);
    if (misaligned(parent, 8) || misaligned(q_starts, 4) || misaligned(bits, 4))
        return fail(FSTA_EINVAL, "%s: parent must be 8-byte, q_starts and bits 4-byte aligned", who);
    const int64_t bits_of_row = (int64_t)words * 32, chunks = (bits_of_row + kTreeRows - 1) / kTreeRows, want = chunks * batch;
    if (bits_of_row > INT32_MAX - kTreeRows) return fail(FSTA_EUNSUPPORTED, "%s: words=%d", who, words);
    const int32_t room = (int32_t)(bits_of_row < kTreeNodes ? bits_of_row : kTreeNodes);
    hipLaunchKernelGGL(tree_bits_kernel, dim3((unsigned)(want < 65536 ? want : 65536)), dim3(kThreads), room * sizeof(TreeNode),
                       static_cast<hipStream_t>(stream), parent, q_starts, batch, tokens, words, room, bits);
    FSTA_HIP_OK(hipGetLastError());
    return FSTA_OK;
}
