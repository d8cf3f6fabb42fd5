// What happens to the pages of a paged cache between two passes of a model: the rows of an accepted path move together, pages are
// given to sequences and taken back, sequences share pages, pages are copied.  All layers in one launch: their pointers travel in
// the kernel's arguments.
//
// Rows are bytes here: a row of head_dim values is 4, 8 or 16 lanes of 16 bytes, an 8-bit row's exponent one byte beside it.
#include "fsta_paged.h"

namespace fsta {
namespace {

typedef unsigned int u32x4 __attribute__((ext_vector_type(4)));

constexpr int kThreads = 256, kWaves = kThreads / 64;
constexpr int kMaxLayers = 32;            // per launch (64 bytes of the 4 KB of kernel arguments each)
constexpr int kPiece = 2048;              // 16-byte units of a page that a workgroup copies
constexpr int kGroup = 2048;              // pages whose free ones a wave lists at a time

struct Layer {
    uint8_t* rows[2];                     // k, v
    uint8_t* exponent[2];                 // or null
    uint8_t* into[2];                     // where pages go to: the same pool, or another
    uint8_t* into_exponent[2];
};
struct Layers {
    Layer at[kMaxLayers];
    uint16_t heads[kMaxLayers], lanes[kMaxLayers];    // lanes: 16-byte units of a row
};

// ---- rows of an accepted path ------------------------------------------------------------------------------------------

struct CompactArgs {
    const int32_t *path, *counts, *page_table, *kv_lens, *q_starts;
    int32_t* new_lens;
    int32_t max_path, batch, width, num_pages, page_shift;
};

// blockIdx.x: layer and tensor, .y: heads in fours, .z: sequence; a wave moves the rows of one head.  A row's place lies at or before
// the place it comes from, and a path's numbers ascend: a place that is written was read before, or nobody reads it, so a
// wave that loads some rows and then stores them, from the front to the back, needs no copy of them.
// Bound by loads that need each other (lengths, path, table, rows) and by starting workgroups that move a handful of rows: 3.9 us for one
// conversation in 32 layers, 11.3 for 96 in 24 layers of 8 bits (15 MB).  Fewer workgroups with several layers each: 17.6.
template <int LANES>
__device__ void move_rows(uint8_t* rows, uint8_t* exponent, const int64_t* from, const int64_t* to, int count, int head, int page_shift) {
    constexpr int kAtOnce = 64 / LANES, kUnits = 4;
    const int lane = threadIdx.x & 63, sub = lane % LANES, mine = lane / LANES;
    for (int i0 = 0; i0 < count; i0 += kAtOnce * kUnits) {
        u32x4 w[kUnits];
        uint8_t e[kUnits];
        int64_t place[kUnits];
#pragma unroll
        for (int u = 0; u < kUnits; ++u) {
            const int i = i0 + u * kAtOnce + mine;
            place[u] = -1;
            e[u] = 0;
            w[u] = u32x4{0u, 0u, 0u, 0u};
            if (i < count) {
                const int64_t source = from[i] + ((int64_t)head << page_shift);
                place[u] = to[i] + ((int64_t)head << page_shift);
                w[u] = reinterpret_cast<const u32x4*>(rows)[source * LANES + sub];
                if (exponent) e[u] = exponent[source];
            }
        }
#pragma unroll
        for (int u = 0; u < kUnits; ++u) {
            if (place[u] < 0) continue;
            reinterpret_cast<u32x4*>(rows)[place[u] * LANES + sub] = w[u];
            if (exponent && sub == 0) exponent[place[u]] = e[u];
        }
    }
}

__global__ __launch_bounds__(kThreads) void compact_kernel(CompactArgs a, Layers layers) {
    __shared__ int64_t from[64], to[64];      // rows of head 0 of the pool
    __shared__ int moved;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int layer = blockIdx.x >> 1, tensor = blockIdx.x & 1, heads = layers.heads[layer], lanes = layers.lanes[layer];
    for (int b = blockIdx.z; b < a.batch; b += gridDim.z) {
        const int keys = (int)min((int64_t)max(a.kv_lens[b], 0), (int64_t)a.width << a.page_shift);
        const int fresh = (int)min(max((int64_t)a.q_starts[b + 1] - a.q_starts[b], (int64_t)0), (int64_t)keys);
        const int base = keys - fresh, count = min(min(max(a.counts[b], 0), fresh), a.max_path);
        if (blockIdx.x == 0 && blockIdx.y == 0 && tid == 0) a.new_lens[b] = base + count;
        for (int i0 = 0; i0 < count; i0 += 64) {
            if (wave == 0) {
                const int i = i0 + lane;
                const int p = i < count ? a.path[(int64_t)b * a.max_path + i] : -1;
                int64_t source = -1, target = -1;
                if (p >= 0 && p < fresh && p != i) {
                    const int mask = (1 << a.page_shift) - 1;
                    const int old = a.page_table[(int64_t)b * a.width + ((base + p) >> a.page_shift)];
                    const int fits = a.page_table[(int64_t)b * a.width + ((base + i) >> a.page_shift)];
                    if (old >= 0 && old < a.num_pages && fits >= 0 && fits < a.num_pages) {
                        source = (((int64_t)old * heads) << a.page_shift) + ((base + p) & mask);
                        target = (((int64_t)fits * heads) << a.page_shift) + ((base + i) & mask);
                    }
                }
                const uint64_t moves = __ballot(source >= 0);
                if (source >= 0) {
                    const int at = __popcll(moves & ((1ull << lane) - 1));
                    from[at] = source;
                    to[at] = target;
                }
                if (lane == 0) moved = __popcll(moves);
            }
            __syncthreads();
            const int n = moved;
            const Layer& at = layers.at[layer];
            for (int head = (int)blockIdx.y * kWaves + wave; head < heads; head += (int)gridDim.y * kWaves) {
                if (lanes == 16) move_rows<16>(at.rows[tensor], at.exponent[tensor], from, to, n, head, a.page_shift);
                else if (lanes == 8) move_rows<8>(at.rows[tensor], at.exponent[tensor], from, to, n, head, a.page_shift);
                else move_rows<4>(at.rows[tensor], at.exponent[tensor], from, to, n, head, a.page_shift);
            }
            __syncthreads();
        }
    }
}

// ---- whole pages, or their first rows ----------------------------------------------------------------------------------

struct Copy { int32_t from, to, rows; };

struct CopyArgs {
    const int32_t *sources, *targets;     // whole pages ..
    const Copy* list;                     // .. or what the page table's kernels listed, *listed of them
    const int32_t* listed;
    int32_t pairs, num_pages, into_pages, page_shift;
};

// blockIdx.x: which copy, .y: layer and tensor, .z: piece of the page's rows.  The rows of all heads of a whole page lie
// together; of a part the rows of one head do.  Bound by memory: 1024 pages of 8 layers, 4.3 GB read and written, 831 us, 5.2 TB/s (past the
// caches: what is copied is not read soon); 336 tails of 12 layers in 8 bits 100 us, 518 MB.
template <bool LIST>
__global__ __launch_bounds__(kThreads) void copy_pages_kernel(CopyArgs a, Layers layers) {
    constexpr int kUnits = kPiece / kThreads;
    const int tid = threadIdx.x, layer = blockIdx.y >> 1, tensor = blockIdx.y & 1;
    const int heads = layers.heads[layer], lanes = layers.lanes[layer], page = 1 << a.page_shift;
    const int count = LIST ? *a.listed : a.pairs;
    for (int i = blockIdx.x; i < count; i += gridDim.x) {
        Copy c{0, 0, page};
        if constexpr (LIST) {
            c = a.list[i];
        } else {
            c.from = a.sources[i];
            c.to = a.targets[i];
            if (c.from < 0 || c.from >= a.num_pages || c.to < 0 || c.to >= a.into_pages) continue;
            if (c.from == c.to && layers.at[layer].rows[tensor] == layers.at[layer].into[tensor]) continue;
        }
        const Layer& at = layers.at[layer];
        const int64_t page_units = ((int64_t)heads * lanes) << a.page_shift;
        const u32x4* src = reinterpret_cast<const u32x4*>(at.rows[tensor]) + c.from * page_units;
        u32x4* dst = reinterpret_cast<u32x4*>(at.into[tensor]) + c.to * page_units;
        const uint32_t head_units = (uint32_t)c.rows * lanes, total = head_units * heads;
        for (uint32_t first = blockIdx.z * kPiece; first < total; first += gridDim.z * kPiece) {
            u32x4 w[kUnits];
            uint32_t where[kUnits];
#pragma unroll
            for (int u = 0; u < kUnits; ++u) {
                const uint32_t n = first + u * kThreads + tid;
                where[u] = n;
                if (LIST) where[u] = n / head_units * (uint32_t)(lanes << a.page_shift) + n % head_units;
                if (n < total) w[u] = __builtin_nontemporal_load(src + where[u]);
            }
#pragma unroll
            for (int u = 0; u < kUnits; ++u)
                if (first + u * kThreads + tid < total) __builtin_nontemporal_store(w[u], dst + where[u]);
        }
        if (at.exponent[tensor] && blockIdx.z == 0) {
            const int64_t rows = (int64_t)heads << a.page_shift;
            const uint8_t* from = at.exponent[tensor] + c.from * rows;
            uint8_t* to = at.into_exponent[tensor] + c.to * rows;
            for (int n = tid; n < heads * c.rows; n += kThreads) {
                const int where = LIST ? (n / c.rows << a.page_shift) + n % c.rows : n;
                to[where] = from[where];
            }
        }
    }
}

// ---- who holds which page ----------------------------------------------------------------------------------------------

struct TableArgs {
    int32_t *refs, *table, *missing;
    const int32_t* lens;                  // fit: the lengths wanted
    int32_t* slot_lens;                   // fork: the slots' own
    const int32_t *sources, *targets;     // fork
    int32_t batch, width, num_pages, page_shift, pairs;
    // workspace
    int32_t* listed;                      // how many tails are to be copied, and which
    Copy* list;
    int32_t* need;                        // [batch or pairs] free pages wanted
    int32_t* group_free;                  // [groups] free pages of each kGroup
    uint32_t* free_bits;                  // [groups][kGroup / 32]
    int32_t *rows, *row_lens;             // fork: [pairs][width] the sources' entries, [pairs] their lengths or -1
};

__device__ __forceinline__ int groups_of(const TableArgs& a) { return (a.num_pages + kGroup - 1) / kGroup; }

__device__ __forceinline__ void list_copy(const TableArgs& a, int from, int to, int rows) {
    a.list[atomicAdd(a.listed, 1)] = Copy{from, to, rows};      // (their order is nobody's concern: no two touch one page)
}

// One wave: which of a group's pages are free, 32 a lane
__device__ void survey_group(const TableArgs& a, int g) {
    const int lane = threadIdx.x & 63;
    const int64_t first = (int64_t)g * kGroup + lane * 32, pages = a.num_pages;
    int4 refs[8];                         // (all on their way at once; places behind the last page are read at its own)
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const int64_t p = first + 4 * i;
        if (pages >= 4) __builtin_memcpy(&refs[i], a.refs + min(p, pages - 4), sizeof(int4));
    }
    uint32_t word = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const int held[4] = {refs[i].x, refs[i].y, refs[i].z, refs[i].w};
#pragma unroll
        for (int e = 0; e < 4; ++e) word |= (uint32_t)(held[e] <= 0) << (4 * i + e);
    }
    if (first + 32 > pages) {             // the last pages, one by one
        word = 0;
        for (int e = 0; e < 32; ++e)
            if (first + e < pages && a.refs[first + e] <= 0) word |= 1u << e;
    }
    a.free_bits[(int64_t)g * (kGroup / 32) + lane] = word;
    const int total = __shfl((int)wave_prefix_sum((uint32_t)__popc(word)), 63);
    if (lane == 0) a.group_free[g] = total;
}

__device__ __forceinline__ int sum_of(int x) {
#pragma unroll
    for (int d = 32; d; d >>= 1) x += __shfl_xor(x, d);
    return x;
}

// A wave's way through the free pages in ascending order: the ones of the group that it stands at lie in LDS
struct FreePages {
    uint16_t* ids;                        // [kGroup]
    int group, first, count;              // group's number, rank of its first free page, how many
    // Moves to the group with the free page of that rank (at or behind the current one's); false: there is none
    __device__ bool seek(const TableArgs& a, int rank) {
        const int lane = threadIdx.x & 63, groups = groups_of(a);
        int base = first + count;
        int next = group + 1 + lane < groups ? a.group_free[group + 1 + lane] : 0;
        for (int g0 = group + 1; g0 < groups; g0 += 64) {
            const int mine = next;
            next = g0 + 64 + lane < groups ? a.group_free[g0 + 64 + lane] : 0;
            const int up_to = (int)wave_prefix_sum((uint32_t)mine);
            const uint64_t hit = __ballot(base + up_to > rank);
            if (hit) {
                const int l = __ffsll((unsigned long long)hit) - 1;
                group = g0 + l;
                count = __shfl(mine, l);
                first = base + __shfl(up_to, l) - count;
                uint32_t word = a.free_bits[(int64_t)group * (kGroup / 32) + lane];
                const int n = __popc(word);
                int at = (int)wave_prefix_sum((uint32_t)n) - n;
                __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
                for (; word; word &= word - 1) ids[at++] = (uint16_t)(lane * 32 + __ffs((int)word) - 1);
                __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
                __builtin_amdgcn_wave_barrier();
                return true;
            }
            base += __shfl(up_to, 63);
        }
        group = groups;
        first = base;
        count = 0;
        return false;
    }
    // The page of each lane that wants one, ranks ascending with the lanes; -1 where there are no more
    __device__ int take(const TableArgs& a, bool wanted, int rank) {
        int page = -1;
        for (;;) {
            if (wanted && rank < first + count) {
                page = group * kGroup + ids[rank - first];
                wanted = false;
            }
            const uint64_t open = __ballot(wanted);
            if (!open || !seek(a, __shfl(rank, __ffsll((unsigned long long)open) - 1))) return page;
        }
    }
};

__device__ __forceinline__ int needed_before(const TableArgs& a, int i) {
    int sum = 0;
    for (int j = threadIdx.x & 63; j < i; j += 8 * 64) {
        int some[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) some[k] = a.need[min(j + 64 * k, i - 1)];
#pragma unroll
        for (int k = 0; k < 8; ++k) sum += j + 64 * k < i ? some[k] : 0;
    }
    return sum_of(sum);
}

// What a sequence of n positions wants of entry `slot` of its row, which now is `page`
struct Entry { bool named, inside, tail, wanted; };
__device__ __forceinline__ Entry judge(const TableArgs& a, int n, int slot, int page) {
    const int keep = (int)(((int64_t)n + (1 << a.page_shift) - 1) >> a.page_shift);
    Entry e;
    e.named = page >= 0 && page < a.num_pages;
    e.inside = slot < keep;
    e.tail = e.named && slot == keep - 1 && (n & ((1 << a.page_shift) - 1));
    e.wanted = e.inside && !e.named;
    return e;
}

// Entries s0 + 64 k + lane of a row, for eight k at once; -1 behind its end
constexpr int kStrips = 8;
__device__ __forceinline__ void load_strips(const int32_t* row, int s0, int end, int (&page)[kStrips]) {
    const int lane = threadIdx.x & 63;
#pragma unroll
    for (int k = 0; k < kStrips; ++k) page[k] = row[min(s0 + 64 * k + lane, end - 1)];
#pragma unroll
    for (int k = 0; k < kStrips; ++k)
        if (s0 + 64 * k + lane >= end) page[k] = -1;
}

__device__ void survey_fit(const TableArgs& a, int b) {
    const int lane = threadIdx.x & 63;
    const int n = (int)min((int64_t)max(a.lens[b], 0), (int64_t)a.width << a.page_shift);
    const int keep = (int)(((int64_t)n + (1 << a.page_shift) - 1) >> a.page_shift);
    const int32_t* row = a.table + (int64_t)b * a.width;
    int need = 0, last = -1;
    if (keep > 0) last = row[keep - 1];   // (meanwhile the others come)
    for (int s0 = 0; s0 < keep; s0 += 64 * kStrips) {
        int page[kStrips];
        load_strips(row, s0, keep, page);
#pragma unroll
        for (int k = 0; k < kStrips; ++k) need += s0 + 64 * k + lane < keep && (page[k] < 0 || page[k] >= a.num_pages);
    }
    need = sum_of(need);
    const bool copies = judge(a, n, keep - 1, last).tail && a.refs[last] > 1;
    if (lane == 0) {
        a.need[b] = need + copies;
        a.row_lens[b] = copies;           // the last page is one that others hold too (refs change in the next launch)
    }
}

__device__ void assign_fit(const TableArgs& a, int b, uint16_t* ids) {
    const int lane = threadIdx.x & 63;
    const int n = (int)min((int64_t)max(a.lens[b], 0), (int64_t)a.width << a.page_shift);
    const int need = a.need[b];
    const bool copies = a.row_lens[b] != 0;
    int32_t* row = a.table + (int64_t)b * a.width;
    int next = need ? needed_before(a, b) : 0, missing = 0;
    FreePages free{ids, -1, 0, 0};
    for (int s0 = 0; s0 < a.width; s0 += 64 * kStrips) {
        int page[kStrips];
        load_strips(row, s0, a.width, page);
#pragma unroll 1
        for (int k = 0; k < kStrips; ++k) {
            int own = page[0];            // (one after the other to the front: a register cannot be chosen by a number)
#pragma unroll
            for (int j = 0; j < kStrips - 1; ++j) page[j] = page[j + 1];
            const int s = s0 + 64 * k + lane;
            const Entry e = judge(a, n, s, own);
            const bool copied = e.tail && copies, wanted = s < a.width && (e.wanted || copied);
            const uint64_t all = __ballot(wanted);
            int fresh = -1;
            if (all) {
                fresh = free.take(a, wanted, next + __popcll(all & ((1ull << lane) - 1)));
                next += __popcll(all);
                missing += __popcll(__ballot(wanted && fresh < 0));
            }
            if (s >= a.width) continue;
            const int now = fresh >= 0 ? fresh : e.inside && e.named ? own : -1;
            if (now == own) continue;
            row[s] = now;
            if (fresh >= 0) a.refs[fresh] = 1;
            if (e.named) atomicSub(a.refs + own, 1);
            if (copied) list_copy(a, own, fresh, n & ((1 << a.page_shift) - 1));
        }
    }
    if (lane == 0) a.missing[b] = missing;
}

// A slot's source as it is before the call, since other pairs may write to it
__device__ void survey_fork(const TableArgs& a, int i) {
    const int lane = threadIdx.x & 63;
    const int source = a.sources[i], target = a.targets[i];
    bool first = source >= 0 && source < a.batch && target >= 0 && target < a.batch;
    for (int j0 = 0; first && j0 < i; j0 += 64) {
        const int j = j0 + lane;
        first = !__ballot(j < i && a.targets[j] == target && a.sources[j] >= 0 && a.sources[j] < a.batch);
    }
    if (!first || source == target) {
        if (lane == 0) {
            a.row_lens[i] = -1;
            a.need[i] = 0;
        }
        return;
    }
    const int n = (int)min((int64_t)max(a.slot_lens[source], 0), (int64_t)a.width << a.page_shift);
    bool tail = false;
    for (int s = lane; s < a.width; s += 64) {
        const int page = a.table[(int64_t)source * a.width + s];
        const Entry e = judge(a, n, s, page);
        tail |= e.tail;
        a.rows[(int64_t)i * a.width + s] = e.named && e.inside ? page : -1;
    }
    const bool need = __ballot(tail) != 0;
    if (lane == 0) {
        a.row_lens[i] = n;
        a.need[i] = need;
    }
}

__device__ void assign_fork(const TableArgs& a, int i, uint16_t* ids) {
    const int lane = threadIdx.x & 63, n = a.row_lens[i];
    if (n < 0) {
        if (lane == 0) a.missing[i] = 0;
        return;
    }
    const int target = a.targets[i];
    int fresh = -1;
    bool good = true;
    if (a.need[i]) {
        FreePages free{ids, -1, 0, 0};
        fresh = free.take(a, lane == 0, needed_before(a, i));
        fresh = __shfl(fresh, 0);
        good = fresh >= 0;
    }
    for (int s = lane; s < a.width; s += 64) {
        const int page = a.rows[(int64_t)i * a.width + s], old = a.table[(int64_t)target * a.width + s];
        const Entry e = judge(a, n, s, page);
        const int now = !good || !e.named ? -1 : e.tail ? fresh : page;
        if (old >= 0 && old < a.num_pages) atomicSub(a.refs + old, 1);
        if (now >= 0) {
            if (e.tail) {
                a.refs[fresh] = 1;
                list_copy(a, page, fresh, n & ((1 << a.page_shift) - 1));
            } else {
                atomicAdd(a.refs + page, 1);
            }
        }
        a.table[(int64_t)target * a.width + s] = now;
    }
    if (lane == 0) {
        a.slot_lens[target] = good ? n : 0;
        a.missing[i] = !good;
    }
}

template <bool FORK> __device__ __forceinline__ void survey(const TableArgs& a, int i) {
    const int rows = FORK ? a.pairs : a.batch;
    if (i >= rows) survey_group(a, i - rows);
    else if (FORK) survey_fork(a, i);
    else survey_fit(a, i);
}
template <bool FORK> __device__ __forceinline__ void assign(const TableArgs& a, int i, uint16_t* ids) {
    if (FORK) assign_fork(a, i, ids);
    else assign_fit(a, i, ids);
}

// Two launches: what is wanted and what is free, a wave per sequence (or pair) and per group of pages; then every wave finds its
// own share of the free pages, whose order makes the result independent of who comes first.  Bound by loads that need each other, so that all
// that a wave looks at is asked for at once: 4.7 and 4.8 us for 48 sequences, 5.5 and 7.3 for 1024 with 300000 pages (a step's two calls
// 50 us while loads waited for each other, 30 now); 8.7 for 336 forks.
template <bool FORK> __global__ __launch_bounds__(kThreads) void survey_kernel(TableArgs a) {
    if (blockIdx.x == 0 && threadIdx.x == 0) *a.listed = 0;
    const int all = (FORK ? a.pairs : a.batch) + groups_of(a);
    for (int i = (int)blockIdx.x * kWaves + (threadIdx.x >> 6); i < all; i += (int)gridDim.x * kWaves) survey<FORK>(a, i);
}
template <bool FORK> __global__ __launch_bounds__(kThreads) void assign_kernel(TableArgs a) {
    __shared__ uint16_t ids[kWaves][kGroup];
    for (int i = (int)blockIdx.x * kWaves + (threadIdx.x >> 6); i < (FORK ? a.pairs : a.batch); i += (int)gridDim.x * kWaves)
        assign<FORK>(a, i, ids[threadIdx.x >> 6]);
}

// ---- host --------------------------------------------------------------------------------------------------------------

int shift_of(int32_t page_size) {
    int s = 0;
    while ((1 << s) < page_size) ++s;
    return s;
}

int check_pools(const char* who, const fsta_paged_pool* pools, const fsta_paged_pool* into, int32_t layers, int32_t num_pages, int32_t page_size) {
    if (layers < 1 || num_pages < 0) return fail(FSTA_EINVAL, "%s: layers=%d num_pages=%d", who, layers, num_pages);
    if (!pools || !into) return fail(FSTA_EINVAL, "%s: null pointer", who);
    if (page_size < 16 || page_size > 4096 || (page_size & (page_size - 1)))
        return fail(FSTA_EUNSUPPORTED, "%s: page_size=%d (a power of two from 16 to 4096)", who, page_size);
    for (int32_t l = 0; l < layers; ++l) {
        const fsta_paged_pool &p = pools[l], &q = into[l];
        if (p.head_dim != 64 && p.head_dim != 128) return fail(FSTA_EUNSUPPORTED, "%s: head_dim=%d (64 or 128)", who, p.head_dim);
        if (p.cache_dtype != FSTA_F16 && p.cache_dtype != FSTA_BF16 && p.cache_dtype != FSTA_FP8)
            return fail(FSTA_EINVAL, "%s: cache_dtype=%d", who, p.cache_dtype);
        if (p.kv_heads <= 0) return fail(FSTA_EINVAL, "%s: kv_heads=%d", who, p.kv_heads);
        if (p.kv_heads > 16384) return fail(FSTA_EUNSUPPORTED, "%s: kv_heads=%d (at most 16384)", who, p.kv_heads);
        if (p.kv_heads != q.kv_heads || p.head_dim != q.head_dim || p.cache_dtype != q.cache_dtype)
            return fail(FSTA_EINVAL, "%s: layer %d goes to pools of another kv_heads, head_dim or cache_dtype", who, l);
        for (const fsta_paged_pool* x : {&p, &q}) {
            if (num_pages > 0 && (!x->k || !x->v)) return fail(FSTA_EINVAL, "%s: null pointer", who);
            if (misaligned(x->k, 16) || misaligned(x->v, 16)) return fail(FSTA_EINVAL, "%s: the cache must be 16-byte aligned", who);
            if (p.cache_dtype == FSTA_FP8 && num_pages > 0 && (!x->k_exponent || !x->v_exponent)) return fail(FSTA_EINVAL, "%s: null pointer", who);
        }
    }
    return FSTA_OK;
}

// The next layers that a launch takes
int32_t fill(Layers* to, const fsta_paged_pool* pools, const fsta_paged_pool* into, int32_t first, int32_t layers, int* most_heads, int64_t* most_units) {
    const int32_t n = layers - first < kMaxLayers ? layers - first : kMaxLayers;
    *most_heads = 0;
    *most_units = 0;
    for (int32_t i = 0; i < n; ++i) {
        const fsta_paged_pool &p = pools[first + i], &q = into[first + i];
        const bool fp8 = p.cache_dtype == FSTA_FP8;
        to->at[i] = Layer{{static_cast<uint8_t*>(p.k), static_cast<uint8_t*>(p.v)}, {fp8 ? p.k_exponent : nullptr, fp8 ? p.v_exponent : nullptr},
                          {static_cast<uint8_t*>(q.k), static_cast<uint8_t*>(q.v)}, {fp8 ? q.k_exponent : nullptr, fp8 ? q.v_exponent : nullptr}};
        to->heads[i] = (uint16_t)p.kv_heads;
        to->lanes[i] = (uint16_t)(p.head_dim * (fp8 ? 1 : 2) / 16);
        if (p.kv_heads > *most_heads) *most_heads = p.kv_heads;
        if ((int64_t)p.kv_heads * to->lanes[i] > *most_units) *most_units = (int64_t)p.kv_heads * to->lanes[i];
    }
    return n;
}

// Copies of whole pages, or of the listed tails; at most `most` of the latter
int launch_copies(const CopyArgs& a, int32_t most, int32_t most_groups, const fsta_paged_pool* pools, const fsta_paged_pool* into, int32_t layers,
                  hipStream_t stream) {
    for (int32_t first = 0; first < layers; first += kMaxLayers) {
        Layers l;
        int heads;
        int64_t units;
        const int32_t n = fill(&l, pools, into, first, layers, &heads, &units);
        const int64_t pieces = ((units << a.page_shift) + kPiece - 1) / kPiece;
        const unsigned z = (unsigned)(pieces < 1024 ? pieces : 1024), y = (unsigned)(2 * n);
        int64_t x = most;
        if (x * y * z > most_groups) x = most_groups / ((int64_t)y * z) > 1 ? most_groups / ((int64_t)y * z) : 1;
        if (a.list) hipLaunchKernelGGL((copy_pages_kernel<true>), dim3((unsigned)x, y, z), dim3(kThreads), 0, stream, a, l);
        else hipLaunchKernelGGL((copy_pages_kernel<false>), dim3((unsigned)x, y, z), dim3(kThreads), 0, stream, a, l);
        FSTA_HIP_OK(hipGetLastError());
    }
    return FSTA_OK;
}

constexpr size_t kAlign = 16;
constexpr int32_t kMaxRows = 1 << 24;     // pairs of pages
constexpr int32_t kMaxSequences = 1 << 16;            // (each looks at what those before it want)
size_t rounded(size_t bytes) { return (bytes + kAlign - 1) / kAlign * kAlign; }

size_t table_workspace(int64_t rows, int64_t width, int64_t num_pages, TableArgs* a, void* at) {
    const size_t groups = (size_t)((num_pages + kGroup - 1) / kGroup);
    size_t offset = 0;
    const auto take = [&](size_t bytes) {
        uint8_t* p = at ? static_cast<uint8_t*>(at) + offset : nullptr;
        offset += rounded(bytes);
        return p;
    };
    TableArgs none = {};
    if (!a) a = &none;
    a->listed = reinterpret_cast<int32_t*>(take(sizeof(int32_t)));
    a->list = reinterpret_cast<Copy*>(take(sizeof(Copy) * (size_t)rows));
    a->need = reinterpret_cast<int32_t*>(take(sizeof(int32_t) * (size_t)rows));
    a->group_free = reinterpret_cast<int32_t*>(take(sizeof(int32_t) * groups));
    a->free_bits = reinterpret_cast<uint32_t*>(take(sizeof(uint32_t) * groups * (kGroup / 32)));
    a->row_lens = reinterpret_cast<int32_t*>(take(sizeof(int32_t) * (size_t)rows));
    a->rows = reinterpret_cast<int32_t*>(take(sizeof(int32_t) * (size_t)rows * (size_t)width));
    return offset;
}

template <bool FORK> int launch_table(const TableArgs& a, const fsta_paged_pool* pools, int32_t layers, hipStream_t stream) {
    const int64_t rows = FORK ? a.pairs : a.batch, groups = ((int64_t)a.num_pages + kGroup - 1) / kGroup;
    const auto blocks = [](int64_t waves) { return dim3((unsigned)(waves < 65536 * kWaves ? (waves + kWaves - 1) / kWaves : 65536)); };
    hipLaunchKernelGGL((survey_kernel<FORK>), blocks(rows + groups), dim3(kThreads), 0, stream, a);
    hipLaunchKernelGGL((assign_kernel<FORK>), blocks(rows), dim3(kThreads), 0, stream, a);
    FSTA_HIP_OK(hipGetLastError());
    CopyArgs c = {};
    c.list = a.list;
    c.listed = a.listed;
    c.num_pages = c.into_pages = a.num_pages;
    c.page_shift = a.page_shift;
    return launch_copies(c, (int32_t)rows, FORK ? 65536 : 512, pools, pools, layers, stream);
}

int check_table(const char* who, int32_t batch, int32_t width, int32_t page_size, const void* refs, const void* table, const void* lens,
                int32_t num_pages, const void* missing, bool any) {
    if (batch < 0 || width < 0) return fail(FSTA_EINVAL, "%s: batch=%d width=%d", who, batch, width);
    if ((int64_t)width * page_size > 0x7fffffc0ll) return fail(FSTA_EUNSUPPORTED, "%s: %d pages of %d keys in a sequence", who, width, page_size);
    // (pages wanted are counted over the batch in 31 bits)
    if (batch > kMaxSequences || (int64_t)batch * width > INT32_MAX) return fail(FSTA_EUNSUPPORTED, "%s: batch=%d width=%d", who, batch, width);
    if (any && ((num_pages > 0 && !refs) || (width > 0 && !table) || !lens || !missing)) return fail(FSTA_EINVAL, "%s: null pointer", who);
    if (misaligned(refs, 4) || misaligned(table, 4) || misaligned(lens, 4) || misaligned(missing, 4))
        return fail(FSTA_EINVAL, "%s: refs, page_table, lens and missing must be 4-byte aligned", who);
    return FSTA_OK;
}

}  // namespace
}  // namespace fsta

using namespace fsta;

extern "C" int fsta_compact_paged_kv(const fsta_paged_pool* pools, int32_t layers, int32_t num_pages, int32_t page_size, const int32_t* path,
                                     int32_t max_path, const int32_t* counts, const int32_t* page_table, const int32_t* kv_lens,
                                     const int32_t* q_starts, int32_t batch, int32_t width, int32_t* new_lens, void* stream) {
    const char* who = "fsta_compact_paged_kv";
    int rc = check_pools(who, pools, pools, layers, num_pages, page_size);
    if (rc != FSTA_OK) return rc;
    if (batch < 0 || width < 0 || max_path < 0) return fail(FSTA_EINVAL, "%s: batch=%d width=%d max_path=%d", who, batch, width, max_path);
    if ((int64_t)width * page_size > 0x7fffffc0ll) return fail(FSTA_EUNSUPPORTED, "%s: %d pages of %d keys in a sequence", who, width, page_size);
    if (batch == 0) return FSTA_OK;
    if ((max_path > 0 && !path) || !counts || (width > 0 && !page_table) || !kv_lens || !q_starts || !new_lens) return fail(FSTA_EINVAL, "%s: null pointer", who);
    if (misaligned(path, 4) || misaligned(counts, 4) || misaligned(page_table, 4) || misaligned(kv_lens, 4) || misaligned(q_starts, 4) || misaligned(new_lens, 4))
        return fail(FSTA_EINVAL, "%s: path, counts, page_table, kv_lens, q_starts and new_lens must be 4-byte aligned", who);
    if (batch > kMaxSequences) return fail(FSTA_EUNSUPPORTED, "%s: batch=%d", who, batch);
    // rows move in place: of two workgroups with the same pool one would read what the other has moved
    for (int32_t l = 0; l < layers && num_pages > 0; ++l) {
        bool twice = pools[l].k == pools[l].v;
        for (int32_t i = 0; i < l; ++i)
            twice |= (pools[i].k == pools[l].k) | (pools[i].v == pools[l].v) | (pools[i].k == pools[l].v) | (pools[i].v == pools[l].k);
        if (twice) return fail(FSTA_EINVAL, "%s: layer %d has a pool that is there twice", who, l);
    }
    const CompactArgs a{path, counts, page_table, kv_lens, q_starts, new_lens, max_path, batch, width, num_pages, shift_of(page_size)};
    for (int32_t first = 0; first < layers; first += kMaxLayers) {
        Layers l;
        int heads;
        int64_t units;
        const int32_t n = fill(&l, pools, pools, first, layers, &heads, &units);
        const unsigned y = (unsigned)((heads + kWaves - 1) / kWaves);
        hipLaunchKernelGGL(compact_kernel, dim3((unsigned)(2 * n), y < 1024 ? y : 1024, (unsigned)(batch < 1024 ? batch : 1024)), dim3(kThreads), 0,
                           static_cast<hipStream_t>(stream), a, l);
        FSTA_HIP_OK(hipGetLastError());
    }
    return FSTA_OK;
}

extern "C" int fsta_copy_pages(const fsta_paged_pool* pools, const fsta_paged_pool* into, int32_t layers, int32_t num_pages, int32_t into_pages,
                               int32_t page_size, const int32_t* sources, const int32_t* targets, int32_t pairs, void* stream) {
    const char* who = "fsta_copy_pages";
    int rc = check_pools(who, pools, into, layers, num_pages, page_size);
    if (rc != FSTA_OK) return rc;
    if (into_pages < 0 || pairs < 0) return fail(FSTA_EINVAL, "%s: into_pages=%d pairs=%d", who, into_pages, pairs);
    if (pairs > kMaxRows) return fail(FSTA_EUNSUPPORTED, "%s: pairs=%d", who, pairs);
    if (pairs == 0 || num_pages == 0 || into_pages == 0) return FSTA_OK;
    if (!sources || !targets) return fail(FSTA_EINVAL, "%s: null pointer", who);
    if (misaligned(sources, 4) || misaligned(targets, 4)) return fail(FSTA_EINVAL, "%s: sources and targets must be 4-byte aligned", who);
    CopyArgs c = {};
    c.sources = sources;
    c.targets = targets;
    c.pairs = pairs;
    c.num_pages = num_pages;
    c.into_pages = into_pages;
    c.page_shift = shift_of(page_size);
    return launch_copies(c, pairs, 1 << 20, pools, into, layers, static_cast<hipStream_t>(stream));
}

extern "C" size_t fsta_fit_pages_workspace_bytes(int32_t batch, int32_t num_pages) {
    return batch < 0 || num_pages < 0 ? 0 : table_workspace(batch, 0, num_pages, nullptr, nullptr);
}

extern "C" int fsta_fit_pages(const fsta_paged_pool* pools, int32_t layers, int32_t num_pages, int32_t page_size, int32_t* refs, int32_t* page_table,
                              const int32_t* lens, int32_t batch, int32_t width, int32_t* missing, void* workspace, size_t workspace_bytes,
                              void* stream) {
    const char* who = "fsta_fit_pages";
    int rc = check_pools(who, pools, pools, layers, num_pages, page_size);
    if (rc != FSTA_OK) return rc;
    rc = check_table(who, batch, width, page_size, refs, page_table, lens, num_pages, missing, batch > 0);
    if (rc != FSTA_OK) return rc;
    if (batch == 0) return FSTA_OK;
    TableArgs a = {};
    if (!workspace || misaligned(workspace, kAlign) || workspace_bytes < table_workspace(batch, 0, num_pages, &a, workspace))
        return fail(FSTA_EINVAL, "%s: workspace of %zu bytes (%zu needed, 16-byte aligned)", who, workspace_bytes, fsta_fit_pages_workspace_bytes(batch, num_pages));
    a.refs = refs;
    a.table = page_table;
    a.missing = missing;
    a.lens = lens;
    a.batch = batch;
    a.width = width;
    a.num_pages = num_pages;
    a.page_shift = shift_of(page_size);
    return launch_table<false>(a, pools, layers, static_cast<hipStream_t>(stream));
}

extern "C" size_t fsta_fork_pages_workspace_bytes(int32_t pairs, int32_t width, int32_t num_pages) {
    return pairs < 0 || width < 0 || num_pages < 0 ? 0 : table_workspace(pairs, width, num_pages, nullptr, nullptr);
}

extern "C" int fsta_fork_pages(const fsta_paged_pool* pools, int32_t layers, int32_t num_pages, int32_t page_size, int32_t* refs, int32_t* page_table,
                               int32_t* lens, int32_t batch, int32_t width, const int32_t* sources, const int32_t* targets, int32_t pairs,
                               int32_t* missing, void* workspace, size_t workspace_bytes, void* stream) {
    const char* who = "fsta_fork_pages";
    int rc = check_pools(who, pools, pools, layers, num_pages, page_size);
    if (rc != FSTA_OK) return rc;
    if (pairs < 0) return fail(FSTA_EINVAL, "%s: pairs=%d", who, pairs);
    if (pairs > kMaxSequences) return fail(FSTA_EUNSUPPORTED, "%s: pairs=%d", who, pairs);
    rc = check_table(who, batch, width, page_size, refs, page_table, lens, num_pages, missing, pairs > 0 && batch > 0);
    if (rc != FSTA_OK) return rc;
    if (pairs == 0) return FSTA_OK;
    if (!sources || !targets || !missing) return fail(FSTA_EINVAL, "%s: null pointer", who);
    if (misaligned(sources, 4) || misaligned(targets, 4)) return fail(FSTA_EINVAL, "%s: sources and targets must be 4-byte aligned", who);
    TableArgs a = {};
    if (!workspace || misaligned(workspace, kAlign) || workspace_bytes < table_workspace(pairs, width, num_pages, &a, workspace))
        return fail(FSTA_EINVAL, "%s: workspace of %zu bytes (%zu needed, 16-byte aligned)", who, workspace_bytes, fsta_fork_pages_workspace_bytes(pairs, width, num_pages));
    a.refs = refs;
    a.table = page_table;
    a.missing = missing;
    a.slot_lens = lens;
    a.sources = sources;
    a.targets = targets;
    a.batch = batch;
    a.width = width;
    a.num_pages = num_pages;
    a.page_shift = shift_of(page_size);
    a.pairs = pairs;
    return launch_table<true>(a, pools, layers, static_cast<hipStream_t>(stream));
}
