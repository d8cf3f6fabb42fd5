// What the kernels of the paged KV cache share: the batch's description and how a token or a key finds its place in it.
#pragma once

#include "fsta_common.h"

namespace fsta {

// Cache [pages, kv_heads, page_size, head_dim]; sequence b's key p is row p % page_size of page page_table[b][p / page_size].
// Its new tokens are q_starts[b] .. q_starts[b + 1] - 1 of the packed tensors, its last positions below kv_lens[b].
struct PagedBatch {
    const int32_t* page_table;   // [batch, width]
    const int32_t* kv_lens;      // [batch]
    const int32_t* q_starts;     // [batch + 1], or null where there are no new tokens
    int32_t batch, width, num_pages, page_shift, kv_heads, tokens;
};

// What a sequence has, kept within what its tensors hold whatever the arrays say
struct SeqLens { int start, fresh, keys; };
__device__ __forceinline__ SeqLens seq_lens(const PagedBatch& p, int b) {
    SeqLens s{0, 0, 0};
    if (b < p.batch) {
        const int first = p.q_starts[b], last = p.q_starts[b + 1];
        s.start = min(max(first, 0), p.tokens);
        s.fresh = max(min(last, p.tokens) - s.start, 0);
        s.keys = (int)min((int64_t)max(p.kv_lens[b], 0), (int64_t)p.width << p.page_shift);
    }
    return s;
}

// Host-side checks the entry points share; `new_tokens`: whether q_starts is needed
int check_paged_batch(const char* who, const PagedBatch& p, int32_t page_size, int32_t head_dim, int32_t cache_dtype, bool new_tokens);

}  // namespace fsta
