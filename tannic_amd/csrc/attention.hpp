// Problem description shared by the attention kernels: queries of several sequences over keys and values that lie in the pages of a
// cache, or in one tensor per batch.
#pragma once

#include "cache.hpp"

namespace th {

// Row i of sequence s (query head h) is   out = sum_j w_j V[j] / sum_j w_j,   w_j = exp(scale * q . K[j] - max_j(scale * q . K[j])),
// over the keys j the row sees; head h reads the keys and values of head h / group.  A row that sees none (or whose scores are all
// -inf) is 0.
//   pages: sequence s has the tokens starts[s] .. starts[s + 1] of q and context[s] keys before them; its i-th token sees the keys up to
//          context[s] + i.  Key j lies in page table[s, j / page], row j % page; a page number outside the cache holds no key.
//   dense: every sequence has `per_sequence` tokens, each of which sees the first lengths[s] of `room` keys (all of them without lengths).
// Strides are in elements, those of the last dim are 1.
struct AttentionProblem {
    uint32_t sequences, per_sequence, tokens;   // tokens: rows of q and of the result over all sequences
    uint32_t heads, kv_heads, group, d;
    FastDiv heads_div, group_div;
    int64_t q_batch, q_token, q_head;
    int64_t k_page, k_head, k_token;
    int64_t v_page, v_head, v_token;
    const int32_t* starts;    // nullptr: dense
    const int32_t* context;
    const int32_t* lengths;
    const int32_t* table;
    int64_t table_row;
    uint32_t columns, pages, page;
    FastDiv page_div;
    uint32_t room;            // keys a sequence can have: columns * page, or the extent of the dense keys
    float scale;
};

struct Span {
    uint32_t begin, count;    // its tokens: rows of the result
    uint32_t keys;            // keys its first token sees
    uint32_t step;            // 1: every further token sees one more; 0: the same
};

// What a kernel may believe of the lengths in device memory: whatever they hold, no row outside q and no key outside the table follows from it.
template <bool PAGED>
__device__ inline Span span_of(const AttentionProblem& p, uint32_t s) {
    Span r;
    if constexpr (PAGED) {
        const int32_t total = static_cast<int32_t>(p.tokens);
        int32_t from = p.starts[s], to = p.starts[s + 1], before = p.context[s];
        from = from < 0 ? 0 : from > total ? total : from;
        to = to < from ? from : to > total ? total : to;
        r.begin = static_cast<uint32_t>(from);
        r.count = static_cast<uint32_t>(to - from);
        r.keys = before < 0 ? 1u : static_cast<uint32_t>(before) + 1u;    // (at most 2^31)
        r.keys = r.keys < p.room ? r.keys : p.room;
        r.step = 1;
    } else {
        r.begin = s * p.per_sequence;
        r.count = p.per_sequence;
        int32_t n = p.lengths ? p.lengths[s] : static_cast<int32_t>(p.room);
        r.keys = n < 0 ? 0u : static_cast<uint32_t>(n) < p.room ? static_cast<uint32_t>(n) : p.room;
        r.step = 0;
    }
    return r;
}

// keys the i-th token of the span sees (i < 2^31, keys <= room < 2^31)
__device__ inline uint32_t keys_seen(const AttentionProblem& p, const Span& s, uint32_t i) {
    const uint32_t n = s.keys + s.step * i;
    return n < p.room ? n : p.room;
}

// Where key j of sequence s lies: the page (or, dense, the sequence) and the row in it; false: nowhere.
template <bool PAGED>
__device__ inline bool place_of(const AttentionProblem& p, uint32_t s, uint32_t j, int64_t& page, uint32_t& row) {
    if constexpr (PAGED) {
        uint32_t column;
        p.page_div.divmod(j, column, row);
        const int32_t id = p.table[static_cast<int64_t>(s) * p.table_row + column];
        page = id;
        return static_cast<uint32_t>(id) < p.pages;
    } else {
        page = s;
        row = j;
        return true;
    }
}

__device__ inline int64_t query_offset(const AttentionProblem& p, uint32_t s, const Span& span, uint32_t i, uint32_t head) {
    // (pages: q_batch is 0 and tokens count through; dense: tokens count within the sequence)
    const int64_t token = p.starts ? static_cast<int64_t>(span.begin) + i : static_cast<int64_t>(i);
    return static_cast<int64_t>(s) * p.q_batch + token * p.q_token + static_cast<int64_t>(head) * p.q_head;
}

inline bool aligned_to(const void* p, size_t bytes) { return reinterpret_cast<uintptr_t>(p) % bytes == 0; }

}  // namespace th
