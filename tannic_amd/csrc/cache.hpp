// What the operators on a paged cache check and read of their descriptors.
//   keys, values [pages, kv heads, page, d]   a page holds `page` tokens; strides as they fall, the elements of a head one after the other
//   table   int32 [sequences, columns]        the page that holds tokens column * page .. of a sequence; a number outside the cache: none
//   starts  int32 [sequences + 1]             sequence s has the new tokens starts[s] .. starts[s + 1]
//   context int32 [sequences]                 tokens of a sequence before its new ones
#pragma once

#include "common.hpp"

namespace th {

inline bool extents_equal(const tannic_tensor_t* a, const tannic_tensor_t* b) {
    if (a->rank != b->rank) return false;
    for (int d = 0; d < a->rank; ++d)
        if (a->shape.sizes[d] != b->shape.sizes[d]) return false;
    return true;
}

inline bool rows_contiguous(const tannic_tensor_t* t) {
    int64_t step = 1;
    for (int d = t->rank - 1; d >= 0; --d) {
        if (t->shape.sizes[d] != 1 && t->strides.sizes[d] != step) return false;
        step *= static_cast<int64_t>(t->shape.sizes[d]);
    }
    return true;
}

inline int64_t stride_of(const tannic_tensor_t* t, int dim) { return t->shape.sizes[dim] == 1 ? 0 : t->strides.sizes[dim]; }

inline int refuse(const char* text) {
    set_error_text(text);
    return TANNIC_ERROR;
}

// All operands on one device, which is made the current one: a kernel's scratch and its launch belong to it.
template <class... Ts>
inline int on_device_of(const char* text, const tannic_tensor_t* first, const Ts*... others) {
    const auto on_device = [](const tannic_tensor_t* t) { return t == nullptr || t->environment.kind == TANNIC_DEVICE; };
    if (!on_device(first) || !(on_device(others) && ...)) return refuse(text);
    const int id = first->environment.resource.device.id;
    if (!((others == nullptr || others->environment.resource.device.id == id) && ...)) return TANNIC_INCOMPATIBLE_DEVICES;
    TH_TRY(hipSetDevice(id));
    return TANNIC_SUCCESS;
}

constexpr uint64_t kMostBlocks = 1u << 24;      // of 256 threads: a launch has fewer than 2^32 of those

struct PageTable {
    uint32_t sequences, columns, pages, page, kv_heads, room;
    const int32_t *starts, *context, *table;
    int64_t table_row;
    FastDiv page_div;
};

// `d` of the cache is keys->shape.sizes[3].
inline int describe_pages(const tannic_tensor_t* keys, const tannic_tensor_t* values, const tannic_tensor_t* table, const tannic_tensor_t* starts, const tannic_tensor_t* context,
                          PageTable& t) {
    if (keys->rank != 4 || !extents_equal(keys, values)) return refuse("paged cache: keys and values [pages, kv heads, page, d] of one shape");
    if (table->rank != 2 || starts->rank != 1 || context->rank != 1 || context->shape.sizes[0] != table->shape.sizes[0] || starts->shape.sizes[0] != table->shape.sizes[0] + 1)
        return refuse("paged cache: table [sequences, columns], starts [sequences + 1], context [sequences]");
    if (!rows_contiguous(starts) || !rows_contiguous(context) || (table->shape.sizes[1] > 1 && table->strides.sizes[1] != 1))
        return refuse("paged cache: starts, context and the rows of the table lie one element after the other");
    if (keys->shape.sizes[3] > 1 && (keys->strides.sizes[3] != 1 || values->strides.sizes[3] != 1)) return refuse("paged cache: the elements of a head lie one after the other");
    const size_t page = keys->shape.sizes[2], columns = table->shape.sizes[1], sequences = table->shape.sizes[0];
    if (page == 0) return refuse("paged cache: a page holds one token at least");
    if (page >= (1ull << 31) || columns >= (1ull << 31) || page * columns >= (1ull << 31) || keys->shape.sizes[0] >= (1ull << 31) || keys->shape.sizes[1] >= (1u << 16) ||
        sequences >= (1ull << 31))
        return refuse("paged cache: sequences of 2^31 tokens or more are not supported");
    t.sequences = static_cast<uint32_t>(sequences);
    t.columns = static_cast<uint32_t>(columns);
    t.pages = static_cast<uint32_t>(keys->shape.sizes[0]);
    t.kv_heads = static_cast<uint32_t>(keys->shape.sizes[1]);
    t.page = static_cast<uint32_t>(page);
    t.room = static_cast<uint32_t>(page * columns);
    t.starts = static_cast<const int32_t*>(starts->address);
    t.context = static_cast<const int32_t*>(context->address);
    t.table = static_cast<const int32_t*>(table->address);
    t.table_row = stride_of(table, 0);
    t.page_div = FastDiv(t.page);
    return TANNIC_SUCCESS;
}

// The sequence that token t belongs to, found by one wavefront: the last one that starts at or before it (every lane gets the same answer).  First among every so-many-th of
// them, then among those behind the one found (all of them, 64 at a time: 56 us to append a token to each of 4096 sequences, 32 / 8 heads of 128; so: 22).
__device__ inline uint32_t sequence_of(const int32_t* starts, uint32_t sequences, uint32_t t) {
    const uint32_t lane = threadIdx.x % 64, each = (sequences + 63) / 64;
    const auto started = [&](uint32_t s, uint32_t end) -> uint32_t { return __popcll(__ballot(s < end && starts[s] <= static_cast<int32_t>(t))); };
    const uint32_t found = started(lane * each, sequences);
    if (found == 0) return 0;
    const uint32_t from = (found - 1) * each, end = from + each < sequences ? from + each : sequences;
    if (each == 1) return from;
    uint32_t before = 0;
    for (uint32_t s0 = from; s0 < end; s0 += 64) before += started(s0 + lane, end);
    return before == 0 ? from : from + before - 1;
}

}  // namespace th
