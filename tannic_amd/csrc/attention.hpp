// Problem description shared by the attention kernels: queries of several sequences over keys and values that lie in the pages of a
// cache, or in one tensor per batch.
#pragma once

#include "cache.hpp"
#include "meeting.hpp"

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
    FastDiv group_div;
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

// Where key j of sequence s is said to lie: the number of its page (dense: of the sequence) and its row there.  Nothing here waits for the number: whether there is such
// a page is asked (page_exists) when the key is.
template <bool PAGED>
__device__ inline uint32_t page_of(const AttentionProblem& p, uint32_t s, uint32_t j, uint32_t& row) {
    if constexpr (PAGED) {
        uint32_t column;
        p.page_div.divmod(j, column, row);
        return static_cast<uint32_t>(p.table[static_cast<int64_t>(s) * p.table_row + column]);
    } else {
        row = j;
        return s;
    }
}
__device__ inline bool page_exists(const AttentionProblem& p, uint32_t page) { return page < p.pages; }

// Both at once.
template <bool PAGED>
__device__ inline bool place_of(const AttentionProblem& p, uint32_t s, uint32_t j, int64_t& page, uint32_t& row) {
    const uint32_t id = page_of<PAGED>(p, s, j, row);
    page = id;
    return page_exists(p, id);
}

__device__ inline int64_t query_offset(const AttentionProblem& p, uint32_t s, const Span& span, uint32_t i, uint32_t head) {
    // (pages: q_batch is 0 and tokens count through; dense: tokens count within the sequence)
    const int64_t token = p.starts ? static_cast<int64_t>(span.begin) + i : static_cast<int64_t>(i);
    return static_cast<int64_t>(s) * p.q_batch + token * p.q_token + static_cast<int64_t>(head) * p.q_head;
}

// ---- sharing the keys of all rows between blocks -------------------------------------------------------------------------------
// A group is a tile of rows of one sequence that read the same keys (a kv head's); its keys come in units.  All groups' units, one group
// after the other, are dealt to the blocks in equal runs, so that every block reads as many keys as the next whatever the lengths are; a
// group that a run's end cuts is put together from its blocks' partial results by the last of them.  Lengths are known on the device only:
// every wavefront works the runs out for itself, 64 sequences at a time.
struct Group {
    uint32_t s, tile, head;      // of kv_heads x `tiles` in the sequence, tiles innermost
    Span span;
    uint32_t tiles, units;       // units of each of the sequence's groups
    uint32_t first;              // the group's first unit among all
};

// Units of all of a sequence's groups.
template <bool PAGED, int ROWS, int UNIT>
__device__ inline uint32_t sequence_units(const AttentionProblem& p, const Span& span, uint32_t& tiles, uint32_t& units) {
    if (span.count == 0) return tiles = units = 0;
    tiles = (span.count * p.group + (ROWS - 1)) / ROWS;
    const uint32_t keys = keys_seen(p, span, span.count - 1);
    units = keys ? (keys + (UNIT - 1)) / UNIT : 1;      // (rows without keys are written all the same)
    return tiles * p.kv_heads * units;
}

// The host sees to it that there are fewer units than this; sequences that overlap, against what the starts may hold, can make more of them,
// and then nothing is done.
constexpr uint32_t kMostUnits = (1u << 31) - 1;
__device__ inline uint32_t sum_units(uint32_t a, uint32_t b) { return a + b < kMostUnits ? a + b : kMostUnits; }

__device__ inline uint32_t lanes_sum_before(uint32_t v, uint32_t& total) {
    const uint32_t lane = threadIdx.x % 64;
    uint32_t upto = v;
#pragma unroll
    for (uint32_t step = 1; step < 64; step *= 2) {
        const uint32_t below = __shfl_up(upto, step);
        if (lane >= step) upto = sum_units(upto, below);
    }
    total = __builtin_amdgcn_readlane(upto, 63);
    return upto - v;
}

// The run of this block: units from .. to, and the group that holds the first; false: there is none.
struct Run {
    uint32_t block, per, from, to;      // the number among the runs
};

// Lane l looks after the sequences l * each .. + each (one of up to 64): f(span) is what a sequence counts for; how much the lane's count for, together.  (64 at a time, twice, one
// after the other: 82 us for a token of 512 sequences behind 128, 32 / 8 heads of 128; so: 76.)
template <bool PAGED, class F>
__device__ inline uint32_t lanes_share(const AttentionProblem& p, uint32_t each, F&& f) {
    const uint32_t from = threadIdx.x % 64 * each;
    uint32_t mine = 0;
#pragma unroll 4
    for (uint32_t i = 0; i < each; ++i) {
        const bool there = from + i < p.sequences;
        Span span = span_of<PAGED>(p, there ? from + i : p.sequences - 1);
        span.count = there ? span.count : 0;
        mine = sum_units(mine, f(span));
    }
    return mine;
}

// The sequence that counts for place `at` of all, and how much those before it count for, from what a lane's sequences count for and those of the lanes before; false: there is none.
template <bool PAGED, class F>
__device__ inline bool sequence_at(const AttentionProblem& p, uint32_t each, uint32_t mine, uint32_t before, uint32_t at, F&& f, uint32_t& s, uint32_t& first) {
    const uint32_t lane = threadIdx.x % 64;
    uint64_t here = __ballot(before <= at && at - before < mine);
    if (here == 0) return false;
    int l = __builtin_ctzll(here);
    s = l * each;
    first = __builtin_amdgcn_readlane(before, l);
    if (each == 1) return true;
    const uint32_t end = s + each < p.sequences ? s + each : p.sequences;
    for (; s < end; s += 64) {
        Span span = span_of<PAGED>(p, s + lane < end ? s + lane : end - 1);
        span.count = s + lane < end ? span.count : 0;
        mine = f(span);
        uint32_t total;
        before = first + lanes_sum_before(mine, total);
        here = __ballot(before <= at && at - before < mine);
        if (here) {
            l = __builtin_ctzll(here);
            s += l;
            first = __builtin_amdgcn_readlane(before, l);
            return true;
        }
        first += total;
    }
    return false;
}

template <bool PAGED, int ROWS, int UNIT>
__device__ inline bool run_of_block(const AttentionProblem& p, uint32_t blocks, Run& run, Group& g) {
    const uint32_t each = (p.sequences + 63) / 64;
    const auto units_of = [&](const Span& span) -> uint32_t {
        uint32_t tiles, units;
        return sequence_units<PAGED, ROWS, UNIT>(p, span, tiles, units);
    };
    const uint32_t mine = lanes_share<PAGED>(p, each, units_of);
    uint32_t all;
    const uint32_t before = lanes_sum_before(mine, all);
    if (all == kMostUnits) return false;
    run.per = (all + blocks - 1) / blocks;
    // Blocks go round the eight dies (blocks is a multiple of eight).  Neighbouring runs belong on one die where its L2 can serve several tiles with the same keys (fp32, 700 tokens
    // of 8 sequences' 16 heads of 64 over 500 to 2000 states 455 us apart and 396 together, 16 tokens of 8 sequences behind 4096 172 and 138), but not short runs (prompts of 17 to
    // 100 tokens 10.9 and 12.4) or single tiles (a token over 1024 states 12.7 and 15.0, 4 tokens of 16 sequences behind 8192, bf16, 111 and 114).
    run.block = blockIdx.x;
    if (run.per >= 8 && p.tokens * p.group > ROWS * p.sequences) {
        const uint32_t of_die = ((all + run.per - 1) / run.per + 7) / 8;
        if (blockIdx.x / 8 >= of_die) return false;
        run.block = blockIdx.x % 8 * of_die + blockIdx.x / 8;
    }
    run.from = run.block * run.per;      // (blocks * per < all + blocks)
    if (run.from >= all) return false;
    run.to = run.from + run.per < all ? run.from + run.per : all;
    if (!sequence_at<PAGED>(p, each, mine, before, run.from, units_of, g.s, g.first)) return false;
    g.span = span_of<PAGED>(p, g.s);
    sequence_units<PAGED, ROWS, UNIT>(p, g.span, g.tiles, g.units);
    const uint32_t number = (run.from - g.first) / g.units;
    g.first += number * g.units;
    g.head = number / g.tiles;
    g.tile = number % g.tiles;
    return true;
}

// The group behind g (there is one).
template <bool PAGED, int ROWS, int UNIT>
__device__ inline void next_group(const AttentionProblem& p, Group& g) {
    g.first += g.units;
    if (++g.tile < g.tiles) return;
    g.tile = 0;
    if (++g.head < p.kv_heads) return;
    g.head = 0;
    while (++g.s < p.sequences) {
        g.span = span_of<PAGED>(p, g.s);
        if (sequence_units<PAGED, ROWS, UNIT>(p, g.span, g.tiles, g.units)) return;
    }
}

// What a block leaves of a group it has a part of: ROWS x d sums, then every row's largest score (in units of log2) and sum of weights.
// A block has at most two such parts: of the group its run starts in, and of the one it ends in.
template <int ROWS> __host__ __device__ inline uint64_t partial_floats(uint32_t d) { return static_cast<uint64_t>(ROWS) * (d + 2); }

typedef float float4a __attribute__((ext_vector_type(4)));
typedef unsigned int uint4a __attribute__((ext_vector_type(4)));
typedef unsigned int uint2a __attribute__((ext_vector_type(2)));

// the largest / the sum over the lanes l, l ^ 16, l ^ 32, l ^ 48
__device__ inline float across_groups_max(float x) {
    uint2a r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    x = fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
    r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ inline float across_groups_sum(float x) {
    uint2a r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    x = __uint_as_float(r[0]) + __uint_as_float(r[1]);
    r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

template <class T> __device__ inline float4a rows_mfma(uint4a a, uint4a b, float4a c) {
    if constexpr (std::is_same_v<T, f16>) {
        typedef _Float16 V __attribute__((ext_vector_type(8)));
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(V, a), __builtin_bit_cast(V, b), c, 0, 0, 0);
    } else if constexpr (std::is_same_v<T, bf16>) {
        typedef __bf16 V __attribute__((ext_vector_type(8)));
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(V, a), __builtin_bit_cast(V, b), c, 0, 0, 0);
    } else {
        // four products of four: element j of both operands is the j-th
#pragma unroll
        for (int j = 0; j < 4; ++j) c = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(a[j]), __uint_as_float(b[j]), c, 0, 0, 0);
        return c;
    }
}

// two weights as the matrix pipe takes them
template <class T> __device__ inline uint32_t pack_weights(float x, float y) {
    typedef float float2a __attribute__((ext_vector_type(2)));
    if constexpr (std::is_same_v<T, bf16>) {
        typedef __bf16 V __attribute__((ext_vector_type(2)));
        return __builtin_bit_cast(uint32_t, __builtin_convertvector((float2a{x, y}), V));
    } else {
        typedef _Float16 V __attribute__((ext_vector_type(2)));
        return __builtin_bit_cast(uint32_t, __builtin_convertvector((float2a{x, y}), V));
    }
}

// Whether one of a register's two 16-bit values (a float) is infinite or NaN.
template <class T> __device__ inline bool not_finite(uint32_t x) {
    constexpr uint32_t E = std::is_same_v<T, f16> ? 0x7C00u : 0x7F80u;
    if constexpr (sizeof(T) == 4) return (x & 0x7F800000u) == 0x7F800000u;
    return (x & E) == E || ((x >> 16) & E) == E;
}

// The same register with those values 0.
template <class T> __device__ inline uint32_t finite_only(uint32_t x) {
    constexpr uint32_t E = std::is_same_v<T, f16> ? 0x7C00u : 0x7F80u;
    if constexpr (sizeof(T) == 4) return not_finite<T>(x) ? 0u : x;
    return ((x & E) == E ? 0u : x & 0xFFFFu) | (((x >> 16) & E) == E ? 0u : x & 0xFFFF0000u);
}

// The register's two 16-bit values times 0: NaN where they are infinite or NaN.
template <class T> __device__ inline uint32_t times_zero(uint32_t x) {
    constexpr uint32_t E = std::is_same_v<T, f16> ? 0x7C00u : 0x7F80u;
    return ((x & E) == E ? 0x7FFFu : 0u) | (((x >> 16) & E) == E ? 0x7FFF0000u : 0u);
}

// fp16 weights are kept 2^8 times as large: those below 2^-22 of the largest lose bits first, not those below 2^-14
template <class T> constexpr float kWeightShift = std::is_same_v<T, f16> ? 8.0f : 0.0f;

// Partial results pass from block to block, and between the L2 caches of the dies, through the memory both see: stores and loads of device
// scope, which no cache in between keeps.  (A store has arrived when the wavefront's count of outstanding ones says so; a release and an
// acquire around plain accesses would write the die's whole L2 back and drop it: 10 us a call, one token behind 2048.)
__device__ inline void store_through(float* at, float x, float y) {
    const uint64_t bits = static_cast<uint64_t>(__float_as_uint(y)) << 32 | __float_as_uint(x);
    __hip_atomic_store(reinterpret_cast<uint64_t*>(at), bits, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ inline void load_through(const float* at, float& x, float& y) {
    const uint64_t bits = __hip_atomic_load(reinterpret_cast<const uint64_t*>(at), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    x = __uint_as_float(static_cast<uint32_t>(bits));
    y = __uint_as_float(static_cast<uint32_t>(bits >> 32));
}
__device__ inline void load_through(const float* at, float4a& v) {
    float x, y, z, w;
    load_through(at, x, y);
    load_through(at + 2, z, w);
    v = float4a{x, y, z, w};
}

// How many blocks of a group have left their part: counts on a stream, 0 between calls.
constexpr uint32_t kAttentionArrivals = 1024;
int attention_arrivals(hipStream_t stream, uint32_t*& arrivals);

// The kernels of 16-byte pieces.  UNSUPPORTED_DTYPE: nothing was done, another kernel has to take the operands.
int attention_rows(int dtype, const AttentionProblem& p, const void* q, const void* k, const void* v, void* out, hipStream_t stream);
int attention_tile(int dtype, const AttentionProblem& p, const void* q, const void* k, const void* v, void* out, hipStream_t stream);

inline bool aligned_to(const void* p, size_t bytes) { return reinterpret_cast<uintptr_t>(p) % bytes == 0; }

}  // namespace th
