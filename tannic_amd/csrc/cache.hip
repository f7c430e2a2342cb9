// Writing into a paged cache (tannic_hip_append_pages) and copying its pages (tannic_hip_copy_pages).
// A Tannic program keeps one dense cache per sequence and writes it by slice assignment, one call for each; sequences that come
// and go, or share a beginning, need pages.  Both operators only move bytes: HBM-bound, launch-bound for few tokens.
#include <algorithm>
#include <new>
#include <vector>

#include "cache.hpp"

namespace th {

// ---- new tokens into their pages --------------------------------------------------------------------------------------------
struct AppendProblem {
    PageTable pages;
    uint32_t tokens, heads, d;              // heads: of q, 0 without it
    uint32_t rows, side;                    // a token's rows of q, k and v; how many of them a block holds side by side
    FastDiv d_vectors_div;                  // vectors of a row
    int64_t q_token, q_head, k_token, k_head, v_token, v_head;
    int64_t kc_page, kc_head, kc_token, vc_page, vc_head, vc_token;
    uint32_t positions;                     // rows of the tables of angles, 0: nothing is rotated
    bool wide_angles;                       // they are float, not of the operands' type
};

// (a vector of 16 bytes lies at a multiple of them; a pair wherever an element may)
template <class T, int N, bool WHOLE>
struct alignas(WHOLE ? 16 : sizeof(T)) Few {
    T v[N];
};

// blockIdx.x: a token, blockIdx.y: ROUNDS times as many of its rows as 256 threads hold side by side.  A thread has the same elements of all its rows, so that the angles
// are loaded once (before: with every vector, 49.5 us for 7500 tokens of 32 + 2 * 8 heads of 128; so: 38, 4.9 TB/s; 32 tokens 3.4), and asks for the rows before the lengths and the table
// have said where they go.  The pairs (2i, 2i + 1) turn in fp32 (float64: in double) and are rounded once, as tannic_hip_rope does.
template <class T, int VEC, bool WHOLE, int ROUNDS>
__global__ __launch_bounds__(256) void append_pages_kernel(AppendProblem p, const T* q, const T* k, const T* v, const void* cs, const void* sn, T* keys, T* values, T* turned) {
    using A = std::conditional_t<std::is_same_v<T, double>, double, float>;
    using Vector = Few<T, VEC, WHOLE>;
    constexpr int PAIRS = VEC > 1 ? VEC / 2 : 1;
    const uint32_t token = blockIdx.x;
    uint32_t beside, e;
    p.d_vectors_div.divmod(threadIdx.x, beside, e);
    e *= VEC;
    if (beside >= p.side) beside = p.rows;      // (threads over: no row)
    const uint32_t first = blockIdx.y * (p.side * ROUNDS) + beside;
    Vector x[ROUNDS];
#pragma unroll
    for (int r = 0; r < ROUNDS; ++r) {
        const uint32_t head = first + r * p.side < p.rows ? first + r * p.side : p.rows - 1;
        const T* const row = head < p.heads ? q + token * p.q_token + head * p.q_head
                             : head < p.heads + p.pages.kv_heads ? k + token * p.k_token + (head - p.heads) * p.k_head
                                                                 : v + token * p.v_token + (head - p.heads - p.pages.kv_heads) * p.v_head;
        x[r] = *reinterpret_cast<const Vector*>(row + e);
    }
    const uint32_t s = sequence_of(p.pages.starts, p.pages.sequences, token);
    const int32_t from = p.pages.starts[s], to = p.pages.starts[s + 1], before = p.pages.context[s];
    if (static_cast<int32_t>(token) < from || static_cast<int32_t>(token) >= to) return;      // no sequence's token
    // (from is at most the token's number; a negative one is taken as 0)
    const uint64_t position = static_cast<uint64_t>(before < 0 ? 0 : before) + (token - static_cast<uint32_t>(from < 0 ? 0 : from));
    bool held = position < p.pages.room;
    uint32_t column = 0, in_page = 0;
    int32_t page = -1;
    if (held) {
        p.pages.page_div.divmod(static_cast<uint32_t>(position), column, in_page);
        page = p.pages.table[static_cast<int64_t>(s) * p.pages.table_row + column];
        held = static_cast<uint32_t>(page) < p.pages.pages;
    }
    A c[PAIRS], n[PAIRS];
    const bool turns = VEC > 1 && p.positions > 0;
    if (turns) {
        const size_t at = static_cast<size_t>(position < p.positions ? position : p.positions - 1) * (p.d / 2) + e / 2;
        if (p.wide_angles) {
            const auto cv = *reinterpret_cast<const Few<float, PAIRS, false>*>(static_cast<const float*>(cs) + at), nv = *reinterpret_cast<const Few<float, PAIRS, false>*>(static_cast<const float*>(sn) + at);
#pragma unroll
            for (int u = 0; u < PAIRS; ++u) c[u] = cv.v[u], n[u] = nv.v[u];
        } else {
            const auto cv = *reinterpret_cast<const Few<T, PAIRS, false>*>(static_cast<const T*>(cs) + at), nv = *reinterpret_cast<const Few<T, PAIRS, false>*>(static_cast<const T*>(sn) + at);
#pragma unroll
            for (int u = 0; u < PAIRS; ++u) c[u] = static_cast<A>(widen(cv.v[u])), n[u] = static_cast<A>(widen(nv.v[u]));
        }
    }
#pragma unroll
    for (int r = 0; r < ROUNDS; ++r) {
        uint32_t head = first + r * p.side;
        if (head >= p.rows) return;
        if (turns && head < p.heads + p.pages.kv_heads) {
#pragma unroll
            for (int u = 0; u + 1 < VEC; u += 2) {
                const A even = static_cast<A>(widen(x[r].v[u])), odd = static_cast<A>(widen(x[r].v[u + 1]));
                x[r].v[u] = narrow<T>(even * c[u / 2] - odd * n[u / 2]);
                x[r].v[u + 1] = narrow<T>(even * n[u / 2] + odd * c[u / 2]);
            }
        }
        T* row;
        if (head < p.heads) row = turned + (static_cast<size_t>(token) * p.heads + head) * p.d;
        else if (!held) return;      // (the rows of q come first)
        else if (head < p.heads + p.pages.kv_heads) row = keys + page * p.kc_page + (head - p.heads) * p.kc_head + in_page * p.kc_token;
        else row = values + page * p.vc_page + (head - p.heads - p.pages.kv_heads) * p.vc_head + in_page * p.vc_token;
        *reinterpret_cast<Vector*>(row + e) = x[r];
    }
}

template <class T, int VEC, bool WHOLE>
int launch_append(AppendProblem& p, const void* q, const void* k, const void* v, const void* cs, const void* sn, void* keys, void* values, void* turned, hipStream_t stream) {
    const uint32_t vectors = p.d / VEC;
    p.rows = p.heads + 2 * p.pages.kv_heads;
    p.side = 256 / vectors;
    p.d_vectors_div = FastDiv(vectors);
    auto launch = [&](auto rounds) {
        constexpr int ROUNDS = decltype(rounds)::value;
        const dim3 grid(p.tokens, (p.rows + p.side * ROUNDS - 1) / (p.side * ROUNDS));
        if (grid.y > 65535) return refuse("append_pages: so many heads of this size are not supported");
        hipLaunchKernelGGL((append_pages_kernel<T, VEC, WHOLE, ROUNDS>), grid, dim3(256), 0, stream, p, static_cast<const T*>(q), static_cast<const T*>(k), static_cast<const T*>(v), cs, sn,
                           static_cast<T*>(keys), static_cast<T*>(values), static_cast<T*>(turned));
        return launch_status("append_pages_kernel");
    };
    // few tokens: a row per thread, on more blocks
    if (p.tokens * static_cast<uint64_t>(p.rows) * vectors < 256 * 1024) return launch(std::integral_constant<int, 1>{});
    return launch(std::integral_constant<int, 3>{});
}

// ---- pages to pages -----------------------------------------------------------------------------------------------------------
typedef uint32_t uint4c __attribute__((ext_vector_type(4)));
constexpr int kCopyDims = 4;      // dims in front of the pages, at most
struct CopyPlace {
    uint32_t lead[kCopyDims];     // extents in front of the pages
    int64_t lead_stride[kCopyDims], page_stride;     // bytes
    uint32_t units;               // vectors of a page
};
// the pages' numbers travel with the launch: nothing is uploaded, and a recorded launch keeps them
template <int N>
struct CopyPairs {
    int32_t source[N], target[N];
};

// One page (of one layer, keys or values) per blockIdx.y and z, a vector per thread (512 MB of pages past the caches, us with one / two / four: 195 / 199 / 201).
template <class V, int N, bool PAST>
__global__ __launch_bounds__(256) void copy_pages_kernel(CopyPlace p, CopyPairs<N> pairs, char* pool) {
    uint32_t rest = blockIdx.z;
    int64_t off = 0;
#pragma unroll
    for (int d = kCopyDims - 1; d >= 0; --d) {
        off += static_cast<int64_t>(rest % p.lead[d]) * p.lead_stride[d];
        rest /= p.lead[d];
    }
    const V* const from = reinterpret_cast<const V*>(pool + off + pairs.source[blockIdx.y] * p.page_stride);
    V* const to = reinterpret_cast<V*>(pool + off + pairs.target[blockIdx.y] * p.page_stride);
    const uint32_t at = blockIdx.x * 256 + threadIdx.x;
    if (at >= p.units) return;
    if constexpr (PAST) __builtin_nontemporal_store(__builtin_nontemporal_load(from + at), to + at);
    else to[at] = from[at];
}

constexpr uint64_t kCopyPast = uint64_t(64) << 20;      // bytes of a launch

template <class V, int N>
int launch_copy(CopyPlace p, uint64_t page_bytes, uint32_t leads, const int32_t* sources, const int32_t* targets, uint32_t count, char* pool, hipStream_t stream) {
    CopyPairs<N> pairs;
    std::memcpy(pairs.source, sources, count * sizeof(int32_t));
    std::memcpy(pairs.target, targets, count * sizeof(int32_t));
    p.units = static_cast<uint32_t>(page_bytes / sizeof(V));
    const dim3 grid((p.units + 255) / 256, count, leads);
    // A compaction goes past the caches (512 MB of pages 210 us through them, 195 past them); what a fork copies is read soon after (4.7 both ways).
    if (page_bytes * leads * count >= kCopyPast) hipLaunchKernelGGL((copy_pages_kernel<V, N, true>), grid, dim3(256), 0, stream, p, pairs, pool);
    else hipLaunchKernelGGL((copy_pages_kernel<V, N, false>), grid, dim3(256), 0, stream, p, pairs, pool);
    return launch_status("copy_pages_kernel");
}

constexpr uint32_t kFewPairs = 16, kManyPairs = 480;     // (a launch's arguments are 4 KB at most)

template <class V>
int launch_copy(const CopyPlace& p, uint64_t page_bytes, uint32_t leads, const int32_t* sources, const int32_t* targets, uint32_t count, char* pool, hipStream_t stream) {
    if (count <= kFewPairs) return launch_copy<V, kFewPairs>(p, page_bytes, leads, sources, targets, count, pool, stream);
    return launch_copy<V, kManyPairs>(p, page_bytes, leads, sources, targets, count, pool, stream);
}

// Copies one after another, as many per launch as do not touch each other.
int run_copies(const CopyPlace& p, uint64_t page_bytes, uint32_t leads, uint32_t pages, int grain, const int32_t* sources, const int32_t* targets, size_t count, char* pool, hipStream_t stream) {
    // bit 0: read by the launch being put together, bit 1: written by it (a few copies are compared with each other instead of marking pages)
    const bool marks = count > 64;
    std::vector<uint8_t> touched(marks ? pages : 0, 0);
    std::vector<int32_t> from, to;
    from.reserve(std::min<size_t>(count, kManyPairs));
    to.reserve(std::min<size_t>(count, kManyPairs));
    auto flush = [&]() -> int {
        if (from.empty()) return TANNIC_SUCCESS;
        const uint32_t n = static_cast<uint32_t>(from.size());
        int status;
        if (grain % 16 == 0) status = launch_copy<uint4c>(p, page_bytes, leads, from.data(), to.data(), n, pool, stream);
        else if (grain % 4 == 0) status = launch_copy<uint32_t>(p, page_bytes, leads, from.data(), to.data(), n, pool, stream);
        else status = launch_copy<uint8_t>(p, page_bytes, leads, from.data(), to.data(), n, pool, stream);
        for (uint32_t i = 0; marks && i < n; ++i) touched[from[i]] = touched[to[i]] = 0;
        from.clear();
        to.clear();
        return status;
    };
    for (size_t i = 0; i < count; ++i) {
        const int32_t a = sources[i], b = targets[i];
        if (a == b) continue;
        const bool meets = marks ? (touched[a] & 2) || touched[b]
                                 : std::find(to.begin(), to.end(), a) != to.end() || std::find(to.begin(), to.end(), b) != to.end() || std::find(from.begin(), from.end(), b) != from.end();
        if (from.size() == kManyPairs || meets) {
            if (int status = flush(); status != TANNIC_SUCCESS) return status;
        }
        if (marks) touched[a] |= 1, touched[b] |= 2;
        from.push_back(a);
        to.push_back(b);
    }
    return flush();
}

}  // namespace th

using namespace th;

extern "C" {

int tannic_hip_append_pages(const tannic_tensor_t* k, const tannic_tensor_t* v, const tannic_tensor_t* table, const tannic_tensor_t* starts, const tannic_tensor_t* context,
                            const tannic_tensor_t* cos, const tannic_tensor_t* sin, const tannic_tensor_t* q, tannic_tensor_t* keys, tannic_tensor_t* values, tannic_tensor_t* turned,
                            tannic_stream_t stream) {
    if (!k || !v || !table || !starts || !context || !keys || !values) return refuse("append_pages: a descriptor is missing");
    if (!cos != !sin || !q != !turned || (q && !cos)) return refuse("append_pages: cos and sin come together, q comes with them and with a place for the rotated queries");
    if (!have_storage(k, v, table, starts, context, cos, sin, q, keys, values, turned)) return TANNIC_ERROR;
    const int dtype = k->dtype;
    if (dtype != TANNIC_FLOAT16 && dtype != TANNIC_BFLOAT16 && dtype != TANNIC_FLOAT32 && dtype != TANNIC_FLOAT64) return TANNIC_UNSUPPORTED_DTYPE;
    if (v->dtype != dtype || keys->dtype != dtype || values->dtype != dtype || (q && (q->dtype != dtype || turned->dtype != dtype)) || table->dtype != TANNIC_INT32 ||
        starts->dtype != TANNIC_INT32 || context->dtype != TANNIC_INT32 || (cos && (cos->dtype != sin->dtype || (cos->dtype != dtype && cos->dtype != TANNIC_FLOAT32))))
        return TANNIC_UNSUPPORTED_DTYPE;
    AppendProblem p{};
    if (int status = describe_pages(keys, values, table, starts, context, p.pages); status != TANNIC_SUCCESS) return status;
    if (k->rank != 3 || !extents_equal(k, v) || k->shape.sizes[1] != keys->shape.sizes[1] || k->shape.sizes[2] != keys->shape.sizes[3])
        return refuse("append_pages: k and v [tokens, kv heads, d] with the cache's kv heads and d");
    if (q && (q->rank != 3 || q->shape.sizes[0] != k->shape.sizes[0] || q->shape.sizes[2] != k->shape.sizes[2] || !extents_equal(q, turned) || !rows_contiguous(turned)))
        return refuse("append_pages: q [tokens, heads, d] with the tokens and d of k, the rotated queries contiguous with q's shape");
    const size_t tokens = k->shape.sizes[0], d = k->shape.sizes[2], heads = q ? q->shape.sizes[1] : 0;
    if (d > 1 && (k->strides.sizes[2] != 1 || v->strides.sizes[2] != 1 || (q && q->strides.sizes[2] != 1))) return refuse("append_pages: the elements of a head lie one after the other");
    if (cos) {
        if (d % 2 != 0 || cos->rank != 2 || !extents_equal(cos, sin) || cos->shape.sizes[1] != d / 2 || cos->shape.sizes[0] == 0 || cos->shape.sizes[0] >= (1ull << 31) ||
            !rows_contiguous(cos) || !rows_contiguous(sin))
            return refuse("append_pages: cos and sin [positions, d/2], contiguous, for an even d");
    }
    if (tokens >= kMostBlocks || heads >= (1u << 16) || d > 256) return refuse("append_pages: 2^24 tokens, 2^16 heads or heads of more than 256 elements are not supported");
    if (tokens == 0 || d == 0 || heads + k->shape.sizes[1] == 0 || p.pages.sequences == 0) return TANNIC_SUCCESS;
    if (int status = on_device_of("append_pages: the operands live on a device", keys, values, k, v, table, starts, context, cos, sin, q, turned); status != TANNIC_SUCCESS) return status;
    p.tokens = static_cast<uint32_t>(tokens);
    p.heads = static_cast<uint32_t>(heads);
    p.d = static_cast<uint32_t>(d);
    p.positions = cos ? static_cast<uint32_t>(cos->shape.sizes[0]) : 0;
    p.wide_angles = cos && cos->dtype == TANNIC_FLOAT32;
    // 16 bytes per access where every row of every operand starts at a multiple of them
    const size_t size = dtype_size(dtype);
    uint64_t grain = d * size;
    auto place = [&](const tannic_tensor_t* t, int first, int second, int64_t& a, int64_t& b) {
        a = stride_of(t, first), b = stride_of(t, second);
        grain |= reinterpret_cast<uintptr_t>(t->address) | static_cast<uint64_t>(a) * size | static_cast<uint64_t>(b) * size;
    };
    int64_t unused;
    place(k, 0, 1, p.k_token, p.k_head);
    place(v, 0, 1, p.v_token, p.v_head);
    if (q) place(q, 0, 1, p.q_token, p.q_head), place(turned, 0, 1, unused, unused);
    place(keys, 0, 1, p.kc_page, p.kc_head), place(keys, 2, 2, p.kc_token, unused);
    place(values, 0, 1, p.vc_page, p.vc_head), place(values, 2, 2, p.vc_token, unused);
    auto run = [&](auto tag) {
        using T = typename decltype(tag)::type;
        const void* const qa = q ? q->address : nullptr;
        void* const ta = turned ? turned->address : nullptr;
        const void *const ca = cos ? cos->address : nullptr, *const sa = sin ? sin->address : nullptr;
        if (grain % 16 == 0) return launch_append<T, 16 / sizeof(T), true>(p, qa, k->address, v->address, ca, sa, keys->address, values->address, ta, as_stream(stream));
        if (d % 2 == 0) return launch_append<T, 2, false>(p, qa, k->address, v->address, ca, sa, keys->address, values->address, ta, as_stream(stream));
        return launch_append<T, 1, false>(p, qa, k->address, v->address, ca, sa, keys->address, values->address, ta, as_stream(stream));
    };
    switch (dtype) {
        case TANNIC_FLOAT16: return run(type_tag<f16>{});
        case TANNIC_BFLOAT16: return run(type_tag<bf16>{});
        case TANNIC_FLOAT32: return run(type_tag<float>{});
        default: return run(type_tag<double>{});
    }
}

int tannic_hip_copy_pages(tannic_tensor_t* pool, tannic_stream_t stream, const int32_t* sources, const int32_t* targets, size_t count) {
    if (!pool || (count > 0 && (!sources || !targets))) return refuse("copy_pages: a descriptor or a list is missing");
    if (!have_storage(pool)) return TANNIC_ERROR;
    const size_t size = dtype_size(pool->dtype);
    if (size == 0) return TANNIC_UNSUPPORTED_DTYPE;
    if (pool->rank < 4) return refuse("copy_pages: a cache is [.., pages, kv heads, page, d]");
    const int at = pool->rank - 4;
    CopyPlace p{};
    int64_t page_elements = 1;
    uint64_t leads = 1;
    for (int d = pool->rank - 1; d > at; --d) {
        if (pool->shape.sizes[d] != 1 && pool->strides.sizes[d] != page_elements) return refuse("copy_pages: the elements of a page lie one after the other");
        page_elements *= static_cast<int64_t>(pool->shape.sizes[d]);
    }
    if (pool->shape.sizes[at] >= (1ull << 31) || static_cast<uint64_t>(page_elements) * size >= (1ull << 31)) return refuse("copy_pages: 2^31 pages, or pages of 2^31 bytes, or more are not supported");
    const uint32_t pages = static_cast<uint32_t>(pool->shape.sizes[at]);
    for (size_t i = 0; i < count; ++i)
        if (static_cast<uint32_t>(sources[i]) >= pages || static_cast<uint32_t>(targets[i]) >= pages) return refuse("copy_pages: a page's number is outside the cache");
    uint64_t grain = static_cast<uint64_t>(page_elements) * size | reinterpret_cast<uintptr_t>(pool->address);
    for (int d = 0; d < kCopyDims; ++d) p.lead[d] = 1;
    for (int d = 0; d < at; ++d) {
        const int to = kCopyDims - at + d;
        p.lead[to] = static_cast<uint32_t>(pool->shape.sizes[d]);
        p.lead_stride[to] = stride_of(pool, d) * static_cast<int64_t>(size);
        grain |= static_cast<uint64_t>(p.lead_stride[to]);
        leads *= pool->shape.sizes[d];
        if (leads >= (1u << 16)) return refuse("copy_pages: 2^16 layers or more in one call are not supported");
    }
    p.page_stride = stride_of(pool, at) * static_cast<int64_t>(size);
    if (pages > 1 && (p.page_stride < 0 ? -p.page_stride : p.page_stride) < page_elements * static_cast<int64_t>(size)) return refuse("copy_pages: pages lie apart from each other");
    grain |= static_cast<uint64_t>(p.page_stride);
    if (count == 0 || leads == 0 || page_elements == 0) return TANNIC_SUCCESS;
    if (int status = on_device_of("copy_pages: the cache lives on a device", static_cast<const tannic_tensor_t*>(pool)); status != TANNIC_SUCCESS) return status;
    try {
        return run_copies(p, static_cast<uint64_t>(page_elements) * size, static_cast<uint32_t>(leads), pages, static_cast<int>(grain & 15), sources, targets, count, static_cast<char*>(pool->address),
                          as_stream(stream));
    } catch (const std::bad_alloc&) {
        return refuse("copy_pages: out of host memory");
    }
}

}  // extern "C"
