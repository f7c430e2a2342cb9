// Attention of new tokens over the pages of a cache (tannic_hip_attend_pages) and over keys and values of another length
// (tannic_hip_attend): checks, the problem's description, the choice of a kernel, and the kernel for what the others do not take.
// A Tannic program writes it as products, a scale, a mask and a softmax, which need keys and values in one dense tensor and move the
// scores through memory four times; here a row's scores live in registers, and its softmax is folded key by key:
//   top' = max(top, s),  sum' = sum * exp(top - top') + exp(s - top'),  acc' = acc * exp(top - top') + exp(s - top') * V
#include <exception>
#include <map>
#include <mutex>

#include "attention.hpp"
#include "lanes.hpp"

namespace th {

struct SumOp {
    template <class A> __device__ static inline A combine(A x, A y) { return x + y; }
};
struct LargerOp {
    __device__ static inline float combine(float x, float y) { return fmaxf(x, y); }
    __device__ static inline double combine(double x, double y) { return fmax(x, y); }
};
__device__ inline float exponential(float x) { return expf(x); }
__device__ inline double exponential(double x) { return exp(x); }

constexpr uint32_t kAttentionHead = 256;   // elements of a head, at most

// Any type, alignment and head size: a block per query row, its four wavefronts taking 64 keys in turns; a lane has one key's score,
// then every lane adds the 64 values' elements lane, lane + 64, ...  Bound by its loads of the keys, a lane's own row each (a token of 32 heads of 128 behind 2048, bf16:
// 453 us, where the others take 11.6).
template <class T, bool PAGED>
__global__ __launch_bounds__(256) void attention_any_kernel(AttentionProblem p, const T* q, const T* k, const T* v, T* out) {
    using A = std::conditional_t<std::is_same_v<T, double>, double, float>;
    __shared__ A query[kAttentionHead], weight[4][64], part[4][kAttentionHead], tops[4], sums[4];
    const uint32_t lane = threadIdx.x % 64, wave = threadIdx.x / 64;
    const uint32_t token = blockIdx.x, head = blockIdx.y;
    const uint32_t s = PAGED ? sequence_of(p.starts, p.sequences, token) : token / p.per_sequence;
    const Span span = span_of<PAGED>(p, s);
    if (token < span.begin || token - span.begin >= span.count) return;   // no sequence's row: left as it is
    const uint32_t i = token - span.begin, seen = keys_seen(p, span, i), kv_head = p.group_div.div(head);
    const T* const row = q + query_offset(p, s, span, i, head);
    for (uint32_t e = threadIdx.x; e < p.d; e += 256) query[e] = static_cast<A>(widen(row[e]));
    __syncthreads();
    A top = -INFINITY, sum = 0, acc[4] = {};
    for (uint32_t j0 = wave * 64; j0 < seen; j0 += 256) {
        int64_t page;
        uint32_t in;
        const uint32_t j = j0 + lane;
        const bool live = j < seen && place_of<PAGED>(p, s, j, page, in);
        A score = -INFINITY;
        if (live) {
            const T* const key = k + page * p.k_page + in * p.k_token + kv_head * p.k_head;
            A dot = 0;
            for (uint32_t e = 0; e < p.d; ++e) dot += query[e] * static_cast<A>(widen(key[e]));
            score = dot * static_cast<A>(p.scale);
        }
        const A above = LargerOp::combine(top, wave_reduce<LargerOp>(score));
        const A base = above == static_cast<A>(-INFINITY) ? A(0) : above;    // (nothing finite yet: every weight below is 0)
        const A w = live ? exponential(score - base) : A(0), old = exponential(top - base);
        sum = sum * old + wave_reduce<SumOp>(w);
        top = above;
        weight[wave][lane] = w;
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
        __builtin_amdgcn_wave_barrier();
#pragma unroll
        for (int c = 0; c < 4; ++c) acc[c] *= old;
        uint64_t todo = __ballot(live);
        while (todo) {
            const uint32_t n = __builtin_ctzll(todo);
            todo &= todo - 1;
            place_of<PAGED>(p, s, j0 + n, page, in);
            const T* const value = v + page * p.v_page + in * p.v_token + kv_head * p.v_head;
            const A each = weight[wave][n];
#pragma unroll
            for (int c = 0; c < 4; ++c)
                if (lane + 64 * c < p.d) acc[c] += each * static_cast<A>(widen(value[lane + 64 * c]));
        }
        __builtin_amdgcn_wave_barrier();
    }
#pragma unroll
    for (int c = 0; c < 4; ++c) part[wave][lane + 64 * c] = acc[c];
    if (lane == 0) {
        tops[wave] = top;
        sums[wave] = sum;
    }
    __syncthreads();
    A above = tops[0];
    for (int w = 1; w < 4; ++w) above = LargerOp::combine(above, tops[w]);
    const A base = above == static_cast<A>(-INFINITY) ? A(0) : above;
    A total = 0, share[4];
    for (int w = 0; w < 4; ++w) {
        share[w] = exponential(tops[w] - base);
        total += sums[w] * share[w];
    }
    if (threadIdx.x < p.d) {
        A value = 0;
        for (int w = 0; w < 4; ++w) value += part[w][threadIdx.x] * share[w];
        out[(static_cast<size_t>(token) * p.heads + head) * p.d + threadIdx.x] = narrow<T>(total == A(0) ? A(0) : value / total);
    }
}

__global__ __launch_bounds__(256) void clear_arrivals_kernel(uint32_t* counts) { counts[blockIdx.x * 256 + threadIdx.x] = 0; }
static_assert(kAttentionArrivals % 256 == 0);

// The counts of blocks that have left their part of a group: one array per stream, 0 between calls.  It is cleared once, on a stream of its
// own, so that a first call that is being recorded does not leave the clearing to the replay; kept until the process ends.
int attention_arrivals(hipStream_t stream, uint32_t*& arrivals) try {
    static std::mutex mutex;
    static std::map<std::pair<int, hipStream_t>, uint32_t*> known;
    int device = 0;
    TH_TRY(hipGetDevice(&device));
    std::lock_guard<std::mutex> lock(mutex);
    const auto at = known.try_emplace({device, stream}, nullptr).first;
    if (at->second == nullptr) {
        void* counts = nullptr;
        hipStream_t own = nullptr;
        hipError_t err = hipMalloc(&counts, kAttentionArrivals * sizeof(uint32_t));
        if (err == hipSuccess) err = hipStreamCreateWithFlags(&own, hipStreamNonBlocking);
        if (err == hipSuccess) {
            hipLaunchKernelGGL(clear_arrivals_kernel, dim3(kAttentionArrivals / 256), dim3(256), 0, own, static_cast<uint32_t*>(counts));
            err = hipGetLastError();
        }
        if (err == hipSuccess) err = hipStreamSynchronize(own);
        if (own) (void)hipStreamDestroy(own);
        if (err != hipSuccess) {
            if (counts) (void)hipFree(counts);
            set_error("attention: counts of arrivals", __FILE__, __LINE__, err);
            return TANNIC_ERROR;
        }
        at->second = static_cast<uint32_t*>(counts);
    }
    arrivals = at->second;
    return TANNIC_SUCCESS;
} catch (const std::exception& e) {
    set_error_text(e.what());
    return TANNIC_ERROR;
}

template <class T>
int run_attention(const AttentionProblem& p, const void* q, const void* k, const void* v, void* out, hipStream_t stream) {
    const dim3 grid(p.tokens, p.heads);
    const T *pq = static_cast<const T*>(q), *pk = static_cast<const T*>(k), *pv = static_cast<const T*>(v);
    if (p.starts) hipLaunchKernelGGL((attention_any_kernel<T, true>), grid, dim3(256), 0, stream, p, pq, pk, pv, static_cast<T*>(out));
    else hipLaunchKernelGGL((attention_any_kernel<T, false>), grid, dim3(256), 0, stream, p, pq, pk, pv, static_cast<T*>(out));
    return launch_status("attention_any_kernel");
}

// The kernels that take every row of every operand in 16-byte pieces: tiles of 128 rows of the matrix pipe where the rows of a sequence and kv head are more on average than the
// 16 of the other's tiles, which reads the keys for each (8 tokens of 32 / 8 heads of 128 of 16 sequences behind 8192 173 us there and 109 here, 12 tokens 287 and 111; 4 tokens,
// one tile for both, 111 and 107, and of 8 sequences' 16 heads of 64 over 2000 states 15 and 20); more than 32 for heads above 128 (12 / 2 heads of 256: 5 tokens of 2 sequences
// behind 4096 37 and 52, of 16 66 and 66, 8 tokens of 16 83 and 67).
// The host does not know the lengths, so it is the average that counts: sequences of like lengths are on the right side, a chunk among many single tokens is not (190 tokens behind
// 8192 with 63 single tokens behind 512 to 8192: 366 us, where the chunk alone takes 74 and the single tokens 139).
int attention_pieces(int dtype, const AttentionProblem& p, const void* q, const void* k, const void* v, void* out, hipStream_t stream) {
    const int64_t size = static_cast<int64_t>(dtype_size(dtype));
    const int64_t grain = p.d | p.q_batch | p.q_token | p.q_head | p.k_page | p.k_head | p.k_token | p.v_page | p.v_head | p.v_token;
    if ((grain * size) % 16 != 0 || !aligned_to(q, 16) || !aligned_to(k, 16) || !aligned_to(v, 16) || !aligned_to(out, 4 * size)) return TANNIC_UNSUPPORTED_DTYPE;
    if (static_cast<uint64_t>(p.tokens) * p.group > (p.d > 128 ? 32ull : 16ull) * p.sequences) {
        if (int status = attention_tile(dtype, p, q, k, v, out, stream); status != TANNIC_UNSUPPORTED_DTYPE) return status;
    }
    return attention_rows(dtype, p, q, k, v, out, stream);
}

int run_attention(int dtype, const AttentionProblem& p, const void* q, const void* k, const void* v, void* out, hipStream_t stream) {
    if (int status = attention_pieces(dtype, p, q, k, v, out, stream); status != TANNIC_UNSUPPORTED_DTYPE) return status;
    switch (dtype) {
        case TANNIC_FLOAT16: return run_attention<f16>(p, q, k, v, out, stream);
        case TANNIC_BFLOAT16: return run_attention<bf16>(p, q, k, v, out, stream);
        case TANNIC_FLOAT32: return run_attention<float>(p, q, k, v, out, stream);
        case TANNIC_FLOAT64: return run_attention<double>(p, q, k, v, out, stream);
        default: return TANNIC_UNSUPPORTED_DTYPE;
    }
}

static bool is_float(int dtype) { return dtype == TANNIC_FLOAT16 || dtype == TANNIC_BFLOAT16 || dtype == TANNIC_FLOAT32 || dtype == TANNIC_FLOAT64; }

}  // namespace th

using namespace th;

extern "C" {

int tannic_hip_attend_pages(const tannic_tensor_t* q, const tannic_tensor_t* keys, const tannic_tensor_t* values, const tannic_tensor_t* table,
                            const tannic_tensor_t* starts, const tannic_tensor_t* context, tannic_tensor_t* dst, tannic_stream_t stream, float scale) {
    if (!q || !keys || !values || !table || !starts || !context || !dst) return refuse("attend_pages: a descriptor is missing");
    if (!have_storage(q, keys, values, table, starts, context, dst)) return TANNIC_ERROR;
    if (!is_float(q->dtype) || keys->dtype != q->dtype || values->dtype != q->dtype || dst->dtype != q->dtype || table->dtype != TANNIC_INT32 ||
        starts->dtype != TANNIC_INT32 || context->dtype != TANNIC_INT32)
        return TANNIC_UNSUPPORTED_DTYPE;
    if (q->rank != 3 || !extents_equal(q, dst) || !rows_contiguous(dst)) return refuse("attend_pages: q [tokens, heads, d], dst contiguous with q's shape");
    PageTable pages;
    if (int status = describe_pages(keys, values, table, starts, context, pages); status != TANNIC_SUCCESS) return status;
    AttentionProblem p{};
    p.heads = static_cast<uint32_t>(q->shape.sizes[1]);
    p.d = static_cast<uint32_t>(q->shape.sizes[2]);
    if (q->shape.sizes[0] >= kMostBlocks || q->shape.sizes[1] >= (1u << 16) || q->shape.sizes[0] * q->shape.sizes[1] >= (1ull << 30))
        return refuse("attend_pages: 2^24 tokens, 2^16 heads or 2^30 rows of queries or more are not supported");
    if (q->shape.sizes[2] != keys->shape.sizes[3] || q->shape.sizes[2] > kAttentionHead) return refuse("attend_pages: q and the keys have one head size, at most 256");
    if (q->shape.sizes[1] == 0 || pages.kv_heads == 0 || q->shape.sizes[1] % pages.kv_heads != 0) return refuse("attend_pages: the number of heads is a multiple of the cache's");
    if (q->shape.sizes[2] > 1 && q->strides.sizes[2] != 1) return refuse("attend_pages: the elements of a head of q lie one after the other");
    if (element_count(q) == 0 || pages.sequences == 0) return TANNIC_SUCCESS;
    if (int status = on_device_of("attend_pages: the operands live on a device", q, keys, values, table, starts, context, dst); status != TANNIC_SUCCESS) return status;
    p.sequences = pages.sequences;
    p.tokens = static_cast<uint32_t>(q->shape.sizes[0]);
    p.kv_heads = pages.kv_heads;
    p.q_token = stride_of(q, 0);
    p.q_head = stride_of(q, 1);
    p.k_page = stride_of(keys, 0), p.k_head = stride_of(keys, 1), p.k_token = stride_of(keys, 2);
    p.v_page = stride_of(values, 0), p.v_head = stride_of(values, 1), p.v_token = stride_of(values, 2);
    p.starts = pages.starts, p.context = pages.context, p.table = pages.table, p.table_row = pages.table_row;
    p.columns = pages.columns, p.pages = pages.pages, p.page = pages.page, p.page_div = pages.page_div, p.room = pages.room;
    p.group = p.heads / p.kv_heads;
    p.group_div = FastDiv(p.group);
    p.scale = scale;
    return run_attention(q->dtype, p, q->address, keys->address, values->address, dst->address, as_stream(stream));
}

int tannic_hip_attend(const tannic_tensor_t* q, const tannic_tensor_t* k, const tannic_tensor_t* v, const tannic_tensor_t* lengths, tannic_tensor_t* dst,
                      tannic_stream_t stream, float scale) {
    if (!q || !k || !v || !dst) return refuse("attend: a descriptor is missing");
    if (!have_storage(q, k, v, lengths, dst)) return TANNIC_ERROR;
    if (!is_float(q->dtype) || k->dtype != q->dtype || v->dtype != q->dtype || dst->dtype != q->dtype || (lengths && lengths->dtype != TANNIC_INT32)) return TANNIC_UNSUPPORTED_DTYPE;
    if (q->rank != 4 || k->rank != 4 || !extents_equal(q, dst) || !rows_contiguous(dst) || !extents_equal(k, v))
        return refuse("attend: q [batch, tokens, heads, d], k and v [batch, states, kv heads, d], dst contiguous with q's shape");
    const size_t batch = q->shape.sizes[0], n = q->shape.sizes[1], heads = q->shape.sizes[2], d = q->shape.sizes[3];
    const size_t states = k->shape.sizes[1], kv_heads = k->shape.sizes[2];
    if (k->shape.sizes[0] != batch || k->shape.sizes[3] != d) return refuse("attend: q, k and v have one batch and one head size");
    if (d > kAttentionHead) return refuse("attend: heads of more than 256 elements are not supported");
    if (heads == 0 || kv_heads == 0 || heads % kv_heads != 0) return refuse("attend: the number of heads is a multiple of the keys'");
    if (batch >= kMostBlocks || n >= kMostBlocks || heads >= (1u << 16) || states >= (1ull << 31) || batch * n >= kMostBlocks || batch * n * heads >= (1ull << 30))
        return refuse("attend: 2^24 tokens, 2^16 heads, 2^30 rows of queries, 2^31 keys or more are not supported");
    if (lengths && (lengths->rank != 1 || lengths->shape.sizes[0] != batch || !rows_contiguous(lengths))) return refuse("attend: lengths [batch], contiguous");
    if (d > 1 && (q->strides.sizes[3] != 1 || (states > 0 && (k->strides.sizes[3] != 1 || v->strides.sizes[3] != 1)))) return refuse("attend: the elements of a head lie one after the other");
    if (element_count(q) == 0) return TANNIC_SUCCESS;
    if (int status = on_device_of("attend: the operands live on a device", q, k, v, lengths, dst); status != TANNIC_SUCCESS) return status;
    AttentionProblem p{};
    p.sequences = static_cast<uint32_t>(batch);
    p.per_sequence = static_cast<uint32_t>(n);
    p.tokens = static_cast<uint32_t>(batch * n);
    p.heads = static_cast<uint32_t>(heads);
    p.kv_heads = static_cast<uint32_t>(kv_heads);
    p.d = static_cast<uint32_t>(d);
    p.q_batch = stride_of(q, 0), p.q_token = stride_of(q, 1), p.q_head = stride_of(q, 2);
    p.k_page = stride_of(k, 0), p.k_token = stride_of(k, 1), p.k_head = stride_of(k, 2);
    p.v_page = stride_of(v, 0), p.v_token = stride_of(v, 1), p.v_head = stride_of(v, 2);
    p.lengths = lengths ? static_cast<const int32_t*>(lengths->address) : nullptr;
    p.room = static_cast<uint32_t>(states);
    p.pages = p.sequences;
    p.page = p.room;
    p.group = p.heads / p.kv_heads;
    p.group_div = FastDiv(p.group);
    p.scale = scale;
    return run_attention(q->dtype, p, q->address, k->address, v->address, dst->address, as_stream(stream));
}

}  // extern "C"
