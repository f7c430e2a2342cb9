// Product of 8-bit integers with a scale for each row of the first operand and each column of the second (tokens and channels):
//   dst[m, n] = (sum_k a[m, k] * b[k, n]) * a_scales[m] * b_scales[n]
// The sum is a whole number and exact in 32 bits (K below 2^17), in any order and in any parts; it is taken to float, multiplied by both scales and rounded once to dst's type.
// As calls of the operators that were there it is an int32 product, a cast and two broadcasting multiplications.
#include "gemm_quantized.hpp"

namespace th {

constexpr size_t kMostInner = (1u << 17) - 1;      // 128 * 128 * K is below 2^31

// Any strides: 64 x 64 results of a block, 4 x 4 of a thread, K in steps of 32 through LDS.
template <class D>
__global__ __launch_bounds__(256) void gemm_quantized_any_kernel(const int8_t* a, const int8_t* b, D* c, GemmProblem p, ScalePlaces s, uint32_t tiles_n) {
    constexpr int T = 64, KT = 32;
    __shared__ int sa[KT][T + 1];
    __shared__ int sb[KT][T + 1];
    int64_t oa, ob, oc;
    batch_offsets(p, blockIdx.y, oa, ob, oc);
    const float *scale_a, *scale_b;
    scale_offsets(p, s, blockIdx.y, scale_a, scale_b);
    a += oa;
    b += ob;
    c += oc;
    const uint32_t m0 = blockIdx.x / tiles_n * T, n0 = blockIdx.x % tiles_n * T;
    const int tx = threadIdx.x % 16, ty = threadIdx.x / 16;
    int acc[4][4] = {};
    for (uint32_t k0 = 0; k0 < p.K; k0 += KT) {
        for (int i = threadIdx.x; i < T * KT; i += 256) {
            // consecutive threads along whichever index is contiguous
            const int ka = p.a_cs == 1 ? i % KT : i / T, ma = p.a_cs == 1 ? i / KT : i % T;
            const uint32_t m = m0 + ma, k = k0 + ka;
            sa[ka][ma] = m < p.M && k < p.K ? a[m * p.a_rs + k * p.a_cs] : 0;
            const int kb = p.b_rs == 1 ? i % KT : i / T, nb = p.b_rs == 1 ? i / KT : i % T;
            const uint32_t n = n0 + nb, k2 = k0 + kb;
            sb[kb][nb] = n < p.N && k2 < p.K ? b[k2 * p.b_rs + n * p.b_cs] : 0;
        }
        __syncthreads();
#pragma unroll 4
        for (int kk = 0; kk < KT; ++kk) {
            int x[4], y[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                x[i] = sa[kk][ty * 4 + i];
                y[i] = sb[kk][tx * 4 + i];
            }
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int j = 0; j < 4; ++j) acc[i][j] += x[i] * y[j];
        }
        __syncthreads();
    }
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const uint32_t m = m0 + ty * 4 + i, n = n0 + tx * 4 + j;
            if (m < p.M && n < p.N) c[m * p.c_rs + n] = rounded<D>(static_cast<float>(acc[i][j]) * scale_a[m * s.a_step] * scale_b[n * s.b_step]);
        }
}

template <class D>
int run_any(const GemmProblem& p, const ScalePlaces& s, const void* a, const void* b, void* c, hipStream_t stream) {
    const uint64_t tiles_m = (static_cast<uint64_t>(p.M) + 63) / 64, tiles_n = (static_cast<uint64_t>(p.N) + 63) / 64;
    if (tiles_m * tiles_n >= kMostBlocks || p.batches > 65535) return refuse("gemm_quantized: a product of so many tiles or batches is not supported");
    hipLaunchKernelGGL((gemm_quantized_any_kernel<D>), dim3(static_cast<uint32_t>(tiles_m * tiles_n), p.batches), dim3(256), 0, stream, static_cast<const int8_t*>(a),
                       static_cast<const int8_t*>(b), static_cast<D*>(c), p, s, static_cast<uint32_t>(tiles_n));
    return launch_status("gemm_quantized_any_kernel");
}

// Batches that lie behind each other under one matrix are rows of one product.
void fold_batches(GemmProblem& p, ScalePlaces& s) {
    while (p.batch_rank > 0) {
        const int d = p.batch_rank - 1;
        const uint64_t extent = p.batch_extent[d], rows = p.M * extent;
        if (extent != 1) {
            if (p.b_bs[d] != 0 || s.b_bs[d] != 0 || rows >= (1ull << 31)) return;
            const int64_t m = p.M;
            if (m == 1) {      // (a single row's pitch is never used)
                p.a_rs = p.a_bs[d];
                s.a_step = s.a_bs[d];
            } else if (p.a_bs[d] != m * p.a_rs || s.a_bs[d] != m * s.a_step) {
                return;
            }
            p.c_rs = p.N;
            p.M = static_cast<uint32_t>(rows);
            p.batches = static_cast<uint32_t>(p.batches / extent);
        }
        p.batch_extent[d] = 1;
        p.a_bs[d] = p.b_bs[d] = p.c_bs[d] = s.a_bs[d] = s.b_bs[d] = 0;
        --p.batch_rank;
    }
}

// Operands that do not lie along K in whole pieces: `q`, the product over copies of them (or over the same, a single row without a pitch), if gemm_repack makes it one that the kernels
// with direct loads take.  (It copies no batch of several dims and no more than 2 GB, and leaves rows far apart or in reverse order as they are.)
bool copies_fit(const GemmProblem& p, const void* a, const void* b, GemmProblem& q, bool copies[2]) {
    return gemm_repack_plan(p, 1, a, b, true, q, copies) == TANNIC_SUCCESS && quantized_operands_fit(q, copies[0] ? nullptr : a, copies[1] ? nullptr : b);
}

template <class D>
int run_quantized(const GemmProblem& p, const ScalePlaces& s, const void* a, const void* b, void* c, hipStream_t stream) {
    GemmProblem q = p;
    const void *pa = a, *pb = b;
    void* held[2] = {nullptr, nullptr};
    int status = TANNIC_UNSUPPORTED_DTYPE;
    bool fit = quantized_operands_fit(p, a, b);
    if (!fit) {
        status = gemm_quantized_bytes<D>(p, true, s, a, b, c, stream);
        if (status != TANNIC_UNSUPPORTED_DTYPE) return status;
        bool copies[2];
        if (copies_fit(p, a, b, q, copies)) {
            status = gemm_repack(p, 1, a, b, stream, true, q, pa, pb, held);
            if (status != TANNIC_SUCCESS && status != TANNIC_UNSUPPORTED_DTYPE) return status;
            fit = status == TANNIC_SUCCESS;
        }
        if (!fit) status = gemm_quantized_bytes<D>(p, false, s, a, b, c, stream);
    }
    if (fit) {
        status = gemm_quantized_rows<D>(q, s, pa, pb, c, stream);
        if (status == TANNIC_UNSUPPORTED_DTYPE) status = gemm_quantized_tile<D>(q, s, pa, pb, c, stream);
    }
    if (status == TANNIC_UNSUPPORTED_DTYPE) status = run_any<D>(p, s, a, b, c, stream);
    for (void* h : held)
        if (h) scratch_release(h, stream);
    return status;
}

// The product and where its scales lie, from the descriptors: everything but the device.
int describe_quantized(const tannic_tensor_t* a, const tannic_tensor_t* a_scales, const tannic_tensor_t* b, const tannic_tensor_t* b_scales, const tannic_tensor_t* dst, GemmProblem& p,
                       ScalePlaces& s) {
    if (!a || !a_scales || !b || !b_scales || !dst) return refuse("gemm_quantized: a descriptor is missing");
    if (!have_storage(a, a_scales, b, b_scales, dst)) return TANNIC_ERROR;
    if (a->dtype != TANNIC_INT8 || b->dtype != TANNIC_INT8 || a_scales->dtype != TANNIC_FLOAT32 || b_scales->dtype != TANNIC_FLOAT32 ||
        (dst->dtype != TANNIC_FLOAT16 && dst->dtype != TANNIC_BFLOAT16 && dst->dtype != TANNIC_FLOAT32))
        return TANNIC_UNSUPPORTED_DTYPE;
    if (int status = describe_gemm(a, b, dst, p)) return status;
    if (!rows_contiguous(dst)) return refuse("gemm_quantized: dst is contiguous");
    if (p.K > kMostInner) return refuse("gemm_quantized: sums over 2^17 elements or more do not fit 32 bits");
    bool fit = a_scales->rank + 1 == a->rank && b_scales->rank + 1 == b->rank;
    for (int d = 0; fit && d < a_scales->rank; ++d) fit = a_scales->shape.sizes[d] == a->shape.sizes[d];
    for (int d = 0; fit && d < b_scales->rank; ++d) fit = b_scales->shape.sizes[d] == b->shape.sizes[d + (d == b_scales->rank - 1)];
    if (!fit) return refuse("gemm_quantized: a scale for each row of a [.., M, K] and each column of b [.., K, N]");
    s.a = static_cast<const float*>(a_scales->address);
    s.b = static_cast<const float*>(b_scales->address);
    s.a_step = stride_of(a_scales, a_scales->rank - 1);
    s.b_step = stride_of(b_scales, b_scales->rank - 1);
    for (int d = 0; d < p.batch_rank; ++d) {
        const auto places = [&](const tannic_tensor_t* scales) -> int64_t {      // (its batch dims are right-aligned with dst's)
            const int at = d + scales->rank - 1 - p.batch_rank;
            return at < 0 ? 0 : stride_of(scales, at);
        };
        s.a_bs[d] = places(a_scales);
        s.b_bs[d] = places(b_scales);
    }
    return TANNIC_SUCCESS;
}

}  // namespace th

using namespace th;

extern "C" int tannic_hip_gemm_quantized(const tannic_tensor_t* a, const tannic_tensor_t* a_scales, const tannic_tensor_t* b, const tannic_tensor_t* b_scales, tannic_tensor_t* dst,
                                         tannic_stream_t stream) {
    GemmProblem p;
    ScalePlaces s{};
    if (int status = describe_quantized(a, a_scales, b, b_scales, dst, p, s)) return status;
    if (int status = on_device_of("gemm_quantized: the operands live on a device", a, a_scales, b, b_scales, dst)) return status;
    if (p.M == 0 || p.N == 0 || p.batches == 0) return TANNIC_SUCCESS;
    fold_batches(p, s);
    switch (dst->dtype) {
        case TANNIC_FLOAT16: return run_quantized<f16>(p, s, a->address, b->address, dst->address, as_stream(stream));
        case TANNIC_BFLOAT16: return run_quantized<bf16>(p, s, a->address, b->address, dst->address, as_stream(stream));
        default: return run_quantized<float>(p, s, a->address, b->address, dst->address, as_stream(stream));
    }
}

extern "C" int tannic_hip_gemm_quantized_plan(const tannic_tensor_t* a, const tannic_tensor_t* a_scales, const tannic_tensor_t* b, const tannic_tensor_t* b_scales, const tannic_tensor_t* dst,
                                              uint32_t out[2]) {
    out[0] = out[1] = 0;
    GemmProblem p;
    ScalePlaces s{};
    if (int status = describe_quantized(a, a_scales, b, b_scales, dst, p, s)) return status;
    if (p.M == 0 || p.N == 0 || p.batches == 0) return TANNIC_SUCCESS;
    fold_batches(p, s);
    GemmProblem q = p;
    bool copies[2] = {false, false};
    const void *pa = a->address, *pb = b->address;
    if (!quantized_operands_fit(p, pa, pb)) {
        if (gemm_quantized_bytes_takes<bf16>(p, true) || !copies_fit(p, pa, pb, q, copies)) {
            out[0] = gemm_quantized_bytes_takes<bf16>(p, false) ? 3 : 0;
            return TANNIC_SUCCESS;
        }
        if (copies[0]) pa = nullptr;
        if (copies[1]) pb = nullptr;
    }
    out[0] = gemm_quantized_rows_takes(q, pa, pb) ? 1 : gemm_quantized_tile_takes(q, pa, pb) ? 2 : 0;
    out[1] = (copies[0] ? 1 : 0) + (copies[1] ? 2 : 0);
    return TANNIC_SUCCESS;
}
