// Problem description shared by the kernels of products of 8-bit integers with scales (gemm_quantized.hip).
#pragma once

#include "gemm_tiles.hpp"
#include "quantized.hpp"

namespace th {

// Where the scales of a product lie: a row's (column's) in a batch.
struct ScalePlaces {
    const float *a, *b;
    int64_t a_step, b_step;
    int64_t a_bs[6], b_bs[6];
};

__device__ inline void scale_offsets(const GemmProblem& p, const ScalePlaces& s, uint32_t batch, const float*& a, const float*& b) {
    int64_t oa = 0, ob = 0;
    for (int d = p.batch_rank - 1; d >= 0; --d) {
        const uint32_t idx = batch % p.batch_extent[d];
        batch /= p.batch_extent[d];
        oa += static_cast<int64_t>(idx) * s.a_bs[d];
        ob += static_cast<int64_t>(idx) * s.b_bs[d];
    }
    a = s.a + oa;
    b = s.b + ob;
}

typedef int int4v __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) void* lds_address;

__device__ inline int4v mfma_i8(const uint4v& first, const uint4v& second, const int4v& sum) {
    int4v x, y;
    __builtin_memcpy(&x, &first, 16);
    __builtin_memcpy(&y, &second, 16);
    return __builtin_amdgcn_mfma_i32_16x16x64_i8(x, y, sum, 0, 0, 0);
}

// Four results of a row, from column `col` on, `live` of them there.
template <class D> __device__ inline void store_four(D* to, const float (&v)[4], uint32_t live) {
    D out[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) out[e] = rounded<D>(v[e]);
    if (live >= 4) {
        typedef unsigned int uint2any __attribute__((ext_vector_type(2), aligned(2)));
        typedef unsigned int uint4any __attribute__((ext_vector_type(4), aligned(4)));
        using Any = std::conditional_t<sizeof(D) == 2, uint2any, uint4any>;
        Any bits;
        __builtin_memcpy(&bits, out, sizeof(Any));
        *reinterpret_cast<Any*>(to) = bits;
    } else {
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (e < static_cast<int>(live)) to[e] = out[e];
    }
}

// Operands that the kernels with direct loads to LDS take: rows along K in whole pieces of 16 bytes at multiples of 4 (what such a load asks of an address), 32-bit offsets
// inside a tile of 256 rows.
inline bool quantized_operands_fit(const GemmProblem& p, const void* a, const void* b) {
    if (p.a_cs != 1 || p.b_rs != 1 || p.K == 0 || p.K % 16 != 0 || p.batches > 65535) return false;
    if (reinterpret_cast<uintptr_t>(a) % 4 || reinterpret_cast<uintptr_t>(b) % 4 || p.a_rs % 4 || p.b_cs % 4) return false;
    for (int d = 0; d < p.batch_rank; ++d)
        if (p.a_bs[d] % 4 || p.b_bs[d] % 4) return false;
    const auto pitch = [](int64_t rows, int64_t stride) { return rows == 1 || (stride >= 0 && stride < (1 << 22)); };
    return pitch(p.M, p.a_rs) && pitch(p.N, p.b_cs);
}

// What a row of an operand is looked up with where its loads are out of the buffer's range, and so zeros.
constexpr uint32_t kBeyond = 0x80000000u;

// The bytes of `rows` rows (256 at most), which end with the last one's K: below kBeyond.
__device__ inline uint32_t bytes_of_rows(uint32_t rows, int64_t pitch, uint32_t K) { return (rows - 1) * static_cast<uint32_t>(pitch) + K; }

// Fewer blocks of bm x bn results than a launch may have.
inline bool few_enough_blocks(const GemmProblem& p, uint64_t bm, uint64_t bn) {
    return (static_cast<uint64_t>(p.M) + bm - 1) / bm * ((static_cast<uint64_t>(p.N) + bn - 1) / bn) * p.batches < kMostBlocks && p.batches <= 65535;
}
inline bool gemm_quantized_tile_takes(const GemmProblem& p, const void* a, const void* b) { return quantized_operands_fit(p, a, b) && few_enough_blocks(p, 256, 256); }

// Up to 32 rows (gemm_quantized_rows.hip) and more (gemm_quantized_tile.hip); TANNIC_UNSUPPORTED_DTYPE: not this kernel's
bool gemm_quantized_rows_takes(const GemmProblem& p, const void* a, const void* b);
template <class D> int gemm_quantized_rows(const GemmProblem& p, const ScalePlaces& s, const void* a, const void* b, void* c, hipStream_t stream);
template <class D> int gemm_quantized_tile(const GemmProblem& p, const ScalePlaces& s, const void* a, const void* b, void* c, hipStream_t stream);
// rows along K that start anywhere and have any length; `or_copies`: not where copying them for the kernels above is faster
template <class D> int gemm_quantized_bytes(const GemmProblem& p, bool or_copies, const ScalePlaces& s, const void* a, const void* b, void* c, hipStream_t stream);
template <class D> bool gemm_quantized_bytes_takes(const GemmProblem& p, bool or_copies);

}  // namespace th
