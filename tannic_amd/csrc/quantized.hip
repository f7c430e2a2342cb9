// Rows in 8-bit integers with a scale each, what a product of integers takes (gemm_quantized.hip): of any values, of a gated activation, of a
// root-mean-square norm with the residual's addition before it; that norm in the operands' type; and the way back.
//   quantize          u = x
//   swiglu_quantize   u = gate / (1 + exp(-gate)) * up
//   add_rms_norm      total = round(x + residual),  u = total * gain,  r = 1 / sqrt(mean(total^2) + eps);  u * r in the operands' type, or in 8 bits
//   values = rint(u * (127 * (1 / max|u|))),  scales = max|u| (* r) / 127
// The norm's r is one number for a row and cancels in the integers, so that these need the row's largest |u| only, which no order of summation changes.
#include "quantized.hpp"

namespace th {

struct SquaresOp {
    template <class A> __device__ static inline A combine(A x, A y) { return x + y; }
};

// One value per block of 256 threads, the same in every thread.
template <class Op, class A>
__device__ inline A block_reduce(A v, A* lds) {
    v = wave_reduce<Op>(v);
    __syncthreads();
    if (threadIdx.x % 64 == 0) lds[threadIdx.x / 64] = v;
    __syncthreads();
    return Op::combine(Op::combine(lds[0], lds[1]), Op::combine(lds[2], lds[3]));
}

enum class RowSource { plain, gated, norm, sum_norm };

struct RowOperands {
    const void *x, *second, *gain;      // second: up, or the residual
    void *total, *dst;                  // dst: the norm in the operands' type, or the integers
    float* scales;                      // nullptr: in the operands' type
    RowsMap rows_x, rows_second;
    uint32_t rows, length;
    double eps;
};

// gate / (1 + exp(-gate)) * up, off by 8 * 2^-24 at most, for gates from -64 on: exp(-gate) is 2^high * (1 + low * ln 2) with high + low = -gate * log2 e (the instruction for
// powers of two is off by 2 units, and high alone would be by |gate|); the sum with 1 takes both in one rounding, its reciprocal is off by 2 units.  The product with log2 e may not be
// beyond all floats: the exponential of -200 is nothing beside 1.
constexpr float kLog2e = 0x1.715476p+0f, kLog2eRest = 0x1.4ae0bep-26f;
__device__ inline float gated(float gate, float up) {
    constexpr float ln2 = 0x1.62e430p-1f;
    const float power = __builtin_amdgcn_fmed3f(-gate, -200.0f, 200.0f), high = power * kLog2e, low = fmaf(power, kLog2eRest, fmaf(power, kLog2e, -high));
    const float sum = fmaf(__builtin_amdgcn_exp2f(high), fmaf(low, ln2, 1.0f), 1.0f);
    return gate * __builtin_amdgcn_rcpf(sum) * up;
}

// Below -64 1 is nothing beside exp(-gate) (2^-92), and gate * exp(gate) * up is it: from -87 on the reciprocal of the sum would be no normal number, from -92 on the quotient, and
// both come out as 0, while up may make either large.  exp(gate) is 2^whole * 2^part with |part| <= 1/2 (off by 2^-25 before the instruction's 2 units), the powers of two of both factors meet in the last step:
// off by 5 * 2^-24 at most, or by half of the smallest subnormal number.  exp(-400) is 0 with any factor; a gate that is not finite is what it is in the formula.
constexpr uint32_t kFarGateBits = 0xC2800000u;      // -64 (what is below it, as an unsigned number, is above this; so is what is not a number and has a sign)
__device__ inline float gated_far(float gate, float up) {
    const float power = fmaxf(gate, -400.0f), whole = rintf(power * kLog2e), part = fmaf(power, kLog2eRest, fmaf(power, kLog2e, -whole));
    const float near = power * 0x1p-64f * __builtin_amdgcn_exp2f(part) * up;
    return fmaf(gate, 0.0f, ldexpf(near, static_cast<int>(whole) + 64));
}

// ---- rows in registers ----------------------------------------------------------------
// 16 bytes of a row and what its integers take, wherever they start.
typedef unsigned int uint4any __attribute__((ext_vector_type(4), aligned(1)));
typedef unsigned int uint2any __attribute__((ext_vector_type(2), aligned(1)));
typedef unsigned int uint1any __attribute__((aligned(1)));
template <class T> constexpr int kPiece = 16 / sizeof(T);
template <class T> struct Piece {
    T v[kPiece<T>];
};

// `live` elements of a piece (the last one of a row may be short), zeros behind them
template <class T, bool PAST = false> __device__ inline Piece<T> load_piece(const T* from, uint32_t live) {
    Piece<T> r;
    if (live >= kPiece<T>) {
        uint4any bits;
        if constexpr (PAST) bits = __builtin_nontemporal_load(reinterpret_cast<const uint4any*>(from));
        else bits = *reinterpret_cast<const uint4any*>(from);
        __builtin_memcpy(&r, &bits, 16);
    } else {
#pragma unroll
        for (int e = 0; e < kPiece<T>; ++e) r.v[e] = e < static_cast<int>(live) ? from[e] : T{};
    }
    return r;
}
template <class T, bool PAST = false> __device__ inline void store_piece(T* to, const Piece<T>& piece, uint32_t live) {
    if (live >= kPiece<T>) {
        uint4any bits;
        __builtin_memcpy(&bits, &piece, 16);
        if constexpr (PAST) __builtin_nontemporal_store(bits, reinterpret_cast<uint4any*>(to));
        else *reinterpret_cast<uint4any*>(to) = bits;
    } else {
#pragma unroll
        for (int e = 0; e < kPiece<T>; ++e)
            if (e < static_cast<int>(live)) to[e] = piece.v[e];
    }
}
template <bool PAST, int N> __device__ inline void store_integers(int8_t* to, const int8_t (&v)[N], uint32_t live) {
    if (live >= N) {
        using Any = std::conditional_t<N == 8, uint2any, uint1any>;
        Any bits;
        __builtin_memcpy(&bits, v, N);
        if constexpr (PAST) __builtin_nontemporal_store(bits, reinterpret_cast<Any*>(to));
        else *reinterpret_cast<Any*>(to) = bits;
    } else {
#pragma unroll
        for (int e = 0; e < N; ++e)
            if (e < static_cast<int>(live)) to[e] = v[e];
    }
}

// A group of G threads (a wavefront, or a block) per row, which is read once and kept in registers as u, NCH pieces of 16 bytes of a thread.  Bound by memory: 8001 x 5120 fp16
// with sum and residual 55.9 us, 5.1 TB/s, 4096 x 14336 bf16 gated 57.2 us, 5.1 TB/s (its arithmetic takes nearly as long), 28672 x 4096 fp16 57.6 us, 6.1 TB/s.
// Wavefronts on a SIMD that the registers have to leave room for: three blocks of 512 on a compute unit where one register too many (81, fp16) would make them two (8001 x 5120 with sum and
// residual 59 / 50 us).  No such limit for the others: with three or four pieces they would spill.
template <RowSource S, int G, int NCH> constexpr int kRowWavefronts = (S == RowSource::norm || S == RowSource::sum_norm) && G == 512 && NCH == 2 ? 6 : 1;

template <class T, RowSource S, bool INTEGERS, int G, int NCH, bool PAST>
__global__ __launch_bounds__(G == 64 ? 256 : G, (kRowWavefronts<S, G, NCH>)) void rows_kernel(RowOperands p) {
    constexpr bool NORM = S == RowSource::norm || S == RowSource::sum_norm;
    constexpr int VEC = kPiece<T>, BLOCK = G == 64 ? 256 : G, WAVES = BLOCK / 64;
    __shared__ float sums[WAVES];
    __shared__ uint32_t largest[WAVES];
    const uint32_t t = threadIdx.x % G;
    const T* const gain = static_cast<const T*>(p.gain);
    for (uint32_t row = blockIdx.x * (BLOCK / G) + threadIdx.x / G; row < p.rows; row += gridDim.x * (BLOCK / G)) {
        const T* const x = static_cast<const T*>(p.x) + p.rows_x.offset(row);
        const T* const second = S == RowSource::gated || S == RowSource::sum_norm ? static_cast<const T*>(p.second) + p.rows_second.offset(row) : nullptr;
        const size_t base = static_cast<size_t>(row) * p.length;
        Piece<T> a[NCH], b[NCH], g[NCH];
#pragma unroll
        for (int i = 0; i < NCH; ++i) {
            const uint32_t at = (t + i * G) * VEC;
            if (at < p.length) {
                a[i] = load_piece<T, PAST>(x + at, p.length - at);
                if constexpr (S == RowSource::gated || S == RowSource::sum_norm) b[i] = load_piece<T, PAST>(second + at, p.length - at);
                if constexpr (NORM) g[i] = load_piece(gain + at, p.length - at);
            }
        }
        float u[NCH][VEC], squares = 0;
        uint32_t most = 0, lowest = 0;      // (the bits of the lowest gate)
#pragma unroll
        for (int i = 0; i < NCH; ++i) {
            const uint32_t at = (t + i * G) * VEC;
            if (at < p.length) {
                if constexpr (S == RowSource::sum_norm) {
#pragma unroll
                    for (int e = 0; e < VEC; ++e) a[i].v[e] = rounded<T>(widen(a[i].v[e]) + widen(b[i].v[e]));
                    store_piece(static_cast<T*>(p.total) + base + at, a[i], p.length - at);
                }
#pragma unroll
                for (int e = 0; e < VEC; ++e) {
                    const float v = widen(a[i].v[e]);
                    if constexpr (NORM) squares += v * v;
                    if constexpr (S == RowSource::gated) u[i][e] = gated(v, widen(b[i].v[e])), lowest = LargestOp::combine(lowest, __float_as_uint(v));
                    else if constexpr (NORM && INTEGERS) u[i][e] = v * widen(g[i].v[e]);
                    else u[i][e] = v;
                    if constexpr (INTEGERS) most = LargestOp::combine(most, magnitude(u[i][e]));
                }
            }
        }
        if constexpr (S == RowSource::gated) {
            // some gate far below zero, hardly ever: the thread's pieces once more, read again so that nothing is kept for it
            if (lowest > kFarGateBits) {
                most = 0;
#pragma unroll
                for (int i = 0; i < NCH; ++i) {
                    const uint32_t at = (t + i * G) * VEC;
                    if (at < p.length) {
                        uint32_t again = at;
                        asm volatile("" : "+v"(again));      // (a number of its own, or the first reading waits piece by piece for what both have in common: 4096 x 14336 fp16 90 us for 88)
                        const Piece<T> gate = load_piece<T, PAST>(x + again, p.length - again), up = load_piece<T, PAST>(second + again, p.length - again);
#pragma unroll
                        for (int e = 0; e < VEC; ++e) {
                            if (__float_as_uint(widen(gate.v[e])) > kFarGateBits) u[i][e] = gated_far(widen(gate.v[e]), widen(up.v[e]));
                            most = LargestOp::combine(most, magnitude(u[i][e]));
                        }
                    }
                }
            }
        }
        if constexpr (NORM) squares = wave_reduce<SquaresOp>(squares);
        if constexpr (INTEGERS) most = wave_reduce<LargestOp>(most);
        if constexpr (G > 64) {
            __syncthreads();      // (the row before has been read)
            if (threadIdx.x % 64 == 0) {
                if constexpr (NORM) sums[threadIdx.x / 64] = squares;
                if constexpr (INTEGERS) largest[threadIdx.x / 64] = most;
            }
            __syncthreads();
            squares = 0;
            most = 0;
#pragma unroll
            for (int w = 0; w < WAVES; ++w) {
                if constexpr (NORM) squares += sums[w];
                if constexpr (INTEGERS) most = LargestOp::combine(most, largest[w]);
            }
        }
        const float r = NORM ? 1.0f / sqrtf(squares / static_cast<float>(p.length) + static_cast<float>(p.eps)) : 1.0f;
        const RowScale scale(most);
#pragma unroll
        for (int i = 0; i < NCH; ++i) {
            const uint32_t at = (t + i * G) * VEC;
            if (at < p.length) {
                if constexpr (INTEGERS) {
                    int8_t out[VEC];
#pragma unroll
                    for (int e = 0; e < VEC; ++e) out[e] = scale.integer(u[i][e]);
                    store_integers<PAST>(static_cast<int8_t*>(p.dst) + base + at, out, p.length - at);
                } else {
                    Piece<T> out;
#pragma unroll
                    for (int e = 0; e < VEC; ++e) out.v[e] = rounded<T>(u[i][e] * r * widen(g[i].v[e]));
                    store_piece(static_cast<T*>(p.dst) + base + at, out, p.length - at);
                }
            }
        }
        if constexpr (INTEGERS)
            if (t == 0) p.scales[row] = scale.scale(r);
    }
}

// Any row, the rows in turns: a block per row, which is read twice (a sum that was written is read again by the thread that wrote it).
template <class T, RowSource S, bool INTEGERS>
__global__ __launch_bounds__(256) void rows_any_kernel(RowOperands p) {
    using A = std::conditional_t<std::is_same_v<T, double>, double, float>;
    constexpr bool NORM = S == RowSource::norm || S == RowSource::sum_norm;
    __shared__ double sums[4];
    __shared__ uint32_t largest[4];
    const T* const gain = static_cast<const T*>(p.gain);
    for (uint32_t row = blockIdx.x; row < p.rows; row += gridDim.x) {
        const T* const x = static_cast<const T*>(p.x) + p.rows_x.offset(row);
        const T* const second = static_cast<const T*>(p.second) + (S == RowSource::gated || S == RowSource::sum_norm ? p.rows_second.offset(row) : 0);
        const size_t base = static_cast<size_t>(row) * p.length;
        T* const total = static_cast<T*>(p.total) + base;
        uint32_t lowest = 0;      // (the bits of the lowest gate)
        using Far = std::true_type;      // the row has gates far below zero, hardly ever
        using Near = std::false_type;
        auto value = [&](uint32_t i, bool first, auto gates) -> A {
            if constexpr (S == RowSource::gated) {
                const float gate = widen(x[i * p.rows_x.step]), up = widen(second[i * p.rows_second.step]);
                lowest = LargestOp::combine(lowest, __float_as_uint(gate));
                if constexpr (decltype(gates)::value)
                    if (__float_as_uint(gate) > kFarGateBits) return gated_far(gate, up);
                return gated(gate, up);
            }
            if constexpr (S == RowSource::sum_norm) {
                if (!first) return static_cast<A>(widen(total[i]));
                const T sum = rounded<T>(static_cast<A>(widen(x[i * p.rows_x.step])) + static_cast<A>(widen(second[i * p.rows_second.step])));
                total[i] = sum;
                return static_cast<A>(widen(sum));
            }
            return static_cast<A>(widen(x[i * p.rows_x.step]));
        };
        double squares = 0;      // (a thread may have millions of them, one after another)
        uint32_t most = 0;
        const auto look = [&](auto gates) {
            for (uint32_t i = threadIdx.x; i < p.length; i += 256) {
                const A v = value(i, true, gates);
                if constexpr (NORM) squares += static_cast<double>(v) * v;
                if constexpr (INTEGERS) most = LargestOp::combine(most, magnitude(static_cast<float>(NORM ? v * static_cast<A>(widen(gain[i])) : v)));
            }
        };
        look(Near{});
        bool far = false;
        if constexpr (S == RowSource::gated) {
            far = block_reduce<LargestOp>(lowest, largest) > kFarGateBits;
            if (far) {
                most = 0;
                look(Far{});
            }
        }
        A r = 1;
        if constexpr (NORM) r = A(1) / sqrt(static_cast<A>(block_reduce<SquaresOp>(squares, sums)) / static_cast<A>(p.length) + static_cast<A>(p.eps));
        if constexpr (INTEGERS) {
            const RowScale scale(block_reduce<LargestOp>(most, largest));
            const auto write = [&](auto gates) {
                for (uint32_t i = threadIdx.x; i < p.length; i += 256) {
                    const A v = value(i, false, gates);
                    static_cast<int8_t*>(p.dst)[base + i] = scale.integer(static_cast<float>(NORM ? v * static_cast<A>(widen(gain[i])) : v));
                }
            };
            if (far) write(Far{});
            else write(Near{});
            if (threadIdx.x == 0) p.scales[row] = scale.scale(static_cast<float>(r));
        } else {
            for (uint32_t i = threadIdx.x; i < p.length; i += 256) static_cast<T*>(p.dst)[base + i] = rounded<T>(value(i, false, Near{}) * r * static_cast<A>(widen(gain[i])));
        }
    }
}

// Eight elements of a row per thread.
template <class T, bool PAST>
__global__ __launch_bounds__(256) void dequantize_kernel(const int8_t* values, RowsMap map, const float* scales, T* dst, uint32_t length, FastDiv per_row, uint32_t items) {
    const uint32_t item = blockIdx.x * 256 + threadIdx.x;
    if (item >= items) return;
    uint32_t row, piece;
    per_row.divmod(item, row, piece);
    const uint32_t at = piece * 8, live = length - at;
    const int8_t* const from = values + map.offset(row) + at;
    int8_t v[8];
    if (live >= 8) {
        const uint2any bits = *reinterpret_cast<const uint2any*>(from);
        __builtin_memcpy(v, &bits, 8);
    } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = e < static_cast<int>(live) ? from[e] : int8_t(0);
    }
    const float scale = scales[row];
    T* const to = dst + static_cast<size_t>(row) * length + at;
    constexpr int VEC = kPiece<T>;
#pragma unroll
    for (int i = 0; i < 8; i += VEC) {
        Piece<T> out;
#pragma unroll
        for (int e = 0; e < VEC; ++e) out.v[e] = rounded<T>(static_cast<float>(v[i + e]) * scale);
        if (static_cast<int>(live) > i) store_piece<T, PAST>(to + i, out, live - i);
    }
}

template <class T>
__global__ __launch_bounds__(256) void dequantize_any_kernel(const int8_t* values, RowsMap map, const float* scales, T* dst, uint32_t rows, uint32_t length) {
    for (uint32_t row = blockIdx.x; row < rows; row += gridDim.x) {
        const int8_t* const x = values + map.offset(row);
        const float scale = scales[row];
        for (uint32_t i = threadIdx.x; i < length; i += 256) dst[static_cast<size_t>(row) * length + i] = rounded<T>(static_cast<float>(x[i * map.step]) * scale);
    }
}

constexpr uint32_t kMostRowBlocks = 1u << 20;      // (rows beyond in turns)

// What does not fit the memory-side cache of 256 MB with its results goes past the caches: a matrix of weights from 128 MB on (28672 x 4096 fp16 with 235 MB 55 us past them, 61 through
// them; 8000 x 4096 bf16 with its sum and residual 39 and 36, so that the other sources, whose results a product takes next, stay with them).
constexpr uint64_t kRowsPastCaches = 128ull << 20;

template <class T, RowSource S, bool INTEGERS, int G, int NCH>
int launch_rows(const RowOperands& p, hipStream_t stream) {
    constexpr uint32_t BLOCK = G == 64 ? 256 : G, ROWS = BLOCK / G;
    const uint32_t blocks = (p.rows + ROWS - 1) / ROWS;
    const dim3 grid(blocks < kMostRowBlocks ? blocks : kMostRowBlocks);
    if constexpr (S == RowSource::plain) {
        if (static_cast<uint64_t>(p.rows) * p.length * sizeof(T) > kRowsPastCaches) {
            hipLaunchKernelGGL((rows_kernel<T, S, INTEGERS, G, NCH, true>), grid, dim3(BLOCK), 0, stream, p);
            return launch_status("rows_kernel");
        }
    }
    hipLaunchKernelGGL((rows_kernel<T, S, INTEGERS, G, NCH, false>), grid, dim3(BLOCK), 0, stream, p);
    return launch_status("rows_kernel");
}

template <class T, RowSource S, bool INTEGERS>
int run_rows(const RowOperands& p, hipStream_t stream) {
    if constexpr (!std::is_same_v<T, double>) {
        // rows whose elements lie one after the other and that the registers of a block hold
        constexpr bool PAIR = S == RowSource::gated || S == RowSource::sum_norm, PLAIN = S == RowSource::plain, NORM = S == RowSource::norm || S == RowSource::sum_norm;
        const uint32_t pieces = (p.length + kPiece<T> - 1) / kPiece<T>;
        if (p.length > 0 && (p.length == 1 || (p.rows_x.step == 1 && (!PAIR || p.rows_second.step == 1))) && pieces <= 4096) {
            // Threads of a row and their pieces, us of a norm with its sum / of values / gated, bf16, operands from memory, in brackets what is nearest: 32768 rows of 128 pieces 64 x 2
            // 37 / 17 / 27 (128 x 1 36 / 19 / 25); 16384 of 256 256 x 1 36 / - / 26, 128 x 2 - / 17 / - (64 x 4 39 / 17 / 29); 8192 of 512 512 x 1 39 / - / 29, 256 x 2 - / 17 / - (the other
            // way round 42 / 18 / 31); 8001 of 640 512 x 2 50 / - / -, 256 x 3 - / 21 / 38 (256 x 4 59 / 22 / 40); 4096 of 1024 512 x 2 43 / 18 / 31 (256 x 4 50 / 17 / 34); 4096 of 1536
            // 512 x 3 67 / 24 / 39 (1024 x 2 74 / 33 / 52); 4096 of 1792 1024 x 2 84 / - / -, 512 x 4 - / 34 / 57 (the other way round 97 / 47 / 68); 2000 of 3584 1024 x 4 94 / 31 / 67.
            if (pieces <= 64) return launch_rows<T, S, INTEGERS, 64, 1>(p, stream);
            if (pieces <= 128 && p.rows >= 1024) return launch_rows<T, S, INTEGERS, 64, 2>(p, stream);
            if constexpr (PLAIN) {
                if (pieces > 128 && pieces <= 256 && p.rows >= 1024) return launch_rows<T, S, INTEGERS, 128, 2>(p, stream);
            }
            if (pieces <= 256) return launch_rows<T, S, INTEGERS, 256, 1>(p, stream);
            if (pieces <= 512) return launch_rows<T, S, INTEGERS, PLAIN ? 256 : 512, PLAIN ? 2 : 1>(p, stream);
            if constexpr (!NORM) {
                if (pieces <= 768) return launch_rows<T, S, INTEGERS, 256, 3>(p, stream);
            }
            if (pieces <= 1024) return launch_rows<T, S, INTEGERS, 512, 2>(p, stream);
            if (pieces <= 1536) return launch_rows<T, S, INTEGERS, 512, 3>(p, stream);
            if constexpr (NORM) {
                if (pieces <= 2048) return launch_rows<T, S, INTEGERS, 1024, 2>(p, stream);
            } else {
                if (pieces <= 2048) return launch_rows<T, S, INTEGERS, 512, 4>(p, stream);
            }
            return launch_rows<T, S, INTEGERS, 1024, 4>(p, stream);
        }
    }
    hipLaunchKernelGGL((rows_any_kernel<T, S, INTEGERS>), dim3(p.rows < kMostRowBlocks ? p.rows : kMostRowBlocks), dim3(256), 0, stream, p);
    return launch_status("rows_any_kernel");
}

template <RowSource S, bool INTEGERS>
int run_rows(int dtype, const RowOperands& p, hipStream_t stream) {
    switch (dtype) {
        case TANNIC_FLOAT16: return run_rows<f16, S, INTEGERS>(p, stream);
        case TANNIC_BFLOAT16: return run_rows<bf16, S, INTEGERS>(p, stream);
        case TANNIC_FLOAT32: return run_rows<float, S, INTEGERS>(p, stream);
        case TANNIC_FLOAT64:
            if constexpr (!INTEGERS) return run_rows<double, S, INTEGERS>(p, stream);
        default: return TANNIC_UNSUPPORTED_DTYPE;
    }
}

// Rows and length of x [.., L]; what is too long for the kernels' 32-bit counts is refused.
int describe_rows(const tannic_tensor_t* x, RowOperands& p, const char* too_large) {
    const size_t length = x->shape.sizes[x->rank - 1];
    size_t rows = 1;
    for (int d = 0; d < x->rank - 1; ++d) {
        if (x->shape.sizes[d] >= (1ull << 31)) return refuse(too_large);
        rows *= x->shape.sizes[d];
        if (rows >= (1ull << 31)) return refuse(too_large);
    }
    if (length >= (1ull << 31)) return refuse(too_large);
    p.rows = static_cast<uint32_t>(rows);
    p.length = static_cast<uint32_t>(length);
    p.x = x->address;
    p.rows_x = rows_of(x);
    return TANNIC_SUCCESS;
}

}  // namespace th

using namespace th;

extern "C" {

int tannic_hip_add_rms_norm(const tannic_tensor_t* x, const tannic_tensor_t* residual, const tannic_tensor_t* gain, tannic_tensor_t* total, tannic_tensor_t* dst,
                            tannic_tensor_t* scales, tannic_stream_t stream, float eps) {
    if (!x || !gain || !dst) return refuse("add_rms_norm: a descriptor is missing");
    if ((residual == nullptr) != (total == nullptr)) return refuse("add_rms_norm: the sum is written where there is a residual, and only there");
    if (!have_storage(x, residual, gain, total, dst, scales)) return TANNIC_ERROR;
    if (!(quantizable(x->dtype) || (x->dtype == TANNIC_FLOAT64 && !scales)) || gain->dtype != x->dtype || (residual && (residual->dtype != x->dtype || total->dtype != x->dtype)) ||
        dst->dtype != (scales ? TANNIC_INT8 : x->dtype) || (scales && scales->dtype != TANNIC_FLOAT32))
        return TANNIC_UNSUPPORTED_DTYPE;
    if (x->rank < 1 || !extents_equal(x, dst) || !rows_contiguous(dst) || (residual && (!extents_equal(x, residual) || !extents_equal(x, total) || !rows_contiguous(total))))
        return refuse("add_rms_norm: x [.., L], the residual, the sum and dst have one shape, the sum and dst are contiguous");
    if (gain->rank != 1 || gain->shape.sizes[0] != x->shape.sizes[x->rank - 1] || !rows_contiguous(gain)) return refuse("add_rms_norm: gain [L], contiguous");
    if (scales && !scales_of(scales, dst)) return refuse("add_rms_norm: scales [..] for values [.., L], contiguous");
    RowOperands p{};
    if (int status = describe_rows(x, p, "add_rms_norm: 2^31 rows, rows of 2^31 elements or more are not supported")) return status;
    if (int status = on_device_of("add_rms_norm: the operands live on a device", x, residual, gain, total, dst, scales)) return status;
    if (p.rows == 0 || (p.length == 0 && !scales)) return TANNIC_SUCCESS;
    p.gain = gain->address;
    p.dst = dst->address;
    p.scales = scales ? static_cast<float*>(scales->address) : nullptr;
    p.eps = eps;
    if (residual) {
        p.second = residual->address;
        p.rows_second = rows_of(residual);
        p.total = total->address;
        return scales ? run_rows<RowSource::sum_norm, true>(x->dtype, p, as_stream(stream)) : run_rows<RowSource::sum_norm, false>(x->dtype, p, as_stream(stream));
    }
    return scales ? run_rows<RowSource::norm, true>(x->dtype, p, as_stream(stream)) : run_rows<RowSource::norm, false>(x->dtype, p, as_stream(stream));
}

int tannic_hip_quantize(const tannic_tensor_t* x, tannic_tensor_t* dst, tannic_tensor_t* scales, tannic_stream_t stream) {
    if (!x || !dst || !scales) return refuse("quantize: a descriptor is missing");
    if (!have_storage(x, dst, scales)) return TANNIC_ERROR;
    if (!quantizable(x->dtype) || dst->dtype != TANNIC_INT8 || scales->dtype != TANNIC_FLOAT32) return TANNIC_UNSUPPORTED_DTYPE;
    if (x->rank < 1 || !extents_equal(x, dst) || !rows_contiguous(dst) || !scales_of(scales, dst)) return refuse("quantize: x and dst [.., L], scales [..], the results contiguous");
    RowOperands p{};
    if (int status = describe_rows(x, p, "quantize: 2^31 rows, rows of 2^31 elements or more are not supported")) return status;
    if (int status = on_device_of("quantize: the operands live on a device", x, dst, scales)) return status;
    if (p.rows == 0) return TANNIC_SUCCESS;
    p.dst = dst->address;
    p.scales = static_cast<float*>(scales->address);
    return run_rows<RowSource::plain, true>(x->dtype, p, as_stream(stream));
}

int tannic_hip_swiglu_quantize(const tannic_tensor_t* gate, const tannic_tensor_t* up, tannic_tensor_t* dst, tannic_tensor_t* scales, tannic_stream_t stream) {
    if (!gate || !up || !dst || !scales) return refuse("swiglu_quantize: a descriptor is missing");
    if (!have_storage(gate, up, dst, scales)) return TANNIC_ERROR;
    if (!quantizable(gate->dtype) || up->dtype != gate->dtype || dst->dtype != TANNIC_INT8 || scales->dtype != TANNIC_FLOAT32) return TANNIC_UNSUPPORTED_DTYPE;
    if (gate->rank < 1 || !extents_equal(gate, up) || !extents_equal(gate, dst) || !rows_contiguous(dst) || !scales_of(scales, dst))
        return refuse("swiglu_quantize: gate, up and dst [.., L], scales [..], the results contiguous");
    RowOperands p{};
    if (int status = describe_rows(gate, p, "swiglu_quantize: 2^31 rows, rows of 2^31 elements or more are not supported")) return status;
    if (int status = on_device_of("swiglu_quantize: the operands live on a device", gate, up, dst, scales)) return status;
    if (p.rows == 0) return TANNIC_SUCCESS;
    p.second = up->address;
    p.rows_second = rows_of(up);
    p.dst = dst->address;
    p.scales = static_cast<float*>(scales->address);
    return run_rows<RowSource::gated, true>(gate->dtype, p, as_stream(stream));
}

int tannic_hip_dequantize(const tannic_tensor_t* values, const tannic_tensor_t* scales, tannic_tensor_t* dst, tannic_stream_t stream) {
    if (!values || !scales || !dst) return refuse("dequantize: a descriptor is missing");
    if (!have_storage(values, scales, dst)) return TANNIC_ERROR;
    if (values->dtype != TANNIC_INT8 || scales->dtype != TANNIC_FLOAT32 || !quantizable(dst->dtype)) return TANNIC_UNSUPPORTED_DTYPE;
    if (values->rank < 1 || !extents_equal(values, dst) || !rows_contiguous(dst) || !scales_of(scales, values))
        return refuse("dequantize: values and dst [.., L], scales [..], dst and scales contiguous");
    RowOperands p{};
    if (int status = describe_rows(values, p, "dequantize: 2^31 rows, rows of 2^31 elements or more are not supported")) return status;
    if (int status = on_device_of("dequantize: the operands live on a device", values, scales, dst)) return status;
    if (p.rows == 0 || p.length == 0) return TANNIC_SUCCESS;
    const auto run = [&](auto tag) {
        using T = typename decltype(tag)::type;
        const uint64_t per_row = (static_cast<uint64_t>(p.length) + 7) / 8, items = per_row * p.rows;
        if ((p.length == 1 || p.rows_x.step == 1) && items < (1ull << 31)) {
            const auto launch = [&](auto kernel) {
                hipLaunchKernelGGL(kernel, dim3(static_cast<uint32_t>((items + 255) / 256)), dim3(256), 0, as_stream(stream), static_cast<const int8_t*>(values->address), p.rows_x,
                                   static_cast<const float*>(scales->address), static_cast<T*>(dst->address), p.length, FastDiv(static_cast<uint32_t>(per_row)), static_cast<uint32_t>(items));
            };
            if (static_cast<uint64_t>(p.rows) * p.length * sizeof(T) > kRowsPastCaches) launch(dequantize_kernel<T, true>);
            else launch(dequantize_kernel<T, false>);
            return launch_status("dequantize_kernel");
        }
        hipLaunchKernelGGL((dequantize_any_kernel<T>), dim3(p.rows < kMostRowBlocks ? p.rows : kMostRowBlocks), dim3(256), 0, as_stream(stream),
                           static_cast<const int8_t*>(values->address), p.rows_x, static_cast<const float*>(scales->address), static_cast<T*>(dst->address), p.rows, p.length);
        return launch_status("dequantize_any_kernel");
    };
    if (dst->dtype == TANNIC_FLOAT16) return run(type_tag<f16>{});
    if (dst->dtype == TANNIC_BFLOAT16) return run(type_tag<bf16>{});
    return run(type_tag<float>{});
}

}  // extern "C"
