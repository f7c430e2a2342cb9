// Products of 8-bit integers with scales for more rows than a few: BM x BN tiles of 2 x 2 wavefronts on v_mfma_i32_16x16x64_i8.
//
// Both operands lie along K and come in steps of 128 bytes of a row, straight to LDS (16 bytes of a lane, 1 KB = eight rows of a load; the 16-byte pieces of a row in LDS are
// turned by the row, on the global side, so that the 16 rows of a fragment are read from different banks).  STAGES steps are in LDS or on their way.  A step multiplies the
// second half of the step before, whose fragments are in registers, and its own first half; behind the products of a half go the reads of the fragments for the next one, and
// behind those of the first half the loads of the step that takes the freed stage.  It ends with a wait for the next step's loads and one barrier.
// The weights are the first operand, so that a lane has four consecutive columns of one row: times the row's and the columns' scales, and to memory by whole rows through LDS (16 bits) or as they are.
// Blocks that share a tile's K leave whole numbers, which a second kernel adds up and scales, or for small tiles the last of the blocks that gets there.
#include <algorithm>

#include "attention.hpp"
#include "gemm_quantized.hpp"

namespace th {

struct SharedK {
    uint32_t splits, steps;      // blocks per tile; steps of 128 per block
    int* partials;               // for the second kernel [split][batch][M][pitch], for the last block [batch][tile][split][16 x 16 of a wavefront][thread][4]
    uint32_t pitch;
    uint32_t* arrivals;          // of a tile's blocks, 0 between calls
};
enum class Sharing { none, second_kernel, last_block };

// Sums pass from block to block, and between the L2 caches of the dies, through the memory both see: stores and loads of device scope, which no cache in between keeps.
__device__ inline void store_through(int* at, const int4v& v) {
    uint64_t bits[2];
    __builtin_memcpy(bits, &v, 16);
#pragma unroll
    for (int i = 0; i < 2; ++i) __hip_atomic_store(reinterpret_cast<uint64_t*>(at) + i, bits[i], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ inline int4v load_through(const int* at) {
    uint64_t bits[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) bits[i] = __hip_atomic_load(reinterpret_cast<const uint64_t*>(at) + i, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    int4v v;
    __builtin_memcpy(&v, bits, 16);
    return v;
}

// Leaves a block's sums for the others of its tile; true for the last of them, whose sums are all parts' then.
template <int TM, int TN>
__device__ inline bool add_parts(int4v (&acc)[TM][TN], const SharedK& shared, uint32_t split, uint32_t tile, unsigned char* lds) {
    int* const parts = shared.partials + (static_cast<size_t>(tile) * shared.splits * (TM * TN) * 256 + threadIdx.x) * 4;
    const auto of = [&](uint32_t part, int at) { return parts + (static_cast<size_t>(part) * (TM * TN) + at) * 1024; };
#pragma unroll
    for (int i = 0; i < TM; ++i)
#pragma unroll
        for (int j = 0; j < TN; ++j) store_through(of(split, i * TN + j), acc[i][j]);
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");      // (they have arrived)
    __syncthreads();
    uint32_t* const before = reinterpret_cast<uint32_t*>(lds);
    if (threadIdx.x == 0) {
        *before = __hip_atomic_fetch_add(shared.arrivals + tile, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        if (*before == shared.splits - 1) __hip_atomic_store(shared.arrivals + tile, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
    __syncthreads();
    if (*before != shared.splits - 1) return false;
    __syncthreads();      // (its place in LDS is used again)
    // the other parts, four on their way at a time (where there are not four, its own in their place, times 0)
    for (uint32_t from = 0; from < shared.splits; from += 4) {
        int4v got[4][TM][TN];
#pragma unroll
        for (uint32_t n = 0; n < 4; ++n)
#pragma unroll
            for (int i = 0; i < TM; ++i)
#pragma unroll
                for (int j = 0; j < TN; ++j) got[n][i][j] = load_through(of(from + n < shared.splits ? from + n : split, i * TN + j));
#pragma unroll
        for (uint32_t n = 0; n < 4; ++n) {
            const int counts = from + n < shared.splits && from + n != split;
#pragma unroll
            for (int i = 0; i < TM; ++i)
#pragma unroll
                for (int j = 0; j < TN; ++j) acc[i][j] += got[n][i][j] * counts;
        }
    }
    return true;
}

// A wavefront's TM x TN sums of 16 x 16 from row `row0` and column `col0` on: as they are, into its share of the partial sums.
template <int TM, int TN>
__device__ inline void leave_sums(const int4v (&acc)[TM][TN], const GemmProblem& p, const SharedK& shared, uint32_t split, uint32_t row0, uint32_t col0) {
    const uint32_t lane = threadIdx.x % 64;
    int* const mine = shared.partials + (static_cast<size_t>(split) * p.batches + blockIdx.y) * p.M * shared.pitch;
#pragma unroll
    for (int i = 0; i < TM; ++i) {
        const uint32_t row = row0 + i * 16 + lane % 16;
#pragma unroll
        for (int j = 0; j < TN; ++j) {
            const uint32_t col = col0 + j * 16 + 4 * (lane / 16);
            if (row < p.M && col < p.N) *reinterpret_cast<int4v*>(mine + static_cast<size_t>(row) * shared.pitch + col) = acc[i][j];
        }
    }
}

// The same scaled and rounded, into the product; `mine`: the wavefront's own part of LDS, in which 16-bit results become whole rows (16 bytes of a lane).
template <class D, int TM, int TN>
__device__ inline void write_scaled(const int4v (&acc)[TM][TN], D* mine, D* c, const GemmProblem& p, const ScalePlaces& s, uint32_t row0, uint32_t col0) {
    const uint32_t lane = threadIdx.x % 64;
    const float *scale_a, *scale_b;
    scale_offsets(p, s, blockIdx.y, scale_a, scale_b);
    float sb[TN][4];
#pragma unroll
    for (int j = 0; j < TN; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const uint32_t col = col0 + j * 16 + 4 * (lane / 16) + e;
            sb[j][e] = scale_b[(col < p.N ? col : p.N - 1) * s.b_step];
        }
    constexpr int WM = TM * 16, WN = TN * 16, PITCH = WN + 8;
#pragma unroll
    for (int i = 0; i < TM; ++i) {
        const uint32_t row = row0 + i * 16 + lane % 16;
        const float sa = scale_a[(row < p.M ? row : p.M - 1) * s.a_step];
#pragma unroll
        for (int j = 0; j < TN; ++j) {
            float out[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) out[e] = static_cast<float>(acc[i][j][e]) * sa * sb[j][e];
            const uint32_t col = col0 + j * 16 + 4 * (lane / 16);
            if constexpr (sizeof(D) == 4) {
                if (row < p.M && col < p.N) store_four<D>(c + static_cast<int64_t>(row) * p.c_rs + col, out, p.N - col);
            } else {
                D narrow[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) narrow[e] = rounded<D>(out[e]);
                uint2 bits;
                __builtin_memcpy(&bits, narrow, 8);
                *reinterpret_cast<uint2*>(mine + (i * 16 + lane % 16) * PITCH + j * 16 + 4 * (lane / 16)) = bits;
            }
        }
    }
    if constexpr (sizeof(D) == 2) {
        constexpr int PIECES = WN / 8, LANES = PIECES <= 2 ? 2 : PIECES <= 4 ? 4 : PIECES <= 8 ? 8 : 16, ROWS = 64 / LANES;      // of a row; of a pass
        const uint32_t piece = lane % LANES, col = col0 + piece * 8;
        if (piece < PIECES && col < p.N) {
#pragma unroll
            for (int r0 = 0; r0 < WM; r0 += ROWS) {
                const uint32_t r = r0 + lane / LANES, row = row0 + r;
                if (r < WM && row < p.M) {
                    const uint4v bits = *reinterpret_cast<const uint4v*>(mine + r * PITCH + piece * 8);
                    store_piece_anywhere(c + static_cast<int64_t>(row) * p.c_rs + col, &bits, p.N - col < 8 ? p.N - col : 8);
                }
            }
        }
    }
}

template <class D, int BM, int BN, int STAGES, int PER_CU, Sharing SHARING>
__global__ __launch_bounds__(256, PER_CU) void gemm_quantized_tile_kernel(const int8_t* A, const int8_t* B, D* C, GemmProblem p, ScalePlaces s, uint32_t tiles_m, uint32_t tiles_n, SharedK shared) {
#if defined(__HIP_DEVICE_COMPILE__)
    constexpr bool SPLIT = SHARING != Sharing::none;
    constexpr int WM = BM / 2, WN = BN / 2, TM = WM / 16, TN = WN / 16;
    constexpr uint32_t A_TILE = BM * 128, B_TILE = BN * 128, STAGE = A_TILE + B_TILE;      // bytes
    constexpr int LOADS_A = BM / 32, LOADS_B = BN / 32, LOADS = LOADS_A + LOADS_B;         // of 1 KB, per wavefront and step
    extern __shared__ __align__(16) unsigned char lds[];

    uint32_t tm, tn;
    const uint32_t split = SPLIT ? blockIdx.x % shared.splits : 0;
    tile_of<true>(SPLIT ? blockIdx.x / shared.splits : blockIdx.x, tiles_m, tiles_n, tm, tn);
    int64_t oa, ob, oc;
    batch_offsets(p, blockIdx.y, oa, ob, oc);
    const uint32_t m0 = tm * BM, n0 = tn * BN;
    const uint32_t all = (p.K + 127) / 128, first = SPLIT ? split * shared.steps : 0;
    const uint32_t steps = SPLIT ? (all - first < shared.steps ? all - first : shared.steps) : all;

    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64), lane = threadIdx.x % 64;
    const uint32_t wm = wave / 2 * WM, wn = wave % 2 * WN, frag_row = lane % 16, frag_piece = lane / 16;
    const uint32_t rows_a = p.M - m0 < BM ? p.M - m0 : BM, rows_b = p.N - n0 < BN ? p.N - n0 : BN;
    const __amdgpu_buffer_rsrc_t rsrc_a =
        __builtin_amdgcn_make_buffer_rsrc(const_cast<int8_t*>(A + oa + static_cast<int64_t>(m0) * p.a_rs), 0, bytes_of_rows(rows_a, p.a_rs, p.K), 0x00020000);
    const __amdgpu_buffer_rsrc_t rsrc_b =
        __builtin_amdgcn_make_buffer_rsrc(const_cast<int8_t*>(B + ob + static_cast<int64_t>(n0) * p.b_cs), 0, bytes_of_rows(rows_b, p.b_cs, p.K), 0x00020000);
    // load j of a wavefront fills 1 KB of a stage (j < LOADS_A: of A's tile): the lane's row and its (turned) piece; rows that are not there are beyond the buffer's range
    uint32_t voff[LOADS];
    const uint32_t turned = (lane % 8) ^ ((lane >> 4) & 3u);      // (rows 8 j + lane / 8: (row / 2) % 8 is (lane / 16) % 4 and 4 for odd j)
#pragma unroll
    for (int j = 0; j < LOADS; ++j) {
        const bool of_a = j < LOADS_A;
        const uint32_t block = of_a ? wave * LOADS_A + j : wave * LOADS_B + (j - LOADS_A), row = block * 8 + lane / 8;
        voff[j] = row < (of_a ? rows_a : rows_b) ? row * static_cast<uint32_t>(of_a ? p.a_rs : p.b_cs) + (turned ^ (block % 2 * 4)) * 16 : kBeyond;
    }
    const auto issue = [&](int j, uint32_t stage, uint32_t step) {
        const bool of_a = j < LOADS_A;
        const uint32_t block = of_a ? wave * LOADS_A + j : wave * LOADS_B + (j - LOADS_A), k = (first + step) * 128;
        uint32_t offset = voff[j];
        // (a step that K ends in: zeros behind it)
        if (k + 128 > p.K && k + (turned ^ (block % 2 * 4)) * 16 >= p.K) offset = kBeyond;
        __builtin_amdgcn_raw_ptr_buffer_load_lds(of_a ? rsrc_a : rsrc_b, (lds_address)(lds + stage * STAGE + (of_a ? 0 : A_TILE) + block * 1024), 16, offset, k, 0, 0);
    };

    int4v acc[TM][TN];
#pragma unroll
    for (int i = 0; i < TM; ++i)
#pragma unroll
        for (int j = 0; j < TN; ++j) acc[i][j] = int4v{0, 0, 0, 0};

    // loads complete in order: with at most AHEAD of them outstanding the next step's are in
    constexpr int AHEAD = (STAGES - 2) * LOADS;
    const auto wait_loads = [](bool every) {
        if (every) asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        else asm volatile("s_waitcnt vmcnt(%0)" ::"n"(AHEAD) : "memory");
    };
    // own reads of LDS done, then everybody's (a fence would also wait for the loads on their way)
    const auto meet = [] {
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
    };
#pragma unroll
    for (int t = 0; t < STAGES - 1; ++t) {
        if (static_cast<uint32_t>(t) < steps) {
#pragma unroll
            for (int j = 0; j < LOADS; ++j) issue(j, t, t);
        }
    }
    wait_loads(steps < static_cast<uint32_t>(STAGES - 1));
    meet();

    constexpr int PRODUCTS = TM * TN;      // of a half
    constexpr int LOAD_EVERY = PRODUCTS / LOADS > 0 ? PRODUCTS / LOADS : 1;
    constexpr int READ_EVERY = PRODUCTS / (TM + TN) > 0 ? PRODUCTS / (TM + TN) : 1;
    uint4v fa[2][TM], fb[2][TN];
    const auto fragment = [&](const unsigned char* tile, uint32_t row, int half) { return *reinterpret_cast<const uint4v*>(tile + tile_offset<int8_t>(row + frag_row, half * 4 + frag_piece)); };
    // read n of a half's fragments: the first of A and all of B, which the first products want, then the others
    const auto read = [&](const unsigned char* stage, int half, int n) {
        if (n == 0) fa[half][0] = fragment(stage, wm, half);
        else if (n <= TN) fb[half][n - 1] = fragment(stage + A_TILE, wn + (n - 1) * 16, half);
        else fa[half][n - TN] = fragment(stage, wm + (n - TN) * 16, half);
    };
    const auto step = [&](uint32_t at, uint32_t now, uint32_t fill, auto first_tag, auto fetch_tag) {      // now: the stage of step `at`; fill: the one that is free
        constexpr bool FIRST = decltype(first_tag)::value, FETCH = decltype(fetch_tag)::value;
        const unsigned char* const stage = lds + now * STAGE;
        if constexpr (FIRST) {
#pragma unroll
            for (int n = 0; n < TM + TN; ++n) read(stage, 0, n);
        }
        __builtin_amdgcn_sched_barrier(0);
        static_for<2 * PRODUCTS>([&](auto tag) {
            constexpr int m = decltype(tag)::value, half = m / PRODUCTS, q = m % PRODUCTS, i = q / TN, j = q % TN;
            constexpr bool multiplies = !(FIRST && half == 0);
            if constexpr (multiplies) acc[i][j] = mfma_i8(fb[1 - half][j], fa[1 - half][i], acc[i][j]);
            // (a half with fewer products than reads has several behind each)
            if constexpr (multiplies) {
                constexpr int from = q * (TM + TN) / PRODUCTS, to = (q + 1) * (TM + TN) / PRODUCTS;
                if constexpr (PRODUCTS >= TM + TN) {
                    if constexpr (q % READ_EVERY == 0 && q / READ_EVERY < TM + TN) read(stage, half, q / READ_EVERY);
                } else {
#pragma unroll
                    for (int n = from; n < to; ++n) read(stage, half, n);
                }
            }
            constexpr int slot = FIRST ? m - PRODUCTS : m;
            if constexpr (FETCH && slot >= 0 && slot < PRODUCTS) {
                if constexpr (PRODUCTS >= LOADS) {
                    if constexpr (slot % LOAD_EVERY == LOAD_EVERY / 2 && slot / LOAD_EVERY < LOADS) issue(slot / LOAD_EVERY, fill, at + STAGES - 1);
                } else {
#pragma unroll
                    for (int n = slot * LOADS / PRODUCTS; n < (slot + 1) * LOADS / PRODUCTS; ++n) issue(n, fill, at + STAGES - 1);
                }
            }
            __builtin_amdgcn_sched_barrier(0);
        });
        wait_loads(!FETCH);
        meet();
    };
    using Yes = std::true_type;
    using No = std::false_type;
    const auto next = [](uint32_t stage) { return stage + 1 == STAGES ? 0u : stage + 1; };
    uint32_t at = 0, now = 0, fill = STAGES - 1;
    if (steps > STAGES - 1) step(0, now, fill, Yes{}, Yes{});
    else step(0, now, fill, Yes{}, No{});
    for (at = 1, now = next(now), fill = next(fill); at + STAGES - 1 < steps; ++at, now = next(now), fill = next(fill)) step(at, now, fill, No{}, Yes{});
    for (; at < steps; ++at, now = next(now), fill = next(fill)) step(at, now, fill, No{}, No{});
#pragma unroll
    for (int i = 0; i < TM; ++i)
#pragma unroll
        for (int j = 0; j < TN; ++j) acc[i][j] = mfma_i8(fb[1][j], fa[1][i], acc[i][j]);

    if constexpr (SHARING == Sharing::last_block) {
        if (!add_parts<TM, TN>(acc, shared, split, blockIdx.y * tiles_m * tiles_n + blockIdx.x / shared.splits, lds)) return;
    }
    if constexpr (SHARING == Sharing::second_kernel) leave_sums<TM, TN>(acc, p, shared, split, m0 + wm, n0 + wn);
    else write_scaled<D, TM, TN>(acc, reinterpret_cast<D*>(lds) + wave * (WM * (WN + 8)), C + oc, p, s, m0 + wm, n0 + wn);
#endif
}

// Rows along K that start anywhere and have any length from 16 on: tiles of BM x 64 on the same 2 x 2 wavefronts, whose pieces go through registers, up to three steps ahead of the products; LDS
// holds two steps.  The last piece of a row that is not whole pieces is its last 16 bytes, of which A's have zeros for those that the piece before has: a whole number of
// products is left out by zeros of one operand, whatever the other holds.  Bound by its loads and writes to LDS, and by the latency of a step where blocks are few; what it saves is copying both
// operands into aligned rows (us with the copies / so: 77 x 2049 x 1030
// 11.7 / 7.1, 1 x 28672 x 4095 60.6 / 31.2, 64 x 4096 x 4095 21.5 / 14.0; 2048 x 4096 x 4095 53 / 117, which are copied).
template <class D, int BM, Sharing SHARING>
__global__ __launch_bounds__(256, 2) void gemm_quantized_bytes_kernel(const int8_t* A, const int8_t* B, D* C, GemmProblem p, ScalePlaces s, uint32_t tiles_m, uint32_t tiles_n, SharedK shared) {
    constexpr bool SPLIT = SHARING != Sharing::none;
    constexpr int BN = 64, WM = BM / 2, WN = BN / 2, TM = WM / 16, TN = WN / 16, LOADS_A = BM / 32, LOADS = LOADS_A + BN / 32;
    constexpr uint32_t A_TILE = BM * 128, STAGE = A_TILE + BN * 128, OUT = sizeof(D) == 2 ? 2 * 4 * WM * (WN + 8) : 0;
    __shared__ __align__(16) unsigned char lds[2 * STAGE > OUT ? 2 * STAGE : OUT];
    uint32_t tm, tn;
    const uint32_t split = SPLIT ? blockIdx.x % shared.splits : 0;
    tile_of<true>(SPLIT ? blockIdx.x / shared.splits : blockIdx.x, tiles_m, tiles_n, tm, tn);
    int64_t oa, ob, oc;
    batch_offsets(p, blockIdx.y, oa, ob, oc);
    const uint32_t m0 = tm * BM, n0 = tn * BN;
    const uint32_t all = (p.K + 127) / 128, first = SPLIT ? split * shared.steps : 0;
    const uint32_t steps = SPLIT ? (all - first < shared.steps ? all - first : shared.steps) : all;
    const uint32_t wave = threadIdx.x / 64, lane = threadIdx.x % 64;
    const uint32_t wm = wave / 2 * WM, wn = wave % 2 * WN, frag_row = lane % 16, frag_piece = lane / 16;
    // load j: piece threadIdx.x % 8 of rows 32 j + threadIdx.x / 8 of A's tile, then of B's
    const uint32_t piece = threadIdx.x % 8, row = threadIdx.x / 8;
    const int8_t* from[LOADS];
    bool there[LOADS];
#pragma unroll
    for (int j = 0; j < LOADS; ++j) {
        const uint32_t r = (j < LOADS_A ? m0 + j * 32 : n0 + (j - LOADS_A) * 32) + row;
        there[j] = r < (j < LOADS_A ? p.M : p.N);
        from[j] = j < LOADS_A ? A + oa + static_cast<int64_t>(there[j] ? r : 0) * p.a_rs : B + ob + static_cast<int64_t>(there[j] ? r : 0) * p.b_cs;
    }
    typedef unsigned int uint4any __attribute__((ext_vector_type(4), aligned(1)));
    uint4v held[2][LOADS];
    const auto load = [&](uint32_t step, auto set_tag) {
        constexpr int set = decltype(set_tag)::value;
        const uint32_t want = (first + step) * 128 + piece * 16;
        const uint32_t k = want + 16 <= p.K ? want : p.K - 16, twice = want < p.K ? want - k : 16;      // bytes that the piece before has
#pragma unroll
        for (int j = 0; j < LOADS; ++j) {
            held[set][j] = uint4v{0, 0, 0, 0};
            if (there[j] && want < p.K) {
                const uint4any bits = *reinterpret_cast<const uint4any*>(from[j] + k);
                held[set][j] = uint4v{bits[0], bits[1], bits[2], bits[3]};
            }
            if (j < LOADS_A && twice != 0) {
#pragma unroll
                for (uint32_t e = 0; e < 4; ++e) {
                    const uint32_t zeros = twice <= 4 * e ? 0u : twice - 4 * e >= 4 ? 4u : twice - 4 * e;      // of the word's bytes
                    held[set][j][e] = zeros == 4 ? 0u : held[set][j][e] >> (8 * zeros) << (8 * zeros);
                }
            }
        }
    };
    const auto keep = [&](auto set_tag) {      // a set's step goes to the stage of its number
        constexpr int set = decltype(set_tag)::value;
#pragma unroll
        for (int j = 0; j < LOADS; ++j) {
            const uint32_t r = (j < LOADS_A ? j : j - LOADS_A) * 32 + row;
            *reinterpret_cast<uint4v*>(lds + set * STAGE + (j < LOADS_A ? 0 : A_TILE) + tile_offset<int8_t>(r, piece)) = held[set][j];
        }
    };
    int4v acc[TM][TN];
#pragma unroll
    for (int i = 0; i < TM; ++i)
#pragma unroll
        for (int j = 0; j < TN; ++j) acc[i][j] = int4v{0, 0, 0, 0};
    using Even = std::integral_constant<int, 0>;
    using Odd = std::integral_constant<int, 1>;
    // step `at` from the stage of its number, the next one's operands into the other, those of the third behind it on their way
    const auto step = [&](uint32_t at, auto here, auto next) {
        const unsigned char* const stage = lds + decltype(here)::value * STAGE;
        if (at + 1 < steps) keep(next);
        if (at + 3 < steps) load(at + 3, next);
#pragma unroll
        for (int half = 0; half < 2; ++half) {
            uint4v fa[TM], fb[TN];
#pragma unroll
            for (int i = 0; i < TM; ++i) fa[i] = *reinterpret_cast<const uint4v*>(stage + tile_offset<int8_t>(wm + i * 16 + frag_row, half * 4 + frag_piece));
#pragma unroll
            for (int j = 0; j < TN; ++j) fb[j] = *reinterpret_cast<const uint4v*>(stage + A_TILE + tile_offset<int8_t>(wn + j * 16 + frag_row, half * 4 + frag_piece));
#pragma unroll
            for (int i = 0; i < TM; ++i)
#pragma unroll
                for (int j = 0; j < TN; ++j) acc[i][j] = mfma_i8(fb[j], fa[i], acc[i][j]);
        }
        __syncthreads();
    };
    load(0, Even{});
    if (steps > 1) load(1, Odd{});
    keep(Even{});
    if (steps > 2) load(2, Even{});
    __syncthreads();
    for (uint32_t at = 0; at < steps; at += 2) {
        step(at, Even{}, Odd{});
        if (at + 1 < steps) step(at + 1, Odd{}, Even{});
    }
    if constexpr (SPLIT) {
        if (!add_parts<TM, TN>(acc, shared, split, blockIdx.y * tiles_m * tiles_n + blockIdx.x / shared.splits, lds)) return;
    }
    write_scaled<D, TM, TN>(acc, reinterpret_cast<D*>(lds) + wave * (WM * (WN + 8)), C + oc, p, s, m0 + wm, n0 + wn);
}

// The sums of the blocks that shared K, scaled: four columns of a row per thread.
template <class D>
__global__ __launch_bounds__(256) void gemm_quantized_join_kernel(D* C, GemmProblem p, ScalePlaces s, SharedK shared, FastDiv per_row, uint32_t items) {
    const uint32_t item = blockIdx.x * 256 + threadIdx.x;
    if (item >= items) return;
    uint32_t row, col;
    per_row.divmod(item, row, col);
    col *= 4;
    int64_t oa, ob, oc;
    batch_offsets(p, blockIdx.y, oa, ob, oc);
    const float *scale_a, *scale_b;
    scale_offsets(p, s, blockIdx.y, scale_a, scale_b);
    const size_t apart = static_cast<size_t>(p.batches) * p.M * shared.pitch;
    const int* from = shared.partials + (static_cast<size_t>(blockIdx.y) * p.M + row) * shared.pitch + col;
    int4v sum = *reinterpret_cast<const int4v*>(from);
    for (uint32_t i = 1; i < shared.splits; ++i) sum += *reinterpret_cast<const int4v*>(from + i * apart);
    const float sa = scale_a[row * s.a_step];
    float out[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) out[e] = static_cast<float>(sum[e]) * sa * scale_b[(col + e < p.N ? col + e : col) * s.b_step];
    store_four<D>(C + oc + static_cast<int64_t>(row) * p.c_rs + col, out, p.N - col);
}

template <class D, int BM, int BN, int STAGES, Sharing SHARING = Sharing::second_kernel>
static int launch_tiles(const GemmProblem& p, const ScalePlaces& s, uint32_t splits, const void* a, const void* b, void* c, hipStream_t stream) {
    const uint32_t tiles_m = (p.M + BM - 1) / BM, tiles_n = (p.N + BN - 1) / BN, steps = (p.K + 127) / 128;
    constexpr size_t tile_bytes = static_cast<size_t>(STAGES) * (BM + BN) * 128, out_bytes = sizeof(D) == 2 ? 2 * 4 * (BM / 2) * (BN / 2 + 8) : 0;
    constexpr size_t lds_bytes = tile_bytes > out_bytes ? tile_bytes : out_bytes;
    static_assert(lds_bytes <= 160 * 1024);
    constexpr int PER_CU = lds_bytes <= 80 * 1024 ? 2 : 1;
    SharedK shared{splits, (steps + splits - 1) / splits, nullptr, (p.N + 3) / 4 * 4, nullptr};
    shared.splits = (steps + shared.steps - 1) / shared.steps;      // (none without a step)
    const auto run = [&](auto kernel, std::atomic<uint64_t>& configured) {
        if (int rc = raise_lds_limit(reinterpret_cast<const void*>(kernel), lds_bytes, configured)) return rc;
        hipLaunchKernelGGL(kernel, dim3(tiles_m * tiles_n * shared.splits, p.batches), dim3(256), lds_bytes, stream, static_cast<const int8_t*>(a), static_cast<const int8_t*>(b),
                           static_cast<D*>(c), p, s, tiles_m, tiles_n, shared);
        return launch_status("gemm_quantized_tile_kernel");
    };
    static std::atomic<uint64_t> configured{0}, configured_split{0};
    if (shared.splits == 1) return run(gemm_quantized_tile_kernel<D, BM, BN, STAGES, PER_CU, Sharing::none>, configured);
    static_assert(kAttentionArrivals >= 256);
    void* held = nullptr;
    const size_t results = SHARING == Sharing::last_block ? static_cast<size_t>(tiles_m) * tiles_n * BM * BN : static_cast<size_t>(p.M) * shared.pitch;
    if (SHARING == Sharing::last_block)
        if (int status = attention_arrivals(stream, shared.arrivals)) return status;
    if (scratch_acquire(&held, shared.splits * p.batches * results * sizeof(int), stream) != TANNIC_SUCCESS) return TANNIC_ERROR;
    shared.partials = static_cast<int*>(held);
    int status = run(gemm_quantized_tile_kernel<D, BM, BN, STAGES, PER_CU, SHARING>, configured_split);
    if (SHARING == Sharing::second_kernel && status == TANNIC_SUCCESS) {
        const uint32_t per_row = shared.pitch / 4, items = p.M * per_row;
        hipLaunchKernelGGL((gemm_quantized_join_kernel<D>), dim3((items + 255) / 256, p.batches), dim3(256), 0, stream, static_cast<D*>(c), p, s, shared, FastDiv(per_row), items);
        status = launch_status("gemm_quantized_join_kernel");
    }
    scratch_release(held, stream);
    return status;
}

// The kernel's tiles: rows, columns, us of a step of 128 with the chip full of them (and of a block that has a compute unit alone, where that is more), us that a block takes beside its
// steps, us that the last of the blocks that share a tile takes for each of their parts (0: a second kernel adds them up).  Two blocks of the last three are on a compute unit at a time and share
// its step times.  Of the 0.50 us of a 128 x 128 step LDS takes 0.35 (32 KB of what is loaded 0.24, 64 KB of fragments 0.20), and no pipe is busy most of it: a SIMD has one wavefront, which
// issues 45 % of the time, waits 35 % for loads, fragments and the others and 20 % for a pipe (counted for 128 x 96; the matrix pipe is busy 30 %, LDS with fragments 19 %).  The largest tile is
// bound by the matrix pipe under the chip's power limit (256 x 256 1.4 us, 3.1 POP/s; MFMAs alone on such values 1.3).  Measured with weights from
// memory: 31 products of 33 to 8000 rows, each tile and up to 16 splits; what comes out first below is within 7 % of the fastest found.
struct Tiles8 {
    uint32_t rows, columns;
    double step, beside, join, alone;
};
constexpr Tiles8 kTiles8[] = {{256, 256, 1.40, 15.0, 0, 0}, {256, 192, 1.13, 12.0, 0, 0}, {256, 128, 0.84, 6.0, 0, 0}, {128, 128, 0.50, 4.0, 0, 0},
                              {128, 96, 0.47, 3.2, 0, 0},   {64, 128, 0.38, 1.1, 0, 0},   {64, 64, 0.235, 0.7, 0.48, 0}, {32, 64, 0.18, 0.6, 0.37, 0}};

struct Choice8 {
    int tile;
    uint32_t splits;
    double cost;
};

template <uint32_t N> using Parts = std::integral_constant<uint32_t, N>;      // (a number that is divided by, known to the compiler)

// The least us of a product by this: the blocks of the busiest compute unit one after another, and the weights from memory, most of the shorter one beside the longer; then the sums of blocks
// that share K.  (Every product goes through it: 0.2 us of a call.)
static Choice8 choose_tiles8(const GemmProblem& p, const Tiles8* tiles, int count) {
    const uint32_t steps = (p.K + 127) / 128, most_parts = p.K / 512;      // (of four steps and more)
    const double loaded = 1.5 + static_cast<double>(p.N) * p.K / 5.2e6, results = 8.0 / 6e6 * p.M * p.N * p.batches;
    Choice8 best{0, 1, -1.0};
    for (int t = 0; t < count; ++t) {
        const Tiles8& tile = tiles[t];
        const uint64_t blocks = static_cast<uint64_t>((p.M - 1) / tile.rows + 1) * ((p.N - 1) / tile.columns + 1) * p.batches;
        if (blocks >= kMostBlocks) continue;      // (a launch has fewer)
        const auto of = [&](auto splits) {
            const double rounds = static_cast<double>(static_cast<int64_t>((blocks * splits + 255) / 256)), of_step = std::max(rounds * tile.step, tile.alone);
            const double multiplied = 3.0 + static_cast<int>((steps + splits - 1) / splits) * of_step + rounds * tile.beside;
            const double joined = splits == 1 ? 0.0 : tile.join > 0 ? 1.0 + tile.join * splits : 2.5 + results * splits;
            const double cost = std::max(multiplied, loaded) + 0.3 * std::min(multiplied, loaded) + joined;
            if (best.cost < 0 || cost < best.cost) best = Choice8{t, splits, cost};
        };
        of(Parts<1>{});
        // (parts so many that they are all there at once: 512, half as many tiles at most, which there are counts of arrivals for)
        const uint32_t most = blocks > 256 ? 1 : static_cast<uint32_t>(std::min<uint64_t>(most_parts, 512 / static_cast<uint32_t>(blocks)));
        const auto each = [&](auto... splits) { ((splits <= most ? of(splits) : void()), ...); };
        each(Parts<2>{}, Parts<3>{}, Parts<4>{}, Parts<6>{}, Parts<8>{}, Parts<12>{}, Parts<16>{});
    }
    return best;
}

template <class D>
int gemm_quantized_tile(const GemmProblem& p, const ScalePlaces& s, const void* a, const void* b, void* c, hipStream_t stream) {
    if (!gemm_quantized_tile_takes(p, a, b)) return TANNIC_UNSUPPORTED_DTYPE;
    const Choice8 choice = choose_tiles8(p, kTiles8, 8);
    switch (choice.tile) {
        case 0: return launch_tiles<D, 256, 256, 2>(p, s, choice.splits, a, b, c, stream);
        case 1: return launch_tiles<D, 256, 192, 2>(p, s, choice.splits, a, b, c, stream);
        case 2: return launch_tiles<D, 256, 128, 3>(p, s, choice.splits, a, b, c, stream);
        case 3: return launch_tiles<D, 128, 128, 4>(p, s, choice.splits, a, b, c, stream);
        case 4: return launch_tiles<D, 128, 96, 5>(p, s, choice.splits, a, b, c, stream);
        case 5: return launch_tiles<D, 64, 128, 3>(p, s, choice.splits, a, b, c, stream);
        case 6: return launch_tiles<D, 64, 64, 5, Sharing::last_block>(p, s, choice.splits, a, b, c, stream);
        default: return launch_tiles<D, 32, 64, 6, Sharing::last_block>(p, s, choice.splits, a, b, c, stream);
    }
}

template <class D, int BM>
static int launch_bytes(const GemmProblem& p, const ScalePlaces& s, uint32_t splits, const void* a, const void* b, void* c, hipStream_t stream) {
    const uint32_t tiles_m = (p.M + BM - 1) / BM, tiles_n = (p.N + 63) / 64, steps = (p.K + 127) / 128;
    SharedK shared{splits, (steps + splits - 1) / splits, nullptr, 0, nullptr};
    shared.splits = (steps + shared.steps - 1) / shared.steps;
    void* held = nullptr;
    if (shared.splits > 1) {
        if (int status = attention_arrivals(stream, shared.arrivals)) return status;
        if (scratch_acquire(&held, static_cast<size_t>(shared.splits) * p.batches * tiles_m * tiles_n * BM * 64 * sizeof(int), stream) != TANNIC_SUCCESS) return TANNIC_ERROR;
        shared.partials = static_cast<int*>(held);
    }
    const auto run = [&](auto kernel) {
        hipLaunchKernelGGL(kernel, dim3(tiles_m * tiles_n * shared.splits, p.batches), dim3(256), 0, stream, static_cast<const int8_t*>(a), static_cast<const int8_t*>(b), static_cast<D*>(c), p,
                           s, tiles_m, tiles_n, shared);
        return launch_status("gemm_quantized_bytes_kernel");
    };
    const int status = shared.splits > 1 ? run(gemm_quantized_bytes_kernel<D, BM, Sharing::last_block>) : run(gemm_quantized_bytes_kernel<D, BM, Sharing::none>);
    if (held) scratch_release(held, stream);
    return status;
}

// The tiles for rows that start anywhere, times as above; four blocks and more on a compute unit share its loads, one alone is not faster than `alone`.
constexpr Tiles8 kBytes8[] = {{64, 64, 0.44, 0.7, 0.48, 0.75}, {32, 64, 0.345, 0.6, 0.37, 0.64}};

static bool choose_bytes8(const GemmProblem& p, bool or_copies, Choice8& choice) {
    if (p.a_cs != 1 || p.b_rs != 1 || p.K < 16 || !few_enough_blocks(p, 64, 64)) return false;
    choice = choose_tiles8(p, kBytes8, 2);
    if (!or_copies) return true;
    // where copies and the tiles of aligned rows are faster those take it: two launches of about 3 us, a read and a write of both operands (and no product is shorter than 4 us)
    const double copies = 6.0 + 2.0 * (static_cast<double>(p.M) + p.N) * p.K * p.batches / 4.5e6;
    GemmProblem q = p;
    q.K = (p.K + 127) / 128 * 128;
    return !(choice.cost > copies + 4.0 && choice.cost > copies + choose_tiles8(q, kTiles8, 8).cost);
}

template <class D> bool gemm_quantized_bytes_takes(const GemmProblem& p, bool or_copies) {
    Choice8 choice;
    return choose_bytes8(p, or_copies, choice);
}

template <class D>
int gemm_quantized_bytes(const GemmProblem& p, bool or_copies, const ScalePlaces& s, const void* a, const void* b, void* c, hipStream_t stream) {
    Choice8 choice;
    if (!choose_bytes8(p, or_copies, choice)) return TANNIC_UNSUPPORTED_DTYPE;
    return choice.tile == 0 ? launch_bytes<D, 64>(p, s, choice.splits, a, b, c, stream) : launch_bytes<D, 32>(p, s, choice.splits, a, b, c, stream);
}

// This file is compiled once for each type of results (TH_TILE_TYPE).
#ifndef TH_TILE_TYPE
#define TH_TILE_TYPE bf16
#endif
template int gemm_quantized_tile<TH_TILE_TYPE>(const GemmProblem&, const ScalePlaces&, const void*, const void*, void*, hipStream_t);
template bool gemm_quantized_bytes_takes<TH_TILE_TYPE>(const GemmProblem&, bool);
template int gemm_quantized_bytes<TH_TILE_TYPE>(const GemmProblem&, bool, const ScalePlaces&, const void*, const void*, void*, hipStream_t);

}  // namespace th
