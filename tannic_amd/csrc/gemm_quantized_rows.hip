// Products of 8-bit integers with scales for up to 32 rows (tokens) and columns enough to fill the chip once: the weights go by once, which is the work (1 row of 4096 x 14336
// from memory 11.5 us, 5.1 TB/s; the kernel's start and end, its first window and the meeting of its wavefronts are 3 us of any of them: 4096 x 4096 6.2 us, 2.7 TB/s).
//
// A block has 16 NB columns (rows of W, which lie along K), its four wavefronts share K in windows of 128 bytes.  A wavefront has a ring of windows in LDS of its own,
// filled by direct global -> LDS loads of whole 128-byte lines (eight lanes a row; the 16-byte pieces of a row in LDS are turned by the row, on the global side, so that the
// 16 rows of a fragment are read from different banks), all but one of them on their way; v_mfma_i32_16x16x64_i8 takes 16 columns and 16 rows.  The
// wavefronts' sums, whole numbers, meet in LDS.
#include "gemm_quantized.hpp"

namespace th {

constexpr int kRowWaves = 4;
constexpr int kRowBytesPerWave = 32 * 1024;

template <class D, int MB, int NB, bool PAST>
__global__ __launch_bounds__(64 * kRowWaves) void gemm_quantized_rows_kernel(const int8_t* x, const int8_t* w, D* c, GemmProblem p, ScalePlaces s, uint32_t windows_per_wave) {
#if defined(__HIP_DEVICE_COMPILE__)
    constexpr int BLOCKS = MB + NB;                       // of 16 rows in a window: W's, then x's
    constexpr int STAGE_BYTES = BLOCKS * 2048, STAGES = kRowBytesPerWave / STAGE_BYTES, LOADS = 2 * BLOCKS;
    static_assert(STAGES >= 3, "a ring of at least three windows");
    extern __shared__ __align__(16) unsigned char lds[];
    int64_t ox, ow, oc;
    batch_offsets(p, blockIdx.y, ox, ow, oc);
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64), lane = threadIdx.x % 64;
    const uint32_t r = lane % 16, kc = lane / 16;
    const uint32_t n0 = blockIdx.x * 16 * NB;
    unsigned char* const ring = lds + wave * kRowBytesPerWave;
    const __amdgpu_buffer_rsrc_t rsrc_w = __builtin_amdgcn_make_buffer_rsrc(const_cast<int8_t*>(w + ow + static_cast<int64_t>(n0) * p.b_cs), 0,
                                                                            bytes_of_rows(p.N - n0 < 16 * NB ? p.N - n0 : 16 * NB, p.b_cs, p.K), 0x00020000);
    const __amdgpu_buffer_rsrc_t rsrc_x = __builtin_amdgcn_make_buffer_rsrc(const_cast<int8_t*>(x + ox), 0, bytes_of_rows(p.M, p.a_rs, p.K), 0x00020000);
    // load j of a window: rows 8 (j % 2) .. + 7 of block j / 2; the lane's row and its (turned) piece.  Rows that are not there are beyond the buffer's range.
    uint32_t voff[LOADS], piece[2];
#pragma unroll
    for (int j = 0; j < LOADS; ++j) {
        const uint32_t row = (j % 2) * 8 + lane / 8;
        piece[j % 2] = (lane % 8) ^ ((row >> 1) & 7u);
        const bool of_w = j / 2 < NB;
        const uint32_t block_row = (of_w ? j / 2 : j / 2 - NB) * 16 + row;
        const bool there = of_w ? n0 + block_row < p.N : block_row < p.M;
        voff[j] = there ? block_row * static_cast<uint32_t>(of_w ? p.b_cs : p.a_rs) + piece[j % 2] * 16 : kBeyond;
    }
    const auto issue = [&](uint32_t window, uint32_t stage) {
        const uint32_t k = window * 128;
        const bool ends = k + 128 > p.K;          // (a window that K ends in: zeros behind it)
        constexpr int POLICY = PAST ? 2 : 0;      // (the non-temporal bit of a load)
#pragma unroll
        for (int j = 0; j < LOADS; ++j) {
            const uint32_t offset = ends && k + piece[j % 2] * 16 >= p.K ? kBeyond : voff[j];
            const auto to = (lds_address)(ring + stage * STAGE_BYTES + j * 1024);
            if (j < 2 * NB) __builtin_amdgcn_raw_ptr_buffer_load_lds(rsrc_w, to, 16, offset, k, 0, POLICY);
            else __builtin_amdgcn_raw_ptr_buffer_load_lds(rsrc_x, to, 16, offset, k, 0, 0);
        }
    };
    const uint32_t all = (p.K + 127) / 128;
    const uint32_t first = wave * windows_per_wave;
    const uint32_t count = first >= all ? 0 : (all - first < windows_per_wave ? all - first : windows_per_wave);

    int4v acc[MB][NB];
#pragma unroll
    for (int mb = 0; mb < MB; ++mb)
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) acc[mb][nb] = int4v{0, 0, 0, 0};
#pragma unroll
    for (int t = 0; t < STAGES - 1; ++t)
        if (static_cast<uint32_t>(t) < count) issue(first + t, t);
    uint32_t stage = 0, fill = STAGES - 1;
    for (uint32_t i = 0; i < count; ++i) {
        if (i + STAGES - 1 < count) {
            issue(first + i + STAGES - 1, fill);
            asm volatile("s_waitcnt vmcnt(%0)" ::"n"((STAGES - 1) * LOADS) : "memory");    // loads complete in order: window i is in
        } else {
            asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        }
        const unsigned char* const at = ring + stage * STAGE_BYTES;
        uint4v fw[2][NB], fx[2][MB];
#pragma unroll
        for (int half = 0; half < 2; ++half) {
#pragma unroll
            for (int nb = 0; nb < NB; ++nb) fw[half][nb] = *reinterpret_cast<const uint4v*>(at + nb * 2048 + tile_offset<int8_t>(r, half * 4 + kc));
#pragma unroll
            for (int mb = 0; mb < MB; ++mb) fx[half][mb] = *reinterpret_cast<const uint4v*>(at + (NB + mb) * 2048 + tile_offset<int8_t>(r, half * 4 + kc));
        }
#pragma unroll
        for (int half = 0; half < 2; ++half)
#pragma unroll
            for (int mb = 0; mb < MB; ++mb)
#pragma unroll
                for (int nb = 0; nb < NB; ++nb) acc[mb][nb] = mfma_i8(fw[half][nb], fx[half][mb], acc[mb][nb]);
        stage = stage + 1 == STAGES ? 0 : stage + 1;
        fill = fill + 1 == STAGES ? 0 : fill + 1;
    }
    // the wavefronts' tiles meet in LDS (every wavefront's ring has been read: its own MFMAs needed the data)
    __syncthreads();
    int4v* const partial = reinterpret_cast<int4v*>(lds);     // [wave][tile][lane]
#pragma unroll
    for (int mb = 0; mb < MB; ++mb)
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) partial[(wave * MB * NB + mb * NB + nb) * 64 + lane] = acc[mb][nb];
    __syncthreads();
    // accumulator: lane -> row of x (m) lane % 16; value v -> column n0 + 4 * (lane / 16) + v; wavefront t adds up tile t, t + 4, ..
    const float *scale_a, *scale_b;
    scale_offsets(p, s, blockIdx.y, scale_a, scale_b);
    for (int t = wave; t < MB * NB; t += kRowWaves) {
        const int mb = t / NB, nb = t % NB;
        int4v sum = partial[t * 64 + lane];
#pragma unroll
        for (int v = 1; v < kRowWaves; ++v) sum += partial[(v * MB * NB + t) * 64 + lane];
        const uint32_t m = mb * 16 + r, col = n0 + nb * 16 + 4 * kc;
        if (m >= p.M || col >= p.N) continue;
        const float sa = scale_a[m * s.a_step];
        float out[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) out[e] = static_cast<float>(sum[e]) * sa * scale_b[(col + e < p.N ? col + e : col) * s.b_step];
        store_four<D>(c + oc + static_cast<int64_t>(m) * p.c_rs + col, out, p.N - col);
    }
#endif
}

template <class D, int MB, int NB, bool PAST>
static int launch_rows(const GemmProblem& p, const ScalePlaces& s, const void* a, const void* b, void* c, hipStream_t stream) {
    auto kernel = gemm_quantized_rows_kernel<D, MB, NB, PAST>;
    constexpr size_t lds = kRowWaves * kRowBytesPerWave;
    static std::atomic<uint64_t> configured{0};
    if (int rc = raise_lds_limit(reinterpret_cast<const void*>(kernel), lds, configured)) return rc;
    const uint32_t windows = (p.K + 127) / 128, per_wave = (windows + kRowWaves - 1) / kRowWaves;
    hipLaunchKernelGGL(kernel, dim3((p.N + 16 * NB - 1) / (16 * NB), p.batches), dim3(64 * kRowWaves), lds, stream, static_cast<const int8_t*>(a), static_cast<const int8_t*>(b),
                       static_cast<D*>(c), p, s, per_wave);
    return launch_status("gemm_quantized_rows_kernel");
}

template <class D, int MB, int NB>
static int launch_rows(const GemmProblem& p, const ScalePlaces& s, const void* a, const void* b, void* c, hipStream_t stream) {
    return rows_past_caches(p, 1, 40ull << 20) ? launch_rows<D, MB, NB, true>(p, s, a, b, c, stream) : launch_rows<D, MB, NB, false>(p, s, a, b, c, stream);
}

static uint64_t blocks_of_16(const GemmProblem& p) { return (static_cast<uint64_t>(p.N) + 15) / 16 * p.batches; }

bool gemm_quantized_rows_takes(const GemmProblem& p, const void* a, const void* b) {
    if (p.M > 32 || !quantized_operands_fit(p, a, b)) return false;
    // Where the columns fill the chip once, 16 or 32 to a block, and the tiles of 32 x 64 do not do better, whose four wavefronts share x.  us here / there, weights from memory: 1 row of
    // 6144 x 4096 7.3 / 9.5, 4096 x 14336 11.5 / 15.2, 14336 x 4096 13.8 / 13.4, 28672 x 4096 25.5 / 24.5; 32 rows of 4096 x 4096 6.9 / 9.5, 6144 x 4096 8.6 / 10.4, 14336 x 4096 15.8 / 14.1,
    // 28672 x 4096 29.6 / 26.6; more than 16 rows under a long K, which those share between blocks: 4096 x 14336 16.6 / 15.3, 1000 x 14336 13.4 / 10.2 (16 rows 13.2 / 15.2, 10.2 / 10.0).
    return blocks_of_16(p) <= 512 && !(p.M > 16 && p.K >= 8192);
}

template <class D>
int gemm_quantized_rows(const GemmProblem& p, const ScalePlaces& s, const void* a, const void* b, void* c, hipStream_t stream) {
    if (!gemm_quantized_rows_takes(p, a, b)) return TANNIC_UNSUPPORTED_DTYPE;
    const bool two = blocks_of_16(p) > 256;
    if (p.M <= 16) return two ? launch_rows<D, 1, 2>(p, s, a, b, c, stream) : launch_rows<D, 1, 1>(p, s, a, b, c, stream);
    return two ? launch_rows<D, 2, 2>(p, s, a, b, c, stream) : launch_rows<D, 2, 1>(p, s, a, b, c, stream);
}

template int gemm_quantized_rows<f16>(const GemmProblem&, const ScalePlaces&, const void*, const void*, void*, hipStream_t);
template int gemm_quantized_rows<bf16>(const GemmProblem&, const ScalePlaces&, const void*, const void*, void*, hipStream_t);
template int gemm_quantized_rows<float>(const GemmProblem&, const ScalePlaces&, const void*, const void*, void*, hipStream_t);

}  // namespace th
