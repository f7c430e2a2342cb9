// Attention of few rows: one token of every sequence (decoding), or a few.  16-bit types and fp32, rows in 16-byte pieces.
// The keys and values have to be read once, and that bounds it (HBM): ROWS = 16 query rows that read the same kv head - a sequence's
// tokens times the heads of a group - are one tile of the matrix pipe, and all keys of all sequences are dealt to the blocks in equal
// runs (attention.hpp).  A block's wavefronts take 32 keys in turns (fp32: 16), each folding its own softmax; they meet in LDS at the end of a run.
//   scores  S^T[key][row] = K Q^T: a lane of the accumulator has one row (lane % 16) and four keys (4 (lane / 16) + i), so a row's maximum and
//           sum are one value per lane and two exchanges between lanes.
//   values  O^T[element][row] = V^T P^T: the weights are already where the second product wants them - a lane's keys of both tiles are its
//           eight of the product's 32 - if V's keys are taken in the same order.  16-bit V is transposed on its way out of LDS (ds_read_b64_tr_b16);
//           fp32 V needs no LDS: an accumulator's four keys are four products.
// Measured, a token of every sequence, 32 / 8 heads of 128: 4 sequences behind 32768 to 131072 (1.22 GB, bf16) 219 us, 5.6 TB/s, in the middle 6.1 as large reads alone; 32
// behind 64 to 4096 (133 MB, fp16) 37.9; one behind 2048 11.2, all of it one access after the other: lengths, table, keys, parts, their join.  fp32 chunks come here too, half
// of the fp32 pipe's rate (512 tokens behind 1024: 158 us).
#include "attention.hpp"

namespace th {

// keys of a unit: a step of each of the four wavefronts (half of that, 16-bit: a token behind 2048 13.2 us instead of 11.5, of 8 sequences' 16 heads of 64 over 1024 states 13.3 and
// 12.6; twice that 13.1 and 11.8)
template <class T> constexpr int kRowsUnit = sizeof(T) == 2 ? 128 : 64;

template <class T> __device__ inline uint4a load16(const T* at) { return *reinterpret_cast<const uint4a*>(at); }

template <class T, int DP> constexpr size_t rows_lds_bytes() {
    constexpr size_t join = 4 * 16 * (DP + 4) * 4 + 4 * 16 * 2 * 4, stage = sizeof(T) == 2 ? 4 * 32 * (DP + 16) * 2 : 0;
    return join > stage ? join : stage;
}

template <class T, int DP, bool PAGED>
__global__ __launch_bounds__(256, DP > 128 ? 1 : 2) void attention_rows_kernel(AttentionProblem p, const T* q, const T* k, const T* v, T* out, float* partial, uint32_t* arrivals) {
    constexpr bool HALF = sizeof(T) == 2;
    constexpr int ROWS = 16, E = 16 / sizeof(T);       // elements of a piece
    constexpr int KT = HALF ? 2 : 1, STEP = 16 * KT;        // tiles of 16 keys of a wavefront's step
    constexpr int KS = DP / (4 * E);                        // steps of a score's product: four pieces each
    constexpr int OT = DP / 16;                             // tiles of 16 elements of the result
    constexpr int PITCH = DP + 16;                          // elements from key to key in LDS: the four rows a transposing read touches, and the 16 of a write, on different banks
    extern __shared__ __align__(16) char lds_raw[];
    const uint32_t lane = threadIdx.x % 64, wave = threadIdx.x / 64, col = lane % 16, quarter = lane / 16;
    __shared__ uint32_t arrived;
    Run run;
    Group g;
    if (!run_of_block<PAGED, ROWS, kRowsUnit<T>>(p, gridDim.x, run, g)) return;
    const float factor = p.scale * 1.44269504088896340736f;      // weights are powers of two
    uint32_t at = run.from;
    while (true) {
        const uint32_t stop = g.first + g.units < run.to ? g.first + g.units : run.to;
        const uint32_t key_from = (at - g.first) * kRowsUnit<T>;
        uint32_t key_to = (stop - g.first) * kRowsUnit<T>;
        const bool whole = at == g.first && stop == g.first + g.units;

        // ---- the tile's rows
        uint4a qf[KS];
        const uint32_t row = g.tile * ROWS + col, i = p.group_div.div(row), head = g.head * p.group + row - i * p.group;
        const bool row_lives = i < g.span.count;
        const uint32_t seen = row_lives ? keys_seen(p, g.span, i) : 0;
        const T* const from_row = q + (row_lives ? query_offset(p, g.s, g.span, i, head) : 0);
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
            const uint32_t e = (ks * 4 + quarter) * E;
            qf[ks] = row_lives && e < p.d ? load16(from_row + e) : uint4a{0, 0, 0, 0};
        }
        // the last key any row of the tile sees
        const uint32_t last_i = p.group_div.div(g.tile * ROWS + ROWS - 1);
        const uint32_t most = keys_seen(p, g.span, last_i < g.span.count ? last_i : g.span.count - 1);
        key_to = key_to < most ? key_to : most;
        // keys up to here are seen by every live row
        const uint32_t all_see = keys_seen(p, g.span, p.group_div.div(g.tile * ROWS));

        float4a acc[OT];
        float top = -INFINITY, sum = 0.0f;
#pragma unroll
        for (int t = 0; t < OT; ++t) acc[t] = float4a{0, 0, 0, 0};

        // ---- keys and values of a step: a lane has key lane % 16 of every tile, pieces lane / 16, lane / 16 + 4, ...
        uint4a kf[KT][KS], vf[KT][KS];
        uint32_t there[KT];
        // which page a step's keys lie in is asked for a step before the keys themselves
        uint32_t page[KT], in_page[KT];
        auto look_up = [&](uint32_t j0) {
#pragma unroll
            for (int kt = 0; kt < KT; ++kt) {
                const uint32_t j = j0 + kt * 16 + col;
                page[kt] = ~0u, in_page[kt] = 0;
                if (j < key_to) page[kt] = page_of<PAGED>(p, g.s, j, in_page[kt]);
            }
        };
        // (fp32, whose chunks are bound by the instructions between their products: mostly every key of the step is there and heads have DP elements, and then nothing is asked of the
        // loads one by one, 159 us instead of 195 for 512 tokens behind 1024; the 16-bit types wait for the memory: 39.1 us with and 37.9 without for 32 sequences behind 64 to 4096)
        auto fetch_step = [&](auto every_tag) {
            constexpr bool EVERY = decltype(every_tag)::value;
#pragma unroll
            for (int kt = 0; kt < KT; ++kt) {
                const bool found = EVERY || page_exists(p, page[kt]);
                const int64_t k_off = found ? page[kt] * p.k_page + in_page[kt] * p.k_token + g.head * p.k_head : 0;
                const int64_t v_off = found ? page[kt] * p.v_page + in_page[kt] * p.v_token + g.head * p.v_head : 0;
#pragma unroll
                for (int ks = 0; ks < KS; ++ks) {
                    const uint32_t e = (ks * 4 + quarter) * E;
                    kf[kt][ks] = EVERY || (found && e < p.d) ? load16(k + k_off + e) : uint4a{0, 0, 0, 0};
                }
                if constexpr (HALF) {
#pragma unroll
                    for (int ks = 0; ks < KS; ++ks) {
                        const uint32_t e = (ks * 4 + quarter) * E;
                        vf[kt][ks] = EVERY || (found && e < p.d) ? load16(v + v_off + e) : uint4a{0, 0, 0, 0};
                    }
                } else {
                    // fp32: piece lane % 16 (+ 16 c) of the keys 4 (lane / 16) + i; vf[0][i * (KS / 4) + c] with KS / 4 = DP / 64
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const int source = 4 * quarter + i;
                        const int64_t off = __shfl(v_off, source);
                        const bool live = EVERY || ((there[kt] >> source) & 1);
#pragma unroll
                        for (int c = 0; c < KS / 4; ++c) {
                            const uint32_t e = (c * 16 + col) * E;
                            vf[kt][i * (KS / 4) + c] = EVERY || (live && e < p.d) ? load16(v + off + e) : uint4a{0, 0, 0, 0};
                        }
                    }
                }
            }
        };
        auto fetch = [&]() {
            bool every = !HALF && p.d == DP;
#pragma unroll
            for (int kt = 0; kt < KT; ++kt) {
                there[kt] = static_cast<uint32_t>(__ballot(page_exists(p, page[kt]))) & 0xFFFFu;
                every = every && there[kt] == 0xFFFFu;
            }
            if constexpr (HALF) fetch_step(std::false_type{});
            else if (every) fetch_step(std::true_type{});
            else fetch_step(std::false_type{});
        };
        T* const mine = reinterpret_cast<T*>(lds_raw) + wave * (32 * PITCH);
        uint32_t j0 = key_from + wave * STEP;
        if (j0 < key_to) {
            look_up(j0);
            fetch();
            look_up(j0 + 4 * STEP);
        }
        for (; j0 < key_to; j0 += 4 * STEP) {
            if constexpr (HALF) {
#pragma unroll
                for (int kt = 0; kt < KT; ++kt)
#pragma unroll
                    for (int ks = 0; ks < KS; ++ks) *reinterpret_cast<uint4a*>(mine + (kt * 16 + col) * PITCH + (ks * 4 + quarter) * E) = vf[kt][ks];
            }
            uint32_t keys_here[KT];
#pragma unroll
            for (int kt = 0; kt < KT; ++kt) keys_here[kt] = there[kt];
            const bool full = j0 + STEP <= all_see && keys_here[0] == 0xFFFFu && keys_here[KT - 1] == 0xFFFFu;
            // values that some rows do not see must not reach them through 0 * inf
            bool odd_values = false;
            if (!(j0 + STEP <= all_see) && j0 < key_to && all_see < key_to) {
#pragma unroll
                for (int kt = 0; kt < KT; ++kt)
#pragma unroll
                    for (int ks = 0; ks < KS; ++ks)
#pragma unroll
                        for (int w = 0; w < 4; ++w) odd_values = odd_values || not_finite<T>(vf[kt][ks][w]);
                odd_values = __ballot(odd_values) != 0;
                if (odd_values) {
#pragma unroll
                    for (int kt = 0; kt < KT; ++kt)
#pragma unroll
                        for (int ks = 0; ks < KS; ++ks) {
#pragma unroll
                            for (int w = 0; w < 4; ++w) vf[kt][ks][w] = finite_only<T>(vf[kt][ks][w]);
                            if constexpr (HALF) *reinterpret_cast<uint4a*>(mine + (kt * 16 + col) * PITCH + (ks * 4 + quarter) * E) = vf[kt][ks];
                        }
                }
            }
            asm volatile("" ::: "memory");      // (a wavefront reads what it wrote in order)
            float4a s[KT];
#pragma unroll
            for (int kt = 0; kt < KT; ++kt) {
                s[kt] = float4a{0, 0, 0, 0};
#pragma unroll
                for (int ks = 0; ks < KS; ++ks) s[kt] = rows_mfma<T>(kf[kt][ks], qf[ks], s[kt]);
            }
            uint4a now[HALF ? 1 : KS];      // (fp32: this step's values stay in registers while the next ones come)
            if constexpr (!HALF) {
#pragma unroll
                for (int c = 0; c < KS; ++c) now[c] = vf[0][c];
            }
            const uint32_t j_now = j0;
            if (j0 + 4 * STEP < key_to) {
                fetch();
                look_up(j0 + 8 * STEP);
            }
            float high = -INFINITY;
#pragma unroll
            for (int kt = 0; kt < KT; ++kt) s[kt] *= factor;
            if (!full) {
#pragma unroll
                for (int kt = 0; kt < KT; ++kt)
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        if (!(((keys_here[kt] >> (4 * quarter + i)) & 1) && j_now + kt * 16 + 4 * quarter + i < seen)) s[kt][i] = -INFINITY;
            }
#pragma unroll
            for (int kt = 0; kt < KT; ++kt)
#pragma unroll
                for (int i = 0; i < 4; ++i) high = fmaxf(high, s[kt][i]);
            high = across_groups_max(high);
            const float above = fmaxf(top, high), base = above == -INFINITY ? 0.0f : above - kWeightShift<T>;
            if (__ballot(above > top) != 0) {
                const float old = __builtin_amdgcn_exp2f(top - kWeightShift<T> - base);
                sum *= old;
#pragma unroll
                for (int t = 0; t < OT; ++t) acc[t] *= old;
            }
            top = above;
#pragma unroll
            for (int kt = 0; kt < KT; ++kt)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    s[kt][i] = __builtin_amdgcn_exp2f(s[kt][i] - base);
                    sum += s[kt][i];
                }
            if constexpr (HALF) {
                using Lds = __attribute__((address_space(3))) short;
                typedef short short4a __attribute__((ext_vector_type(4)));
                using Lds4 = __attribute__((address_space(3))) short4a;
                const uint4a weights{pack_weights<T>(s[0][0], s[0][1]), pack_weights<T>(s[0][2], s[0][3]), pack_weights<T>(s[KT - 1][0], s[KT - 1][1]), pack_weights<T>(s[KT - 1][2], s[KT - 1][3])};
                const T* const read_from = mine + (4 * quarter + col / 4) * PITCH + 4 * (col % 4);
#pragma unroll
                for (int t = 0; t < OT; ++t) {
                    const short4a low = __builtin_amdgcn_ds_read_tr16_b64_v4i16((Lds4*)(read_from + t * 16)), high = __builtin_amdgcn_ds_read_tr16_b64_v4i16((Lds4*)(read_from + 16 * PITCH + t * 16));
                    uint4a values;
                    __builtin_memcpy(&values, &low, 8);
                    __builtin_memcpy(reinterpret_cast<char*>(&values) + 8, &high, 8);
                    acc[t] = rows_mfma<T>(values, weights, acc[t]);
                }
            } else {
                // product i has the keys 4 (lane / 16) + i; tile 4 c + w holds the elements 64 c + 4 (row of the tile) + w
#pragma unroll
                for (int i = 0; i < 4; ++i)
#pragma unroll
                    for (int c = 0; c < KS / 4; ++c)
#pragma unroll
                        for (int w = 0; w < 4; ++w)
                            acc[4 * c + w] = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(now[i * (KS / 4) + c][w]), s[0][i], acc[4 * c + w], 0, 0, 0);
            }
            if (odd_values) {
                // the infinite and the NaN, key by key, where they are seen
#pragma unroll 1
                for (uint32_t n = 0; n < STEP; ++n) {
                    int64_t page;
                    uint32_t in;
                    const uint32_t j = j_now + n;
                    if (j >= key_to || !place_of<PAGED>(p, g.s, j, page, in)) continue;
                    const T* const value = v + page * p.v_page + in * p.v_token + g.head * p.v_head;
                    const uint32_t n16 = n % 16;
                    float mine_w = 0.0f;
#pragma unroll
                    for (int kt = 0; kt < KT; ++kt)
#pragma unroll
                        for (int i = 0; i < 4; ++i) mine_w = n == static_cast<uint32_t>(kt * 16) + 4 * (n16 / 4) + i ? s[kt][i] : mine_w;
                    const float w = __shfl(mine_w, static_cast<int>(16 * (n16 / 4) + col));
                    if (j < seen) {
#pragma unroll
                        for (int t = 0; t < OT; ++t)
#pragma unroll
                            for (int i = 0; i < 4; ++i) {
                                const uint32_t e = HALF ? t * 16 + 4 * quarter + i : 64 * (t / 4) + 4 * (4 * quarter + i) + t % 4;
                                const float x = e < p.d ? static_cast<float>(widen(value[e])) : 0.0f;
                                if (!(fabsf(x) < INFINITY)) acc[t][i] += w * x;
                            }
                    }
                }
            }
            asm volatile("" ::: "memory");
        }

        // ---- the wavefronts meet
        float* const join = reinterpret_cast<float*>(lds_raw);
        float* const stats = join + 4 * 16 * (DP + 4);
        const uint32_t pieces = p.d / 4, rows_left = g.span.count * p.group - g.tile * ROWS, rows = rows_left < ROWS ? rows_left : ROWS;
        auto write_row = [&](uint32_t r, uint32_t piece, const float4a& value, float total) {
            const uint32_t row = g.tile * ROWS + r, i = p.group_div.div(row), head = g.head * p.group + row - i * p.group;
            T* const to = out + (static_cast<int64_t>(g.span.begin + i) * p.heads + head) * p.d + piece * 4;
            const float inverse = 1.0f / total;
            T result[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) result[e] = narrow_result<T>(total == 0.0f ? 0.0f : value[e] * inverse);
            __builtin_memcpy(__builtin_assume_aligned(to, 4 * sizeof(T)), result, sizeof result);
        };
        const uint32_t slot = static_cast<uint32_t>(partial_floats<ROWS>(p.d)), level_floats = 2 * gridDim.x * slot;      // (9 million floats at most)
        // (a block has two parts at most: of the group its run starts in, and of one that starts behind that)
        auto part_of = [&](uint32_t level, uint32_t block) -> float* {
            return partial + (level % 2) * level_floats + (2 * block + (block * run.per < g.first ? 1 : 0)) * slot;
        };
        auto leave = [&](float* left, uint32_t r, uint32_t piece, const float4a& value, float above, float total) {
            store_through(left + r * p.d + piece * 4, value[0], value[1]);
            store_through(left + r * p.d + piece * 4 + 2, value[2], value[3]);
            if (piece == 0) store_through(left + static_cast<size_t>(ROWS) * p.d + 2 * r, above, total);
        };
        __syncthreads();
#pragma unroll
        for (int t = 0; t < OT; ++t) {
            if constexpr (HALF) {
                *reinterpret_cast<float4a*>(join + (wave * 16 + col) * (DP + 4) + t * 16 + 4 * quarter) = acc[t];
            } else {
#pragma unroll
                for (int i = 0; i < 4; ++i) join[(wave * 16 + col) * (DP + 4) + 64 * (t / 4) + 4 * (4 * quarter + i) + t % 4] = acc[t][i];
            }
        }
        const float total = across_groups_sum(sum);
        if (quarter == 0) {
            stats[(wave * 16 + col) * 2] = top;
            stats[(wave * 16 + col) * 2 + 1] = total;
        }
        __syncthreads();
        for (uint32_t x = threadIdx.x; x < 16 * (DP / 4); x += 256) {
            const uint32_t r = x / (DP / 4), piece = x % (DP / 4);
            if (piece >= pieces || r >= rows) continue;
            float above = -INFINITY;
#pragma unroll
            for (int w = 0; w < 4; ++w) above = fmaxf(above, stats[(w * 16 + r) * 2]);
            const float base = above == -INFINITY ? 0.0f : above;
            float total_weight = 0.0f;
            float4a value{0, 0, 0, 0};
#pragma unroll
            for (int w = 0; w < 4; ++w) {
                const float share = __builtin_amdgcn_exp2f(stats[(w * 16 + r) * 2] - base);
                total_weight += stats[(w * 16 + r) * 2 + 1] * share;
                value += *reinterpret_cast<const float4a*>(join + (w * 16 + r) * (DP + 4) + piece * 4) * share;
            }
            if (whole) write_row(r, piece, value, total_weight);
            else leave(part_of(0, run.block), r, piece, value, above, total_weight);
        }
        if (!whole) {
            // So many parts that lie beside each other are put together by the last of their blocks to get here, what comes of them by the last of those that have so many of
            // these, and so on: always the same ones in the same order, whichever block is last.  A count is 0 again behind its last block; a group's lie behind its first block
            // and up to its last, where the next group's may begin.
            // (All parts by one block: 3 tokens of 16 / 4 heads of 128 behind 117 and 12655, fp32, 53 us; so: 29.)
            const uint32_t first = g.first / run.per, last = (g.first + g.units - 1) / run.per;      // the blocks that have its parts
            const uint32_t results = rows * pieces;
            const uint32_t log_most = results <= 128 ? 6 : results <= 256 ? 5 : 4;      // (as many as 256 threads read in eight turns, or sixteen)
            // where that leaves threads idle, several share a result's parts
            uint32_t sharing = 1;
            while (2 * sharing * results <= 256) sharing *= 2;
            const uint32_t in_share = sharing == 1 ? 0 : threadIdx.x / results;
            uint32_t parts = last - first + 1, mine_at = run.block - first;
#pragma unroll 1
            for (uint32_t level = 0, apart = 0; parts > 1; ++level, apart += log_most) {
                const uint32_t from = mine_at >> log_most << log_most, here = parts - from < 1u << log_most ? parts - from : 1u << log_most, leader = first + (from << apart);
                asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
                __syncthreads();
                if (here > 1) {
                    if (threadIdx.x == 0) {
                        uint32_t* const count = arrivals + first + meeting_count(from, 1u << apart);
                        const uint32_t before = __hip_atomic_fetch_add(count, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
                        if (before == here - 1) __hip_atomic_store(count, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
                        arrived = before;
                    }
                    __syncthreads();
                    if (arrived != here - 1) break;
                }
                parts = (parts + (1u << log_most) - 1) >> log_most;
                mine_at >>= log_most;
                float* const left = part_of(level + 1, leader);
                const float* const its_first = part_of(level, leader);
                const float* const its_others = partial + (level % 2) * level_floats + 2 * leader * slot;
                const uint32_t its_step = 2 * slot << apart;
                for (uint32_t x0 = 0; x0 < results; x0 += 256) {
                    uint32_t x = sharing == 1 ? x0 + threadIdx.x : threadIdx.x % results;
                    float above = -INFINITY, total = 0.0f;
                    float4a value{0, 0, 0, 0};
                    if (x < results && in_share < sharing) {
                        const uint32_t r = x / pieces, piece = x % pieces;
                        constexpr int N = HALF ? 4 : 8;      // parts on their way at once (fp32, 8 instead of 4: 41 us instead of 43 for 36 tokens of 2 sequences behind 53 and 2516)
                        for (uint32_t n0 = in_share; n0 < here; n0 += N * sharing) {
                            float its_top[N], its_sum[N];
                            float4a its_value[N];
#pragma unroll
                            for (int n = 0; n < N; ++n) {
                                const uint32_t at_part = n0 + n * sharing < here ? n0 + n * sharing : here - 1;
                                const float* const its = (at_part == 0 ? its_first : its_others) + at_part * its_step;
                                load_through(its + ROWS * p.d + 2 * r, its_top[n], its_sum[n]);
                                load_through(its + r * p.d + piece * 4, its_value[n]);
                            }
                            float higher = above;
#pragma unroll
                            for (int n = 0; n < N; ++n) {
                                if (n0 + n * sharing >= here) its_top[n] = -INFINITY, its_sum[n] = 0.0f, its_value[n] = float4a{0, 0, 0, 0};
                                higher = fmaxf(higher, its_top[n]);
                            }
                            const float base = higher == -INFINITY ? 0.0f : higher, old = __builtin_amdgcn_exp2f(above - base);
                            total *= old;
                            value *= old;
#pragma unroll
                            for (int n = 0; n < N; ++n) {
                                const float share = __builtin_amdgcn_exp2f(its_top[n] - base);
                                total += its_sum[n] * share;
                                value += its_value[n] * share;
                            }
                            above = higher;
                        }
                    }
                    if (sharing > 1) {      // (then there is one turn)
                        *reinterpret_cast<float4a*>(join + threadIdx.x * 4) = value;
                        join[1024 + threadIdx.x * 2] = above;
                        join[1024 + threadIdx.x * 2 + 1] = total;
                        __syncthreads();
                        x = threadIdx.x;
                        if (x < results) {
                            above = -INFINITY, total = 0.0f, value = float4a{0, 0, 0, 0};
                            for (uint32_t n = 0; n < sharing; ++n) above = fmaxf(above, join[1024 + (n * results + x) * 2]);
                            const float base = above == -INFINITY ? 0.0f : above;
                            for (uint32_t n = 0; n < sharing; ++n) {
                                const uint32_t its = n * results + x;
                                const float share = __builtin_amdgcn_exp2f(join[1024 + its * 2] - base);
                                total += join[1024 + its * 2 + 1] * share;
                                value += *reinterpret_cast<const float4a*>(join + its * 4) * share;
                            }
                        }
                    }
                    if (x < results) {
                        if (__builtin_expect(parts == 1, 1)) write_row(x / pieces, x % pieces, value, total);
                        else leave(left, x / pieces, x % pieces, value, above, total);
                    }
                }
            }
        }
        if (stop == run.to) return;
        at = stop;
        next_group<PAGED, ROWS, kRowsUnit<T>>(p, g);
        __syncthreads();      // (LDS is read to the end before the next group's values are put there)
    }
}

// as many as run at a time: two on every compute unit, of the largest heads one (512 of those: 51 us instead of 40 for a token of 16 sequences behind 4096, 12 heads of 256)
template <int DP> constexpr uint32_t kRowsBlocks = DP > 128 ? 256 : 512;
static_assert(kRowsBlocks<64> <= kAttentionArrivals);

template <class T, int DP, bool PAGED>
int launch_rows(const AttentionProblem& p, const void* q, const void* k, const void* v, void* out, hipStream_t stream) {
    constexpr int ROWS = 16;
    constexpr size_t LDS = rows_lds_bytes<T, DP>();
    static std::atomic<uint64_t> raised{0};
    if (LDS > (64u << 10))
        if (int status = raise_lds_limit(reinterpret_cast<const void*>(attention_rows_kernel<T, DP, PAGED>), LDS, raised); status != TANNIC_SUCCESS) return status;
    // no more blocks than units there can be
    const uint64_t tiles = static_cast<uint64_t>(p.tokens) * p.group / ROWS + p.sequences;
    const uint64_t most = tiles * p.kv_heads * (p.room / kRowsUnit<T> + 1);
    if (most >= kMostUnits) return TANNIC_UNSUPPORTED_DTYPE;
    const uint32_t blocks = most < kRowsBlocks<DP> ? (static_cast<uint32_t>(most) + 7) / 8 * 8 : kRowsBlocks<DP>;      // (as many on each die)
    uint32_t* arrivals = nullptr;
    if (int status = attention_arrivals(stream, arrivals); status != TANNIC_SUCCESS) return status;
    float* partial = nullptr;
    if (scratch_acquire(reinterpret_cast<void**>(&partial), 4 * blocks * partial_floats<ROWS>(p.d) * sizeof(float), stream) != TANNIC_SUCCESS) return TANNIC_ERROR;
    hipLaunchKernelGGL((attention_rows_kernel<T, DP, PAGED>), dim3(blocks), dim3(256), LDS, stream, p, static_cast<const T*>(q), static_cast<const T*>(k), static_cast<const T*>(v),
                       static_cast<T*>(out), partial, arrivals);
    const int status = launch_status("attention_rows_kernel");
    scratch_release(partial, stream);
    return status;
}

template <class T, bool PAGED>
int pick_head(const AttentionProblem& p, const void* q, const void* k, const void* v, void* out, hipStream_t stream) {
    if (p.d <= 64) return launch_rows<T, 64, PAGED>(p, q, k, v, out, stream);
    if (p.d <= 128) return launch_rows<T, 128, PAGED>(p, q, k, v, out, stream);
    return launch_rows<T, 256, PAGED>(p, q, k, v, out, stream);
}

template <class T>
int pick_cache(const AttentionProblem& p, const void* q, const void* k, const void* v, void* out, hipStream_t stream) {
    if (p.starts) return pick_head<T, true>(p, q, k, v, out, stream);
    return pick_head<T, false>(p, q, k, v, out, stream);
}

int attention_rows(int dtype, const AttentionProblem& p, const void* q, const void* k, const void* v, void* out, hipStream_t stream) {
    switch (dtype) {
        case TANNIC_FLOAT16: return pick_cache<f16>(p, q, k, v, out, stream);
        case TANNIC_BFLOAT16: return pick_cache<bf16>(p, q, k, v, out, stream);
        case TANNIC_FLOAT32: return pick_cache<float>(p, q, k, v, out, stream);
        default: return TANNIC_UNSUPPORTED_DTYPE;
    }
}

}  // namespace th
