// Attention of many rows (chunks of a prompt, a decoder's inputs over an encoder's states), 16-bit types: bound by the matrix pipe.
// A block's four wavefronts have 32 rows each of one tile (a sequence's tokens times the heads of a group) and walk through the keys in steps of KT:
// keys and values of the next step go from memory straight to LDS while this step's are multiplied, all wavefronts reading the same ones.
//   scores  S^T[key][row] = K Q^T on v_mfma_f32_32x32x16: a lane has one row (lane % 32) and 16 of the tile's 32 keys, so that a row's
//           maximum and sum are one value per lane, and one exchange with the lane 32 further;
//   values  O^T[element][row] = V^T P^T: the lane's weights are the second product's operand as they are, if V's keys are taken in the
//           accumulator's order; V is transposed on its way out of LDS (ds_read_b64_tr_b16).
// The running maximum follows the scores only when one exceeds it by 2^8 (in the weights' power of two): sums in fp32 have the room, and the
// 64 to 128 sums of a lane are rescaled a few times in a row's life instead of every step.
// Measured, bf16: 2048 tokens of 32 / 8 heads of 128 behind 30720 1035 us, 1.03 PFLOP/s, the matrix pipe busy 49 % of the time (6.2 vector instructions to a product, two
// wavefronts on a SIMD); 512 behind 4096 62 us, 10 of them parts written and put together; 700 tokens of 8 sequences' 16 heads of 64 over 500 to 2000 states 52 us, 0.49 PFLOP/s
// (half the products to a weight).
#include <algorithm>

#include "attention.hpp"
#include "gemm_tiles.hpp"

namespace th {

// ---- items: a tile's rows of one kv head over a chunk of its keys -----------------------------------------------------------------
// Every sequence has tiles x kv heads groups of items, those of the last tile (which see the most keys) first.  With `places` blocks that run at a time, a place's share of all
// keys is as many as a group should have: one that has a quarter more is cut into equal chunks, and the last of its blocks puts the parts together.  (Cut only where there are fewer groups than places: 64 sequences behind 64 to 32768, 16 tokens of
// 32 / 8 heads of 128 each, 751 us; so: 302.)
struct Item {
    uint32_t s, tile, head, chunk, share;            // share: units of a place
    uint32_t part;                                   // of the parts of all groups that are cut, its group's first
    Span span;
};

__device__ inline uint32_t chunks_of(uint32_t units, uint32_t share) { return units > share + share / 4 ? (units + share - 1) / share : 1; }

template <bool PAGED, int ROWS, int UNIT>
__device__ inline bool item_of_block(const AttentionProblem& p, uint32_t most_groups, uint32_t places, uint32_t least_units, Item& item) {
    const uint32_t each = (p.sequences + 63) / 64;
    uint32_t all, groups, units = 0, tiles = 0, share = 0;
    Span span{};
    uint32_t my_groups = 0, my_parts = 0;
    const uint32_t my_units = lanes_share<PAGED>(p, each, [&](const Span& its) -> uint32_t {
        span = its;
        const uint32_t n = sequence_units<PAGED, ROWS, UNIT>(p, span, tiles, units);
        my_groups = sum_units(my_groups, tiles * p.kv_heads);
        return n;
    });
    lanes_sum_before(my_units, all);
    lanes_sum_before(my_groups, groups);
    // (more groups than the rows of q make: sequences that overlap, against what the starts may hold; there are not the blocks for them)
    if (all == kMostUnits || groups > most_groups) return false;
    share = (all + places - 1) / places;
    share = share > least_units ? share : least_units;
    const auto items_of = [&](const Span& its) -> uint32_t {
        sequence_units<PAGED, ROWS, UNIT>(p, its, tiles, units);
        const uint32_t chunks = chunks_of(units, share), mine = tiles * p.kv_heads * chunks;
        my_parts += chunks > 1 ? mine : 0;
        return mine;
    };
    uint32_t mine;
    if (each == 1) {      // (the lanes still have what they found)
        const uint32_t chunks = chunks_of(units, share);
        mine = tiles * p.kv_heads * chunks;
        my_parts = chunks > 1 ? mine : 0;
    } else {
        mine = lanes_share<PAGED>(p, each, items_of);
    }
    uint32_t total, parts;
    uint32_t before = lanes_sum_before(mine, total), parts_before = lanes_sum_before(my_parts, parts);
    const auto holds_block = [&]() -> uint64_t { return __ballot(before <= blockIdx.x && blockIdx.x - before < mine); };
    uint64_t here = holds_block();
    if (here == 0) return false;
    int at = __builtin_ctzll(here);
    item.s = at * each;
    if (each > 1) {
        const uint32_t lane = threadIdx.x % 64, end = item.s + each < p.sequences ? item.s + each : p.sequences;
        uint32_t first = __builtin_amdgcn_readlane(before, at), first_part = __builtin_amdgcn_readlane(parts_before, at);
        for (;; item.s += 64) {
            if (item.s >= end) return false;
            const bool there = item.s + lane < end;
            span = span_of<PAGED>(p, there ? item.s + lane : end - 1);
            span.count = there ? span.count : 0;
            my_parts = 0;
            mine = items_of(span);
            before = first + lanes_sum_before(mine, total);
            parts_before = first_part + lanes_sum_before(my_parts, parts);
            if ((here = holds_block()) != 0) break;
            first += total;
            first_part += parts;
        }
        at = __builtin_ctzll(here);
        item.s += at;
    }
    item.span.begin = __builtin_amdgcn_readlane(span.begin, at);
    item.span.count = __builtin_amdgcn_readlane(span.count, at);
    item.span.keys = __builtin_amdgcn_readlane(span.keys, at);
    item.span.step = PAGED ? 1 : 0;
    const uint32_t its_chunks = chunks_of(__builtin_amdgcn_readlane(units, at), share), in_sequence = blockIdx.x - __builtin_amdgcn_readlane(before, at);
    uint32_t rest = in_sequence / its_chunks;
    item.chunk = in_sequence - rest * its_chunks;
    item.part = __builtin_amdgcn_readlane(parts_before, at) + rest * its_chunks;
    item.head = rest % p.kv_heads;
    item.tile = __builtin_amdgcn_readlane(tiles, at) - 1 - rest / p.kv_heads;
    item.share = share;
    return true;
}

typedef float float16a __attribute__((ext_vector_type(16)));

template <class T> __device__ inline float16a tile_mfma(uint4a a, uint4a b, float16a c) {
    if constexpr (std::is_same_v<T, f16>) {
        typedef _Float16 V __attribute__((ext_vector_type(8)));
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(V, a), __builtin_bit_cast(V, b), c, 0, 0, 0);
    } else {
        typedef __bf16 V __attribute__((ext_vector_type(8)));
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(V, a), __builtin_bit_cast(V, b), c, 0, 0, 0);
    }
}

// the other half's value (lane ^ 32) beside this lane's
__device__ inline float halves_max(float x) {
    const uint2a r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ inline float halves_sum(float x) {
    const uint2a r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

using LdsVoid = __attribute__((address_space(3))) void*;

// Loads from memory straight to LDS: the wavefront's 64 lanes' 16 bytes each, one after the other from `to` on.  They are written as assembly because a builtin makes the
// compiler put a wait for all of them before every transposing read that follows (the two might touch the same bytes, for all it knows), which would leave nothing of a
// step's head start.  They have no register that anything could read too early; arrive() waits for them.
// (Scalar registers that a vector instruction has written are not there for a load in the five states behind it, and the compiler, which cannot see these loads, does not wait:
// it keeps the descriptors in scalar arithmetic, and a test looks its listing over.  Waits in every load instead: 1045 us for 1035, 2048 tokens behind 30720.)
typedef int int4a __attribute__((ext_vector_type(4)));
__device__ inline void load_to_lds(int4a from, uint32_t offset, uint32_t to) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds" ::"s"(to), "v"(offset), "s"(from) : "memory", "m0");
}
__device__ inline void load_to_lds(const void* from, uint32_t to) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" ::"s"(to), "v"(from) : "memory", "m0");
}

typedef short short4a __attribute__((ext_vector_type(4)));
using LdsShort4 = __attribute__((address_space(3))) short4a;
// the lane's element of a tile's 16 keys: two of its four rows each, `next` bytes apart
template <int NEXT> __device__ inline uint4a read_values(const char* at) {
    const short4a low = __builtin_amdgcn_ds_read_tr16_b64_v4i16((LdsShort4*)at), high = __builtin_amdgcn_ds_read_tr16_b64_v4i16((LdsShort4*)(at + NEXT));
    uint4a v;
    __builtin_memcpy(&v, &low, 8);
    __builtin_memcpy(reinterpret_cast<char*>(&v) + 8, &high, 8);
    return v;
}

// parts put together at a time: a block reads them at no more than a compute unit's rate, so few and often of the larger heads (4 / 8, us: 16 tokens of 32 heads of 128 behind 32768
// 56 / 59, 20 tokens of 12 heads of 256 behind 28185 72 / 85, 198 over 1422 states 44 / 43; 128 tokens of 8 * 16 heads of 64 over 2000 states 27 / 24)
template <int DP> constexpr uint32_t kTileJoin = DP > 64 ? 4 : 8;
constexpr int kTileWaves = 4, kTileRows = 32 * kTileWaves;
template <int DP> constexpr int kTileKeys = DP > 128 ? 32 : 64;
template <int DP> __host__ __device__ constexpr uint64_t tile_partial_floats() { return static_cast<uint64_t>(kTileRows) * (DP + 2); }
template <int V> using Index = std::integral_constant<int, V>;
template <int DP> constexpr size_t tile_lds_bytes() { return 4 * kTileKeys<DP> * DP * 2 + 16 + 4 * 1024; }

template <class T, int DP, bool PAGED>
__global__ __launch_bounds__(64 * kTileWaves, DP > 128 ? 1 : DP > 64 ? 2 : 3) void attention_tile_kernel(AttentionProblem p, const T* q, const T* k, const T* v, T* out, float* partial, uint32_t* arrivals,
                                                                                          uint32_t most_groups, uint32_t places, uint32_t least_units) {
#if defined(__HIP_DEVICE_COMPILE__)
    constexpr int KT = kTileKeys<DP>, NT = KT / 32;         // keys of a step, tiles of 32 of them
    constexpr int KS = DP / 16, OT = DP / 32;               // products of a tile's scores; tiles of 32 elements
    constexpr int LPR = DP / 8, RPI = 64 / LPR;             // 16-byte pieces of a row; rows of a load
    constexpr int KPW = KT / kTileWaves, LOADS = KPW / RPI; // keys a wavefront brings, in so many loads each for K and V
    constexpr uint32_t TILE = KT * DP * 2;                  // bytes
    extern __shared__ __align__(16) char lds_raw[];         // keys of two steps, values of two
    volatile uint32_t* const arrived = reinterpret_cast<volatile uint32_t*>(lds_raw + 4 * TILE);
    volatile uint32_t* const odd_step = arrived + 1;     // the step in which a value was not finite
    const uint32_t lane = threadIdx.x % 64, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64), col = lane % 32, half = lane / 32;
    Item item;
    if (!item_of_block<PAGED, kTileRows, KT>(p, most_groups, places, least_units, item)) return;
    const Span span = item.span;
    const uint32_t first_i = p.group_div.div(item.tile * kTileRows);
    uint32_t last_i = p.group_div.div(item.tile * kTileRows + kTileRows - 1);
    last_i = last_i < span.count ? last_i : span.count - 1;
    const uint32_t all_see = keys_seen(p, span, first_i), most = keys_seen(p, span, last_i);     // by every row of the tile, by the last
    const uint32_t units = most ? (most + KT - 1) / KT : 1, chunks = chunks_of(units, item.share), chunk_units = (units + chunks - 1) / chunks;
    if (item.chunk >= chunks) return;      // (the tile sees fewer keys than the sequence's last)
    const uint32_t key_from = item.chunk * chunk_units * KT, key_end = key_from + chunk_units * KT, key_to = key_end < most ? key_end : most;

    // ---- this lane's row
    const uint32_t row = item.tile * kTileRows + wave * 32 + col, i_row = p.group_div.div(row), q_head = item.head * p.group + row - i_row * p.group;
    const bool row_lives = i_row < span.count;
    const uint32_t seen = row_lives ? keys_seen(p, span, i_row) : 0;
    // a negative scale turns the queries round, so that the largest score is that of the largest product; a scale of 0 leaves nothing of them but what is infinite or NaN
    const uint32_t flip = p.scale < 0.0f ? 0x80008000u : 0u;
    const float factor = (p.scale == 0.0f ? 1.0f : fabsf(p.scale)) * 1.44269504088896340736f;
    uint4a qf[KS];
    {
        const T* const from = q + (row_lives ? query_offset(p, item.s, span, i_row, q_head) : 0);
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
            const uint32_t e = ks * 16 + half * 8;
            uint4a x = row_lives && e < p.d ? *reinterpret_cast<const uint4a*>(from + e) : uint4a{0, 0, 0, 0};
#pragma unroll
            for (int w = 0; w < 4; ++w) x[w] = p.scale == 0.0f ? times_zero<T>(x[w]) : x[w] ^ flip;
            qf[ks] = x;
        }
    }

    // ---- bringing a step's keys and values to LDS
    const uint32_t lds_at = static_cast<uint32_t>(reinterpret_cast<uintptr_t>((LdsVoid)lds_raw));
    // A row's pieces lie in an order of their own, so that the 16 rows a score's operand takes the same piece of, and the four rows of a transposing read, fall
    // on different banks.
    auto k_place = [](uint32_t r) -> uint32_t { return DP == 64 ? (r >> 1) & 7u : r & 15u; };
    auto v_place = [](uint32_t r) -> uint32_t { return DP == 64 ? ((r >> 1) & 1u) * 4 : (r & 3u) * 4; };
    // Rows that are not there, and the pieces behind a head of less than DP elements, are beyond what the loads may reach: 0 is put in their place.
    constexpr uint32_t BEYOND = 0x80000000u;
    uint32_t k_lane[LOADS], v_lane[LOADS];      // bytes from the wavefront's first key
    const uint32_t piece = lane % LPR, row_in = lane / LPR;
#pragma unroll
    for (int i = 0; i < LOADS; ++i) {
        const uint32_t r = i * RPI + row_in, in_tile = wave * KPW + r, k_piece = piece ^ k_place(in_tile), v_piece = piece ^ v_place(in_tile);
        k_lane[i] = k_piece * 8 < p.d ? r * static_cast<uint32_t>(p.k_token) * 2 + k_piece * 16 : BEYOND;
        v_lane[i] = v_piece * 8 < p.d ? r * static_cast<uint32_t>(p.v_token) * 2 + v_piece * 16 : BEYOND;
    }
    // The second buffer of values starts as 0 (see below).
    for (uint32_t x = threadIdx.x; x < TILE / 16; x += 64 * kTileWaves) reinterpret_cast<uint4a*>(lds_raw + 3 * TILE)[x] = uint4a{0, 0, 0, 0};
    struct Fetch {      // loads that are to be issued: from where, and to where in LDS
        int4a from;
        uint32_t to;
    };
    const Fetch nothing{{0, 0, 0, 0x00020000}, static_cast<uint32_t>(__builtin_amdgcn_readfirstlane(lds_at + 4 * TILE + 16))};      // (a place that nobody reads)
    auto fetch_from = [&](const T* base, int64_t offset, uint32_t token_stride, uint32_t here, uint32_t to) -> Fetch {
        const uint64_t start = reinterpret_cast<uint64_t>(base + offset);
        return Fetch{{__builtin_amdgcn_readfirstlane(static_cast<int>(start)), __builtin_amdgcn_readfirstlane(static_cast<int>(start >> 32) & 0xFFFF),
                      __builtin_amdgcn_readfirstlane(static_cast<int>(here ? (here - 1) * token_stride * 2 + p.d * 2 : 0)), 0x00020000},
                     static_cast<uint32_t>(__builtin_amdgcn_readfirstlane(lds_at + to + wave * (LOADS * 1024)))};
    };
    // A wavefront's keys of a step mostly lie in one page: lane w holds the number of wavefront w's, asked for a step before it is needed, and which keys of the step are there
    // follows from the four.  Where pages end inside a wavefront's keys lane n holds the number of key n's.
    const bool together = !PAGED || p.page % KPW == 0;
    const T* const k_head = k + static_cast<int64_t>(item.head) * p.k_head;
    const T* const v_head = v + static_cast<int64_t>(item.head) * p.v_head;
    const bool alike = p.k_page == p.v_page && p.k_token == p.v_token;
    uint32_t next_page = ~0u, next_in = 0;
    auto look_up = [&](uint32_t j0) {
        const uint32_t j = j0 + (together ? (lane % kTileWaves) * KPW : lane % KT);
        next_page = ~0u;
        if (j < key_to) next_page = page_of<PAGED>(p, item.s, j, next_in);
    };
    // the values of a step's keys are brought one (one tile a step: two) steps after them
    struct Pending {
        int64_t offset;
        uint32_t here;
    };
    Pending values_next{0, 0}, values_after{0, 0};
    uint32_t v_next_page = ~0u, v_next_in = 0, v_after_page = ~0u, v_after_in = 0;      // (key by key)
    constexpr uint64_t ALL = ~0ull >> (64 - KT);
    auto one_by_one = [&](auto of_keys, uint32_t key_page, uint32_t key_in, uint32_t buffer) {
        constexpr bool KEYS = decltype(of_keys)::value;
        const uint32_t place = (KEYS ? buffer : 2 + buffer) * TILE + wave * (LOADS * 1024), to = __builtin_amdgcn_readfirstlane(lds_at + place);
        uint32_t pages_of[LOADS], ins_of[LOADS];
#pragma unroll
        for (uint32_t i = 0; i < LOADS; ++i) pages_of[i] = __shfl(key_page, wave * KPW + i * RPI + row_in), ins_of[i] = __shfl(key_in, wave * KPW + i * RPI + row_in);
#pragma unroll
        for (uint32_t i = 0; i < LOADS; ++i) {
            const uint32_t in_tile = wave * KPW + i * RPI + row_in, its_piece = piece ^ (KEYS ? k_place(in_tile) : v_place(in_tile));
            const uint32_t page = pages_of[i], in = ins_of[i];
            if (page_exists(p, page) && its_piece * 8 < p.d)
                load_to_lds((KEYS ? k_head + page * p.k_page + in * p.k_token : v_head + page * p.v_page + in * p.v_token) + its_piece * 8, to + i * 1024);
            else *reinterpret_cast<uint4a*>(lds_raw + place + i * 1024 + lane * 16) = uint4a{0, 0, 0, 0};
        }
    };
    auto bring_keys = [&](uint32_t j0, uint32_t buffer, uint64_t& keys) -> Fetch {
        if (!together) {
            v_after_page = v_next_page, v_after_in = v_next_in;
            v_next_page = next_page, v_next_in = next_in;
            keys = __ballot(page_exists(p, next_page)) & ALL;
            one_by_one(std::true_type{}, next_page, next_in, buffer);
            return nothing;
        }
        const uint32_t live = static_cast<uint32_t>(__ballot(page_exists(p, next_page))) & ((1u << kTileWaves) - 1);
        const uint32_t page = __builtin_amdgcn_readlane(next_page, wave), in = __builtin_amdgcn_readlane(next_in, wave), j = j0 + wave * KPW;
        const uint32_t here = !((live >> wave) & 1) ? 0 : key_to - j < KPW ? key_to - j : KPW;
        const int64_t k_off = here ? page * p.k_page + in * p.k_token : 0, v_off = alike ? k_off : here ? page * p.v_page + in * p.v_token : 0;
        values_after = values_next;
        values_next = Pending{v_off, here};
        keys = ALL;
        if (live != (1u << kTileWaves) - 1 || j0 + KT > key_to) {
            keys = 0;
#pragma unroll
            for (uint32_t w = 0; w < kTileWaves; ++w) keys |= static_cast<uint64_t>((live >> w) & 1 ? (1u << KPW) - 1 : 0u) << (w * KPW);
            const uint32_t left = key_to > j0 ? key_to - j0 : 0;
            if (left < KT) keys &= (1ull << left) - 1;
        }
        return fetch_from(k_head, k_off, static_cast<uint32_t>(p.k_token), here, buffer * TILE);
    };
    auto bring_values = [&](const Pending& of, uint32_t key_page, uint32_t key_in, uint32_t buffer) -> Fetch {
        if (!together) {
            one_by_one(std::false_type{}, key_page, key_in, buffer);
            return nothing;
        }
        return fetch_from(v_head, of.offset, static_cast<uint32_t>(p.v_token), of.here, (2 + buffer) * TILE);
    };
    auto fetch_keys = [&](const Fetch& f, int i) { load_to_lds(f.from, k_lane[i], f.to + i * 1024); };
    auto fetch_values = [&](const Fetch& f, int i) { load_to_lds(f.from, v_lane[i], f.to + i * 1024); };
    auto fetch_all = [&](const Fetch& f, auto&& fetch) {
#pragma unroll
        for (int i = 0; i < LOADS; ++i) fetch(f, i);
    };
    auto arrive = [] {
        asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
    };

    float16a acc[OT];
#pragma unroll
    for (int t = 0; t < OT; ++t)
#pragma unroll
        for (int i = 0; i < 16; ++i) acc[t][i] = 0.0f;
    float top = -INFINITY, base = 0.0f, sum = 0.0f;      // of the products before the scale, and what it takes off a score; the sum over the lane's own keys

    // where this lane reads: K's row col (+ 32 per tile); V's rows 4 half + lane / 4 % 4 (+ 8 per read), elements 16 (lane / 16 % 2) + 4 (lane % 4)
    const uint32_t k_at = col * (DP * 2) + (half ^ k_place(col)) * 16;      // (piece 2 ks + half: ks changes other bits of the place)
    const uint32_t v_row = 4 * half + (lane % 16) / 4;
    uint32_t v_at[OT];
#pragma unroll
    for (int t = 0; t < OT; ++t) {
        const uint32_t v_piece = t * 4 + ((lane / 16) % 2) * 2 + (lane % 4) / 2;
        v_at[t] = 2 * TILE + v_row * (DP * 2) + (v_piece ^ v_place(v_row)) * 16 + (lane % 2) * 8;
    }

    // The work on a tile of 32 keys is spread over three turns, so that the matrix pipe has the tiles before and after to work on while a tile's weights are
    // computed: in turn n the scores of tile n + 1 (from K), the weights of tile n, the sums of tile n - 1 (from V).  Between the turns of a step's last but one
    // and last tile the wavefronts meet: the next step's keys and this one's values have come, and the buffers before them are free for the ones after.
    float16a s;                      // scores of the tile whose turn it is
    uint32_t weights[8];             // of the tile before
    uint32_t odd_from = ~0u, buffer = 0;
    const uint32_t steps = key_from < key_to ? (key_to - key_from + KT - 1) / KT : 0;
    auto scores_of = [&](uint32_t from_buffer, uint32_t tile, int ks) -> uint4a {
        return *reinterpret_cast<const uint4a*>(lds_raw + from_buffer * TILE + tile * (32 * DP * 2) + (k_at ^ (ks * 32)));
    };
    // (The first tile has none before it: its weights are 0, and so is that buffer of values.  What the last one's turn makes of the keys behind it is not used.)
    // FETCH: the loads of the next step's values and of the keys behind those go out one by one between the products (all at once they keep the wavefront waiting for the
    // memory pipe's queue: 1700 of a step's 4600 clocks).
    auto turn = [&](auto fetch_tag, const Fetch& next_values, const Fetch& next_keys, auto value_tile_tag, uint32_t keys, uint32_t j, uint32_t k_buffer, uint32_t k_tile, uint32_t v_buffer) {
        constexpr bool FETCH = decltype(fetch_tag)::value;
        constexpr int V_FROM = decltype(value_tile_tag)::value * (32 * DP * 2);
        uint4a kf[2][2];
        kf[0][0] = scores_of(k_buffer, k_tile, 0), kf[0][1] = scores_of(k_buffer, k_tile, 1);
        uint4a values[3];
        auto value_of = [&](const char* tile, int n) -> uint4a { return read_values<8 * DP * 2>(tile + v_at[n % OT] + (n / OT) * (16 * DP * 2)); };
        {
            const char* const tile = lds_raw + v_buffer * TILE + V_FROM;
            values[0] = value_of(tile, 0), values[1] = value_of(tile, 1);
        }
        // a lane's keys are 8 (i / 4) + 4 half + i % 4
        if (keys != ~0u || j + 32 > all_see) {
            const uint32_t left = seen > j ? seen - j : 0;
            const uint32_t mine = (keys & (left < 32 ? (1u << left) - 1 : ~0u)) >> (4 * half);
#pragma unroll
            for (int i = 0; i < 16; ++i)
                if (!(mine & (1u << (8 * (i / 4) + i % 4)))) s[i] = -INFINITY;
        }
        // The weights are computed against the largest score so far while this tile's is still being found; if it turns out to be too much larger they are computed again.
        float high = -INFINITY, part = 0.0f;
        float16a next;
#pragma unroll
        for (int i = 0; i < 16; ++i) next[i] = 0.0f;
        uint32_t fresh[8];
        uint4a w{};
        const char* const v_tile = lds_raw + v_buffer * TILE + V_FROM;
        float first_of_pair = 0.0f;
        static_for<KS>([&](auto c_tag) {
            constexpr int c = decltype(c_tag)::value;
            if constexpr (c % 2 == 0 && c + 2 < KS) kf[(c / 2 + 1) % 2][0] = scores_of(k_buffer, k_tile, c + 2), kf[(c / 2 + 1) % 2][1] = scores_of(k_buffer, k_tile, c + 3);
            constexpr int kk = c / OT, t = c % OT;
            if constexpr (t == 0) w = uint4a{weights[kk * 4], weights[kk * 4 + 1], weights[kk * 4 + 2], weights[kk * 4 + 3]};
            if constexpr (c + 2 < KS) values[(c + 2) % 3] = value_of(v_tile, c + 2);
            acc[t] = tile_mfma<T>(values[c % 3], w, acc[t]);
            next = tile_mfma<T>(kf[(c / 2) % 2][c % 2], qf[c], next);
            if constexpr (FETCH && c < 2 * LOADS) {
                if constexpr (c % 2 == 0) fetch_values(next_values, c / 2);
                else fetch_keys(next_keys, c / 2);
            }
            // 16 / KS weights of this tile
#pragma unroll
            for (int i = c * 16 / KS; i < (c + 1) * 16 / KS; ++i) {
                const float x = __builtin_amdgcn_exp2f(__builtin_fmaf(s[i], factor, -base));
                part += x;
                if (i % 2 == 0) {
                    first_of_pair = x;
                } else {
                    fresh[i / 2] = pack_weights<T>(first_of_pair, x);
                    high = fmaxf(fmaxf(high, s[i - 1]), s[i]);
                    asm volatile("" : "+v"(fresh[i / 2]), "+v"(part), "+v"(high));      // (here, and not where they are used)
                }
            }
            __builtin_amdgcn_sched_barrier(0);
        });
        high = halves_max(high);
        if (__ballot(high * factor > top * factor + 8.0f || (top == -INFINITY && high > -INFINITY)) != 0) {
            const float above = fmaxf(top, high), old = top == above ? 1.0f : __builtin_amdgcn_exp2f((top - above) * factor);
            top = above;
            base = above == -INFINITY ? 0.0f : above * factor - kWeightShift<T> / 2;
            sum *= old;
            part = 0.0f;
#pragma unroll
            for (int i = 0; i < 16; i += 2) {
                const float x = __builtin_amdgcn_exp2f(__builtin_fmaf(s[i], factor, -base)), y = __builtin_amdgcn_exp2f(__builtin_fmaf(s[i + 1], factor, -base));
                part += x;
                part += y;
                fresh[i / 2] = pack_weights<T>(x, y);
            }
#pragma unroll
            for (int t = 0; t < OT; ++t)
#pragma unroll
                for (int i = 0; i < 16; ++i) acc[t][i] *= old;
        }
        sum += part;
        s = next;
#pragma unroll
        for (int i = 0; i < 8; ++i) weights[i] = fresh[i];
    };
    // Values that some of the tile's rows do not see must not reach those through 0 * inf: where there are such keys, the infinite and the NaN
    // among the values are 0 for the product, and are added in the end where they are seen.
    auto sort_values = [&](uint32_t j0, uint32_t v_buffer) {
        if (j0 + KT <= all_see || all_see >= most) return;
#pragma unroll 1
        for (int i = 0; i < LOADS; ++i) {
            uint4a* const at = reinterpret_cast<uint4a*>(lds_raw + (2 + v_buffer) * TILE + wave * (LOADS * 1024) + i * 1024 + lane * 16);
            uint4a x = *at;
            bool odd = false;
#pragma unroll
            for (int w = 0; w < 4; ++w) odd = odd || not_finite<T>(x[w]);
            if (odd) {
#pragma unroll
                for (int w = 0; w < 4; ++w) x[w] = finite_only<T>(x[w]);
                *at = x;
                *odd_step = j0 + 1;
            }
        }
        __syncthreads();
        if (*odd_step == j0 + 1 && odd_from == ~0u) odd_from = j0;
    };
    using Yes = std::true_type;
    using No = std::false_type;
    if (threadIdx.x == 0) *odd_step = 0;
    uint64_t keys = 0, keys_next = 0, keys_after = 0;      // which keys of this step, the next and the one behind it are there
    if (steps > 0) {
        look_up(key_from);
        fetch_all(bring_keys(key_from, 0, keys), fetch_keys);
        if constexpr (NT == 2) fetch_all(bring_values(values_next, v_next_page, v_next_in, 0), fetch_values);
        look_up(key_from + KT);
        fetch_all(bring_keys(key_from + KT, 1, keys_next), fetch_keys);
        look_up(key_from + 2 * KT);
    }
    arrive();
    if (steps > 0) {
        // the first tile's scores
#pragma unroll
        for (int i = 0; i < 8; ++i) weights[i] = 0;
#pragma unroll
        for (int i = 0; i < 16; ++i) s[i] = 0.0f;
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) s = tile_mfma<T>(scores_of(0, 0, ks), qf[ks], s);
        for (uint32_t step = 0; step < steps; ++step, buffer ^= 1) {
            const uint32_t j0 = key_from + step * KT;
            if constexpr (NT == 2) turn(No{}, nothing, nothing, Index<1>{}, static_cast<uint32_t>(keys), j0, buffer, 1, buffer ^ 1);
            // Here the keys of the next step and the values of this one (one tile a step: of the one before) are there, and what is before them has been read.
            arrive();
            // (behind the last step's keys there are none: nothing comes)
            const Fetch next_values = NT == 2 ? bring_values(values_next, v_next_page, v_next_in, buffer ^ 1) : bring_values(values_after, v_after_page, v_after_in, buffer);
            const Fetch next_keys = bring_keys(j0 + 2 * KT, buffer, keys_after);
            look_up(j0 + 3 * KT);
            if (NT == 2) sort_values(j0, buffer);
            else if (step > 0) sort_values(j0 - KT, buffer ^ 1);
            if constexpr (NT == 2) turn(Yes{}, next_values, next_keys, Index<0>{}, static_cast<uint32_t>(keys >> 32), j0 + 32, buffer ^ 1, 0, buffer);
            else turn(Yes{}, next_values, next_keys, Index<0>{}, static_cast<uint32_t>(keys), j0, buffer ^ 1, 0, buffer ^ 1);
            keys = keys_next;
            keys_next = keys_after;
        }
        // the last tile's sums
        if constexpr (NT == 1) {
            arrive();
            sort_values(key_from + (steps - 1) * KT, buffer ^ 1);
        }
#pragma unroll
        for (int kk = 0; kk < 2; ++kk) {
            const uint4a w{weights[kk * 4], weights[kk * 4 + 1], weights[kk * 4 + 2], weights[kk * 4 + 3]};
#pragma unroll
            for (int t = 0; t < OT; ++t) acc[t] = tile_mfma<T>(read_values<8 * DP * 2>(lds_raw + v_at[t] + (buffer ^ 1) * TILE + ((NT - 1) * 32 + kk * 16) * (DP * 2)), w, acc[t]);
        }
    }
    sum = halves_sum(sum);
    if (odd_from < key_to) {
#pragma unroll 1
        for (uint32_t j = odd_from; j < key_to; ++j) {
            int64_t page;
            uint32_t in;
            if (!place_of<PAGED>(p, item.s, j, page, in) || j >= seen) continue;
            const T* const value = v + page * p.v_page + static_cast<int64_t>(in) * p.v_token + item.head * p.v_head;
#pragma unroll
            for (int t = 0; t < OT; ++t)
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    const uint32_t e = t * 32 + 8 * (i / 4) + 4 * half + i % 4;
                    const float x = e < p.d ? static_cast<float>(widen(value[e])) : 0.0f;
                    if (!(fabsf(x) < INFINITY)) acc[t][i] += x;      // (any weight above 0 says the same)
                    if (i % 4 == 3) __builtin_amdgcn_sched_barrier(0);
                }
        }
    }

    // ---- a lane has its row's elements 32 t + 8 (i / 4) + 4 half + i % 4
    auto write_row = [&](const float16a* of, float total) {
        if (!row_lives) return;
        T* const to = out + (static_cast<int64_t>(span.begin + i_row) * p.heads + q_head) * p.d;
        const float inverse = total == 0.0f ? 0.0f : 1.0f / total;
#pragma unroll
        for (int t = 0; t < OT; ++t)
#pragma unroll
            for (int i = 0; i < 16; i += 4) {
                const uint32_t e = t * 32 + 2 * i + 4 * half;
                if (e < p.d) {
                    T result[4];
#pragma unroll
                    for (int u = 0; u < 4; ++u) result[u] = narrow_result<T>(total == 0.0f ? 0.0f : of[t][i + u] * inverse);
                    __builtin_memcpy(__builtin_assume_aligned(to + e, 8), result, 8);
                }
            }
    };
    if (chunks == 1) {
        write_row(acc, sum);
        return;
    }
    // ---- or a part of it, as the lanes have it.  kTileJoin<DP> parts that lie beside each other are put together by the last of their blocks to get here, what comes of
    // them by the last of those that have kTileJoin<DP> of these, and so on: always the same ones in the same order, whichever block is last.  (One block that reads all 64
    // parts of a group: 166 us for 16 tokens of 32 heads behind 32768; so: 60.)
    constexpr uint64_t SLOT = tile_partial_floats<DP>(), STATS = static_cast<uint64_t>(kTileRows) * DP;
    constexpr uint32_t AT_ONCE = DP > 64 ? 4 : 2;      // parts whose loads are on their way, 8 of each (4 of the small heads: registers of the loop above spill)
    const uint32_t my_row = wave * 32 + col;
    float* const group_parts = partial + static_cast<uint64_t>(item.part) * SLOT;
    uint32_t* const group_arrivals = arrivals + item.part;
    top = top == -INFINITY ? -INFINITY : top * factor;
    uint32_t parts = chunks, mine = item.chunk, apart = 1;      // a part's place is `apart` from the next one's
#pragma unroll 1
    for (; parts > 1; parts = (parts + kTileJoin<DP> - 1) / kTileJoin<DP>, mine /= kTileJoin<DP>, apart *= kTileJoin<DP>) {
        const uint32_t first = mine - mine % kTileJoin<DP>, together_here = parts - first < kTileJoin<DP> ? parts - first : kTileJoin<DP>;
        if (together_here == 1) continue;
        float* const its = group_parts + static_cast<uint64_t>(first * apart) * SLOT;
        if (row_lives) {
            float* const left = its + static_cast<uint64_t>((mine - first) * apart) * SLOT;
#pragma unroll
            for (int t = 0; t < OT; ++t)
#pragma unroll
                for (int i = 0; i < 16; i += 2) store_through(left + ((t * 8 + i / 2) * (64 * kTileWaves) + threadIdx.x) * 2, acc[t][i], acc[t][i + 1]);
            if (half == 0) store_through(left + STATS + 2 * my_row, top, sum);
        }
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        __syncthreads();
        if (threadIdx.x == 0) {
            uint32_t* const count = group_arrivals + meeting_count(first, apart);
            const uint32_t before = __hip_atomic_fetch_add(count, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            if (before == together_here - 1) __hip_atomic_store(count, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            *arrived = before;
        }
        __syncthreads();
        if (*arrived != together_here - 1) return;
        if (row_lives) {
            float its_top[kTileJoin<DP>], its_sum[kTileJoin<DP>];
#pragma unroll
            for (uint32_t c = 0; c < kTileJoin<DP>; ++c) {
                its_top[c] = -INFINITY, its_sum[c] = 0.0f;
                if (c < together_here) load_through(its + static_cast<uint64_t>(c * apart) * SLOT + STATS + 2 * my_row, its_top[c], its_sum[c]);
            }
            top = -INFINITY;
#pragma unroll
            for (uint32_t c = 0; c < kTileJoin<DP>; ++c) top = fmaxf(top, its_top[c]);
            sum = 0.0f;
#pragma unroll
            for (uint32_t c = 0; c < kTileJoin<DP>; ++c) {
                its_top[c] = __builtin_amdgcn_exp2f(its_top[c] - (top == -INFINITY ? 0.0f : top));      // its share
                sum += its_sum[c] * its_top[c];
            }
#pragma unroll
            for (int t = 0; t < OT; ++t) {
#pragma unroll
                for (int i = 0; i < 16; ++i) acc[t][i] = 0.0f;
#pragma unroll
                for (uint32_t c0 = 0; c0 < kTileJoin<DP>; c0 += AT_ONCE) {
                    float x[AT_ONCE][16];
#pragma unroll
                    for (uint32_t c = 0; c < AT_ONCE; ++c)
                        if (c0 + c < together_here) {
#pragma unroll
                            for (int i = 0; i < 16; i += 2)
                                load_through(its + static_cast<uint64_t>((c0 + c) * apart) * SLOT + ((t * 8 + i / 2) * (64 * kTileWaves) + threadIdx.x) * 2, x[c][i], x[c][i + 1]);
                        }
#pragma unroll
                    for (uint32_t c = 0; c < AT_ONCE; ++c)
                        if (c0 + c < together_here) {
#pragma unroll
                            for (int i = 0; i < 16; ++i) acc[t][i] += x[c][i] * its_top[c0 + c];
                        }
                }
            }
        }
    }
    write_row(acc, sum);
#endif
}

// blocks that run at a time: two on every compute unit, of the largest heads one (8 tokens of 16 sequences, us with 512 / 256: 32 heads of 128 behind 8192 109 / 121, 12 heads of
// 256 behind 4096 105 / 67); of heads up to 64 there are three, but with 768 places 128 tokens of 8 * 16 heads over 2000 states take 28 us instead of 24
template <int DP> constexpr uint32_t kTilePlaces = DP > 128 ? 256 : 512;
// units of a chunk, at least: 256 keys (128 / 256 / 512, us: 8 tokens of 32 heads of 128 behind 1000 21 / 19 / 22, 16 behind 4096 35 / 33 / 36; 198 tokens of 12 heads of 256
// over 1422 states 55 / 46 / 42, 91 tokens of 25 sequences 70 / 63 / 63, 3 tokens over 4069 states 47 / 51 / 52)
template <int DP> constexpr uint32_t kTileLeast = 256 / kTileKeys<DP>;

template <class T, int DP, bool PAGED>
int launch_tile(const AttentionProblem& p, const void* q, const void* k, const void* v, void* out, hipStream_t stream) {
    constexpr size_t LDS = tile_lds_bytes<DP>();
    static std::atomic<uint64_t> raised{0};
    if (LDS > (64u << 10))
        if (int status = raise_lds_limit(reinterpret_cast<const void*>(attention_tile_kernel<T, DP, PAGED>), LDS, raised); status != TANNIC_SUCCESS) return status;
    // As many blocks as there can be items: what is cut has no more items than places and groups together, none of fewer units than kTileLeast but a group's last.  Groups are
    // cut if they have more than 5 / 4 of a place's share: there are fewer than 4 / 5 of the places of those, and fewer than 9 / 5 parts of them.
    const uint64_t groups = (static_cast<uint64_t>(p.tokens) * p.group / kTileRows + p.sequences) * p.kv_heads, units = p.room / kTileKeys<DP> + 1;
    if (groups * units >= kMostUnits || groups + kTilePlaces<DP> >= kMostBlocks) return TANNIC_UNSUPPORTED_DTYPE;
    const uint64_t items = std::min<uint64_t>(groups + kTilePlaces<DP>, groups * ((units + kTileLeast<DP> - 1) / kTileLeast<DP>)), parts = std::min<uint64_t>(items, 2 * kTilePlaces<DP>);
    uint32_t* arrivals = nullptr;
    if (int status = attention_arrivals(stream, arrivals); status != TANNIC_SUCCESS) return status;
    static_assert(2 * kTilePlaces<DP> <= kAttentionArrivals);
    float* partial = nullptr;
    if (scratch_acquire(reinterpret_cast<void**>(&partial), parts * tile_partial_floats<DP>() * sizeof(float), stream) != TANNIC_SUCCESS) return TANNIC_ERROR;
    hipLaunchKernelGGL((attention_tile_kernel<T, DP, PAGED>), dim3(static_cast<uint32_t>(items)), dim3(64 * kTileWaves), LDS, stream, p, static_cast<const T*>(q),
                       static_cast<const T*>(k), static_cast<const T*>(v), static_cast<T*>(out), partial, arrivals, static_cast<uint32_t>(groups), kTilePlaces<DP>, kTileLeast<DP>);
    const int status = launch_status("attention_tile_kernel");
    scratch_release(partial, stream);
    return status;
}

template <class T, bool PAGED>
int pick_tile(const AttentionProblem& p, const void* q, const void* k, const void* v, void* out, hipStream_t stream) {
    if (p.d <= 64) return launch_tile<T, 64, PAGED>(p, q, k, v, out, stream);
    if (p.d <= 128) return launch_tile<T, 128, PAGED>(p, q, k, v, out, stream);
    return launch_tile<T, 256, PAGED>(p, q, k, v, out, stream);
}

int attention_tile(int dtype, const AttentionProblem& described, const void* q, const void* k, const void* v, void* out, hipStream_t stream) {
    AttentionProblem p = described;
    if (p.page == 1) p.k_token = p.v_token = p.d;      // (of one row there is no next: what the loads take for it is behind the last byte that they may reach)
    // (a lane's offsets from its wavefront's first key fit 32 bits, and rows ascend)
    const int64_t far = int64_t(1) << 25;
    if (p.k_token < p.d || p.v_token < p.d || p.k_token >= far || p.v_token >= far) return TANNIC_UNSUPPORTED_DTYPE;
    if (dtype == TANNIC_FLOAT16) return p.starts ? pick_tile<f16, true>(p, q, k, v, out, stream) : pick_tile<f16, false>(p, q, k, v, out, stream);
    if (dtype == TANNIC_BFLOAT16) return p.starts ? pick_tile<bf16, true>(p, q, k, v, out, stream) : pick_tile<bf16, false>(p, q, k, v, out, stream);
    return TANNIC_UNSUPPORTED_DTYPE;
}

}  // namespace th
