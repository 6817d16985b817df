// A paged key/value cache in four bits: writing it, reading it back and
// attention over it.
//
// A (page, key head) is one record of page_size * (D + D / 16) bytes:
//
//   key codes    [page_size][D / 2]      byte j of a row: elements 2 j (low bits), 2 j + 1
//   value codes  [D / 2][page_size]      the same bytes, token-minor
//   key scales   [page_size][D / 32]
//   value scales [D / 32][page_size]
//
// The operands of v_mfma_f32_16x16x32_bf16 are rows of eight consecutive k a
// lane: a key row is contiguous in d, which the score product sums over, and a
// value row in tokens, which the other one does. A transposed value row costs
// the append a turn of 4 x 4 bytes between lanes, once a token; the attention
// reads every byte of it for every token that follows.
#include <algorithm>
#include <type_traits>

#include "fp4.h"

namespace mlk {
namespace {

constexpr int kRun = 16;     // tokens of a page that one lane takes: page sizes are multiples of it
constexpr int kTile = 64;    // keys a wave takes at a time
constexpr int W = 8;         // waves of an attention block

struct Cache {
    uint8_t* bytes;
    int64_t record;  // bytes of a (page, head)
    int32_t pages, kv_heads, page_size;
    int32_t runs;     // page_size / kRun
    uint32_t magic;   // ceil(2^31 / runs)
    const int32_t* table;
    int32_t width;
    const int32_t* positions;
    int32_t batch, length;

    int64_t value_codes(int dim) const { return static_cast<int64_t>(page_size) * (dim / 2); }
};

// Page index of a run of 16 tokens and the run's place in it. run < 2^25 (a table's, and those looked up past its end),
// runs <= 64: the quotient by the rounded-up reciprocal is above the true one by less than run / 2^31 < 1 / runs.
__device__ __forceinline__ void split_run(const Cache& c, uint32_t run, uint32_t& page, uint32_t& token) {
    page = __umulhi(2 * run, c.magic);
    token = (run - page * static_cast<uint32_t>(c.runs)) * kRun;
}

// The record of token `at` of sequence b, and its place in the page; null where the table has no such page.
__device__ __forceinline__ uint8_t* record_of(const Cache& c, int b, int at, int head, int& offset) {
    if (at >= c.width * c.page_size) return nullptr;
    uint32_t page, first;
    split_run(c, static_cast<uint32_t>(at) / kRun, page, first);
    offset = static_cast<int>(first) + at % kRun;
    const int id = c.table[static_cast<int64_t>(b) * c.width + page];
    if (id < 0 || id >= c.pages) return nullptr;
    return c.bytes + (static_cast<int64_t>(id) * c.kv_heads + head) * c.record;
}

// ------------------------------------------------------------- append and read

struct Rows3 {
    const void* p;
    int64_t bs, ts, hs;  // element strides of a sequence, a token, a head
};

// Eight elements of a row at any alignment.
template <bool F32>
__device__ __forceinline__ void load8(const void* p, int64_t first, float (&x)[8]) {
    if constexpr (F32) {
        const u32x4_any* const from = reinterpret_cast<const u32x4_any*>(static_cast<const float*>(p) + first);
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = __uint_as_float(from[i / 4][i % 4]);
    } else {
        const u32x4 v = *reinterpret_cast<const u32x4_any*>(static_cast<const uint16_t*>(p) + first);
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = __uint_as_float(i % 2 ? v[i / 2] & 0xFFFF0000u : v[i / 2] << 16);
    }
}

// Eight results of a lane: elements first .. first + 7 of an output row.
template <bool F32>
__device__ __forceinline__ void put8(void* out, int64_t first, const float (&v)[8]) {
    if constexpr (F32) {
        float* const o = static_cast<float*>(out) + first;
        *reinterpret_cast<f32x4*>(o) = f32x4{v[0], v[1], v[2], v[3]};
        *reinterpret_cast<f32x4*>(o + 4) = f32x4{v[4], v[5], v[6], v[7]};
    } else {
        u32x4 w;
#pragma unroll
        for (int i = 0; i < 4; ++i) w[i] = float_to_bf16(v[2 * i]) | float_to_bf16(v[2 * i + 1]) << 16;
        *reinterpret_cast<u32x4*>(static_cast<uint16_t*>(out) + first) = w;
    }
}

// N bytes of a lane.
template <int N>
struct Bytes;
template <>
struct Bytes<1> {
    using type = uint8_t;
};
template <>
struct Bytes<2> {
    using type = uint16_t;
};
template <>
struct Bytes<4> {
    using type = uint32_t;
};
template <>
struct Bytes<8> {
    using type = uint64_t;
};

// A wave moves the keys, or the values, of 16 consecutive tokens of the call and one head: lane 4 t + q the eight elements
// 32 s + 8 q .. of token t for each group s, a dword of codes. A value dword is four rows of one token, where the cache
// holds rows of tokens: four lanes that hold a run of four tokens turn their 4 x 4 bytes, so that a lane moves one row's
// four tokens. Tokens that are no such run are moved byte by byte. Bound by memory: 4 x 2048 tokens of 8 heads of 128 in
// fp32 are written in 14.4 us and read in 16.4 (4.8 and 4.2 TB/s).

// Byte k of the lane whose token is i of its four against byte i of the one whose token is k; its own inverse.
__device__ __forceinline__ uint32_t turn4(uint32_t v, int i) {
    const uint32_t a = __shfl_xor(v, 4, kWave);
    v = i & 1 ? __builtin_amdgcn_perm(v, a, 0x07030501u) : __builtin_amdgcn_perm(a, v, 0x06020400u);
    const uint32_t c = __shfl_xor(v, 8, kWave);
    return i & 2 ? __builtin_amdgcn_perm(v, c, 0x07060302u) : __builtin_amdgcn_perm(c, v, 0x05040100u);
}

// Where a lane's token lies: its record (null: nowhere), its place in the page, and whether the lane's four tokens are
// four places side by side from a multiple of four.
struct Place {
    uint8_t* record;
    int offset;
    bool run;
};
__device__ __forceinline__ Place place_of(const Cache& c, uint32_t token, uint32_t b, int head) {
    Place p{nullptr, 0, false};
    const int i = (threadIdx.x >> 2) & 3;
    if (token < static_cast<uint32_t>(c.batch) * static_cast<uint32_t>(c.length)) {
        const int at = c.positions[token];
        if (at >= 0) p.record = record_of(c, static_cast<int>(b), at, head, p.offset);
    }
    bool same = p.record != nullptr && (p.offset & 3) == i;
#pragma unroll
    for (int m = 4; m <= 8; m += 4) {
        const uint64_t bits = reinterpret_cast<uint64_t>(p.record) + static_cast<uint64_t>(p.offset & ~3);
        const uint32_t low = __shfl_xor(static_cast<uint32_t>(bits), m, kWave), high = __shfl_xor(static_cast<uint32_t>(bits >> 32), m, kWave);
        same = same && (static_cast<uint64_t>(high) << 32 | low) == bits;
        const int other = __shfl_xor(static_cast<int>(same), m, kWave);
        same = same && other != 0;
    }
    p.run = same;
    return p;
}

template <int D, bool F32>
__global__ __launch_bounds__(256) void kv4_append_kernel(Cache c, Rows3 k, Rows3 v, uint32_t waves) {
    constexpr int S = D / 32;
    using Scales = typename Bytes<S>::type;
    const uint32_t id = blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
    if (id >= waves) return;
    const bool values = id & 1;
    const uint32_t tile = (id >> 1) / static_cast<uint32_t>(c.kv_heads), length = static_cast<uint32_t>(c.length);
    const int lane = threadIdx.x & 63, q = lane & 3, i = lane >> 2 & 3, head = static_cast<int>((id >> 1) - tile * c.kv_heads);
    const uint32_t token = tile * 16 + (lane >> 2), held = min(token, c.batch * length - 1), b = held / length;
    const Rows3& r = values ? v : k;
    const int64_t from = b * r.bs + static_cast<int64_t>(held - b * length) * r.ts + head * r.hs + 8 * q;
    float x[S][8];
#pragma unroll
    for (int s = 0; s < S; ++s) load8<F32>(r.p, from + 32 * s, x[s]);
    const Place place = place_of(c, token, b, head);
    uint32_t codes[S];
    uint64_t bytes = 0;
#pragma unroll
    for (int s = 0; s < S; ++s) {
        // The largest magnitude's bits; those of an infinity or a NaN are larger than any number's.
        uint32_t most = 0;
#pragma unroll
        for (int e = 0; e < 8; ++e) most = max(most, __float_as_uint(x[s][e]) & 0x7FFFFFFFu);
        most = max(most, static_cast<uint32_t>(__builtin_amdgcn_mov_dpp(static_cast<int>(most), 0xB1, 0xF, 0xF, false)));
        most = max(most, static_cast<uint32_t>(__builtin_amdgcn_mov_dpp(static_cast<int>(most), 0x4E, 0xF, 0xF, false)));
        const bool fine = most < 0x7F800000u;
        const uint32_t byte = fine ? scale_byte(__uint_as_float(most)) : 255;
        const float scale = scale_of(byte);
        uint32_t w = 0;
        w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[s][0], x[s][1], scale, 0);
        w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[s][2], x[s][3], scale, 1);
        w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[s][4], x[s][5], scale, 2);
        w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[s][6], x[s][7], scale, 3);
        codes[s] = fine ? w : 0;
        bytes |= static_cast<uint64_t>(byte) << (8 * s);
    }
    const int64_t half = static_cast<int64_t>(c.page_size) * (D / 2);
    if (!values) {
        if (place.record == nullptr) return;
        uint32_t* const to = reinterpret_cast<uint32_t*>(place.record + place.offset * (D / 2)) + q;
#pragma unroll
        for (int s = 0; s < S; ++s) to[4 * s] = codes[s];
        if (q == 0) *reinterpret_cast<Scales*>(place.record + 2 * half + place.offset * S) = static_cast<Scales>(bytes);
        return;
    }
    uint32_t turned[S];
#pragma unroll
    for (int s = 0; s < S; ++s) turned[s] = turn4(codes[s], i);
    if (place.record == nullptr) return;
    uint8_t* const to = place.record + half + 4 * q * c.page_size;
    if (place.run) {
#pragma unroll
        for (int s = 0; s < S; ++s) *reinterpret_cast<uint32_t*>(to + (16 * s + i) * c.page_size + (place.offset & ~3)) = turned[s];
    } else {
#pragma unroll
        for (int s = 0; s < S; ++s)
#pragma unroll
            for (int e = 0; e < 4; ++e) to[(16 * s + e) * c.page_size + place.offset] = static_cast<uint8_t>(codes[s] >> (8 * e));
    }
    if (q == 0) {
        uint8_t* const scales = place.record + 2 * half + S * c.page_size + place.offset;
#pragma unroll
        for (int s = 0; s < S; ++s) scales[s * c.page_size] = static_cast<uint8_t>(bytes >> (8 * s));
    }
}

template <int D, bool F32>
__global__ __launch_bounds__(256) void kv4_read_kernel(Cache c, void* k, void* v, uint32_t waves) {
    constexpr int S = D / 32;
    using Scales = typename Bytes<S>::type;
    const uint32_t id = blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
    if (id >= waves) return;
    const bool values = id & 1;
    const uint32_t tile = (id >> 1) / static_cast<uint32_t>(c.kv_heads), length = static_cast<uint32_t>(c.length);
    const int lane = threadIdx.x & 63, q = lane & 3, i = lane >> 2 & 3, head = static_cast<int>((id >> 1) - tile * c.kv_heads);
    const uint32_t token = tile * 16 + (lane >> 2), all = c.batch * length;
    const Place place = place_of(c, token, token / length, head);
    const int64_t half = static_cast<int64_t>(c.page_size) * (D / 2);
    uint32_t codes[S];
    uint64_t bytes = 0;
#pragma unroll
    for (int s = 0; s < S; ++s) codes[s] = 0;
    if (place.record != nullptr) {
        if (!values) {
            const uint32_t* const from = reinterpret_cast<const uint32_t*>(place.record + place.offset * (D / 2)) + q;
#pragma unroll
            for (int s = 0; s < S; ++s) codes[s] = from[4 * s];
            bytes = *reinterpret_cast<const Scales*>(place.record + 2 * half + place.offset * S);
        } else {
            const uint8_t* const from = place.record + half + 4 * q * c.page_size;
            if (place.run) {
#pragma unroll
                for (int s = 0; s < S; ++s) codes[s] = *reinterpret_cast<const uint32_t*>(from + (16 * s + i) * c.page_size + (place.offset & ~3));
            } else {
#pragma unroll
                for (int s = 0; s < S; ++s)
#pragma unroll
                    for (int e = 0; e < 4; ++e) codes[s] |= static_cast<uint32_t>(from[(16 * s + e) * c.page_size + place.offset]) << (8 * e);
            }
            const uint8_t* const scales = place.record + 2 * half + S * c.page_size + place.offset;
#pragma unroll
            for (int s = 0; s < S; ++s) bytes |= static_cast<uint64_t>(scales[s * c.page_size]) << (8 * s);
        }
    }
    if (values) {
#pragma unroll
        for (int s = 0; s < S; ++s) {
            const uint32_t turned = turn4(codes[s], i);
            if (place.run) codes[s] = turned;
        }
    }
    if (token >= all) return;
    if (place.record == nullptr) bytes = c.positions[token] < 0 ? 0 : ~uint64_t{0};  // zero codes, or NaN
    const int64_t to = (static_cast<int64_t>(token) * c.kv_heads + head) * D + 8 * q;
#pragma unroll
    for (int s = 0; s < S; ++s) {
        const bf16x8 x = fp4_octet(codes[s], scale_of(static_cast<uint32_t>(bytes >> (8 * s)) & 0xFF));
        float out[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) out[e] = static_cast<float>(x[e]);
        put8<F32>(values ? v : k, to + 32 * s, out);
    }
}

// ------------------------------------------------------------- attention

struct AttentionArgs {
    Cache c;
    const void* q;
    int64_t q_bs, q_ts, q_hs;
    int32_t heads, group;  // query heads; query heads to a key head
    int32_t rows;          // of a (sequence, key head): length * group; row r = token r / group, head r % group
    int32_t row_tiles, splits;
    float scale_log2;
    void* out;    // [batch, length, heads, D]
    float* part;  // [batch, kv_heads, rows, splits][D], then [...][2] (maximum, sum)
    int64_t part_rows;
};

// Of 16 lanes each: `v` of the lane 4, 8 or 12 below (kUp) or above (kDown), or 4 or 8 around, in the lanes of the
// quarters that `kQuarters` names; `old` elsewhere, 0 past the ends.
constexpr int kDown4 = 0x104, kDown8 = 0x108, kDown12 = 0x10C, kUp4 = 0x114, kUp8 = 0x118, kUp12 = 0x11C, kAround4 = 0x124, kAround8 = 0x128;
template <int kMove, int kQuarters>
__device__ __forceinline__ float from_lanes(float old, float v) {
    return __int_as_float(__builtin_amdgcn_update_dpp(__float_as_int(old), __float_as_int(v), kMove, 0xF, kQuarters, true));
}
__device__ __forceinline__ float max_over_groups(float v) {
    v = fmaxf(v, __shfl_xor(v, 16, kWave));
    return fmaxf(v, __shfl_xor(v, 32, kWave));
}
__device__ __forceinline__ float sum_over_groups(float v) {
    v += __shfl_xor(v, 16, kWave);
    return v + __shfl_xor(v, 32, kWave);
}
__device__ __forceinline__ float finite_or_zero(float m) { return m == -INFINITY ? 0.0f : m; }

// What a wave holds in LDS of its tile of 64 keys: their codes, then, once they are in registers, the values'.
template <int S>
struct TileLds {
    u32x4 codes[64 * S];        // keys: row l of key tile a, 16-byte piece c at (16 a + l) S + (c ^ turn(l)); values: row j,
                                // piece c at 4 j + (c ^ (j / 2 & 3))
    uint8_t key_scale[64 * S];  // of row l of key tile a at (4 l + a) S
    uint8_t value_scale[64 * S];  // [S][64]
    // Eight lanes that read, or write, together meet in different banks.
    static __device__ __forceinline__ int turn(int l) { return S == 8 ? l & 7 : S == 4 ? l >> 1 & 3 : S == 2 ? l >> 2 & 1 : 0; }
};

// A block takes 16 rows of a (sequence, key head) and every p.splits-th group of W tiles of 64 keys, a tile a wave.
//
// Bound by memory in bf16 (64 sequences of 10000 keys, 32 heads on 8 of 128: 127 us, 5.5 TB/s), by the latencies of some
// 400 vector and 96 matrix instructions a tile in fp32 (172 us, 4.0 TB/s: three planes of each query and weight), with the
// two waves a SIMD that the registers allow; one tile a wave alone takes about 5 us, most of it waiting for memory.
//
// Scores are key tile x q^T, so that lane (g, l) holds row l's scores of 16 tokens, in the registers from which the
// product with the values takes its weights: nothing moves between lanes but the maximum (a column's sum is formed at
// the end). Key tile a, row 4 g' + r is token 16 g' + 4 a + r of the 64, so that a lane's scores (rows 4 g .. 4 g + 3 of
// every tile) are its 16 tokens 16 g .. 16 g + 15 of the value product.
// WHOLE: pages of whole tiles. A tile then has one page, and its addresses are scalar. Not for D = 256, where the
// registers that this takes are spilled (64 x 4000 keys of 8 heads, fp32: 161 against 138 us).
// FEW: up to four rows, a token of as many query heads a key head. 12 of 16 columns of a product are then idle, and their
// lanes take three quarters of the rows' softmax (64 x 10000 keys, fp32 181 -> 172 us; 16 x 16000 of 8 heads of 64, fp32
// 45 -> 41; of 32, bf16 22 -> 20).
template <int D, bool F32, bool WHOLE, bool FEW>
__global__ __launch_bounds__(W * 64, D == 32 || (D == 64 && !F32) ? 4 : 2) void kv4_attention_kernel(AttentionArgs p) {
    constexpr int S = D / 32;       // k steps of a score product, groups of a token, 1 KB loads of a tile's keys (or values)
    constexpr int P = F32 ? 3 : 1;  // bf16 operands that make up a query or a weight
    constexpr bool kShared = F32 || S == 8;  // q in LDS: its registers would cost the second wave a SIMD
    using Scales = typename Bytes<S>::type;
    struct Exchange {
        f32x4 acc[W][2 * S][64];
        float stats[W][2][16];
    };
    __shared__ union {
        TileLds<S> tile[W];
        Exchange end;
    } lds;
    __shared__ bf16x8 shared_q[kShared ? P * S : 1][64];
    const Cache& c = p.c;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64), lane = threadIdx.x & 63, g = lane >> 4, l = lane & 15;
    unsigned id = blockIdx.x;
    const int split = id % p.splits;
    id /= p.splits;
    const int row0 = static_cast<int>(id % p.row_tiles) * 16;
    id /= p.row_tiles;
    const int head = id % c.kv_heads, b = id / c.kv_heads;
    const int capacity = c.width * c.page_size;
    const int64_t half = static_cast<int64_t>(c.page_size) * (D / 2), page_stride = c.kv_heads * c.record;
    const int32_t* const table = c.table + static_cast<int64_t>(b) * c.width;
    const uint8_t* const records = c.bytes + head * c.record;
    TileLds<S>& mine = lds.tile[wave];

    // Loads take 16 bytes a lane of whole stretches of memory (in operand order every lane would be a cache access of its
    // own); a tile is 4 runs of 16 tokens, each on a page of its own for all that is known. Keys: load t is bytes 1024 t ..
    // of [64][D / 2]; values: rows 16 t .. of [D / 2][64], run lane & 3; scales: S bytes a lane of [64][S] and [S][64].
    // A run on no page is read from page 0 and its keys made NaN, which only rows that see them take.
    struct Ids {
        int32_t by_group, by_piece;  // pages of runs g and lane & 3; the tile's page
    };
    uint32_t no_lane;
    asm("v_mov_b32 %0, 0" : "=v"(no_lane));
    auto lookup = [&](int tile) {
        auto page_of = [&](int run) {
            uint32_t page, token;
            split_run(c, 4 * tile + run, page, token);
            return page < static_cast<uint32_t>(c.width) ? table[page] : -1;
        };
        if constexpr (WHOLE) {
            // A vector load, waited for with the tile's: the scalar unit's would be waited for by the next read of LDS.
            uint32_t page, token;
            split_run(c, 4 * tile, page, token);
            return Ids{page < static_cast<uint32_t>(c.width) ? table[page + no_lane] : -1, 0};
        }
        return Ids{page_of(g), page_of(lane & 3)};
    };
    u32x4 key_ahead[S], value_ahead[S];
    Scales key_scale_ahead, value_scale_ahead;
    bool missing = false;  // the page of key_scale_ahead: looked at when the tile is used, a select here would wait for the loads
    auto load_whole = [&](int tile, const Ids& ids) {
        const int id = __builtin_amdgcn_readfirstlane(ids.by_group);
        missing = id < 0 || id >= c.pages;
        uint32_t page, token;
        split_run(c, 4 * tile, page, token);
        const uint8_t* const record = records + (missing ? 0 : id) * page_stride;
        const uint8_t* const keys = record + token * (D / 2);
        const uint8_t* const values = record + half + token;
        const uint8_t* const scales = record + 2 * half;
#pragma unroll
        for (int t = 0; t < S; ++t) key_ahead[t] = *reinterpret_cast<const u32x4*>(keys + static_cast<uint32_t>(1024 * t + 16 * lane));
#pragma unroll
        for (int t = 0; t < S; ++t)
            value_ahead[t] = *reinterpret_cast<const u32x4*>(values + static_cast<uint32_t>((16 * t + (lane >> 2)) * c.page_size + 16 * (lane & 3)));
        key_scale_ahead = *reinterpret_cast<const Scales*>(scales + token * S + static_cast<uint32_t>(lane * S));
        value_scale_ahead = *reinterpret_cast<const Scales*>(scales + S * c.page_size + token +
                                                             static_cast<uint32_t>(lane * S / 64 * c.page_size + lane * S % 64));
    };
    auto load = [&](int tile, const Ids& ids) {
        if constexpr (WHOLE) return load_whole(tile, ids);
        missing = ids.by_group < 0 || ids.by_group >= c.pages;
        const int group_id = missing ? 0 : ids.by_group, piece_id = ids.by_piece < 0 || ids.by_piece >= c.pages ? 0 : ids.by_piece;
        uint32_t page, token;
#pragma unroll
        for (int t = 0; t < S; ++t) {
            const int run = S == 8 ? t / 2 : S == 4 ? t : S == 2 ? 2 * t + (lane >> 5) : g;
            const int key_id = S >= 4 ? __builtin_amdgcn_readlane(group_id, 16 * run) : S == 2 ? __shfl(group_id, 16 * run, kWave) : group_id;
            split_run(c, 4 * tile + run, page, token);
            key_ahead[t] = *reinterpret_cast<const u32x4*>(records + key_id * page_stride + (token * (D / 2) + 1024 * t + 16 * lane - run * (8 * D)));
        }
        split_run(c, 4 * tile + (lane & 3), page, token);
        const uint8_t* const value = records + piece_id * page_stride + half + ((lane >> 2) * c.page_size + static_cast<int>(token));
#pragma unroll
        for (int t = 0; t < S; ++t) value_ahead[t] = *reinterpret_cast<const u32x4*>(value + 16 * t * c.page_size);
        split_run(c, 4 * tile + g, page, token);
        key_scale_ahead = *reinterpret_cast<const Scales*>(records + group_id * page_stride + 2 * half + (static_cast<int>(token) + l) * S);
        const int at = lane * S % 64, run = at / 16;  // token of the lane's value scales
        split_run(c, 4 * tile + run, page, token);
        const int value_id = S == 1 ? group_id : __shfl(group_id, 16 * run, kWave);
        value_scale_ahead = *reinterpret_cast<const Scales*>(records + value_id * page_stride + 2 * half +
                                                             ((S + lane * S / 64) * c.page_size + static_cast<int>(token) + at % 16));
    };
    // The first tile is on its way before the rows are known.
    const int stride = W * p.splits, first_tile = split * W + wave;
    Ids ids = lookup(first_tile);
    load(first_tile, ids);
    ids = lookup(first_tile + stride);

    // Rows, their positions, and q as operands, times the sign of the scale: the largest score is then the one of the
    // largest weight.
    const float factor = p.scale_log2 > 0.0f ? 1.0f : p.scale_log2 < 0.0f ? -1.0f : 0.0f;
    const float scale = p.scale_log2 == 0.0f ? 1.0f : fabsf(p.scale_log2);
    const int row = row0 + l, token = min(row, p.rows - 1) / p.group, of_group = min(row, p.rows - 1) - token * p.group;
    const int at = c.positions[static_cast<int64_t>(b) * c.length + token];
    const int position = row < p.rows && at < capacity ? at : -1;
    bf16x8 q[P][kShared ? 1 : S];
    const int64_t q_from = b * p.q_bs + token * p.q_ts + (head * p.group + of_group) * p.q_hs + (D / 4) * g;
#pragma unroll
    for (int s = 0; s < S; ++s) {
        if (kShared && s % W != wave) continue;
        float x[8];
        load8<F32>(p.q, q_from + 8 * s, x);
        bf16x8 operand[P];
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] *= factor;
        if constexpr (F32) {
            planes_of<true>(x, operand);
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) operand[0][i] = static_cast<__bf16>(x[i]);
        }
#pragma unroll
        for (int i = 0; i < P; ++i) {
            if constexpr (kShared) {
                shared_q[s * P + i][lane] = operand[i];
            } else {
                q[i][s] = operand[i];
            }
        }
    }
    int last = position, least = position < 0 ? 0x7FFFFFFF : position;
#pragma unroll
    for (int i = 1; i < 16; i *= 2) {
        last = max(last, __shfl_xor(last, i, kWave));
        least = min(least, __shfl_xor(least, i, kWave));
    }
    last = __builtin_amdgcn_readfirstlane(last);  // of all lanes alike
    least = __builtin_amdgcn_readfirstlane(least);
    if constexpr (kShared) __syncthreads();

    float top = -INFINITY, sum = 0.0f;  // the largest score so far, and the lane's part of the sum of 2^(scale (score - top))
    f32x4 acc[S][2];                    // elements 32 s + 8 g + 2 r and the next, of row l
#pragma unroll
    for (int s = 0; s < S; ++s) acc[s][0] = acc[s][1] = f32x4{0, 0, 0, 0};

    for (int tile = first_tile; tile * kTile <= last; tile += stride) {
        const int first = tile * kTile;
#pragma unroll
        for (int t = 0; t < S; ++t) {
            const int at = 64 * t + lane, token = at / S, row = token >> 4 << 2 | (token & 3), a = token >> 2 & 3;
            mine.codes[(16 * a + row) * S + (at % S ^ mine.turn(row))] = key_ahead[t];
        }
        reinterpret_cast<Scales*>(mine.key_scale)[4 * (4 * g + (l & 3)) + (l >> 2)] =
            missing ? static_cast<Scales>(~uint64_t{0}) : key_scale_ahead;  // token 16 g + l
        reinterpret_cast<Scales*>(mine.value_scale)[lane] = value_scale_ahead;
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        uint32_t kc[4][S], ks[4];
        // The scales of a lane's part of a key row: byte g of four (S = 4), g / 2 of two, the only one, or 2 g and 2 g + 1.
        const uint8_t* const key_scales = mine.key_scale + 4 * l * S;
#pragma unroll
        for (int a = 0; a < 4; ++a) {
            const uint8_t* const row = reinterpret_cast<const uint8_t*>(mine.codes + (16 * a + l) * S);
            if constexpr (S == 1) {
                kc[a][0] = reinterpret_cast<const uint32_t*>(row)[g];
                ks[a] = key_scales[a];
            }
            if constexpr (S == 2) {
                const u32x2 v = reinterpret_cast<const u32x2*>(row + 16 * (g >> 1 ^ mine.turn(l)))[g & 1];
                kc[a][0] = v[0], kc[a][1] = v[1];
                ks[a] = key_scales[2 * a + (g >> 1)];
            }
            if constexpr (S >= 4) {
#pragma unroll
                for (int i = 0; i < S / 4; ++i) {
                    const u32x4 v = reinterpret_cast<const u32x4*>(row)[(S / 4 * g + i) ^ mine.turn(l)];
#pragma unroll
                    for (int j = 0; j < 4; ++j) kc[a][4 * i + j] = v[j];
                }
                ks[a] = S == 4 ? key_scales[4 * a + g] : reinterpret_cast<const uint16_t*>(key_scales)[4 * a + g];
            }
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
#pragma unroll
        for (int t = 0; t < S; ++t) {
            const int j = 16 * t + (lane >> 2);
            mine.codes[4 * j + ((lane & 3) ^ (j >> 1 & 3))] = value_ahead[t];
        }
        if ((tile + stride) * kTile <= last) {
            load(tile + stride, ids);
            ids = lookup(tile + 2 * stride);
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");

        f32x4 score[4];
#pragma unroll
        for (int a = 0; a < 4; ++a) score[a] = f32x4{0, 0, 0, 0};
#pragma unroll
        for (int s = 0; s < S; ++s) {
            bf16x8 qs[P];
#pragma unroll
            for (int i = 0; i < P; ++i) {
                if constexpr (kShared) {
                    qs[i] = shared_q[s * P + i][lane];
                } else {
                    qs[i] = q[i][s];
                }
            }
#pragma unroll
            for (int a = 0; a < 4; ++a) {
                const bf16x8 k = fp4_octet(kc[a][s], s < 4 ? scale_at<0>(ks[a]) : scale_at<1>(ks[a]));
#pragma unroll
                for (int i = P - 1; i >= 0; --i) score[a] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(k, qs[i], score[a], 0, 0, 0);
            }
        }

        const bool masked = first + kTile - 1 > least;  // some row does not see the whole tile
        if (masked) {
#pragma unroll
            for (int i = 0; i < 16; ++i) score[i / 4][i % 4] = first + 16 * g + i > position ? -INFINITY : score[i / 4][i % 4];
        }
        // Scores to weights 2^(scale (score - top)), `top` the largest of a row so far.
        auto soften = [&](auto& v, auto over_lanes) {
            float most = -INFINITY;
#pragma unroll
            for (float x : v) most = fmaxf(most, x);
            const float now = fmaxf(top, max_over_groups(over_lanes(most)));
            if (__ballot(now != top) != 0) {  // seldom after the first tiles
                const float shrink = __builtin_amdgcn_exp2f(fmaf(top, scale, -finite_or_zero(now) * scale));
                top = now;
                sum *= shrink;
#pragma unroll
                for (int s = 0; s < S; ++s) {
                    acc[s][0] *= shrink;
                    acc[s][1] *= shrink;
                }
            }
            const float base = finite_or_zero(top) * scale;
#pragma unroll
            for (float& x : v) {
                x = __builtin_amdgcn_exp2f(fmaf(x, scale, -base));
                sum += x;
            }
        };
        // Eight weights as operands. fp32: of finite values, or NaN. bf16: rounded to nearest, by up to 2^-8 of a weight; the
        // sum is of the unrounded. An output's error grows by it from the 0.0016 or 0.0017 of its own rounding to 0.0017 (one
        // stream of 131072 keys) to 0.0020 (32 x 8000); what is left of each weight as a second operand would take it away
        // again, in 5 to 8% more time (32 x 8000 keys 40.2 -> 43.5 us, 64 x 10000 93 -> 98).
        auto operand_of = [&](const float (&w)[8], bf16x8 (&to)[P]) {
            if constexpr (F32) {
                planes_of<false>(w, to);
            } else {
#pragma unroll
                for (int i = 0; i < 8; ++i) to[0][i] = static_cast<__bf16>(w[i]);
            }
        };
        bf16x8 weight[P][2];
        if constexpr (FEW) {
            // Lane 4 a + r of 16 takes row r's scores of key tile a from lane r, and gives its weights back.
            float v[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                v[i] = score[0][i];
                v[i] = from_lanes<kUp4, 2>(v[i], score[1][i]);
                v[i] = from_lanes<kUp8, 4>(v[i], score[2][i]);
                v[i] = from_lanes<kUp12, 8>(v[i], score[3][i]);
            }
            soften(v, [](float most) {
                most = fmaxf(most, from_lanes<kAround4, 15>(most, most));
                return fmaxf(most, from_lanes<kAround8, 15>(most, most));
            });
            const float both[8] = {v[0], v[1], v[2], v[3], 0, 0, 0, 0};
            bf16x8 mine_of[P];
            operand_of(both, mine_of);
#pragma unroll
            for (int i = 0; i < P; ++i) {
                const u32x4 w = __builtin_bit_cast(u32x4, mine_of[i]);
                u32x4 first, second;
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    const float x = __uint_as_float(w[j]);
                    first[j] = w[j];
                    first[2 + j] = __float_as_uint(from_lanes<kDown4, 15>(0.0f, x));
                    second[j] = __float_as_uint(from_lanes<kDown8, 15>(0.0f, x));
                    second[2 + j] = __float_as_uint(from_lanes<kDown12, 15>(0.0f, x));
                }
                weight[i][0] = __builtin_bit_cast(bf16x8, first);
                weight[i][1] = __builtin_bit_cast(bf16x8, second);
            }
        } else {
            float v[16];
#pragma unroll
            for (int i = 0; i < 16; ++i) v[i] = score[i / 4][i % 4];
            soften(v, [](float most) { return most; });
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                float w[8];
#pragma unroll
                for (int i = 0; i < 8; ++i) w[i] = v[8 * h + i];
                bf16x8 to[P];
                operand_of(w, to);
#pragma unroll
                for (int i = 0; i < P; ++i) weight[i][h] = to[i];
            }
        }

        uint32_t poison = 0;
#pragma unroll
        for (int s = 0; s < S; ++s) {
            u32x4 vs = reinterpret_cast<const u32x4*>(mine.value_scale)[4 * s + g];
            if (masked) {
                // A value that no row may see must not reach a sum as 0 * NaN, or 0 * infinity (values under bytes 253 and
                // 254 can pass bf16's largest): such a scale goes, and the rows that do see it are made NaN below.
#pragma unroll
                for (int i = 0; i < 16; ++i)
                    if ((vs[i / 4] >> (8 * (i % 4)) & 0xFF) > kMostScale) {
                        vs[i / 4] &= ~(0xFFu << (8 * (i % 4)));
                        if (first + 16 * g + i <= position) poison |= 1u << s;
                    }
            }
            const u32x4 codes = mine.codes[4 * (16 * s + l) + (g ^ (l >> 1 & 3))];
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                uint32_t pair[8];  // elements 2 j and 2 j + 1 of a token
#pragma unroll
                for (int w = 0; w < 2; ++w) {
                    const uint32_t code = codes[2 * h + w], scales = vs[2 * h + w];
                    pair[4 * w] = fp4_pair<0>(code, scale_at<0>(scales));
                    pair[4 * w + 1] = fp4_pair<1>(code, scale_at<1>(scales));
                    pair[4 * w + 2] = fp4_pair<2>(code, scale_at<2>(scales));
                    pair[4 * w + 3] = fp4_pair<3>(code, scale_at<3>(scales));
                }
                u32x4 even, odd;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    even[i] = __builtin_amdgcn_perm(pair[2 * i + 1], pair[2 * i], 0x05040100u);
                    odd[i] = __builtin_amdgcn_perm(pair[2 * i + 1], pair[2 * i], 0x07060302u);
                }
#pragma unroll
                for (int i = P - 1; i >= 0; --i) {
                    acc[s][0] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, even), weight[i][h], acc[s][0], 0, 0, 0);
                    acc[s][1] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, odd), weight[i][h], acc[s][1], 0, 0, 0);
                }
            }
        }
        if (masked && __ballot(poison != 0) != 0) {
            poison |= __shfl_xor(poison, 16, kWave);
            poison |= __shfl_xor(poison, 32, kWave);
#pragma unroll
            for (int s = 0; s < S; ++s)
                if (poison >> s & 1) acc[s][0] = acc[s][1] = f32x4{NAN, NAN, NAN, NAN};
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    }

    // The waves' parts joined: each writes its own, wave s adds up elements 32 s .. 32 s + 31 of the rows.
    __syncthreads();
    auto& stats = lds.end.stats;
    if constexpr (FEW) {
        sum += __shfl_xor(sum, 4, kWave);
        sum += __shfl_xor(sum, 8, kWave);
    }
    sum = sum_over_groups(sum);
    if (g == 0) {
        stats[wave][0][l] = top;
        stats[wave][1][l] = sum;
    }
#pragma unroll
    for (int s = 0; s < S; ++s) {
        lds.end.acc[wave][2 * s][lane] = acc[s][0];
        lds.end.acc[wave][2 * s + 1][lane] = acc[s][1];
    }
    __syncthreads();
    static_assert(W >= S);
    if (wave >= S || row >= p.rows) return;
    float all_top = -INFINITY, all_sum = 0.0f;
#pragma unroll
    for (int w = 0; w < W; ++w) all_top = fmaxf(all_top, stats[w][0][l]);
    const float base = finite_or_zero(all_top) * scale;
    float v[8] = {0, 0, 0, 0, 0, 0, 0, 0};
#pragma unroll
    for (int w = 0; w < W; ++w) {
        const float by = __builtin_amdgcn_exp2f(fmaf(stats[w][0][l], scale, -base));
        all_sum = fmaf(stats[w][1][l], by, all_sum);
        const f32x4 even = lds.end.acc[w][2 * wave][lane], odd = lds.end.acc[w][2 * wave + 1][lane];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            v[2 * i] = fmaf(even[i], by, v[2 * i]);
            v[2 * i + 1] = fmaf(odd[i], by, v[2 * i + 1]);
        }
    }
    const int first = 32 * wave + 8 * g;
    if (p.splits > 1) {
        const int64_t part = ((static_cast<int64_t>(b) * c.kv_heads + head) * p.rows + row) * p.splits + split;
        put8<true>(p.part, part * D + first, v);
        if (wave == 0 && g == 0) {
            float* const st = p.part + p.part_rows * D + 2 * part;
            st[0] = all_top * scale;
            st[1] = all_sum;
        }
        return;
    }
    const float by = 1.0f / all_sum;
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = at < 0 ? 0.0f : (at >= capacity ? NAN : v[i] * by);
    put8<F32>(p.out, ((static_cast<int64_t>(b) * c.length + token) * p.heads + head * p.group + of_group) * D + first, v);
}

// Heads of 128 only: with 64, what the lanes convert for themselves is half as much, and sharing it gained nothing.
constexpr int kSharedDim = 128;
// Tiles of 16 rows of a wave: what its queries, sums and scores leave of the registers of two waves a SIMD.
template <bool F32>
constexpr int kRowTiles = F32 ? 1 : 2;

// Many rows: a block takes 16 MT rows a wave of a (sequence, key head), and its waves share each tile of 64 keys as bf16
// operands in LDS. A wave of the kernel above spends most of its instructions on converting keys and values, for 16 rows
// (512 tokens of two sequences over 8192 keys took 270 us so); here it converts an eighth of them, for 128 MT. A tile
// passes through registers (three tiles ahead), LDS as it lies in memory (two ahead) and LDS as operands (one ahead).
// 1 x 512 tokens over 8192 keys, 32 heads on 8: 111 us, 620 TFLOP/s; while a CU is at work its vector units issue for 55%
// of the time, its matrix cores are busy for 33% and its LDS for 29%. Converting at the end of a tile in one of the two
// waves, so that the other's products meet it, took 6% longer.
//
// Operands: key tile a, k step s is unit a S + s; values of group s and half h of a lane's 16 tokens, their even and odd
// elements, are unit 2 s + h.
template <bool F32>
__global__ __launch_bounds__(W * 64, 2) void kv4_attention_rows_kernel(AttentionArgs p) {
    constexpr int D = kSharedDim, S = D / 32, P = F32 ? 3 : 1, MT = kRowTiles<F32>;
    using Scales = typename Bytes<S>::type;
    constexpr int kKeyUnits = 4 * S, kValueUnits = 2 * S;  // a value unit is two operands
    static_assert(2 * S == W, "a wave loads 1 KB of keys or values, and converts two key units and a value unit");
    struct Raw {
        u32x4 key[64 * S], value[64 * S];  // as TileLds has them
        uint8_t key_scale[64 * S], value_scale[64 * S];
    };
    __shared__ Raw raw[2];
    __shared__ bf16x8 key_lds[2][kKeyUnits][64], value_lds[2][kValueUnits][2][64];
    __shared__ int nan_tile[2];  // the last tile of the buffer that held a value group under a byte above kMostScale, plus one
    __shared__ int wave_last[W];
    const Cache& c = p.c;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64), lane = threadIdx.x & 63, g = lane >> 4, l = lane & 15;
    unsigned id = blockIdx.x;
    const int split = id % p.splits;
    id /= p.splits;
    const int block_row = static_cast<int>(id % p.row_tiles) * (W * 16 * MT), row0 = block_row + wave * (16 * MT);
    id /= p.row_tiles;
    const int head = id % c.kv_heads, b = id / c.kv_heads;
    const int capacity = c.width * c.page_size;
    const int64_t half = static_cast<int64_t>(c.page_size) * (D / 2), page_stride = c.kv_heads * c.record;
    const int32_t* const table = c.table + static_cast<int64_t>(b) * c.width;
    const uint8_t* const records = c.bytes + head * c.record;
    if (threadIdx.x < 2) nan_tile[threadIdx.x] = 0;

    struct Ids {
        int32_t by_group, by_piece;  // pages of runs g and lane & 3
    };
    auto lookup = [&](int tile) {
        auto page_of = [&](int run) {
            uint32_t page, token;
            split_run(c, 4 * tile + run, page, token);
            return page < static_cast<uint32_t>(c.width) ? table[page] : -1;
        };
        return Ids{page_of(g), page_of(lane & 3)};
    };
    u32x4 ahead;
    Scales scale_ahead = 0;
    bool missing = false;  // the page of scale_ahead: put in its place with keep, a select at the load would wait for it
    auto load = [&](int tile, const Ids& ids) {
        missing = ids.by_group < 0 || ids.by_group >= c.pages;
        const int group_id = missing ? 0 : ids.by_group, piece_id = ids.by_piece < 0 || ids.by_piece >= c.pages ? 0 : ids.by_piece;
        uint32_t page, token;
        if (wave < S) {
            const int at = (64 * wave + lane) / S, run = at / 16;
            const int key_id = __shfl(group_id, 16 * run, kWave);
            split_run(c, 4 * tile + run, page, token);
            ahead = *reinterpret_cast<const u32x4*>(records + key_id * page_stride + ((static_cast<int>(token) + at % 16) * (D / 2) + lane % S * 16));
        } else {
            split_run(c, 4 * tile + (lane & 3), page, token);
            const int at = (16 * (wave - S) + (lane >> 2)) * c.page_size + static_cast<int>(token);
            ahead = *reinterpret_cast<const u32x4*>(records + piece_id * page_stride + half + at);
        }
        if (wave == W - 1) {
            split_run(c, 4 * tile + g, page, token);
            scale_ahead = *reinterpret_cast<const Scales*>(records + group_id * page_stride + 2 * half + (static_cast<int>(token) + l) * S);
        }
        if (wave == W - 2) {
            const int at = lane * S % 64, run = at / 16;
            const int value_id = __shfl(group_id, 16 * run, kWave);
            split_run(c, 4 * tile + run, page, token);
            const int place = (S + lane * S / 64) * c.page_size + static_cast<int>(token) + at % 16;
            scale_ahead = *reinterpret_cast<const Scales*>(records + value_id * page_stride + 2 * half + place);
        }
    };
    auto keep = [&](int buffer) {
        if (wave < S) {
            const int at = 64 * wave + lane, token = at / S, row = token >> 4 << 2 | (token & 3), a = token >> 2 & 3;
            raw[buffer].key[(16 * a + row) * S + (at % S ^ TileLds<S>::turn(row))] = ahead;
        } else {
            const int j = 16 * (wave - S) + (lane >> 2);
            raw[buffer].value[4 * j + ((lane & 3) ^ (j >> 1 & 3))] = ahead;
        }
        if (wave == W - 1)
            reinterpret_cast<Scales*>(raw[buffer].key_scale)[4 * (4 * g + (l & 3)) + (l >> 2)] = missing ? static_cast<Scales>(~uint64_t{0}) : scale_ahead;
        if (wave == W - 2) reinterpret_cast<Scales*>(raw[buffer].value_scale)[lane] = scale_ahead;
    };
    auto convert = [&](int tile, int buffer) {
        const Raw& from = raw[buffer];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int unit = W * i + wave, a = unit / S, step = unit % S;  // a lane's 8 elements: D / 4 g + 8 step ..
            const int byte = D / 8 * g + 4 * step;
            const uint32_t code = reinterpret_cast<const uint32_t*>(from.key + (16 * a + l) * S + (byte / 16 ^ TileLds<S>::turn(l)))[byte % 16 / 4];
            key_lds[buffer][unit][lane] = fp4_octet(code, scale_of(from.key_scale[(4 * l + a) * S + byte / 16]));
        }
        bool nan = false;
        const int s = wave / 2, h = wave % 2;
        const u32x2 codes = reinterpret_cast<const u32x2*>(from.value + 4 * (16 * s + l) + (g ^ (l >> 1 & 3)))[h];
        const u32x2 scales_of = reinterpret_cast<const u32x2*>(from.value_scale + 64 * s + 16 * g)[h];
        uint32_t pair[8];
#pragma unroll
        for (int w = 0; w < 2; ++w) {
            const uint32_t code = codes[w];
            uint32_t scales = scales_of[w];
            // A NaN group, or one that may hold infinities, must not meet the weight 0 of a row that does not see it: it
            // counts as small here, and the rows that see it are made NaN by themselves.
            if (((scales & 0x7F7F7F7Fu) + 0x01010101u * (0x7F - (kMostScale & 0x7F))) & scales & 0x80808080u) {
                nan = true;
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if ((scales >> (8 * e) & 0xFF) > kMostScale) scales &= ~(0xFFu << (8 * e));
            }
            pair[4 * w] = fp4_pair<0>(code, scale_at<0>(scales));
            pair[4 * w + 1] = fp4_pair<1>(code, scale_at<1>(scales));
            pair[4 * w + 2] = fp4_pair<2>(code, scale_at<2>(scales));
            pair[4 * w + 3] = fp4_pair<3>(code, scale_at<3>(scales));
        }
        u32x4 even, odd;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            even[e] = __builtin_amdgcn_perm(pair[2 * e + 1], pair[2 * e], 0x05040100u);
            odd[e] = __builtin_amdgcn_perm(pair[2 * e + 1], pair[2 * e], 0x07060302u);
        }
        value_lds[buffer][wave][0][lane] = __builtin_bit_cast(bf16x8, even);
        value_lds[buffer][wave][1][lane] = __builtin_bit_cast(bf16x8, odd);
        if (nan) nan_tile[buffer] = tile + 1;
    };

    const float factor = p.scale_log2 > 0.0f ? 1.0f : p.scale_log2 < 0.0f ? -1.0f : 0.0f;
    const float scale = p.scale_log2 == 0.0f ? 1.0f : fabsf(p.scale_log2);
    int position[MT], least = 0x7FFFFFFF, last = -1;
    bf16x8 q[MT][P][S];
#pragma unroll
    for (int m = 0; m < MT; ++m) {
        const int row = row0 + 16 * m + l, clamped = min(row, p.rows - 1), token = clamped / p.group;
        const int at = c.positions[static_cast<int64_t>(b) * c.length + token];
        position[m] = row < p.rows && at < capacity ? at : -1;
        last = max(last, position[m]);
        least = min(least, position[m] < 0 ? 0x7FFFFFFF : position[m]);
        const int64_t from = b * p.q_bs + token * p.q_ts + (head * p.group + clamped - token * p.group) * p.q_hs + (D / 4) * g;
#pragma unroll
        for (int s = 0; s < S; ++s) {
            float x[8];
            load8<F32>(p.q, from + 8 * s, x);
#pragma unroll
            for (int i = 0; i < 8; ++i) x[i] *= factor;
            if constexpr (F32) {
                bf16x8 plane[3];
                planes_of<true>(x, plane);
#pragma unroll
                for (int i = 0; i < 3; ++i) q[m][i][s] = plane[i];
            } else {
#pragma unroll
                for (int i = 0; i < 8; ++i) q[m][0][s][i] = static_cast<__bf16>(x[i]);
            }
        }
    }
#pragma unroll
    for (int i = 1; i < 16; i *= 2) {
        last = max(last, __shfl_xor(last, i, kWave));
        least = min(least, __shfl_xor(least, i, kWave));
    }
    // The block goes as far as its furthest row.
    if (lane == 0) wave_last[wave] = last;
    __syncthreads();
    int block_last = -1;
#pragma unroll
    for (int w = 0; w < W; ++w) block_last = max(block_last, wave_last[w]);

    float top[MT], sum[MT];
    f32x4 acc[MT][S][2];
#pragma unroll
    for (int m = 0; m < MT; ++m) {
        top[m] = -INFINITY;
        sum[m] = 0.0f;
#pragma unroll
        for (int s = 0; s < S; ++s) acc[m][s][0] = acc[m][s][1] = f32x4{0, 0, 0, 0};
    }
    auto at_step = [&](int n) { return split + n * p.splits; };
    load(split, lookup(split));
    keep(0);
    load(at_step(1), lookup(at_step(1)));
    __syncthreads();
    convert(split, 0);
    keep(1);
    load(at_step(2), lookup(at_step(2)));
    Ids ids = lookup(at_step(3));
    __syncthreads();
    for (int step = 0, buffer = 0; at_step(step) * kTile <= block_last; ++step, buffer ^= 1) {
        const int tile = at_step(step), first = tile * kTile;
        if (at_step(step + 1) * kTile <= block_last) {
            convert(at_step(step + 1), buffer ^ 1);
            keep(buffer);
            load(at_step(step + 3), ids);
            ids = lookup(at_step(step + 4));
        }
        if (first <= last) {
            f32x4 score[MT][4];
#pragma unroll
            for (int m = 0; m < MT; ++m)
#pragma unroll
                for (int a = 0; a < 4; ++a) score[m][a] = f32x4{0, 0, 0, 0};
#pragma unroll
            for (int s = 0; s < S; ++s)
#pragma unroll
                for (int a = 0; a < 4; ++a) {
                    const bf16x8 k = key_lds[buffer][a * S + s][lane];
#pragma unroll
                    for (int i = P - 1; i >= 0; --i)
#pragma unroll
                        for (int m = 0; m < MT; ++m) score[m][a] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(k, q[m][i][s], score[m][a], 0, 0, 0);
                }
            const bool masked = first + kTile - 1 > least;
            float now[MT];
            bool moved = false;
#pragma unroll
            for (int m = 0; m < MT; ++m) {
                if (masked) {
#pragma unroll
                    for (int i = 0; i < 16; ++i) score[m][i / 4][i % 4] = first + 16 * g + i > position[m] ? -INFINITY : score[m][i / 4][i % 4];
                }
                float most = -INFINITY;
#pragma unroll
                for (int i = 0; i < 16; ++i) most = fmaxf(most, score[m][i / 4][i % 4]);
                now[m] = fmaxf(top[m], max_over_groups(most));
                moved = moved || now[m] != top[m];
            }
            if (__ballot(moved) != 0) {
#pragma unroll
                for (int m = 0; m < MT; ++m) {
                    const float shrink = __builtin_amdgcn_exp2f(fmaf(top[m], scale, -finite_or_zero(now[m]) * scale));
                    top[m] = now[m];
                    sum[m] *= shrink;
#pragma unroll
                    for (int s = 0; s < S; ++s) {
                        acc[m][s][0] *= shrink;
                        acc[m][s][1] *= shrink;
                    }
                }
            }
            bf16x8 weight[MT][P][2];
#pragma unroll
            for (int m = 0; m < MT; ++m) {
                const float base = finite_or_zero(top[m]) * scale;
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    float w[8];
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        w[i] = __builtin_amdgcn_exp2f(fmaf(score[m][2 * h + i / 4][i % 4], scale, -base));
                        sum[m] += w[i];
                    }
                    if constexpr (F32) {
                        bf16x8 plane[3];
                        planes_of<false>(w, plane);
#pragma unroll
                        for (int i = 0; i < 3; ++i) weight[m][i][h] = plane[i];
                    } else {
#pragma unroll
                        for (int i = 0; i < 8; ++i) weight[m][0][h][i] = static_cast<__bf16>(w[i]);
                    }
                }
            }
#pragma unroll
            for (int s = 0; s < S; ++s)
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const bf16x8 even = value_lds[buffer][2 * s + h][0][lane], odd = value_lds[buffer][2 * s + h][1][lane];
#pragma unroll
                    for (int i = P - 1; i >= 0; --i)
#pragma unroll
                        for (int m = 0; m < MT; ++m) {
                            acc[m][s][0] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(even, weight[m][i][h], acc[m][s][0], 0, 0, 0);
                            acc[m][s][1] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(odd, weight[m][i][h], acc[m][s][1], 0, 0, 0);
                        }
                }
            if (nan_tile[buffer] == tile + 1) {  // rare: the scales again, from memory
                uint32_t page, token;
                split_run(c, 4 * tile + g, page, token);
                const int32_t page_id = page < static_cast<uint32_t>(c.width) ? table[page] : -1;
                const uint8_t* const scales = records + (page_id < 0 || page_id >= c.pages ? 0 : page_id) * page_stride + 2 * half;
#pragma unroll
                for (int m = 0; m < MT; ++m)
#pragma unroll
                    for (int s = 0; s < S; ++s) {
                        int poison = 0;
                        for (int i = 0; i < 16; ++i)
                            if (first + 16 * g + i <= position[m] && scales[(S + s) * c.page_size + static_cast<int>(token) + i] > kMostScale) poison = 1;
                        poison |= __shfl_xor(poison, 16, kWave);
                        poison |= __shfl_xor(poison, 32, kWave);
                        if (poison) acc[m][s][0] = acc[m][s][1] = f32x4{NAN, NAN, NAN, NAN};
                    }
            }
        }
        __syncthreads();
    }

#pragma unroll
    for (int m = 0; m < MT; ++m) {
        sum[m] = sum_over_groups(sum[m]);
        const int row = row0 + 16 * m + l;
        if (row >= p.rows) continue;
        const int token = row / p.group, at = c.positions[static_cast<int64_t>(b) * c.length + token];
        const int64_t part = ((static_cast<int64_t>(b) * c.kv_heads + head) * p.rows + row) * p.splits + split;
        const int64_t to = ((static_cast<int64_t>(b) * c.length + token) * p.heads + head * p.group + row - token * p.group) * D;
        const float by = 1.0f / sum[m];
#pragma unroll
        for (int s = 0; s < S; ++s) {
            float v[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = acc[m][s][i % 2][i / 2];
            if (p.splits > 1) {
                put8<true>(p.part, part * D + 32 * s + 8 * g, v);
            } else {
#pragma unroll
                for (int i = 0; i < 8; ++i) v[i] = at < 0 ? 0.0f : (at >= capacity ? NAN : v[i] * by);
                put8<F32>(p.out, to + 32 * s + 8 * g, v);
            }
        }
        if (p.splits > 1 && g == 0) {
            float* const st = p.part + p.part_rows * D + 2 * part;
            st[0] = top[m] * scale;
            st[1] = sum[m];
        }
    }
}

// The splits of a row joined: D / 8 lanes across it, and TEAMS such groups that take a split each at a time (more than 16
// splits: one group a row walked 64 of them for 20 us; up to 16 of them it saves 0.3 to 1.5 us).
template <int D, bool F32, int TEAMS>
__global__ __launch_bounds__(256) void kv4_join_kernel(AttentionArgs p) {
    constexpr int kLanes = D / 8, kRows = 256 / kLanes / TEAMS;
    __shared__ float joined[TEAMS > 1 ? kRows * TEAMS : 1][D + 4];  // a team's part, then its maximum and sum
    const int lane = threadIdx.x % kLanes, team = threadIdx.x / kLanes % TEAMS, in_block = threadIdx.x / kLanes / TEAMS;
    const Cache& c = p.c;
    const uint32_t all = static_cast<uint32_t>(c.batch * c.kv_heads) * static_cast<uint32_t>(p.rows);  // below 2^31
    const uint32_t idx = min(blockIdx.x * kRows + in_block, all - 1);
    const int bh = static_cast<int>(idx / static_cast<uint32_t>(p.rows)), row = static_cast<int>(idx - static_cast<uint32_t>(bh * p.rows));
    const int b = bh / c.kv_heads, head = bh - b * c.kv_heads, token = row / p.group;
    const int at = c.positions[static_cast<int64_t>(b) * c.length + token];
    const int64_t first = static_cast<int64_t>(idx) * p.splits;
    const float* const st = p.part + p.part_rows * D + 2 * first;
    float top = -INFINITY, sum = 0.0f, v[8] = {0, 0, 0, 0, 0, 0, 0, 0};
    auto add = [&](float its, float its_sum, const float (&part)[8]) {
        const float before = top;
        top = fmaxf(top, its);
        const float base = finite_or_zero(top), shrink = __builtin_amdgcn_exp2f(before - base), by = __builtin_amdgcn_exp2f(its - base);
        sum = fmaf(its_sum, by, sum * shrink);
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = fmaf(part[j], by, v[j] * shrink);
    };
#pragma unroll 4
    for (int i = team; i < p.splits; i += TEAMS) {
        float part[8];
        load8<true>(p.part, (first + i) * D + 8 * lane, part);
        add(st[2 * i], st[2 * i + 1], part);
    }
    if constexpr (TEAMS > 1) {
        float* const mine = joined[in_block * TEAMS + team];
#pragma unroll
        for (int j = 0; j < 8; ++j) mine[8 * lane + j] = v[j];
        if (lane == 0) {
            mine[D] = top;
            mine[D + 1] = sum;
        }
        __syncthreads();
        if (team != 0) return;
        for (int i = 1; i < TEAMS; ++i) {
            const float* const other = joined[in_block * TEAMS + i];
            float part[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) part[j] = other[8 * lane + j];
            add(other[D], other[D + 1], part);
        }
    }
    if (blockIdx.x * kRows + in_block >= all) return;
    const float by = 1.0f / sum;
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = at < 0 ? 0.0f : (at >= c.width * c.page_size ? NAN : v[j] * by);
    put8<F32>(p.out, ((static_cast<int64_t>(b) * c.length + token) * p.heads + head * p.group + row - token * p.group) * D + 8 * lane, v);
}

// ------------------------------------------------------------- host

bool dim_ok(int64_t dim) { return dim == 32 || dim == 64 || dim == 128 || dim == 256; }

template <typename Body>
void by_dim(int64_t dim, Body body) {
    if (dim == 32) body(std::integral_constant<int, 32>{});
    if (dim == 64) body(std::integral_constant<int, 64>{});
    if (dim == 128) body(std::integral_constant<int, 128>{});
    if (dim == 256) body(std::integral_constant<int, 256>{});
}

mlk_status cache_of(Cache& c, uint8_t* bytes, int64_t pages, int64_t page_size, int64_t kv_heads, int64_t dim, const int32_t* table,
                    int64_t width, const int32_t* positions, int64_t batch, int64_t length) {
    MLK_CHECK(batch >= 0 && length >= 0 && kv_heads > 0, "invalid cache geometry");
    MLK_CHECK(dim_ok(dim), "head_dim must be 32, 64, 128 or 256");
    MLK_CHECK(page_size > 0 && page_size % kRun == 0 && page_size <= 1024, "page_size must be a multiple of 16, at most 1024");
    MLK_CHECK(pages > 0 && pages < (int64_t{1} << 31), "the cache must have between 1 and 2^31 - 1 pages");
    MLK_CHECK(width > 0 && width <= (int64_t{1} << 28) / page_size, "page_table must hold between 1 and 2^28 / page_size pages a sequence");
    MLK_CHECK(kv_heads < (int64_t{1} << 20) && batch < (int64_t{1} << 31) && length < (int64_t{1} << 31) && batch * length < (int64_t{1} << 36),
              "too many heads, sequences or tokens");
    c = Cache{};
    c.bytes = bytes;
    c.record = page_size * (dim + dim / 16);
    c.pages = static_cast<int32_t>(pages);
    c.kv_heads = static_cast<int32_t>(kv_heads);
    c.page_size = static_cast<int32_t>(page_size);
    c.runs = static_cast<int32_t>(page_size / kRun);
    c.magic = static_cast<uint32_t>(((int64_t{1} << 31) + c.runs - 1) / c.runs);
    c.table = table;
    c.width = static_cast<int32_t>(width);
    c.positions = positions;
    c.batch = static_cast<int32_t>(batch);
    c.length = static_cast<int32_t>(length);
    if (batch == 0 || length == 0) return MLK_OK;
    MLK_CHECK(bytes && table && positions, "null tensor pointer");
    MLK_CHECK((reinterpret_cast<uintptr_t>(bytes) & 15) == 0, "the cache must be 16-byte aligned");
    return MLK_OK;
}

constexpr int64_t kThreads = int64_t{1} << 32;  // a launch's threads stay below

// Rows of all (sequence, key head) pairs below 2^31: every count of the plan then fits.
bool rows_fit(int64_t batch, int64_t length, int64_t heads, int64_t kv_heads) {
    if (batch <= 0 || length <= 0 || kv_heads <= 0) return true;  // nothing to do, or refused as geometry
    const int64_t most = int64_t{1} << 31;
    return batch < most && length < (most >> 1) && heads < (int64_t{1} << 20) && length * (heads / kv_heads) < (most >> 1) && batch * length < most &&
           batch * length * heads < most;
}

struct Plan {
    int64_t splits, rows, part_rows;
    bool many;  // kv4_attention_rows_kernel
    size_t bytes;

    int64_t row_tiles(bool f32) const { return ceil_div(rows, many ? 16 * W * (f32 ? kRowTiles<true> : kRowTiles<false>) : 16); }
};
// Few blocks are split over the keys, as far as the chip takes them at once (256 blocks of eight waves, 512 with heads up to
// 64; a second round of them cost more than uneven shares: 131072 keys, 8 key heads 67 us with 512 blocks, 39 with 256), a
// tile a wave at least, in whole rounds of tiles (20 tiles in 3 blocks 9.8 us, in 2 11.0), and not for up to 16 tiles:
// joining the parts takes a launch of its own (32 tiles: 14.5 us in one block, 10.5 in four).
//
// The waves share the keys (kv4_attention_rows_kernel) from 2048 tiles of 256 rows by 64 keys on (us; heads of 128, 32 query
// heads on 8 key heads):
//
//   sequences x tokens over keys   tiles   shared bf16  fp32   each wave its own bf16  fp32
//   1 x 64 over 8192                1024       36                     28
//   8 x 64 over 4000 (12 on 4)      2016       44        73          47                 65
//   4 x 300 over 1000               2560       49        93          90                112
//   1 x 512 over 8192               8192      111       193         170                224
//   1 x 250 over 60000             30016      320                   490
//
// One round of its blocks: two took 20 us more for sequences of one length and 15 less for two of which one is half as
// long (2 x 512 over 8192).
Plan plan_of(int64_t batch, int64_t length, int64_t heads, int64_t kv_heads, int64_t dim, int64_t capacity) {
    Plan t{};
    t.rows = length * (heads / kv_heads);
    const int64_t tiles = ceil_div(capacity, kTile), shared_blocks = batch * kv_heads * ceil_div(t.rows, 16 * W * 2);
    t.many = dim == kSharedDim && t.rows >= 128 && shared_blocks * tiles >= 2048;
    if (t.many) {
        t.splits = std::max<int64_t>(1, std::min(256 / shared_blocks, tiles / 4));
    } else {
        const int64_t blocks = std::max<int64_t>(1, batch * kv_heads * ceil_div(t.rows, 16)), resident = dim <= 64 ? 512 : 256;
        const int64_t groups = ceil_div(tiles, W), most = std::max<int64_t>(1, std::min(resident / blocks, groups));
        t.splits = tiles <= 2 * W ? 1 : ceil_div(groups, ceil_div(groups, most));
    }
    t.part_rows = batch * kv_heads * t.rows * t.splits;
    t.bytes = t.splits > 1 ? static_cast<size_t>(t.part_rows) * (dim + 2) * sizeof(float) : 0;
    return t;
}

template <int D, bool F32>
void launch_attention(AttentionArgs p, const Plan& t, hipStream_t s) {
    p.row_tiles = static_cast<int32_t>(t.row_tiles(F32));
    const int64_t blocks = int64_t{p.c.batch} * p.c.kv_heads * p.row_tiles * t.splits;
    if (t.many) {
        if constexpr (D == kSharedDim) hipLaunchKernelGGL(kv4_attention_rows_kernel<F32>, dim3(static_cast<unsigned>(blocks)), dim3(W * 64), 0, s, p);
    } else {
        auto launch = [&](auto whole, auto few) {
            constexpr bool kWhole = decltype(whole)::value, kFew = decltype(few)::value;
            hipLaunchKernelGGL((kv4_attention_kernel<D, F32, kWhole, kFew>), dim3(static_cast<unsigned>(blocks)), dim3(W * 64), 0, s, p);
        };
        auto by_rows = [&](auto whole) { t.rows <= 4 ? launch(whole, std::true_type{}) : launch(whole, std::false_type{}); };
        if (D < 256 && p.c.runs % 4 == 0) {
            by_rows(std::bool_constant<D < 256>{});
        } else {
            by_rows(std::false_type{});
        }
    }
    if (t.splits == 1) return;
    const int64_t rows = t.part_rows / t.splits;
    constexpr int kAtOnce = 256 / (D / 8), kTeams = 8;
    if (t.splits > 16) {
        hipLaunchKernelGGL((kv4_join_kernel<D, F32, kTeams>), dim3(static_cast<unsigned>(ceil_div(rows, kAtOnce / kTeams))), dim3(256), 0, s, p);
    } else {
        hipLaunchKernelGGL((kv4_join_kernel<D, F32, 1>), dim3(static_cast<unsigned>(ceil_div(rows, kAtOnce))), dim3(256), 0, s, p);
    }
}

}  // namespace
}  // namespace mlk

using namespace mlk;

extern "C" mlk_status mlk_kv4_append(const void* k, const int64_t* k_strides, const void* v, const int64_t* v_strides, int32_t dtype,
                                     int64_t batch, int64_t length, int64_t kv_heads, int64_t head_dim, uint8_t* cache,
                                     int64_t pages, int64_t page_size, const int32_t* page_table, int64_t table_width,
                                     const int32_t* positions, mlk_stream_t stream) {
    MLK_CHECK(dtype == MLK_DTYPE_F32 || dtype == MLK_DTYPE_BF16, "dtype must be f32 or bf16");
    Cache c;
    const mlk_status status = cache_of(c, cache, pages, page_size, kv_heads, head_dim, page_table, table_width, positions, batch, length);
    if (status != MLK_OK || batch == 0 || length == 0) return status;
    MLK_CHECK(k && k_strides && v && v_strides, "null tensor pointer");
    const int64_t waves = ceil_div(batch * length, 16) * kv_heads * 2;
    MLK_CHECK(ceil_div(waves, 4) * 256 < kThreads, "too many tokens for one launch");
    const Rows3 kr{k, k_strides[0], k_strides[1], k_strides[2]}, vr{v, v_strides[0], v_strides[1], v_strides[2]};
    by_dim(head_dim, [&](auto dim) {
        constexpr int D = decltype(dim)::value;
        const auto kernel = dtype == MLK_DTYPE_F32 ? kv4_append_kernel<D, true> : kv4_append_kernel<D, false>;
        hipLaunchKernelGGL(kernel, dim3(static_cast<unsigned>(ceil_div(waves, 4))), dim3(256), 0,
                           reinterpret_cast<hipStream_t>(stream), c, kr, vr, static_cast<uint32_t>(waves));
    });
    return launch_status("kv4 append");
}

extern "C" mlk_status mlk_kv4_read(const uint8_t* cache, int64_t pages, int64_t page_size, const int32_t* page_table, int64_t table_width,
                                   const int32_t* positions, int64_t batch, int64_t length, int64_t kv_heads, int64_t head_dim,
                                   int32_t dtype, void* k, void* v, mlk_stream_t stream) {
    MLK_CHECK(dtype == MLK_DTYPE_F32 || dtype == MLK_DTYPE_BF16, "dtype must be f32 or bf16");
    Cache c;
    const mlk_status status = cache_of(c, const_cast<uint8_t*>(cache), pages, page_size, kv_heads, head_dim, page_table, table_width,
                                       positions, batch, length);
    if (status != MLK_OK || batch == 0 || length == 0) return status;
    MLK_CHECK(k && v, "null tensor pointer");
    MLK_CHECK((reinterpret_cast<uintptr_t>(k) & 15) == 0 && (reinterpret_cast<uintptr_t>(v) & 15) == 0, "k and v must be 16-byte aligned");
    const int64_t waves = ceil_div(batch * length, 16) * kv_heads * 2;
    MLK_CHECK(ceil_div(waves, 4) * 256 < kThreads, "too many tokens for one launch");
    by_dim(head_dim, [&](auto dim) {
        constexpr int D = decltype(dim)::value;
        const auto kernel = dtype == MLK_DTYPE_F32 ? kv4_read_kernel<D, true> : kv4_read_kernel<D, false>;
        hipLaunchKernelGGL(kernel, dim3(static_cast<unsigned>(ceil_div(waves, 4))), dim3(256), 0,
                           reinterpret_cast<hipStream_t>(stream), c, k, v, static_cast<uint32_t>(waves));
    });
    return launch_status("kv4 read");
}

extern "C" size_t mlk_kv4_attention_workspace_bytes(int64_t batch, int64_t length, int64_t heads, int64_t kv_heads, int64_t head_dim,
                                                    int64_t page_size, int64_t table_width) {
    if (batch <= 0 || length <= 0 || kv_heads <= 0 || heads <= 0 || heads % kv_heads != 0 || !dim_ok(head_dim) || page_size <= 0 ||
        page_size > 1024 || !rows_fit(batch, length, heads, kv_heads) || table_width <= 0 || table_width > (int64_t{1} << 28) / page_size)
        return 0;
    return plan_of(batch, length, heads, kv_heads, head_dim, page_size * table_width).bytes;
}

extern "C" mlk_status mlk_kv4_attention(const void* q, const int64_t* q_strides, int32_t dtype, int64_t batch, int64_t length,
                                        int64_t heads, int64_t kv_heads, int64_t head_dim, const uint8_t* cache, int64_t pages,
                                        int64_t page_size, const int32_t* page_table, int64_t table_width, const int32_t* positions,
                                        double scale, void* out, void* workspace, size_t workspace_bytes, mlk_stream_t stream) {
    MLK_CHECK(dtype == MLK_DTYPE_F32 || dtype == MLK_DTYPE_BF16, "dtype must be f32 or bf16");
    MLK_CHECK(kv_heads <= 0 || (heads > 0 && heads % kv_heads == 0), "heads must be a multiple of kv_heads");
    MLK_CHECK(rows_fit(batch, length, heads, kv_heads), "too many tokens for one launch");
    AttentionArgs p{};
    const mlk_status status = cache_of(p.c, const_cast<uint8_t*>(cache), pages, page_size, kv_heads, head_dim, page_table, table_width,
                                       positions, batch, length);
    if (status != MLK_OK) return status;
    if (batch == 0 || length == 0) return MLK_OK;
    MLK_CHECK(q && q_strides && out, "null tensor pointer");
    MLK_CHECK((reinterpret_cast<uintptr_t>(out) & 15) == 0, "out must be 16-byte aligned");
    const Plan t = plan_of(batch, length, heads, kv_heads, head_dim, page_size * table_width);
    MLK_CHECK(batch * kv_heads * t.row_tiles(dtype == MLK_DTYPE_F32) * t.splits * (64 * W) < kThreads, "too many tokens for one launch");
    MLK_CHECK(workspace_bytes >= t.bytes && (t.bytes == 0 || (workspace && (reinterpret_cast<uintptr_t>(workspace) & 15) == 0)),
              "workspace must be 16-byte aligned and hold mlk_kv4_attention_workspace_bytes");
    p.q = q;
    p.q_bs = q_strides[0];
    p.q_ts = q_strides[1];
    p.q_hs = q_strides[2];
    p.heads = static_cast<int32_t>(heads);
    p.group = static_cast<int32_t>(heads / kv_heads);
    p.rows = static_cast<int32_t>(t.rows);
    p.splits = static_cast<int32_t>(t.splits);
    p.scale_log2 = static_cast<float>(scale * 1.4426950408889634);
    p.out = out;
    p.part = static_cast<float*>(workspace);
    p.part_rows = t.part_rows;
    by_dim(head_dim, [&](auto dim) {
        constexpr int D = decltype(dim)::value;
        dtype == MLK_DTYPE_F32 ? launch_attention<D, true>(p, t, reinterpret_cast<hipStream_t>(stream))
                               : launch_attention<D, false>(p, t, reinterpret_cast<hipStream_t>(stream));
    });
    return launch_status("kv4 attention");
}
