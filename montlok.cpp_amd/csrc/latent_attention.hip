// Attention in the latents' space over a cache of token rows (latent c, shared rotated key part r):
//
//   s[key] = (q_latent . c[key] + q_rope . r[key]) * scale,   out = sum softmax(s)[key] c[key]
//
// One pass over a sequence's rows with a running maximum and sum; all heads of a token, and all tokens of a call, read the
// same rows: 16 heads make 56 operations a byte of eight-bit rows (bound by memory), 64 heads 224 (memory and products alike),
// a chunk's tokens any number (products).
#include <algorithm>
#include <cfloat>
#include <climits>
#include <cmath>
#include <type_traits>

#include "latent.h"

namespace mlk {
namespace {

// Read in place of rows that no page holds, or that no token of a block sees.
__device__ const uint8_t kZeroRow[2 * (512 + 64) + 16] __attribute__((aligned(16))) = {};

struct LatentAttentionArgs {
    const void *q, *qr;
    int64_t qs[3], rs[3];
    LatentCache c;
    const int32_t* positions;
    const int64_t* ancestors;  // or null
    void* out;
    float* partial;   // sums of the parts: of fp32 rows [sequence][row][split][R], else [share][2][row of a unit][R]
    float* stats;     // maxima and sums of the parts' weights, two in place of R
    int32_t* starts;  // tiles before each unit
    int32_t length, heads, rows, row_blocks, splits;
    int32_t units, shares;  // 0 shares: a unit a block
    int32_t wide;           // the cache is larger than an offset of 32 bits reaches
    float scale;      // times log2(e), not negative
    uint32_t negate;  // the sign bits of two bf16 where it was
};

constexpr int kTile = 64;   // tokens of a tile, for plans and fp32 queries
constexpr int kPPitch = 72;  // bf16 elements from one row of weights to the next in LDS: 36 dwords, eight rows on eight bank groups

__device__ __forceinline__ float max_over_groups(float v) {
    v = fmaxf(v, __shfl_xor(v, 16, kWave));
    return fmaxf(v, __shfl_xor(v, 32, kWave));
}
__device__ __forceinline__ float sum_over_groups(float v) {
    v += __shfl_xor(v, 16, kWave);
    return v + __shfl_xor(v, 32, kWave);
}
__device__ __forceinline__ float finite_or_zero(float m) { return m == -INFINITY ? 0.0f : m; }

__device__ __forceinline__ f32x4 mfma(const bf16x8& a, const bf16x8& b, const f32x4& c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }

typedef short i16x4 __attribute__((ext_vector_type(4)));
typedef int i32x2 __attribute__((ext_vector_type(2)));
typedef __attribute__((address_space(3))) const uint8_t LdsByte;

// Sixteen bytes a lane from memory to LDS at `to` + 16 * lane, without a register between them. The compiler does not count
// these loads (of its builtin it does, and waits for every read of LDS in turn): wait_for_rows() ends every one.
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"  // m0 as a clobber: nothing else here uses it
__device__ __forceinline__ void load_row_pieces(const uint8_t* from, uint32_t to) {
    asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, off" ::"v"(from), "s"(to) : "memory", "m0");
}
// The same from `from` + offset. Beside waves that keep the matrix cores busy the form above is issued once in 246 cycles, this
// one once in 71 as without them: a vector of 64-bit addresses waits for the matrix instructions' operands.
__device__ __forceinline__ void load_row_pieces(const uint8_t* from, uint32_t offset, uint32_t to) {
    asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, %1" ::"v"(offset), "s"(from), "s"(to) : "memory", "m0");
}
#pragma clang diagnostic pop
__device__ __forceinline__ void wait_for_rows() {
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_waitcnt(0x0F70);  // vmcnt 0, the other counters at their most
    asm volatile("" ::: "memory");
}

// What a token of a call sees: the places below `base`, and base + j where bit j is set; nothing from `end` on. The base is
// kNowhere where that is nothing, 0 past the table, where it is nothing either but the result NaN.
struct Sight {
    int base, end;
    uint64_t bits;
};
constexpr int kNowhere = -(1 << 30);
__device__ __forceinline__ Sight sight_of(const LatentAttentionArgs& p, int64_t sequence, int token) {
    const int64_t at = sequence * p.length + token;
    const int32_t position = p.positions[at];
    Sight s{position < 0 ? kNowhere : 0, 0, 0};
    if (position < 0 || position >= static_cast<int64_t>(p.c.width) * p.c.page_size) return s;
    s.end = s.base = position + 1;
    if (p.ancestors == nullptr) return s;
    s.base = position - token;
    s.bits = static_cast<uint64_t>(p.ancestors[at]);
    if (p.length < 64) s.bits &= (uint64_t{1} << p.length) - 1;
    s.end = max(s.bits == 0 ? s.base : s.base + 64 - __builtin_clzll(s.bits), 0);
    if (s.end == 0) s.base = kNowhere;
    return s;
}

// What a row's sums are multiplied by. Where it sees tokens its sum is 1 at least, its largest weight; it is 0 where it sees
// nothing, which gives zeros, and where all its scores are -infinity or it is past the table, which gives NaN. A part's maximum
// tells the join which: -infinity for the first, kNoWeight for the others where no weight of theirs is in the part.
__device__ __forceinline__ float inverse_of(float sum, bool nothing) { return sum != 0.0f ? 1.0f / sum : nothing ? 0.0f : NAN; }
constexpr float kNoWeight = -FLT_MAX;

// fp32 queries: 16 rows (a row is a token and a query head) of one sequence over every `splits`-th part of its tokens. Queries
// and weights are three bf16 planes each, which hold every bit of them (from 2^-110 on), so that products with the cache's
// values are exact.
// Wave i scores tokens 16 i .. of a tile of 64, then takes R / 4 columns of all rows' sums. Every product has the rows as its
// columns (scores are tokens x rows, sums are columns x rows), so that a lane's numbers all belong to row lane & 15: its
// maximum, sum and rescaling are one number, its weights of four tokens and its sums of four columns lie side by side.
//
// Bound by latency where it is small (480 tokens of 8 heads, R = 64: 6.7 us and 3.8 for the join) and by the products of the
// planes, three of each, where it is not: 64 sequences of up to 4096 tokens, 64 heads, R = 512, take 257 us, 90 TFLOP/s.
template <int R, int P, bool E4M3>
__global__ __launch_bounds__(256) void latent_attention_f32_kernel(LatentAttentionArgs p) {
    constexpr int ROW = row_bytes<E4M3>(R, P), PIECES = ROW / 16, COLS = R / 4, CT = COLS / 16, kPlanes = 3;
    constexpr int KS = R / 32, RS = (P + 31) / 32;  // 32-deep steps over the latent and the key part
    __shared__ __attribute__((aligned(16))) uint8_t tiles[2][kTile * ROW];
    __shared__ __attribute__((aligned(16))) uint16_t weights[kPlanes][16 * kPPitch];
    __shared__ float maxima[4][16];
    __shared__ const uint8_t* row_at[kTile];
    __shared__ float missing[2][kTile];  // NaN where a token's page is missing, else 0
    __shared__ int tainted[2];           // some score of the tile is not finite
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64), lane = threadIdx.x & 63, g = lane >> 4, l = lane & 15;
    unsigned id = blockIdx.x;
    const int split = id % p.splits;
    id /= p.splits;
    const int row = static_cast<int>(id % p.row_blocks) * 16 + l, token_of_row = row / p.heads, head = row - token_of_row * p.heads;
    const int64_t b = id / p.row_blocks;
    const bool real = row < p.rows;
    Sight sight{0, 0, 0};
    if (real) sight = sight_of(p, b, token_of_row);
    int end = sight.end;
#pragma unroll
    for (int m = 1; m < 16; m *= 2) end = max(end, __shfl_xor(end, m, kWave));
    end = __builtin_amdgcn_readfirstlane(end);

    const int tile_count = (end + kTile - 1) / kTile, per_split = (tile_count + p.splits - 1) / p.splits;
    const int first = min(split * per_split, tile_count), last = min(first + per_split, tile_count);

    // The lane's queries: of each step the dimensions that its piece of a key row holds (codes come 16 to a piece, bf16 values 8).
    bf16x8 q[KS + RS][kPlanes];
    const int64_t ql = b * p.qs[0] + token_of_row * p.qs[1] + head * p.qs[2], qr = b * p.rs[0] + token_of_row * p.rs[1] + head * p.rs[2];
#pragma unroll
    for (int t = 0; t < KS + RS; ++t) {
        const int d = t >= KS ? 32 * (t - KS) + 8 * g : E4M3 ? 64 * (t / 2) + 16 * g + 8 * (t % 2) : 32 * t + 8 * g;
        const float* const from = static_cast<const float*>(t < KS ? p.q : p.qr) + (t < KS ? ql : qr) + d;
        float v[8] = {};
        if (real && (t < KS || d < P)) {
            const u32x4 lo = *reinterpret_cast<const u32x4_any*>(from), hi = *reinterpret_cast<const u32x4_any*>(from + 4);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                v[i] = __uint_as_float(lo[i]);
                v[4 + i] = __uint_as_float(hi[i]);
            }
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = p.negate == 0 ? v[i] : -v[i];
        planes_of<true>(v, q[t]);
    }

    // Row addresses of a tile: by the first wave, a token a lane. The page's number is looked at a tile after it was asked for.
    auto page_of = [&](int tile) {
        const uint32_t token = static_cast<uint32_t>(tile) * kTile + lane, page = token / static_cast<uint32_t>(p.c.page_size);
        return static_cast<int>(token) < end && page < static_cast<uint32_t>(p.c.width) ? p.c.table[b * p.c.width + page] : -1;
    };
    auto set_rows = [&](int tile, int page_id) {
        const uint32_t token = static_cast<uint32_t>(tile) * kTile + lane, in_page = token % static_cast<uint32_t>(p.c.page_size);
        const bool held = page_id >= 0 && page_id < p.c.pages;
        row_at[lane] = held ? p.c.bytes + (static_cast<int64_t>(page_id) * p.c.page_size + in_page) * ROW : kZeroRow;
        // Tokens that no row sees are no missing ones.
        missing[tile & 1][lane] = held || static_cast<int>(token) >= end ? 0.0f : NAN;
    };
    auto load_tile = [&](int tile) {
        const uint32_t to = static_cast<uint32_t>(reinterpret_cast<uintptr_t>((LdsByte*)tiles[tile & 1]));
#pragma unroll
        for (int i = 0; i < (PIECES + 3) / 4; ++i) {
            const int part = i * 4 + wave;  // 64 pieces
            if (part < PIECES) {
                const int piece = part * 64 + lane, from = piece / PIECES;
                load_row_pieces(row_at[from] + (piece - from * PIECES) * 16, __builtin_amdgcn_readfirstlane(to + part * 1024));
            }
        }
    };

    f32x4 acc[CT] = {};
    float top = -INFINITY, sum = 0.0f;
    if (first < last) {
        if (wave == 0) set_rows(first, page_of(first));
        if (threadIdx.x == 0) tainted[0] = tainted[1] = 0;
        __syncthreads();
        load_tile(first);
        wait_for_rows();
        __syncthreads();
        if (wave == 0 && first + 1 < last) set_rows(first + 1, page_of(first + 1));
    }
    for (int tile = first; tile < last; ++tile) {
        __syncthreads();  // the tile, and the next one's row addresses
        int next_page = 0;
        if (wave == 0 && tile + 2 < last) next_page = page_of(tile + 2);
        if (tile + 1 < last) load_tile(tile + 1);
        const uint8_t* const rows = tiles[tile & 1];

        // Scores of tokens 16 wave + 4 g + i with the lane's row.
        f32x4 s = {}, r = {};
        const uint8_t* const key = rows + (16 * wave + l) * ROW;
#pragma unroll
        for (int t = 0; t < KS; t += E4M3 ? 2 : 1) {
            const u32x4 v = *reinterpret_cast<const u32x4*>(key + (E4M3 ? 32 : 64) * t + 16 * g);
            if constexpr (E4M3) {
                const bf16x8 a = e4m3_octet(v[0], v[1], 1.0f), c = e4m3_octet(v[2], v[3], 1.0f);
#pragma unroll
                for (int i = kPlanes - 1; i >= 0; --i) {
                    s = mfma(a, q[t][i], s);
                    s = mfma(c, q[t + 1][i], s);
                }
            } else {
#pragma unroll
                for (int i = kPlanes - 1; i >= 0; --i) s = mfma(__builtin_bit_cast(bf16x8, v), q[t][i], s);
            }
        }
#pragma unroll
        for (int t = 0; t < RS; ++t) {
            const int d = 32 * t + 8 * g;
            // Where the key part is 16 wide the upper lanes' queries are zeros, and so are their keys.
            bf16x8 a = __builtin_bit_cast(bf16x8, u32x4{0, 0, 0, 0});
            if (P >= 32 || d < P) a = *reinterpret_cast<const bf16x8*>(key + (E4M3 ? R : 2 * R) + 2 * d);
#pragma unroll
            for (int i = kPlanes - 1; i >= 0; --i) r = mfma(a, q[KS + t][i], r);
        }
        float key_scale[4];
        bool odd = false;
        float most = -INFINITY;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int in_tile = 16 * wave + 4 * g + i, past = tile * kTile + in_tile - sight.base;
            key_scale[i] = E4M3 ? *reinterpret_cast<const float*>(rows + in_tile * ROW + R + 2 * P) : 1.0f;
            const float v = (E4M3 ? fmaf(s[i], key_scale[i], r[i]) : s[i] + r[i]) * p.scale + missing[tile & 1][in_tile];
            odd |= !(fabsf(v) < INFINITY);
            const bool seen = past < 0 || (past < 64 && (sight.bits >> (past & 63) & 1));
            s[i] = seen ? v : -INFINITY;
            most = fmaxf(most, s[i]);
        }
        most = max_over_groups(most);
        if (g == 0) maxima[wave][l] = most;
        if (odd) tainted[tile & 1] = 1;
        __syncthreads();  // the rows' maxima
        const bool clean = tainted[tile & 1] == 0;
        if (threadIdx.x == 0) tainted[~tile & 1] = 0;
        most = top;
#pragma unroll
        for (int i = 0; i < 4; ++i) most = fmaxf(most, maxima[i][l]);
        const float under = finite_or_zero(most), by = __builtin_amdgcn_exp2f(top - under);
        top = most;
        float w[4], total = 0.0f;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float e = __builtin_amdgcn_exp2f(s[i] - under);
            total += e;
            w[i] = E4M3 ? (s[i] == -INFINITY ? 0.0f : e * key_scale[i]) : e;
        }
        sum = fmaf(sum, by, total);
        Parts3 x[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) x[i] = parts_of<true>(w[i]);
        const int to = l * kPPitch + 16 * wave + 4 * g;
        *reinterpret_cast<u32x2*>(&weights[0][to]) = u32x2{pack_upper(x[0].a, x[1].a), pack_upper(x[2].a, x[3].a)};
        *reinterpret_cast<u32x2*>(&weights[1][to]) = u32x2{pack_upper(x[0].b, x[1].b), pack_upper(x[2].b, x[3].b)};
        *reinterpret_cast<u32x2*>(&weights[2][to]) = u32x2{pack_upper(x[0].c, x[1].c), pack_upper(x[2].c, x[3].c)};
#pragma unroll
        for (int c = 0; c < CT; ++c) acc[c] *= by;
        if (!clean) {
            // A latent that is no number makes its scores none, and the weight of every row that sees it; where a row does not,
            // its weight 0 has to meet a number. Seldom: rows of a cache hold numbers, or codes 0 under a scale of NaN.
            uint8_t* const mine = tiles[tile & 1];
            for (int i = threadIdx.x; i < kTile * R / 4; i += 256) {
                const int token = i / (R / 4), d = i % (R / 4) * 4;
                if constexpr (E4M3) {
                    uint32_t* const at4 = reinterpret_cast<uint32_t*>(mine + token * ROW + d);
                    uint32_t v = *at4;
#pragma unroll
                    for (int j = 0; j < 4; ++j)
                        if ((v >> (8 * j) & 127) == 127) v &= ~(255u << (8 * j));
                    *at4 = v;
                } else {
                    uint32_t* const at4 = reinterpret_cast<uint32_t*>(mine + token * ROW + 2 * d);
#pragma unroll
                    for (int j = 0; j < 2; ++j) {
                        uint32_t v = at4[j];
                        if ((v & 0x7F80u) == 0x7F80u) v &= 0xFFFF0000u;
                        if ((v & 0x7F800000u) == 0x7F800000u) v &= 0xFFFFu;
                        at4[j] = v;
                    }
                }
            }
        }
        __syncthreads();  // the weights
#pragma unroll
        for (int t = 0; t < kTile / 32; ++t) {
            bf16x8 w8[kPlanes];
#pragma unroll
            for (int i = 0; i < kPlanes; ++i) w8[i] = *reinterpret_cast<const bf16x8*>(&weights[i][l * kPPitch + 32 * t + 8 * g]);
#pragma unroll
            for (int c = 0; c < CT; ++c) {
                // Eight tokens of a column a lane: the rows' bytes turned as they are read.
                const int column = wave * COLS + 16 * c;
                bf16x8 v;
                if constexpr (E4M3) {
                    const i32x2 y = __builtin_amdgcn_ds_read_tr8_b64_v2i32(
                        (__attribute__((address_space(3))) i32x2*)(rows + (32 * t + 8 * g + l / 2) * ROW + column + 8 * (l & 1)));
                    v = e4m3_octet(y[0], y[1], 1.0f);
                } else {
                    i16x4 y[2];
#pragma unroll
                    for (int h = 0; h < 2; ++h)
                        y[h] = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                            (__attribute__((address_space(3))) i16x4*)(rows + (32 * t + 8 * g + 4 * h + l / 4) * ROW + 2 * column + 8 * (l & 3)));
                    v = __builtin_bit_cast(bf16x8, __builtin_shufflevector(y[0], y[1], 0, 1, 2, 3, 4, 5, 6, 7));
                }
#pragma unroll
                for (int i = kPlanes - 1; i >= 0; --i) acc[c] = mfma(v, w8[i], acc[c]);
            }
        }
        wait_for_rows();  // of the next tile
        if (wave == 0 && tile + 2 < last) set_rows(tile + 2, next_page);
    }

    // A row's sum lies with the lanes and waves that scored its tokens.
    __syncthreads();
    sum = sum_over_groups(sum);
    if (g == 0) maxima[wave][l] = sum;
    __syncthreads();
    if (!real) return;
    sum = maxima[0][l] + maxima[1][l] + maxima[2][l] + maxima[3][l];
    const int64_t at_row = b * p.rows + row;
    // Asked for again where it matters: held through the loop over tiles it costs more (64 x 4096 tokens 259 us for 257).
    const bool nothing = top == -INFINITY && sight_of(p, b, row / p.heads).base == kNowhere;
    if (p.splits == 1) {
        const float inverse = inverse_of(sum, nothing);
#pragma unroll
        for (int c = 0; c < CT; ++c) *reinterpret_cast<f32x4*>(static_cast<float*>(p.out) + at_row * R + wave * COLS + 16 * c + 4 * g) = acc[c] * inverse;
    } else {
        const int64_t part = at_row * p.splits + split;
        if (first < last) {
#pragma unroll
            for (int c = 0; c < CT; ++c) *reinterpret_cast<f32x4*>(p.partial + part * R + wave * COLS + 16 * c + 4 * g) = acc[c];
        }
        if (wave == 0 && g == 0) {
            p.stats[part * 2] = top == -INFINITY && !nothing ? kNoWeight : top;
            p.stats[part * 2 + 1] = sum;
        }
    }
}

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
__device__ __forceinline__ f32x16 mfma(const bf16x8& a, const bf16x8& b, const f32x16& c) { return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0); }

// The maximum, or the sum, of a row: its scores lie with the lanes l and l + 32.
__device__ __forceinline__ float max_over_halves(float v) {
    const auto x = __builtin_amdgcn_permlane32_swap(__float_as_int(v), __float_as_int(v), false, false);
    return fmaxf(__int_as_float(x[0]), __int_as_float(x[1]));
}
__device__ __forceinline__ float sum_over_halves(float v) {
    const auto x = __builtin_amdgcn_permlane32_swap(__float_as_int(v), __float_as_int(v), false, false);
    return __int_as_float(x[0]) + __int_as_float(x[1]);
}

// At most N of the loads that this wave asked for are still on their way.
template <int N>
__device__ __forceinline__ void wait_for_rows_but() {
    static_assert(N >= 0 && N < 64, "the counter's range");
    __builtin_amdgcn_s_waitcnt((N & 15) | 0x0F70 | (N >> 4) << 14);
    asm volatile("" ::: "memory");
}

// A row's sums are rescaled when its maximum has grown by more than this (log2): weights are then at most 2^16, which
// changes no rounding, and after a row's first tokens next to no tile rescales.
constexpr float kSlack = 16.0f;

constexpr int kMaxUnits = 1024;  // that blocks share out among them
constexpr int kLeastShare = 2;   // tiles of a block, so that a block is worth its beginning
constexpr int kIds = 512;  // page numbers that are looked up at a time

// Waves of two kinds, RW groups of 32 rows: a scorer takes the rows' scores of 32 tokens of a tile (KW of them a group) and
// turns them into weights, a summer adds all tokens' latents to a part of the columns, and sees to the loads. Scorers
// hold the queries, summers the sums. With 64 rows what either holds leaves room for a wave of the other kind on its SIMD, and
// the one's exponents and conversions run beside the other's products (both in one wave, which then has a SIMD to itself: 6500
// cycles a tile of 64 tokens and 64 rows, of which the matrix cores are busy for 2200). Up to 32 rows are half of that, two
// scorers and two summers with a SIMD each; LDS holds one such block, or two where a tile is small.
//
// A tile is scored while the one before it is summed, with one barrier between.
//
// Measured with R = 512, P = 64 in eight bits, the kernel alone: 24 sequences of up to 8000 tokens, 16 heads, 32.0 us; one of
// 131072 tokens, 32 heads, 28.2 us (84 MB); 64 of up to 16384, 64 heads, 126 us (435 MB, 3.5 TB/s, 735 TFLOP/s); two chunks of
// 256 tokens of 24 heads over up to 8000 173 us (950 TFLOP/s). A launch's first 8 us (positions, page numbers, row addresses, a
// tile, each after the other) and its last 2 are no work on tiles; a tile of 64 rows and 64 tokens then takes 2.0 us where its
// products alone take 1.1: LDS reads and conversions of the operands share the SIMD with them (a product of 32 cycles takes 47
// beside its operand's read, 50 with its conversion too), and the clock is 1.8 to 2.1 GHz under them. That form takes all 256
// registers of a lane, and one more in scratch memory (its wide one four).
template <int R, int P, bool E4M3, int RW>
struct Shape {
    static constexpr int ROW = row_bytes<E4M3>(R, P), KW = 64 * ROW * 3 <= 140 * 1024 ? 2 : 1, KEYS = 32 * KW, BYTES = KEYS * ROW;
    static constexpr int STAGES = BYTES * 4 <= 76 * 1024 ? 4 : 3;
    static constexpr int SCORERS = RW * KW, SUMMERS = RW * 2, WAVES = SCORERS + SUMMERS;
    // A summer takes all rows of a quarter of the columns where it can: it then turns and converts half as many latents as for
    // one group's rows of half of the columns, with as many sums.
    static constexpr int GROUPS = RW == 2 && R % 128 == 0 ? 2 : 1, COLUMNS = R / (2 * GROUPS);
    static constexpr int LOADS = BYTES / 1024 + (BYTES % 1024 != 0);  // of 64 lanes, 16 bytes each
};

template <int R, int P, bool E4M3, int RW, bool WIDE>
__global__ __launch_bounds__((Shape<R, P, E4M3, RW>::WAVES * 64), RW) void latent_attention_rows_kernel(LatentAttentionArgs p) {
    using S = Shape<R, P, E4M3, RW>;
    constexpr int ROW = S::ROW, KW = S::KW, KEYS = S::KEYS, STAGES = S::STAGES, SUMMERS = S::SUMMERS, PIECES = ROW / 16;
    constexpr int KS = R / 16, RS = P / 16, RG = S::GROUPS, CT = S::COLUMNS / 32;  // 16-deep steps over the latent and the key part, 32-wide tiles of columns
    // Tiles are asked for AHEAD iterations before they are scored. Where their pieces lie is read at the end of the iteration
    // before that, from addresses set in the one before, from page numbers looked up one before that: each is there for all
    // summers after a barrier.
    constexpr int AHEAD = STAGES - 2, SLOTS = AHEAD == 1 ? 4 : 8;
    __shared__ __attribute__((aligned(16))) uint8_t tiles[STAGES][S::BYTES];
    __shared__ bf16x8 shared_weights[2][RW][KW][2][64];
    __shared__ uint64_t row_at[SLOTS][KEYS];      // offsets of a tile's rows in the cache, or addresses where these are wide
    __shared__ uint32_t missing[SLOTS][KEYS];     // all ones where a token's page is missing: its row becomes NaN
    __shared__ __attribute__((aligned(16))) float scales[S::SCORERS][32];
    __shared__ float tops[RW][KW][32], factors[RW][32];
    __shared__ int32_t ids[2][kIds];
    __shared__ int ends[RW];
    __shared__ int starts[kMaxUnits + 1];
    __shared__ int grown[2], odd[2];  // 1 + the tile where a maximum has outgrown its row's, or a score is no number
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
    const bool scorer = wave < S::SCORERS;
    const int rw = scorer ? wave / KW : (wave - S::SCORERS) / 2, part = scorer ? wave % KW : RG == 1 ? (wave - S::SCORERS) % 2 : wave - S::SCORERS;

    // The block's share: of the tiles of all units (RW * 32 rows of a sequence), laid end to end, as many as any other block's;
    // or one unit.
    int unit = blockIdx.x, from_tile = 0, until = INT_MAX, share = 0;
    if (p.shares != 0) {
        for (int u = threadIdx.x; u < p.units; u += S::WAVES * 64) starts[u + 1] = 1;  // a unit that sees nothing has outputs all the same
        __syncthreads();
        for (int i = threadIdx.x; i < p.units / p.row_blocks * p.length; i += S::WAVES * 64) {
            const int sequence = i / p.length, token = i - sequence * p.length, row0 = token * p.heads, end = sight_of(p, sequence, token).end;
            for (int u = row0 / (RW * 32); u <= (row0 + p.heads - 1) / (RW * 32); ++u) atomicMax(&starts[sequence * p.row_blocks + u + 1], end);
        }
        __syncthreads();
        if (wave == 0) {  // sums of everything before: a run of units a lane, then the lanes
            const int lane = threadIdx.x;
            const int run = (p.units + 63) / 64, u0 = min(lane * run, p.units), u1 = min(u0 + run, p.units);
            int sum = 0;
            for (int u = u0; u < u1; ++u) sum += starts[u + 1] = (starts[u + 1] + KEYS - 1) / KEYS;
            int before = sum;
#pragma unroll
            for (int m = 1; m < 64; m *= 2) {
                const int other = __shfl_up(before, m, kWave);
                before += lane >= m ? other : 0;
            }
            before -= sum;
            for (int u = u0; u < u1; ++u) starts[u + 1] = before += starts[u + 1];
            if (lane == 0) starts[0] = 0;
        }
        __syncthreads();
        const int total = starts[p.units], each = max((total + p.shares - 1) / p.shares, kLeastShare);
        // Neighbouring shares on one XCD, whose cache then holds one sequence's rows for many units.
        share = blockIdx.x % 8 * (p.shares / 8) + blockIdx.x / 8;
        const int share_first = share * each;
        until = min(share_first + each, total);
        if (blockIdx.x == 0) {  // for the join
            for (int u = threadIdx.x; u <= p.units; u += S::WAVES * 64) p.starts[u] = starts[u];
        }
        if (share_first >= until) return;
        int low = 0, high = p.units - 1;  // the last unit that begins at or before the share
        while (low < high) {
            const int middle = (low + high + 1) / 2;
            if (starts[middle] <= share_first) low = middle;
            else high = middle - 1;
        }
        unit = __builtin_amdgcn_readfirstlane(low);
        from_tile = __builtin_amdgcn_readfirstlane(share_first - starts[unit]);
        until = __builtin_amdgcn_readfirstlane(until);
    }

    for (int part_of_share = 0;; ++part_of_share) {
    // Formed anew for every part: what follows from the lane alone is otherwise kept through all of them, in registers that the
    // loop over tiles needs.
    int lane = threadIdx.x & 63;
    asm volatile("" : "+v"(lane));
    const int h = lane >> 5, l = lane & 31;
    const int64_t b = unit / p.row_blocks;
    const int row0 = static_cast<int>(unit - b * p.row_blocks) * (RW * 32), row = row0 + 32 * rw + l;
    const bool real = row < p.rows;
    const int token_of_row = row / p.heads, head = row - token_of_row * p.heads;
    // Page numbers for the summers, looked up kIds at a time.
    const int own = wave - S::SCORERS;
    const uint32_t page_size = static_cast<uint32_t>(p.c.page_size);
    int held_page = 0, held_end = 0, holds = 0;  // ids[holds] begins with page held_page and serves tiles before held_end
    auto hold = [&](int tile) {
        constexpr int EACH = kIds / (SUMMERS * 64);
        static_assert(kIds % (SUMMERS * 64) == 0, "as many for every lane");
        const int page0 = static_cast<int>(static_cast<uint32_t>(tile) * KEYS / page_size);
        held_end = static_cast<int>((static_cast<int64_t>(page0) + kIds) * page_size / KEYS);
        holds ^= 1;
        held_page = page0;
        int32_t id[EACH];
#pragma unroll
        for (int i = 0; i < EACH; ++i) {
            const int page = page0 + (i * SUMMERS + own) * 64 + lane;
            id[i] = -1;
            if (page < p.c.width) id[i] = p.c.table[b * p.c.width + page];
        }
#pragma unroll
        for (int i = 0; i < EACH; ++i) ids[holds][(i * SUMMERS + own) * 64 + lane] = id[i];
    };
    if (!scorer) hold(from_tile);
    Sight sight{0, 0, 0};
    if (real) sight = sight_of(p, b, token_of_row);
    const int base = sight.base;
    const uint64_t bits = sight.bits;
    int all = sight.end, every = real ? base : INT_MAX;  // where the tokens that some row sees end, and those that every row of the wave sees
#pragma unroll
    for (int m = 1; m < 32; m *= 2) {
        all = max(all, __shfl_xor(all, m, kWave));
        every = min(every, __shfl_xor(every, m, kWave));
    }
    const int plain = __builtin_amdgcn_readfirstlane(every);
    if (!scorer) ends[rw] = all;
    if (threadIdx.x < 2) grown[threadIdx.x] = odd[threadIdx.x] = 0;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < RW; ++i) all = max(all, ends[i]);
    all = __builtin_amdgcn_readfirstlane(all);

    const int tile_count = (all + KEYS - 1) / KEYS;
    const int unit_start = p.shares == 0 ? 0 : starts[unit], unit_end = p.shares == 0 ? INT_MAX : starts[unit + 1];
    const int first = min(from_tile, tile_count), last = p.shares == 0 ? tile_count : min(until - unit_start, tile_count);
    const bool whole = p.shares == 0 || (from_tile == 0 && until >= unit_end);
    // A share has at most two parts of units, its first and its last.
    const int64_t place = (static_cast<int64_t>(share) * 2 + (part_of_share != 0)) * (RW * 32) + 32 * rw + l;

    if (scorer) {
        float top = -INFINITY, sum = 0.0f;
        if (first < last) {
            bf16x8 q[KS + RS];
            {
                // A lane without a row takes the first row's: what it makes of it goes nowhere.
                const int64_t ql = b * p.qs[0] + (real ? token_of_row * p.qs[1] + head * p.qs[2] : 0);
                const int64_t qr = b * p.rs[0] + (real ? token_of_row * p.rs[1] + head * p.rs[2] : 0);
#pragma unroll
                for (int t = 0; t < KS + RS; ++t) {
                    // The dimensions that the lane's piece of a row holds: codes come 16 to a piece, bf16 values 8.
                    const int d = t >= KS ? 16 * (t - KS) + 8 * h : E4M3 ? 32 * (t / 2) + 16 * h + 8 * (t % 2) : 16 * t + 8 * h;
                    u32x4 v = *reinterpret_cast<const u32x4_any*>(static_cast<const uint16_t*>(t < KS ? p.q : p.qr) + (t < KS ? ql : qr) + d);
#pragma unroll
                    for (int i = 0; i < 4; ++i) v[i] ^= p.negate;  // a negative scale is the queries'
                    q[t] = __builtin_bit_cast(bf16x8, v);
                }
            }
#pragma unroll
            for (int i = 0; i < 2; ++i) __syncthreads();  // row addresses, the first tile
            int stage = 0;
            for (int tile = first; tile < last; ++tile) {
                const uint8_t* const rows = tiles[stage];
                stage = stage == STAGES - 1 ? 0 : stage + 1;
                // Scores of the wave's tokens with the lane's row: register i holds token 8 (i / 4) + 4 h + i % 4. Pieces of the
                // key row are read six ahead of their use, and turned into an operand beside the product before theirs; nothing
                // moves over the bars (the scheduler on its own reads each piece right before it is used).
                f32x16 s = {};
                const uint8_t* const key = rows + (32 * part + l) * ROW;
                constexpr int PARTS = E4M3 ? KS / 2 : KS, ALL = PARTS + RS, RING = ALL < 6 ? ALL : 6;
                auto piece = [&](int t) {
                    return *reinterpret_cast<const u32x4*>(key + (t < PARTS ? 32 * t : (E4M3 ? R : 2 * R) + 32 * (t - PARTS)) + 16 * h);
                };
                float scale = 1.0f;
                if constexpr (E4M3) scale = *reinterpret_cast<const float*>(key + R + 2 * P);
                const uint32_t lost = missing[tile % SLOTS][32 * part + l];
                u32x4 ring[RING];
#pragma unroll
                for (int t = 0; t < RING; ++t) ring[t] = piece(t);
                if constexpr (E4M3) scales[wave][l] = scale;
                ring[0][0] |= lost;
                __builtin_amdgcn_sched_barrier(0);
                auto operand = [&](int k) {  // of product k; its piece makes room for a later one
                    const int t = !E4M3 ? k : k < KS ? k / 2 : k - KS + PARTS;
                    const u32x4 x = ring[t % RING];
                    const bool codes = E4M3 && k < KS;
                    if (t + RING < ALL && (!codes || k % 2 == 1)) ring[t % RING] = piece(t + RING);
                    return codes ? e4m3_octet(x[k % 2 * 2], x[k % 2 * 2 + 1], scale) : __builtin_bit_cast(bf16x8, x);
                };
                bf16x8 next = operand(0);
                f32x4 key_scale[4];
#pragma unroll
                for (int k = 0; k < KS + RS; ++k) {
                    const bf16x8 now = next;
                    if (k + 1 < KS + RS) next = operand(k + 1);
                    s = mfma(now, q[k], s);
                    if constexpr (E4M3) {
                        if (k >= KS + RS - 4) key_scale[k - (KS + RS - 4)] = *reinterpret_cast<const f32x4*>(&scales[wave][8 * (k - (KS + RS - 4)) + 4 * h]);
                    }
                    __builtin_amdgcn_sched_barrier(0);
                }
                const int first_token = tile * KEYS + 32 * part;
                const bool masked = first_token + 32 > plain;
                if (masked) {
                    float none = 0.0f;
#pragma unroll
                    for (int i = 0; i < 16; ++i) {
                        none = fmaf(s[i], 0.0f, none);  // NaN once a score is an infinity or none
                        const int past = first_token + 8 * (i / 4) + 4 * h + i % 4 - base;
                        const bool seen = (past < 0) | ((past < 64) & static_cast<bool>(bits >> (past & 63) & 1));
                        s[i] = seen ? s[i] : -INFINITY;
                        // A scale of NaN is no matter to a row that does not see its token.
                        if constexpr (E4M3) key_scale[i / 4][i % 4] = seen ? key_scale[i / 4][i % 4] : 0.0f;
                    }
                    if (__any(none != none)) odd[tile & 1] = tile + 1;
                }
                float most = s[0];
#pragma unroll
                for (int i = 1; i < 16; ++i) most = fmaxf(most, s[i]);
                most = max_over_halves(most);
                most = most == -INFINITY ? most : most * p.scale;  // a scale of 0 is one too

                float total;
                auto weigh = [&] {
                    const float under = finite_or_zero(top);
                    total = 0.0f;
                    float e[16];
#pragma unroll
                    for (int i = 0; i < 16; ++i) e[i] = __builtin_amdgcn_exp2f(fmaf(s[i], p.scale, -under));
                    if (masked && p.scale == 0.0f) {  // the infinity of an unseen token times 0
#pragma unroll
                        for (int i = 0; i < 16; ++i) e[i] = s[i] == -INFINITY ? 0.0f : e[i];
                    }
                    u32x4 packed[2];
#pragma unroll
                    for (int i = 0; i < 16; i += 2) {
                        total += e[i] + e[i + 1];
                        if constexpr (E4M3) {
                            e[i] *= key_scale[i / 4][i % 4];
                            e[i + 1] *= key_scale[i / 4][i % 4 + 1];
                        }
                        // Rounded to bf16 for the product with the latents: 2^-8 of a weight at most, without a bias; the sum keeps them whole.
                        packed[i / 8][i / 2 % 4] = __builtin_bit_cast(uint32_t, bf16x2{static_cast<__bf16>(e[i]), static_cast<__bf16>(e[i + 1])});
                    }
                    shared_weights[tile & 1][rw][part][0][lane] = __builtin_bit_cast(bf16x8, packed[0]);
                    shared_weights[tile & 1][rw][part][1][lane] = __builtin_bit_cast(bf16x8, packed[1]);
                };
                // Weights under the maximum so far, which all waves of the rows know. Where it is outgrown they learn the others'
                // and weigh again, and the summers rescale.
                weigh();
                tops[rw][part][l] = most;
                if (__any(most > top + kSlack)) grown[tile & 1] = tile + 1;
                __syncthreads();
                if (__builtin_expect(grown[tile & 1] == tile + 1, 0)) {
                    float now = top;
#pragma unroll
                    for (int i = 0; i < KW; ++i) now = fmaxf(now, tops[rw][i][l]);
                    const float by = __builtin_amdgcn_exp2f(top - finite_or_zero(now));
                    if (part == 0) factors[rw][l] = by;
                    top = now;
                    sum *= by;
                    weigh();
                    __syncthreads();
                }
                sum += total;
            }
        }
        sum = sum_over_halves(sum);
        const bool weightless = top == -INFINITY && base != kNowhere;
        tops[rw][part][l] = whole && weightless ? NAN : sum;
        __syncthreads();
        if (!whole && part == 0 && h == 0) {
#pragma unroll
            for (int i = 1; i < KW; ++i) sum += tops[rw][i][l];
            p.stats[place * 2] = weightless ? kNoWeight : top;
            p.stats[place * 2 + 1] = sum;
        }
    } else {

    // A summer. Row addresses: of the pages whose numbers ids[] holds, by one wave, a token a lane.
    auto set_rows = [&](int tile) {
        if (lane < KEYS) {
            // Behind the last token that some row sees that token's row again, which stands for nothing there.
            const uint32_t token = min(static_cast<uint32_t>(tile) * KEYS + lane, static_cast<uint32_t>(all) - 1), page = token / page_size;
            const int32_t page_id = ids[holds][page - held_page];
            const bool held = page_id >= 0 && page_id < p.c.pages;
            const uint64_t at = held ? (static_cast<uint64_t>(page_id) * page_size + (token - page * page_size)) * ROW : 0;
            row_at[tile % SLOTS][lane] = WIDE ? reinterpret_cast<uint64_t>(p.c.bytes) + at : at;
            missing[tile % SLOTS][lane] = held ? 0 : 0xFFFFFFFFu;
        }
    };
    const uint32_t lds0 = static_cast<uint32_t>(reinterpret_cast<uintptr_t>((LdsByte*)tiles[0]));
    // A wave's loads of a tile, in two steps: all their places, which are read from LDS, then the loads one by one.
    constexpr int ASKS = (S::LOADS + SUMMERS - 1) / SUMMERS;
    struct Asks {
        uint32_t offset[ASKS], to;
    };
    auto whole_wave = [&](int i) { return (i + 1) * SUMMERS * 64 <= KEYS * PIECES; };
    auto active = [&](int i) { return (i * SUMMERS + own) * 64 + lane < KEYS * PIECES; };
    uint32_t places[WIDE ? 1 : ASKS];  // a piece's row in the upper half and bytes in the lower, one register for both
    if constexpr (!WIDE) {
#pragma unroll
        for (int i = 0; i < ASKS; ++i) {
            const int piece = min((i * SUMMERS + own) * 64 + lane, KEYS * PIECES - 1), r = piece / PIECES;
            places[i] = static_cast<uint32_t>(r * 8) << 16 | (piece - r * PIECES) * 16;
            asm volatile("" : "+v"(places[i]));
        }
    }
    auto find_one = [&](Asks& asks, int tile, int i) {
        const uint8_t* const table = reinterpret_cast<const uint8_t*>(row_at[tile % SLOTS]);
        asks.offset[i] = *reinterpret_cast<const uint32_t*>(table + (places[i] >> 16)) + (places[i] & 0xFFFF);
    };
    auto find = [&](Asks& asks, int tile, int stage) {
        asks.to = __builtin_amdgcn_readfirstlane(lds0 + stage * S::BYTES + own * 1024);
#pragma unroll
        for (int i = 0; i < ASKS; ++i) find_one(asks, tile, i);
    };
    auto ask = [&](const Asks& asks, int i) {
        if (whole_wave(i) || active(i)) load_row_pieces(p.c.bytes, asks.offset[i], __builtin_amdgcn_readfirstlane(asks.to + i * SUMMERS * 1024));
    };
    auto ask_wide = [&](int tile, int stage) {
        const uint32_t to = __builtin_amdgcn_readfirstlane(lds0 + stage * S::BYTES + own * 1024);
        for (int i = 0; i < ASKS; ++i) {
            const int piece = (i * SUMMERS + own) * 64 + lane, r = piece / PIECES;
            const uint32_t at = __builtin_amdgcn_readfirstlane(to + i * SUMMERS * 1024);
            if (piece < KEYS * PIECES) load_row_pieces(reinterpret_cast<const uint8_t*>(row_at[tile % SLOTS][r] + (piece - r * PIECES) * 16), at);
        }
    };
    auto load_tile = [&](int tile, int stage) {
        if constexpr (WIDE) {
            ask_wide(tile, stage);
        } else {
            Asks asks;
            find(asks, tile, stage);
#pragma unroll
            for (int i = 0; i < ASKS; ++i) ask(asks, i);
        }
    };
    f32x16 acc[RG][CT];
#pragma unroll
    for (int r = 0; r < RG; ++r)
#pragma unroll
        for (int c = 0; c < CT; ++c) acc[r][c] = f32x16{};

    // The latents of the tokens whose weights a lane holds, eight of a column: the rows' bytes turned as they are read.
    // Beside its products go the loads of a later tile (at once they would fill the memory's queue and hold the wave up, 1450
    // cycles of a tile's 4400), then the places of the one after that, `find_tile`.
    auto add_tile = [&](int tile, const uint8_t* rows, Asks& asks, int find_tile, auto with_asks) {
        constexpr int VS = 2 * KW, GROUP = E4M3 && CT % 2 == 0 ? 2 : 1, N = GROUP * VS;  // column tiles read ahead of their products
        struct Codes {
            i32x2 v;
        };
        struct Words {
            i16x4 lo, hi;
        };
        using Fragment = std::conditional_t<E4M3, Codes, Words>;
        const uint8_t* const at0 = rows + (E4M3 ? 1 : 2) * (part * CT * 32 + 16 * (lane >> 4 & 1)) +
                                   (E4M3 ? ((lane >> 1 & 3) + 8 * (lane >> 3 & 1) + 4 * h) * ROW + 8 * (lane & 1) : ((lane >> 2 & 3) + 4 * h) * ROW + 8 * (lane & 3));
        auto read = [&](Fragment (&f)[N], int c) {
#pragma unroll
            for (int i = 0; i < N; ++i) {
                const uint8_t* const at = at0 + (i / GROUP) * 16 * ROW + (c + i % GROUP) * (E4M3 ? 32 : 64);
                if constexpr (E4M3) {
                    f[i].v = __builtin_amdgcn_ds_read_tr8_b64_v2i32((__attribute__((address_space(3))) i32x2*)at);
                } else {
                    f[i].lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) i16x4*)at);
                    f[i].hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) i16x4*)(at + 8 * ROW));
                }
            }
        };
        // A latent that is no number makes its scores none, and the weight of every row that sees it; where a row does not, its
        // weight 0 has to meet a number. Seldom: rows that were written hold numbers, and a scale of NaN.
        auto scrub = [&](Fragment (&f)[N]) {
#pragma unroll
            for (int i = 0; i < N; ++i) {
                if constexpr (E4M3) {
#pragma unroll
                    for (int k = 0; k < 8; ++k) {
                        const uint32_t byte = 255u << (8 * (k & 3)), nan = 127u << (8 * (k & 3)), word = static_cast<uint32_t>(f[i].v[k / 4]);
                        if ((word & nan) == nan) f[i].v[k / 4] = static_cast<int>(word & ~byte);
                    }
                } else {
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        if ((f[i].lo[k] & 0x7F80) == 0x7F80) f[i].lo[k] = 0;
                        if ((f[i].hi[k] & 0x7F80) == 0x7F80) f[i].hi[k] = 0;
                    }
                }
            }
        };
        Fragment ahead[2][N];
        read(ahead[0], 0);
        bf16x8 w[RG][VS];
#pragma unroll
        for (int r = 0; r < RG; ++r)
#pragma unroll
            for (int i = 0; i < VS; ++i) w[r][i] = shared_weights[tile & 1][RG == 1 ? rw : r][i / 2][i % 2][lane];
        const bool tainted = odd[tile & 1] == tile + 1;
#pragma unroll
        for (int c = 0; c < CT; c += GROUP) {
            Fragment(&f)[N] = ahead[c / GROUP & 1];
            if (c + GROUP < CT) read(ahead[c / GROUP + 1 & 1], c + GROUP);
            if (__builtin_expect(tainted, 0)) scrub(f);
            auto latents = [&](int i) {
                if constexpr (E4M3) return e4m3_octet(f[i].v[0], f[i].v[1], 1.0f);
                else return __builtin_bit_cast(bf16x8, __builtin_shufflevector(f[i].lo, f[i].hi, 0, 1, 2, 3, 4, 5, 6, 7));
            };
            bf16x8 next = latents(0);
#pragma unroll
            for (int i = 0; i < N; ++i) {
                const bf16x8 now = next;
                if (i + 1 < N) next = latents(i + 1);
#pragma unroll
                for (int r = 0; r < RG; ++r) {
                    acc[r][c + i % GROUP] = mfma(now, w[r][i / GROUP], acc[r][c + i % GROUP]);
                    if constexpr (decltype(with_asks)::value) {
                        // One load with every second product, with fewer products as many as it takes.
                        constexpr int STEPS = CT * VS * RG, PER = (ASKS + STEPS - 1) / STEPS, EVERY = STEPS >= 2 * ASKS ? 2 : 1;
                        const int step = (c * VS + i) * RG + r;
#pragma unroll
                        for (int k = 0; k < PER; ++k)
                            if (step % EVERY == 0 && step / EVERY * PER + k < ASKS) ask(asks, step / EVERY * PER + k);
                        // Their registers are free for the next places, one a product, the last product's for what is left.
                        constexpr int FREE = ((ASKS + PER - 1) / PER - 1) * EVERY + 1;
#pragma unroll
                        for (int k = 0; k < ASKS; ++k)
                            if (k == step - FREE || (step == STEPS - 1 && k > step - FREE)) find_one(asks, find_tile, k);
                    }
                }
                __builtin_amdgcn_sched_barrier(0);
            }
        }
    };

    if (first < last) {
        for (int i = own; i < AHEAD + 2; i += SUMMERS) set_rows(first + i);
        __syncthreads();
#pragma unroll
        for (int i = 0; i < AHEAD; ++i)
            if (first + i < last) load_tile(first + i, i);
        if (first + AHEAD <= last) wait_for_rows_but<(AHEAD - 1) * (S::LOADS / SUMMERS)>();
        else wait_for_rows();
        Asks asks{};
        if constexpr (!WIDE) find(asks, first + AHEAD, AHEAD);
        __syncthreads();
        // Before the scorers, whose weights are not needed until the barrier: 64 x 16384 tokens 139 -> 134 us (a chunk of 256 188 -> 189).
        __builtin_amdgcn_s_setprio(2);
        int stage = 0;  // of the tile that is scored
        for (int tile = first; tile < last; ++tile) {
            // The stage that is loaded now was summed in the iteration before this one. Behind the last tile that tile is loaded
            // again, and not read.
            const int free_stage = stage >= STAGES - AHEAD ? stage + AHEAD - STAGES : stage + AHEAD;
            if constexpr (WIDE) {
                if (tile + AHEAD < last) ask_wide(tile + AHEAD, free_stage);
            }
            if (tile > first) {
                add_tile(tile - 1, tiles[stage == 0 ? STAGES - 1 : stage - 1], asks, min(tile + AHEAD + 1, last - 1), std::bool_constant<!WIDE>{});
            } else if constexpr (!WIDE) {
#pragma unroll
                for (int i = 0; i < ASKS; ++i) ask(asks, i);
                find(asks, min(tile + AHEAD + 1, last - 1), 0);
            }
            if constexpr (!WIDE) asks.to = __builtin_amdgcn_readfirstlane(lds0 + (free_stage == STAGES - 1 ? 0 : free_stage + 1) * S::BYTES + own * 1024);
            if (own == tile % SUMMERS && tile + AHEAD + 2 < last) set_rows(tile + AHEAD + 2);
            if (tile + AHEAD + 3 < last && tile + AHEAD + 3 >= held_end) hold(tile + AHEAD + 3);
            if (tile + AHEAD < last) wait_for_rows_but<(AHEAD - 1) * (S::LOADS / SUMMERS)>();
            else wait_for_rows();
            __syncthreads();
            if (__builtin_expect(grown[tile & 1] == tile + 1, 0)) {
                __syncthreads();
                if (tile > first) {
#pragma unroll
                    for (int r = 0; r < RG; ++r) {
                        const float by = factors[RG == 1 ? rw : r][l];
#pragma unroll
                        for (int c = 0; c < CT; ++c) acc[r][c] *= by;
                    }
                }
            }
            stage = stage == STAGES - 1 ? 0 : stage + 1;
        }
        add_tile(last - 1, tiles[stage == 0 ? STAGES - 1 : stage - 1], asks, 0, std::false_type{});
    }
    __syncthreads();  // the rows' sums
    const int column = part * S::COLUMNS + 4 * h;
#pragma unroll
    for (int r = 0; r < RG; ++r) {
        const int group = RG == 1 ? rw : r, in_unit = 32 * group + l, out_row = row0 + in_unit;
        if (whole && out_row < p.rows) {
            float sum = 0.0f;
#pragma unroll
            for (int i = 0; i < KW; ++i) sum += tops[group][i][l];
            const float inverse = inverse_of(sum, true);
            uint16_t* const to = static_cast<uint16_t*>(p.out) + (b * p.rows + out_row) * R + column;
#pragma unroll
            for (int c = 0; c < CT; ++c)
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    float x[4];
#pragma unroll
                    for (int e = 0; e < 4; ++e) x[e] = acc[r][c][4 * j + e] * inverse;
                    *reinterpret_cast<u32x2*>(to + 32 * c + 8 * j) =
                        u32x2{__builtin_bit_cast(uint32_t, bf16x2{static_cast<__bf16>(x[0]), static_cast<__bf16>(x[1])}),
                              __builtin_bit_cast(uint32_t, bf16x2{static_cast<__bf16>(x[2]), static_cast<__bf16>(x[3])})};
                }
        } else if (!whole && first < last) {
            float* const to = p.partial + (static_cast<int64_t>(share) * 2 + (part_of_share != 0)) * (RW * 32) * R + in_unit * R + column;
#pragma unroll
            for (int c = 0; c < CT; ++c)
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const f32x16& v = acc[r][c];
                    *reinterpret_cast<f32x4*>(to + 32 * c + 8 * j) = f32x4{v[4 * j], v[4 * j + 1], v[4 * j + 2], v[4 * j + 3]};
                }
        }
    }
    }
    if (p.shares == 0 || until <= unit_end) return;
    ++unit;
    from_tile = 0;
    __syncthreads();
    }
}

// The parts of a unit's rows: a row and 64 of its columns a block, 4 a lane, 16 parts at a time.
// 256 parts of 32 rows of 512 columns (17 MB): 6.8 us.
template <int R>
__global__ __launch_bounds__(256) void latent_join_rows_kernel(LatentAttentionArgs p, int rows_per_unit) {
    constexpr int COLUMNS = 64, LANES = COLUMNS / 4, GROUPS = 256 / LANES, BATCH = 8;
    __shared__ float by[256];
    __shared__ float reduced[4];
    __shared__ f32x4 sums[GROUPS][LANES];
    const int unit = blockIdx.x / (rows_per_unit * (R / COLUMNS)), in = blockIdx.x % (rows_per_unit * (R / COLUMNS));
    const int r = in / (R / COLUMNS), column = in % (R / COLUMNS) * COLUMNS + threadIdx.x % LANES * 4, group = threadIdx.x / LANES;
    const int64_t b = unit / p.row_blocks;
    const int row = static_cast<int>(unit - b * p.row_blocks) * rows_per_unit + r;
    if (row >= p.rows) return;
    // The shares that hold the unit's tiles: share g is of tiles each * g ..; where it is a share's first unit its part is the first.
    const int begin = p.starts[unit], end = p.starts[unit + 1], total = p.starts[p.units];
    const int each = max((total + p.shares - 1) / p.shares, kLeastShare), g0 = begin / each, parts = (end - 1) / each - g0 + 1;
    if (parts == 1) return;
    auto place = [&](int i) { return (static_cast<int64_t>(g0 + i) * 2 + (i == 0 && begin > g0 * each)) * rows_per_unit + r; };
    const int lane = threadIdx.x & 63, wave = threadIdx.x / 64;
    const bool mine = static_cast<int>(threadIdx.x) < parts;  // at most 256 of them
    const float top = mine ? p.stats[place(threadIdx.x) * 2] : -INFINITY;
    const float sum0 = mine ? p.stats[place(threadIdx.x) * 2 + 1] : 0.0f;
    float most = top;
#pragma unroll
    for (int m = 1; m < 64; m *= 2) most = fmaxf(most, __shfl_xor(most, m, kWave));
    if (lane == 0) reduced[wave] = most;
    __syncthreads();
    most = fmaxf(fmaxf(reduced[0], reduced[1]), fmaxf(reduced[2], reduced[3]));
    const float factor = __builtin_amdgcn_exp2f(top - finite_or_zero(most));
    by[threadIdx.x] = sum0 == 0.0f ? 0.0f : factor;  // of a part that saw nothing: its sums may not have been written
    float sum = sum0 == 0.0f ? 0.0f : sum0 * factor;
#pragma unroll
    for (int m = 1; m < 64; m *= 2) sum += __shfl_xor(sum, m, kWave);
    __syncthreads();
    if (lane == 0) reduced[wave] = sum;
    __syncthreads();
    sum = (reduced[0] + reduced[1]) + (reduced[2] + reduced[3]);
    const float inverse = inverse_of(sum, most == -INFINITY);
    f32x4 acc = {0.0f, 0.0f, 0.0f, 0.0f};
    for (int i = group; i < parts; i += GROUPS * BATCH) {
        f32x4 v[BATCH];
        float f[BATCH];
#pragma unroll
        for (int k = 0; k < BATCH; ++k) {
            const int j = i + k * GROUPS;
            f[k] = j < parts ? by[j] : 0.0f;
            if (f[k] != 0.0f) v[k] = *reinterpret_cast<const f32x4*>(p.partial + place(j) * R + column);
        }
#pragma unroll
        for (int k = 0; k < BATCH; ++k) {
            if (f[k] != 0.0f) {
#pragma unroll
                for (int j = 0; j < 4; ++j) acc[j] = fmaf(v[k][j], f[k], acc[j]);
            }
        }
    }
    sums[group][threadIdx.x % LANES] = acc;
    __syncthreads();
    if (group != 0) return;
#pragma unroll
    for (int i = 1; i < GROUPS; ++i) acc += sums[i][threadIdx.x];
    acc *= inverse;
    *reinterpret_cast<u32x2*>(static_cast<uint16_t*>(p.out) + (b * p.rows + row) * R + column) =
        u32x2{__builtin_bit_cast(uint32_t, bf16x2{static_cast<__bf16>(acc[0]), static_cast<__bf16>(acc[1])}),
              __builtin_bit_cast(uint32_t, bf16x2{static_cast<__bf16>(acc[2]), static_cast<__bf16>(acc[3])})};
}

// The same where rows have few parts: a wave a row (of 64 lanes or as many as its columns take, 4 or 8 a lane), eight parts and
// their statistics asked for at a time, under a running maximum. 12,288 rows of 512 columns in two or three parts each (58 MB):
// 12.4 us; by the kernel above 24.9.
template <int R>
__global__ __launch_bounds__(256) void latent_join_few_kernel(LatentAttentionArgs p, int rows_per_unit) {
    constexpr int LANES = R / 4 < 64 ? R / 4 : 64, ROWS = 256 / LANES, EACH = R / 4 / LANES, BATCH = 8;
    const int blocks = rows_per_unit / ROWS, unit = blockIdx.x / blocks, r = (blockIdx.x - unit * blocks) * ROWS + threadIdx.x / LANES;
    const int column = threadIdx.x % LANES * 4;
    const int begin = p.starts[unit], end = p.starts[unit + 1], total = p.starts[p.units];
    const int each = max((total + p.shares - 1) / p.shares, kLeastShare), g0 = begin / each, parts = (end - 1) / each - g0 + 1;
    const int64_t b = unit / p.row_blocks;
    const int row = static_cast<int>(unit - b * p.row_blocks) * rows_per_unit + r;
    if (parts == 1 || row >= p.rows) return;
    float most = -INFINITY, sum = 0.0f;
    f32x4 acc[EACH] = {};
    for (int i = 0; i < parts; i += BATCH) {
        f32x2 stats[BATCH];
        f32x4 v[BATCH][EACH];
#pragma unroll
        for (int k = 0; k < BATCH; ++k) {
            stats[k] = f32x2{-INFINITY, 0.0f};
            if (i + k >= parts) continue;
            const int part = i + k;
            const int64_t place = (static_cast<int64_t>(g0 + part) * 2 + (part == 0 && begin > g0 * each)) * rows_per_unit + r;
            stats[k] = *reinterpret_cast<const f32x2*>(p.stats + place * 2);
#pragma unroll
            for (int j = 0; j < EACH; ++j) v[k][j] = *reinterpret_cast<const f32x4*>(p.partial + place * R + column + 256 * j);
        }
        float now = most;
#pragma unroll
        for (int k = 0; k < BATCH; ++k) now = fmaxf(now, stats[k][0]);
        const float before = __builtin_amdgcn_exp2f(most - finite_or_zero(now));
        most = now;
        sum *= before;
#pragma unroll
        for (int j = 0; j < EACH; ++j) acc[j] *= before;
#pragma unroll
        for (int k = 0; k < BATCH; ++k) {
            // Of a part that saw nothing the sums may not have been written.
            const float f = stats[k][1] == 0.0f ? 0.0f : __builtin_amdgcn_exp2f(stats[k][0] - finite_or_zero(now));
            sum = fmaf(stats[k][1], f, sum);
            if (f != 0.0f) {
#pragma unroll
                for (int j = 0; j < EACH; ++j)
#pragma unroll
                    for (int e = 0; e < 4; ++e) acc[j][e] = fmaf(v[k][j][e], f, acc[j][e]);
            }
        }
    }
    const float inverse = inverse_of(sum, most == -INFINITY);
#pragma unroll
    for (int j = 0; j < EACH; ++j) {
        const f32x4 x = acc[j] * inverse;
        *reinterpret_cast<u32x2*>(static_cast<uint16_t*>(p.out) + (b * p.rows + row) * R + column + 256 * j) =
            u32x2{__builtin_bit_cast(uint32_t, bf16x2{static_cast<__bf16>(x[0]), static_cast<__bf16>(x[1])}),
                  __builtin_bit_cast(uint32_t, bf16x2{static_cast<__bf16>(x[2]), static_cast<__bf16>(x[3])})};
    }
}

// The parts of a row of fp32, 64 columns a block: 16 lanes side by side, 16 parts at a time.
template <int R>
__global__ __launch_bounds__(256) void latent_join_f32_kernel(const float* partial, const float* stats, int splits, float* out) {
    __shared__ float by[256];
    __shared__ float reduced[4];
    __shared__ f32x4 sums[16][16];
    const int64_t row = blockIdx.x / (R / 64);
    const int lane = threadIdx.x & 63, wave = threadIdx.x / 64, group = threadIdx.x / 16, column = blockIdx.x % (R / 64) * 64 + threadIdx.x % 16 * 4;
    const float* const from = partial + (row * splits + group) * R + column;
    // Every load is issued before the first is waited for; a part that saw nothing may hold anything.
    f32x4 v[16];
#pragma unroll
    for (int i = 0; i < 16; ++i)
        if (group + 16 * i < splits) v[i] = *reinterpret_cast<const f32x4*>(from + 16 * i * R);
    const bool mine = static_cast<int>(threadIdx.x) < splits;  // at most 256 of them
    const float top = mine ? stats[(row * splits + threadIdx.x) * 2] : -INFINITY;
    const float total = mine ? stats[(row * splits + threadIdx.x) * 2 + 1] : 0.0f;
    float most = top;
#pragma unroll
    for (int m = 1; m < 64; m *= 2) most = fmaxf(most, __shfl_xor(most, m, kWave));
    if (lane == 0) reduced[wave] = most;
    __syncthreads();
    most = fmaxf(fmaxf(reduced[0], reduced[1]), fmaxf(reduced[2], reduced[3]));
    const float factor = __builtin_amdgcn_exp2f(top - finite_or_zero(most));
    by[threadIdx.x] = total == 0.0f ? 0.0f : factor;
    float sum = total == 0.0f ? 0.0f : total * factor;
#pragma unroll
    for (int m = 1; m < 64; m *= 2) sum += __shfl_xor(sum, m, kWave);
    __syncthreads();
    if (lane == 0) reduced[wave] = sum;
    __syncthreads();
    sum = (reduced[0] + reduced[1]) + (reduced[2] + reduced[3]);
    const float inverse = inverse_of(sum, most == -INFINITY);
    f32x4 acc = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int i = 0; i < 16; ++i) {
        const float f = group + 16 * i < splits ? by[group + 16 * i] : 0.0f;
        if (f != 0.0f) {
#pragma unroll
            for (int j = 0; j < 4; ++j) acc[j] = fmaf(v[i][j], f, acc[j]);
        }
    }
    sums[group][threadIdx.x % 16] = acc;
    __syncthreads();
    if (group != 0) return;
#pragma unroll
    for (int i = 1; i < 16; ++i) acc += sums[i][threadIdx.x];
    acc *= inverse;
    *reinterpret_cast<f32x4*>(out + row * R + column) = acc;
}

struct Plan {
    int64_t row_blocks, splits, units, shares, workspace;
};
constexpr int kChip = 256;  // compute units
// Rows a block by the rows a sequence has: the cache is read, and turned into bf16, once for all of them. Up to 32 rows are
// half a block of 64: 24 sequences of 16 heads 38.7 us (64: 45.0), one of 32 heads and 131072 tokens 35.0 (39.7).
int64_t rows_per_block(int64_t rows, bool f32) { return f32 ? 16 : rows <= 32 ? 32 : 64; }
Plan plan_of(int64_t batch, int64_t rows, int64_t rank, bool f32, int64_t capacity) {
    Plan plan{};
    const int64_t per = rows_per_block(rows, f32);
    plan.row_blocks = ceil_div(rows, per);
    plan.units = batch * plan.row_blocks;
    const int64_t tiles = ceil_div(capacity, kTile);
    if (f32) {
        plan.splits = std::max<int64_t>(1, std::min<int64_t>(std::min<int64_t>(tiles / 2, 256), ceil_div(512, std::max<int64_t>(plan.units, 1))));
        plan.workspace = plan.splits == 1 ? 0 : batch * rows * plan.splits * (rank + 2) * 4;
        return plan;
    }
    // Shares where there are few units; with more a unit a block balances well enough where sequences are of like lengths, and
    // has nothing to join. One long sequence among more than 1024 units is then one block's work a unit.
    if (plan.units <= kMaxUnits && tiles > kLeastShare && plan.units * 2 * tiles < (int64_t{1} << 31)) {
        plan.shares = kChip;
        plan.workspace = plan.shares * 2 * per * (rank + 2) * 4 + (kMaxUnits + 1) * 4;
    }
    return plan;
}

template <int R, int P, bool F32, bool E4M3>
void launch_attention(const LatentAttentionArgs& p, int64_t blocks, hipStream_t s) {
    const dim3 grid(static_cast<unsigned>(blocks));
    if constexpr (F32) {
        hipLaunchKernelGGL((latent_attention_f32_kernel<R, P, E4M3>), grid, dim3(256), 0, s, p);
    } else {
        const int64_t rows = rows_per_block(p.rows, false);
        auto go = [&](auto groups) {
            constexpr int RW = decltype(groups)::value;
            const dim3 threads(Shape<R, P, E4M3, RW>::WAVES * 64);
            if (p.wide) hipLaunchKernelGGL((latent_attention_rows_kernel<R, P, E4M3, RW, true>), grid, threads, 0, s, p);
            else hipLaunchKernelGGL((latent_attention_rows_kernel<R, P, E4M3, RW, false>), grid, threads, 0, s, p);
        };
        if (rows == 32) go(std::integral_constant<int, 1>{});
        else go(std::integral_constant<int, 2>{});
    }
}
template <int R, int P>
void launch_attention(const LatentAttentionArgs& p, bool f32, bool e4m3, int64_t blocks, hipStream_t s) {
    if (f32) e4m3 ? launch_attention<R, P, true, true>(p, blocks, s) : launch_attention<R, P, true, false>(p, blocks, s);
    else e4m3 ? launch_attention<R, P, false, true>(p, blocks, s) : launch_attention<R, P, false, false>(p, blocks, s);
}
template <int R>
void launch_attention(const LatentAttentionArgs& p, int64_t rope, bool f32, bool e4m3, int64_t blocks, hipStream_t s) {
    if (rope == 16) launch_attention<R, 16>(p, f32, e4m3, blocks, s);
    else if (rope == 32) launch_attention<R, 32>(p, f32, e4m3, blocks, s);
    else launch_attention<R, 64>(p, f32, e4m3, blocks, s);
    if (!f32) {
        if (p.shares == 0) return;
        const int per = static_cast<int>(rows_per_block(p.rows, false));
        // A row of many parts falls to several blocks of 64 columns: 256 parts of each of 32 rows 35.0 us with the attention, by
        // one wave a row 78.9. Where rows have some ten parts a wave each is faster: 24 units 6.0 us, by 64 columns 9.8. How many
        // a row has is not known here: units stand for it, and of 17 or more with one long sequence among them that one's rows,
        // of up to 256 parts, are joined by a wave each.
        if (p.units * 16 <= p.shares) hipLaunchKernelGGL((latent_join_rows_kernel<R>), dim3(static_cast<unsigned>(p.units * per * (R / 64))), dim3(256), 0, s, p, per);
        else hipLaunchKernelGGL((latent_join_few_kernel<R>), dim3(static_cast<unsigned>(p.units * per / (R / 4 < 64 ? 1024 / R : 4))), dim3(256), 0, s, p, per);
        return;
    }
    if (p.splits == 1) return;
    const int64_t rows = static_cast<int64_t>(p.units) / p.row_blocks * p.rows;
    hipLaunchKernelGGL((latent_join_f32_kernel<R>), dim3(static_cast<unsigned>(rows * (R / 64))), dim3(256), 0, s, p.partial, p.stats, p.splits,
                       static_cast<float*>(p.out));
}

mlk_status check_attention(int64_t batch, int64_t length, int64_t heads) {
    MLK_CHECK(heads > 0 && heads < (int64_t{1} << 16), "heads must be between 1 and 65535");
    MLK_CHECK(length < (int64_t{1} << 31) / heads, "too many tokens");
    MLK_CHECK(batch * ceil_div(length * heads, 16) < (int64_t{1} << 22), "too many tokens for one launch");
    return MLK_OK;
}

}  // namespace
}  // namespace mlk

using namespace mlk;

extern "C" size_t mlk_latent_attention_workspace_bytes(int64_t batch, int64_t length, int64_t heads, int64_t rank, int64_t rope_dim, int32_t dtype,
                                                       int32_t cache_dtype, int64_t page_size, int64_t table_width) {
    if (check_latent_cache(batch, length, rank, rope_dim, dtype, cache_dtype, 1, page_size, table_width) != MLK_OK ||
        check_attention(batch, length, heads) != MLK_OK || batch == 0 || length == 0)
        return 0;
    return static_cast<size_t>(plan_of(batch, length * heads, rank, dtype == MLK_DTYPE_F32, page_size * table_width).workspace);
}

extern "C" mlk_status mlk_latent_attention(const void* q_latent, const int64_t* q_latent_strides, const void* q_rope, const int64_t* q_rope_strides,
                                           int32_t dtype, int64_t batch, int64_t length, int64_t heads, int64_t rank, int64_t rope_dim,
                                           const uint8_t* cache, int32_t cache_dtype, int64_t pages, int64_t page_size, const int32_t* page_table,
                                           int64_t table_width, const int32_t* positions, const int64_t* ancestors, double scale, void* out,
                                           void* workspace, size_t workspace_bytes, mlk_stream_t stream) {
    mlk_status checked = check_latent_cache(batch, length, rank, rope_dim, dtype, cache_dtype, pages, page_size, table_width);
    if (checked == MLK_OK) checked = check_attention(batch, length, heads);
    if (checked != MLK_OK) return checked;
    MLK_CHECK(ancestors == nullptr || length <= 64, "a tree holds at most 64 tokens");
    MLK_CHECK(std::isfinite(static_cast<float>(scale * 1.4426950408889634074)), "scale must be finite");
    if (batch == 0 || length == 0) return MLK_OK;
    MLK_CHECK(q_latent && q_latent_strides && q_rope && q_rope_strides && cache && page_table && positions && out, "null tensor pointer");
    MLK_CHECK((reinterpret_cast<uintptr_t>(cache) & 15) == 0 && (reinterpret_cast<uintptr_t>(out) & 15) == 0, "cache and out must be 16-byte aligned");
    const bool f32 = dtype == MLK_DTYPE_F32, e4m3 = cache_dtype == MLK_DTYPE_E4M3;
    const Plan plan = plan_of(batch, length * heads, rank, f32, page_size * table_width);
    MLK_CHECK(plan.workspace == 0 || (workspace && workspace_bytes >= static_cast<size_t>(plan.workspace) &&
                                      (reinterpret_cast<uintptr_t>(workspace) & 15) == 0),
              "the workspace is too small or not 16-byte aligned");
    LatentAttentionArgs p{};
    p.q = q_latent;
    p.qr = q_rope;
    for (int i = 0; i < 3; ++i) {
        p.qs[i] = q_latent_strides[i];
        p.rs[i] = q_rope_strides[i];
    }
    p.c = {cache, page_table, static_cast<int32_t>(pages), static_cast<int32_t>(page_size), static_cast<int32_t>(table_width)};
    p.positions = positions;
    p.ancestors = ancestors;
    p.out = out;
    p.partial = static_cast<float*>(workspace);
    p.length = static_cast<int32_t>(length);
    p.heads = static_cast<int32_t>(heads);
    p.rows = static_cast<int32_t>(length * heads);
    p.row_blocks = static_cast<int32_t>(plan.row_blocks);
    p.splits = static_cast<int32_t>(plan.splits);
    p.scale = static_cast<float>(std::fabs(scale) * 1.4426950408889634074);
    p.negate = std::signbit(scale) ? 0x80008000u : 0;
    p.wide = pages * page_size * (e4m3 ? rank + 2 * rope_dim + 16 : 2 * (rank + rope_dim) + 16) > (int64_t{1} << 32);
    p.units = static_cast<int32_t>(plan.units);
    p.shares = static_cast<int32_t>(plan.shares);
    if (f32) p.stats = p.partial + batch * p.rows * plan.splits * rank;
    if (plan.shares != 0) {
        const int64_t parts = plan.shares * 2 * rows_per_block(p.rows, f32);
        p.stats = p.partial + parts * rank;
        p.starts = reinterpret_cast<int32_t*>(p.stats + parts * 2);
    }
    const int64_t blocks = f32 ? plan.units * plan.splits : plan.shares != 0 ? plan.shares : plan.units;
    hipStream_t s = reinterpret_cast<hipStream_t>(stream);
    switch (rank) {
        case 64: launch_attention<64>(p, rope_dim, f32, e4m3, blocks, s); break;
        case 128: launch_attention<128>(p, rope_dim, f32, e4m3, blocks, s); break;
        case 256: launch_attention<256>(p, rope_dim, f32, e4m3, blocks, s); break;
        default: launch_attention<512>(p, rope_dim, f32, e4m3, blocks, s); break;
    }
    return launch_status("latent attention");
}
