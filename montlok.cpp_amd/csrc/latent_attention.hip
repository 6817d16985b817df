// Attention in the latents' space over a cache of token rows (latent c, shared rotated key part r):
//
//   s[key] = (q_latent . c[key] + q_rope . r[key]) * scale,   out = sum softmax(s)[key] c[key]
//
// One pass over a sequence's rows with a running maximum and sum; all heads of a token, and all tokens of a call, read the
// same rows.
#include <algorithm>
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
    float* partial;  // [sequence][row][split][R], then the maxima and sums [sequence][row][split][2]
    int32_t length, heads, rows, row_blocks, splits;
    float scale;  // times log2(e)
};

constexpr int kTile = 64;   // tokens of a tile
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
#pragma clang diagnostic pop
__device__ __forceinline__ void wait_for_rows() {
    __builtin_amdgcn_s_waitcnt(0x0F70);  // vmcnt 0, the other counters at their most
    asm volatile("" ::: "memory");
}

// MT tiles of 16 rows (a row is a token and a query head) of one sequence over every `splits`-th part of its tokens.
// Wave (rg, kg) scores the row tiles of group rg with 16 tokens of a tile, then takes R / WAVES columns of all rows' sums.
// Every product has the rows as its columns (scores are tokens x rows, sums are columns x rows), so that a lane's numbers all
// belong to row lane & 15 of a tile: its maximum, sum and rescaling are one number, its weights of four tokens and its sums
// of four columns lie side by side.
template <int R, int P, bool F32, bool E4M3, int MT, int WAVES>
__global__ __launch_bounds__(WAVES * 64, F32 ? 1 : WAVES / 4) void latent_attention_kernel(LatentAttentionArgs p) {
    constexpr int ROW = row_bytes<E4M3>(R, P), PIECES = ROW / 16, kPlanes = F32 ? 3 : 1;
    constexpr int RG = WAVES / 4, RT = MT / RG, COLS = R / WAVES, CT = COLS / 16;
    constexpr int KS = R / 32, RS = (P + 31) / 32;  // 32-deep steps over the latent and the key part
    static_assert(MT % RG == 0 && COLS % 16 == 0, "rows and columns fall to whole tiles");
    __shared__ __attribute__((aligned(16))) uint8_t tiles[2][kTile * ROW];
    __shared__ __attribute__((aligned(16))) uint16_t weights[kPlanes][MT * 16 * kPPitch];
    __shared__ float maxima[4][MT * 16];
    __shared__ const uint8_t* row_at[kTile];
    __shared__ float missing[2][kTile];  // NaN where a token's page is missing, else 0
    __shared__ int tainted[2];           // some score of the tile is not finite
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64), lane = threadIdx.x & 63, g = lane >> 4, l = lane & 15;
    const int kg = wave % 4, rg = wave / 4;
    unsigned id = blockIdx.x;
    const int split = id % p.splits;
    id /= p.splits;
    const int row0 = static_cast<int>(id % p.row_blocks) * (MT * 16);
    const int64_t b = id / p.row_blocks;

    // What each of the lane's rows sees: tokens below `base`, and base + j where bit j is set. A plain row sees base = its
    // position + 1 tokens.
    int base[MT], end = 0, at[MT];
    uint64_t bits[MT];
    bool beyond[MT];
    const int64_t capacity = static_cast<int64_t>(p.c.width) * p.c.page_size;
#pragma unroll
    for (int m = 0; m < MT; ++m) {
        const int row = row0 + 16 * m + l;
        const int token = row / p.heads;
        at[m] = row < p.rows ? p.positions[b * p.length + token] : -1;
        beyond[m] = at[m] >= capacity;
        base[m] = 0;
        bits[m] = 0;
        if (at[m] >= 0 && !beyond[m]) {
            if (p.ancestors == nullptr) {
                base[m] = at[m] + 1;
                end = max(end, base[m]);
            } else {
                base[m] = at[m] - token;
                bits[m] = static_cast<uint64_t>(p.ancestors[b * p.length + token]);
                if (p.length < 64) bits[m] &= (uint64_t{1} << p.length) - 1;
                end = max(end, bits[m] == 0 ? base[m] : base[m] + 64 - __builtin_clzll(bits[m]));
            }
        }
    }
#pragma unroll
    for (int m = 1; m < 16; m *= 2) end = max(end, __shfl_xor(end, m, kWave));
    end = __builtin_amdgcn_readfirstlane(end);

    const int tile_count = (end + kTile - 1) / kTile, per_split = (tile_count + p.splits - 1) / p.splits;
    const int first = min(split * per_split, tile_count), last = min(first + per_split, tile_count);

    // The lane's queries: of row tile m, step s, the dimensions that its piece of a key row holds.
    bf16x8 q[RT][KS + RS][kPlanes];
    auto dimension = [&](int s) {  // of the latent; codes come 16 to a piece, bf16 values 8
        return E4M3 ? 64 * (s / 2) + 16 * g + 8 * (s % 2) : 32 * s + 8 * g;
    };
#pragma unroll
    for (int m = 0; m < RT; ++m) {
        const int row = row0 + 16 * (rg * RT + m) + l, token = row / p.heads, head = row - token * p.heads;
        const bool real = row < p.rows;
        const int64_t ql = b * p.qs[0] + token * p.qs[1] + head * p.qs[2], qr = b * p.rs[0] + token * p.rs[1] + head * p.rs[2];
#pragma unroll
        for (int s = 0; s < KS + RS; ++s) {
            const bool in_latent = s < KS;
            const int d = in_latent ? dimension(s) : 32 * (s - KS) + 8 * g;
            const void* const from = in_latent ? p.q : p.qr;
            const int64_t start = (in_latent ? ql : qr) + d;
            const bool take = real && (in_latent || d < P);
            if constexpr (F32) {
                float v[8] = {};
                if (take) {
                    const u32x4 lo = *reinterpret_cast<const u32x4_any*>(static_cast<const float*>(from) + start);
                    const u32x4 hi = *reinterpret_cast<const u32x4_any*>(static_cast<const float*>(from) + start + 4);
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        v[i] = __uint_as_float(lo[i]);
                        v[4 + i] = __uint_as_float(hi[i]);
                    }
                }
                bf16x8 plane[3];
                planes_of<true>(v, plane);
#pragma unroll
                for (int i = 0; i < 3; ++i) q[m][s][i] = plane[i];
            } else {
                u32x4 v = {0, 0, 0, 0};
                if (take) v = *reinterpret_cast<const u32x4_any*>(static_cast<const uint16_t*>(from) + start);
                q[m][s][0] = __builtin_bit_cast(bf16x8, v);
            }
        }
    }

    // Row addresses of a tile: by the first wave, a token a lane.
    auto page_of = [&](int tile) {
        const uint32_t token = static_cast<uint32_t>(tile) * kTile + lane;
        if (static_cast<int>(token) >= end) return -2;
        const uint32_t page = token / static_cast<uint32_t>(p.c.page_size);
        return page < static_cast<uint32_t>(p.c.width) ? p.c.table[b * p.c.width + page] : -1;
    };
    auto set_rows = [&](int tile, int page_id) {
        const uint32_t token = static_cast<uint32_t>(tile) * kTile + lane, in_page = token % static_cast<uint32_t>(p.c.page_size);
        const bool held = page_id >= 0 && page_id < p.c.pages;
        row_at[lane] = held ? p.c.bytes + (static_cast<int64_t>(page_id) * p.c.page_size + in_page) * ROW : kZeroRow;
        missing[tile & 1][lane] = held || page_id == -2 ? 0.0f : NAN;
    };
    auto load_tile = [&](int tile) {
        const uint32_t to = static_cast<uint32_t>(reinterpret_cast<uintptr_t>((LdsByte*)tiles[tile & 1]));
#pragma unroll
        for (int i = 0; i < (PIECES + WAVES - 1) / WAVES; ++i) {
            const int part = i * WAVES + wave;  // 64 pieces
            if (part < PIECES) {
                const int piece = part * 64 + lane, row = piece / PIECES;
                load_row_pieces(row_at[row] + (piece - row * PIECES) * 16, __builtin_amdgcn_readfirstlane(to + part * 1024));
            }
        }
    };

    f32x4 acc[MT][CT];
    float top[MT], sum[RT];
#pragma unroll
    for (int m = 0; m < MT; ++m) {
        top[m] = -INFINITY;
#pragma unroll
        for (int c = 0; c < CT; ++c) acc[m][c] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    }
#pragma unroll
    for (int m = 0; m < RT; ++m) sum[m] = 0.0f;

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

        // Scores of tokens 16 kg + 4 g + i with row l of each row tile.
        f32x4 s[RT], r[RT];
#pragma unroll
        for (int m = 0; m < RT; ++m) s[m] = r[m] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
        const uint8_t* const key = rows + (16 * kg + l) * ROW;
        if constexpr (E4M3) {
#pragma unroll
            for (int t = 0; t < KS / 2; ++t) {
                const u32x4 v = *reinterpret_cast<const u32x4*>(key + 64 * t + 16 * g);
                const bf16x8 a = e4m3_octet(v[0], v[1]), c = e4m3_octet(v[2], v[3]);
#pragma unroll
                for (int m = 0; m < RT; ++m)
#pragma unroll
                    for (int i = kPlanes - 1; i >= 0; --i) {
                        s[m] = mfma(a, q[m][2 * t][i], s[m]);
                        s[m] = mfma(c, q[m][2 * t + 1][i], s[m]);
                    }
            }
        } else {
#pragma unroll
            for (int t = 0; t < KS; ++t) {
                const bf16x8 a = *reinterpret_cast<const bf16x8*>(key + 64 * t + 16 * g);
#pragma unroll
                for (int m = 0; m < RT; ++m)
#pragma unroll
                    for (int i = kPlanes - 1; i >= 0; --i) s[m] = mfma(a, q[m][t][i], s[m]);
            }
        }
#pragma unroll
        for (int t = 0; t < RS; ++t) {
            const int d = 32 * t + 8 * g;
            // Where the key part is 16 wide the upper lanes' queries are zeros; they read the row's tail or zeros in its place.
            bf16x8 a = __builtin_bit_cast(bf16x8, u32x4{0, 0, 0, 0});
            if (P >= 32 || d < P) a = *reinterpret_cast<const bf16x8*>(key + (E4M3 ? R : 2 * R) + 2 * d);
#pragma unroll
            for (int m = 0; m < RT; ++m)
#pragma unroll
                for (int i = kPlanes - 1; i >= 0; --i) r[m] = mfma(a, q[m][KS + t][i], r[m]);
        }
        float key_scale[4], lost[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int token = 16 * kg + 4 * g + i;
            key_scale[i] = E4M3 ? *reinterpret_cast<const float*>(rows + token * ROW + R + 2 * P) : 1.0f;
            lost[i] = missing[tile & 1][token];
        }
        bool odd = false;
#pragma unroll
        for (int m = 0; m < RT; ++m) {
            const int row = rg * RT + m;
            float most = -INFINITY;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int token = tile * kTile + 16 * kg + 4 * g + i, past = token - base[row];
                float v = (E4M3 ? fmaf(s[m][i], key_scale[i], r[m][i]) : s[m][i] + r[m][i]) * p.scale + lost[i];
                odd |= !(fabsf(v) < INFINITY);
                const bool seen = past < 0 || (past < 64 && (bits[row] >> (past & 63) & 1));
                v = seen ? v : -INFINITY;
                s[m][i] = v;
                most = fmaxf(most, v);
            }
            most = max_over_groups(most);
            if (g == 0) maxima[kg][16 * row + l] = most;
        }
        if (odd) tainted[tile & 1] = 1;
        __syncthreads();  // the rows' maxima
        const bool clean = tainted[tile & 1] == 0;
        if (threadIdx.x == 0) tainted[~tile & 1] = 0;
        float by[MT];
#pragma unroll
        for (int m = 0; m < MT; ++m) {
            float most = top[m];
#pragma unroll
            for (int i = 0; i < 4; ++i) most = fmaxf(most, maxima[i][16 * m + l]);
            by[m] = __builtin_amdgcn_exp2f(top[m] - finite_or_zero(most));
            top[m] = most;
        }
#pragma unroll
        for (int m = 0; m < RT; ++m) {
            const int row = rg * RT + m;
            const float under = finite_or_zero(top[row]);
            float w[4], total = 0.0f;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float e = __builtin_amdgcn_exp2f(s[m][i] - under);
                total += e;
                w[i] = E4M3 ? (s[m][i] == -INFINITY ? 0.0f : e * key_scale[i]) : e;
            }
            sum[m] = fmaf(sum[m], by[row], total);
            uint16_t* const to = &weights[0][(16 * row + l) * kPPitch + 16 * kg + 4 * g];
            if constexpr (F32) {
                Parts3 x[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) x[i] = parts_of<true>(w[i]);
                *reinterpret_cast<u32x2*>(to) = u32x2{pack_upper(x[0].a, x[1].a), pack_upper(x[2].a, x[3].a)};
                *reinterpret_cast<u32x2*>(to + MT * 16 * kPPitch) = u32x2{pack_upper(x[0].b, x[1].b), pack_upper(x[2].b, x[3].b)};
                *reinterpret_cast<u32x2*>(to + 2 * MT * 16 * kPPitch) = u32x2{pack_upper(x[0].c, x[1].c), pack_upper(x[2].c, x[3].c)};
            } else {
                // Rounded to bf16 for the product with the latents: 2^-8 of a weight at most, without a bias; the sum keeps them whole.
                *reinterpret_cast<u32x2*>(to) = u32x2{__builtin_bit_cast(uint32_t, bf16x2{static_cast<__bf16>(w[0]), static_cast<__bf16>(w[1])}),
                                                      __builtin_bit_cast(uint32_t, bf16x2{static_cast<__bf16>(w[2]), static_cast<__bf16>(w[3])})};
            }
        }
#pragma unroll
        for (int m = 0; m < MT; ++m)
#pragma unroll
            for (int c = 0; c < CT; ++c) acc[m][c] *= by[m];
        if (!clean) {
            // A latent that is no number makes its scores none, and the weight of every row that sees it; where a row does not,
            // its weight 0 has to meet a number. Seldom: rows of a cache hold numbers, or codes 0 under a scale of NaN.
            uint8_t* const mine = tiles[tile & 1];
            for (int i = threadIdx.x; i < kTile * R / 4; i += WAVES * 64) {
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
            bf16x8 w[MT][kPlanes];
#pragma unroll
            for (int m = 0; m < MT; ++m)
#pragma unroll
                for (int i = 0; i < kPlanes; ++i) w[m][i] = *reinterpret_cast<const bf16x8*>(&weights[i][(16 * m + l) * kPPitch + 32 * t + 8 * g]);
#pragma unroll
            for (int c = 0; c < CT; ++c) {
                // Eight tokens of a column a lane: the rows' bytes turned as they are read.
                const int column = wave * COLS + 16 * c;
                bf16x8 v;
                if constexpr (E4M3) {
                    const i32x2 x = __builtin_amdgcn_ds_read_tr8_b64_v2i32(
                        (__attribute__((address_space(3))) i32x2*)(rows + (32 * t + 8 * g + l / 2) * ROW + column + 8 * (l & 1)));
                    v = e4m3_octet(x[0], x[1]);
                } else {
                    i16x4 x[2];
#pragma unroll
                    for (int h = 0; h < 2; ++h)
                        x[h] = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                            (__attribute__((address_space(3))) i16x4*)(rows + (32 * t + 8 * g + 4 * h + l / 4) * ROW + 2 * column + 8 * (l & 3)));
                    v = __builtin_bit_cast(bf16x8, __builtin_shufflevector(x[0], x[1], 0, 1, 2, 3, 4, 5, 6, 7));
                }
#pragma unroll
                for (int m = 0; m < MT; ++m)
#pragma unroll
                    for (int i = kPlanes - 1; i >= 0; --i) acc[m][c] = mfma(v, w[m][i], acc[m][c]);
            }
        }
        wait_for_rows();  // of the next tile
        if (wave == 0 && tile + 2 < last) set_rows(tile + 2, next_page);
    }

    // A row's sum lies with the lanes and waves that scored its tokens.
    __syncthreads();
#pragma unroll
    for (int m = 0; m < RT; ++m) {
        const float total = sum_over_groups(sum[m]);
        if (g == 0) maxima[kg][16 * (rg * RT + m) + l] = total;
    }
    __syncthreads();
#pragma unroll
    for (int m = 0; m < MT; ++m) {
        const int row = row0 + 16 * m + l;
        if (row >= p.rows) continue;
        const float total = maxima[0][16 * m + l] + maxima[1][16 * m + l] + maxima[2][16 * m + l] + maxima[3][16 * m + l];
        const int64_t at_row = b * p.rows + row;
        if (p.splits == 1) {
            // A row that sees nothing has no sum: zeros. One past the table: NaN.
            const float inverse = beyond[m] ? NAN : total == 0.0f ? 0.0f : 1.0f / total;
#pragma unroll
            for (int c = 0; c < CT; ++c) {
                const int64_t to = at_row * R + wave * COLS + 16 * c + 4 * g;
                const f32x4 v = acc[m][c] * inverse;
                if constexpr (F32) {
                    *reinterpret_cast<f32x4*>(static_cast<float*>(p.out) + to) = v;
                } else {
                    *reinterpret_cast<u32x2*>(static_cast<uint16_t*>(p.out) + to) =
                        u32x2{__builtin_bit_cast(uint32_t, bf16x2{static_cast<__bf16>(v[0]), static_cast<__bf16>(v[1])}),
                              __builtin_bit_cast(uint32_t, bf16x2{static_cast<__bf16>(v[2]), static_cast<__bf16>(v[3])})};
                }
            }
        } else {
            const int64_t part = at_row * p.splits + split;
            if (first < last) {
#pragma unroll
                for (int c = 0; c < CT; ++c) *reinterpret_cast<f32x4*>(p.partial + part * R + wave * COLS + 16 * c + 4 * g) = acc[m][c];
            }
            if (wave == 0 && g == 0) {
                float* const stats = p.partial + static_cast<int64_t>(gridDim.x / (p.splits * p.row_blocks)) * p.rows * p.splits * R + part * 2;
                stats[0] = first < last ? top[m] : -INFINITY;
                stats[1] = beyond[m] ? NAN : first < last ? total : 0.0f;
            }
        }
    }
}

// The parts of a row, R / 4 lanes a row.
template <int R, bool F32>
__global__ __launch_bounds__(256) void latent_join_kernel(const float* partial, const float* stats, int64_t rows, int splits, void* out) {
    constexpr int LANES = R / 4;
    const int64_t row = static_cast<int64_t>(blockIdx.x) * (256 / LANES) + threadIdx.x / LANES;
    const int column = threadIdx.x % LANES * 4;
    if (row >= rows) return;
    float top = -INFINITY;
    for (int i = 0; i < splits; ++i) top = fmaxf(top, stats[(row * splits + i) * 2]);
    const float under = finite_or_zero(top);
    f32x4 acc = {0.0f, 0.0f, 0.0f, 0.0f};
    float sum = 0.0f;
    for (int i = 0; i < splits; ++i) {
        const int64_t part = row * splits + i;
        const float by = __builtin_amdgcn_exp2f(stats[part * 2] - under), total = stats[part * 2 + 1];
        if (total == 0.0f) continue;  // nothing seen: its sums may not have been written
        sum = fmaf(total, by, sum);
        const f32x4 v = *reinterpret_cast<const f32x4*>(partial + part * R + column);
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[j] = fmaf(v[j], by, acc[j]);
    }
    const float inverse = sum == 0.0f ? 0.0f : 1.0f / sum;
    acc *= inverse;
    if constexpr (F32) {
        *reinterpret_cast<f32x4*>(static_cast<float*>(out) + row * R + column) = acc;
    } else {
        *reinterpret_cast<u32x2*>(static_cast<uint16_t*>(out) + row * R + column) =
            u32x2{__builtin_bit_cast(uint32_t, bf16x2{static_cast<__bf16>(acc[0]), static_cast<__bf16>(acc[1])}),
                  __builtin_bit_cast(uint32_t, bf16x2{static_cast<__bf16>(acc[2]), static_cast<__bf16>(acc[3])})};
    }
}

struct Plan {
    int tiles;  // of 16 rows a block
    int64_t row_blocks, splits, workspace;
};
// Row tiles a block by the rows a sequence has: the cache is read, and turned into bf16, once for all of them.
Plan plan_of(int64_t batch, int64_t rows, int64_t rank, bool f32, int64_t capacity) {
    Plan plan{};
    plan.tiles = f32 || rows <= 16 ? 1 : rows <= 32 ? 2 : 4;
    plan.row_blocks = ceil_div(rows, 16 * plan.tiles);
    const int64_t blocks = batch * plan.row_blocks, tiles = ceil_div(capacity, kTile);
    plan.splits = std::max<int64_t>(1, std::min<int64_t>(std::min<int64_t>(tiles / 2, 256), ceil_div(512, std::max<int64_t>(blocks, 1))));
    plan.workspace = plan.splits == 1 ? 0 : batch * rows * plan.splits * (rank + 2) * 4;
    return plan;
}

template <int R, int P, bool F32, bool E4M3>
void launch_attention(const LatentAttentionArgs& p, int tiles, int64_t blocks, hipStream_t s) {
    const dim3 grid(static_cast<unsigned>(blocks));
    if constexpr (F32) {
        hipLaunchKernelGGL((latent_attention_kernel<R, P, true, E4M3, 1, 4>), grid, dim3(256), 0, s, p);
    } else {
        if (tiles == 1) hipLaunchKernelGGL((latent_attention_kernel<R, P, false, E4M3, 1, 4>), grid, dim3(256), 0, s, p);
        else if (tiles == 2) hipLaunchKernelGGL((latent_attention_kernel<R, P, false, E4M3, 2, 4>), grid, dim3(256), 0, s, p);
        else if constexpr (R >= 256) hipLaunchKernelGGL((latent_attention_kernel<R, P, false, E4M3, 4, 8>), grid, dim3(512), 0, s, p);
        else hipLaunchKernelGGL((latent_attention_kernel<R, P, false, E4M3, 4, 4>), grid, dim3(256), 0, s, p);
    }
}
template <int R, int P>
void launch_attention(const LatentAttentionArgs& p, bool f32, bool e4m3, int tiles, int64_t blocks, hipStream_t s) {
    if (f32) e4m3 ? launch_attention<R, P, true, true>(p, tiles, blocks, s) : launch_attention<R, P, true, false>(p, tiles, blocks, s);
    else e4m3 ? launch_attention<R, P, false, true>(p, tiles, blocks, s) : launch_attention<R, P, false, false>(p, tiles, blocks, s);
}
template <int R>
void launch_attention(const LatentAttentionArgs& p, int64_t rope, bool f32, bool e4m3, int tiles, int64_t blocks, hipStream_t s) {
    if (rope == 16) launch_attention<R, 16>(p, f32, e4m3, tiles, blocks, s);
    else if (rope == 32) launch_attention<R, 32>(p, f32, e4m3, tiles, blocks, s);
    else launch_attention<R, 64>(p, f32, e4m3, tiles, blocks, s);
    if (p.splits == 1) return;
    const int64_t rows = blocks / p.splits / p.row_blocks * p.rows;
    const float* const stats = p.partial + rows * p.splits * R;
    const dim3 grid(static_cast<unsigned>(ceil_div(rows, 1024 / R)));
    if (f32) hipLaunchKernelGGL((latent_join_kernel<R, true>), grid, dim3(256), 0, s, p.partial, stats, rows, p.splits, p.out);
    else hipLaunchKernelGGL((latent_join_kernel<R, false>), grid, dim3(256), 0, s, p.partial, stats, rows, p.splits, p.out);
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
    p.scale = static_cast<float>(scale * 1.4426950408889634074);
    const int64_t blocks = batch * plan.row_blocks * plan.splits;
    hipStream_t s = reinterpret_cast<hipStream_t>(stream);
    switch (rank) {
        case 64: launch_attention<64>(p, rope_dim, f32, e4m3, plan.tiles, blocks, s); break;
        case 128: launch_attention<128>(p, rope_dim, f32, e4m3, plan.tiles, blocks, s); break;
        case 256: launch_attention<256>(p, rope_dim, f32, e4m3, plan.tiles, blocks, s); break;
        default: launch_attention<512>(p, rope_dim, f32, e4m3, plan.tiles, blocks, s); break;
    }
    return launch_status("latent attention");
}
