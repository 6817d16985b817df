// Every head's own matrix times its part of the activations: y[t, h] = W[h] x[t, h], the products that take an MLA layer's
// queries into the latents' space and its attended latents back to the heads' values. W is dense along its inputs or along
// its outputs, so that both products read the same projection's rows.
//
// Products have the outputs as rows and the tokens as columns, so that a lane ends with runs of outputs of one token. Sums are
// fp32, and rounded once.
#include <algorithm>
#include <type_traits>

#include "fp4.h"

namespace mlk {
namespace {

struct HeadArgs {
    const void *x, *w;
    void* y;
    int64_t xs_token, xs_head, ws_head, ws_out, ws_in;
    int64_t tokens, chunk;  // chunk: tokens of a block
    int32_t heads, k, n;
};

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef short i16x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef u32x2 u32x2_any __attribute__((aligned(2)));

// The unit of a block: blocks of one die (every eighth) take neighbouring units, which read the same weights or tokens.
__device__ __forceinline__ unsigned unit_of(unsigned units) { return blockIdx.x % 8 * ((units + 7) / 8) + blockIdx.x / 8; }

// Eight elements from k of a row of `count`, zeros behind it.
__device__ __forceinline__ u32x4 eight(const uint16_t* row, int k, int count) {
    u32x4 v = {0, 0, 0, 0};
    if (k + 8 <= count) {
        v = *reinterpret_cast<const u32x4_any*>(row + k);
    } else if (k < count) {
        for (int i = 0; i < count - k; ++i) v[i / 2] |= static_cast<uint32_t>(row[k + i]) << (16 * (i & 1));
    }
    return v;
}

constexpr int kBatch = 8, kTurn = 40;  // steps turned at a time; bf16 elements of a row of 32 in LDS: 20 dwords, four rows on other banks

// A wave's weights of 32 outputs from n and KS steps of 16 inputs from k, zeros behind the last input. IN_DENSE: W's rows are
// dense along the inputs and are operands as they lie; else 16 inputs x 32 outputs at a time go through LDS (`turn`, the
// wave's own) and are turned as they are read.
template <int KS, bool IN_DENSE>
__device__ __forceinline__ void load_weights(bf16x8 (&w)[KS], const HeadArgs& p, int64_t head, int n, int k, uint16_t* turn) {
    constexpr int BATCH = KS < kBatch ? KS : kBatch;
    const int lane = threadIdx.x & 63, h = lane >> 5, l = lane & 31;
    const uint16_t* const w0 = static_cast<const uint16_t*>(p.w) + head * p.ws_head;
    if constexpr (IN_DENSE) {
        const uint16_t* const row = w0 + static_cast<int64_t>(min(n + l, p.n - 1)) * p.ws_out;
#pragma unroll
        for (int s = 0; s < KS; ++s) w[s] = __builtin_bit_cast(bf16x8, eight(row, k + 16 * s + 8 * h, p.k));
    } else {
        const int k_of = lane >> 2, n_of = (lane & 3) * 8;  // a lane's piece of 16 inputs x 32 outputs
#pragma unroll
        for (int s0 = 0; s0 < KS; s0 += BATCH) {
            u32x4 v[BATCH];
#pragma unroll
            for (int s = 0; s < BATCH; ++s) {
                const int row = k + 16 * (s0 + s) + k_of;
                v[s] = eight(w0 + static_cast<int64_t>(min(row, p.k - 1)) * p.ws_in, n + n_of, row < p.k ? p.n : 0);
            }
#pragma unroll
            for (int s = 0; s < BATCH; ++s) *reinterpret_cast<u32x4*>(turn + (16 * s + k_of) * kTurn + n_of) = v[s];
            __builtin_amdgcn_wave_barrier();
#pragma unroll
            for (int s = 0; s < BATCH; ++s) {
                i16x4 x[2];
#pragma unroll
                for (int i = 0; i < 2; ++i)
                    x[i] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) i16x4*)(
                        turn + (16 * s + 8 * h + 4 * i + (lane >> 2 & 3)) * kTurn + 16 * (lane >> 4 & 1) + 4 * (lane & 3)));
                w[s0 + s] = __builtin_bit_cast(bf16x8, __builtin_shufflevector(x[0], x[1], 0, 1, 2, 3, 4, 5, 6, 7));
            }
            __builtin_amdgcn_wave_barrier();
        }
    }
}

// The 32 outputs from n of a lane's token. Register i holds output 8 (i / 4) + 4 h + i % 4: the halves exchange four each, so
// that each has eight in a row.
__device__ __forceinline__ void store_outputs(const HeadArgs& p, const f32x16& acc, int64_t head, int64_t token, bool in, int n) {
    const int h = (threadIdx.x & 63) >> 5;
    uint16_t* const y = static_cast<uint16_t*>(p.y) + (token * p.heads + head) * p.n;
#pragma unroll
    for (int g = 0; g < 2; ++g) {
        uint32_t a[2], b[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int r = 8 * g + 2 * i;
            a[i] = __builtin_bit_cast(uint32_t, bf16x2{static_cast<__bf16>(acc[r]), static_cast<__bf16>(acc[r + 1])});
            b[i] = __builtin_bit_cast(uint32_t, bf16x2{static_cast<__bf16>(acc[r + 4]), static_cast<__bf16>(acc[r + 5])});
            const auto swapped = __builtin_amdgcn_permlane32_swap(a[i], b[i], false, false);
            a[i] = swapped[0];
            b[i] = swapped[1];
        }
        const int at = n + 16 * g + 8 * h;
        const u32x4 v = {a[0], a[1], b[0], b[1]};
        if (!in || at >= p.n) continue;
        if (at + 8 <= p.n) {
            *reinterpret_cast<u32x4_any*>(y + at) = v;
        } else {
            for (int i = 0; i < p.n - at; ++i) y[at + i] = static_cast<uint16_t>(v[i / 2] >> (16 * (i & 1)));
        }
    }
}

// bf16 in and out, many tokens. A wave's weights, of NT x 32 outputs and all inputs, are kept in registers and read once; the
// tokens of all waves go through LDS, the next 32 being loaded while these are multiplied.
//
// Bound by memory: 512 outputs of 128 inputs make 51 operations a byte. 4096 tokens of 64 heads take 140 us (W dense along its
// inputs) or 122 with 512 outputs of 128 inputs, 91 with 128 of 512: 2.4, 2.8 and 3.7 TB/s (210 and 275 with each wave reading
// the tokens by itself, 32 bytes of a row a load). The form for more than 256 inputs takes all 256 registers of a lane, and two
// (W dense along its outputs) or four more in scratch memory.
template <int KS, int NT, bool IN_DENSE>
__global__ __launch_bounds__(256, 2) void head_linear_kernel(HeadArgs p, unsigned n_blocks, unsigned chunks, unsigned blocks) {
    constexpr int ROW = KS * 16 + 8, PIECES = 64 * KS, EACH = (PIECES + 255) / 256;
    constexpr int TURN = (KS < kBatch ? KS : kBatch) * 16 * kTurn, TURNED = IN_DENSE ? 0 : 4 * TURN, TOKENS = 2 * 32 * ROW;
    __shared__ __attribute__((aligned(16))) uint16_t shared[TURNED > TOKENS ? TURNED : TOKENS];
    const unsigned id = unit_of(blocks);
    if (id >= blocks) return;
    const int wave = threadIdx.x / 64, lane = threadIdx.x & 63, h = lane >> 5, l = lane & 31;
    const unsigned nb = id % n_blocks, rest = id / n_blocks, chunk = rest % chunks, head = rest / chunks;
    const int n0 = (static_cast<int>(nb) * 4 + wave) * (NT * 32);
    const int64_t begin = static_cast<int64_t>(chunk) * p.chunk, end = min(begin + p.chunk, p.tokens);
    const uint16_t* const x0 = static_cast<const uint16_t*>(p.x) + head * p.xs_head;
    u32x4 next[EACH];
    auto load = [&](int64_t t0) {
#pragma unroll
        for (int i = 0; i < EACH; ++i) {
            const int piece = threadIdx.x + i * 256;
            next[i] = eight(x0 + min(t0 + piece / (2 * KS), end - 1) * p.xs_token, piece % (2 * KS) * 8, p.k);
        }
    };
    load(begin);
    bf16x8 w[NT][KS];
#pragma unroll
    for (int a = 0; a < NT; ++a) load_weights<KS, IN_DENSE>(w[a], p, head, n0 + 32 * a, 0, shared + wave * TURN);
    if constexpr (!IN_DENSE) __syncthreads();  // the tokens take the same LDS
    int half = 0;
    for (int64_t t0 = begin; t0 < end; t0 += 32, half ^= 1) {
        uint16_t* const xs = shared + half * (32 * ROW);
#pragma unroll
        for (int i = 0; i < EACH; ++i) {
            const int piece = threadIdx.x + i * 256;
            if (piece < PIECES) *reinterpret_cast<u32x4*>(xs + piece / (2 * KS) * ROW + piece % (2 * KS) * 8) = next[i];
        }
        __syncthreads();  // one a tile: a wave writes a half again only behind the next barrier, which follows its readers' products
        if (t0 + 32 < end) load(t0 + 32);
        f32x16 acc[NT] = {};
#pragma unroll
        for (int s = 0; s < KS; ++s) {
            const bf16x8 x = *reinterpret_cast<const bf16x8*>(xs + l * ROW + 16 * s + 8 * h);
#pragma unroll
            for (int a = 0; a < NT; ++a) acc[a] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(w[a][s], x, acc[a], 0, 0, 0);
        }
#pragma unroll
        for (int a = 0; a < NT; ++a) store_outputs(p, acc[a], head, t0 + l, t0 + l < end, n0 + 32 * a);
    }
}

// bf16 in and out, few tokens: 32 tokens x 32 outputs a block, whose WAVES waves take KS steps of the inputs each; the first
// adds their sums in order.
//
// Bound by latency, one load of everything and a store: 24 tokens of 64 heads, 512 outputs of 128 inputs, 4.1 us a call (10 MB
// at 5 TB/s are 2.1); with 512 inputs 4.5 to 5.4 (7.7 to 9.6 where one wave takes all of them).
template <int KS, int WAVES, bool IN_DENSE>
__global__ __launch_bounds__(WAVES * 64) void head_linear_few_kernel(HeadArgs p, unsigned n_blocks, unsigned chunks, unsigned blocks) {
    constexpr int TURN = (KS < kBatch ? KS : kBatch) * 16 * kTurn, TURNED = IN_DENSE ? 0 : WAVES * TURN, PARTS = (WAVES - 1) * 64 * 40;
    __shared__ __attribute__((aligned(16))) uint16_t shared[TURNED > PARTS ? TURNED : PARTS > 0 ? PARTS : 8];
    const unsigned id = unit_of(blocks);
    if (id >= blocks) return;
    const int wave = threadIdx.x / 64, lane = threadIdx.x & 63, h = lane >> 5, l = lane & 31;
    const unsigned nb = id % n_blocks, rest = id / n_blocks, chunk = rest % chunks, head = rest / chunks;
    const int n0 = static_cast<int>(nb) * 32, k0 = wave * (KS * 16);
    const int64_t t = static_cast<int64_t>(chunk) * 32 + l;
    const uint16_t* const x = static_cast<const uint16_t*>(p.x) + head * p.xs_head + min(t, p.tokens - 1) * p.xs_token;
    u32x4 xv[KS];
#pragma unroll
    for (int s = 0; s < KS; ++s) xv[s] = eight(x, k0 + 16 * s + 8 * h, p.k);
    bf16x8 w[KS];
    load_weights<KS, IN_DENSE>(w, p, head, n0, k0, shared + wave * TURN);
    f32x16 acc = {};
#pragma unroll
    for (int s = 0; s < KS; ++s) acc = __builtin_amdgcn_mfma_f32_32x32x16_bf16(w[s], __builtin_bit_cast(bf16x8, xv[s]), acc, 0, 0, 0);
    if constexpr (WAVES > 1) {
        float* const parts = reinterpret_cast<float*>(shared) + lane * 20;
        if constexpr (!IN_DENSE) __syncthreads();  // the parts take the turned weights' LDS
        if (wave > 0) {
#pragma unroll
            for (int i = 0; i < 16; i += 4) *reinterpret_cast<f32x4*>(parts + (wave - 1) * (64 * 20) + i) = f32x4{acc[i], acc[i + 1], acc[i + 2], acc[i + 3]};
        }
        __syncthreads();
        if (wave > 0) return;
#pragma unroll
        for (int from = 0; from < WAVES - 1; ++from)
#pragma unroll
            for (int i = 0; i < 16; i += 4) {
                const f32x4 v = *reinterpret_cast<const f32x4*>(parts + from * (64 * 20) + i);
#pragma unroll
                for (int j = 0; j < 4; ++j) acc[i + j] += v[j];
            }
    }
    store_outputs(p, acc, head, t, t < p.tokens, n0);
}

// Four elements from k of a row of `count`, zeros behind it: as they are stored, and as numbers.
__device__ __forceinline__ u32x4 four(const float* row, int k, int count) {
    u32x4 v = {0, 0, 0, 0};
    if (k + 4 <= count) {
        v = *reinterpret_cast<const u32x4_any*>(row + k);
    } else {
#pragma unroll
        for (int i = 0; i < 3; ++i)
            if (k + i < count) v[i] = __builtin_bit_cast(uint32_t, row[k + i]);
    }
    return v;
}
__device__ __forceinline__ u32x2 four(const uint16_t* row, int k, int count) {
    u32x2 v = {0, 0};
    if (k + 4 <= count) {
        v = *reinterpret_cast<const u32x2_any*>(row + k);
    } else {
#pragma unroll
        for (int i = 0; i < 3; ++i)
            if (k + i < count) v[i / 2] |= static_cast<uint32_t>(row[k + i]) << (16 * (i & 1));
    }
    return v;
}
__device__ __forceinline__ u32x4 numbers(u32x4 v) { return v; }
__device__ __forceinline__ u32x4 numbers(u32x2 v) { return u32x4{v[0] << 16, v[0] & 0xffff0000u, v[1] << 16, v[1] & 0xffff0000u}; }

// fp32 in and out, weights of either type, on the fp32 matrix cores (16 x 16 x 4): products are exact and sums fp32. A block
// of four waves brings TILE tokens and TILE outputs to LDS, TK inputs at a time, the next being loaded while these are
// multiplied. A wave makes 32 tokens x 32 outputs; its lane holds four inputs, 4 g .. 4 g + 3 of a step of 16, and product j
// takes the j-th of each.
//
// SPLIT: all waves make the same 32 x 32, from a quarter of the inputs each, and the first adds the four in order; else each
// makes a quarter of 64 x 64. One half of LDS is enough to split, where the sixth block on a compute unit is worth more.
//
// Bound by the fp32 products: 600 tokens of 24 heads, 96 outputs of 512 inputs, take 21 us (9.2 at the 154 TFLOP/s of a large
// fp32 product; 31 with operands read from memory lane by lane, 16 rows a load), 4096 tokens of 64 heads, 512 of 128, 365 us,
// 94 TFLOP/s. Both types of weights take the same.
template <bool W32, bool IN_DENSE, bool SPLIT>
__global__ __launch_bounds__(256, SPLIT ? 6 : 4) void head_linear_f32_kernel(HeadArgs p, unsigned n_blocks, unsigned chunks, unsigned blocks) {
    constexpr int TILE = SPLIT ? 32 : 64, TK = SPLIT ? 64 : 32, STEPS = SPLIT ? 1 : 2;
    // Rows of x and of an IN_DENSE w hold TK inputs, else those of w TILE outputs; with 4 more, rows that are read together
    // (16 of 16 bytes, or every fourth) lie on other banks.
    constexpr int X_ROW = TK + 4, W_ROW = IN_DENSE ? TK + 4 : TILE + 4, W_SIZE = IN_DENSE ? TILE * W_ROW : TK * W_ROW;
    __shared__ __attribute__((aligned(16))) float shared[SPLIT ? 1 : 2][TILE * X_ROW + W_SIZE];
    static_assert(sizeof shared >= 3 * 64 * 20 * sizeof(float), "the waves' parts take the same LDS");
    const unsigned id = unit_of(blocks);
    if (id >= blocks) return;
    const int thread = threadIdx.x, wave = thread / 64, lane = thread & 63, g = lane >> 4, l = lane & 15;
    const unsigned nb = id % n_blocks, rest = id / n_blocks, chunk = rest % chunks, head = rest / chunks;
    const int n0 = static_cast<int>(nb) * TILE;
    const int64_t begin = static_cast<int64_t>(chunk) * p.chunk, end = min(begin + p.chunk, p.tokens);
    using Weight = std::conditional_t<W32, float, uint16_t>;
    const float* const x = static_cast<const float*>(p.x) + head * p.xs_head;
    const Weight* const w = static_cast<const Weight*>(p.w) + head * p.ws_head;
    constexpr int X_PIECES = TK / 4, W_PIECES = IN_DENSE ? TK / 4 : TILE / 4;  // of a row; a thread takes two pieces of each
    u32x4 next_x[2];
    std::conditional_t<W32, u32x4, u32x2> next_w[2];
    auto load = [&](int64_t t0, int k0) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int at = thread + 256 * i, row = at / W_PIECES, piece = at % W_PIECES * 4;
            next_x[i] = four(x + min(t0 + at / X_PIECES, end - 1) * p.xs_token, k0 + at % X_PIECES * 4, p.k);
            if constexpr (IN_DENSE) next_w[i] = four(w + static_cast<int64_t>(min(n0 + row, p.n - 1)) * p.ws_out, k0 + piece, p.k);
            else next_w[i] = four(w + static_cast<int64_t>(min(k0 + row, p.k - 1)) * p.ws_in, n0 + piece, k0 + row < p.k ? p.n : 0);
        }
    };
    f32x4 acc[2][2] = {};  // [outputs][tokens]
    const int at_t = (SPLIT ? 0 : wave / 2 * 32) + l, at_n = (SPLIT ? 0 : wave % 2 * 32) + l, at_k = (SPLIT ? 16 * wave : 0) + 4 * g;
    load(begin, 0);
    int half = 0;
    for (int64_t t0 = begin; t0 < end; t0 += TILE) {
        for (int k0 = 0; k0 < p.k; k0 += TK, half ^= !SPLIT) {
            if (SPLIT && k0 > 0) __syncthreads();
            float* const xs = shared[half];
            float* const ws = xs + TILE * X_ROW;
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const int at = thread + 256 * i;
                *reinterpret_cast<u32x4*>(xs + at / X_PIECES * X_ROW + at % X_PIECES * 4) = next_x[i];
                *reinterpret_cast<u32x4*>(ws + at / W_PIECES * W_ROW + at % W_PIECES * 4) = numbers(next_w[i]);
            }
            __syncthreads();  // one a tile: a wave writes a half again only behind the next barrier, which follows its readers' products
            if (k0 + TK < p.k) load(t0, k0 + TK);
            else if (!SPLIT && t0 + TILE < end) load(t0 + TILE, 0);
#pragma unroll
            for (int s = 0; s < STEPS; ++s) {
                const int k = at_k + 16 * s;
                f32x4 xv[2], wv[2];
#pragma unroll
                for (int m = 0; m < 2; ++m) {
                    xv[m] = *reinterpret_cast<const f32x4*>(xs + (at_t + 16 * m) * X_ROW + k);
                    if constexpr (IN_DENSE) {
                        wv[m] = *reinterpret_cast<const f32x4*>(ws + (at_n + 16 * m) * W_ROW + k);
                    } else {
#pragma unroll
                        for (int j = 0; j < 4; ++j) wv[m][j] = ws[(k + j) * W_ROW + at_n + 16 * m];
                    }
                }
#pragma unroll
                for (int j = 0; j < 4; ++j)
#pragma unroll
                    for (int a = 0; a < 2; ++a)
#pragma unroll
                        for (int b = 0; b < 2; ++b) acc[a][b] = __builtin_amdgcn_mfma_f32_16x16x4f32(wv[a][j], xv[b][j], acc[a][b], 0, 0, 0);
            }
        }
        if constexpr (SPLIT) {
            float* const parts = shared[0] + lane * 20;
            __syncthreads();
            if (wave > 0) {
#pragma unroll
                for (int i = 0; i < 4; ++i) *reinterpret_cast<f32x4*>(parts + (wave - 1) * (64 * 20) + 4 * i) = acc[i / 2][i % 2];
            }
            __syncthreads();
            if (wave > 0) return;
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int from = 0; from < 3; ++from) acc[i / 2][i % 2] += *reinterpret_cast<const f32x4*>(parts + from * (64 * 20) + 4 * i);
        }
#pragma unroll
        for (int b = 0; b < 2; ++b) {
            const int64_t t = t0 + at_t + 16 * b;
            float* const y = static_cast<float*>(p.y) + (t * p.heads + head) * p.n;
#pragma unroll
            for (int a = 0; a < 2; ++a) {
                const int n = n0 + at_n - l + 16 * a + 4 * g;
                const f32x4 v = acc[a][b];
                acc[a][b] = f32x4{};
                if (t >= end) continue;
                if (n + 4 <= p.n) {
                    *reinterpret_cast<u32x4_any*>(y + n) = __builtin_bit_cast(u32x4, v);
                } else {
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        if (n + i < p.n) y[n + i] = v[i];
                }
            }
        }
        if constexpr (SPLIT) break;
    }
}

// bf16 with more inputs than a wave's registers hold (above 512): 32 tokens x 32 outputs a block on the vector units.
__global__ __launch_bounds__(256) void head_linear_any_kernel(HeadArgs p, unsigned token_tiles, unsigned n_tiles) {
    __shared__ float xs[32][33], ws[32][33];
    const unsigned id = blockIdx.x, tile = id % token_tiles, rest = id / token_tiles, nt = rest % n_tiles, head = rest / n_tiles;
    const int64_t t0 = static_cast<int64_t>(tile) * 32;
    const int n0 = nt * 32, a = threadIdx.x % 32, b = threadIdx.x / 32;
    float sum[4] = {};
    for (int k0 = 0; k0 < p.k; k0 += 32) {
        for (int i = b; i < 32; i += 8) {
            const bool in = t0 + i < p.tokens && k0 + a < p.k;
            xs[i][a] = in ? Element<false>::get(p.x, (t0 + i) * p.xs_token + head * p.xs_head + k0 + a) : 0.0f;
            const int n = p.ws_in == 1 ? i : a, k = p.ws_in == 1 ? a : i;
            const bool has = n0 + n < p.n && k0 + k < p.k;
            ws[n][k] = has ? Element<false>::get(p.w, head * p.ws_head + (n0 + n) * p.ws_out + (k0 + k) * p.ws_in) : 0.0f;
        }
        __syncthreads();
        for (int k = 0; k < 32; ++k)
#pragma unroll
            for (int i = 0; i < 4; ++i) sum[i] = fmaf(xs[b + 8 * i][k], ws[a][k], sum[i]);
        __syncthreads();
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int64_t t = t0 + b + 8 * i;
        if (t < p.tokens && n0 + a < p.n) Element<false>::put(p.y, (t * p.heads + head) * p.n + n0 + a, sum[i]);
    }
}

constexpr int kChip = 256;  // compute units

dim3 grid_of(unsigned blocks) { return dim3((blocks + 7) / 8 * 8); }

// Cuts the tokens into pieces of whole tiles, as many as make `blocks` blocks of `units` a piece.
unsigned cut(HeadArgs& p, int64_t tile, int64_t units, int64_t blocks) {
    const int64_t tiles = ceil_div(p.tokens, tile), pieces = std::min(tiles, std::max<int64_t>(1, ceil_div(blocks, units)));
    p.chunk = ceil_div(tiles, pieces) * tile;
    return static_cast<unsigned>(ceil_div(p.tokens, p.chunk));
}

template <int KS>
void launch_bf16(HeadArgs p, hipStream_t s) {
    constexpr int NT = KS > 8 ? 1 : 2;
    const bool in_dense = p.ws_in == 1;
    // A block of many tokens reads its weights once for all of them; up to four such a compute unit, at least one: of 456
    // blocks (600 tokens of 24 heads, 512 -> 96) 10.8 us against 13.4 in tiles of few tokens, of 256 (64 of 64 heads, 128 ->
    // 512) 5.6 against 6.6, of 160 (300 of 16 heads, 512 -> 128) 8.0 against 7.8.
    const unsigned wide = static_cast<unsigned>(ceil_div(p.n, 128 * NT)), chunks = cut(p, 32, p.heads * wide, 4 * kChip);
    if (const unsigned blocks = p.heads * wide * chunks; blocks >= kChip) {
        if (in_dense) hipLaunchKernelGGL((head_linear_kernel<KS, NT, true>), grid_of(blocks), dim3(256), 0, s, p, wide, chunks, blocks);
        else hipLaunchKernelGGL((head_linear_kernel<KS, NT, false>), grid_of(blocks), dim3(256), 0, s, p, wide, chunks, blocks);
    } else {
        constexpr int WAVES = KS > 8 ? 4 : 1, EACH = KS / WAVES;
        const unsigned n_blocks = static_cast<unsigned>(ceil_div(p.n, 32)), tiles = static_cast<unsigned>(ceil_div(p.tokens, 32));
        const unsigned few = p.heads * n_blocks * tiles;
        if (in_dense) hipLaunchKernelGGL((head_linear_few_kernel<EACH, WAVES, true>), grid_of(few), dim3(WAVES * 64), 0, s, p, n_blocks, tiles, few);
        else hipLaunchKernelGGL((head_linear_few_kernel<EACH, WAVES, false>), grid_of(few), dim3(WAVES * 64), 0, s, p, n_blocks, tiles, few);
    }
}

template <bool W32>
void launch_f32(HeadArgs p, hipStream_t s) {
    auto launch = [&](auto split) {
        constexpr bool SPLIT = decltype(split)::value;
        constexpr int TILE = SPLIT ? 32 : 64;
        const unsigned n_blocks = static_cast<unsigned>(ceil_div(p.n, TILE)), chunks = cut(p, TILE, p.heads * n_blocks, SPLIT ? 1 << 30 : 8 * kChip);
        const unsigned blocks = p.heads * n_blocks * chunks;
        if (p.ws_in == 1) hipLaunchKernelGGL((head_linear_f32_kernel<W32, true, SPLIT>), grid_of(blocks), dim3(256), 0, s, p, n_blocks, chunks, blocks);
        else hipLaunchKernelGGL((head_linear_f32_kernel<W32, false, SPLIT>), grid_of(blocks), dim3(256), 0, s, p, n_blocks, chunks, blocks);
    };
    // Tiles of 32 x 32 that give every SIMD two waves are not split: 2048 tiles (64 tokens of 64 heads, 128 -> 512) take 9.4 us,
    // split 11.1; 1368 (600 tokens of 24 heads, 512 -> 96) 24.7, split 21.6; 640 (300 of 16, 512 -> 128) 16.2, split 12.0.
    if (p.heads * ceil_div(p.n, 32) * ceil_div(p.tokens, 32) >= 8 * kChip) launch(std::false_type{});
    else launch(std::true_type{});
}

}  // namespace
}  // namespace mlk

using namespace mlk;

extern "C" mlk_status mlk_head_linear(const void* x, int64_t tokens, int64_t heads, int64_t in_features, const int64_t* x_strides, int32_t dtype,
                                      const void* weight, const int64_t* weight_strides, int32_t weight_dtype, int64_t out_features, void* out,
                                      mlk_stream_t stream) {
    MLK_CHECK(dtype == MLK_DTYPE_F32 || dtype == MLK_DTYPE_BF16, "dtype must be f32 or bf16");
    MLK_CHECK(weight_dtype == MLK_DTYPE_BF16 || (weight_dtype == MLK_DTYPE_F32 && dtype == MLK_DTYPE_F32), "the weight must be bf16, or f32 with f32 input");
    MLK_CHECK(tokens >= 0 && heads > 0 && in_features > 0 && out_features > 0, "invalid head_linear geometry");
    MLK_CHECK(heads < (int64_t{1} << 20) && in_features < (int64_t{1} << 20) && out_features < (int64_t{1} << 20), "head_linear: heads and features must be below 2^20");
    MLK_CHECK(tokens < (int64_t{1} << 31), "too many tokens");
    const int64_t token_tiles = ceil_div(tokens, 32), n_tiles = ceil_div(out_features, 32);
    MLK_CHECK(token_tiles < (int64_t{1} << 23) / heads / n_tiles, "too many tokens for one launch");  // of 256 threads a tile: below 2^32
    if (tokens == 0) return MLK_OK;
    MLK_CHECK(x && x_strides && weight && weight_strides && out, "null tensor pointer");
    MLK_CHECK(weight_strides[1] == 1 || weight_strides[2] == 1, "the weight must be dense along its inputs or its outputs");
    MLK_CHECK((reinterpret_cast<uintptr_t>(out) & 15) == 0, "out must be 16-byte aligned");
    const HeadArgs p{x, weight, out, x_strides[0], x_strides[1], weight_strides[0], weight_strides[1], weight_strides[2], tokens, 0,
                     static_cast<int32_t>(heads), static_cast<int32_t>(in_features), static_cast<int32_t>(out_features)};
    hipStream_t s = reinterpret_cast<hipStream_t>(stream);
    if (dtype == MLK_DTYPE_F32) {
        weight_dtype == MLK_DTYPE_F32 ? launch_f32<true>(p, s) : launch_f32<false>(p, s);
    } else if (in_features <= 32) {
        launch_bf16<2>(p, s);
    } else if (in_features <= 64) {
        launch_bf16<4>(p, s);
    } else if (in_features <= 128) {
        launch_bf16<8>(p, s);
    } else if (in_features <= 256) {
        launch_bf16<16>(p, s);
    } else if (in_features <= 512) {
        launch_bf16<32>(p, s);
    } else {
        hipLaunchKernelGGL(head_linear_any_kernel, dim3(static_cast<unsigned>(token_tiles * n_tiles * heads)), dim3(256), 0, s, p,
                           static_cast<unsigned>(token_tiles), static_cast<unsigned>(n_tiles));
    }
    return launch_status("head linear");
}
