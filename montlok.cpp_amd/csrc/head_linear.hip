// Every head's own matrix times its part of the activations: y[t, h] = W[h] x[t, h], the products that take an MLA layer's
// queries into the latents' space and its attended latents back to the heads' values. W is dense along its inputs or along
// its outputs, so that both products read the same projection's rows.
//
// A wave takes 32 outputs of a head and goes over tokens, 32 (or 64) at a time: products have the outputs as rows and the
// tokens as columns, so that a lane ends with runs of outputs of one token. All waves of a block read the same tokens.
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

// bf16 in and out. The wave's weights are kept in registers, KS steps of 16 inputs (zeros behind the last), and read once.
// IN_DENSE: W's rows are dense along the inputs and are operands as they lie; else 16 inputs x 32 outputs at a time go
// through LDS and are turned as they are read.
//
// Bound by memory: 512 outputs of 128 inputs make 51 operations a byte of weights and activations.
template <int KS, bool IN_DENSE, int WAVES>
__global__ __launch_bounds__(WAVES * 64) void head_linear_kernel(HeadArgs p, unsigned n_blocks, unsigned chunks) {
    constexpr int BATCH = KS < 8 ? KS : 8, PITCH = 40;  // bf16 elements of a row of 32 in LDS: 20 dwords, four rows on other banks
    __shared__ __attribute__((aligned(16))) uint16_t turned[IN_DENSE ? 1 : WAVES][IN_DENSE ? 8 : BATCH * 16 * PITCH];
    const int wave = threadIdx.x / 64, lane = threadIdx.x & 63, h = lane >> 5, l = lane & 31;
    const unsigned id = blockIdx.x, chunk = id % chunks, rest = id / chunks, nb = rest % n_blocks, head = rest / n_blocks;
    const int n0 = static_cast<int>(nb) * (WAVES * 32) + wave * 32;
    const uint16_t* const w0 = static_cast<const uint16_t*>(p.w) + head * p.ws_head;
    bf16x8 w[KS];
    if constexpr (IN_DENSE) {
        const uint16_t* const row = w0 + static_cast<int64_t>(min(n0 + l, p.n - 1)) * p.ws_out;
#pragma unroll
        for (int s = 0; s < KS; ++s) {
            const int k = 16 * s + 8 * h;
            u32x4 v = {0, 0, 0, 0};
            if (k + 8 <= p.k) {
                v = *reinterpret_cast<const u32x4_any*>(row + k);
            } else if (k < p.k) {
                for (int i = 0; i < p.k - k; ++i) v[i / 2] |= static_cast<uint32_t>(row[k + i]) << (16 * (i & 1));
            }
            w[s] = __builtin_bit_cast(bf16x8, v);
        }
    } else {
        uint16_t* const mine = turned[wave];
        const int k_of = lane >> 2, n_of = (lane & 3) * 8;  // a lane's piece of 16 inputs x 32 outputs
#pragma unroll
        for (int s0 = 0; s0 < KS; s0 += BATCH) {
            u32x4 v[BATCH];
#pragma unroll
            for (int s = 0; s < BATCH; ++s) {
                const int k = 16 * (s0 + s) + k_of, n = n0 + n_of;
                const uint16_t* const at = w0 + static_cast<int64_t>(min(k, p.k - 1)) * p.ws_in + n;
                v[s] = u32x4{0, 0, 0, 0};
                if (k < p.k) {
                    if (n + 8 <= p.n) {
                        v[s] = *reinterpret_cast<const u32x4_any*>(at);
                    } else {
                        for (int i = 0; i < p.n - n; ++i) v[s][i / 2] |= static_cast<uint32_t>(at[i]) << (16 * (i & 1));
                    }
                }
            }
#pragma unroll
            for (int s = 0; s < BATCH; ++s) *reinterpret_cast<u32x4*>(mine + (16 * s + k_of) * PITCH + n_of) = v[s];
            __builtin_amdgcn_wave_barrier();
#pragma unroll
            for (int s = 0; s < BATCH; ++s) {
                i16x4 x[2];
#pragma unroll
                for (int i = 0; i < 2; ++i)
                    x[i] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) i16x4*)(
                        mine + (16 * s + 8 * h + 4 * i + (lane >> 2 & 3)) * PITCH + 16 * (lane >> 4 & 1) + 4 * (lane & 3)));
                w[s0 + s] = __builtin_bit_cast(bf16x8, __builtin_shufflevector(x[0], x[1], 0, 1, 2, 3, 4, 5, 6, 7));
            }
            __builtin_amdgcn_wave_barrier();
        }
    }
    const uint16_t* const x0 = static_cast<const uint16_t*>(p.x) + head * p.xs_head;
    const int64_t end = min((static_cast<int64_t>(chunk) + 1) * p.chunk, p.tokens);
    for (int64_t t0 = static_cast<int64_t>(chunk) * p.chunk; t0 < end; t0 += 32) {
        const int64_t t = t0 + l;
        const uint16_t* const x = x0 + min(t, end - 1) * p.xs_token;
        f32x16 acc = {};
#pragma unroll
        for (int s = 0; s < KS; ++s) {
            const int k = 16 * s + 8 * h;
            u32x4 v = {0, 0, 0, 0};
            if (k + 8 <= p.k) {
                v = *reinterpret_cast<const u32x4_any*>(x + k);
            } else if (k < p.k) {
                for (int i = 0; i < p.k - k; ++i) v[i / 2] |= static_cast<uint32_t>(x[k + i]) << (16 * (i & 1));
            }
            acc = __builtin_amdgcn_mfma_f32_32x32x16_bf16(w[s], __builtin_bit_cast(bf16x8, v), acc, 0, 0, 0);
        }
        // Register i holds output 8 (i / 4) + 4 h + i % 4: the halves exchange four each, so that each has eight in a row.
        uint16_t* const y = static_cast<uint16_t*>(p.y) + (t * p.heads + head) * p.n;
#pragma unroll
        for (int g = 0; g < 2; ++g) {
            uint32_t a[2], b[2];
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                a[i] = __builtin_bit_cast(uint32_t, bf16x2{static_cast<__bf16>(acc[8 * g + 2 * i]), static_cast<__bf16>(acc[8 * g + 2 * i + 1])});
                b[i] = __builtin_bit_cast(uint32_t, bf16x2{static_cast<__bf16>(acc[8 * g + 4 + 2 * i]), static_cast<__bf16>(acc[8 * g + 5 + 2 * i])});
                const auto swapped = __builtin_amdgcn_permlane32_swap(a[i], b[i], false, false);
                a[i] = swapped[0];
                b[i] = swapped[1];
            }
            const int n = n0 + 16 * g + 8 * h;
            const u32x4 v = {a[0], a[1], b[0], b[1]};
            if (t >= end || n >= p.n) continue;
            if (n + 8 <= p.n) {
                *reinterpret_cast<u32x4_any*>(y + n) = v;
            } else {
                for (int i = 0; i < p.n - n; ++i) y[n + i] = static_cast<uint16_t>(v[i / 2] >> (16 * (i & 1)));
            }
        }
    }
}

// fp32 in and out, weights of either type, on the fp32 matrix cores (32 x 32 x 2): products are exact and sums fp32. A lane
// holds four inputs, 4 h .. 4 h + 3 of a step of 8, and product j takes the j-th of each. Two tiles of 32 tokens a wave, the
// next step's operands asked for before a step's products; weights are read again for every 64 tokens.
template <bool W32, bool IN_DENSE, int WAVES>
__global__ __launch_bounds__(WAVES * 64, 2) void head_linear_f32_kernel(HeadArgs p, unsigned n_blocks, unsigned chunks) {
    const int wave = threadIdx.x / 64, lane = threadIdx.x & 63, h = lane >> 5, l = lane & 31;
    const unsigned id = blockIdx.x, chunk = id % chunks, rest = id / chunks, nb = rest % n_blocks, head = rest / n_blocks;
    const int n0 = static_cast<int>(nb) * (WAVES * 32) + wave * 32;
    using Weight = std::conditional_t<W32, float, uint16_t>;
    const Weight* const w = static_cast<const Weight*>(p.w) + head * p.ws_head + static_cast<int64_t>(min(n0 + l, p.n - 1)) * p.ws_out;
    const int64_t t0 = static_cast<int64_t>(chunk) * 64;
    const float* x[2];
#pragma unroll
    for (int m = 0; m < 2; ++m) x[m] = static_cast<const float*>(p.x) + head * p.xs_head + min(t0 + 32 * m + l, p.tokens - 1) * p.xs_token;
    auto number = [](Weight v) {
        if constexpr (W32) return v;
        else return bf16_to_float(v);
    };
    struct Step {
        f32x4 w, x[2];
    };
    auto load = [&](int k0) {
        const int k = k0 + 4 * h;
        Step s;
        if (k + 4 <= p.k) {
#pragma unroll
            for (int m = 0; m < 2; ++m) s.x[m] = __builtin_bit_cast(f32x4, *reinterpret_cast<const u32x4_any*>(x[m] + k));
            if constexpr (IN_DENSE && W32) {
                s.w = __builtin_bit_cast(f32x4, *reinterpret_cast<const u32x4_any*>(w + k));
            } else {
#pragma unroll
                for (int j = 0; j < 4; ++j) s.w[j] = number(w[static_cast<int64_t>(k + j) * p.ws_in]);
            }
        } else {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const bool in = k + j < p.k;
                s.w[j] = in ? number(w[static_cast<int64_t>(k + j) * p.ws_in]) : 0.0f;
#pragma unroll
                for (int m = 0; m < 2; ++m) s.x[m][j] = in ? x[m][k + j] : 0.0f;
            }
        }
        return s;
    };
    f32x16 acc[2] = {};
    constexpr int DEPTH = 4;
    Step ahead[DEPTH];
#pragma unroll
    for (int i = 0; i < DEPTH; ++i) ahead[i] = load(8 * i);
    for (int k0 = 0; k0 < p.k; k0 += 8 * DEPTH) {
#pragma unroll
        for (int i = 0; i < DEPTH; ++i) {
            const Step now = ahead[i];
            ahead[i] = load(k0 + 8 * (DEPTH + i));
#pragma unroll
            for (int j = 0; j < 4; ++j)
#pragma unroll
                for (int m = 0; m < 2; ++m) acc[m] = __builtin_amdgcn_mfma_f32_32x32x2f32(now.w[j], now.x[m][j], acc[m], 0, 0, 0);
        }
    }
#pragma unroll
    for (int m = 0; m < 2; ++m) {
        const int64_t t = t0 + 32 * m + l;
        if (t >= p.tokens) continue;
        float* const y = static_cast<float*>(p.y) + (t * p.heads + head) * p.n;
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            const int n = n0 + 8 * g + 4 * h;
            if (n + 4 <= p.n) {
                *reinterpret_cast<u32x4_any*>(y + n) = __builtin_bit_cast(u32x4, f32x4{acc[m][4 * g], acc[m][4 * g + 1], acc[m][4 * g + 2], acc[m][4 * g + 3]});
            } else {
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    if (n + i < p.n) y[n + i] = acc[m][4 * g + i];
            }
        }
    }
}

// bf16 with more inputs than a wave's registers hold: 32 tokens x 32 outputs a block, sums in fp32.
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

// Blocks of four waves (128 outputs) where these fill the chip, else of one.
template <typename Launch>
void launch_blocks(const HeadArgs& p, int64_t chunks, Launch launch) {
    const int64_t wide = ceil_div(p.n, 128);
    if (p.heads * wide * chunks >= 2 * kChip) launch(std::integral_constant<int, 4>{}, wide);
    else launch(std::integral_constant<int, 1>{}, ceil_div(p.n, 32));
}

template <int KS>
void launch_bf16(HeadArgs p, hipStream_t s) {
    // A block reads its weights once for its tokens: as many of them as leave four blocks a compute unit.
    const int64_t tiles = ceil_div(p.tokens, 32), units = p.heads * ceil_div(p.n, 128);
    const int64_t most = std::max<int64_t>(1, ceil_div(4 * kChip, units)), chunks = std::min(tiles, most);
    p.chunk = ceil_div(tiles, chunks) * 32;
    const unsigned used = static_cast<unsigned>(ceil_div(p.tokens, p.chunk));
    launch_blocks(p, used, [&](auto waves, int64_t n_blocks) {
        constexpr int W = decltype(waves)::value;
        const dim3 grid(static_cast<unsigned>(p.heads * n_blocks * used));
        if (p.ws_in == 1) hipLaunchKernelGGL((head_linear_kernel<KS, true, W>), grid, dim3(W * 64), 0, s, p, static_cast<unsigned>(n_blocks), used);
        else hipLaunchKernelGGL((head_linear_kernel<KS, false, W>), grid, dim3(W * 64), 0, s, p, static_cast<unsigned>(n_blocks), used);
    });
}

template <bool W32>
void launch_f32(const HeadArgs& p, hipStream_t s) {
    const unsigned chunks = static_cast<unsigned>(ceil_div(p.tokens, 64));
    launch_blocks(p, chunks, [&](auto waves, int64_t n_blocks) {
        constexpr int W = decltype(waves)::value;
        const dim3 grid(static_cast<unsigned>(p.heads * n_blocks * chunks));
        if (p.ws_in == 1) hipLaunchKernelGGL((head_linear_f32_kernel<W32, true, W>), grid, dim3(W * 64), 0, s, p, static_cast<unsigned>(n_blocks), chunks);
        else hipLaunchKernelGGL((head_linear_f32_kernel<W32, false, W>), grid, dim3(W * 64), 0, s, p, static_cast<unsigned>(n_blocks), chunks);
    });
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
    MLK_CHECK(token_tiles < (int64_t{1} << 24) / heads / n_tiles, "too many tokens for one launch");  // of 256 threads a tile: below 2^32
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
