// Every head's own matrix times its part of the activations: y[t, h] = W[h] x[t, h], the products that take an MLA layer's
// queries into the latents' space and its attended latents back to the heads' values. W is dense along its inputs or along
// its outputs, so that both products read the same projection's rows.
#include "fp4.h"

namespace mlk {
namespace {

struct HeadArgs {
    const void *x, *w;
    void* y;
    int64_t xs_token, xs_head, ws_head, ws_out, ws_in;
    int64_t tokens;
    int32_t heads, k, n;
};

// 32 tokens x 32 outputs a block, sums in fp32.
template <bool X32, bool W32>
__global__ __launch_bounds__(256) void head_linear_any_kernel(HeadArgs p, unsigned token_tiles, unsigned n_tiles) {
    __shared__ float xs[32][33], ws[32][33];
    const unsigned id = blockIdx.x, tile = id % token_tiles, rest = id / token_tiles, nt = rest % n_tiles, head = rest / n_tiles;
    const int64_t t0 = static_cast<int64_t>(tile) * 32;
    const int n0 = nt * 32, a = threadIdx.x % 32, b = threadIdx.x / 32;
    float sum[4] = {};
    for (int k0 = 0; k0 < p.k; k0 += 32) {
        for (int i = b; i < 32; i += 8) {
            const bool in = t0 + i < p.tokens && k0 + a < p.k;
            xs[i][a] = in ? Element<X32>::get(p.x, (t0 + i) * p.xs_token + head * p.xs_head + k0 + a) : 0.0f;
            const int n = p.ws_in == 1 ? i : a, k = p.ws_in == 1 ? a : i;
            const bool has = n0 + n < p.n && k0 + k < p.k;
            ws[n][k] = has ? Element<W32>::get(p.w, head * p.ws_head + (n0 + n) * p.ws_out + (k0 + k) * p.ws_in) : 0.0f;
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
        if (t < p.tokens && n0 + a < p.n) Element<X32>::put(p.y, (t * p.heads + head) * p.n + n0 + a, sum[i]);
    }
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
    MLK_CHECK(token_tiles < (int64_t{1} << 24) / heads / n_tiles, "too many tokens for one launch");
    if (tokens == 0) return MLK_OK;
    MLK_CHECK(x && x_strides && weight && weight_strides && out, "null tensor pointer");
    MLK_CHECK(weight_strides[1] == 1 || weight_strides[2] == 1, "the weight must be dense along its inputs or its outputs");
    MLK_CHECK((reinterpret_cast<uintptr_t>(out) & 15) == 0, "out must be 16-byte aligned");
    const HeadArgs p{x, weight, out, x_strides[0], x_strides[1], weight_strides[0], weight_strides[1], weight_strides[2], tokens,
                     static_cast<int32_t>(heads), static_cast<int32_t>(in_features), static_cast<int32_t>(out_features)};
    hipStream_t s = reinterpret_cast<hipStream_t>(stream);
    const dim3 grid(static_cast<unsigned>(token_tiles * n_tiles * heads));
    const unsigned tt = static_cast<unsigned>(token_tiles), nt = static_cast<unsigned>(n_tiles);
    if (dtype == MLK_DTYPE_BF16) hipLaunchKernelGGL((head_linear_any_kernel<false, false>), grid, dim3(256), 0, s, p, tt, nt);
    else if (weight_dtype == MLK_DTYPE_BF16) hipLaunchKernelGGL((head_linear_any_kernel<true, false>), grid, dim3(256), 0, s, p, tt, nt);
    else hipLaunchKernelGGL((head_linear_any_kernel<true, true>), grid, dim3(256), 0, s, p, tt, nt);
    return launch_status("head linear");
}
