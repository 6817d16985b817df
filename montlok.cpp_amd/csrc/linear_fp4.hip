// y = x W^T + b with four-bit weights (groups of 32 under a power of two), on
// the bf16 matrix cores with fp32 accumulation. Every weight is exact in bf16,
// a bf16 x is too, and an fp32 x is the exact sum of three bf16 values, so the
// only rounding is that of the sums.
#include "fp4.h"

namespace mlk {
namespace {

struct Fp4LinearArgs {
    const void* x;
    int64_t x_stride;
    const uint8_t* codes;
    const uint8_t* scales;
    const float* bias;
    void* out;
    int32_t rows, K, N;
};

constexpr int kStep = 128;  // k of one 16-byte load of a wave's four lane groups
constexpr int kWaves = 4;

// Block: 16 columns of y (rows of W) by 16 rows, its waves' share of K interleaved. Lane (g, l) holds group
// 4 step + g of row l of W (16 bytes) and the same 32 elements of row l of x: the products sum over k in an order of
// their own, the same for both operands.
template <bool F32>
__global__ __launch_bounds__(kWaves * 64) void linear_fp4_kernel(Fp4LinearArgs p) {
    constexpr int P = F32 ? 3 : 1;
    __shared__ float part[kWaves][16][17];
    const int wave = threadIdx.x / 64, lane = threadIdx.x & 63, g = lane >> 4, l = lane & 15;
    const int n0 = blockIdx.x * 16, m0 = blockIdx.y * 16;
    const int64_t n = min(n0 + l, p.N - 1), m = min(m0 + l, p.rows - 1);
    f32x4 acc = {0, 0, 0, 0};
    for (int step = wave; step * kStep < p.K; step += kWaves) {
        const int k0 = step * kStep + kGroup * g;
        const bool live = k0 < p.K;
        const int k = live ? k0 : 0;
        const u32x4 w = *reinterpret_cast<const u32x4*>(p.codes + n * (p.K / 2) + k / 2);
        const float scale = scale_of(p.scales[n * (p.K / kGroup) + k / kGroup]);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            float v[8];
            bf16x8 xs[P];
#pragma unroll
            for (int j = 0; j < 8; ++j) v[j] = live ? Element<F32>::get(p.x, m * p.x_stride + k + 8 * i + j) : 0.0f;
            if constexpr (F32) {
                planes_of(v, xs);
            } else {
#pragma unroll
                for (int j = 0; j < 8; ++j) xs[0][j] = static_cast<__bf16>(v[j]);
            }
            const bf16x8 ws = fp4_octet(live ? w[i] : 0, live ? scale : 1.0f);
#pragma unroll
            for (int j = P - 1; j >= 0; --j) acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(ws, xs[j], acc, 0, 0, 0);
        }
    }
#pragma unroll
    for (int r = 0; r < 4; ++r) part[wave][l][4 * g + r] = acc[r];
    __syncthreads();
    const int row = threadIdx.x / 16, col = threadIdx.x % 16;
    if (m0 + row >= p.rows || n0 + col >= p.N) return;
    float y = part[0][row][col];
#pragma unroll
    for (int w = 1; w < kWaves; ++w) y += part[w][row][col];
    if (p.bias != nullptr) y += p.bias[n0 + col];
    Element<F32>::put(p.out, static_cast<int64_t>(m0 + row) * p.N + n0 + col, y);
}

}  // namespace
}  // namespace mlk

using namespace mlk;

extern "C" mlk_status mlk_linear_fp4(const void* x, int64_t rows, int64_t in_features, int64_t x_stride, int32_t dtype,
                                     const uint8_t* codes, const uint8_t* scales, const float* bias, int64_t out_features, void* out,
                                     mlk_stream_t stream) {
    MLK_CHECK(dtype == MLK_DTYPE_F32 || dtype == MLK_DTYPE_BF16, "dtype must be f32 or bf16");
    MLK_CHECK(rows >= 0 && out_features > 0, "invalid linear geometry");
    MLK_CHECK(in_features > 0 && in_features % kGroup == 0, "in_features must be a positive multiple of 32");
    MLK_CHECK(rows < (int64_t{1} << 20) - 16 && in_features < (int64_t{1} << 31) && out_features < (int64_t{1} << 31) - 16, "too many rows or features");
    if (rows == 0) return MLK_OK;
    MLK_CHECK(x && codes && scales && out, "null tensor pointer");
    MLK_CHECK((reinterpret_cast<uintptr_t>(codes) & 15) == 0, "codes must be 16-byte aligned");
    Fp4LinearArgs p{x, x_stride, codes, scales, bias, out, static_cast<int32_t>(rows), static_cast<int32_t>(in_features), static_cast<int32_t>(out_features)};
    const dim3 grid(static_cast<unsigned>(ceil_div(out_features, 16)), static_cast<unsigned>(ceil_div(rows, 16)));
    hipStream_t s = reinterpret_cast<hipStream_t>(stream);
    if (dtype == MLK_DTYPE_F32) {
        hipLaunchKernelGGL(linear_fp4_kernel<true>, grid, dim3(kWaves * 64), 0, s, p);
    } else {
        hipLaunchKernelGGL(linear_fp4_kernel<false>, grid, dim3(kWaves * 64), 0, s, p);
    }
    return launch_status("linear fp4");
}
