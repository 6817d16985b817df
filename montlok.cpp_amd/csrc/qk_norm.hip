// RMSNorm of every query and key head and the rotation of its last lanes, in
// one pass: each head row is read once and written once.
//
//   y = x / sqrt(mean(x^2) + eps) * w                          (over head_dim)
//   out[nope + i]        = y[nope + i] cos[i] - y[nope + half + i] sin[i]
//   out[nope + half + i] = y[nope + half + i] cos[half + i] + y[nope + i] sin[half + i]
//
// with the token's own row of the tables. Everything is formed in double and
// rounded once, as rms_norm and mla_rope_qk are.
#include <cmath>

#include "fp4.h"

namespace mlk {
namespace {

struct Head {
    const void* x;
    int64_t bs, ts, hs;
    const float* weight;
    void* out;
};

struct NormArgs {
    Head q, k;
    const float* cosine;
    const float* sine;
    const int32_t* positions;
    int64_t table_rows, tokens, length;
    int32_t heads, kv_heads, dim, rope;
    double eps;
};

// One wave a head row.
template <bool F32>
__global__ __launch_bounds__(256) void qk_norm_rope_kernel(NormArgs p) {
    const int per_token = p.heads + p.kv_heads, lane = threadIdx.x & 63;
    const int64_t row = static_cast<int64_t>(blockIdx.x) * 4 + threadIdx.x / 64;
    const int64_t token = row / per_token;
    if (token >= p.tokens) return;
    const int which = static_cast<int>(row - token * per_token), head = which < p.heads ? which : which - p.heads;
    const Head& t = which < p.heads ? p.q : p.k;
    const int64_t b = token / p.length;
    const int64_t from = b * t.bs + (token - b * p.length) * t.ts + head * t.hs;
    const int64_t to = (token * (which < p.heads ? p.heads : p.kv_heads) + head) * p.dim;
    double sum = 0.0;
    for (int d = lane; d < p.dim; d += 64) {
        const double v = Element<F32>::get(t.x, from + d);
        sum = fma(v, v, sum);
    }
    const double by = 1.0 / sqrt(group_sum_d<64>(sum) / p.dim + p.eps);
    const int64_t at = p.positions[token];
    const bool inside = at < p.table_rows;
    const int nope = p.dim - p.rope, half = p.rope / 2;
    auto norm = [&](int d) { return Element<F32>::get(t.x, from + d) * by * t.weight[d]; };
    for (int d = lane; d < p.dim; d += 64) {
        double y = 0.0;
        if (at >= 0) {
            if (d < nope) {
                y = norm(d);
            } else if (inside) {
                const int i = d - nope;
                const double c = p.cosine[at * p.rope + i], s = p.sine[at * p.rope + i];
                const double other = norm(i < half ? d + half : d - half);
                y = norm(d) * c + (i < half ? -other * s : other * s);
            }
            if (!inside) y = NAN;
        }
        Element<F32>::put(t.out, to + d, static_cast<float>(y));
    }
}

}  // namespace
}  // namespace mlk

using namespace mlk;

extern "C" mlk_status mlk_qk_norm_rope(const void* q, const int64_t* q_strides, const void* k, const int64_t* k_strides, int32_t dtype,
                                       const float* q_weight, const float* k_weight, double eps, const float* cosine,
                                       const float* sine, int64_t table_rows, int64_t rope_dim, const int32_t* positions,
                                       int64_t batch, int64_t length, int64_t heads, int64_t kv_heads, int64_t head_dim, void* q_out,
                                       void* k_out, mlk_stream_t stream) {
    MLK_CHECK(dtype == MLK_DTYPE_F32 || dtype == MLK_DTYPE_BF16, "dtype must be f32 or bf16");
    MLK_CHECK(batch >= 0 && length >= 0 && heads > 0 && kv_heads > 0 && table_rows >= 0, "invalid norm geometry");
    MLK_CHECK(head_dim > 0 && head_dim <= 1024, "head_dim must be between 1 and 1024");
    MLK_CHECK(rope_dim >= 0 && rope_dim <= head_dim && rope_dim % 2 == 0, "rope_dim must be even and at most head_dim");
    MLK_CHECK(heads < (int64_t{1} << 20) && kv_heads < (int64_t{1} << 20), "too many heads");
    MLK_CHECK(batch < (int64_t{1} << 31) && length < (int64_t{1} << 31) && batch * length < (int64_t{1} << 36), "too many tokens");
    const int64_t blocks = ceil_div(batch * length * (heads + kv_heads), 4);
    MLK_CHECK(blocks < (int64_t{1} << 31), "too many tokens for one launch");
    if (batch == 0 || length == 0) return MLK_OK;
    MLK_CHECK(q && q_strides && k && k_strides && q_weight && k_weight && positions && q_out && k_out, "null tensor pointer");
    MLK_CHECK(rope_dim == 0 || table_rows == 0 || (cosine && sine), "null tensor pointer");
    NormArgs p{};
    p.q = Head{q, q_strides[0], q_strides[1], q_strides[2], q_weight, q_out};
    p.k = Head{k, k_strides[0], k_strides[1], k_strides[2], k_weight, k_out};
    p.cosine = cosine;
    p.sine = sine;
    p.positions = positions;
    p.table_rows = table_rows;
    p.tokens = batch * length;
    p.length = length;
    p.heads = static_cast<int32_t>(heads);
    p.kv_heads = static_cast<int32_t>(kv_heads);
    p.dim = static_cast<int32_t>(head_dim);
    p.rope = static_cast<int32_t>(rope_dim);
    p.eps = eps;
    hipStream_t s = reinterpret_cast<hipStream_t>(stream);
    if (dtype == MLK_DTYPE_F32) {
        hipLaunchKernelGGL(qk_norm_rope_kernel<true>, dim3(static_cast<unsigned>(blocks)), dim3(256), 0, s, p);
    } else {
        hipLaunchKernelGGL(qk_norm_rope_kernel<false>, dim3(static_cast<unsigned>(blocks)), dim3(256), 0, s, p);
    }
    return launch_status("qk norm rope");
}
