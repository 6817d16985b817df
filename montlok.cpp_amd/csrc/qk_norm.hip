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
#include <type_traits>

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
    int64_t table_rows, tokens, length;  // tokens below 2^26
    int32_t heads, kv_heads, dim, rope;
    double eps;
};

// 1 / sqrt(v) for v >= 0: the hardware's approximation (some 23 bits) and one third-order step, to a double's last place.
__device__ __forceinline__ double inv_sqrt(double v) {
    const double r = __builtin_amdgcn_rsq(v), e = fma(-(v * r), r, 1.0);
    return __builtin_isinf(v) ? 0.0 : fma(r * e, fma(0.375, e, 0.5), r);
}

// E consecutive floats, or elements of x, at any alignment.
typedef float f32x4_any __attribute__((ext_vector_type(4), aligned(4)));
template <int E>
__device__ __forceinline__ void load_floats(const float* from, float (&v)[E]) {
#pragma unroll
    for (int i = 0; i < E; i += 4) {
        const f32x4 x = *reinterpret_cast<const f32x4_any*>(from + i);
#pragma unroll
        for (int j = 0; j < 4; ++j) v[i + j] = x[j];
    }
}
template <bool F32>
__device__ __forceinline__ u32x4 load_elements(const void* p, int64_t first) {
    return *reinterpret_cast<const u32x4_any*>(static_cast<const char*>(p) + first * (F32 ? 4 : 2));
}
template <bool F32>
__device__ __forceinline__ double element(const u32x4& v, int i) {
    if constexpr (F32) return __uint_as_float(v[i]);
    return __uint_as_float(i % 2 ? v[i / 2] & 0xFFFF0000u : v[i / 2] << 16);
}

// The float that v is stored through. For bf16 the upper word of v, and a float's last bit where the lower word is not 0: the
// middle between two bf16 values only where v is one, so that v is rounded once (from 2^-126 on; a subnormal float may lose
// that bit).
template <bool F32>
__device__ __forceinline__ float to_store(double v) {
    if constexpr (F32) return static_cast<float>(v);
    uint32_t cut = __double2loint(v);
    asm("v_min_u32 %0, 1, %0" : "+v"(cut));  // the compiler makes a comparison and a selection of it
    return static_cast<float>(__hiloint2double(__double2hiint(v), static_cast<int>(cut << 29)));
}

// A head row on LPG lanes of E elements (16 bytes) each, a wave on R * 64 / LPG query rows, or key rows, of one token.
// What the rows share is formed once, weight times cosine and partner's weight times sine in double, so that an element
// costs three double operations beside its square (with all of it per row, 8000 tokens x 40 heads of 128 in bf16 took
// 56 us, and 39 so). A rotated lane loads its partners' 16 bytes as well (from the L1: the partner lane has them) instead of
// exchanging doubles. Every load is issued before the first sum.
template <bool F32, int LPG, int R>
__global__ __launch_bounds__(256) void qk_norm_rope_vec_kernel(NormArgs p, unsigned chunks, unsigned q_chunks) {
    constexpr int E = F32 ? 4 : 8, D = LPG * E, G = 64 / LPG;
    const unsigned wave = blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
    const unsigned token = wave / chunks;  // below 2^26, as a launch's waves
    if (token >= p.tokens) return;
    const unsigned chunk = wave - token * chunks, length = static_cast<unsigned>(p.length), b = token / length;
    const bool query = chunk < q_chunks;
    const Head& t = query ? p.q : p.k;
    const int rows = query ? p.heads : p.kv_heads;
    const int lane = threadIdx.x & 63, d = lane % LPG * E, first = static_cast<int>(query ? chunk : chunk - q_chunks) * (G * R) + lane / LPG;
    const int64_t at = p.positions[token];
    const int nope = D - p.rope, half = p.rope / 2;
    const bool turned = d >= nope, upper = d >= nope + half, inside = at >= 0 && at < p.table_rows;
    const int other = !turned ? d : upper ? d - half : d + half;
    const int64_t from = b * t.bs + static_cast<int64_t>(token - b * length) * t.ts;
    u32x4 x[R], y[R];
#pragma unroll
    for (int r = 0; r < R; ++r) {
        const int64_t start = from + min(first + r * G, rows - 1) * t.hs;
        x[r] = load_elements<F32>(t.x, start + d);
        y[r] = load_elements<F32>(t.x, start + other);
    }
    float weight[E], partner[E], cosine[E], sine[E];
    load_floats<E>(t.weight + d, weight);
    load_floats<E>(t.weight + other, partner);
#pragma unroll
    for (int i = 0; i < E; ++i) {
        cosine[i] = 1.0f;
        sine[i] = 0.0f;
    }
    if (turned && inside) {
        load_floats<E>(p.cosine + at * p.rope + (d - nope), cosine);
        load_floats<E>(p.sine + at * p.rope + (d - nope), sine);
    }
    const uint32_t fill = at < 0 ? 0 : F32 ? 0x7FC00000u : 0x7FC07FC0u;  // zeros, or NaN, where the position has no row
    double sum[R];
#pragma unroll
    for (int r = 0; r < R; ++r) {
        sum[r] = 0.0;
#pragma unroll
        for (int i = 0; i < E; ++i) sum[r] = fma(element<F32>(x[r], i), element<F32>(x[r], i), sum[r]);
    }
    group_sums_d(sum, LPG);
    double own[E], others[E];
#pragma unroll
    for (int i = 0; i < E; ++i) {
        own[i] = static_cast<double>(weight[i]) * cosine[i];
        others[i] = turned ? static_cast<double>(upper ? partner[i] : -partner[i]) * sine[i] : 0.0;
    }
#pragma unroll
    for (int r = 0; r < R; ++r) {
        const int row = first + r * G;
        if (row >= rows) break;
        const double by = inv_sqrt(fma(sum[r], 1.0 / D, p.eps));
        float out[E];
#pragma unroll
        for (int i = 0; i < E; ++i) {
            // A lane that is not rotated is its own partner, times 0: an infinity of it is NaN here, and in its row's norm.
            out[i] = to_store<F32>(fma(element<F32>(y[r], i), others[i], element<F32>(x[r], i) * own[i]) * by);
        }
        u32x4 w;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            w[i] = F32 ? __float_as_uint(out[i]) : __builtin_bit_cast(uint32_t, bf16x2{static_cast<__bf16>(out[E / 4 * i]), static_cast<__bf16>(out[E / 4 * i + E / 8])});
            w[i] = inside ? w[i] : fill;
        }
        const int64_t to = (static_cast<int64_t>(token) * rows + row) * D + d;
        *reinterpret_cast<u32x4*>(static_cast<char*>(t.out) + to * (F32 ? 4 : 2)) = w;
    }
}

// Any head_dim and rope_dim, one wave a head row.
template <bool F32>
__global__ __launch_bounds__(256) void qk_norm_rope_kernel(NormArgs p) {
    const int per_token = p.heads + p.kv_heads, lane = threadIdx.x & 63;
    const unsigned row = blockIdx.x * 4 + threadIdx.x / 64, token = row / static_cast<unsigned>(per_token);
    if (token >= p.tokens) return;
    const int which = static_cast<int>(row - token * per_token), head = which < p.heads ? which : which - p.heads;
    const Head& t = which < p.heads ? p.q : p.k;
    const unsigned length = static_cast<unsigned>(p.length), b = token / length;
    const int64_t from = b * t.bs + static_cast<int64_t>(token - b * length) * t.ts + head * t.hs;
    const int64_t to = (static_cast<int64_t>(token) * (which < p.heads ? p.heads : p.kv_heads) + head) * p.dim;
    double sum = 0.0;
    for (int d = lane; d < p.dim; d += 64) {
        const double v = Element<F32>::get(t.x, from + d);
        sum = fma(v, v, sum);
    }
    const double by = inv_sqrt(group_sum_d<64>(sum) / p.dim + p.eps);
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
                y = norm(d) * c + (i < half ? -other : other) * s;
            }
            if (!inside) y = NAN;
        }
        Element<F32>::put(t.out, to + d, to_store<F32>(y));
    }
}

template <bool F32, int LPG>
void launch_vec(const NormArgs& p, hipStream_t s) {
    auto chunks = [&](int64_t rows, int64_t r) { return ceil_div(rows, 64 / LPG * r); };
    auto slots = [&](int64_t r) { return (chunks(p.heads, r) + chunks(p.kv_heads, r)) * r; };
    auto launch = [&](auto per) {
        constexpr int R = decltype(per)::value;
        const int64_t q = chunks(p.heads, R), all = q + chunks(p.kv_heads, R);
        hipLaunchKernelGGL((qk_norm_rope_vec_kernel<F32, LPG, R>), dim3(static_cast<unsigned>(ceil_div(p.tokens * all, 4))), dim3(256), 0, s, p,
                           static_cast<unsigned>(all), static_cast<unsigned>(q));
    };
    // Several rows a lane group where the waves still fill the chip and few of the groups' turns go empty.
    if (p.tokens * slots(4) >= 4 * 4096 && 4 * slots(4) <= 5 * slots(1)) return launch(std::integral_constant<int, 4>{});
    if (p.tokens * slots(2) >= 2 * 4096 && 4 * slots(2) <= 5 * slots(1)) return launch(std::integral_constant<int, 2>{});
    launch(std::integral_constant<int, 1>{});
}

// False where the head's elements do not fall to a power of two of lanes, halves of the rotation to whole lanes.
template <bool F32>
bool launch_vec(const NormArgs& p, hipStream_t s) {
    constexpr int E = F32 ? 4 : 8;
    if (p.rope / 2 % E != 0 || p.dim % E != 0) return false;
    switch (p.dim / E) {
        case 4: launch_vec<F32, 4>(p, s); return true;
        case 8: launch_vec<F32, 8>(p, s); return true;
        case 16: launch_vec<F32, 16>(p, s); return true;
        case 32: launch_vec<F32, 32>(p, s); return true;
        case 64: launch_vec<F32, 64>(p, s); return true;
        default: return false;
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
    MLK_CHECK(blocks < (int64_t{1} << 24), "too many tokens for one launch");  // of 256 threads: below 2^32
    if (batch == 0 || length == 0) return MLK_OK;
    MLK_CHECK(q && q_strides && k && k_strides && q_weight && k_weight && positions && q_out && k_out, "null tensor pointer");
    MLK_CHECK((reinterpret_cast<uintptr_t>(q_out) & 15) == 0 && (reinterpret_cast<uintptr_t>(k_out) & 15) == 0, "outputs must be 16-byte aligned");
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
    if (dtype == MLK_DTYPE_F32 ? launch_vec<true>(p, s) : launch_vec<false>(p, s)) return launch_status("qk norm rope");
    if (dtype == MLK_DTYPE_F32) {
        hipLaunchKernelGGL(qk_norm_rope_kernel<true>, dim3(static_cast<unsigned>(blocks)), dim3(256), 0, s, p);
    } else {
        hipLaunchKernelGGL(qk_norm_rope_kernel<false>, dim3(static_cast<unsigned>(blocks)), dim3(256), 0, s, p);
    }
    return launch_status("qk norm rope");
}
