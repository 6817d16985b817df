// The rotation of queries and keys at their own positions, neighbours (2 i, 2 i + 1) or halves (i, i + rope / 2) of a
// head's last `rope` lanes paired:
//
//   (a, b) -> m (a cos t - b sin t), m (b cos t + a sin t),   t = position * frequency[i]
//
// Angles, sines and products are double, rounded once: t of a far position keeps no correct digit in fp32 (2^20 positions:
// 0.06 radians). Bound by memory, each head row read once and written once: 8,002 tokens of 16 + 16 heads of 64 in fp32 take
// 24.6 us, 5.1 TB/s; one token each of 16 sequences 3.4 us, a launch and a chain of two loads.
#include <algorithm>
#include <cmath>
#include <type_traits>

#include "fp4.h"

namespace mlk {
namespace {

struct RopeHead {
    const void* x;
    int64_t bs, ts, hs;
    void* out;
};
struct RopeArgs {
    RopeHead q, k;
    const double* frequencies;
    const int32_t* positions;
    unsigned tokens, length;  // tokens below 2^31
    int32_t heads, kv_heads, dim, rope;
    double magnitude;
};

// sine and cosine of position * frequency. The product is kept whole (hi + lo); pi / 2 in two doubles leaves 2^-107 of
// every quarter turn, so up to 2^31 radians the angle in its quarter is right to a double's last places.
__device__ __forceinline__ void sincos_at(int32_t position, double frequency, double* sine, double* cosine) {
    const double at = position, hi = at * frequency, lo = fma(at, frequency, -hi);
    const double turns = __builtin_rint(hi * 0.63661977236758134308);
    const double r = fma(-turns, 6.123233995736765886e-17, fma(-turns, 1.5707963267948965580, hi)) + lo;
    double s, c;
    sincos_d(r, &s, &c);
    const double quarter = turns - 4.0 * __builtin_floor(turns * 0.25);
    const bool swap = quarter == 1.0 || quarter == 3.0;
    const double so = swap ? c : s, co = swap ? s : c;
    *sine = quarter >= 2.0 ? -so : so;
    *cosine = quarter == 1.0 || quarter == 2.0 ? -co : co;
}

// The float that v is stored through: rounded to bf16 it is v rounded once (the upper word of v, and a float's last bit where
// the lower word is not 0).
template <bool F32>
__device__ __forceinline__ float to_store(double v) {
    if constexpr (F32) return static_cast<float>(v);
    uint32_t cut = __double2loint(v);
    asm("v_min_u32 %0, 1, %0" : "+v"(cut));
    return static_cast<float>(__hiloint2double(__double2hiint(v), static_cast<int>(cut << 29)));
}

template <bool F32>
struct Piece {
    static constexpr int E = F32 ? 4 : 8;
    u32x4 w;
    __device__ __forceinline__ double get(int i) const {
        if constexpr (F32) return __uint_as_float(w[i]);
        return __uint_as_float(i % 2 ? w[i / 2] & 0xFFFF0000u : w[i / 2] << 16);
    }
    static __device__ __forceinline__ Piece load(const void* p, int64_t first) {
        return {*reinterpret_cast<const u32x4_any*>(static_cast<const char*>(p) + first * (F32 ? 4 : 2))};
    }
    static __device__ __forceinline__ Piece of(const double (&v)[E]) {
        Piece r;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if constexpr (F32) r.w[i] = __float_as_uint(to_store<true>(v[i]));
            else r.w[i] = __builtin_bit_cast(uint32_t, bf16x2{static_cast<__bf16>(to_store<false>(v[2 * i])), static_cast<__bf16>(to_store<false>(v[2 * i + 1]))});
        }
        return r;
    }
    __device__ __forceinline__ void store(void* p, int64_t first) const { *reinterpret_cast<u32x4*>(static_cast<char*>(p) + first * (F32 ? 4 : 2)) = w; }
};

// A block takes `tokens_per` tokens and `rows_per` of their head rows. `items` threads serve a row: a piece of 16 bytes each
// of what is copied, then a piece (neighbours) or one in each half (halves) of what is rotated; a thread keeps its place in
// the row and walks over rows. Sines and cosines of a token are formed once in a block, while its first pieces are loaded.
template <bool F32, bool NEIGHBOURS>
__global__ __launch_bounds__(256) void rope_kernel(RopeArgs p, int items, int tokens_per, int rows_per, unsigned row_chunks) {
    constexpr int E = Piece<F32>::E;
    extern __shared__ double2 turn[];  // [tokens_per][rope / 2]: cosine, sine
    const int pairs = p.rope / 2, all = p.heads + p.kv_heads;
    const unsigned chunk = blockIdx.x % row_chunks, first_token = blockIdx.x / row_chunks * tokens_per;
    for (int i = threadIdx.x; i < tokens_per * pairs; i += 256) {
        const int t = i / pairs;
        double s = 0.0, c = 0.0;
        if (first_token + t < p.tokens) sincos_at(p.positions[first_token + t], p.frequencies[i - t * pairs], &s, &c);
        turn[i] = double2{c * p.magnitude, s * p.magnitude};
    }
    __syncthreads();
    const int row_step = 256 / (items * tokens_per);  // rows of each token that the threads take at a time
    const int slot = threadIdx.x / items, item = threadIdx.x - slot * items;
    const int t = slot / row_step;
    const unsigned token = first_token + t;
    if (t >= tokens_per || token >= p.tokens) return;
    const int32_t at = p.positions[token];
    const int nope = p.dim - p.rope, copied = nope / E;
    const bool turned = item >= copied;
    const int d = turned && !NEIGHBOURS ? nope + (item - copied) * E : item * E;
    const unsigned b = token / p.length, in = token - b * p.length;
    const double2* const mine = turn + t * pairs;
    const int end = min(static_cast<int>(chunk + 1) * rows_per, all);
    for (int row = chunk * rows_per + slot - t * row_step; row < end; row += row_step) {
        const bool query = row < p.heads;
        const RopeHead& h = query ? p.q : p.k;
        const int head = query ? row : row - p.heads;
        const int64_t from = b * h.bs + in * h.ts + head * h.hs + d;
        const int64_t to = (static_cast<int64_t>(token) * (query ? p.heads : p.kv_heads) + head) * p.dim + d;
        Piece<F32> x = Piece<F32>::load(h.x, from);
        if (!turned) {
            if (at < 0) x.w = u32x4{0, 0, 0, 0};
            x.store(h.out, to);
        } else if constexpr (NEIGHBOURS) {
            double y[E];
#pragma unroll
            for (int i = 0; i < E; i += 2) {
                const double2 cs = mine[(d - nope + i) / 2];
                y[i] = fma(x.get(i), cs.x, -(x.get(i + 1) * cs.y));
                y[i + 1] = fma(x.get(i + 1), cs.x, x.get(i) * cs.y);
            }
            x = Piece<F32>::of(y);
            if (at < 0) x.w = u32x4{0, 0, 0, 0};
            x.store(h.out, to);
        } else {
            Piece<F32> z = Piece<F32>::load(h.x, from + pairs);
            double y[E], u[E];
#pragma unroll
            for (int i = 0; i < E; ++i) {
                const double2 cs = mine[d - nope + i];
                y[i] = fma(x.get(i), cs.x, -(z.get(i) * cs.y));
                u[i] = fma(z.get(i), cs.x, x.get(i) * cs.y);
            }
            x = Piece<F32>::of(y);
            z = Piece<F32>::of(u);
            if (at < 0) x.w = z.w = u32x4{0, 0, 0, 0};
            x.store(h.out, to);
            z.store(h.out, to + pairs);
        }
    }
}

// Any head_dim and rope_dim: a thread an element, or a pair.
template <bool F32>
__global__ __launch_bounds__(256) void rope_any_kernel(RopeArgs p, bool neighbours) {
    const int nope = p.dim - p.rope, pairs = p.rope / 2, items = nope + pairs, all = p.heads + p.kv_heads;
    const int64_t id = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x, row = id / items;
    const int item = static_cast<int>(id - row * items);
    const int64_t token = row / all;
    if (token >= p.tokens) return;
    const int which = static_cast<int>(row - token * all), head = which < p.heads ? which : which - p.heads;
    const RopeHead& h = which < p.heads ? p.q : p.k;
    const int64_t b = token / p.length, in = token - b * p.length;
    const int64_t from = b * h.bs + in * h.ts + head * h.hs, to = (token * (which < p.heads ? p.heads : p.kv_heads) + head) * p.dim;
    const int32_t at = p.positions[token];
    if (item < nope) {
        Element<F32>::put(h.out, to + item, at < 0 ? 0.0f : Element<F32>::get(h.x, from + item));
        return;
    }
    const int i = item - nope, first = nope + (neighbours ? 2 * i : i), second = neighbours ? first + 1 : first + pairs;
    double s, c;
    sincos_at(at, p.frequencies[i], &s, &c);
    c *= p.magnitude;
    s *= p.magnitude;
    const double x = Element<F32>::get(h.x, from + first), y = Element<F32>::get(h.x, from + second);
    Element<F32>::put(h.out, to + first, at < 0 ? 0.0f : to_store<F32>(fma(x, c, -(y * s))));
    Element<F32>::put(h.out, to + second, at < 0 ? 0.0f : to_store<F32>(fma(y, c, x * s)));
}

template <bool F32>
bool launch_pieces(const RopeArgs& p, bool neighbours, hipStream_t s) {
    constexpr int E = Piece<F32>::E;
    if (p.dim % E != 0 || p.rope % (neighbours ? E : 2 * E) != 0) return false;
    const int items = (p.dim - p.rope) / E + p.rope / E / (neighbours ? 1 : 2);
    if (items == 0 || items > 256) return false;
    const int all = p.heads + p.kv_heads;
    // Several tokens a block where one has few pieces; several rows a thread once the blocks fill the chip.
    const int tokens_per = std::max(1, 256 / (items * all)), row_step = 256 / (items * tokens_per);
    const int64_t groups = ceil_div(p.tokens, tokens_per);
    int passes = 1;
    while (passes < 8 && groups * ceil_div(all, row_step * passes) > 4096) passes *= 2;
    const int64_t chunks = ceil_div(all, row_step * passes);
    if (groups * chunks >= (int64_t{1} << 24)) return false;
    const dim3 grid(static_cast<unsigned>(groups * chunks));
    const size_t lds = static_cast<size_t>(tokens_per) * (p.rope / 2) * sizeof(double2);
    if (neighbours) {
        hipLaunchKernelGGL((rope_kernel<F32, true>), grid, dim3(256), lds, s, p, items, tokens_per, row_step * passes, static_cast<unsigned>(chunks));
    } else {
        hipLaunchKernelGGL((rope_kernel<F32, false>), grid, dim3(256), lds, s, p, items, tokens_per, row_step * passes, static_cast<unsigned>(chunks));
    }
    return true;
}

}  // namespace
}  // namespace mlk

using namespace mlk;

extern "C" mlk_status mlk_rope(const void* q, const int64_t* q_strides, const void* k, const int64_t* k_strides, int32_t dtype,
                               const double* frequencies, int64_t rope_dim, int32_t interleaved, double magnitude, const int32_t* positions,
                               int64_t batch, int64_t length, int64_t heads, int64_t kv_heads, int64_t head_dim, void* q_out, void* k_out,
                               mlk_stream_t stream) {
    MLK_CHECK(dtype == MLK_DTYPE_F32 || dtype == MLK_DTYPE_BF16, "dtype must be f32 or bf16");
    MLK_CHECK(batch >= 0 && length >= 0 && heads > 0 && kv_heads > 0, "invalid rotation geometry");
    MLK_CHECK(head_dim > 0 && head_dim <= 1024, "head_dim must be between 1 and 1024");
    MLK_CHECK(rope_dim > 0 && rope_dim <= head_dim && rope_dim % 2 == 0, "rope_dim must be even, positive and at most head_dim");
    MLK_CHECK(heads < (int64_t{1} << 20) && kv_heads < (int64_t{1} << 20), "too many heads");
    MLK_CHECK(batch < (int64_t{1} << 31) && length < (int64_t{1} << 31) && batch * length < (int64_t{1} << 31), "too many tokens");
    const int64_t threads = batch * length * (heads + kv_heads);
    MLK_CHECK(threads < (int64_t{1} << 32) / head_dim, "too many tokens for one launch");  // a thread an element at most
    if (batch == 0 || length == 0) return MLK_OK;
    MLK_CHECK(q && q_strides && k && k_strides && frequencies && positions && q_out && k_out, "null tensor pointer");
    MLK_CHECK((reinterpret_cast<uintptr_t>(q_out) & 15) == 0 && (reinterpret_cast<uintptr_t>(k_out) & 15) == 0, "outputs must be 16-byte aligned");
    RopeArgs p{};
    p.q = RopeHead{q, q_strides[0], q_strides[1], q_strides[2], q_out};
    p.k = RopeHead{k, k_strides[0], k_strides[1], k_strides[2], k_out};
    p.frequencies = frequencies;
    p.positions = positions;
    p.tokens = static_cast<unsigned>(batch * length);
    p.length = static_cast<unsigned>(length);
    p.heads = static_cast<int32_t>(heads);
    p.kv_heads = static_cast<int32_t>(kv_heads);
    p.dim = static_cast<int32_t>(head_dim);
    p.rope = static_cast<int32_t>(rope_dim);
    p.magnitude = magnitude;
    hipStream_t s = reinterpret_cast<hipStream_t>(stream);
    const bool f32 = dtype == MLK_DTYPE_F32, neighbours = interleaved != 0;
    if (f32 ? launch_pieces<true>(p, neighbours, s) : launch_pieces<false>(p, neighbours, s)) return launch_status("rope");
    const int64_t blocks = ceil_div(threads * (head_dim - rope_dim / 2), 256);
    if (f32) {
        hipLaunchKernelGGL(rope_any_kernel<true>, dim3(static_cast<unsigned>(blocks)), dim3(256), 0, s, p, neighbours);
    } else {
        hipLaunchKernelGGL(rope_any_kernel<false>, dim3(static_cast<unsigned>(blocks)), dim3(256), 0, s, p, neighbours);
    }
    return launch_status("rope");
}
