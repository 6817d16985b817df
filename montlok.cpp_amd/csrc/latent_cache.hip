// Latents and rotated key parts into a paged cache and back out of it, each read once and written once.
//
// Bound by memory: 32,000 padded fp32 tokens of 512 + 64 take 15.4 us into eight bits and 17.4 us back, 5.1 TB/s over both; 16
// tokens 2.9 and 2.5 us, a chain of position, page number and row. Lanes take eight latents each, so that a row's largest
// value is found in at most six exchanges and every load and store is of 8 to 32 bytes side by side.
#include <cmath>

#include "latent.h"

namespace mlk {

mlk_status check_latent_cache(int64_t batch, int64_t length, int64_t rank, int64_t rope, int32_t dtype, int32_t cache_dtype,
                              int64_t pages, int64_t page_size, int64_t width) {
    MLK_CHECK(dtype == MLK_DTYPE_F32 || dtype == MLK_DTYPE_BF16, "dtype must be f32 or bf16");
    MLK_CHECK(cache_dtype == MLK_DTYPE_E4M3 || cache_dtype == MLK_DTYPE_BF16, "the cache's dtype must be e4m3 or bf16");
    MLK_CHECK(rank == 64 || rank == 128 || rank == 256 || rank == 512, "rank must be 64, 128, 256 or 512");
    MLK_CHECK(rope == 16 || rope == 32 || rope == 64, "rope_dim must be 16, 32 or 64");
    MLK_CHECK(page_size > 0 && page_size <= 65536, "page_size must be between 1 and 65536");
    MLK_CHECK(pages > 0 && pages < (int64_t{1} << 31), "pages must be between 1 and 2^31 - 1");
    MLK_CHECK(width > 0 && width <= (int64_t{1} << 28) && width * page_size <= (int64_t{1} << 28), "page_table must hold 1 to 2^28 tokens");
    MLK_CHECK(batch >= 0 && length >= 0 && batch < (int64_t{1} << 31) && length < (int64_t{1} << 31), "invalid cache geometry");
    return MLK_OK;
}

namespace {

struct CopyArgs {
    LatentCache c;
    const int32_t* positions;
    unsigned tokens, length;  // tokens below 2^29
    // append: the tensors and their strides {sequence, token}; read: outputs, contiguous
    const void *latent, *rope;
    int64_t ls[2], rs[2];
    void *latent_out, *rope_out;
    uint8_t* bytes;
};

// Eight consecutive values at any element's alignment.
template <bool F32>
__device__ __forceinline__ void load8(const void* p, int64_t first, float (&v)[8]) {
    if constexpr (F32) {
        const char* const at = static_cast<const char*>(p) + first * 4;
        const u32x4 a = *reinterpret_cast<const u32x4_any*>(at), b = *reinterpret_cast<const u32x4_any*>(at + 16);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            v[i] = __uint_as_float(a[i]);
            v[4 + i] = __uint_as_float(b[i]);
        }
    } else {
        const u32x4 a = *reinterpret_cast<const u32x4_any*>(static_cast<const char*>(p) + first * 2);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            v[2 * i] = __uint_as_float(a[i] << 16);
            v[2 * i + 1] = __uint_as_float(a[i] & 0xFFFF0000u);
        }
    }
}
__device__ __forceinline__ u32x4 pack8(const float (&v)[8]) {
    u32x4 w;
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = __builtin_bit_cast(uint32_t, bf16x2{static_cast<__bf16>(v[2 * i]), static_cast<__bf16>(v[2 * i + 1])});
    return w;
}
// Eight values to a contiguous, 16-byte aligned tensor.
template <bool F32>
__device__ __forceinline__ void store8(void* p, int64_t first, const float (&v)[8]) {
    if constexpr (F32) {
        float* const to = static_cast<float*>(p) + first;
        *reinterpret_cast<f32x4*>(to) = f32x4{v[0], v[1], v[2], v[3]};
        *reinterpret_cast<f32x4*>(to + 4) = f32x4{v[4], v[5], v[6], v[7]};
    } else {
        *reinterpret_cast<u32x4*>(static_cast<uint16_t*>(p) + first) = pack8(v);
    }
}

// R / 8 lanes a token, eight latents each; the first P / 8 of them take the key part too.
template <int R, bool F32, bool E4M3>
__global__ __launch_bounds__(256) void latent_append_kernel(CopyArgs p, int rope) {
    constexpr int LPT = R / 8;
    const unsigned token = blockIdx.x * (256 / LPT) + threadIdx.x / LPT;
    const int l = threadIdx.x % LPT;
    const bool real = token < p.tokens;
    const unsigned b = real ? token / p.length : 0, t = real ? token - b * p.length : 0;
    const int32_t at = real ? p.positions[token] : -1;
    float v[8], k[8];
    if (at >= 0) {
        load8<F32>(p.latent, b * p.ls[0] + t * p.ls[1] + 8 * l, v);
        if (8 * l < rope) load8<F32>(p.rope, b * p.rs[0] + t * p.rs[1] + 8 * l, k);
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = 0.0f;
    }
    // The row's largest magnitude as bits, which order as the values do; an infinity or a NaN is at least 0x7F800000. In the
    // bf16 cache a value that would round to an infinity counts as one.
    uint32_t most = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) most = max(most, __float_as_uint(v[i]) & 0x7FFFFFFFu);
#pragma unroll
    for (int m = 1; m < LPT; m *= 2) most = max(most, static_cast<uint32_t>(__shfl_xor(static_cast<int>(most), m, kWave)));
    if (at < 0) return;
    uint8_t* const row = row_of(p.bytes, p.c, b, static_cast<uint32_t>(at), row_bytes<E4M3>(R, rope));
    if (row == nullptr) return;
    if constexpr (E4M3) {
        const bool fine = most < 0x7F800000u;
        // The smallest power of two with most <= 448 * 2^power: 448 is 1.75 * 2^8. At least 2^-117, so that every value of
        // the row is a normal fp32 number, and at most 2^119, so that all are finite: what is above 448 * 2^119 is held there.
        const int power = min(max(static_cast<int>((most + 0x1FFFFFu) >> 23) - 135, -117), 119);
        const float by = __uint_as_float(static_cast<uint32_t>(127 - power) << 23);
        u32x2 codes = {0, 0};
        if (fine) {
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = __builtin_amdgcn_fmed3f(v[i] * by, -448.0f, 448.0f);
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                codes[i] = __builtin_amdgcn_cvt_pk_fp8_f32(v[4 * i], v[4 * i + 1], 0, false);
                codes[i] = __builtin_amdgcn_cvt_pk_fp8_f32(v[4 * i + 2], v[4 * i + 3], codes[i], true);
            }
        }
        *reinterpret_cast<u32x2*>(row + 8 * l) = codes;
        if (l == 0) *reinterpret_cast<u32x4*>(row + R + 2 * rope) = u32x4{fine ? static_cast<uint32_t>(127 + power) << 23 : 0x7FC00000u, 0, 0, 0};
    } else {
        const bool fine = most < 0x7F7F8000u;  // halfway from the largest bf16 to 2^128, which rounds to an infinity
        *reinterpret_cast<u32x4*>(row + 16 * l) = fine ? pack8(v) : u32x4{0x7FC07FC0u, 0x7FC07FC0u, 0x7FC07FC0u, 0x7FC07FC0u};
        if (l == 0) *reinterpret_cast<u32x4*>(row + 2 * (R + rope)) = u32x4{0, 0, 0, 0};
    }
    if (8 * l < rope) *reinterpret_cast<u32x4*>(row + (E4M3 ? R : 2 * R) + 16 * l) = pack8(k);
}

template <int R, bool F32, bool E4M3>
__global__ __launch_bounds__(256) void latent_read_kernel(CopyArgs p, int rope) {
    constexpr int LPT = R / 8;
    const unsigned token = blockIdx.x * (256 / LPT) + threadIdx.x / LPT;
    const int l = threadIdx.x % LPT;
    if (token >= p.tokens) return;
    const int32_t at = p.positions[token];
    const uint8_t* const row = at < 0 ? nullptr : row_of(p.c.bytes, p.c, token / p.length, static_cast<uint32_t>(at), row_bytes<E4M3>(R, rope));
    float v[8], k[8];
    if (row == nullptr) {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = k[i] = at < 0 ? 0.0f : NAN;
    } else {
        if constexpr (E4M3) {
            const u32x2 codes = *reinterpret_cast<const u32x2*>(row + 8 * l);
            const float scale = *reinterpret_cast<const float*>(row + R + 2 * rope);
            load8<false>(row + R, 8 * (8 * l < rope ? l : 0), k);
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const auto a = __builtin_amdgcn_cvt_pk_f32_fp8(codes[i], false), c = __builtin_amdgcn_cvt_pk_f32_fp8(codes[i], true);
                v[4 * i] = a[0] * scale;
                v[4 * i + 1] = a[1] * scale;
                v[4 * i + 2] = c[0] * scale;
                v[4 * i + 3] = c[1] * scale;
            }
        } else {
            load8<false>(row, 8 * l, v);
            load8<false>(row, R + 8 * (8 * l < rope ? l : 0), k);
        }
    }
    store8<F32>(p.latent_out, static_cast<int64_t>(token) * R + 8 * l, v);
    if (8 * l < rope) store8<F32>(p.rope_out, static_cast<int64_t>(token) * rope + 8 * l, k);
}

template <bool APPEND, bool F32, bool E4M3>
void launch_copy(const CopyArgs& p, int rank, int rope, hipStream_t s) {
    auto go = [&](auto r) {
        constexpr int R = decltype(r)::value;
        const dim3 grid(static_cast<unsigned>(ceil_div(p.tokens, 256 / (R / 8))));
        if constexpr (APPEND) {
            hipLaunchKernelGGL((latent_append_kernel<R, F32, E4M3>), grid, dim3(256), 0, s, p, rope);
        } else {
            hipLaunchKernelGGL((latent_read_kernel<R, F32, E4M3>), grid, dim3(256), 0, s, p, rope);
        }
    };
    switch (rank) {
        case 64: return go(std::integral_constant<int, 64>{});
        case 128: return go(std::integral_constant<int, 128>{});
        case 256: return go(std::integral_constant<int, 256>{});
        default: return go(std::integral_constant<int, 512>{});
    }
}
template <bool APPEND>
mlk_status launch_copy(const CopyArgs& p, int64_t rank, int64_t rope, int32_t dtype, int32_t cache_dtype, mlk_stream_t stream) {
    hipStream_t s = reinterpret_cast<hipStream_t>(stream);
    const bool f32 = dtype == MLK_DTYPE_F32, e4m3 = cache_dtype == MLK_DTYPE_E4M3;
    const int r = static_cast<int>(rank), q = static_cast<int>(rope);
    if (f32) {
        e4m3 ? launch_copy<APPEND, true, true>(p, r, q, s) : launch_copy<APPEND, true, false>(p, r, q, s);
    } else {
        e4m3 ? launch_copy<APPEND, false, true>(p, r, q, s) : launch_copy<APPEND, false, false>(p, r, q, s);
    }
    return launch_status(APPEND ? "latent append" : "latent read");
}

}  // namespace
}  // namespace mlk

using namespace mlk;

extern "C" mlk_status mlk_latent_append(const void* latent, const int64_t* latent_strides, const void* k_rope, const int64_t* k_rope_strides,
                                        int32_t dtype, int64_t batch, int64_t length, int64_t rank, int64_t rope_dim, uint8_t* cache,
                                        int32_t cache_dtype, int64_t pages, int64_t page_size, const int32_t* page_table, int64_t table_width,
                                        const int32_t* positions, mlk_stream_t stream) {
    const mlk_status checked = check_latent_cache(batch, length, rank, rope_dim, dtype, cache_dtype, pages, page_size, table_width);
    if (checked != MLK_OK) return checked;
    MLK_CHECK(batch * length < (int64_t{1} << 32) / 64, "too many tokens for one launch");  // of 64 lanes a token at most: below 2^32 threads
    if (batch == 0 || length == 0) return MLK_OK;
    MLK_CHECK(latent && latent_strides && k_rope && k_rope_strides && cache && page_table && positions, "null tensor pointer");
    MLK_CHECK((reinterpret_cast<uintptr_t>(cache) & 15) == 0, "the cache must be 16-byte aligned");
    CopyArgs p{};
    p.c = {cache, page_table, static_cast<int32_t>(pages), static_cast<int32_t>(page_size), static_cast<int32_t>(table_width)};
    p.bytes = cache;
    p.positions = positions;
    p.tokens = static_cast<unsigned>(batch * length);
    p.length = static_cast<unsigned>(length);
    p.latent = latent;
    p.rope = k_rope;
    for (int i = 0; i < 2; ++i) {
        p.ls[i] = latent_strides[i];
        p.rs[i] = k_rope_strides[i];
    }
    return launch_copy<true>(p, rank, rope_dim, dtype, cache_dtype, stream);
}

extern "C" mlk_status mlk_latent_read(const uint8_t* cache, int32_t cache_dtype, int64_t pages, int64_t page_size, const int32_t* page_table,
                                      int64_t table_width, const int32_t* positions, int64_t batch, int64_t length, int64_t rank,
                                      int64_t rope_dim, int32_t dtype, void* latent, void* k_rope, mlk_stream_t stream) {
    const mlk_status checked = check_latent_cache(batch, length, rank, rope_dim, dtype, cache_dtype, pages, page_size, table_width);
    if (checked != MLK_OK) return checked;
    MLK_CHECK(batch * length < (int64_t{1} << 32) / 64, "too many tokens for one launch");
    if (batch == 0 || length == 0) return MLK_OK;
    MLK_CHECK(cache && page_table && positions && latent && k_rope, "null tensor pointer");
    MLK_CHECK((reinterpret_cast<uintptr_t>(cache) & 15) == 0, "the cache must be 16-byte aligned");
    MLK_CHECK((reinterpret_cast<uintptr_t>(latent) & 15) == 0 && (reinterpret_cast<uintptr_t>(k_rope) & 15) == 0, "outputs must be 16-byte aligned");
    CopyArgs p{};
    p.c = {cache, page_table, static_cast<int32_t>(pages), static_cast<int32_t>(page_size), static_cast<int32_t>(table_width)};
    p.positions = positions;
    p.tokens = static_cast<unsigned>(batch * length);
    p.length = static_cast<unsigned>(length);
    p.latent_out = latent;
    p.rope_out = k_rope;
    return launch_copy<false>(p, rank, rope_dim, dtype, cache_dtype, stream);
}
