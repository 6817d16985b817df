// A cache of latents: pages of token rows, as latent_append writes them and latent_attention reads them.
//
//   eight bits   R e4m3 codes | P bf16 | fp32 scale, 12 unused bytes        value = code * scale, the scale a power of two
//   bf16         R bf16       | P bf16 | 16 unused bytes
//
// A row is an odd number of 16-byte pieces: sixteen rows laid end to end in LDS then begin in different banks, whatever
// piece of them is read. A power of two of the whole row is enough for a format with an exponent of its own: e4m3 holds
// 2^-9 .. 448, so what a row's largest value leaves of the smallest ones is 2^-18 of it.
#pragma once

#include "fp4.h"

namespace mlk {

template <bool E4M3>
constexpr int row_bytes(int rank, int rope) {
    return E4M3 ? rank + 2 * rope + 16 : 2 * (rank + rope) + 16;
}

struct LatentCache {
    const uint8_t* bytes;
    const int32_t* table;
    int32_t pages, page_size, width;
};

// The row of a token, or null where the table does not name its page.
template <typename Byte>
__device__ __forceinline__ Byte* row_of(Byte* bytes, const LatentCache& c, int64_t sequence, uint32_t token, int row) {
    const uint32_t page = token / static_cast<uint32_t>(c.page_size);
    if (page >= static_cast<uint32_t>(c.width)) return nullptr;
    const int32_t id = c.table[sequence * c.width + page];
    if (id < 0 || id >= c.pages) return nullptr;
    return bytes + (static_cast<int64_t>(id) * c.page_size + (token - page * static_cast<uint32_t>(c.page_size))) * row;
}

// Eight e4m3 codes times a power of two as bf16 values, exactly (NaN for 0x7F and 0xFF, and under a scale of NaN: all codes
// under every exponent byte).
__device__ __forceinline__ bf16x8 e4m3_octet(uint32_t lo, uint32_t hi, float scale) {
    const u32x4 v = {__builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, scale, false)),
                     __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, scale, true)),
                     __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, scale, false)),
                     __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, scale, true))};
    return __builtin_bit_cast(bf16x8, v);
}

// What every call over a cache is checked for; MLK_OK or the refusal.
mlk_status check_latent_cache(int64_t batch, int64_t length, int64_t rank, int64_t rope, int32_t dtype, int32_t cache_dtype,
                              int64_t pages, int64_t page_size, int64_t width);

}  // namespace mlk
