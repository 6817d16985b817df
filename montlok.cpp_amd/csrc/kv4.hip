// A paged key/value cache in four bits: writing it, reading it back and
// attention over it.
//
// A (page, key head) is one record of page_size * (D + D / 16) bytes:
//
//   key codes    [page_size][D / 2]      byte j of a row: elements 2 j (low bits), 2 j + 1
//   value codes  [D / 2][page_size]      the same bytes, token-minor
//   key scales   [page_size][D / 32]
//   value scales [D / 32][page_size]
//
// Both products of attention then load their operands straight into the
// registers that v_mfma_f32_16x16x32_bf16 takes them from (lane (g, l) = 16 g + l
// holds row l of A, 8 consecutive k): a key row is contiguous in d, which the
// score product sums over, and a value row in tokens, which the other one does.
// A transposed value row in the cache costs the append 16-byte-apart byte
// stores, once a token; the attention reads every byte of it for every token
// that follows.
#include <algorithm>

#include "fp4.h"

namespace mlk {
namespace {

constexpr int kRun = 16;     // tokens of a page that one lane takes: page sizes are multiples of it
constexpr int kTile = 64;    // keys a wave takes at a time
constexpr int kWaves = 4;    // of an attention block

struct Cache {
    uint8_t* bytes;
    int64_t record;  // bytes of a (page, head)
    int32_t pages, kv_heads, page_size;
    int32_t runs;     // page_size / kRun
    uint32_t magic;   // ceil(2^32 / runs); runs = 1: 0
    const int32_t* table;
    int32_t width;
    const int32_t* positions;
    int32_t batch, length;

    int64_t value_codes(int dim) const { return static_cast<int64_t>(page_size) * (dim / 2); }
};

// Page index of a run of 16 tokens and the run's place in it. run < 2^26, runs <= 64: the product with the
// rounded-up reciprocal is exact.
__device__ __forceinline__ void split_run(const Cache& c, uint32_t run, uint32_t& page, uint32_t& token) {
    page = c.magic == 0 ? run : __umulhi(run, c.magic);
    token = (run - page * static_cast<uint32_t>(c.runs)) * kRun;
}

// The record of token `at` of sequence b, and its place in the page; null where the table has no such page.
__device__ __forceinline__ uint8_t* record_of(const Cache& c, int b, int at, int head, int& offset) {
    uint32_t page, first;
    split_run(c, static_cast<uint32_t>(at) / kRun, page, first);
    offset = static_cast<int>(first) + at % kRun;
    if (page >= static_cast<uint32_t>(c.width)) return nullptr;
    const int id = c.table[static_cast<int64_t>(b) * c.width + page];
    if (id < 0 || id >= c.pages) return nullptr;
    return c.bytes + (static_cast<int64_t>(id) * c.kv_heads + head) * c.record;
}

// ------------------------------------------------------------- append and read

struct Rows3 {
    const void* p;
    int64_t bs, ts, hs;  // element strides of a sequence, a token, a head
};

// One thread a group of 32.
template <bool F32>
__global__ __launch_bounds__(256) void kv4_append_kernel(Cache c, Rows3 k, Rows3 v, int dim) {
    const int groups = dim / kGroup;
    const int64_t idx = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
    const int64_t row = idx / groups;  // (token, head)
    const int group = static_cast<int>(idx - row * groups);
    const int64_t token = row / c.kv_heads;
    if (token >= static_cast<int64_t>(c.batch) * c.length) return;
    const int head = static_cast<int>(row - token * c.kv_heads), b = static_cast<int>(token / c.length);
    const int at = c.positions[token];
    if (at < 0) return;
    int offset;
    uint8_t* const record = record_of(c, b, at, head, offset);
    if (record == nullptr) return;
    const bool values = blockIdx.y != 0;
    const Rows3& r = values ? v : k;
    const int64_t from = b * r.bs + (token - static_cast<int64_t>(b) * c.length) * r.ts + head * r.hs + group * kGroup;
    float x[kGroup];
    float most = 0.0f;
    bool fine = true;
#pragma unroll
    for (int i = 0; i < kGroup; ++i) {
        x[i] = Element<F32>::get(r.p, from + i);
        most = fmaxf(most, fabsf(x[i]));
        fine = fine && (__float_as_uint(x[i]) & 0x7F800000u) != 0x7F800000u;
    }
    const uint32_t byte = fine ? scale_byte(most) : 255;
    const float scale = scale_of(byte);
    u32x4 codes = {0, 0, 0, 0};
    if (fine) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            uint32_t w = 0;
            w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[8 * i], x[8 * i + 1], scale, 0);
            w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[8 * i + 2], x[8 * i + 3], scale, 1);
            w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[8 * i + 4], x[8 * i + 5], scale, 2);
            w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[8 * i + 6], x[8 * i + 7], scale, 3);
            codes[i] = w;
        }
    }
    const int64_t half = static_cast<int64_t>(c.page_size) * (dim / 2), scales = static_cast<int64_t>(c.page_size) * groups;
    if (!values) {
        *reinterpret_cast<u32x4*>(record + static_cast<int64_t>(offset) * (dim / 2) + 16 * group) = codes;
        record[2 * half + static_cast<int64_t>(offset) * groups + group] = static_cast<uint8_t>(byte);
    } else {
        uint8_t* const to = record + half + static_cast<int64_t>(16 * group) * c.page_size + offset;
#pragma unroll
        for (int j = 0; j < 16; ++j) to[static_cast<int64_t>(j) * c.page_size] = static_cast<uint8_t>(codes[j / 4] >> (8 * (j % 4)));
        record[2 * half + scales + static_cast<int64_t>(group) * c.page_size + offset] = static_cast<uint8_t>(byte);
    }
}

template <bool F32>
__global__ __launch_bounds__(256) void kv4_read_kernel(Cache c, void* k, void* v, int dim) {
    const int groups = dim / kGroup;
    const int64_t idx = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
    const int64_t row = idx / groups;
    const int group = static_cast<int>(idx - row * groups);
    const int64_t token = row / c.kv_heads;
    if (token >= static_cast<int64_t>(c.batch) * c.length) return;
    const int head = static_cast<int>(row - token * c.kv_heads), b = static_cast<int>(token / c.length);
    const bool values = blockIdx.y != 0;
    void* const out = values ? v : k;
    const int64_t to = row * dim + group * kGroup;
    const int at = c.positions[token];
    uint32_t byte = 3;
    u32x4 codes = {0, 0, 0, 0};
    if (at >= 0) {
        int offset;
        const uint8_t* const record = record_of(c, b, at, head, offset);
        const int64_t half = static_cast<int64_t>(c.page_size) * (dim / 2), scales = static_cast<int64_t>(c.page_size) * groups;
        if (record == nullptr) {
            byte = 255;
        } else if (!values) {
            codes = *reinterpret_cast<const u32x4*>(record + static_cast<int64_t>(offset) * (dim / 2) + 16 * group);
            byte = record[2 * half + static_cast<int64_t>(offset) * groups + group];
        } else {
            const uint8_t* const from = record + half + static_cast<int64_t>(16 * group) * c.page_size + offset;
#pragma unroll
            for (int j = 0; j < 16; ++j) codes[j / 4] |= static_cast<uint32_t>(from[static_cast<int64_t>(j) * c.page_size]) << (8 * (j % 4));
            byte = record[2 * half + scales + static_cast<int64_t>(group) * c.page_size + offset];
        }
    }
    const float scale = scale_of(byte);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const bf16x8 x = fp4_octet(codes[i], scale);
#pragma unroll
        for (int j = 0; j < 8; ++j) Element<F32>::put(out, to + 8 * i + j, static_cast<float>(x[j]));
    }
}

// ------------------------------------------------------------- attention

struct AttentionArgs {
    Cache c;
    const void* q;
    int64_t q_bs, q_ts, q_hs;
    int32_t heads, group;  // query heads; query heads to a key head
    int32_t rows;          // of a (sequence, key head): length * group; row r = token r / group, head r % group
    int32_t row_tiles, splits;
    float scale_log2;
    void* out;    // [batch, length, heads, D]
    float* part;  // [batch, kv_heads, rows, splits][D], then [...][2] (maximum, sum)
    int64_t part_rows;
};

__device__ __forceinline__ float max_over_groups(float v) {
    v = fmaxf(v, __shfl_xor(v, 16, kWave));
    return fmaxf(v, __shfl_xor(v, 32, kWave));
}
__device__ __forceinline__ float sum_over_groups(float v) {
    v += __shfl_xor(v, 16, kWave);
    return v + __shfl_xor(v, 32, kWave);
}
__device__ __forceinline__ float finite_or_zero(float m) { return m == -INFINITY ? 0.0f : m; }

// Eight results of a lane: elements first .. first + 7 of an output row.
template <bool F32>
__device__ __forceinline__ void put8(void* out, int64_t first, const float (&v)[8]) {
    if constexpr (F32) {
        float* const o = static_cast<float*>(out) + first;
        *reinterpret_cast<f32x4*>(o) = f32x4{v[0], v[1], v[2], v[3]};
        *reinterpret_cast<f32x4*>(o + 4) = f32x4{v[4], v[5], v[6], v[7]};
    } else {
        u32x4 w;
#pragma unroll
        for (int i = 0; i < 4; ++i) w[i] = float_to_bf16(v[2 * i]) | float_to_bf16(v[2 * i + 1]) << 16;
        *reinterpret_cast<u32x4*>(static_cast<uint16_t*>(out) + first) = w;
    }
}

template <int D, bool F32, int MT>
__global__ __launch_bounds__(kWaves * 64) void kv4_attention_kernel(AttentionArgs p) {
    constexpr int S = D / 32;          // k steps of a score product, and groups of a token
    constexpr int P = F32 ? 3 : 1;     // bf16 operands that make up a query or a weight
    constexpr int kScales = D == 256 ? 2 : 1;  // scales that a lane's part of a key row meets
    __shared__ float exchange[2][2 * S * 4 * MT][64];
    __shared__ float stats[kWaves][2][16 * MT];
    const Cache& c = p.c;
    const int wave = threadIdx.x / 64, lane = threadIdx.x & 63, g = lane >> 4, l = lane & 15;
    unsigned id = blockIdx.x;
    const int split = id % p.splits;
    id /= p.splits;
    const int row0 = static_cast<int>(id % p.row_tiles) * (16 * MT);
    id /= p.row_tiles;
    const int head = id % c.kv_heads, b = id / c.kv_heads;
    const int capacity = c.width * c.page_size;

    // Rows, their positions, and q as operands.
    int position[MT];
    bf16x8 q[MT][P][S];
    int last = -1, least = 0x7FFFFFFF;
#pragma unroll
    for (int m = 0; m < MT; ++m) {
        const int row = row0 + 16 * m + l, clamped = min(row, p.rows - 1), token = clamped / p.group;
        const int at = c.positions[static_cast<int64_t>(b) * c.length + token];
        position[m] = row < p.rows && at < capacity ? at : -1;
        last = max(last, position[m]);
        least = min(least, position[m] < 0 ? 0x7FFFFFFF : position[m]);
        const int64_t from = b * p.q_bs + token * p.q_ts + (head * p.group + clamped % p.group) * p.q_hs + (D / 4) * g;
#pragma unroll
        for (int s = 0; s < S; ++s) {
            float x[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) x[i] = Element<F32>::get(p.q, from + 8 * s + i);
            if constexpr (F32) {
                bf16x8 plane[3];
                planes_of<true>(x, plane);
#pragma unroll
                for (int i = 0; i < 3; ++i) q[m][i][s] = plane[i];
            } else {
#pragma unroll
                for (int i = 0; i < 8; ++i) q[m][0][s][i] = static_cast<__bf16>(x[i]);
            }
        }
    }
#pragma unroll
    for (int i = 1; i < 16; i *= 2) {
        last = max(last, __shfl_xor(last, i, kWave));
        least = min(least, __shfl_xor(least, i, kWave));
    }
    const int tiles = (last + kTile) / kTile;  // 0 where no row has a key
    const int begin = static_cast<int>(static_cast<int64_t>(tiles) * split / p.splits);
    const int end = static_cast<int>(static_cast<int64_t>(tiles) * (split + 1) / p.splits);

    float top[MT], sum[MT];
    f32x4 acc[MT][S][2];
#pragma unroll
    for (int m = 0; m < MT; ++m) {
        top[m] = -INFINITY;
        sum[m] = 0.0f;
#pragma unroll
        for (int s = 0; s < S; ++s) acc[m][s][0] = acc[m][s][1] = f32x4{0, 0, 0, 0};
    }

    const int64_t half = static_cast<int64_t>(c.page_size) * (D / 2);
    const int32_t* const table = c.table + static_cast<int64_t>(b) * c.width;
    for (int tile = begin + wave; tile < end; tile += kWaves) {
        const int first = tile * kTile;
        // Key tile a, row 4 g' + r is token 16 g' + 4 a + r of the 64, so that a lane's scores (rows 4 g .. 4 g + 3
        // of every tile) are its 16 tokens 16 g .. 16 g + 15 of the value product.
        uint32_t page, run;
        split_run(c, (first >> 4) + (l >> 2), page, run);
        bool held = first + 16 * (l >> 2) <= last;
        int id_k = held ? table[page] : 0;
        const bool bad = id_k < 0 || id_k >= c.pages;
        if (bad) id_k = 0;
        const uint8_t* const key = c.bytes + (static_cast<int64_t>(id_k) * c.kv_heads + head) * c.record;
        uint32_t kc[4][S], ks[4];
#pragma unroll
        for (int a = 0; a < 4; ++a) {
            const int token = run + 4 * a + (l & 3);
            const uint8_t* const from = key + token * (D / 2) + (D / 8) * g;
            const uint8_t* const scale = key + 2 * half + token * S;
            if constexpr (S == 1) {
                kc[a][0] = *reinterpret_cast<const uint32_t*>(from);
                ks[a] = scale[0];
            } else if constexpr (S == 2) {
                const u32x2 v = *reinterpret_cast<const u32x2*>(from);
                kc[a][0] = v[0], kc[a][1] = v[1];
                ks[a] = scale[g >> 1];
            } else {
#pragma unroll
                for (int i = 0; i < S / 4; ++i) {
                    const u32x4 v = reinterpret_cast<const u32x4*>(from)[i];
#pragma unroll
                    for (int j = 0; j < 4; ++j) kc[a][4 * i + j] = v[j];
                }
                ks[a] = S == 4 ? scale[g] : reinterpret_cast<const uint16_t*>(scale)[g];
            }
            if (bad) ks[a] = 0xFFFF;
        }
        split_run(c, (first >> 4) + g, page, run);
        held = first + 16 * g <= last;
        int id_v = held ? table[page] : 0;
        if (id_v < 0 || id_v >= c.pages) id_v = 0;
        const uint8_t* const value = c.bytes + (static_cast<int64_t>(id_v) * c.kv_heads + head) * c.record;
        u32x4 vc[S], vs[S];
#pragma unroll
        for (int s = 0; s < S; ++s) {
            vc[s] = *reinterpret_cast<const u32x4*>(value + half + static_cast<int64_t>(16 * s + l) * c.page_size + run);
            vs[s] = *reinterpret_cast<const u32x4*>(value + 2 * half + static_cast<int64_t>(S + s) * c.page_size + run);
        }

        f32x4 score[MT][4];
#pragma unroll
        for (int a = 0; a < 4; ++a) {
#pragma unroll
            for (int m = 0; m < MT; ++m) score[m][a] = f32x4{0, 0, 0, 0};
#pragma unroll
            for (int s = 0; s < S; ++s) {
                const bf16x8 k = fp4_octet(kc[a][s], kScales == 1 ? scale_at<0>(ks[a]) : (s < 4 ? scale_at<0>(ks[a]) : scale_at<1>(ks[a])));
#pragma unroll
                for (int m = 0; m < MT; ++m)
#pragma unroll
                    for (int i = P - 1; i >= 0; --i) score[m][a] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(k, q[m][i][s], score[m][a], 0, 0, 0);
            }
        }

        const bool masked = first + kTile - 1 > least;  // some row does not see the whole tile
        uint32_t poison[MT];
        if (masked) {
            // A value that no row may see must not reach a sum as 0 * NaN: its NaN scale goes, and the rows that do
            // see it are made NaN below.
#pragma unroll
            for (int m = 0; m < MT; ++m) poison[m] = 0;
#pragma unroll
            for (int s = 0; s < S; ++s)
#pragma unroll
                for (int i = 0; i < 16; ++i)
                    if ((vs[s][i / 4] >> (8 * (i % 4)) & 0xFF) == 0xFF) {
                        vs[s][i / 4] &= ~(0xFFu << (8 * (i % 4)));
#pragma unroll
                        for (int m = 0; m < MT; ++m)
                            if (first + 16 * g + i <= position[m]) poison[m] |= 1u << s;
                    }
        }

        bf16x8 weight[MT][P][2];
#pragma unroll
        for (int m = 0; m < MT; ++m) {
            float x[16];
            float most = -INFINITY;
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                x[i] = score[m][i / 4][i % 4] * p.scale_log2;
                if (masked && first + 16 * g + i > position[m]) x[i] = -INFINITY;
                most = fmaxf(most, x[i]);
            }
            const float before = top[m];
            top[m] = fmaxf(before, max_over_groups(most));
            const float base = finite_or_zero(top[m]), shrink = __builtin_amdgcn_exp2f(before - base);
            float part = 0.0f;
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                x[i] = __builtin_amdgcn_exp2f(x[i] - base);
                part += x[i];
            }
            sum[m] = fmaf(sum[m], shrink, part);
#pragma unroll
            for (int s = 0; s < S; ++s) {
                acc[m][s][0] *= shrink;
                acc[m][s][1] *= shrink;
            }
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                float w[8];
#pragma unroll
                for (int i = 0; i < 8; ++i) w[i] = x[8 * h + i];
                if constexpr (F32) {
                    bf16x8 plane[3];
                    planes_of<false>(w, plane);  // of finite values, or NaN
#pragma unroll
                    for (int i = 0; i < 3; ++i) weight[m][i][h] = plane[i];
                } else {
#pragma unroll
                    for (int i = 0; i < 8; ++i) weight[m][0][h][i] = static_cast<__bf16>(w[i]);
                }
            }
        }

#pragma unroll
        for (int s = 0; s < S; ++s)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                uint32_t pair[8];  // elements 2 j and 2 j + 1 of a token
#pragma unroll
                for (int w = 0; w < 2; ++w) {
                    const uint32_t codes = vc[s][2 * h + w], scales = vs[s][2 * h + w];
                    pair[4 * w] = fp4_pair<0>(codes, scale_at<0>(scales));
                    pair[4 * w + 1] = fp4_pair<1>(codes, scale_at<1>(scales));
                    pair[4 * w + 2] = fp4_pair<2>(codes, scale_at<2>(scales));
                    pair[4 * w + 3] = fp4_pair<3>(codes, scale_at<3>(scales));
                }
                u32x4 even, odd;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    even[i] = __builtin_amdgcn_perm(pair[2 * i + 1], pair[2 * i], 0x05040100u);
                    odd[i] = __builtin_amdgcn_perm(pair[2 * i + 1], pair[2 * i], 0x07060302u);
                }
#pragma unroll
                for (int m = 0; m < MT; ++m)
#pragma unroll
                    for (int i = P - 1; i >= 0; --i) {
                        acc[m][s][0] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, even), weight[m][i][h], acc[m][s][0], 0, 0, 0);
                        acc[m][s][1] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, odd), weight[m][i][h], acc[m][s][1], 0, 0, 0);
                    }
            }
        if (masked) {
#pragma unroll
            for (int m = 0; m < MT; ++m) {
                if (__ballot(poison[m] != 0) == 0) continue;
                uint32_t any = poison[m];
                any |= __shfl_xor(any, 16, kWave);
                any |= __shfl_xor(any, 32, kWave);
#pragma unroll
                for (int s = 0; s < S; ++s)
                    if (any >> s & 1) acc[m][s][0] = acc[m][s][1] = f32x4{NAN, NAN, NAN, NAN};
            }
        }
    }

    // The four waves' parts joined.
#pragma unroll
    for (int m = 0; m < MT; ++m) {
        sum[m] = sum_over_groups(sum[m]);
        if (g == 0) {
            stats[wave][0][16 * m + l] = top[m];
            stats[wave][1][16 * m + l] = sum[m];
        }
    }
    __syncthreads();
    float all_top[MT], all_sum[MT];
#pragma unroll
    for (int m = 0; m < MT; ++m) {
        all_top[m] = -INFINITY;
#pragma unroll
        for (int w = 0; w < kWaves; ++w) all_top[m] = fmaxf(all_top[m], stats[w][0][16 * m + l]);
        const float base = finite_or_zero(all_top[m]);
        all_sum[m] = 0.0f;
#pragma unroll
        for (int w = 0; w < kWaves; ++w) all_sum[m] = fmaf(stats[w][1][16 * m + l], __builtin_amdgcn_exp2f(stats[w][0][16 * m + l] - base), all_sum[m]);
        const float shrink = __builtin_amdgcn_exp2f(top[m] - base);
#pragma unroll
        for (int s = 0; s < S; ++s) {
            acc[m][s][0] *= shrink;
            acc[m][s][1] *= shrink;
        }
    }
#pragma unroll
    for (int other = 2; other > 0; other /= 2) {
        if (wave >= other && wave < 2 * other) {
#pragma unroll
            for (int m = 0; m < MT; ++m)
#pragma unroll
                for (int s = 0; s < S; ++s)
#pragma unroll
                    for (int i = 0; i < 8; ++i) exchange[wave - other][(m * S + s) * 8 + i][lane] = acc[m][s][i / 4][i % 4];
        }
        __syncthreads();
        if (wave < other) {
#pragma unroll
            for (int m = 0; m < MT; ++m)
#pragma unroll
                for (int s = 0; s < S; ++s)
#pragma unroll
                    for (int i = 0; i < 8; ++i) acc[m][s][i / 4][i % 4] += exchange[wave][(m * S + s) * 8 + i][lane];
        }
        __syncthreads();
    }
    if (wave != 0) return;
#pragma unroll
    for (int m = 0; m < MT; ++m) {
        const int row = row0 + 16 * m + l;
        if (row >= p.rows) continue;
        const int64_t part = ((static_cast<int64_t>(b) * c.kv_heads + head) * p.rows + row) * p.splits + split;
        const int token = row / p.group;
        const int64_t to = ((static_cast<int64_t>(b) * c.length + token) * p.heads + head * p.group + row % p.group) * D;
        const int at = c.positions[static_cast<int64_t>(b) * c.length + token];
        const float by = 1.0f / all_sum[m];
#pragma unroll
        for (int s = 0; s < S; ++s) {
            float v[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = acc[m][s][i % 2][i / 2];
            if (p.splits > 1) {
                put8<true>(p.part, part * D + 32 * s + 8 * g, v);
            } else {
#pragma unroll
                for (int i = 0; i < 8; ++i) v[i] = at < 0 ? 0.0f : (at >= capacity ? NAN : v[i] * by);
                put8<F32>(p.out, to + 32 * s + 8 * g, v);
            }
        }
        if (p.splits > 1 && g == 0) {
            float* const st = p.part + p.part_rows * D + 2 * part;
            st[0] = all_top[m];
            st[1] = all_sum[m];
        }
    }
}

// The splits of a row joined: D / 8 lanes a row.
template <int D, bool F32>
__global__ __launch_bounds__(256) void kv4_join_kernel(AttentionArgs p) {
    constexpr int kLanes = D / 8;
    const int64_t idx = static_cast<int64_t>(blockIdx.x) * (256 / kLanes) + threadIdx.x / kLanes;  // (sequence, key head, row)
    const int lane = threadIdx.x % kLanes;
    const Cache& c = p.c;
    if (idx >= static_cast<int64_t>(c.batch) * c.kv_heads * p.rows) return;
    const int64_t bh = idx / p.rows;
    const int row = static_cast<int>(idx - bh * p.rows), head = static_cast<int>(bh % c.kv_heads), b = static_cast<int>(bh / c.kv_heads);
    const int token = row / p.group;
    const float* const st = p.part + p.part_rows * D + 2 * idx * p.splits;
    float top = -INFINITY;
    for (int i = 0; i < p.splits; ++i) top = fmaxf(top, st[2 * i]);
    const float base = finite_or_zero(top);
    float sum = 0.0f, v[8] = {0, 0, 0, 0, 0, 0, 0, 0};
    for (int i = 0; i < p.splits; ++i) {
        const float by = __builtin_amdgcn_exp2f(st[2 * i] - base);
        const float* const from = p.part + (idx * p.splits + i) * D + 8 * lane;
        const f32x4 lo = *reinterpret_cast<const f32x4*>(from), hi = *reinterpret_cast<const f32x4*>(from + 4);
        sum = fmaf(st[2 * i + 1], by, sum);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            v[j] = fmaf(lo[j], by, v[j]);
            v[4 + j] = fmaf(hi[j], by, v[4 + j]);
        }
    }
    const int at = c.positions[static_cast<int64_t>(b) * c.length + token];
    const float by = 1.0f / sum;
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = at < 0 ? 0.0f : (at >= c.width * c.page_size ? NAN : v[j] * by);
    put8<F32>(p.out, ((static_cast<int64_t>(b) * c.length + token) * p.heads + head * p.group + row % p.group) * D + 8 * lane, v);
}

// ------------------------------------------------------------- host

bool dim_ok(int64_t dim) { return dim == 32 || dim == 64 || dim == 128 || dim == 256; }

mlk_status cache_of(Cache& c, uint8_t* bytes, int64_t pages, int64_t page_size, int64_t kv_heads, int64_t dim, const int32_t* table,
                    int64_t width, const int32_t* positions, int64_t batch, int64_t length) {
    MLK_CHECK(batch >= 0 && length >= 0 && kv_heads > 0, "invalid cache geometry");
    MLK_CHECK(dim_ok(dim), "head_dim must be 32, 64, 128 or 256");
    MLK_CHECK(page_size > 0 && page_size % kRun == 0 && page_size <= 1024, "page_size must be a multiple of 16, at most 1024");
    MLK_CHECK(pages > 0 && pages < (int64_t{1} << 31), "the cache must have between 1 and 2^31 - 1 pages");
    MLK_CHECK(width > 0 && width <= (int64_t{1} << 30) / page_size, "page_table must hold between 1 and 2^30 / page_size pages a sequence");
    MLK_CHECK(kv_heads < (int64_t{1} << 20) && batch < (int64_t{1} << 31) && length < (int64_t{1} << 31) && batch * length < (int64_t{1} << 36),
              "too many heads, sequences or tokens");
    c = Cache{};
    c.bytes = bytes;
    c.record = page_size * (dim + dim / 16);
    c.pages = static_cast<int32_t>(pages);
    c.kv_heads = static_cast<int32_t>(kv_heads);
    c.page_size = static_cast<int32_t>(page_size);
    c.runs = static_cast<int32_t>(page_size / kRun);
    c.magic = c.runs == 1 ? 0 : static_cast<uint32_t>(((int64_t{1} << 32) + c.runs - 1) / c.runs);
    c.table = table;
    c.width = static_cast<int32_t>(width);
    c.positions = positions;
    c.batch = static_cast<int32_t>(batch);
    c.length = static_cast<int32_t>(length);
    if (batch == 0 || length == 0) return MLK_OK;
    MLK_CHECK(bytes && table && positions, "null tensor pointer");
    MLK_CHECK((reinterpret_cast<uintptr_t>(bytes) & 15) == 0, "the cache must be 16-byte aligned");
    return MLK_OK;
}

// Rows of all (sequence, key head) pairs below 2^31: every count of the plan then fits.
bool rows_fit(int64_t batch, int64_t length, int64_t heads, int64_t kv_heads) {
    if (batch <= 0 || length <= 0 || kv_heads <= 0) return true;  // nothing to do, or refused as geometry
    const int64_t most = int64_t{1} << 31;
    return batch < most && length < (most >> 1) && heads < (int64_t{1} << 20) && length * (heads / kv_heads) < (most >> 1) && batch * length < most &&
           batch * length * heads < most;
}

struct Plan {
    int mt;
    int64_t row_tiles, splits, rows, part_rows;
    size_t bytes;
};
Plan plan_of(int64_t batch, int64_t length, int64_t heads, int64_t kv_heads, int64_t dim, int64_t capacity) {
    Plan t{};
    t.rows = length * (heads / kv_heads);
    t.mt = 1;
    t.row_tiles = ceil_div(t.rows, 16 * t.mt);
    const int64_t blocks = std::max<int64_t>(1, batch * kv_heads * t.row_tiles), tiles = ceil_div(capacity, kTile);
    t.splits = std::max<int64_t>(1, std::min(ceil_div(1024, blocks), tiles / (2 * kWaves)));
    t.part_rows = batch * kv_heads * t.rows * t.splits;
    t.bytes = t.splits > 1 ? static_cast<size_t>(t.part_rows) * (dim + 2) * sizeof(float) : 0;
    return t;
}

template <int D, bool F32>
void launch_attention(const AttentionArgs& p, const Plan& t, hipStream_t s) {
    const int64_t blocks = int64_t{p.c.batch} * p.c.kv_heads * t.row_tiles * t.splits;
    hipLaunchKernelGGL((kv4_attention_kernel<D, F32, 1>), dim3(static_cast<unsigned>(blocks)), dim3(kWaves * 64), 0, s, p);
    if (t.splits > 1) {
        const int64_t rows = int64_t{p.c.batch} * p.c.kv_heads * p.rows;
        hipLaunchKernelGGL((kv4_join_kernel<D, F32>), dim3(static_cast<unsigned>(ceil_div(rows, 256 / (D / 8)))), dim3(256), 0, s, p);
    }
}

template <bool F32>
void launch_attention(int64_t dim, const AttentionArgs& p, const Plan& t, hipStream_t s) {
    if (dim == 32) launch_attention<32, F32>(p, t, s);
    if (dim == 64) launch_attention<64, F32>(p, t, s);
    if (dim == 128) launch_attention<128, F32>(p, t, s);
    if (dim == 256) launch_attention<256, F32>(p, t, s);
}

}  // namespace
}  // namespace mlk

using namespace mlk;

extern "C" mlk_status mlk_kv4_append(const void* k, const int64_t* k_strides, const void* v, const int64_t* v_strides, int32_t dtype,
                                     int64_t batch, int64_t length, int64_t kv_heads, int64_t head_dim, uint8_t* cache,
                                     int64_t pages, int64_t page_size, const int32_t* page_table, int64_t table_width,
                                     const int32_t* positions, mlk_stream_t stream) {
    MLK_CHECK(dtype == MLK_DTYPE_F32 || dtype == MLK_DTYPE_BF16, "dtype must be f32 or bf16");
    Cache c;
    const mlk_status status = cache_of(c, cache, pages, page_size, kv_heads, head_dim, page_table, table_width, positions, batch, length);
    if (status != MLK_OK || batch == 0 || length == 0) return status;
    MLK_CHECK(k && k_strides && v && v_strides, "null tensor pointer");
    const int64_t blocks = ceil_div(batch * length * kv_heads * (head_dim / kGroup), 256);
    MLK_CHECK(blocks < (int64_t{1} << 31), "too many tokens for one launch");
    const Rows3 kr{k, k_strides[0], k_strides[1], k_strides[2]}, vr{v, v_strides[0], v_strides[1], v_strides[2]};
    const dim3 grid(static_cast<unsigned>(blocks), 2);
    hipStream_t s = reinterpret_cast<hipStream_t>(stream);
    if (dtype == MLK_DTYPE_F32) {
        hipLaunchKernelGGL(kv4_append_kernel<true>, grid, dim3(256), 0, s, c, kr, vr, static_cast<int>(head_dim));
    } else {
        hipLaunchKernelGGL(kv4_append_kernel<false>, grid, dim3(256), 0, s, c, kr, vr, static_cast<int>(head_dim));
    }
    return launch_status("kv4 append");
}

extern "C" mlk_status mlk_kv4_read(const uint8_t* cache, int64_t pages, int64_t page_size, const int32_t* page_table, int64_t table_width,
                                   const int32_t* positions, int64_t batch, int64_t length, int64_t kv_heads, int64_t head_dim,
                                   int32_t dtype, void* k, void* v, mlk_stream_t stream) {
    MLK_CHECK(dtype == MLK_DTYPE_F32 || dtype == MLK_DTYPE_BF16, "dtype must be f32 or bf16");
    Cache c;
    const mlk_status status = cache_of(c, const_cast<uint8_t*>(cache), pages, page_size, kv_heads, head_dim, page_table, table_width,
                                       positions, batch, length);
    if (status != MLK_OK || batch == 0 || length == 0) return status;
    MLK_CHECK(k && v, "null tensor pointer");
    const int64_t blocks = ceil_div(batch * length * kv_heads * (head_dim / kGroup), 256);
    MLK_CHECK(blocks < (int64_t{1} << 31), "too many tokens for one launch");
    const dim3 grid(static_cast<unsigned>(blocks), 2);
    hipStream_t s = reinterpret_cast<hipStream_t>(stream);
    if (dtype == MLK_DTYPE_F32) {
        hipLaunchKernelGGL(kv4_read_kernel<true>, grid, dim3(256), 0, s, c, k, v, static_cast<int>(head_dim));
    } else {
        hipLaunchKernelGGL(kv4_read_kernel<false>, grid, dim3(256), 0, s, c, k, v, static_cast<int>(head_dim));
    }
    return launch_status("kv4 read");
}

extern "C" size_t mlk_kv4_attention_workspace_bytes(int64_t batch, int64_t length, int64_t heads, int64_t kv_heads, int64_t head_dim,
                                                    int64_t page_size, int64_t table_width) {
    if (batch <= 0 || length <= 0 || kv_heads <= 0 || heads <= 0 || heads % kv_heads != 0 || !dim_ok(head_dim) || page_size <= 0 ||
        page_size > 1024 || !rows_fit(batch, length, heads, kv_heads) || table_width <= 0 || table_width > (int64_t{1} << 30) / page_size)
        return 0;
    return plan_of(batch, length, heads, kv_heads, head_dim, page_size * table_width).bytes;
}

extern "C" mlk_status mlk_kv4_attention(const void* q, const int64_t* q_strides, int32_t dtype, int64_t batch, int64_t length,
                                        int64_t heads, int64_t kv_heads, int64_t head_dim, const uint8_t* cache, int64_t pages,
                                        int64_t page_size, const int32_t* page_table, int64_t table_width, const int32_t* positions,
                                        double scale, void* out, void* workspace, size_t workspace_bytes, mlk_stream_t stream) {
    MLK_CHECK(dtype == MLK_DTYPE_F32 || dtype == MLK_DTYPE_BF16, "dtype must be f32 or bf16");
    MLK_CHECK(kv_heads <= 0 || (heads > 0 && heads % kv_heads == 0), "heads must be a multiple of kv_heads");
    MLK_CHECK(rows_fit(batch, length, heads, kv_heads), "too many tokens for one launch");
    AttentionArgs p{};
    const mlk_status status = cache_of(p.c, const_cast<uint8_t*>(cache), pages, page_size, kv_heads, head_dim, page_table, table_width,
                                       positions, batch, length);
    if (status != MLK_OK) return status;
    if (batch == 0 || length == 0) return MLK_OK;
    MLK_CHECK(q && q_strides && out, "null tensor pointer");
    MLK_CHECK((reinterpret_cast<uintptr_t>(out) & 15) == 0, "out must be 16-byte aligned");
    const Plan t = plan_of(batch, length, heads, kv_heads, head_dim, page_size * table_width);
    MLK_CHECK(batch * kv_heads * t.row_tiles * t.splits < (int64_t{1} << 31), "too many tokens for one launch");
    MLK_CHECK(workspace_bytes >= t.bytes && (t.bytes == 0 || (workspace && (reinterpret_cast<uintptr_t>(workspace) & 15) == 0)),
              "workspace must be 16-byte aligned and hold mlk_kv4_attention_workspace_bytes");
    p.q = q;
    p.q_bs = q_strides[0];
    p.q_ts = q_strides[1];
    p.q_hs = q_strides[2];
    p.heads = static_cast<int32_t>(heads);
    p.group = static_cast<int32_t>(heads / kv_heads);
    p.rows = static_cast<int32_t>(t.rows);
    p.row_tiles = static_cast<int32_t>(t.row_tiles);
    p.splits = static_cast<int32_t>(t.splits);
    p.scale_log2 = static_cast<float>(scale * 1.4426950408889634);
    p.out = out;
    p.part = static_cast<float*>(workspace);
    p.part_rows = t.part_rows;
    if (dtype == MLK_DTYPE_F32) {
        launch_attention<true>(head_dim, p, t, reinterpret_cast<hipStream_t>(stream));
    } else {
        launch_attention<false>(head_dim, p, t, reinterpret_cast<hipStream_t>(stream));
    }
    return launch_status("kv4 attention");
}
