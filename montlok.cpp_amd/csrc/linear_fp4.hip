// y = x W^T + b with four-bit weights (groups of 32 under a power of two), on
// the bf16 matrix cores with fp32 accumulation. Every weight below 2^128 is
// exact in bf16, a bf16 x is too, and an fp32 x from 2^-110 on is the exact sum
// of three bf16 values, so the only rounding is that of the sums.
#include <algorithm>
#include <type_traits>

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

// Four results side by side; `first` a multiple of 4 from an aligned base.
template <bool F32>
__device__ __forceinline__ void put4(void* out, int64_t first, const float (&y)[4]) {
    if constexpr (F32) {
        *reinterpret_cast<f32x4*>(static_cast<float*>(out) + first) = f32x4{y[0], y[1], y[2], y[3]};
    } else {
        *reinterpret_cast<u32x2*>(static_cast<uint16_t*>(out) + first) =
            u32x2{float_to_bf16(y[0]) | float_to_bf16(y[1]) << 16, float_to_bf16(y[2]) | float_to_bf16(y[3]) << 16};
    }
}

// Few rows: a block takes 16 NT columns of y (rows of W) by 16 rows, its kWaves waves interleaved blocks of 256 k. A wave
// loads its block of W whole lines at a time (128 bytes of 8 rows an instruction; the order of the matrix instruction, lane
// (g, l) = group of row l, straight from memory costs a cache access a lane and bounded this kernel: 31 us where it takes
// 8 now) and turns it in its own piece of LDS. x comes the same way (TURN), or, for up to kFew rows, straight to the lanes
// whose row exists. Past K a lane's x is zero (its W is that of the last group, which counts anyway). An infinity or a NaN
// in fp32 x makes the quick planes NaN; a wave that sees one in its sums forms them again.
//
// One bf16 row is bound by the reading of W (12288 x 4096: 7.4 us, 3.6 TB/s); 16 rows of fp32 by what a block does for
// each of its columns' x, which it reads whole from L2 and takes apart (4100 x 4096: 9.5 us, 0.9 TB/s).
constexpr int kFew = 4, kWaves = 8, kSteps = 2;
template <bool F32, bool TURN, int NT>
__global__ __launch_bounds__(kWaves * 64) void linear_fp4_stream_kernel(Fp4LinearArgs p) {
    constexpr int KW = kWaves, U = kSteps;
    constexpr int P = F32 ? 3 : 1, kPieces = F32 ? 8 : 4;  // 16-byte pieces of 32 elements of x
    constexpr int kRow = 4 * U;                            // groups of a row that an iteration takes, 4 a matrix instruction
    constexpr int kTurn = 16 * kRow * NT + (TURN ? 16 * 4 * kPieces : 0), kPart = (16 * (16 * NT + 1) + 3) / 4;
    __shared__ u32x4 lds[KW][kTurn > kPart ? kTurn : kPart];
    const int wave = threadIdx.x / 64, lane = threadIdx.x & 63, g = lane >> 4, l = lane & 15;
    const int n0 = blockIdx.x * (16 * NT), m0 = blockIdx.y * 16, groups = p.K / kGroup;
    const uint8_t* const codes = p.codes + static_cast<int64_t>(n0) * (p.K / 2);
    const uint8_t* const scales = p.scales + static_cast<int64_t>(n0) * groups;
    const char* const xs = static_cast<const char*>(p.x) + static_cast<int64_t>(m0) * p.x_stride * (F32 ? 4 : 2);
    u32x4* const turn_w = lds[wave];
    u32x4* const turn_x = lds[wave] + 16 * kRow * NT;
    f32x4 acc[NT];
    auto sum = [&](auto careful) {
#pragma unroll
        for (int n = 0; n < NT; ++n) acc[n] = f32x4{0, 0, 0, 0};
#pragma unroll 1
        for (int group0 = kRow * wave; group0 < groups; group0 += kRow * KW) {
            u32x4 w[NT][U];
            uint32_t byte[NT][U];
            u32x4 x[U][kPieces];
#pragma unroll
            for (int n = 0; n < NT; ++n) {
#pragma unroll
                for (int t = 0; t < U; ++t) {
                    const int row = min(16 * n + t * (64 / kRow) + lane / kRow, p.N - 1 - n0), group = min(group0 + lane % kRow, groups - 1);
                    w[n][t] = *reinterpret_cast<const u32x4*>(codes + static_cast<int64_t>(row) * (p.K / 2) + 16 * group);
                }
                const uint8_t* const from = scales + static_cast<int64_t>(min(16 * n + l, p.N - 1 - n0)) * groups;
                if (group0 + kRow <= groups) {
                    typedef uint32_t Scales __attribute__((ext_vector_type(U), aligned(1)));
                    const Scales v = *reinterpret_cast<const Scales*>(from + group0);
#pragma unroll
                    for (int u = 0; u < U; ++u) byte[n][u] = v[u] >> (8 * g);
                } else {
#pragma unroll
                    for (int u = 0; u < U; ++u) byte[n][u] = from[min(group0 + 4 * u + g, groups - 1)];
                }
            }
#pragma unroll
            for (int u = 0; u < U; ++u) {
                if constexpr (TURN) {
                    // 4 kPieces pieces of a row side by side; past K the last of the row, zeroed below.
#pragma unroll
                    for (int i = 0; i < kPieces; ++i) {
                        const int at = 64 * i + lane, row = min(at / (4 * kPieces), p.rows - 1 - m0);
                        const int piece = min((group0 + 4 * u) * kPieces + at % (4 * kPieces), groups * kPieces - 1);
                        x[u][i] = *reinterpret_cast<const u32x4_any*>(xs + static_cast<int64_t>(row) * p.x_stride * (F32 ? 4 : 2) + 16 * piece);
                    }
                } else {
#pragma unroll
                    for (int i = 0; i < kPieces; ++i) x[u][i] = u32x4{0, 0, 0, 0};
                    if (group0 + 4 * u + g < groups && m0 + l < p.rows) {
#pragma unroll
                        for (int i = 0; i < kPieces; ++i)
                            x[u][i] = reinterpret_cast<const u32x4_any*>(xs + static_cast<int64_t>(l) * p.x_stride * (F32 ? 4 : 2) +
                                                                         16 * kPieces * (group0 + 4 * u + g))[i];
                    }
                }
            }
            __builtin_amdgcn_sched_barrier(0);  // every load of the iteration in flight before the first wait
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int t = 0; t < U; ++t) {
                    const int row = t * (64 / kRow) + lane / kRow;
                    turn_w[(16 * n + row) * kRow + ((lane % kRow) ^ (row % kRow))] = w[n][t];
                }
#pragma unroll
            for (int u = 0; u < U; ++u) {
                if constexpr (TURN) {
                    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
#pragma unroll
                    for (int i = 0; i < kPieces; ++i) {
                        const int at = 64 * i + lane, row = at / (4 * kPieces), piece = at % (4 * kPieces);
                        const bool inside = (group0 + 4 * u) * kPieces + piece < groups * kPieces;
                        turn_x[row * (4 * kPieces) + (piece ^ row)] = inside ? x[u][i] : u32x4{0, 0, 0, 0};
                    }
                }
                __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
                u32x4 ws[NT];
                float scale[NT];
#pragma unroll
                for (int n = 0; n < NT; ++n) {
                    ws[n] = turn_w[(16 * n + l) * kRow + ((4 * u + g) ^ (l % kRow))];
                    scale[n] = scale_of(byte[n][u] & 0xFF);
                }
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    u32x4 piece[F32 ? 2 : 1];
#pragma unroll
                    for (int j = 0; j < (F32 ? 2 : 1); ++j) {
                        const int at = (F32 ? 2 * i : i) + j;
                        piece[j] = TURN ? turn_x[l * (4 * kPieces) + ((kPieces * g + at) ^ l)] : x[u][at];
                    }
                    bf16x8 xv[P];
                    if constexpr (F32) {
                        float v[8];
#pragma unroll
                        for (int j = 0; j < 8; ++j) v[j] = __uint_as_float(piece[j / 4][j % 4]);
                        planes_of<decltype(careful)::value>(v, xv);
                    } else {
                        xv[0] = __builtin_bit_cast(bf16x8, piece[0]);
                    }
#pragma unroll
                    for (int n = 0; n < NT; ++n) {
                        const bf16x8 wv = fp4_octet(ws[n][i], scale[n]);
#pragma unroll
                        for (int j = P - 1; j >= 0; --j) acc[n] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(wv, xv[j], acc[n], 0, 0, 0);
                    }
                }
            }
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        }
    };
    sum(std::false_type{});
    if constexpr (F32) {
        bool odd = false;
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int r = 0; r < 4; ++r) odd = odd || acc[n][r] != acc[n][r];
        if (__ballot(odd) != 0) sum(std::true_type{});
    }
    __syncthreads();
    float* const part = reinterpret_cast<float*>(lds);  // [KW][16][16 NT + 1]
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int r = 0; r < 4; ++r) part[(wave * 16 + l) * (16 * NT + 1) + 16 * n + 4 * g + r] = acc[n][r];
    __syncthreads();
    for (int at = threadIdx.x; at < 256 * NT; at += KW * 64) {
        const int row = at / (16 * NT), col = at % (16 * NT);
        if (m0 + row >= p.rows || n0 + col >= p.N) continue;
        float y = part[row * (16 * NT + 1) + col];
#pragma unroll
        for (int w = 1; w < KW; ++w) y += part[(w * 16 + row) * (16 * NT + 1) + col];
        if (p.bias != nullptr) y += p.bias[n0 + col];
        Element<F32>::put(p.out, static_cast<int64_t>(m0 + row) * p.N + n0 + col, y);
    }
}

// More rows: a block of WN KW waves (two by four) takes 16 NT WN columns of y by 16 MT rows. WN waves share the columns and KW the k of
// a step, 64 each, so that a wave's products need MT P LDS reads for NT MT P matrix instructions and every weight is
// converted once. Codes, scales and x are staged in LDS a step ahead, from registers loaded the step before that, x as
// bf16 (three planes for fp32): loaded in rows, 8 lanes to 128 bytes, read in operand order. Unit u (8 consecutive k) of
// row m of x lies at u * rows + (m ^ (u & 7)), piece c (32 codes) of row n of W at n * pieces + (c ^ (n & 7)): what
// 8 lanes write, or read, together lies in different banks. The KW partial sums meet in LDS.
//
// 256 rows of bf16, 8192 x 8192: 38 us, 900 TFLOP/s, 69% of what a large library product reaches. While a CU is at work its
// matrix cores are busy for 39% of the time, its vector units issue for 28%, its LDS is busy for 39%, and one block a CU
// leaves little to overlap them with; a step staged after its products, or two steps in registers, took 2 to 6 us longer.
template <bool F32, int NT, int MT>
struct TileShape {
    static constexpr int WN = 2, KW = 4;
    static constexpr int P = F32 ? 3 : 1, kRows = 16 * MT, kCols = 16 * NT * WN, kThreads = 64 * WN * KW;
    static constexpr int kK = 64 * KW, kUnits = kK / 8, kPieces = kK / kGroup;
    static constexpr int kX = P * kUnits * kRows, kW = kCols * kPieces, kScales = kCols * kPieces / 16;  // 16-byte units a buffer
    static constexpr int kBuffer = kX + kW + kScales;
    // A wave's partial sums of the tiles t = n MT + m that others finish (t mod KW is the wave that does).
    static constexpr int kParts = NT * MT - NT * MT / KW;
    static constexpr __device__ int part_of(int kw, int tile) { return tile - tile / KW - (tile % KW > kw ? 1 : 0); }
    static constexpr size_t kLds = std::max(size_t{2} * kBuffer * 16, size_t{WN} * KW * kParts * 1024);
};
template <bool F32, int NT, int MT>
__global__ __launch_bounds__((TileShape<F32, NT, MT>::kThreads)) void linear_fp4_tile_kernel(Fp4LinearArgs p, int n_tiles, int m_tiles) {
    using T = TileShape<F32, NT, MT>;
    constexpr int WN = T::WN, KW = T::KW, P = T::P, kBytes = F32 ? 4 : 2;
    constexpr int kXLoads = T::kRows * T::kUnits / T::kThreads, kWLoads = (T::kW + T::kThreads - 1) / T::kThreads;
    static_assert(kXLoads * T::kThreads == T::kRows * T::kUnits && T::kThreads % T::kUnits == 0 && T::kPieces == 8);
    extern __shared__ u32x4 lds[];
    // Blocks of the same columns side by side on one XCD: W comes from memory once, then from that L2.
    const int xcd = blockIdx.x & 7, index = blockIdx.x >> 3;
    const int n_tile = xcd + 8 * (index / m_tiles), m_tile = index % m_tiles;
    if (n_tile >= n_tiles) return;
    const int wave = threadIdx.x / 64, lane = threadIdx.x & 63, g = lane >> 4, l = lane & 15;
    const int wn = wave % WN, kw = wave / WN;
    const int n0 = n_tile * T::kCols, m0 = m_tile * T::kRows;

    // Offsets from the block's first rows in 32 bits: the rows' once, the step's added.
    const int groups = p.K / kGroup;
    const uint8_t* const codes = p.codes + static_cast<int64_t>(n0) * (p.K / 2);
    const uint8_t* const scales = p.scales + static_cast<int64_t>(n0) * groups;
    const char* const xs = static_cast<const char*>(p.x) + static_cast<int64_t>(m0) * p.x_stride * kBytes;
    const int unit = threadIdx.x % T::kUnits;  // of x, the same in every load
    const int x_first = static_cast<int>(threadIdx.x) / T::kUnits, x_rows = T::kThreads / T::kUnits;

    struct {  // what a thread has loaded of the step that is staged next
        u32x4 w[kWLoads], x[kXLoads][F32 ? 2 : 1];
        u32x2 scale_bytes;
    } ahead;
    auto load = [&](int step) {
        // Past K: the last group's, x is zeroed when it is staged, and that group counts anyway.
#pragma unroll
        for (int i = 0; i < kWLoads; ++i) {
            const int at = i * T::kThreads + static_cast<int>(threadIdx.x), row = at / T::kPieces, piece = at % T::kPieces;
            if (T::kW % T::kThreads != 0 && at >= T::kW) break;
            const uint32_t offset = static_cast<uint32_t>(min(row, p.N - 1 - n0)) * static_cast<uint32_t>(groups) +
                                    static_cast<uint32_t>(min(step * T::kPieces + piece, groups - 1));
            ahead.w[i] = *reinterpret_cast<const u32x4*>(codes + 16 * static_cast<uint64_t>(offset));
        }
        if (static_cast<int>(threadIdx.x) < T::kCols) {
            const uint8_t* const from = scales + static_cast<int64_t>(min(static_cast<int>(threadIdx.x), p.N - 1 - n0)) * groups;
            const int first = step * T::kPieces;
            typedef uint32_t u32x2_any __attribute__((ext_vector_type(2), aligned(1)));
            if (first + T::kPieces <= groups) ahead.scale_bytes = *reinterpret_cast<const u32x2_any*>(from + first);
            if (first + T::kPieces > groups) {
#pragma unroll
                for (int i = 0; i < T::kPieces / 4; ++i) {
                    ahead.scale_bytes[i] = 0;
#pragma unroll
                    for (int j = 0; j < 4; ++j) ahead.scale_bytes[i] |= static_cast<uint32_t>(from[min(first + 4 * i + j, groups - 1)]) << (8 * j);
                }
            }
        }
        const int kx = min(step * T::kK + 8 * unit, p.K - 8) * kBytes;
#pragma unroll
        for (int i = 0; i < kXLoads; ++i) {
            const uint32_t row = static_cast<uint32_t>(min(x_first + i * x_rows, p.rows - 1 - m0));
            const char* const from = xs + (row * static_cast<uint32_t>(p.x_stride * kBytes) + kx);
#pragma unroll
            for (int j = 0; j < (F32 ? 2 : 1); ++j) ahead.x[i][j] = reinterpret_cast<const u32x4_any*>(from)[j];
        }
    };
    auto stage = [&](int step, int buffer) {
        u32x4* const to_x = lds + buffer * T::kBuffer;
        u32x4* const to_w = to_x + T::kX;
        if (step * T::kK + T::kK > p.K && step * T::kK + 8 * unit >= p.K) {
#pragma unroll
            for (int i = 0; i < kXLoads; ++i)
#pragma unroll
                for (int j = 0; j < (F32 ? 2 : 1); ++j) ahead.x[i][j] = u32x4{0, 0, 0, 0};
        }
#pragma unroll
        for (int i = 0; i < kXLoads; ++i) {
            const int row = x_first + i * x_rows;
            u32x4* const to = to_x + unit * T::kRows + (row ^ (unit & 7));
            if constexpr (F32) {
                float v[8];
#pragma unroll
                for (int j = 0; j < 8; ++j) v[j] = __uint_as_float(ahead.x[i][j / 4][j % 4]);
                bf16x8 planes[3];
                planes_of<true>(v, planes);
#pragma unroll
                for (int j = 0; j < 3; ++j) to[j * (T::kUnits * T::kRows)] = __builtin_bit_cast(u32x4, planes[j]);
            } else {
                to[0] = ahead.x[i][0];
            }
        }
#pragma unroll
        for (int i = 0; i < kWLoads; ++i) {
            const int at = i * T::kThreads + static_cast<int>(threadIdx.x), row = at / T::kPieces, piece = at % T::kPieces;
            if (T::kW % T::kThreads != 0 && at >= T::kW) break;
            to_w[row * T::kPieces + (piece ^ (row & 7))] = ahead.w[i];
        }
        if (static_cast<int>(threadIdx.x) < T::kCols) {
            uint32_t* const to = reinterpret_cast<uint32_t*>(to_w + T::kW) + threadIdx.x * (T::kPieces / 4);
#pragma unroll
            for (int i = 0; i < T::kPieces / 4; ++i) to[i] = ahead.scale_bytes[i];
        }
    };

    f32x4 acc[NT][MT];
#pragma unroll
    for (int i = 0; i < NT; ++i)
#pragma unroll
        for (int m = 0; m < MT; ++m) acc[i][m] = f32x4{0, 0, 0, 0};
    const int steps = (p.K + T::kK - 1) / T::kK;
    load(0);
    stage(0, 0);
    if (steps > 1) load(1);
    // A lane's 16 elements of the wave's 64 are k = 64 kw + 16 g ..: half (g & 1) of piece 2 kw + g / 2, units 8 kw + 2 g
    // and the next.
    const int piece = 2 * kw + (g >> 1);
    auto advance = [&](int step, auto place) {  // place: step modulo 2
        constexpr int kPlace = decltype(place)::value;
        const u32x4* const from_x = lds + kPlace * T::kBuffer;
        const u32x4* const from_w = from_x + T::kX;
        __syncthreads();
        if (step + 1 < steps) stage(step + 1, 1 - kPlace);
        if (step + 2 < steps) load(step + 2);
        __builtin_amdgcn_sched_barrier(0);
        bf16x8 xv[2][MT][P];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int u = 8 * kw + 2 * g + i;
#pragma unroll
            for (int m = 0; m < MT; ++m)
#pragma unroll
                for (int j = 0; j < P; ++j)
                    xv[i][m][j] = __builtin_bit_cast(bf16x8, from_x[j * (T::kUnits * T::kRows) + u * T::kRows + 16 * m + (l ^ (u & 7))]);
        }
        u32x2 codes_of[NT];
        float scale[NT];
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            const int row = 16 * (NT * wn + n) + l;
            codes_of[n] = reinterpret_cast<const u32x2*>(from_w + row * T::kPieces + (piece ^ (row & 7)))[g & 1];
            scale[n] = scale_of(reinterpret_cast<const uint8_t*>(from_w + T::kW)[row * T::kPieces + piece]);
        }
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                const bf16x8 wv = fp4_octet(codes_of[n][i], scale[n]);
#pragma unroll
                for (int j = P - 1; j >= 0; --j)
#pragma unroll
                    for (int m = 0; m < MT; ++m) acc[n][m] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(wv, xv[i][m][j], acc[n][m], 0, 0, 0);
            }
    };
    for (int step = 0; step < steps; step += 2) {
        advance(step, std::integral_constant<int, 0>{});
        if (step + 1 < steps) advance(step + 1, std::integral_constant<int, 1>{});
    }

    __syncthreads();
    float* const part = reinterpret_cast<float*>(lds) + wn * KW * T::kParts * 256 + lane;
#pragma unroll
    for (int t = 0; t < NT * MT; ++t)
        if (t % KW != kw)
#pragma unroll
            for (int r = 0; r < 4; ++r) part[(kw * T::kParts + T::part_of(kw, t)) * 256 + r * 64] = acc[t / MT][t % MT][r];
    __syncthreads();
#pragma unroll
    for (int n = 0; n < NT; ++n) {
        const int col = n0 + 16 * (NT * wn + n) + 4 * g;
#pragma unroll
        for (int m = 0; m < MT; ++m) {
            const int row = m0 + 16 * m + l, t = n * MT + m;
            if (t % KW != kw) continue;
            float y[4];
#pragma unroll
            for (int r = 0; r < 4; ++r) y[r] = acc[n][m][r];
#pragma unroll
            for (int other = 0; other < KW; ++other)
                if (other != t % KW)
#pragma unroll
                    for (int r = 0; r < 4; ++r) y[r] += part[(other * T::kParts + T::part_of(other, t)) * 256 + r * 64];
            if (row >= p.rows || col >= p.N) continue;
            if (p.bias != nullptr) {
#pragma unroll
                for (int r = 0; r < 4; ++r) y[r] += p.bias[min(col + r, p.N - 1)];
            }
            const int64_t to = static_cast<int64_t>(row) * p.N + col;
            if (p.N % 4 == 0) {
                put4<F32>(p.out, to, y);
            } else {
#pragma unroll
                for (int r = 0; r < 4; ++r)
                    if (col + r < p.N) Element<F32>::put(p.out, to + r, y[r]);
            }
        }
    }
}

template <bool F32, int NT, int MT>
void launch_tile(const Fp4LinearArgs& p, hipStream_t s) {
    using T = TileShape<F32, NT, MT>;
    static_assert(T::kLds <= 160 * 1024);
    const int64_t n_tiles = ceil_div(p.N, T::kCols), m_tiles = ceil_div(p.rows, T::kRows);
    hipLaunchKernelGGL((linear_fp4_tile_kernel<F32, NT, MT>), dim3(static_cast<unsigned>(8 * ceil_div(n_tiles, 8) * m_tiles)),
                       dim3(T::kThreads), T::kLds, s, p, static_cast<int>(n_tiles), static_cast<int>(m_tiles));
}
template <bool F32, int NT>
void launch_stream(const Fp4LinearArgs& p, hipStream_t s) {
    const dim3 grid(static_cast<unsigned>(ceil_div(p.N, 16 * NT)), static_cast<unsigned>(ceil_div(p.rows, 16)));
    if (p.rows <= kFew) {
        hipLaunchKernelGGL((linear_fp4_stream_kernel<F32, false, NT>), grid, dim3(kWaves * 64), 0, s, p);
    } else {
        hipLaunchKernelGGL((linear_fp4_stream_kernel<F32, true, NT>), grid, dim3(kWaves * 64), 0, s, p);
    }
}

// The forms' times go as the rounds of blocks on 256 CUs. Measured for K = 4096 in bf16 (us, launch included):
//
//   N      rows  stream  64-column tiles  128-column tiles
//   4096    64     9.6        15.0             20.7
//   4096   128    16.7        15.4             21.1
//   4096   256    30.2        16.5             21.7
//   12288   32    17.0        17.4             24.7
//   12288   64    26.7        19.3             25.7
//   12288  128    49          34               26.6
//   12288  256    91          51               48.9
//
// that is 3.7 us for 256 stream blocks of 32 columns and 16 rows (fractions of a round count, blocks are many to a CU),
// 15.5 and 22 for a round of tiles by 64 rows. fp32: 12 for 256 stream blocks of 64 columns, 30 for a round of 128-column
// tiles by 32 rows. A stream block that takes more columns shares what its x costs among them, and leaves CUs idle where
// there are few: the round of 256 blocks of 16, 32 and 64 columns takes 4.0 and 4.9 us in bf16 (2.9 and 3.8 with 4 rows
// and less), 6.7, 8.1 and 11.6 in fp32 (5.2, 6.8 and 9.5). 12288 x 16 rows in bf16: 14.8 us with 16 columns, 11.2 with
// 32; 4096 x 16 rows 6.0 and 6.9; fp32 12288 x 1 row 16.9, 18.2 and 14.5; 4100 x 16 rows 14.2 (257 blocks) and 10.0.
template <bool F32>
void launch(const Fp4LinearArgs& p, hipStream_t s) {
    const int64_t tiles16 = ceil_div(p.rows, 16);
    auto rounds = [&](int64_t cols, int64_t rows) { return static_cast<double>(ceil_div(ceil_div(p.N, cols) * ceil_div(p.rows, rows), 256)); };
    auto full = [&](int64_t cols) { return std::max(1.0, static_cast<double>(ceil_div(p.N, cols) * tiles16) / 256); };
    const bool offsets_fit = p.x_stride < (int64_t{1} << 24);  // a tile's rows of x are addressed in 32 bits
    const bool few = p.rows <= kFew;
    if constexpr (F32) {
        if (offsets_fit && 30 * rounds(128, 32) < 12 * full(64)) return launch_tile<true, 4, 2>(p, s);
        const double by16 = (few ? 5.2 : 6.7) * rounds(16, 16), by32 = (few ? 6.8 : 8.1) * rounds(32, 16), by64 = (few ? 9.5 : 11.6) * rounds(64, 16);
        if (by64 < std::min(by16, by32)) return launch_stream<true, 4>(p, s);
        by16 <= by32 ? launch_stream<true, 1>(p, s) : launch_stream<true, 2>(p, s);
    } else {
        const double stream = 3.7 * full(32), narrow = 15.5 * rounds(64, 64), wide = 22 * rounds(128, 64);
        if (offsets_fit && std::min(narrow, wide) < stream)
            return narrow < wide ? launch_tile<false, 2, 4>(p, s) : launch_tile<false, 4, 4>(p, s);
        (few ? 2.9 : 4.0) * rounds(16, 16) <= (few ? 3.8 : 4.9) * rounds(32, 16) ? launch_stream<false, 1>(p, s) : launch_stream<false, 2>(p, s);
    }
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
    MLK_CHECK(rows < (int64_t{1} << 20) - 16 && in_features < (int64_t{1} << 24) && out_features < (int64_t{1} << 26) &&
                  rows * out_features <= (int64_t{1} << 34),
              "too many rows or features");  // the grids: 65,535 blocks along y, 2^32 threads along x
    MLK_CHECK(x_stride >= 0, "x_stride must not be negative");
    if (rows == 0) return MLK_OK;
    MLK_CHECK(x && codes && scales && out, "null tensor pointer");
    MLK_CHECK((reinterpret_cast<uintptr_t>(codes) & 15) == 0 && (reinterpret_cast<uintptr_t>(out) & 15) == 0,
              "codes and out must be 16-byte aligned");
    Fp4LinearArgs p{x, x_stride, codes, scales, bias, out, static_cast<int32_t>(rows), static_cast<int32_t>(in_features),
                    static_cast<int32_t>(out_features)};
    hipStream_t s = reinterpret_cast<hipStream_t>(stream);
    if (dtype == MLK_DTYPE_F32) {
        launch<true>(p, s);
    } else {
        launch<false>(p, s);
    }
    return launch_status("linear fp4");
}
