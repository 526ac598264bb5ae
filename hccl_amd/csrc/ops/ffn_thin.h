// The forward products for few rows per rank (a decoding step), where the time is that of reading the weights once.
//
// A workgroup takes 16 columns of C (of both weights) of one rank and all its rows, 16 x MB at a time; its eight wavefronts share
// out k in turns of 64 and add up their parts in LDS, in the order of the wavefronts.  Weights go from memory to the matrix
// instruction's registers without LDS: nobody else needs them.  A lane's two chunks of 16 bytes of a turn lie next to each other
// (k = 16 (lane / 16) .. + 15), so that four lanes read a cache line of a row; the same k of the rows of x, which come from the L2.
//
// What bounds it: the weights' way from memory, with too little time to reach its rate.  Block of 1 row x 4096 x 2048 16 us (3.1 TB/s;
// 10.9 and 5.5 us of kernels) where the last-level cache holds the weights, 17.7 (2.8) from memory; 2 ranks 26.5 (3.8), 4 ranks x
// 7168 x 2048 74.5 (4.7).
//
// Limits as in ffn_gemm.h: range-checked loads give zeros behind the last row, column and k.
#pragma once
#include "ops/ffn_gemm.h"

namespace hcclx {
namespace ffn {

constexpr uint32_t kThinWaves = 8;
constexpr uint32_t kTurnK = 64;
// Turns whose loads are on their way together.  (Two, four, eight: 8 ranks x 1 row x 7168 x 2048, for which tiles are taken otherwise,
// second product 67, 80, 113 us; first 95, 93, 104.  More registers leave fewer wavefronts on a CU, and a turn behind the last costs as much as any.  Sixteen
// wavefronts instead of eight: 73 and 101.)
constexpr int kTurnsAhead = 2;

// HALF: eight columns of both weights share a matrix instruction's sixteen, in twice as many workgroups.
template <int DT, int KIND, int MB, bool X8, bool HALF>
__global__ void __launch_bounds__(kThinWaves * 64)
k_ffn_thin(FfnArgs a)
{
    constexpr int kWeights = KIND == kFfnGateUp && !HALF ? 2 : 1;   // fragments of weights
    constexpr uint32_t kCols = HALF ? 8 : 16;
    constexpr int kAhead = HALF ? 2 * kTurnsAhead : kTurnsAhead;    // (of half the bytes)
    static_assert(KIND == kFfnGateUp || (KIND == kFfnDown && !X8 && !HALF), "the forward products");
    __shared__ f32x4 s_part[kThinWaves][MB * kWeights][64];
    __shared__ uint32_t s_rows[2];
    const FfnRows &s = a.rows;
    const uint32_t rank = blockIdx.y;
    const uint32_t wave = uniform(threadIdx.x / 64);
    const uint32_t lane = threadIdx.x & 63;
    // (read together, before the wait for the rows: otherwise the way to the first load is a row of waits)
    const char *const p0 = a.p[0][rank];
    const char *const p1 = a.p[1][rank];
    const char *const p2 = a.p[2][rank];
    asm volatile("" ::"s"(p0), "s"(p1), "s"(p2), "s"(s.counts), "s"(s.per_rank), "s"(s.unit), "s"(s.n), "s"(s.capacity), "s"(s.most), "s"(s.dim),
                 "s"(s.hidden), "s"(a.h), "s"(a.saved), "s"(a.act));
    if (wave == 0) {
        const RankRows mine(s);
        if (lane == rank) {
            s_rows[0] = mine.rows;
            s_rows[1] = mine.start;
        }
    }
    __syncthreads();
    const uint32_t rows = uniform(s_rows[0]);
    const uint32_t start = uniform(s_rows[1]);
    const uint32_t dim = s.dim;
    const uint32_t hidden = s.hidden;
    const uint32_t ks = KIND == kFfnGateUp ? dim : hidden;
    const uint32_t cols = KIND == kFfnGateUp ? hidden : dim;
    const uint32_t n0 = blockIdx.x * kCols;
    const uint32_t w_ld = ks * 2;
    const uint32_t x_ld = X8 ? dim + HCCLX_ROW8_TAIL : ks * 2;
    const uint32_t have = cols - n0 < kCols ? cols - n0 : kCols;
    const Window gate((KIND == kFfnGateUp ? p1 : p0) + static_cast<uint64_t>(n0) * w_ld, have * w_ld);
    const Window up((KIND == kFfnGateUp ? p2 : p0) + static_cast<uint64_t>(n0) * w_ld, have * w_ld);
    const char *x = KIND == kFfnGateUp ? p0 : a.h + static_cast<uint64_t>(start) * w_ld;
    const uint32_t w_row = lane % kCols * w_ld;
    const bool of_up = HALF && lane % 16 >= 8;
    const uint32_t x_row = lane % 16 * x_ld;
    const uint32_t k_in = lane / 16 * 16;
    const uint32_t turns = (ks + kTurnK * kThinWaves - 1) / (kTurnK * kThinWaves);

    for (uint32_t m0 = 0; m0 < rows; m0 += 16 * MB) {
        const uint32_t here = rows - m0 < 16 * MB ? rows - m0 : 16 * MB;
        const Window in(x + static_cast<uint64_t>(m0) * x_ld, here * x_ld);
        f32x4 acc[MB][kWeights];
#pragma unroll
        for (int m = 0; m < MB; ++m) {
#pragma unroll
            for (int w = 0; w < kWeights; ++w) acc[m][w] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
        }
        u32x4 fw[kAhead][kWeights][2];
        u32x4 fu[kAhead][2];
        u32x4 fx[kAhead][MB][X8 ? 1 : 2];
        auto load = [&](uint32_t turn, int to) {
            const uint32_t k = (turn * kThinWaves + wave) * kTurnK + k_in;
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const uint32_t o = k + h * 8 < ks ? w_row + (k + h * 8) * 2 : kOut;
                if constexpr (HALF) {   // (what a lane does not have is zeros)
                    fw[to][0][h] = __builtin_bit_cast(u32x4, gate.load(of_up ? kOut : o));
                    fu[to][h] = __builtin_bit_cast(u32x4, up.load(of_up ? o : kOut));
                } else {
                    fw[to][0][h] = __builtin_bit_cast(u32x4, gate.load(o));
                    if constexpr (kWeights == 2) fw[to][1][h] = __builtin_bit_cast(u32x4, up.load(o));
                }
            }
#pragma unroll
            for (int m = 0; m < MB; ++m) {
                const uint32_t row = x_row + m * 16 * x_ld;
                if constexpr (X8) {
                    fx[to][m][0] = __builtin_bit_cast(u32x4, in.load(k < ks ? row + k : kOut));   // (dim is a multiple of 16)
                } else {
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        fx[to][m][h] = __builtin_bit_cast(u32x4, in.load(k + h * 8 < ks ? row + (k + h * 8) * 2 : kOut));
                    }
                }
            }
        };
        auto multiply = [&](int from) {
#pragma unroll
            for (int m = 0; m < MB; ++m) {
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const u32x4 f = X8 ? widen8<DT>(fx[from][m][0][2 * h], fx[from][m][0][2 * h + 1]) : fx[from][m][X8 ? 0 : h];
#pragma unroll
                    for (int w = 0; w < kWeights; ++w) {
                        acc[m][w] = Mma<DT>::run(HALF ? fw[from][w][h] | fu[from][h] : fw[from][w][h], f, acc[m][w]);
                    }
                }
            }
        };
#pragma unroll
        for (int t = 0; t < kAhead; ++t) load(t, t);
        for (uint32_t turn = 0; turn < turns; turn += kAhead) {
#pragma unroll
            for (int t = 0; t < kAhead; ++t) {
                multiply(t);
                load(turn + t + kAhead, t);   // (behind the last turn: nothing, which loads zeros)
            }
        }

        __syncthreads();   // the parts of the rows before have been read
#pragma unroll
        for (int m = 0; m < MB; ++m) {
#pragma unroll
            for (int w = 0; w < kWeights; ++w) s_part[wave][m * kWeights + w][lane] = acc[m][w];
        }
        __syncthreads();
        if (wave >= MB) continue;
        if (HALF && lane >= 32) continue;   // lanes 0 .. 31 have the gate's columns and get up's from the others' places
        constexpr int kSums = KIND == kFfnGateUp ? 2 : 1;
        f32x4 sum[kSums];
#pragma unroll
        for (int w = 0; w < kSums; ++w) {
            const uint32_t part = HALF ? wave : wave * kWeights + w;
            const uint32_t place = HALF ? lane + w * 32 : lane;
            sum[w] = s_part[0][part][place];
#pragma unroll
            for (uint32_t v = 1; v < kThinWaves; ++v) sum[w] += s_part[v][part][place];
        }
        const uint32_t row = m0 + wave * 16 + lane % 16;
        const uint32_t col = n0 + lane / 16 * 4;
        if (row >= rows || col >= cols) continue;
        if constexpr (KIND == kFfnGateUp) {
            if constexpr (X8) {
                const float scale = *reinterpret_cast<const float *>(x + static_cast<uint64_t>(row) * x_ld + dim);
                sum[0] *= scale;
                sum[kSums - 1] *= scale;
            }
            const uint64_t packed = static_cast<uint64_t>(start) + row;
            if (a.saved != nullptr) {
                float *to = a.saved + packed * 2 * hidden + col;
                *reinterpret_cast<f32x4 *>(to) = sum[0];
                *reinterpret_cast<f32x4 *>(to + hidden) = sum[kSums - 1];
            }
            f32x4 h;
#pragma unroll
            for (int e = 0; e < 4; ++e) h[e] = Act(sum[0][e], ActTerms(a.act)).value * sum[kSums - 1][e];
            *reinterpret_cast<uint2 *>(a.h + (packed * hidden + col) * 2) = narrow4<DT>(h);
        } else {
            char *c = const_cast<char *>(p1);
            *reinterpret_cast<uint2 *>(c + (static_cast<uint64_t>(row) * dim + col) * 2) = narrow4<DT>(sum[0]);
        }
    }
}

template <int DT, int KIND, int MB, bool HALF>
void launch_thin(const FfnArgs &a, hipStream_t st)
{
    constexpr uint32_t kCols = HALF ? 8 : 16;
    const dim3 grid((columns<KIND>(a.rows) + kCols - 1) / kCols, a.rows.n);
    if constexpr (KIND == kFfnGateUp) {
        if (a.x8) {
            HCCLX_LAUNCH((k_ffn_thin<DT, KIND, MB, true, HALF>), grid, dim3(kThinWaves * 64), 0, st, a);
            return;
        }
    }
    HCCLX_LAUNCH((k_ffn_thin<DT, KIND, MB, false, HALF>), grid, dim3(kThinWaves * 64), 0, st, a);
}

}  // namespace ffn
}  // namespace hcclx
