// The matrix products of the experts' feed-forward block on the matrix cores, one expert (rank) per group of rows.
//
// Every product is  C[m][n] = sum over k of A[m][k] B[n][k]  in tiles of BM x BN, with the operands as they lie in memory: "k-wise"
// (k runs along a row of the buffer) or "crosswise" (k counts the rows of the buffer).  A tile of either operand comes to LDS by
// loads that write LDS directly, 64 k at a time, two stages deep; crosswise tiles are read back with the transposing LDS read.
// v_mfma 16x16x32 takes B as its first operand, so that a lane ends up with four neighbouring columns of C.
//
// LDS layout: chunks of 16 bytes (k-wise) or 32 bytes (crosswise) of a row are permuted by an exclusive or with the row's number,
// so that the lanes of a read meet different banks.  The loads write LDS in lane order, hence the permutation is applied to the
// addresses that they read; those stay within the same cache lines.
//
// Bounds: the loads are range-checked by the hardware against the rows and columns that exist, and give zeros behind them, which
// add nothing; so no buffer needs padding, and garbage (NaN) behind a rank's last row is not seen.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>
#include "hcclx_ops.h"
#include "kernels/elem.h"
#include "kernels/launch.h"
#include "ops/ffn.h"
#include "ops/lanes.h"

namespace hcclx {
namespace ffn {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) char lds_char;
typedef __attribute__((address_space(3))) void lds_void;
typedef __attribute__((address_space(3))) s16x4 lds_s16x4;
typedef __attribute__((address_space(3))) u32x4 lds_u32x4;

constexpr uint32_t kBK = 64;             // k of a stage
constexpr uint32_t kOut = 0x80000000u;   // an offset behind every range

template <int DT> struct Mma;
template <> struct Mma<HCCL_DATA_TYPE_BFP16> {
    typedef __bf16 E;
    typedef __bf16 V8 __attribute__((ext_vector_type(8)));
    static __device__ __forceinline__ f32x4 run(u32x4 a, u32x4 b, f32x4 c)
    {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(V8, a), __builtin_bit_cast(V8, b), c, 0, 0, 0);
    }
};
template <> struct Mma<HCCL_DATA_TYPE_FP16> {
    typedef _Float16 E;
    typedef _Float16 V8 __attribute__((ext_vector_type(8)));
    static __device__ __forceinline__ f32x4 run(u32x4 a, u32x4 b, f32x4 c)
    {
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(V8, a), __builtin_bit_cast(V8, b), c, 0, 0, 0);
    }
};

// Four floats rounded to nearest even, as 8 bytes.
template <int DT>
__device__ __forceinline__ uint2 narrow4(f32x4 v)
{
    typedef typename Mma<DT>::E E;
    typedef E E4 __attribute__((ext_vector_type(4)));
    const E4 r = {static_cast<E>(v[0]), static_cast<E>(v[1]), static_cast<E>(v[2]), static_cast<E>(v[3])};
    return __builtin_bit_cast(uint2, r);
}

__device__ __forceinline__ uint32_t uniform(uint32_t x) { return __builtin_amdgcn_readfirstlane(x); }
__device__ __forceinline__ uint32_t of_lane(uint32_t x, uint32_t lane) { return __builtin_amdgcn_readlane(x, lane); }

__device__ __forceinline__ uint32_t inclusive_sum(uint32_t v)
{
    const uint32_t lane = threadIdx.x & 63;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const uint32_t o = __shfl_up(v, d, 64);
        if (lane >= static_cast<uint32_t>(d)) v += o;
    }
    return v;
}

// Lane j of every wavefront: the rows of rank j, and where they begin among the packed rows.
struct RankRows {
    uint32_t rows;
    uint32_t start;
    __device__ __forceinline__ explicit RankRows(const FfnRows &s)
    {
        const uint32_t j = threadIdx.x & 63;
        uint32_t r = 0;
        if (j < s.n) {
            r = s.capacity;
            if (s.counts != nullptr) {
                uint64_t sum = 0;
                for (uint32_t i = 0; i < s.per_rank; ++i) sum += s.counts[static_cast<uint64_t>(j) * s.per_rank + i];
                const uint64_t rows64 = (sum >> 32) == 0 ? static_cast<uint32_t>(sum) / s.unit : sum / s.unit;
                r = rows64 < s.capacity ? static_cast<uint32_t>(rows64) : s.capacity;
            }
        }
        // n * capacity may pass 32 bits where the counts do not bind: what is behind `most` is cut before it is summed
        r = r < s.most ? r : s.most;
        uint64_t before = 0;
        uint32_t mine = 0, from = 0;
        for (uint32_t k = 0; k < s.n; ++k) {
            const uint32_t rk = of_lane(r, k);
            const uint32_t left = s.most - static_cast<uint32_t>(before);
            const uint32_t take = rk < left ? rk : left;
            if (k == j) {
                mine = take;
                from = static_cast<uint32_t>(before);
            }
            before += take;
        }
        rows = mine;
        start = from;
    }
};

struct Tile {
    uint32_t rank;
    uint32_t m0;      // first row, of the rank
    uint32_t rows;    // of the rank
    uint32_t start;   // the rank's first packed row
    uint32_t nt;      // number of the column tile
};

// Which tile workgroup `id` computes.  The eight XCDs take workgroups in turn and have an L2 each: every XCD gets a stretch of
// tiles of its own, and neighbours in a stretch are kGroup row tiles by a few column tiles, which share operands.
constexpr uint32_t kGroup = 4;
template <uint32_t BM>
__device__ __forceinline__ bool locate(const FfnRows &s, uint32_t nts, Tile *t)
{
    const RankRows mine(s);
    const uint32_t tiles = (mine.rows + BM - 1) / BM;
    const uint32_t upto = inclusive_sum(tiles);
    const uint32_t total = of_lane(upto, 63);
    const uint32_t all = total * nts;
    const uint32_t per = (all + 7) / 8;
    const uint32_t slot = blockIdx.x / 8;
    const uint32_t at = (blockIdx.x % 8) * per + slot;
    if (slot >= per || at >= all) return false;
    const uint32_t group = at / (kGroup * nts);
    const uint32_t first = group * kGroup;
    const uint32_t height = total - first < kGroup ? total - first : kGroup;
    const uint32_t inside = at - first * nts;
    const uint32_t mt = first + inside % height;
    t->nt = inside / height;
    t->rank = __builtin_ctzll(__ballot(upto > mt));
    t->rows = of_lane(mine.rows, t->rank);
    t->start = of_lane(mine.start, t->rank);
    t->m0 = (mt - (of_lane(upto, t->rank) - of_lane(tiles, t->rank))) * BM;
    return true;
}

// Brings R rows (k-wise: of the operand; crosswise: R columns of 64 rows) of a stage to LDS, 16 bytes per lane and load.
template <uint32_t R, uint32_t WAVES, bool KWISE, bool PAIR>
struct Stager {
    static constexpr uint32_t kLoads = R / 8 / WAVES;
    static_assert(kLoads * 8 * WAVES == R, "every wavefront loads as much");
    uint32_t offset[kLoads];
    uint32_t k_at;   // k-wise: of this lane's chunk in a stage

    // ld: bytes of a row of the buffer; cols: crosswise, columns that exist from the tile's first on
    __device__ __forceinline__ void init(uint32_t wave, uint32_t lane, uint32_t ld, uint32_t cols)
    {
        if constexpr (KWISE) {
            const uint32_t chunk = (lane % 8) ^ (lane / 8);
            k_at = chunk * 8;
#pragma unroll
            for (uint32_t i = 0; i < kLoads; ++i) {
                uint32_t row = (wave * kLoads + i) * 8 + lane / 8;
                if (PAIR) row %= R / 2;
                offset[i] = row * ld + chunk * 16;
            }
        } else {
            constexpr uint32_t kChunks = R / 8;   // of a row
            k_at = 0;
#pragma unroll
            for (uint32_t i = 0; i < kLoads; ++i) {
                const uint32_t at = (wave * kLoads + i) * 64 + lane;
                const uint32_t k = at / kChunks;
                const uint32_t place = at % kChunks;
                const uint32_t turn = (k & 3) | ((k >> 3) & 1) << 2;
                const uint32_t chunk = ((place / 2) ^ turn) * 2 + place % 2;
                offset[i] = chunk * 8 < cols ? k * ld + chunk * 16 : kOut;
            }
        }
    }
    // base: of the stage (uniform); range: bytes from there on that exist; left: k-wise, k that exist from the stage's first on
    __device__ __forceinline__ void issue(const char *base, uint32_t range, uint32_t left, lds_char *lds, uint32_t wave) const
    {
        const __amdgpu_buffer_rsrc_t rsrc = __builtin_amdgcn_make_buffer_rsrc(const_cast<char *>(base), 0, static_cast<int>(range), 0x00027000);
        const bool beyond = KWISE && k_at >= left;
#pragma unroll
        for (uint32_t i = 0; i < kLoads; ++i) {
            const uint32_t o = beyond ? kOut : offset[i];
            __builtin_amdgcn_raw_ptr_buffer_load_lds(rsrc, (lds_void *)(lds + (wave * kLoads + i) * 1024), 16, o, 0, 0, 0);
        }
    }
};

// A fragment of 16 rows by 32 k out of a staged tile.
template <bool KWISE, uint32_t R>
struct Reader {
    uint32_t base;
    uint32_t turn;
    __device__ __forceinline__ explicit Reader(uint32_t lane)
    {
        if constexpr (KWISE) {
            base = (lane % 16) * 128 + (((lane / 16) ^ (lane & 7)) * 16);
            turn = 0;
        } else {
            const uint32_t k = lane / 16 * 8 + lane % 16 / 4;
            turn = (k & 3) | ((k >> 3) & 1) << 2;
            base = k * (R * 2) + lane % 4 * 8;
        }
    }
    // f: number of the 16 rows in the tile; half: which 32 of the stage's 64 k
    __device__ __forceinline__ u32x4 operator()(const lds_char *tile, uint32_t f, uint32_t half) const
    {
        if constexpr (KWISE) {
            return *(const lds_u32x4 *)(tile + (base ^ (half * 64)) + f * 2048);
        } else {
            const lds_char *p = tile + base + (f ^ turn) * 32 + half * (32 * R * 2);
            const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4 *)(p));
            const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4 *)(p + 4 * R * 2));
            struct Both {
                s16x4 lo, hi;
            } both = {lo, hi};
            return __builtin_bit_cast(u32x4, both);
        }
    }
};

// act(a) and its derivative.
struct Act {
    float value;
    float slope;
    __device__ __forceinline__ Act(float a, int act)
    {
        if (act == HCCLX_ACT_SILU) {
            const float s = 1.0f / (1.0f + __expf(-a));
            value = a * s;
            slope = s * (1.0f + a * (1.0f - s));
        } else {
            constexpr float kRoot = 0.7978845608028654f;   // sqrt(2 / pi)
            const float t = 1.0f - 2.0f / (__expf(2.0f * kRoot * (a + 0.044715f * a * a * a)) + 1.0f);
            value = 0.5f * a * (1.0f + t);
            slope = 0.5f * (1.0f + t) + 0.5f * a * (1.0f - t * t) * (kRoot * (1.0f + 3.0f * 0.044715f * a * a));
        }
    }
};

// One operand of a product: where its tile begins and how its stages follow each other.
struct Operand {
    const char *base;
    uint32_t ld;      // bytes of a row
    uint32_t extent;  // k-wise: rows from the tile's first on; crosswise: columns
};
template <bool KWISE>
__device__ __forceinline__ void stage_of(const Operand &o, uint32_t rows, uint32_t k0, uint32_t k, const char **base, uint32_t *range)
{
    if constexpr (KWISE) {
        const uint32_t have = o.extent < rows ? o.extent : rows;
        *base = o.base + static_cast<uint64_t>(k0) * 2;
        *range = (have - 1) * o.ld + (k - k0) * 2;
    } else {
        const uint32_t have = k - k0 < kBK ? k - k0 : kBK;
        *base = o.base + static_cast<uint64_t>(k0) * o.ld;
        *range = (have - 1) * o.ld + o.extent * 2;
    }
}

// WM x WN wavefronts of FM x FN fragments each.
template <int DT, int KIND, int WM, int WN, int FM, int FN>
__global__ void __launch_bounds__(WM *WN * 64)
k_ffn(FfnArgs a)
{
    constexpr uint32_t BM = WM * FM * 16;
    constexpr uint32_t BN = WN * FN * 16;
    constexpr uint32_t kWaves = WM * WN;
    constexpr bool kPair = KIND == kFfnGateUp;             // half of the columns from either weight
    constexpr bool kAk = KIND != kFfnGradWeights;          // A lies k-wise
    constexpr bool kBk = KIND == kFfnGateUp || KIND == kFfnDown;
    constexpr uint32_t kCols = kPair ? BN / 2 : BN;        // columns of C
    constexpr uint32_t kStage = (BM + BN) * kBK * 2;
    __shared__ __attribute__((aligned(1024))) char s_tile[2][kStage];

    const FfnRows &s = a.rows;
    const uint32_t wave = uniform(threadIdx.x / 64);
    const uint32_t lane = threadIdx.x & 63;
    const uint32_t dim = s.dim;
    const uint32_t hidden = s.hidden;

    // what is multiplied: up to two pairs of operands along k, one after the other
    Operand oa[2], ob[2];
    uint32_t ks = 0;          // length of k, of each pair
    uint32_t pairs = 1;
    Tile t;
    uint32_t n0 = 0;
    uint32_t weight = 0;      // kFfnGradWeights: 0 the projections', 1 w_down's
    if constexpr (KIND == kFfnGradWeights) {
        const uint32_t first_tiles = (2 * hidden + BM - 1) / BM * ((dim + BN - 1) / BN);
        const uint32_t second_tiles = (dim + BM - 1) / BM * ((hidden + BN - 1) / BN);
        const uint32_t per = (first_tiles + second_tiles + 7) / 8;   // of an XCD and rank
        const uint32_t rank = blockIdx.x / (per * 8);
        const uint32_t inside = blockIdx.x % (per * 8);
        uint32_t at = inside % 8 * per + inside / 8;
        if (at >= first_tiles + second_tiles) return;
        weight = at >= first_tiles ? 1 : 0;
        if (weight != 0) at -= first_tiles;
        const uint32_t mts = ((weight != 0 ? dim : 2 * hidden) + BM - 1) / BM;
        const uint32_t nts = ((weight != 0 ? hidden : dim) + BN - 1) / BN;
        const uint32_t first = at / (kGroup * nts) * kGroup;
        const uint32_t height = mts - first < kGroup ? mts - first : kGroup;
        const uint32_t left = at - first * nts;
        const RankRows mine(s);
        t.rank = rank;
        t.rows = of_lane(mine.rows, rank);
        t.start = of_lane(mine.start, rank);
        t.m0 = (first + left % height) * BM;
        t.nt = left / height;
        n0 = t.nt * BN;
        ks = t.rows;
        if (weight == 0) {
            oa[0] = {a.dproj + static_cast<uint64_t>(t.start) * hidden * 4 + static_cast<uint64_t>(t.m0) * 2, hidden * 4, 2 * hidden - t.m0};
            ob[0] = {a.p[0][rank] + static_cast<uint64_t>(n0) * 2, dim * 2, dim - n0};
        } else {
            oa[0] = {a.p[1][rank] + static_cast<uint64_t>(t.m0) * 2, dim * 2, dim - t.m0};
            ob[0] = {a.h + static_cast<uint64_t>(t.start) * hidden * 2 + static_cast<uint64_t>(n0) * 2, hidden * 2, hidden - n0};
        }
    } else {
        const uint32_t cols = KIND == kFfnGateUp || KIND == kFfnGradHidden ? hidden : dim;
        if (!locate<BM>(s, (cols + kCols - 1) / kCols, &t)) return;
        n0 = t.nt * kCols;
        const uint64_t row = static_cast<uint64_t>(t.start) + t.m0;
        const uint32_t rows = t.rows - t.m0;
        if constexpr (KIND == kFfnGateUp) {
            ks = dim;
            const char *x = a.x16 != nullptr ? a.x16 + row * dim * 2 : a.p[0][t.rank] + static_cast<uint64_t>(t.m0) * dim * 2;
            oa[0] = {x, dim * 2, rows};
            const char *w = a.p[wave * (BN / kWaves) >= BN / 2 ? 2 : 1][t.rank];   // of the rows that this wavefront stages
            ob[0] = {w + static_cast<uint64_t>(n0) * dim * 2, dim * 2, hidden - n0};
        } else if constexpr (KIND == kFfnDown) {
            ks = hidden;
            oa[0] = {a.h + row * hidden * 2, hidden * 2, rows};
            ob[0] = {a.p[0][t.rank] + static_cast<uint64_t>(n0) * hidden * 2, hidden * 2, dim - n0};
        } else if constexpr (KIND == kFfnGradHidden) {
            ks = dim;
            oa[0] = {a.p[0][t.rank] + static_cast<uint64_t>(t.m0) * dim * 2, dim * 2, rows};
            ob[0] = {a.p[1][t.rank] + static_cast<uint64_t>(n0) * 2, hidden * 2, hidden - n0};
        } else {
            ks = hidden;
            pairs = 2;
            oa[0] = {a.dproj + row * hidden * 4, hidden * 4, rows};
            oa[1] = {oa[0].base + static_cast<uint64_t>(hidden) * 2, hidden * 4, rows};
            ob[0] = {a.p[0][t.rank] + static_cast<uint64_t>(n0) * 2, dim * 2, dim - n0};
            ob[1] = {a.p[1][t.rank] + static_cast<uint64_t>(n0) * 2, dim * 2, dim - n0};
        }
    }

    Stager<BM, kWaves, kAk, false> sa;
    Stager<BN, kWaves, kBk, kPair> sb;
    sa.init(wave, lane, oa[0].ld, oa[0].extent);
    sb.init(wave, lane, ob[0].ld, ob[0].extent);
    const uint32_t steps = (ks + kBK - 1) / kBK;   // of a pair
    const uint32_t total = steps * pairs;
    auto stage = [&](uint32_t step, lds_char *lds) {
        const bool second = KIND == kFfnGradInput && step >= steps;
        const uint32_t k0 = (second ? step - steps : step) * kBK;
        const char *base;
        uint32_t range;
        stage_of<kAk>(second ? oa[1] : oa[0], BM, k0, ks, &base, &range);
        sa.issue(base, range, ks - k0, lds, wave);
        stage_of<kBk>(second ? ob[1] : ob[0], kCols, k0, ks, &base, &range);
        sb.issue(base, range, ks - k0, lds + BM * kBK * 2, wave);
    };

    const uint32_t wm = wave / WN;
    const uint32_t wn = wave % WN;
    const Reader<kAk, BM> ra(lane);
    const Reader<kBk, BN> rb(lane);
    f32x4 acc[FM][FN];
#pragma unroll
    for (int m = 0; m < FM; ++m) {
#pragma unroll
        for (int n = 0; n < FN; ++n) acc[m][n] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    }
    // the fragments of B that this wavefront takes: of a pair, half from either weight
    auto b_frag = [&](int n) -> uint32_t {
        if constexpr (kPair) {
            constexpr int kHalf = FN / 2;
            return n < kHalf ? wn * kHalf + n : BN / 32 + wn * kHalf + (n - kHalf);
        } else {
            return wn * FN + n;
        }
    };

    if (total != 0) stage(0, (lds_char *)s_tile[0]);
    for (uint32_t step = 0; step < total; ++step) {
        __syncthreads();   // this stage's loads have landed, and everybody has read the one before
        const lds_char *tile = (const lds_char *)s_tile[step & 1];
        if (step + 1 < total) stage(step + 1, (lds_char *)s_tile[(step + 1) & 1]);
#pragma unroll
        for (uint32_t half = 0; half < 2; ++half) {
            u32x4 fa[FM], fb[FN];
#pragma unroll
            for (int m = 0; m < FM; ++m) fa[m] = ra(tile, wm * FM + m, half);
#pragma unroll
            for (int n = 0; n < FN; ++n) fb[n] = rb(tile + BM * kBK * 2, b_frag(n), half);
#pragma unroll
            for (int m = 0; m < FM; ++m) {
#pragma unroll
                for (int n = 0; n < FN; ++n) acc[m][n] = Mma<DT>::run(fb[n], fa[m], acc[m][n]);
            }
        }
    }

    // a lane holds columns 4 (lane / 16) .. + 3 of row lane % 16 of every fragment
    const uint32_t row_in = wm * (FM * 16) + lane % 16;
    const uint32_t col_in = lane / 16 * 4;
#pragma unroll
    for (int m = 0; m < FM; ++m) {
        const uint32_t row = t.m0 + row_in + m * 16;
        if constexpr (KIND == kFfnGradWeights) {
            if (row >= (weight != 0 ? dim : 2 * hidden)) continue;
            const uint32_t width = weight != 0 ? hidden : dim;
            const char *to = weight != 0 ? a.p[4][t.rank] : row < hidden ? a.p[2][t.rank] : a.p[3][t.rank];
            const uint32_t r = weight == 0 && row >= hidden ? row - hidden : row;
            char *c = const_cast<char *>(to) + static_cast<uint64_t>(r) * width * 2;
#pragma unroll
            for (int n = 0; n < FN; ++n) {
                const uint32_t col = n0 + (wn * FN + n) * 16 + col_in;
                if (col < width) *reinterpret_cast<uint2 *>(c + static_cast<uint64_t>(col) * 2) = narrow4<DT>(acc[m][n]);
            }
        } else {
            if (row >= t.rows) continue;
            const uint64_t packed = static_cast<uint64_t>(t.start) + row;
            if constexpr (KIND == kFfnGateUp) {
                float scale = 1.0f;
                if (a.x16 != nullptr) scale = *reinterpret_cast<const float *>(a.p[0][t.rank] + static_cast<uint64_t>(row) * (dim + HCCLX_ROW8_TAIL) + dim);
#pragma unroll
                for (int n = 0; n < FN / 2; ++n) {
                    const uint32_t col = n0 + (wn * (FN / 2) + n) * 16 + col_in;
                    if (col >= hidden) continue;
                    const f32x4 g = acc[m][n] * scale;
                    const f32x4 u = acc[m][n + FN / 2] * scale;
                    if (a.saved != nullptr) {
                        float *to = a.saved + packed * 2 * hidden + col;
                        *reinterpret_cast<f32x4 *>(to) = g;
                        *reinterpret_cast<f32x4 *>(to + hidden) = u;
                    }
                    f32x4 h;
#pragma unroll
                    for (int e = 0; e < 4; ++e) h[e] = Act(g[e], a.act).value * u[e];
                    *reinterpret_cast<uint2 *>(a.h + (packed * hidden + col) * 2) = narrow4<DT>(h);
                }
            } else if constexpr (KIND == kFfnGradHidden) {
#pragma unroll
                for (int n = 0; n < FN; ++n) {
                    const uint32_t col = n0 + (wn * FN + n) * 16 + col_in;
                    if (col >= hidden) continue;
                    const float *from = a.saved + packed * 2 * hidden + col;
                    const f32x4 g = *reinterpret_cast<const f32x4 *>(from);
                    const f32x4 u = *reinterpret_cast<const f32x4 *>(from + hidden);
                    f32x4 h, dg, du;
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const Act f(g[e], a.act);
                        h[e] = f.value * u[e];
                        dg[e] = acc[m][n][e] * u[e] * f.slope;
                        du[e] = acc[m][n][e] * f.value;
                    }
                    *reinterpret_cast<uint2 *>(a.h + (packed * hidden + col) * 2) = narrow4<DT>(h);
                    char *to = a.dproj + (packed * 2 * hidden + col) * 2;
                    *reinterpret_cast<uint2 *>(to) = narrow4<DT>(dg);
                    *reinterpret_cast<uint2 *>(to + static_cast<uint64_t>(hidden) * 2) = narrow4<DT>(du);
                }
            } else {
                char *c = const_cast<char *>(KIND == kFfnDown ? a.p[1][t.rank] : a.p[2][t.rank]) + static_cast<uint64_t>(row) * dim * 2;
#pragma unroll
                for (int n = 0; n < FN; ++n) {
                    const uint32_t col = n0 + (wn * FN + n) * 16 + col_in;
                    if (col < dim) *reinterpret_cast<uint2 *>(c + static_cast<uint64_t>(col) * 2) = narrow4<DT>(acc[m][n]);
                }
            }
        }
    }
}

// The values of 8-bit codes in 16 bits, which hold every e4m3 value exactly; the rows' scales are applied to the products.  A
// wavefront per packed row.
template <int DT>
__global__ void __launch_bounds__(256)
k_ffn_widen(FfnArgs a)
{
    const FfnRows &s = a.rows;
    const RankRows mine(s);
    const uint32_t lane = threadIdx.x & 63;
    const uint32_t packed = blockIdx.x * 4 + uniform(threadIdx.x / 64);
    const uint64_t has = __ballot(packed - mine.start < mine.rows && packed >= mine.start);
    if (has == 0) return;
    const uint32_t rank = __builtin_ctzll(has);
    const uint32_t row = packed - of_lane(mine.start, rank);
    const char *from = a.p[0][rank] + static_cast<uint64_t>(row) * (s.dim + HCCLX_ROW8_TAIL);
    char *to = a.x16 + static_cast<uint64_t>(packed) * s.dim * 2;
    for (uint32_t c = lane * 16; c < s.dim; c += 1024) {
        const u32x4 codes = *reinterpret_cast<const u32x4 *>(from + c);
#pragma unroll
        for (int q = 0; q < 2; ++q) {
            float f[8];
            from_e4m3(codes[2 * q], *reinterpret_cast<float(*)[4]>(f));
            from_e4m3(codes[2 * q + 1], *reinterpret_cast<float(*)[4]>(f + 4));
            const uint2 lo = narrow4<DT>(f32x4{f[0], f[1], f[2], f[3]});
            const uint2 hi = narrow4<DT>(f32x4{f[4], f[5], f[6], f[7]});
            *reinterpret_cast<u32x4 *>(to + (c + q * 8) * 2) = u32x4{lo.x, lo.y, hi.x, hi.y};
        }
    }
}

// Workgroups of a product in tiles of bm x (columns of C per tile): at most one tile more per rank than the rows fill.
inline uint64_t row_tiles(const FfnRows &s, uint64_t bm)
{
    const uint64_t by_rows = s.most / bm + s.n;
    const uint64_t by_rank = s.n * ((s.capacity + bm - 1) / bm);
    return by_rows < by_rank ? by_rows : by_rank;
}

template <int DT, int KIND, int WM, int WN, int FM, int FN>
hipError_t run(const FfnArgs &a, hipStream_t st)
{
    constexpr uint64_t BM = WM * FM * 16;
    constexpr uint64_t BN = WN * FN * 16;
    const FfnRows &s = a.rows;
    uint64_t groups;
    if (KIND == kFfnGradWeights) {
        const uint64_t tiles = (2ull * s.hidden + BM - 1) / BM * ((s.dim + BN - 1) / BN) + (s.dim + BM - 1) / BM * ((s.hidden + BN - 1) / BN);
        groups = (tiles + 7) / 8 * 8 * s.n;
    } else {
        const uint64_t cols = KIND == kFfnGateUp || KIND == kFfnGradHidden ? s.hidden : s.dim;
        const uint64_t width = KIND == kFfnGateUp ? BN / 2 : BN;
        groups = (row_tiles(s, BM) * ((cols + width - 1) / width) + 7) / 8 * 8;
    }
    if (groups > 0xffffffffull / (WM * WN * 64)) return hipErrorInvalidValue;
    if (groups == 0) return hipSuccess;
    HCCLX_LAUNCH((k_ffn<DT, KIND, WM, WN, FM, FN>), dim3(static_cast<uint32_t>(groups)), dim3(WM * WN * 64), 0, st, a);
    return hipGetLastError();
}

template <int DT, int KIND>
hipError_t pick(const FfnArgs &a, uint32_t num_cus, hipStream_t st)
{
    const FfnRows &s = a.rows;
    const uint64_t cols = KIND == kFfnGateUp || KIND == kFfnGradHidden ? s.hidden : s.dim;
    const uint64_t rows = KIND == kFfnGradWeights ? 3ull * s.hidden * s.n : s.most;
    const bool large = (rows / 256) * (cols / 256) >= num_cus && (KIND == kFfnGradWeights || s.most / s.n >= 128);
    if (large) return run<DT, KIND, 2, 4, 8, 4>(a, st);
    return run<DT, KIND, 2, 2, 4, 4>(a, st);
}

}  // namespace ffn

template <int DT>
hipError_t launch_ffn_widen(const FfnArgs &a, hipStream_t st)
{
    if (a.rows.most == 0) return hipSuccess;
    HCCLX_LAUNCH((ffn::k_ffn_widen<DT>), dim3((a.rows.most + 3) / 4), dim3(256), 0, st, a);
    return hipGetLastError();
}

template <int DT>
hipError_t launch_ffn(FfnKind kind, const FfnArgs &a, uint32_t num_cus, hipStream_t st)
{
    switch (kind) {
        case kFfnGateUp: return ffn::pick<DT, kFfnGateUp>(a, num_cus, st);
        case kFfnDown: return ffn::pick<DT, kFfnDown>(a, num_cus, st);
        case kFfnGradHidden: return ffn::pick<DT, kFfnGradHidden>(a, num_cus, st);
        case kFfnGradInput: return ffn::pick<DT, kFfnGradInput>(a, num_cus, st);
        default: return ffn::pick<DT, kFfnGradWeights>(a, num_cus, st);
    }
}

}  // namespace hcclx
