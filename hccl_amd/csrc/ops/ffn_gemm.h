// The matrix products of the experts' feed-forward block on the matrix cores, one expert (rank) per group of rows.
//
// Every product is  C[m][n] = sum over k of A[m][k] B[n][k]  in tiles of BM x BN, with the operands as they lie in memory: "k-wise"
// (k runs along a row of the buffer) or "crosswise" (k counts the rows of the buffer).  A tile of either operand comes to LDS by
// loads that write LDS directly, 64 k at a time, two stages deep; crosswise tiles are read back with the transposing LDS read.
// v_mfma 16x16x32 takes B as its first operand, so that a lane ends up with four neighbouring columns of C.  (From registers alone
// it reaches 2100 TFLOP/s here, 32x32x16 1350.)
//
// What bounds it: the matrix instructions, at the clock that the card's power leaves.  8 ranks x 4096 rows x 7168 x 2048: 1400 us for
// the first product (1370 TFLOP/s; its pipes are busy 71 % of the time, at 1.75 to 1.9 GHz), 750 for the second (1280; 66 %).  With
// rows of 4096 they are busy for 59 to 61 %, with those of the hidden rows' gradient, which reads and writes four streams between its
// tiles while nothing is multiplied, for 38 %.  A wavefront has 128 x
// 128 of a tile of 256 x 256, which is one wavefront per SIMD, 256 accumulators in the second half of its registers and one LDS
// read of 1 KiB for four matrix instructions; eight wavefronts of 128 x 64 read half as much again and took 1580 and 820.  With
// nobody else on its SIMD a wavefront has to keep the matrix pipe busy by itself: between two matrix instructions there is one
// LDS read, or one load, or a few scalar instructions (all of a stage's loads at once: as slow as eight wavefronts), and what is
// read is a row of fragments ahead.  Stages of 32 k, more of them, took 1890.
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
typedef __attribute__((address_space(3))) s16x4 lds_s16x4;
typedef __attribute__((address_space(3))) u32x4 lds_u32x4;

constexpr uint32_t kOut = 0x80000000u;   // an offset behind every range
constexpr uint32_t kRaw = 0x00027000u;        // last word of a buffer resource: plain bytes, range-checked
constexpr uint32_t kMostRange = 0x7fffffffu;
constexpr uint32_t kBK = 64;             // k of a stage: a cache line of a k-wise row
constexpr uint32_t kWaves = 4;           // of a workgroup, two by two
constexpr uint32_t kWaveRows = 2;
constexpr uint32_t kWaveCols = 2;
constexpr uint32_t kTile = 256;          // rows and columns of a whole tile
constexpr uint32_t kLdsBytes = 160 * 1024;

// add: of accumulators that stay in the second half of the registers and between instructions that stay in their order.  (Where the
// compiler chooses, 256 accumulators move from one half to the other and back: first product 2435 us.)
template <int DT> struct Mma;
template <> struct Mma<HCCL_DATA_TYPE_BFP16> {
    typedef __bf16 E;
    typedef __bf16 V8 __attribute__((ext_vector_type(8)));
    static __device__ __forceinline__ f32x4 run(u32x4 a, u32x4 b, f32x4 c)
    {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(V8, a), __builtin_bit_cast(V8, b), c, 0, 0, 0);
    }
    static __device__ __forceinline__ void add(f32x4 &c, u32x4 a, u32x4 b)
    {
        asm volatile("v_mfma_f32_16x16x32_bf16 %0, %1, %2, %0" : "+a"(c) : "v"(a), "v"(b));
    }
};
template <> struct Mma<HCCL_DATA_TYPE_FP16> {
    typedef _Float16 E;
    typedef _Float16 V8 __attribute__((ext_vector_type(8)));
    static __device__ __forceinline__ f32x4 run(u32x4 a, u32x4 b, f32x4 c)
    {
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(V8, a), __builtin_bit_cast(V8, b), c, 0, 0, 0);
    }
    static __device__ __forceinline__ void add(f32x4 &c, u32x4 a, u32x4 b)
    {
        asm volatile("v_mfma_f32_16x16x32_f16 %0, %1, %2, %0" : "+a"(c) : "v"(a), "v"(b));
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

// Eight codes' values.
template <int DT>
__device__ __forceinline__ u32x4 widen8(uint32_t low, uint32_t high)
{
    float f[4];
    from_e4m3(low, f);
    const uint2 lo = narrow4<DT>(f32x4{f[0], f[1], f[2], f[3]});
    from_e4m3(high, f);
    const uint2 hi = narrow4<DT>(f32x4{f[0], f[1], f[2], f[3]});
    return u32x4{lo.x, lo.y, hi.x, hi.y};
}

// Two fragments of C as 16-bit values, four columns to a lane: afterwards lanes 0..15 and 32..47 hold columns 0..7 and 8..15 of the
// first, the others of the second.  16-byte stores of half a cache line per row instead of 8-byte ones of a quarter.
__device__ __forceinline__ u32x4 pair_up(uint2 first, uint2 second)
{
    typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
    const u32x2 x = __builtin_amdgcn_permlane16_swap(first.x, second.x, false, false);
    const u32x2 y = __builtin_amdgcn_permlane16_swap(first.y, second.y, false, false);
    return u32x4{x[0], y[0], x[1], y[1]};
}
// A stretch of memory that results go to or come from, at offsets of 32 bits; what does not exist has the offset kOut, where loads
// give zeros and stores do nothing.  (No branches: the number of stores of a tile is known when they are waited for.)
struct Window {
    __amdgpu_buffer_rsrc_t rsrc;
    __device__ __forceinline__ explicit Window(const void *base, uint32_t range = kMostRange)
        : rsrc(__builtin_amdgcn_make_buffer_rsrc(const_cast<void *>(base), 0, static_cast<int>(range), kRaw))
    {
    }
    __device__ __forceinline__ void store(uint32_t offset, u32x4 v) const { __builtin_amdgcn_raw_buffer_store_b128(v, rsrc, offset, 0, 0); }
    __device__ __forceinline__ f32x4 load(uint32_t offset) const
    {
        return __builtin_bit_cast(f32x4, __builtin_amdgcn_raw_buffer_load_b128(rsrc, offset, 0, 0));
    }
};

__device__ __forceinline__ uint32_t uniform(uint32_t x) { return __builtin_amdgcn_readfirstlane(x); }
// The same where the compiler, knowing that x is uniform, would drop the instruction and keep x and all that is computed from it in
// vector registers (quotients of the tiles' numbers).
__device__ __forceinline__ uint32_t scalar(uint32_t x)
{
    asm("" : "+v"(x));
    return uniform(x);
}
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
                const uint64_t *mine = s.counts + static_cast<uint64_t>(j) * s.per_rank;
                for (uint32_t i = 0; i < s.per_rank; i += 8) {   // eight loads at a time
                    uint64_t c[8];
#pragma unroll
                    for (uint32_t e = 0; e < 8; ++e) c[e] = mine[i + e < s.per_rank ? i + e : i];
#pragma unroll
                    for (uint32_t e = 0; e < 8; ++e) sum += i + e < s.per_rank ? c[e] : 0;
                }
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

// A tile of C, or a part of one.
struct Tile {
    uint32_t rank;
    uint32_t rows;    // of the rank
    uint32_t start;   // the rank's first packed row
    uint32_t m0;      // first row and column
    uint32_t n0;
    uint32_t weight;  // kFfnGradWeights: of w_gate, w_up or w_down
};

// Tiles are numbered rank by rank, kGroup rows of tiles at a time, down these first: 32 neighbours are 4 x 8 tiles, which share
// operands.
constexpr uint32_t kGroup = 4;
__device__ __forceinline__ void in_groups(uint32_t at, uint32_t mts, uint32_t nts, uint32_t *mt, uint32_t *nt)
{
    const uint32_t first = at / (kGroup * nts) * kGroup;
    const uint32_t height = mts - first < kGroup ? mts - first : kGroup;
    const uint32_t inside = at - first * nts;
    *mt = scalar(first + inside % height);
    *nt = scalar(inside / height);
}

// How whole tiles are shared out.  T of them on W CUs take T / W rounds and one more for what is left, however little; so what is
// left is cut into parts, of which a CU has at most one: quarters of up to W / 4 tiles, halves (of the columns) of up to W / 2.  One
// rank, bf16, cut : whole, forward and gradients: 1024 rows x 2048 x 2048 53 + 120 : 102 + 220 us, 2048 x 4096 x 2048 (a round and
// halves or quarters of one) 101 + 220 : 156 + 343.  More than W / 2 are left whole: three quarters of a tile take as long as it.
// The eight XCDs take workgroups in turn and have an L2 each: every XCD gets a run of neighbours out of each round.
struct Share {
    uint32_t whole;   // tiles that are not cut
    uint32_t parts;   // of each tile that is: 2 or 4
    uint32_t left;    // tiles that are
    __device__ __forceinline__ Share(uint32_t tiles, uint32_t groups)
    {
        left = scalar(tiles % groups);
        parts = left <= groups / 4 ? 4 : 2;
        if (left > groups / 2) left = 0;
        whole = tiles - left;
    }
};

// Columns of C, and of a whole tile.
template <int KIND>
__host__ __device__ inline uint32_t columns(const FfnRows &s)
{
    return KIND == kFfnGateUp || KIND == kFfnGradHidden ? s.hidden : s.dim;
}
template <int KIND> constexpr uint32_t kTileCols = KIND == kFfnGateUp ? kTile / 2 : kTile;   // half of a tile from either weight

// A load of 16 bytes per lane, from the range-checked buffer at the lanes' offsets to lds + 16 * lane.  Written out because the
// compiler waits for every such load that it knows of before it lets a transposing LDS read go, whatever that reads; here loads and
// reads keep apart by meet().  There is no register that the load writes.  s_nop: a wait state behind a write of m0.  A buffer
// whose scalars a vector instruction may have written takes five, which are between the making of a buffer and its first load.
typedef uint32_t Resource __attribute__((ext_vector_type(4)));
__device__ __forceinline__ void load_to_lds(Resource buffer, uint32_t lds, uint32_t offset)
{
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds" ::"s"(lds), "v"(offset), "s"(buffer) : "memory");
}

// Brings R rows (k-wise: of the operand; crosswise: R columns of kBK rows) of a stage to LDS.
template <uint32_t R, bool KWISE, bool PAIR>
struct Stager {
    static constexpr uint32_t kLoads = R * kBK * 2 / 1024 / kWaves;
    static constexpr uint32_t kChunks = KWISE ? kBK / 8 : R / 8;   // of 16 bytes, of a row
    static constexpr uint32_t kRows = 64 / kChunks;                // of a load
    static_assert(kLoads * 1024 * kWaves == R * kBK * 2 && kRows * kChunks == 64, "every wavefront loads as much, in whole rows");
    uint32_t row_at;   // offset of the first load's row
    uint32_t chunk;    // and the chunk of it

    // ld: bytes of a row of the buffer
    __device__ __forceinline__ void init(uint32_t wave, uint32_t lane, uint32_t ld)
    {
        uint32_t row = wave * kLoads * kRows + lane / kChunks;
        if constexpr (KWISE) {
            chunk = (lane % 8) ^ (lane / 8);
            if (PAIR) row %= R / 2;
        } else {
            const uint32_t turn = (row & 3) | ((row >> 3) & 1) << 2;
            chunk = ((lane % kChunks / 2) ^ turn) * 2 + lane % 2;
        }
        row_at = row * ld;
    }
    // Load i of a stage in `buffer`.  end: k (k-wise) or columns (crosswise) that exist
    __device__ __forceinline__ void issue(uint32_t i, Resource buffer, uint32_t end, uint32_t ld, uint32_t lds, uint32_t wave) const
    {
        load_to_lds(buffer, uniform(lds + (wave * kLoads + i) * 1024), at(i, end, ld));
    }

private:
    __device__ __forceinline__ uint32_t at(uint32_t i, uint32_t end, uint32_t ld) const
    {
        // (crosswise: of the row's number, the first two bits and the fourth turn the chunks; a load is kRows rows further on)
        constexpr bool kTurns = !KWISE;
        const uint32_t c = kTurns ? chunk ^ (((i * kRows) & 3) | (((i * kRows) >> 3) & 1) << 2) * 2 : chunk;
        return (c * 8 < end ? row_at + c * 16 : kOut) + i * kRows * ld;
    }
};

// base: of a stage; range: bytes from there on that exist
__device__ __forceinline__ Resource resource(const char *base, uint32_t range)
{
    const uint64_t at = reinterpret_cast<uint64_t>(base);
    return {uniform(static_cast<uint32_t>(at)), uniform(static_cast<uint32_t>(at >> 32) & 0xffffu), uniform(range), kRaw};
}

// A fragment of 16 rows by 32 k out of a staged tile.
template <bool KWISE, uint32_t R>
struct Reader {
    uint32_t base;
    uint32_t turn;
    __device__ __forceinline__ explicit Reader(uint32_t lane)
    {
        if constexpr (KWISE) {
            base = (lane % 16) * (kBK * 2) + ((lane / 16) ^ (lane % 8)) * 16;
            turn = 0;
        } else {
            const uint32_t k = lane / 16 * 8 + lane % 16 / 4;
            turn = ((k & 3) | ((k >> 3) & 1) << 2) * 32;
            base = k * (R * 2) + lane % 4 * 8;
        }
    }
    // f: number of the 16 rows in the tile; half: which 32 k of the stage's
    __device__ __forceinline__ u32x4 operator()(const lds_char *tile, uint32_t f, uint32_t half) const
    {
        if constexpr (KWISE) {
            return *(const lds_u32x4 *)(tile + (base ^ (half * 64)) + f * (kBK * 32));
        } else {
            uint32_t t = turn;
            asm("" : "+v"(t));   // (computed for each read: kept for every fragment it would take a register each)
            const lds_char *p = tile + base + ((f * 32) ^ t) + half * (32 * R * 2);
            const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4 *)(p));
            const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4 *)(p + 4 * R * 2));
            struct Both {
                s16x4 lo, hi;
            } both = {lo, hi};
            return __builtin_bit_cast(u32x4, both);
        }
    }
};

// act(a) = a / (1 + exp(-w(a))) and its derivative: both activations with w = a (p + q a^2), SILU with 1 and 0, and GELU_TANH, whose
// (1 + tanh z) / 2 is 1 / (1 + exp(-2 z)).
struct ActTerms {
    float p;
    float q;
    __device__ __forceinline__ explicit ActTerms(int act)
    {
        constexpr float kTwice = 1.5957691216057308f;   // 2 sqrt(2 / pi)
        p = act == HCCLX_ACT_SILU ? 1.0f : kTwice;
        q = act == HCCLX_ACT_SILU ? 0.0f : kTwice * 0.044715f;
    }
};
struct Act {
    float value;
    float slope;
    __device__ __forceinline__ Act(float a, const ActTerms &t)
    {
        // (0 times infinity is not 0.  Far out, where s is 0 or 1, so is value or 1 - s, and what it is multiplied by is finite: the
        // square by its limit, which s has long ceased to notice, and not times a, which has none.)
        const float square = __builtin_fminf(a * a, 1e30f);
        const float s = 1.0f / (1.0f + __expf(-a * (t.p + t.q * square)));
        value = a * s;
        slope = s + value * (1.0f - s) * (t.p + 3.0f * t.q * square);
    }
};

// Where the stages of a tile come from: two pairs of operands along k, one after the other (the second of kFfnGradInput alone).
struct Feed {
    const char *a[2];
    const char *b[2];
    uint32_t a_ld;       // bytes of a row
    uint32_t b_ld;
    uint32_t a_extent;   // k-wise: rows from the tile's first on; crosswise: columns
    uint32_t b_extent;
    uint32_t k;          // of each pair
};
template <int KIND, uint32_t BN>
__device__ __forceinline__ Feed feed_of(const FfnArgs &a, const Tile &t, uint32_t wave)
{
    const uint32_t dim = a.rows.dim;
    const uint32_t hidden = a.rows.hidden;
    const uint64_t n0 = t.n0;
    Feed f;
    f.a[1] = f.b[1] = nullptr;
    if constexpr (KIND == kFfnGradWeights) {
        f.k = t.rows;
        if (t.weight < 2) {
            f.a[0] = a.dproj + static_cast<uint64_t>(t.start) * hidden * 4 + (static_cast<uint64_t>(t.weight) * hidden + t.m0) * 2;
            f.b[0] = a.p[0][t.rank] + n0 * 2;
            f.a_ld = hidden * 4;
            f.b_ld = dim * 2;
            f.a_extent = hidden - t.m0;
            f.b_extent = dim - t.n0;
        } else {
            f.a[0] = a.p[1][t.rank] + static_cast<uint64_t>(t.m0) * 2;
            f.b[0] = a.h + static_cast<uint64_t>(t.start) * hidden * 2 + n0 * 2;
            f.a_ld = dim * 2;
            f.b_ld = hidden * 2;
            f.a_extent = dim - t.m0;
            f.b_extent = hidden - t.n0;
        }
    } else {
        const uint64_t row = static_cast<uint64_t>(t.start) + t.m0;
        f.a_extent = t.rows - t.m0;
        if constexpr (KIND == kFfnGateUp) {
            f.k = dim;
            f.a[0] = a.x16 != nullptr ? a.x16 + row * dim * 2 : a.p[0][t.rank] + static_cast<uint64_t>(t.m0) * dim * 2;
            f.b[0] = a.p[wave * (BN / kWaves) >= BN / 2 ? 2 : 1][t.rank] + n0 * dim * 2;   // of the rows that this wavefront stages
            f.a_ld = f.b_ld = dim * 2;
            f.b_extent = hidden - t.n0;
        } else if constexpr (KIND == kFfnDown) {
            f.k = hidden;
            f.a[0] = a.h + row * hidden * 2;
            f.b[0] = a.p[0][t.rank] + n0 * hidden * 2;
            f.a_ld = f.b_ld = hidden * 2;
            f.b_extent = dim - t.n0;
        } else if constexpr (KIND == kFfnGradHidden) {
            f.k = dim;
            f.a[0] = a.p[0][t.rank] + static_cast<uint64_t>(t.m0) * dim * 2;
            f.b[0] = a.p[1][t.rank] + n0 * 2;
            f.a_ld = dim * 2;
            f.b_ld = hidden * 2;
            f.b_extent = hidden - t.n0;
        } else {
            f.k = hidden;
            f.a[0] = a.dproj + row * hidden * 4;
            f.a[1] = f.a[0] + static_cast<uint64_t>(hidden) * 2;
            f.b[0] = a.p[0][t.rank] + n0 * 2;
            f.b[1] = a.p[1][t.rank] + n0 * 2;
            f.a_ld = hidden * 4;
            f.b_ld = dim * 2;
            f.b_extent = dim - t.n0;
        }
    }
    return f;
}

// All but the youngest LOADS loads of this wavefront and all its LDS reads are done, and everybody has got here.
template <int LOADS>
__device__ __forceinline__ void meet()
{
    static_assert(LOADS < 64, "the counter's range");
    __builtin_amdgcn_sched_barrier(0);   // the matrix instructions in front stay there and run while this waits
    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"(LOADS) : "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
}

// Writes a tile of C, or what becomes of it.
template <int DT, int KIND, int FM, int FN>
__device__ __forceinline__ void results(const FfnArgs &a, const Tile &t, const f32x4 (&acc)[FM][FN], uint32_t wm, uint32_t wn, uint32_t lane)
{
    const uint32_t dim = a.rows.dim;
    const uint32_t hidden = a.rows.hidden;
    asm volatile("" : "+v"(lane));   // what follows from it is not computed ahead of the products, which need the registers
    // A lane holds columns 4 (lane / 16) .. + 3 of row lane % 16 of every fragment of C (col_of), and after pair_up() eight columns
    // of one fragment of two (col_in of the first).  Offsets are from the tile's first row on, in bytes.
    const uint32_t row_in = wm * (FM * 16) + lane % 16;
    const uint32_t col_in = (lane / 16 % 2) * 16 + lane / 32 * 8;
    const uint32_t col_of = lane / 16 * 4;
    constexpr int kOwn = KIND == kFfnGateUp ? FN / 2 : FN;   // fragments of C across
    const uint32_t first = t.n0 + wn * (kOwn * 16);
    const ActTerms terms(a.act);
    if constexpr (KIND == kFfnGradWeights) {
        const uint32_t width = t.weight == 2 ? hidden : dim;
        const uint32_t height = t.weight == 2 ? dim : hidden;
        const Window c(a.p[2 + t.weight][t.rank] + static_cast<uint64_t>(t.m0) * width * 2);
#pragma unroll
        for (int m = 0; m < FM; ++m) {
            const uint32_t row = row_in + m * 16;
            const bool live = t.m0 + row < height;
#pragma unroll
            for (int n = 0; n < FN; n += 2) {
                const uint32_t col = first + n * 16 + col_in;
                c.store(live && col < width ? row * width * 2 + col * 2 : kOut, pair_up(narrow4<DT>(acc[m][n]), narrow4<DT>(acc[m][n + 1])));
            }
        }
    } else {
        const uint64_t packed = static_cast<uint64_t>(t.start) + t.m0;
        if constexpr (KIND == kFfnGateUp) {
            const Window to_h(a.h + packed * hidden * 2);
            const Window to_saved(a.saved + packed * 2 * hidden);
            // the scale of row m0, if rows are of 8 bits
            const char *wire = a.p[0][t.rank] + static_cast<uint64_t>(t.m0) * (dim + HCCLX_ROW8_TAIL) + dim;
#pragma unroll
            for (int m = 0; m < FM; ++m) {
                const uint32_t row = row_in + m * 16;
                const bool live = t.m0 + row < t.rows;
                float scale = 1.0f;
                const char *of_row = wire + static_cast<uint64_t>(row) * (dim + HCCLX_ROW8_TAIL);
                if (a.x16 != nullptr && live) scale = *reinterpret_cast<const float *>(of_row);
                uint2 h[kOwn];
#pragma unroll
                for (int n = 0; n < kOwn; ++n) {
                    const f32x4 g = acc[m][n] * scale;
                    const f32x4 u = acc[m][n + kOwn] * scale;
                    const uint32_t col = first + n * 16 + col_of;
                    if (a.saved != nullptr) {
                        const bool there = live && col < hidden;
                        to_saved.store(there ? row * hidden * 8 + col * 4 : kOut, __builtin_bit_cast(u32x4, g));
                        to_saved.store(there ? row * hidden * 8 + (hidden + col) * 4 : kOut, __builtin_bit_cast(u32x4, u));
                    }
                    f32x4 r;
#pragma unroll
                    for (int e = 0; e < 4; ++e) r[e] = Act(g[e], terms).value * u[e];
                    h[n] = narrow4<DT>(r);
                }
#pragma unroll
                for (int n = 0; n < kOwn; n += 2) {
                    const uint32_t col = first + n * 16 + col_in;
                    to_h.store(live && col < hidden ? row * hidden * 2 + col * 2 : kOut, pair_up(h[n], h[n + 1]));
                }
            }
        } else if constexpr (KIND == kFfnGradHidden) {
            const Window to_h(a.h + packed * hidden * 2);
            const Window to_d(a.dproj + packed * 2 * hidden * 2);
            const Window from(a.saved + packed * 2 * hidden);
#pragma unroll
            for (int m = 0; m < FM; ++m) {
                const uint32_t row = row_in + m * 16;
                const bool live = t.m0 + row < t.rows;
                f32x4 g[FN], u[FN];
#pragma unroll
                for (int n = 0; n < FN; ++n) {
                    const uint32_t col = first + n * 16 + col_of;
                    const bool there = live && col < hidden;
                    g[n] = from.load(there ? row * hidden * 8 + col * 4 : kOut);
                    u[n] = from.load(there ? row * hidden * 8 + (hidden + col) * 4 : kOut);
                }
                uint2 h[FN], dg[FN], du[FN];
#pragma unroll
                for (int n = 0; n < FN; ++n) {
                    f32x4 r, d0, d1;
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const Act f(g[n][e], terms);
                        r[e] = f.value * u[n][e];
                        d0[e] = acc[m][n][e] * u[n][e] * f.slope;
                        d1[e] = acc[m][n][e] * f.value;
                    }
                    h[n] = narrow4<DT>(r);
                    dg[n] = narrow4<DT>(d0);
                    du[n] = narrow4<DT>(d1);
                }
#pragma unroll
                for (int n = 0; n < FN; n += 2) {
                    const uint32_t col = first + n * 16 + col_in;
                    const bool there = live && col < hidden;
                    to_h.store(there ? row * hidden * 2 + col * 2 : kOut, pair_up(h[n], h[n + 1]));
                    to_d.store(there ? row * hidden * 4 + col * 2 : kOut, pair_up(dg[n], dg[n + 1]));
                    to_d.store(there ? row * hidden * 4 + (hidden + col) * 2 : kOut, pair_up(du[n], du[n + 1]));
                }
            }
        } else {
            const Window c((KIND == kFfnDown ? a.p[1][t.rank] : a.p[2][t.rank]) + static_cast<uint64_t>(t.m0) * dim * 2);
#pragma unroll
            for (int m = 0; m < FM; ++m) {
                const uint32_t row = row_in + m * 16;
                const bool live = t.m0 + row < t.rows;
#pragma unroll
                for (int n = 0; n < FN; n += 2) {
                    const uint32_t col = first + n * 16 + col_in;
                    c.store(live && col < dim ? row * dim * 2 + col * 2 : kOut, pair_up(narrow4<DT>(acc[m][n]), narrow4<DT>(acc[m][n + 1])));
                }
            }
        }
    }
}

// Waits until the accumulators' last products, or zeros, are in their registers: what the compiler does by itself for instructions
// that it knows.
template <int FM, int FN>
__device__ __forceinline__ void settle(f32x4 (&acc)[FM][FN])
{
    asm volatile("s_nop 15\n\ts_nop 7" ::: "memory");
#pragma unroll
    for (int m = 0; m < FM; ++m) {
#pragma unroll
        for (int n = 0; n < FN; n += 4) asm volatile("" : "+a"(acc[m][n]), "+a"(acc[m][n + 1]), "+a"(acc[m][n + 2]), "+a"(acc[m][n + 3]));
    }
}

// Tiles of wavefronts of FM x FN fragments each: t and what next(&t) gives after it, until it says no; their operands' rows have the
// same lengths.  The stages of one tile follow those of the one before without a break, so that the first of them are on their way
// while results are written.
template <int DT, int KIND, int FM, int FN, typename Next>
__device__ __forceinline__ void products(const FfnArgs &a, Tile t, char *s_tile, Next &&next)
{
    constexpr uint32_t BM = kWaveRows * FM * 16;
    constexpr uint32_t BN = kWaveCols * FN * 16;
    constexpr bool kPair = KIND == kFfnGateUp;             // half of the columns from either weight
    constexpr bool kAk = KIND != kFfnGradWeights;          // A lies k-wise
    constexpr bool kBk = KIND == kFfnGateUp || KIND == kFfnDown;
    constexpr uint32_t kCols = kPair ? BN / 2 : BN;        // columns of C
    constexpr uint32_t kStageA = BM * kBK * 2;
    constexpr uint32_t kStageB = BN * kBK * 2;
    // As many stages as fit, with one more of A: A's loads go out in the first half of a stage's products and B's in the second.
    constexpr uint32_t kStages = (kLdsBytes - kStageA) / (kStageA + kStageB);
    constexpr uint32_t kPairs = KIND == kFfnGradInput ? 2 : 1;

    const uint32_t wave = uniform(threadIdx.x / 64);
    const uint32_t lane = threadIdx.x & 63;
    const uint32_t wm = wave / kWaveCols;
    const uint32_t wn = wave % kWaveCols;
    auto place_a = [&](uint32_t slot) { return (lds_char *)s_tile + slot * kStageA; };
    auto place_b = [&](uint32_t slot) { return (lds_char *)s_tile + (kStages + 1) * kStageA + slot * kStageB; };
    auto after_a = [](uint32_t slot) { return slot == kStages ? 0 : slot + 1; };
    auto after_b = [](uint32_t slot) { return slot + 1 == kStages ? 0 : slot + 1; };

    Stager<BM, kAk, false> sa;
    Stager<BN, kBk, kPair> sb;
    Feed from = feed_of<KIND, BN>(a, t, wave);
    sa.init(wave, lane, from.a_ld);
    sb.init(wave, lane, from.b_ld);
    constexpr int kLoadsA = decltype(sa)::kLoads;
    constexpr int kLoadsB = decltype(sb)::kLoads;
    constexpr int kLoads = kLoadsA + kLoadsB;
    static_assert(kStages >= 2, "two stages fit");

    // The loads run ahead of the products: `from` is where they are, `then` what follows (if `more`), `left` k of this pair are to
    // come in `steps` stages.  A tile has kStages stages at least (of zeros, if need be): when its products begin, all of those
    // are its own.  Without branches, and in pieces that fit between two matrix instructions; the empty asm keeps the compiler
    // from moving a piece.
    auto stages_of = [&](const Feed &f) -> int {
        const uint32_t n = (f.k + kBK - 1) / kBK * kPairs;
        return n < kStages ? kStages : n;
    };
    Feed then = from;
    uint32_t more = 0;
    uint32_t left = from.k;
    int steps = stages_of(from);
    uint32_t pair = 0;
    struct Stage {
        Resource r;
        uint32_t end, ld;
    };
    Stage ga, gb;   // the next of A to be loaded, and of B
    uint32_t k = 0, rows = 0, range = 0, on = 0;
    auto k_left = [&] { return left < kBK ? left : kBK; };
    constexpr int kPiecesA = 3;
    auto next_a = [&](int i) {
        if (i == 0) {
            k = k_left();
            rows = kAk ? (from.a_extent < BM ? from.a_extent : BM) : k;
            asm volatile("" : "+s"(k), "+s"(rows));
        }
        if (i == 1) {
            range = k == 0 ? 0 : (rows - 1) * from.a_ld + (kAk ? k : from.a_extent) * 2;
            asm volatile("" : "+s"(range));
        }
        if (i == 2) {
            ga = {resource(from.a[0], range), kAk ? k : from.a_extent, from.a_ld};
            asm volatile("" : "+s"(ga.r));
        }
    };
    constexpr int kPiecesB = 11;
    constexpr int kPiecesOfB = 3;   // the others take `from` on to the next stage, or to the next tile if this one's are all on their way
    auto next_b = [&](int i) {
        if (i == 0) {
            k = k_left();
            rows = kBk ? (from.b_extent < kCols ? from.b_extent : kCols) : k;
            asm volatile("" : "+s"(k), "+s"(rows));
        }
        if (i == 1) {
            range = k == 0 ? 0 : (rows - 1) * from.b_ld + (kBk ? k : from.b_extent) * 2;
            asm volatile("" : "+s"(range));
        }
        if (i == 2) {
            gb = {resource(from.b[0], range), kBk ? k : from.b_extent, from.b_ld};
            asm volatile("" : "+s"(gb.r));
        }
        if (i == 3) {
            left -= k;
            from.a[0] += kAk ? kBK * 2 : static_cast<uint64_t>(from.a_ld) * kBK;
            asm volatile("" : "+s"(left), "+s"(from.a[0]));
        }
        if (i == 4) {
            from.b[0] += kBk ? kBK * 2 : static_cast<uint64_t>(from.b_ld) * kBK;
            asm volatile("" : "+s"(from.b[0]));
        }
        if (KIND == kFfnGradInput && i == 5) {
            const bool second = left == 0 && pair == 0;
            pair = second ? 1 : pair;
            left = second ? from.k : left;
            from.a[0] = second ? from.a[1] : from.a[0];
            from.b[0] = second ? from.b[1] : from.b[0];
            asm volatile("" : "+s"(left), "+s"(pair), "+s"(from.a[0]), "+s"(from.b[0]));
        }
        if (i == 6) {
            --steps;
            on = steps <= 0 ? more : 0;
            more -= on;
            asm volatile("" : "+s"(steps), "+s"(on), "+s"(more));
        }
        if (i == 7) {
            from.a[0] = on != 0 ? then.a[0] : from.a[0];
            from.a[1] = on != 0 ? then.a[1] : from.a[1];
            asm volatile("" : "+s"(from.a[0]), "+s"(from.a[1]));
        }
        if (i == 8) {
            from.b[0] = on != 0 ? then.b[0] : from.b[0];
            from.b[1] = on != 0 ? then.b[1] : from.b[1];
            asm volatile("" : "+s"(from.b[0]), "+s"(from.b[1]));
        }
        if (i == 9) {
            from.a_extent = on != 0 ? then.a_extent : from.a_extent;
            from.b_extent = on != 0 ? then.b_extent : from.b_extent;
            from.k = on != 0 ? then.k : from.k;
            asm volatile("" : "+s"(from.a_extent), "+s"(from.b_extent), "+s"(from.k));
        }
        if (i == 10) {
            left = on != 0 ? then.k : left;
            steps = on != 0 ? stages_of(then) : steps;
            pair = on != 0 ? 0 : pair;
            asm volatile("" : "+s"(left), "+s"(steps), "+s"(pair));
        }
    };

    auto issue_a = [&](int i, uint32_t slot) {
        sa.issue(i, ga.r, ga.end, ga.ld, static_cast<uint32_t>(reinterpret_cast<uintptr_t>(place_a(slot))), wave);
    };
    auto issue_b = [&](int i, uint32_t slot) {
        sb.issue(i, gb.r, gb.end, gb.ld, static_cast<uint32_t>(reinterpret_cast<uintptr_t>(place_b(slot))), wave);
    };

    const Reader<kAk, BM> ra(lane);
    const Reader<kBk, BN> rb(lane);
    // the fragments of B that this wavefront takes: of a pair, half from either weight
    auto b_frag = [&](int n) -> uint32_t {
        if constexpr (kPair) {
            constexpr int kHalf = FN / 2;
            return n < kHalf ? wn * kHalf + n : BN / 32 + wn * kHalf + (n - kHalf);
        } else {
            return wn * FN + n;
        }
    };
    // Fragments of 32 k at a time.  While they are multiplied, row of fragments by row, the next ones are read: A's into the
    // registers of the rows done, of which there are kEarly more than rows, so that the last of a stage is read kEarly rows before
    // its end, and B's into a second set.  When everybody has read the last of a stage, the one kStages behind it is loaded into its
    // place, B's in the half that follows and A's in the one after.
    f32x4 acc[FM][FN];
    constexpr int kEarly = 2;
    u32x4 fa[FM + kEarly], fb[2][FN];
    static_assert(FM * 2 >= FN && FN >= 4, "every row of fragments reads two of B at most");
    auto second_of = [](int m) { return m < kEarly ? FM + m : m - kEarly; };   // registers of row m of the second half
    auto fence = [] { __builtin_amdgcn_sched_barrier(0); };
    // Does its share of the pieces before product (m, n) of a half, where nothing is read or loaded.
    auto pieces = [&](int m, int n, int count, auto &&piece) {
        constexpr int kPer = FN == 8 ? 3 : 1;              // places of a row
        constexpr int kPlaces = kPer * 4;
        if (FN == 8 ? n != 1 && n != 3 && n != 6 : n != 1) return;
        const int place = m * kPer + n / 3;
#pragma unroll
        for (int i = 0; i < kPiecesB; ++i) {
            if (i * kPlaces / kPiecesB == place && i < count) piece(i);
        }
    };
    // multiplies the first half of a stage, reads its second half, loads A into slot `to`
    auto first_half = [&](const lds_char *pa, const lds_char *pb, uint32_t to) {
#pragma unroll
        for (int m = 0; m < FM; ++m) {
#pragma unroll
            for (int n = 0; n < FN; ++n) {
                if (m == 0 && n < kEarly) fa[second_of(n)] = ra(pa, wm * FM + n, 1);
                if (m > 0 && n == 0 && m + kEarly - 1 < FM) fa[second_of(m + kEarly - 1)] = ra(pa, wm * FM + m + kEarly - 1, 1);
                if (n * 2 == FN && m * 2 < FN) fb[1][m * 2] = rb(pb, b_frag(m * 2), 1);
                if (n * 2 == FN + 2 && m * 2 + 1 < FN) fb[1][m * 2 + 1] = rb(pb, b_frag(m * 2 + 1), 1);
                if (n == FN - 1) {
#pragma unroll
                    for (int i = m; i < kLoadsA; i += FM) issue_a(i, to);
                }
                pieces(m, n, kPiecesB, next_b);
                Mma<DT>::add(acc[m][n], fb[0][n], fa[m]);
                fence();
            }
        }
    };
    // multiplies the second half, reads the first half of the next stage, loads B into slot `to`
    auto second_half = [&](const lds_char *pa, const lds_char *pb, uint32_t to) {
#pragma unroll
        for (int m = 0; m < FM; ++m) {
#pragma unroll
            for (int n = 0; n < FN; ++n) {
                if (n == 0 && m < kEarly) fa[FM - kEarly + m] = ra(pa, wm * FM + FM - kEarly + m, 0);
                if (n == 0 && m > kEarly) fa[m - 1 - kEarly] = ra(pa, wm * FM + m - 1 - kEarly, 0);
                if (n * 2 == FN) {
#pragma unroll
                    for (int i = m; i < FN; i += FM) fb[0][i] = rb(pb, b_frag(i), 0);
                }
                if (n == FN - 1) {
#pragma unroll
                    for (int i = m; i < kLoadsB; i += FM) issue_b(i, to);
                }
                pieces(m, n, kPiecesA, next_a);
                Mma<DT>::add(acc[m][n], fb[1][n], fa[second_of(m)]);
                fence();
            }
        }
        fa[FM - 1 - kEarly] = ra(pa, wm * FM + FM - 1 - kEarly, 0);
    };
    int total = steps;
    uint32_t at_a = 0, at_b = 0;
#pragma unroll 1
    for (uint32_t slot = 0; slot < kStages; ++slot) {   // (a loop: this runs once, and takes as long as its instructions take to come)
        for (int i = 0; i < kPiecesA; ++i) next_a(i);
        for (int i = 0; i < kPiecesOfB; ++i) next_b(i);
        asm volatile("s_nop 4" ::: "memory");
#pragma unroll
        for (int i = 0; i < kLoadsA; ++i) issue_a(i, slot);
#pragma unroll
        for (int i = 0; i < kLoadsB; ++i) issue_b(i, slot);
        for (int i = kPiecesOfB; i < kPiecesB; ++i) next_b(i);
    }
    bool landed = false;   // the tile's first stage, with the others
    for (;;) {
        Tile after = t;
        const bool last = !next(&after);
        if (!last) then = feed_of<KIND, BN>(a, after, wave);
        more = scalar(last ? 0 : 1);
        if (steps <= 0 && more != 0) {   // this tile's stages are all on their way already
            more = 0;
            from = then;
            left = from.k;
            steps = stages_of(from);
            pair = 0;
        }
        if (!landed) meet<kLoads *(kStages - 1)>();
        landed = true;
        {   // (read here, not by the last turn of the tile before: writing results needs the registers)
#pragma unroll
            for (int m = 0; m < FM; ++m) fa[m] = ra(place_a(at_a), wm * FM + m, 0);
#pragma unroll
            for (int n = 0; n < FN; ++n) fb[0][n] = rb(place_b(at_b), b_frag(n), 0);
        }
#pragma unroll
        for (int m = 0; m < FM; ++m) {
#pragma unroll
            for (int n = 0; n < FN; ++n) acc[m][n] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
        }
        for (int i = 0; i < kPiecesA; ++i) next_a(i);
        settle<FM, FN>(acc);
        for (int step = 0; step < total; ++step) {
            first_half(place_a(at_a), place_b(at_b), at_a == 0 ? kStages : at_a - 1);
            meet<kLoads *(kStages - 2) + kLoadsA>();   // the next stage has landed; of a new tile's first, the results before it have left, too
            const uint32_t to = at_b;
            at_a = after_a(at_a);
            at_b = after_b(at_b);
            second_half(place_a(at_a), place_b(at_b), to);
        }
        settle<FM, FN>(acc);
        results<DT, KIND, FM, FN>(a, t, acc, wm, wn, lane);
        if (last) break;
        t = after;
        total = stages_of(then);
    }
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");   // nothing may be on its way to LDS when it is given back
}

// How C is cut: into whole tiles and their parts; or, for ranks of fewer rows than a whole tile has, into tiles of 128 x 128 (four
// stages on their way instead of two) or of 128 x 256 (three).
enum Cut { kCutWhole, kCutSmall, kCutWide };

// One workgroup per CU.  It takes its share of the tiles, one of every round, and then of the parts.
template <int DT, int KIND, Cut CUT>
__global__ void __launch_bounds__(kWaves * 64, 1)
k_ffn(FfnArgs a)
{
    static_assert(CUT == kCutWhole || KIND != kFfnGradWeights, "whose tiles are full however few the rows");
    constexpr uint32_t kEdge = CUT == kCutWhole ? kTile : kTile / 2;
    constexpr uint32_t kWide = CUT == kCutSmall ? kTileCols<KIND> / 2 : kTileCols<KIND>;
    __shared__ __attribute__((aligned(1024))) char s_tile[kLdsBytes];
    const FfnRows &s = a.rows;
    // (read together; otherwise the way to the first load is a row of waits for one argument each)
    asm volatile("" ::"s"(s.counts), "s"(s.per_rank), "s"(s.unit), "s"(s.n), "s"(s.capacity), "s"(s.most), "s"(s.dim), "s"(s.hidden), "s"(a.h),
                 "s"(a.dproj), "s"(a.saved), "s"(a.x16), "s"(a.act));
    auto count = [](uint32_t size, uint32_t edge) { return (size + edge - 1) / edge; };
    // kFfnGradWeights: all ranks' tiles of the projections' gradients, then those of w_down's
    const uint32_t across = count(KIND == kFfnGradWeights ? s.dim : columns<KIND>(s), KIND == kFfnGradWeights ? kEdge : kWide);
    const uint32_t across1 = count(s.hidden, kEdge);
    const uint32_t tiles0 = 2 * across1 * across;
    const uint32_t tiles1 = count(s.dim, kEdge) * across1;
    const uint32_t both0 = scalar(s.n) * tiles0;   // of all ranks (read by a part of the workgroup too, which makes it a vector)
    const uint32_t both1 = scalar(s.n) * tiles1;
    const RankRows mine(s);   // (of the lane's rank)
    const uint32_t mine_down = count(mine.rows, kEdge);
    const uint32_t mine_upto = inclusive_sum(mine_down * across);   // tiles of this rank and those before it
    auto tile = [&](uint32_t at, Tile *t) {
        t->weight = 0;
        if constexpr (KIND == kFfnGradWeights) {
            const bool down = at >= both0;
            at -= down ? both0 : 0;
            t->rank = scalar(at / (down ? tiles1 : tiles0));
            in_groups(at % (down ? tiles1 : tiles0), down ? across : 2 * across1, down ? across1 : across, &t->m0, &t->n0);
            t->weight = down ? 2 : t->m0 >= across1 ? 1 : 0;
            t->m0 -= t->weight == 1 ? across1 : 0;
        } else {
            t->rank = __builtin_ctzll(__ballot(mine_upto > at));
            const uint32_t down = of_lane(mine_down, t->rank);
            in_groups(at - (of_lane(mine_upto, t->rank) - down * across), down, across, &t->m0, &t->n0);
        }
        t->rows = of_lane(mine.rows, t->rank);
        t->start = of_lane(mine.start, t->rank);
        t->m0 *= kEdge;
        t->n0 *= kWide;
    };
    const uint32_t tiles = KIND == kFfnGradWeights ? both0 + both1 : of_lane(mine_upto, kFfnRanks - 1);
    const uint32_t turned = blockIdx.x % 8 * (gridDim.x / 8) + blockIdx.x / 8;
    uint32_t at = turned;
    uint32_t end = tiles;
    auto next = [&](Tile *then) {
        at += gridDim.x;
        if (at >= end) return false;
        tile(at, then);
        return true;
    };
    Tile t;
    if constexpr (CUT != kCutWhole) {
        if (at >= end) return;
        tile(at, &t);
        products<DT, KIND, 4, CUT == kCutWide ? 8 : 4>(a, t, s_tile, next);
    } else {
        const Share share(tiles, gridDim.x);
        for (uint32_t group = 0; group < (KIND == kFfnGradWeights ? 2 : 1); ++group) {
            end = group == 0 && KIND == kFfnGradWeights && share.whole > both0 ? both0 : share.whole;
            if (at >= end) continue;
            __syncthreads();   // everybody is done with the LDS of the tiles before
            tile(at, &t);
            products<DT, KIND, 8, 8>(a, t, s_tile, next);
        }
        if (turned >= share.left * share.parts) return;
        const uint32_t part = scalar(turned % share.parts);
        tile(scalar(share.whole + turned / share.parts), &t);
        t.n0 += part % 2 * (kTileCols<KIND> / 2);
        if (share.parts == 4) t.m0 += part / 2 * (kTile / 2);
        // a part may have no column or row
        if constexpr (KIND == kFfnGradWeights) {
            if (t.n0 >= (t.weight == 2 ? s.hidden : s.dim) || t.m0 >= (t.weight == 2 ? s.dim : s.hidden)) return;
        } else {
            if (t.n0 >= columns<KIND>(s) || t.m0 >= t.rows) return;
        }
        __syncthreads();   // everybody is done with the last whole tile's LDS
        auto none = [](Tile *) { return false; };
        if (share.parts == 2) {
            products<DT, KIND, 8, 4>(a, t, s_tile, none);
        } else {
            products<DT, KIND, 4, 4>(a, t, s_tile, none);
        }
    }
}

// The values of 8-bit codes in 16 bits, which hold every e4m3 value exactly; the rows' scales are applied to the products.  A
// workgroup per packed row: 8 ranks x 64 rows of 7168 6.4 us (a wavefront per row: 8.6).
template <int DT>
__global__ void __launch_bounds__(256)
k_ffn_widen(FfnArgs a)
{
    const FfnRows &s = a.rows;
    const RankRows mine(s);
    const uint32_t packed = blockIdx.x;
    const uint64_t has = __ballot(packed - mine.start < mine.rows && packed >= mine.start);
    if (has == 0) return;
    const uint32_t rank = __builtin_ctzll(has);
    const uint32_t row = packed - of_lane(mine.start, rank);
    const char *from = a.p[0][rank] + static_cast<uint64_t>(row) * (s.dim + HCCLX_ROW8_TAIL);
    char *to = a.x16 + static_cast<uint64_t>(packed) * s.dim * 2;
    for (uint32_t c = threadIdx.x * 16; c < s.dim; c += 4096) {
        const u32x4 codes = *reinterpret_cast<const u32x4 *>(from + c);
#pragma unroll
        for (int q = 0; q < 2; ++q) *reinterpret_cast<u32x4 *>(to + (c + q * 8) * 2) = widen8<DT>(codes[2 * q], codes[2 * q + 1]);
    }
}

template <int DT, int KIND>
hipError_t run(const FfnArgs &a, Cut cut, uint32_t num_cus, hipStream_t st)
{
    if (a.rows.most == 0 && KIND != kFfnGradWeights) return hipSuccess;
    const dim3 groups(num_cus < 32 ? 32 : num_cus / 32 * 32);   // a multiple of eight, and its half and quarter too
    const dim3 block(kWaves * 64);
    if constexpr (KIND == kFfnGradWeights) {
        HCCLX_LAUNCH((k_ffn<DT, KIND, kCutWhole>), groups, block, 0, st, a);
    } else if (cut == kCutWhole) {
        HCCLX_LAUNCH((k_ffn<DT, KIND, kCutWhole>), groups, block, 0, st, a);
    } else if (cut == kCutSmall) {
        HCCLX_LAUNCH((k_ffn<DT, KIND, kCutSmall>), groups, block, 0, st, a);
    } else {
        HCCLX_LAUNCH((k_ffn<DT, KIND, kCutWide>), groups, block, 0, st, a);
    }
    return hipGetLastError();
}

}  // namespace ffn

}  // namespace hcclx
