// Logits whose columns are split over the ranks (include/hcclx_ops.h: hcclx_logits_t): how a kernel finds its way through a row, and
// what the kernels that read rows share.
//
// A row is cut into chunks of 64 vectors of 16 bytes, which begin anew with every rank's columns: a wavefront reads a chunk with one
// load per lane, at any alignment of the row.  Chunks are numbered in the order of their columns.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>
#include <string>
#include <vector>
#include "hcclx_internal.h"
#include "hcclx_ops.h"
#include "kernels/elem.h"
#include "kernels/fold.h"
#include "ops/lanes.h"

namespace hcclx {
namespace logits {

constexpr uint32_t kMostRanks = 64;
constexpr uint32_t kMostRows = (1u << 22) - 1;   // a workgroup of up to 1024 for each, in one launch

// Neighbouring columns of one rank: a chunk, or all of a rank's.
struct alignas(32) Stretch {
    const char *at;    // of row 0
    char *to;          // where row 0's gradient goes
    uint64_t step;     // bytes from one row to the next
    uint32_t first;    // number of the first column
    uint32_t elems;
};

struct Rows {
    const Stretch *chunks;
    const Stretch *ranks;   // those that have columns
    uint32_t nchunks;
    uint32_t nranks;
    uint32_t rows;
    uint32_t vocab;
};

template <int DT> constexpr uint32_t kChunk = 64 * Vec16<DT>::NE;   // elements

__device__ __forceinline__ float minus_infinity() { return -__builtin_inff(); }

// Lane `lane`'s vector of a chunk whose row begins at `at`; what does not exist is minus infinity.
template <int DT, bool ONCE>
__device__ __forceinline__ u32x4 load_piece(const char *at, uint32_t lane, uint32_t elems)
{
    using V = Vec16<DT>;
    using S = typename V::S;
    const uint32_t from = lane * V::NE;
    if (from + V::NE <= elems) {
        const char *p = at + lane * 16;
        return ONCE ? __builtin_nontemporal_load(as_global(p)) : ld16_cached(p);
    }
    S tmp[V::NE];
#pragma unroll
    for (int e = 0; e < V::NE; ++e) tmp[e] = from + e < elems ? reinterpret_cast<const S *>(at)[from + e] : V::D::narrow(minus_infinity());
    u32x4 raw;
    __builtin_memcpy(&raw, tmp, 16);
    return raw;
}

// One element, widened.
template <int DT>
__device__ __forceinline__ float load_one(const char *at, uint32_t k)
{
    using D = DTypeOf<DT>;
    return D::widen(reinterpret_cast<const typename D::S *>(at)[k]);
}

// The stretch that column k lies in (k < vocab).
__device__ __forceinline__ const Stretch *rank_of(const Rows &r, uint32_t k)
{
    uint32_t j = 0;
    for (uint32_t i = 1; i < r.nranks; ++i) j = r.ranks[i].first <= k ? i : j;
    return r.ranks + j;
}

// 2^x, good to a unit or two in the last place from 2^-126 up, 0 below.
__device__ __forceinline__ float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }

// 2^y for y <= 0, good to a few units in 2^53 of the result: y = n + f with |f| <= 1/2, and the power series of exp(f ln 2), whose first
// omitted term is below 2^-52.  Anything that is no number above -1000, NaN too, gives 0.
__device__ __forceinline__ double exp2_exact(double y)
{
    if (!(y > -1000.0)) return 0.0;
    const double n = rint(y);
    const double z = (y - n) * 0.69314718055994530942;
    double p = 1.0 / 479001600;
    p = __builtin_fma(p, z, 1.0 / 39916800);
    p = __builtin_fma(p, z, 1.0 / 3628800);
    p = __builtin_fma(p, z, 1.0 / 362880);
    p = __builtin_fma(p, z, 1.0 / 40320);
    p = __builtin_fma(p, z, 1.0 / 5040);
    p = __builtin_fma(p, z, 1.0 / 720);
    p = __builtin_fma(p, z, 1.0 / 120);
    p = __builtin_fma(p, z, 1.0 / 24);
    p = __builtin_fma(p, z, 1.0 / 6);
    p = __builtin_fma(p, z, 0.5);
    p = __builtin_fma(p, z, 1.0);
    p = __builtin_fma(p, z, 1.0);
    return ldexp(p, static_cast<int>(n));
}

typedef unsigned long long u64;

// v of the lane that DPP control CTRL names, in the rows of 16 lanes that ROWS names; 0 elsewhere.
template <int CTRL, int ROWS, typename T>
__device__ __forceinline__ T dpp_or_zero(T v)
{
    static_assert(sizeof(T) == 4 || sizeof(T) == 8, "");
    if constexpr (sizeof(T) == 4) {
        return __builtin_bit_cast(T, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), CTRL, ROWS, 0xf, false));
    } else {
        const u64 x = __builtin_bit_cast(u64, v);
        const uint32_t lo = __builtin_amdgcn_update_dpp(0, static_cast<int>(x), CTRL, ROWS, 0xf, false);
        const uint32_t hi = __builtin_amdgcn_update_dpp(0, static_cast<int>(x >> 32), CTRL, ROWS, 0xf, false);
        return __builtin_bit_cast(T, static_cast<u64>(hi) << 32 | lo);
    }
}
// v of the last lane.
template <typename T>
__device__ __forceinline__ T of_last_lane(T v)
{
    if constexpr (sizeof(T) == 4) {
        return __builtin_bit_cast(T, __builtin_amdgcn_readlane(__builtin_bit_cast(int, v), 63));
    } else {
        const u64 x = __builtin_bit_cast(u64, v);
        const uint32_t lo = __builtin_amdgcn_readlane(static_cast<int>(x), 63);
        const uint32_t hi = __builtin_amdgcn_readlane(static_cast<int>(x >> 32), 63);
        return __builtin_bit_cast(T, static_cast<u64>(hi) << 32 | lo);
    }
}
// Sums over the lanes up to this one, and over all; the largest.  All in registers (through LDS a step takes ten times as long).
template <typename T>
__device__ __forceinline__ T wave_sums(T v)
{
    v += dpp_or_zero<0x111, 0xf>(v);   // row_shr 1, 2, 4, 8
    v += dpp_or_zero<0x112, 0xf>(v);
    v += dpp_or_zero<0x114, 0xf>(v);
    v += dpp_or_zero<0x118, 0xf>(v);
    v += dpp_or_zero<0x142, 0xa>(v);   // lane 15 of rows 0 and 2 to the rows behind
    v += dpp_or_zero<0x143, 0xc>(v);   // lane 31 to rows 2 and 3
    return v;
}
template <typename T>
__device__ __forceinline__ T wave_total(T v) { return of_last_lane(wave_sums(v)); }

// The largest, or NaN if there is one.
__device__ __forceinline__ double larger(double a, double b) { return b > a || b != b ? b : a; }
template <int CTRL, int ROWS>
__device__ __forceinline__ double larger_of_lane(double v)
{
    const u64 x = __builtin_bit_cast(u64, v);
    const int low = static_cast<int>(x), high = static_cast<int>(x >> 32);
    const uint32_t lo = __builtin_amdgcn_update_dpp(low, low, CTRL, ROWS, 0xf, false);
    const uint32_t hi = __builtin_amdgcn_update_dpp(high, high, CTRL, ROWS, 0xf, false);
    return larger(v, __builtin_bit_cast(double, static_cast<u64>(hi) << 32 | lo));
}
__device__ __forceinline__ double wave_largest(double v)
{
    v = larger_of_lane<0x111, 0xf>(v);
    v = larger_of_lane<0x112, 0xf>(v);
    v = larger_of_lane<0x114, 0xf>(v);
    v = larger_of_lane<0x118, 0xf>(v);
    v = larger_of_lane<0x142, 0xa>(v);
    return of_last_lane(larger_of_lane<0x143, 0xc>(v));
}

// ---- host -------------------------------------------------------------------------------------------------------------

// The stretches of a plan in device memory.
struct Table {
    DeviceBlock block;
    uint64_t bytes = 0;
    Rows rows{};
};

// Checks what a caller says about its logits.  to: pointers that gradients go to, or nullptr.
int check(const hcclx_logits_t &l, void *const *to, uint32_t *vocab);
// Bytes between the first and the last element of a rank's rows, and its row in bytes.
uint64_t extent(const hcclx_logits_t &l, uint32_t j);
uint64_t stride(const hcclx_logits_t &l, uint32_t j);
// Refuses what is written on what is read: `bytes` at p against every rank's columns of `of`.
int check_apart(const hcclx_logits_t &l, const char *of_what, const void *const *of, const char *what, const void *p, uint64_t bytes);
int check_apart(const char *what, const void *p, uint64_t bytes, const char *other, const void *q, uint64_t other_bytes);
// Gradients may lie on their own rank's logits, and on nothing else that is read.
int check_gradients(const hcclx_logits_t &l, void *const *to);
int check_array(const void *p, uint64_t align, bool optional, const char *what);
// Lays the table out and copies it to the device.
int lay_out(const hcclx_logits_t &l, void *const *to, uint32_t vocab, Table *table);

}  // namespace logits
}  // namespace hcclx
