// The loss of a student against a teacher's top logits, and its gradient (include/hcclx_ops.h: hcclx_distill_*).
//
// With c = log2(e) / T, r the row's largest logit and S the sum over the row of 2^((l - r) c):
//     q = 2^((l - r) c) / S,   log q = (l - r) c ln 2 - log S
// so a row needs one pass for r and S (a running reference and sum per lane, joined at the end) and one for the gradient.  The
// difference comes first, so that the largest term is 1 whatever the logits' magnitude, and c is held in two floats: with one, as far off as
// 2^-25 of itself, S of logits some 20 powers of two below the largest was off by 2e-7, which the difference q - p of a student that mostly
// agrees showed twentyfold.  What concerns the teacher's k entries alone is computed in 64 bits: the loss is a small difference of
// logarithms.
#include "ops/logits.h"

#include <algorithm>
#include <cmath>

using namespace hcclx;
using namespace hcclx::logits;

namespace {

constexpr uint32_t kThreads = 512;
constexpr uint32_t kSmall = 256;                                 // of a workgroup for a short row
constexpr uint32_t kMostWaves = kThreads / 64;
constexpr int kAhead = 4;                                        // chunks of a wavefront that are on their way together
constexpr int kHeld = 8;                                         // vectors of a thread that holds its part of a row
constexpr uint32_t kFree = 0xffffffffu;
constexpr double kLn2 = 0.69314718055994530942;

struct DistillArgs {
    Rows rows;
    const char *teacher;
    const int32_t *indices;
    const float *weight;   // nullptr: 1
    float *loss;
    float2 *stats;         // written with the loss; read where there is none
    float2 *parts;         // r and S of the parts of every row: [rows][nparts]
    float *student;        // [rows][k]: the student's logits at the teacher's entries, where several workgroups share a row
    uint32_t nparts;       // of the rows whose r and S are in `parts`
    uint32_t k;
    uint32_t mask;         // slots of the table of the entries' columns, less one
    int teacher_dtype;
    float c;               // log2(e) / T: the float below it, and what is left, which is more than 0
    float c_low;
    double T;
    double c64;
};

// r and S of a set of columns: S = sum of 2^((l - r) c).  r = -infinity: nothing in it (S = 0).
struct Sum {
    float r;
    float s;
};
// (l - r) c.  (The second part of c is positive: minus infinity stays that.)
__device__ __forceinline__ float exponent(const DistillArgs &a, float l, float r)
{
    const float d = l - r;
    return __builtin_fmaf(d, a.c_low, d * a.c);
}
// S with the reference r, of which v.r is no more.  (A NaN among the logits is in S, not in r.)
__device__ __forceinline__ float with(const DistillArgs &a, Sum v, float r) { return r == minus_infinity() ? v.s : v.s * exp2_fast(exponent(a, v.r, r)); }
__device__ __forceinline__ Sum join(const DistillArgs &a, Sum v, Sum o)
{
    const float r = fmaxf(v.r, o.r);
    return {r, with(a, v, r) + with(a, o, r)};
}
// Over a wavefront, the same in every lane: a common reference first.
__device__ __forceinline__ Sum wave_join(const DistillArgs &a, Sum v)
{
    float r = v.r;
    r = fmaxf(r, dpp_or<0x111>(r, r));
    r = fmaxf(r, dpp_or<0x112>(r, r));
    r = fmaxf(r, dpp_or<0x114>(r, r));
    r = fmaxf(r, dpp_or<0x118>(r, r));
    r = fmaxf(r, dpp_or<0x142>(r, r));
    r = of_last_lane(fmaxf(r, dpp_or<0x143>(r, r)));
    return {r, wave_total(with(a, v, r))};
}

// (fmaxf first makes a quiet NaN of every operand that may be a signalling one, half as much work again.  What NaN does to the largest is
// of no matter: it is in the sum.)
__device__ __forceinline__ float max3(float a, float b, float c)
{
    float r;
    asm("v_max3_f32 %0, %1, %2, %3" : "=v"(r) : "v"(a), "v"(b), "v"(c));
    return r;
}

// What N vectors add to a sum whose reference is `mine.r`, of a lane.
template <int DT, int N>
__device__ __forceinline__ Sum lane_sum(const DistillArgs &a, Sum mine, const u32x4 (&raw)[N])
{
    using V = Vec16<DT>;
    constexpr int NE = V::NE;
    float most = minus_infinity();
#pragma unroll
    for (int u = 0; u < N; ++u) {
        float f[NE];
        V::unpack(raw[u], f);
#pragma unroll
        for (int e = 0; e < NE; e += 2) most = max3(most, f[e], f[e + 1]);
    }
    const float r = fmaxf(mine.r, most);
    const float ref = r == minus_infinity() ? 0.0f : r;   // (nothing yet: the terms are 2^-infinity)
    float sum = mine.s * exp2_fast(exponent(a, mine.r, ref));
#pragma unroll
    for (int u = 0; u < N; ++u) {
        float f[NE];
        V::unpack(raw[u], f);
        float part = exp2_fast(exponent(a, f[0], ref));
#pragma unroll
        for (int e = 1; e < NE; ++e) part += exp2_fast(exponent(a, f[e], ref));
        sum += part;
    }
    return {r, sum};
}
template <int NT>
__device__ __forceinline__ Sum all_sum(const DistillArgs &a, Sum mine, Sum *s)
{
    mine = wave_join(a, mine);
    if ((threadIdx.x & 63) == 0) s[threadIdx.x / 64] = mine;
    __syncthreads();
    float r = s[0].r;
#pragma unroll
    for (uint32_t w = 1; w < NT / 64; ++w) r = fmaxf(r, s[w].r);
    float sum = 0.0f;
#pragma unroll
    for (uint32_t w = 0; w < NT / 64; ++w) sum += with(a, s[w], r);
    return {r, sum};
}

// r and S over the chunks from..to of a row, of all threads (s: one for each wavefront).
template <int DT, int NT, bool ONCE>
__device__ __forceinline__ Sum row_sum(const DistillArgs &a, uint64_t row, uint32_t from, uint32_t to, Sum *s)
{
    constexpr uint32_t kWaves = NT / 64;
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
    const uint32_t lane = threadIdx.x & 63;
    Sum mine = {minus_infinity(), 0.0f};
    for (uint32_t first = from + wave; first < to; first += kWaves * kAhead) {
        u32x4 raw[kAhead];
#pragma unroll
        for (int u = 0; u < kAhead; ++u) {
            const uint32_t i = first + u * kWaves;
            const Stretch t = a.rows.chunks[i < to ? i : from];
            raw[u] = load_piece<DT, ONCE>(t.at + row * t.step, lane, i < to ? t.elems : 0);
        }
        mine = lane_sum<DT>(a, mine, raw);
    }
    return all_sum<NT>(a, mine, s);
}

__device__ __forceinline__ double teacher_logit(const DistillArgs &a, uint64_t at)
{
    if (a.teacher_dtype == HCCL_DATA_TYPE_FP32) return load_one<HCCL_DATA_TYPE_FP32>(a.teacher + at * 4, 0);
    return a.teacher_dtype == HCCL_DATA_TYPE_FP16 ? load_one<HCCL_DATA_TYPE_FP16>(a.teacher + at * 2, 0)
                                                  : load_one<HCCL_DATA_TYPE_BFP16>(a.teacher + at * 2, 0);
}

// Sum or largest of a double over all threads, in a fixed order.  One barrier: s is written once.
template <int NT, bool MAX>
__device__ __forceinline__ double all_of(double v, double *s)
{
    v = MAX ? wave_largest(v) : wave_total(v);
    if ((threadIdx.x & 63) == 0) s[threadIdx.x / 64] = v;
    __syncthreads();
    v = s[0];
#pragma unroll
    for (uint32_t w = 1; w < NT / 64; ++w) v = MAX ? larger(v, s[w]) : v + s[w];
    return v;
}

// The teacher's entries of a row: thread t has the entries t, t + NT, ...
template <int NT>
struct Entries {
    static constexpr uint32_t kEach = (HCCLX_TOP_MAX + NT - 1) / NT;
    uint32_t at[kEach];    // column, or kFree: no entry, or one that names no column
    double t[kEach];       // its logit / T
    double p[kEach];
    bool any;              // whether the row has one that is not minus infinity
    bool nan;              // whether p is no number: the teacher has NaN or infinity

    __device__ __forceinline__ void read(const DistillArgs &a, uint64_t row)
    {
#pragma unroll
        for (uint32_t i = 0; i < kEach; ++i) {
            const uint32_t e = threadIdx.x + i * NT;
            at[i] = kFree;
            t[i] = -__builtin_inf();
            if (e < a.k) {
                const uint32_t c = static_cast<uint32_t>(a.indices[row * a.k + e]);
                if (c < a.rows.vocab) {
                    at[i] = c;
                    t[i] = teacher_logit(a, row * a.k + e) / a.T;
                }
            }
        }
    }
    // p of every entry, log p in t
    __device__ __forceinline__ void normalise(double (*s)[kMostWaves])
    {
        double most = t[0];
#pragma unroll
        for (uint32_t i = 1; i < kEach; ++i) most = larger(most, t[i]);
        most = all_of<NT, true>(most, s[0]);
        any = !(most == -__builtin_inf());
        double sum = 0.0;
#pragma unroll
        for (uint32_t i = 0; i < kEach; ++i) {
            p[i] = any && at[i] != kFree ? exp(t[i] - most) : 0.0;
            sum += p[i];
        }
        sum = all_of<NT, false>(sum, s[1]);
        const double log_sum = log(sum);
        nan = sum != sum;
#pragma unroll
        for (uint32_t i = 0; i < kEach; ++i) {
            p[i] = any ? p[i] / sum : 0.0;
            t[i] = t[i] - most - log_sum;
        }
    }
};

struct DistillShared {
    Sum sums[kMostWaves];
    double reduce[3][kMostWaves];
};
extern __shared__ unsigned long long s_table[];   // sums and columns of the entries, as many as the plan's k needs (Together)

// Sums p over the entries that name the same column: where the entry's sum is.  Sums are of whole numbers, so that their order does not
// show: p is rounded to 2^-62 there, 2^-24 of what is as improbable as 2^-38.  A column that one entry names has that entry's p as it is.  Between
// the table's making and the first entry lies a barrier of the caller's.
template <int NT>
struct Together {
    unsigned long long *const sum;
    uint32_t *const column;
    const uint32_t mask;
    // (used: false where the launch has no memory for it)
    __device__ __forceinline__ Together(uint32_t last, bool used) : sum(s_table), column(reinterpret_cast<uint32_t *>(s_table + last + 1)), mask(last)
    {
        for (uint32_t i = threadIdx.x; used && i <= mask; i += NT) {
            column[i] = kFree;
            sum[i] = 0;
        }
    }
    static constexpr uint32_t kShared = 0x80000000u;   // (no column has this bit)
    __device__ __forceinline__ uint32_t add(uint32_t c, double p)
    {
        uint32_t i = (c * 2654435769u) >> 16 & mask;
        for (;;) {   // (at most half of the slots are taken)
            const uint32_t was = atomicCAS(&column[i], kFree, c);
            if (was == c) atomicOr(&column[i], kShared);
            if (was == kFree || (was & ~kShared) == c) break;
            i = (i + 1) & mask;
        }
        atomicAdd(&sum[i], static_cast<unsigned long long>(p * 0x1p62));
        return i;
    }
    // The sum at i, given an entry of it.
    __device__ __forceinline__ double of(uint32_t i, double p) const
    {
        const bool shared = (column[i] & kShared) != 0;
        const double all = static_cast<double>(sum[i]) * 0x1p-62;
        return shared ? all : p;
    }
};

template <int DT>
__device__ __forceinline__ void store_piece(char *to, uint32_t lane, uint32_t elems, const float (&f)[Vec16<DT>::NE])
{
    using V = Vec16<DT>;
    using S = typename V::S;
    const uint32_t from = lane * V::NE;
    if (from + V::NE <= elems) {
        if constexpr (DT == HCCL_DATA_TYPE_BFP16) {   // (two at once, to nearest even as D::narrow)
            typedef float f2 __attribute__((ext_vector_type(2)));
            typedef __bf16 b2 __attribute__((ext_vector_type(2)));
            u32x4 raw;
#pragma unroll
            for (int e = 0; e < 4; ++e) raw[e] = __builtin_bit_cast(uint32_t, __builtin_convertvector((f2{f[2 * e], f[2 * e + 1]}), b2));
            st16(to + lane * 16, raw);
        } else {
            st16(to + lane * 16, V::pack(f));
        }
        return;
    }
#pragma unroll
    for (int e = 0; e < V::NE; ++e) {
        if (from + e < elems) reinterpret_cast<S *>(to)[from + e] = V::D::narrow(f[e]);
    }
}

// Gradient of the chunks from..to of a row where p is 0: scale 2^((l - r) c); or zeros.
template <int DT, int NT, bool ZERO>
__device__ __forceinline__ void row_gradient(const DistillArgs &a, uint64_t row, uint32_t from, uint32_t to, float r, float scale)
{
    using V = Vec16<DT>;
    constexpr int NE = V::NE;
    constexpr uint32_t kWaves = NT / 64;
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
    const uint32_t lane = threadIdx.x & 63;
    for (uint32_t first = from + wave; first < to; first += kWaves * kAhead) {
        u32x4 raw[kAhead];
        if constexpr (!ZERO) {
#pragma unroll
            for (int u = 0; u < kAhead; ++u) {
                const uint32_t i = first + u * kWaves;
                const Stretch t = a.rows.chunks[i < to ? i : from];
                raw[u] = load_piece<DT, true>(t.at + row * t.step, lane, i < to ? t.elems : 0);
            }
        }
#pragma unroll
        for (int u = 0; u < kAhead; ++u) {
            const uint32_t i = first + u * kWaves;
            if (i >= to) continue;
            const Stretch t = a.rows.chunks[i];
            float f[NE];
            if constexpr (!ZERO) V::unpack(raw[u], f);
#pragma unroll
            for (int e = 0; e < NE; ++e) f[e] = ZERO ? 0.0f : scale * exp2_fast(DT == HCCL_DATA_TYPE_FP32 ? exponent(a, f[e], r) : (f[e] - r) * a.c);   // (16 bits do not show c_low)
            store_piece<DT>(t.to + row * t.step, lane, t.elems, f);
        }
    }
}

// What is left of a row, or of its chunks from..to, once r and S are known.  student: the row's logits at the entries if not nullptr.
// gradient(scale): writes scale 2^((l - r) c) everywhere.
template <int DT, int NT, bool LOSS, bool GRAD, typename Gradient>
__device__ __forceinline__ void finish(const DistillArgs &a, DistillShared &s, uint64_t row, uint32_t from, uint32_t to, Sum all, float w,
                                       Entries<NT> &e, Together<NT> &together, const float *student, Gradient &&gradient)
{
    using D = DTypeOf<DT>;
    constexpr uint32_t kEach = Entries<NT>::kEach;
    const Stretch *of[kEach];
    float l[kEach];
    // columns of these chunks
    const uint32_t low = a.rows.chunks[from].first;
    const uint32_t high = a.rows.chunks[to - 1].first + a.rows.chunks[to - 1].elems;
#pragma unroll
    for (uint32_t i = 0; i < kEach; ++i) {
        of[i] = a.rows.ranks;
        l[i] = 0.0f;
        const bool mine = e.at[i] >= low && e.at[i] < high;
        if (mine) {   // (kFree is no column)
            of[i] = rank_of(a.rows, e.at[i]);
            // (all are read before the first gradient is written: it may lie on the logits)
            l[i] = student != nullptr ? student[threadIdx.x + i * NT] : load_one<DT>(of[i]->at + row * of[i]->step, e.at[i] - of[i]->first);
        } else if (LOSS && e.at[i] != kFree) {
            l[i] = student[threadIdx.x + i * NT];
        }
        if (!mine && GRAD && !LOSS) e.at[i] = kFree;   // (after the entries' weights are known)
    }
    const bool empty = all.r == minus_infinity() && all.s == 0.0f;   // every logit is minus infinity: q is 0
    const double r = all.r;
    const double log_s = log(static_cast<double>(all.s));
    if constexpr (LOSS) {
        double sum = 0.0;
#pragma unroll
        for (uint32_t i = 0; i < kEach; ++i) {
            const double log_q = empty ? -__builtin_inf() : (l[i] - r) * a.c64 * kLn2 - log_s;
            if (!(e.p[i] == 0.0)) sum += e.p[i] * (e.t[i] - log_q);
        }
        sum = all_of<NT, false>(sum, s.reduce[2]);
        if (threadIdx.x == 0) {
            if (a.loss != nullptr) a.loss[row] = e.any ? static_cast<float>(w * a.T * a.T * sum) : 0.0f;
            if (a.stats != nullptr) a.stats[row] = {all.r, all.s};
        }
    }
    if constexpr (GRAD) {
        const float scale = e.nan ? __builtin_nanf("") : static_cast<float>(w * a.T);
        if (!LOSS) __syncthreads();   // the entries' logits have been read (or by the loss's sum)
        uint32_t slot[kEach];
#pragma unroll
        for (uint32_t i = 0; i < kEach; ++i) slot[i] = e.any && e.at[i] != kFree ? together.add(e.at[i], e.p[i]) : 0;
        if ((empty && !e.nan) || !e.any) {
            row_gradient<DT, NT, true>(a, row, from, to, 0.0f, 0.0f);
        } else {
            gradient(scale / all.s);
        }
        if (!e.any) return;
        // the entries' gradients replace what the threads of their columns have written: that is in memory by then
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        __syncthreads();
#pragma unroll
        for (uint32_t i = 0; i < kEach; ++i) {
            if (e.at[i] < low || e.at[i] >= high) continue;
            const double p = together.of(slot[i], e.p[i]);
            const double q = empty ? 0.0 : exp2((l[i] - r) * a.c64) / all.s;
            reinterpret_cast<typename D::S *>(of[i]->to + row * of[i]->step)[e.at[i] - of[i]->first] =
                D::narrow(static_cast<float>(scale * (q - p)));
        }
    }
}

// A row that counts nothing.
template <int DT, int NT, bool LOSS, bool GRAD>
__device__ __forceinline__ void nothing(const DistillArgs &a, uint64_t row, uint32_t from, uint32_t to)
{
    if (LOSS && threadIdx.x == 0) {
        if (a.loss != nullptr) a.loss[row] = 0.0f;
        if (a.stats != nullptr) a.stats[row] = {0.0f, 0.0f};
    }
    if (GRAD) row_gradient<DT, NT, true>(a, row, from, to, 0.0f, 0.0f);
}

// A row per workgroup.  Bound by the bytes on their way where there are many rows: 8 ranks, 4096 x 131072 bf16, loss and gradient 482 us, 3.0 GB
// at 6.2 TB/s, of which the gradient's second reading comes from the last-level cache (four workgroups of 512 on a CU; of 256 540 us, of
// 1024 497, with the row kept in registers in between 586); 2048 x 65536 fp16, loss alone, 52 us, 270 MB at
// 5.2 TB/s, a tenth of which are lines of 128 bytes for the entries' logits, out of the caches by then.
template <int DT, bool GRAD, int NT>
__global__ void __launch_bounds__(NT)
k_distill_row(DistillArgs a)
{
    __shared__ DistillShared s;
    const uint64_t row = blockIdx.x;
    const uint32_t n = a.rows.nchunks;
    const float w = a.weight != nullptr ? a.weight[row] : 1.0f;
    if (w == 0.0f) {
        nothing<DT, NT, true, GRAD>(a, row, 0, n);
        return;
    }
    Together<NT> together(a.mask, GRAD);
    Entries<NT> e;
    e.read(a, row);
    const Sum all = row_sum<DT, NT, !GRAD>(a, row, 0, n, s.sums);
    e.normalise(s.reduce);
    finish<DT, NT, true, GRAD>(a, s, row, 0, n, all, w, e, together, nullptr,
                                 [&](float scale) { row_gradient<DT, NT, false>(a, row, 0, n, all.r, scale); });
}

// The same where rows are few and short: a row stays in the threads' registers, N vectors in each, instead of being read twice.  What counts
// there is the chain of one row: with more chunks than a turn of the workgroup it saves a turn's wait, with fewer the code of N vectors costs
// more than that.  16 rows bf16 of 33, 48 and 64 chunks 10.1, 9.8 and 9.9 us, read twice 11.2, 11.7 and 11.2; of 16 and 32 9.4 and 9.7, read
// twice 8.8 and 8.7.  Of up to the two rows that a CU has room for: 512 rows of 33 to 64 chunks 15.6 to 17.1 and 15.0 to 22.5; 600 of 33 21 and
// 18, 4096 of 33, 48 and 64 97, 103 and 113 and 78, 102 and 124.
template <int DT, int N>
__global__ void __launch_bounds__(kThreads)
k_distill_held(DistillArgs a)
{
    constexpr int NT = kThreads;
    using V = Vec16<DT>;
    constexpr int NE = V::NE;
    constexpr uint32_t kWaves = kThreads / 64;
    __shared__ DistillShared s;
    const uint64_t row = blockIdx.x;
    const uint32_t n = a.rows.nchunks;
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
    const uint32_t lane = threadIdx.x & 63;
    const float w = a.weight != nullptr ? a.weight[row] : 1.0f;
    if (w == 0.0f) {
        nothing<DT, kThreads, true, true>(a, row, 0, n);
        return;
    }
    u32x4 raw[N];
#pragma unroll
    for (int u = 0; u < N; ++u) {
        const uint32_t i = wave + u * kWaves;
        const Stretch t = a.rows.chunks[i < n ? i : 0];
        raw[u] = load_piece<DT, true>(t.at + row * t.step, lane, i < n ? t.elems : 0);
    }
    Together<NT> together(a.mask, true);
    Entries<kThreads> e;
    e.read(a, row);
    const Sum all = all_sum<kThreads>(a, lane_sum<DT>(a, {minus_infinity(), 0.0f}, raw), s.sums);
    e.normalise(s.reduce);
    finish<DT, kThreads, true, true>(a, s, row, 0, n, all, w, e, together, nullptr, [&](float scale) {
#pragma unroll
        for (int u = 0; u < N; ++u) {
            const uint32_t i = wave + u * kWaves;
            if (i >= n) break;
            const Stretch t = a.rows.chunks[i];
            float f[NE];
            V::unpack(raw[u], f);
#pragma unroll
            for (int k = 0; k < NE; ++k) f[k] = scale * exp2_fast(DT == HCCL_DATA_TYPE_FP32 ? exponent(a, f[k], all.r) : (f[k] - all.r) * a.c);
            store_piece<DT>(t.to + row * t.step, lane, t.elems, f);
        }
    });
}

// The chunks of a part of a row, of which there are `parts`.
struct Part {
    uint64_t row;
    uint32_t from;
    uint32_t to;
    uint32_t part;
    __device__ __forceinline__ Part(const DistillArgs &a, uint32_t parts)
    {
        row = blockIdx.x / parts;
        part = blockIdx.x % parts;
        from = static_cast<uint32_t>(static_cast<uint64_t>(a.rows.nchunks) * part / parts);
        to = static_cast<uint32_t>(static_cast<uint64_t>(a.rows.nchunks) * (part + 1) / parts);
    }
};

// Several workgroups per row, two launches: r and S of every part, then what is left.  Bound by the chain of one row (16 of
// 131072 bf16 12 us).
template <int DT>
__global__ void __launch_bounds__(kThreads)
k_distill_sums(DistillArgs a)
{
    __shared__ Sum s[kMostWaves];
    const Part p(a, a.nparts);
    if (a.weight != nullptr && a.weight[p.row] == 0.0f) return;
    if (p.part == 0) {   // the student's logits at the entries, before another workgroup writes their gradients there
        for (uint32_t e = threadIdx.x; e < a.k; e += kThreads) {
            const uint32_t c = static_cast<uint32_t>(a.indices[p.row * a.k + e]);
            if (c >= a.rows.vocab) continue;
            const Stretch *of = rank_of(a.rows, c);
            a.student[p.row * a.k + e] = load_one<DT>(of->at + p.row * of->step, c - of->first);
        }
    }
    const Sum all = row_sum<DT, kThreads, false>(a, p.row, p.from, p.to, s);
    if (threadIdx.x == 0) a.parts[p.row * a.nparts + p.part] = {all.r, all.s};
}

// grid: `parts` workgroups per row.  SAVED: r and S are those that the loss saved.
template <int DT, bool SAVED, bool GRAD>
__global__ void __launch_bounds__(kThreads)
k_distill_parts(DistillArgs a, uint32_t parts)
{
    constexpr int NT = kThreads;
    __shared__ DistillShared s;
    const Part p(a, parts);
    const float w = a.weight != nullptr ? a.weight[p.row] : 1.0f;
    Sum all = {0.0f, 0.0f};
    if (w != 0.0f) {
        if constexpr (SAVED) {
            const float2 v = a.stats[p.row];
            all = {v.x, v.y};
        } else {
            const float2 *of = a.parts + p.row * a.nparts;
            all = {of[0].x, of[0].y};
            for (uint32_t i = 1; i < a.nparts; ++i) all = join(a, all, {of[i].x, of[i].y});
        }
    }
    const auto gradient = [&](float scale) { row_gradient<DT, kThreads, false>(a, p.row, p.from, p.to, all.r, scale); };
    const bool none = w == 0.0f || (SAVED && all.r == 0.0f && all.s == 0.0f);   // (a row that counted has S >= 1, is empty or NaN)
    if (!SAVED && p.part == 0) {
        if (none) {
            nothing<DT, kThreads, true, GRAD>(a, p.row, p.from, p.to);
            return;
        }
        Together<NT> together(a.mask, GRAD);
        Entries<kThreads> e;
        e.read(a, p.row);
        e.normalise(s.reduce);
        finish<DT, kThreads, true, GRAD>(a, s, p.row, p.from, p.to, all, w, e, together, a.student + p.row * a.k, gradient);
    } else if constexpr (GRAD) {
        if (none) {
            nothing<DT, kThreads, false, true>(a, p.row, p.from, p.to);
            return;
        }
        Together<NT> together(a.mask, true);
        Entries<kThreads> e;
        e.read(a, p.row);
        e.normalise(s.reduce);
        finish<DT, kThreads, false, true>(a, s, p.row, p.from, p.to, all, w, e, together, SAVED ? nullptr : a.student + p.row * a.k, gradient);
    }
}

// Workgroups that share a row, where `most` are to be had.
uint32_t parts_of(uint32_t rows, uint32_t nchunks, uint32_t most)
{
    const uint32_t fill = rows >= most ? 1 : most / rows;
    // (four chunks for a wavefront: 16 rows of 131072 bf16 12.2 us in eight workgroups each, in four 14.2, in one 29; of 32000 11.7 in three, 11.3 in one)
    return std::max(1u, std::min(fill, nchunks / (kThreads / 64 * kAhead)));
}

struct DistillWork : PlanWork {
    DistillArgs args{};
    Table table;
    DeviceBlock scratch;   // parts, student
    uint32_t parts = 1;
    int dtype = 0;
    bool saved = false;    // the gradient from what the loss saved
    bool grad = false;
    bool held = false;     // rows in registers
    bool short_rows = false;   // small workgroups

    template <int DT>
    void run(hipStream_t st) const
    {
        const uint32_t rows = args.rows.rows;
        const dim3 grid(rows * parts), block(kThreads), small(kSmall);
        const uint32_t table = (args.mask + 1) * 12;
        if (saved) {
            HCCLX_LAUNCH((k_distill_parts<DT, true, true>), grid, block, table, st, args, parts);
        } else if (held) {
            HCCLX_LAUNCH((k_distill_held<DT, kHeld>), grid, block, table, st, args);
        } else if (parts == 1 && short_rows) {
            if (grad) {
                HCCLX_LAUNCH((k_distill_row<DT, true, kSmall>), grid, small, table, st, args);
            } else {
                HCCLX_LAUNCH((k_distill_row<DT, false, kSmall>), grid, small, 0, st, args);
            }
        } else if (parts == 1) {
            if (grad) {
                HCCLX_LAUNCH((k_distill_row<DT, true, kThreads>), grid, block, table, st, args);
            } else {
                HCCLX_LAUNCH((k_distill_row<DT, false, kThreads>), grid, block, 0, st, args);
            }
        } else {
            HCCLX_LAUNCH((k_distill_sums<DT>), grid, block, 0, st, args);
            if (grad) {
                HCCLX_LAUNCH((k_distill_parts<DT, false, true>), grid, block, table, st, args, parts);
            } else {
                HCCLX_LAUNCH((k_distill_parts<DT, false, false>), dim3(rows), block, 0, st, args, 1u);
            }
        }
    }

    int launch(const DeviceCtx *, hipStream_t st) const override
    {
        if (args.rows.rows == 0) return HCCL_SUCCESS;
        if (dtype == HCCL_DATA_TYPE_FP32) {
            run<HCCL_DATA_TYPE_FP32>(st);
        } else if (dtype == HCCL_DATA_TYPE_FP16) {
            run<HCCL_DATA_TYPE_FP16>(st);
        } else {
            run<HCCL_DATA_TYPE_BFP16>(st);
        }
        const hipError_t e = hipGetLastError();
        return e == hipSuccess ? HCCL_SUCCESS : fail_hip(e, "distillation kernels");
    }
};

// What a loss and a gradient have in common.
int prepare(const hcclx_logits_t &l, const hcclx_teacher_t &t, const float *weight, void *const *dlogits, std::unique_ptr<DistillWork> *work)
{
    uint32_t vocab = 0;
    int rc = logits::check(l, dlogits, &vocab);
    if (rc != HCCL_SUCCESS) return rc;
    if (t.k == 0 || t.k > HCCLX_TOP_MAX) return fail(HCCL_E_PARA, "k outside 1.." + std::to_string(HCCLX_TOP_MAX));
    if (t.dtype != HCCL_DATA_TYPE_FP32 && t.dtype != HCCL_DATA_TYPE_FP16 && t.dtype != HCCL_DATA_TYPE_BFP16) {
        return fail(HCCL_E_NOT_SUPPORT, "the teacher's logits are fp32, fp16 or bf16");
    }
    if (!(t.temperature >= 1e-6f && t.temperature <= 1e6f)) return fail(HCCL_E_PARA, "temperature outside 1e-6 .. 1e6");
    const bool none = l.rows == 0;
    if ((rc = check_array(t.logits, dtype_size(t.dtype), none, "teacher")) != HCCL_SUCCESS) return rc;
    if ((rc = check_array(t.indices, 4, none, "indices")) != HCCL_SUCCESS) return rc;
    if ((rc = check_array(weight, 4, true, "weight")) != HCCL_SUCCESS) return rc;
    const uint64_t rows = l.rows;
    if (dlogits != nullptr) {
        if ((rc = check_gradients(l, dlogits)) != HCCL_SUCCESS) return rc;
        if ((rc = check_apart(l, "dlogits", dlogits, "teacher", t.logits, rows * t.k * dtype_size(t.dtype))) != HCCL_SUCCESS) return rc;
        if ((rc = check_apart(l, "dlogits", dlogits, "indices", t.indices, rows * t.k * 4)) != HCCL_SUCCESS) return rc;
        if ((rc = check_apart(l, "dlogits", dlogits, "weight", weight, rows * 4)) != HCCL_SUCCESS) return rc;
    }
    auto w = std::make_unique<DistillWork>();
    w->args.teacher = static_cast<const char *>(t.logits);
    w->args.indices = t.indices;
    w->args.weight = weight;
    w->args.k = t.k;
    w->args.teacher_dtype = t.dtype;
    w->args.T = t.temperature;
    w->args.c64 = 1.4426950408889634074 / t.temperature;
    w->args.c = static_cast<float>(w->args.c64);
    if (w->args.c >= w->args.c64) w->args.c = std::nextafter(w->args.c, 0.0f);
    w->args.c_low = static_cast<float>(w->args.c64 - w->args.c);
    w->args.rows.vocab = vocab;
    w->args.mask = 63;
    while (w->args.mask + 1 < 2 * t.k) w->args.mask = 2 * w->args.mask + 1;   // (at most half are taken)
    w->dtype = l.dtype;
    w->grad = dlogits != nullptr;
    *work = std::move(w);
    return HCCL_SUCCESS;
}

// Bytes of the rows' logits.
uint64_t row_bytes(const hcclx_logits_t &l, uint32_t vocab) { return static_cast<uint64_t>(l.rows) * vocab * dtype_size(l.dtype); }

int make_distill(const hcclx_distill_t &d, hcclx_plan_t **plan)
{
    std::unique_ptr<DistillWork> w;
    int rc = prepare(d.logits, d.teacher, d.weight, d.dlogits, &w);
    if (rc != HCCL_SUCCESS) return rc;
    const hcclx_logits_t &l = d.logits;
    const uint64_t rows = l.rows;
    const uint64_t loss_bytes = rows * sizeof(float), stats_bytes = rows * sizeof(float2);
    if ((rc = check_array(d.loss, 4, true, "loss")) != HCCL_SUCCESS) return rc;
    if ((rc = check_array(d.stats, 8, true, "stats")) != HCCL_SUCCESS) return rc;
    struct {
        const char *what;
        void *p;
        uint64_t bytes;
    } const out[2] = {{"loss", d.loss, loss_bytes}, {"stats", d.stats, stats_bytes}};
    for (const auto &o : out) {
        if ((rc = check_apart(l, "logits", l.logits, o.what, o.p, o.bytes)) != HCCL_SUCCESS) return rc;
        if ((rc = check_apart(l, "dlogits", d.dlogits, o.what, o.p, o.bytes)) != HCCL_SUCCESS) return rc;
        if ((rc = check_apart(o.what, o.p, o.bytes, "teacher", d.teacher.logits, rows * d.teacher.k * dtype_size(d.teacher.dtype))) != HCCL_SUCCESS) return rc;
        if ((rc = check_apart(o.what, o.p, o.bytes, "indices", d.teacher.indices, rows * d.teacher.k * 4)) != HCCL_SUCCESS) return rc;
        if ((rc = check_apart(o.what, o.p, o.bytes, "weight", d.weight, rows * 4)) != HCCL_SUCCESS) return rc;
    }
    if ((rc = check_apart("loss", d.loss, loss_bytes, "stats", d.stats, stats_bytes)) != HCCL_SUCCESS) return rc;
    DeviceCtx *ctx = device_ctx();
    if (!ctx) return HCCL_E_RUNTIME;
    const uint32_t vocab = w->args.rows.vocab;
    if ((rc = lay_out(l, d.dlogits, vocab, &w->table)) != HCCL_SUCCESS) return rc;
    w->args.rows = w->table.rows;
    w->args.loss = d.loss;
    w->args.stats = reinterpret_cast<float2 *>(d.stats);
    uint64_t held = w->table.bytes;
    const uint32_t cus = static_cast<uint32_t>(ctx->num_cus), turn = kThreads / 64 * kAhead;
    w->held = w->grad && l.rows <= 2 * cus && w->args.rows.nchunks > turn && w->args.rows.nchunks <= kThreads / 64 * kHeld;
    // Short rows: smaller workgroups find room for more of them at once.  With a gradient that pays while a row is one turn of theirs (bf16, 16 rows
    // of 16 chunks 8.1 us, by workgroups of 512 8.8; of 24 10.6 and 8.6), or two where rows fill the device (4096 rows of 5000 35 and 53, of
    // 16000 66 and 68, of 24000 99 and 100, of 32000 127 and 116; fp32 of 8000 59 and 63, of 16000 121 and 110).  The loss alone reads a row once:
    // 4096 rows of 16 chunks 25 and 42, of 64 50 and 57, of 128 93 and 94, of 160 114 and 113; 1000 of 128 27 and 29; 300 of 64 10.7 and 10.7, of 128
    // 16.8 and 15.3.
    w->short_rows = w->args.rows.nchunks <= (!w->grad ? 128 : l.rows > 2 * cus ? 32 : 16);
    if (rows != 0 && !w->held) w->parts = parts_of(l.rows, w->args.rows.nchunks, cus);
    if (w->parts > 1) {
        w->args.nparts = w->parts;
        const uint64_t sums = rows * w->parts * sizeof(float2);
        const uint64_t bytes = sums + rows * d.teacher.k * sizeof(float);
        if ((rc = w->scratch.get(bytes)) != HCCL_SUCCESS) return rc;
        w->args.parts = reinterpret_cast<float2 *>(w->scratch.p);
        w->args.student = reinterpret_cast<float *>(w->scratch.p + sums);
        held += bytes;
    }
    const uint64_t algo = row_bytes(l, vocab) * (1 + w->grad);
    return plan_of(ctx, std::move(w), algo, held, plan);
}

int make_distill_grad(const hcclx_distill_grad_t &d, hcclx_plan_t **plan)
{
    std::unique_ptr<DistillWork> w;
    if (d.dlogits == nullptr) return fail(HCCL_E_PTR, "dlogits pointer array is null");
    int rc = prepare(d.logits, d.teacher, d.weight, d.dlogits, &w);
    if (rc != HCCL_SUCCESS) return rc;
    const hcclx_logits_t &l = d.logits;
    if ((rc = check_array(d.stats, 8, l.rows == 0, "stats")) != HCCL_SUCCESS) return rc;
    if ((rc = check_apart(l, "dlogits", d.dlogits, "stats", d.stats, l.rows * sizeof(float2))) != HCCL_SUCCESS) return rc;
    DeviceCtx *ctx = device_ctx();
    if (!ctx) return HCCL_E_RUNTIME;
    const uint32_t vocab = w->args.rows.vocab;
    if ((rc = lay_out(l, d.dlogits, vocab, &w->table)) != HCCL_SUCCESS) return rc;
    w->args.rows = w->table.rows;
    w->args.stats = reinterpret_cast<float2 *>(const_cast<float *>(d.stats));
    w->saved = true;
    // The parts of a row have nothing to wait for: 32 workgroups for a CU, four of which it holds, even out what a last round of them leaves
    // idle (1500 rows of 100003 fp32: 256 us, one for a row 277).
    if (l.rows != 0) w->parts = parts_of(l.rows, w->args.rows.nchunks, 32 * static_cast<uint32_t>(ctx->num_cus));
    const uint64_t held = w->table.bytes;
    return plan_of(ctx, std::move(w), 2 * row_bytes(l, vocab), held, plan);
}

}  // namespace

extern "C" {

int hcclx_distill_plan_create(const hcclx_distill_t *distill, hcclx_plan_t **plan)
{
    if (plan == nullptr) return fail(HCCL_E_PTR, "plan is null");
    *plan = nullptr;
    if (distill == nullptr) return fail(HCCL_E_PTR, "distill is null");
    return guarded([&] { return make_distill(*distill, plan); });
}

int hcclx_distill_grad_plan_create(const hcclx_distill_grad_t *distill, hcclx_plan_t **plan)
{
    if (plan == nullptr) return fail(HCCL_E_PTR, "plan is null");
    *plan = nullptr;
    if (distill == nullptr) return fail(HCCL_E_PTR, "distill is null");
    return guarded([&] { return make_distill_grad(*distill, plan); });
}

}  // extern "C"
