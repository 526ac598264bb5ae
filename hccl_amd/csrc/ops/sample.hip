// The largest logits of a row, and the draw of the next token (include/hcclx_ops.h: hcclx_top_logits_*, hcclx_sample_*).
//
// The first launch reads every logit once and leaves, of every 64 neighbouring columns (a group), the largest, and for runs of a few chunks
// the sum of exp((l - most) / T) where it is wanted.  The second, a workgroup per row, works on what that left:
//
// Of the order of a row's logits (descending, of equal ones the first), the first k lie in those k groups that come first when groups
// are ordered the same way by their largest: an element of any other group has k elements before it.  So the k groups are found among
// the largest values, their elements that reach the k-th group's largest are listed in the order of their columns, and the
// list, little longer than k, is sorted.
//
// The order is that of whole numbers: a float's bits, turned so that they grow with it.  A threshold is found by counting numbers into
// 2048 equal stretches of the range that is left, which leaves one of them, and so on: three rounds at most.
//
// Weights of the draw are whole numbers too, exp((l - most) / T) 2^s from 64-bit arithmetic: their sums do not go by the order.
//
// A row whose draw goes by more than such a list is left to several workgroups.  Next to the second launch they count its elements by
// levels of their weight, 64 to a power of two, which says in which level the cut lies; in a third those over that level are weighed and
// those in it are listed; and a fourth finds the cut among these, and draws.  (One workgroup for all of that: 64 rows of 131072 bf16,
// a sixth of them such, 112 us instead of 36 to 42.)
//
// What bounds it: the first launch, by reading (8 x 4096 x 131072 bf16 197 us, 5.5 TB/s, with a sum that keeps the vector units four fifths
// busy); the others, by how long one row takes: some twenty steps of a workgroup, each with a barrier, and the fetch of their code.  1 row
// of 131072 3 us + 10 us + two launches that find nothing to do.
#include "ops/logits.h"

#include <algorithm>

using namespace hcclx;
using namespace hcclx::logits;

namespace {

constexpr uint32_t kGroup = 64;          // columns
constexpr uint32_t kRunWaves = 4;        // of a workgroup of the first launch, a run each
constexpr uint32_t kList = 2048;         // elements that are sorted at once
constexpr uint32_t kSmallTop = 256;      // the longest list of a small workgroup, and the elements that it sorts
constexpr uint32_t kSmallList = 1024;
constexpr uint32_t kNucleus = 64;        // listed where no top_k bounds the list (192: 1024 draws 194 us instead of 186, 64 42.5 instead of 40)
constexpr uint32_t kLevels = 2048;       // of the weights of a row
constexpr uint32_t kWholeBits = 51;      // of a weight's whole number where there is no filter
constexpr uint32_t kBand = 8192;         // elements of a cut's level, shared out to the parts of a row (each lists kList at most: of the most rows 4096)
constexpr uint32_t kNone = 0;            // the number of what does not exist
constexpr uint32_t kLeast = 0x007fffffu;   // of minus infinity

// What a row's token is drawn by.
struct Choice {
    const float *temperature;
    const int32_t *top_k;
    const float *top_p;
    const float *min_p;
    const float *random;
    int32_t *token;
    float *logprob;
};

struct Run {
    double sum;
    float most;
    uint32_t unused;
};

// A row that is left to the launches behind the second.
struct Wide {
    uint32_t wide;     // 0: it is not; 2: it is, but its cut is not found by levels, or it has none
    uint32_t top;      // its largest number
    unsigned long long p_low;    // between which what top_p asks for lies
    unsigned long long p_high;
};

// What a part of such a row holds nearer than the band, and how many in it.
struct Found {
    unsigned long long weight;
    uint32_t over;
    uint32_t listed;
};

// Distances of the elements that the cut lies among: low .. high - 1.  Those nearer all stay, those further don't.
struct Band {
    float low;
    float high;
    bool by_level;   // by top_k or top_p
    bool by_min;
    bool known;      // false: the cut is not found by levels
};

struct SelectArgs {
    Rows rows;
    uint32_t *most;     // [rows][nchunks * groups of a chunk]: the numbers of the groups' largest
    Run *runs;          // [rows][nruns]
    uint32_t nruns;
    uint32_t per_run;   // chunks
    uint32_t bits;      // s
    // rows that are left to the launches behind the second, of the `batch` rows from `first` on
    struct Wide *wide;  // [batch]
    unsigned long long *levels;   // [batch][kLevels]
    struct Band *bands;           // [batch]
    struct Found *found;          // [batch][wide_parts]
    unsigned long long *listed;   // [batch][wide_parts][band_each]: the elements that the cut lies among
    unsigned long long *spans;    // [batch][kMostSpans]: weights over them
    uint32_t span;      // chunks that are weighed together
    uint32_t nspans;
    uint32_t wide_parts;   // workgroups of a row
    uint32_t band_each;    // elements that a part may list
    uint32_t first;
    // the largest
    uint32_t k;
    char *values;
    int32_t *indices;
    float *lse;
    Choice choice;
};

__device__ __forceinline__ uint32_t number_of(float v)
{
    const uint32_t u = __float_as_uint(v + 0.0f);   // (-0 is 0)
    return u ^ (static_cast<uint32_t>(static_cast<int32_t>(u) >> 31) | 0x80000000u);
}
__device__ __forceinline__ float value_of(uint32_t n) { return __uint_as_float(n ^ ((n >> 31) != 0 ? 0x80000000u : 0xffffffffu)); }
// NaN counts as minus infinity.
__device__ __forceinline__ float no_nan(float v) { return fmaxf(v, minus_infinity()); }

// Bits of a number that are the same for all values of a type and sign.
template <int DT> constexpr uint32_t kIdle = DT == HCCL_DATA_TYPE_BFP16 ? 16 : DT == HCCL_DATA_TYPE_FP16 ? 13 : 0;

template <int CTRL>
__device__ __forceinline__ float dpp(float v) { return dpp_or<CTRL>(v, v); }

__device__ __forceinline__ uint32_t wave_most(uint32_t v)
{
    v = max(v, dpp_or_zero<0x111, 0xf>(v));
    v = max(v, dpp_or_zero<0x112, 0xf>(v));
    v = max(v, dpp_or_zero<0x114, 0xf>(v));
    v = max(v, dpp_or_zero<0x118, 0xf>(v));
    v = max(v, dpp_or_zero<0x142, 0xa>(v));
    return of_last_lane(max(v, dpp_or_zero<0x143, 0xc>(v)));
}

// 2^(up - y / 64) for y >= 0: y = n + f with |f| <= 1/2, a power out of the table (64 of them) and five terms of the power series, the
// first omitted of which is below 2^-54.  What is below 2^-53, or no number, is 0.  (No branch: several of them run side by side.)
__device__ __forceinline__ double power(const double *powers, double y, int up)
{
    constexpr double kEnd = 53.0 * 64.0;
    const double in = __builtin_fmin(y, kEnd);   // (of NaN kEnd)
    const double n = rint(in);
    const double z = (in - n) * (-0.69314718055994530942 / 64);
    double p = 1.0 / 120;
    p = __builtin_fma(p, z, 1.0 / 24);
    p = __builtin_fma(p, z, 1.0 / 6);
    p = __builtin_fma(p, z, 0.5);
    p = __builtin_fma(p, z, 1.0);
    p = __builtin_fma(p, z, 1.0);
    const int whole = static_cast<int>(n);
    // (the product is a normal number between 2^-1 and 2^1: its exponent is added to)
    const double q = p * powers[whole & 63];
    const u64 r = __builtin_bit_cast(u64, q) + (static_cast<u64>(static_cast<uint32_t>(up - (whole >> 6)) << 20) << 32);
    return in < kEnd ? __builtin_bit_cast(double, r) : 0.0;
}

struct RowChoice {
    bool greedy;
    bool by_k;
    bool by_p;
    bool by_min;
    uint32_t k;
    float p;        // where top_p is below 1
    double least;
    double c;   // log2(e) / T

    __device__ __forceinline__ RowChoice(const Choice &a, uint64_t row, uint32_t vocab)
    {
        const float T = a.temperature != nullptr ? a.temperature[row] : 1.0f;
        const int32_t top = a.top_k != nullptr ? a.top_k[row] : 0;
        const float tp = a.top_p != nullptr ? a.top_p[row] : 1.0f;
        const float mp = a.min_p != nullptr ? a.min_p[row] : 0.0f;
        greedy = !(T > 0.0f);
        by_k = greedy || (top > 0 && static_cast<uint32_t>(top) < vocab);
        k = greedy ? 1 : static_cast<uint32_t>(top);
        by_p = !greedy && tp < 1.0f;
        by_min = !greedy && mp > 0.0f;
        p = tp;
        least = mp < 1.0f ? mp : 1.0f;
        c = greedy ? 1.0 : 1.4426950408889634074 / static_cast<double>(T);
    }
    // whether elements are counted by levels, in case that no list holds what stays
    __device__ __forceinline__ bool by_levels() const { return by_k ? k > HCCLX_TOP_MAX && !by_p : by_p; }
    __device__ __forceinline__ bool none() const { return !by_k && !by_p && !by_min; }
    // whether the sum over the whole row is needed
    __device__ __forceinline__ bool whole() const { return !by_k && (by_p || !by_min); }
};

// The first launch: U chunks per wavefront.  SUM: exp(l - most) in 32 bits; CHOICE: by the row's temperature in 64, where it is needed.
enum RunKind { kRunPlain, kRunSum, kRunChoice };
template <int DT, int U, int KIND>
__global__ void __launch_bounds__(kRunWaves * 64)
k_logit_runs(SelectArgs a, uint32_t parts)
{
    using V = Vec16<DT>;
    constexpr int NE = V::NE;
    constexpr uint32_t kPer = kChunk<DT> / kGroup;   // groups of a chunk
    const uint64_t row = a.first + blockIdx.x / parts;
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
    const uint32_t run = blockIdx.x % parts * kRunWaves + wave;
    const uint32_t lane = threadIdx.x & 63;
    const uint32_t from = run * U;
    __shared__ double s_powers[64];
    if constexpr (KIND == kRunChoice) {
        if (threadIdx.x < 64) s_powers[threadIdx.x] = exp2_exact(threadIdx.x / -64.0);
        __syncthreads();
        if (a.wide_parts != 0 && RowChoice(a.choice, row, a.rows.vocab).by_levels()) {   // (the second launch counts)
            const uint32_t part = blockIdx.x % parts;
            u64 *const levels = a.levels + static_cast<uint64_t>(blockIdx.x / parts) * kLevels;
            for (uint32_t i = kLevels * part / parts + threadIdx.x; i < kLevels * (part + 1) / parts; i += kRunWaves * 64) levels[i] = 0;
        }
    }
    if (from >= a.rows.nchunks) return;
    u32x4 raw[U];
    uint32_t elems[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const uint32_t i = from + u;
        const Stretch t = a.rows.chunks[i < a.rows.nchunks ? i : from];
        elems[u] = i < a.rows.nchunks ? t.elems : 0;
        raw[u] = load_piece<DT, false>(t.at + row * t.step, lane, elems[u]);
    }
    float most = minus_infinity();
    uint32_t *to = a.most + row * a.rows.nchunks * kPer + from * kPer;
#pragma unroll
    for (int u = 0; u < U; ++u) {
        float f[NE];
        V::unpack(raw[u], f);
        float m = minus_infinity();
#pragma unroll
        for (int e = 0; e < NE; ++e) m = fmaxf(m, f[e]);
        // over the 8 or 16 lanes of a group
        m = fmaxf(m, dpp<0xb1>(m));    // lane ^ 1
        m = fmaxf(m, dpp<0x4e>(m));    // lane ^ 2
        m = fmaxf(m, dpp<0x141>(m));   // 7 - lane of each 8
        if (NE == 4) m = fmaxf(m, dpp<0x140>(m));   // 15 - lane of each 16
        constexpr uint32_t kLanes = kGroup / NE;
        if (lane % kLanes == 0 && from + u < a.rows.nchunks) to[u * kPer + lane / kLanes] = lane * NE < elems[u] ? number_of(m) : kNone;
        most = fmaxf(most, m);
    }
    if constexpr (KIND != kRunPlain) {
        const RowChoice choice(a.choice, row, a.rows.vocab);
        if (KIND == kRunChoice && !choice.whole()) return;
#pragma unroll
        for (int d = 8; d < 64; d <<= 1) most = fmaxf(most, __shfl_xor(most, d, 64));
        double sum = 0.0;
        if constexpr (KIND == kRunSum) {
            // (bounded: minus infinity and NaN become a term of 0, and infinity has a distance of 0 from itself)
            constexpr float kBound = 0x1.fffffep+125f;
            const float c = 1.44269504f;
            const float most_bounded = fminf(fmaxf(most, -kBound), kBound);
            float s = 0.0f;
            if (__builtin_fabsf(most_bounded) < 0x1p20f) {
                const float ref = most_bounded * c;
#pragma unroll
                for (int u = 0; u < U; ++u) {
                    float f[NE];
                    V::unpack(raw[u], f);
#pragma unroll
                    for (int e = 0; e < NE; ++e) s += exp2_fast(__builtin_fmaf(fminf(fmaxf(f[e], -kBound), kBound), c, -ref));
                }
                s *= exp2_fast(-__builtin_fmaf(most_bounded, c, -ref));   // (what rounding the reference did to all terms)
            } else {   // where that is more than a part of a power of two: the difference first, one operation more
#pragma unroll
                for (int u = 0; u < U; ++u) {
                    float f[NE];
                    V::unpack(raw[u], f);
#pragma unroll
                    for (int e = 0; e < NE; ++e) s += exp2_fast((fminf(fmaxf(f[e], -kBound), kBound) - most_bounded) * c);
                }
            }
            sum = most == minus_infinity() ? 0.0 : static_cast<double>(wave_sum(s));
        } else if (most != minus_infinity()) {
            const double step = 64.0 * choice.c;
#pragma unroll
            for (int u = 0; u < U; ++u) {
                float f[NE];
                V::unpack(raw[u], f);
#pragma unroll
                for (int e = 0; e < NE; ++e) {
                    const float l = no_nan(f[e]);
                    const double w = power(s_powers, (static_cast<double>(most) - l) * step, 0);
                    sum += l == most ? 1.0 : w;
                }
            }
            sum = wave_total(sum);
        }
        if (lane == 0) a.runs[row * a.nruns + run] = {sum, most, 0};
    }
}

// ---- the second launch ---------------------------------------------------------------------------------------------------

// What a list holds of an element, so that larger ones come first in its order: number, ~place.  A place counts kChunk for each chunk in
// front of the element's; places are in the order of the columns.
template <int DT>
__device__ __forceinline__ uint32_t column_of(const SelectArgs &a, u64 x)
{
    const uint32_t place = ~static_cast<uint32_t>(x);
    return a.rows.chunks[place / kChunk<DT>].first + place % kChunk<DT>;
}

struct Range {
    uint32_t low;      // numbers (without their idle bits) that are left, both included
    uint32_t high;
    uint32_t above;    // how many are over them
    uint32_t inside;   // and in them
    u64 weight_above;
    u64 weight_inside;
};

constexpr uint32_t kBatch = 4096;        // rows that are drawn from together: 36 to 84 KB for the wide draw of each, 150 KB where they are few
constexpr uint32_t kMostParts = 32;      // workgroups of a wide row
constexpr uint32_t kMostSpans = 512;
constexpr uint32_t kCounted = 256;       // elements of a list that is put in order by counting
constexpr uint32_t kMostWaves = 8;
constexpr uint32_t kCached = 320;        // chunks whose places in the row are kept in LDS
constexpr uint32_t kNoEnd = 0xffffffffu;
constexpr uint32_t kNotSure = 1 << 16;   // counts for more elements than a list has
constexpr uint32_t kStretches = 1000;    // of the range of a list's numbers
constexpr uint32_t kMostAlike = 32;      // elements of a stretch that are put in order by counting
constexpr uint32_t kQueue = 512;         // elements of a chunk that a wavefront weighs

// What is used at different times lies in the same place.
template <uint32_t LIST, uint32_t GROUPS>
struct SharedOf {
    static constexpr uint32_t kList = LIST;        // elements of a list
    static constexpr uint32_t kBins = LIST;        // stretches that are counted into
    static constexpr uint32_t kMostGroups = GROUPS;
    union {
        struct {
            u64 weight[kBins];
            uint32_t count[kBins];
        } bins;
        struct {
            u64 listed[kList];   // in the order of the columns
            u64 sorted[kList];
        } list;
        struct {
            u64 weight[512];   // of the chunks of a row
            uint32_t equal[512];
        } walk;
        struct {
            u64 listed[kList];   // (where list.listed is)
            float queue[LIST < 2048 ? 1 : kMostWaves][kQueue];
        } wide;
        struct {
            uint32_t unused[LIST * 4 - GROUPS];
            uint32_t groups[GROUPS];   // behind the bins and what counting uses of `sorted`; before anything is sorted by exchanges
        };
    };
    union {
        struct {
            uint64_t at[kCached];     // of the row's chunks
            uint32_t elems[kCached];
        };
        u64 span_weight[kMostSpans];
        uint32_t stretch[kStretches + 1];   // begins in a list that is sorted
    };
    double powers[64];   // 2^(-i / 64)
    u64 part[2][kMostWaves];
    uint32_t most[kMostWaves];
    uint32_t least[kMostWaves];
    uint32_t place[kMostWaves];
    Range range;
    u64 word64[2];
    uint32_t word[4];
    u64 one;
};
constexpr uint32_t groups_for(uint32_t k) { return k + k / 2 + 32; }
using Shared = SharedOf<kList, groups_for(HCCLX_TOP_MAX)>;            // 38 KB: four workgroups on a CU
using SmallShared = SharedOf<kSmallList, groups_for(kSmallTop)>;      // 22 KB: seven
template <typename S> constexpr bool kApart = S::kList * 16 - S::kMostGroups * 4 >= S::kBins * 12 && S::kList * 16 - S::kMostGroups * 4 >= S::kList * 8 + 3 * kCounted * 8;
static_assert(kApart<Shared> && kApart<SmallShared> && sizeof(Shared) <= 160 * 1024 / 4 && sizeof(SmallShared) <= 160 * 1024 / 7, "");

// A lane's vector of a group: lanes kGroup / NE in a row hold one.
struct Piece {
    u32x4 raw;
    uint32_t place;
    uint32_t have;    // elements that exist
};

// What the threads of a workgroup do together about a row.
template <int NT, typename S = Shared>
struct Team {
    static constexpr uint32_t kWaves = NT / 64;
    static_assert(kWaves <= kMostWaves, "");

    const SelectArgs &a;
    S &s;
    const uint64_t row;
    uint32_t top;      // the largest number of the row
    double top_value;
    double c;          // log2(e) / T, where weights are asked for
    uint32_t flip;     // which partial sums are free

    __device__ __forceinline__ Team(const SelectArgs &args, S &shared, uint64_t of, uint32_t largest, double scale)
        : a(args), s(shared), row(of), top(largest), top_value(value_of(largest)), c(scale), flip(0)
    {
        if (threadIdx.x < 64) s.powers[threadIdx.x] = exp2_exact(threadIdx.x / -64.0);
    }

    // Sums over the threads before this one, and over all.  One barrier: partial sums alternate between two places, and who is here for the
    // third time has seen everybody leave the first.
    template <typename T>
    __device__ __forceinline__ T before(T v, T *all)
    {
        T *part = reinterpret_cast<T *>(s.part[flip]);
        flip ^= 1;
        const uint32_t wave = threadIdx.x / 64;
        const T sum = wave_sums(v);
        if ((threadIdx.x & 63) == 63) part[wave] = sum;
        __syncthreads();
        T from = 0, whole = 0;
#pragma unroll
        for (uint32_t w = 0; w < kWaves; ++w) {
            from += w < wave ? part[w] : T(0);
            whole += part[w];
        }
        *all = whole;
        return from + sum - v;
    }
    template <typename T>
    __device__ __forceinline__ T total(T v)
    {
        T all;
        (void)before(v, &all);
        return all;
    }

    // exp((l - most) / T) times 2^up
    __device__ __forceinline__ double share(float l, int up) const
    {
        const double far = power(s.powers, (top_value - l) * (64.0 * c), up);
        return static_cast<double>(l) == top_value ? ldexp(1.0, up) : far;   // (of infinities too)
    }
    __device__ __forceinline__ double share(uint32_t number) const { return share(value_of(number), 0); }
    // The same times 2^bits as a whole number: 2^52 added, the last place of a double is 1.
    __device__ __forceinline__ u64 weight(float l, uint32_t bits) const
    {
        return static_cast<u64>(__double_as_longlong(share(l, static_cast<int>(bits)) + 0x1p52)) & ((u64(1) << 52) - 1);
    }
    __device__ __forceinline__ u64 weight(float l) const { return weight(l, a.bits); }
    __device__ __forceinline__ u64 weight(uint32_t number) const { return weight(value_of(number)); }

    // Sorts s.list.listed[0 .. n) into s.list.sorted, descending: into equal stretches of the range of their numbers, and in those by counting
    // (301 rows of 32003, lists of 700: 31 us with the first launch, 44 by exchanges alone).  Where many are alike, by exchanges.
    __device__ __forceinline__ void sort(uint32_t n)
    {
        constexpr uint32_t kMine = S::kList / NT;
        u64 key[kMine];
        uint32_t least = kNoEnd;
#pragma unroll
        for (uint32_t i = 0; i < kMine; ++i) {
            const uint32_t at = threadIdx.x + i * NT;
            key[i] = at < n ? s.list.listed[at] : 0;
            if (at < n) least = min(least, static_cast<uint32_t>(key[i] >> 32));
        }
        least = ~wave_most(~least);
        if ((threadIdx.x & 63) == 0) s.least[threadIdx.x / 64] = least;
        for (uint32_t i = threadIdx.x; i <= kStretches; i += NT) s.stretch[i] = 0;
        if (threadIdx.x == 0) s.word[3] = 0;
        __syncthreads();
        least = s.least[0];
#pragma unroll
        for (uint32_t w = 1; w < kWaves; ++w) least = min(least, s.least[w]);
        // (the largest number of the list is the row's)
        const uint32_t each = (top - least) / kStretches + 1;
        uint32_t bin[kMine], place[kMine];
#pragma unroll
        for (uint32_t i = 0; i < kMine; ++i) {
            bin[i] = place[i] = 0;
            if (threadIdx.x + i * NT >= n) continue;
            bin[i] = (top - static_cast<uint32_t>(key[i] >> 32)) / each;
            place[i] = atomicAdd(&s.stretch[bin[i]], 1u);
            if (place[i] == kMostAlike) s.word[3] = 1;
        }
        __syncthreads();
        if (s.word[3] != 0) {
            exchange(n);
            return;
        }
        constexpr uint32_t kBegins = (kStretches + NT) / NT;   // neighbours of a thread
        uint32_t count[kBegins], sum = 0, all;
#pragma unroll
        for (uint32_t i = 0; i < kBegins; ++i) {
            const uint32_t b = threadIdx.x * kBegins + i;
            sum += count[i] = b <= kStretches ? s.stretch[b] : 0;
        }
        sum = before(sum, &all);
#pragma unroll
        for (uint32_t i = 0; i < kBegins; ++i) {
            const uint32_t b = threadIdx.x * kBegins + i;
            if (b <= kStretches) s.stretch[b] = sum;
            sum += count[i];
        }
        __syncthreads();
#pragma unroll
        for (uint32_t i = 0; i < kMine; ++i) {
            if (threadIdx.x + i * NT < n) s.list.sorted[s.stretch[bin[i]] + place[i]] = key[i];
        }
        __syncthreads();
#pragma unroll
        for (uint32_t i = 0; i < kMine; ++i) {
            if (threadIdx.x + i * NT >= n) continue;
            const uint32_t from = s.stretch[bin[i]], to = s.stretch[bin[i] + 1];
            place[i] = from;
            for (uint32_t k = from; k < to; ++k) place[i] += s.list.sorted[k] > key[i];
        }
        __syncthreads();
#pragma unroll
        for (uint32_t i = 0; i < kMine; ++i) {
            if (threadIdx.x + i * NT < n) s.list.sorted[place[i]] = key[i];
        }
        __syncthreads();
    }
    __device__ __forceinline__ void exchange(uint32_t n) const
    {
        uint32_t size = 64;
        while (size < n) size *= 2;
        const uint32_t t = threadIdx.x;
        if (size <= NT) {   // an element per thread; a wavefront's own steps need no barrier
            u64 x = t < n ? s.list.listed[t] : 0;
            for (uint32_t width = 2; width <= size; width *= 2) {
                for (uint32_t step = width / 2; step >= 1; step /= 2) {
                    u64 y;
                    if (step >= 64) {
                        s.list.sorted[t] = x;
                        __syncthreads();
                        y = s.list.sorted[t ^ step];
                        __syncthreads();
                    } else {
                        y = __shfl_xor(x, static_cast<int>(step), 64);
                    }
                    const bool larger = ((t & step) == 0) == ((t & width) == 0);
                    x = (x > y) == larger ? x : y;
                }
            }
            s.list.sorted[t] = x;
            __syncthreads();
            return;
        }
        for (uint32_t i = t; i < size; i += NT) s.list.sorted[i] = i < n ? s.list.listed[i] : 0;
        __syncthreads();
        for (uint32_t width = 2; width <= size; width *= 2) {
            for (uint32_t step = width / 2; step >= 1; step /= 2) {
                for (uint32_t k = t; k < size / 2; k += NT) {
                    const uint32_t i = (k & ~(step - 1)) * 2 + (k & (step - 1));
                    const u64 x = s.list.sorted[i], y = s.list.sorted[i + step];
                    const bool down = (i & width) == 0;
                    if ((x < y) == down) {
                        s.list.sorted[i] = y;
                        s.list.sorted[i + step] = x;
                    }
                }
                __syncthreads();
            }
        }
    }

    // A short list (n <= kCounted), thread t < n: how many elements come before s.list.listed[t], and their weight, given the element's own.
    // The threads share out the comparisons, whose sums meet in LDS.  (WEIGH false: the number alone.)
    template <bool WEIGH>
    __device__ __forceinline__ uint32_t count_before(uint32_t n, u64 own, u64 *weight_before)
    {
        static_assert(3 * kCounted <= S::kList && kCounted <= S::kMostGroups && kCounted <= NT, "");
        u64 *const weights = s.list.sorted, *const sums = s.list.sorted + kCounted;
        uint32_t *const ranks = s.groups;
        if (threadIdx.x < kCounted) {
            if (WEIGH) {
                weights[threadIdx.x] = threadIdx.x < n ? own : 0;
                sums[threadIdx.x] = 0;
            }
            ranks[threadIdx.x] = 0;
            if (threadIdx.x >= n && threadIdx.x < ((n + 7) & ~7u)) s.list.listed[threadIdx.x] = 0;   // (comes before nothing)
        }
        __syncthreads();
        uint32_t each = 64;   // threads of a share: all elements
        while (each < n) each *= 2;
        const uint32_t i = threadIdx.x & (each - 1);
        const uint32_t shares = NT / each;
        const uint32_t eights = (n + 7) / 8;
        if (i < n) {
            const u64 x = s.list.listed[i];
            uint32_t rank = 0;
            u64 sum = 0;
            for (uint32_t k = threadIdx.x / each; k < eights; k += shares) {
#pragma unroll
                for (uint32_t j = 0; j < 8; ++j) {
                    const bool first = s.list.listed[k * 8 + j] > x;
                    rank += first;
                    if (WEIGH) sum += first ? weights[k * 8 + j] : 0;
                }
            }
            atomicAdd(&ranks[i], rank);
            if (WEIGH) atomicAdd(&sums[i], sum);
        }
        __syncthreads();
        if (WEIGH) *weight_before = threadIdx.x < kCounted ? sums[threadIdx.x] : 0;
        return threadIdx.x < kCounted ? ranks[threadIdx.x] : 0;
    }

    // whole: the sum of what could have been drawn, of exp((l - most) / T).
    __device__ __forceinline__ void write_choice(uint32_t column, uint32_t number, double whole) const
    {
        a.choice.token[row] = static_cast<int32_t>(column);
        if (a.choice.logprob != nullptr) {
            const double x = number == top ? 0.0 : (static_cast<double>(value_of(number)) - top_value) * c * 0.69314718055994530942;
            a.choice.logprob[row] = static_cast<float>(x - log(whole));
        }
    }
    __device__ __forceinline__ double run_sum(uint32_t i) const   // of a run, of exp((l - most) / T)
    {
        const Run run = a.runs[row * a.nruns + i];
        return run.sum * share(run.most, 0);
    }
};

template <int DT, int NT, typename S = Shared>
struct Row : Team<NT, S> {
    using V = Vec16<DT>;
    using B = Team<NT, S>;
    using B::a;
    using B::s;
    using B::row;
    using B::top;
    using B::top_value;
    using B::before;
    using B::total;
    using B::weight;
    using B::kWaves;
    static constexpr uint32_t NE = V::NE;
    static constexpr uint32_t kPer = kChunk<DT> / kGroup;
    static constexpr uint32_t kLanes = kGroup / NE;
    static constexpr uint32_t kTurn = NT / kLanes;   // groups of a turn
    static constexpr uint32_t kShift = kIdle<DT>;
    static constexpr uint32_t kHeld = 4096 / NT;     // groups of a thread whose largest it holds, where all find room
    static_assert(kHeld % 4 == 0, "");

    const uint32_t *most;
    const uint32_t ngroups;
    uint32_t held[kHeld];
    uint32_t bottom;   // the least of the groups' largest

    __device__ __forceinline__ Row(const SelectArgs &args, S &shared, uint64_t of)
        : Team<NT, S>(args, shared, of, 0, 0.0), most(args.most + of * args.rows.nchunks * kPer), ngroups(args.rows.nchunks * kPer)
    {
        uint32_t t = 0, least = kNoEnd;
        // (rows of the largest are whole vectors: a chunk has four or eight groups)
#pragma unroll
        for (uint32_t i = 0; i < kHeld; i += 4) {
            const uint32_t at = threadIdx.x * kHeld + i;
            const u32x4 v = at < ngroups ? *reinterpret_cast<const u32x4 *>(most + at) : u32x4{kNone, kNone, kNone, kNone};
#pragma unroll
            for (uint32_t j = 0; j < 4; ++j) {
                held[i + j] = v[j];
                t = max(t, v[j]);
                least = min(least, v[j] != kNone ? v[j] : kNoEnd);
            }
        }
        find_chunks();
        for (uint32_t i = NT * kHeld + threadIdx.x; i < ngroups; i += NT) {
            t = max(t, most[i]);
            least = min(least, most[i] != kNone ? most[i] : kNoEnd);
        }
        t = wave_most(t);
        least = ~wave_most(~least);
        if ((threadIdx.x & 63) == 0) {
            s.most[threadIdx.x / 64] = t;
            s.least[threadIdx.x / 64] = least;
        }
        __syncthreads();
        t = s.most[0];
        least = s.least[0];
#pragma unroll
        for (uint32_t w = 1; w < kWaves; ++w) {
            t = max(t, s.most[w]);
            least = min(least, s.least[w]);
        }
        top = t;
        bottom = least;
        top_value = value_of(top);
    }

    // f(group, its largest) of neighbouring groups per thread, in their order
    template <typename F>
    __device__ __forceinline__ void each_group(F &&f) const
    {
        if (ngroups <= NT * kHeld) {
#pragma unroll
            for (uint32_t i = 0; i < kHeld; ++i) f(threadIdx.x * kHeld + i, held[i]);   // (kNone behind the last)
        } else {
            const uint32_t each = (ngroups + NT - 1) / NT;
            const uint32_t from = min(threadIdx.x * each, ngroups), to = min(from + each, ngroups);
            for (uint32_t i = from; i < to; ++i) f(i, most[i]);
        }
    }

    __device__ __forceinline__ void find_chunks()
    {
        if (a.rows.nchunks > kCached) return;
        for (uint32_t i = threadIdx.x; i < a.rows.nchunks; i += NT) {
            const Stretch of = a.rows.chunks[i];
            s.at[i] = reinterpret_cast<uint64_t>(of.at + row * of.step);
            s.elems[i] = of.elems;
        }
    }
    // Where the row's part of a chunk lies, and how much it has.
    __device__ __forceinline__ const char *chunk_at(uint32_t chunk, uint32_t *elems) const
    {
        if (a.rows.nchunks <= kCached) {
            *elems = s.elems[chunk];
            return reinterpret_cast<const char *>(s.at[chunk]);
        }
        const Stretch t = a.rows.chunks[chunk];
        *elems = t.elems;
        return t.at + row * t.step;
    }
    __device__ __forceinline__ Piece piece(uint32_t group, bool there) const
    {
        const uint32_t chunk = there ? group / kPer : 0;
        uint32_t elems;
        const char *at = chunk_at(chunk, &elems);
        const uint32_t lane = group % kPer * kLanes + threadIdx.x % kLanes;   // of the chunk
        const uint32_t first = lane * NE;
        Piece p;
        p.have = !there || first >= elems ? 0 : elems - first < NE ? elems - first : NE;
        p.place = chunk * kChunk<DT> + first;
        p.raw = load_piece<DT, false>(at, lane, there ? elems : 0);
        return p;
    }

    // f(piece, values) of the vectors of n groups: those of the list, or (nullptr) all
    template <typename F>
    __device__ __forceinline__ void each_piece(const uint32_t *list, uint32_t n, F &&f) const
    {
        constexpr int kAhead = 4;
        for (uint32_t g = threadIdx.x / kLanes; g < n; g += kTurn * kAhead) {
            Piece p[kAhead];
#pragma unroll
            for (int u = 0; u < kAhead; ++u) {
                const uint32_t i = g + u * kTurn;
                p[u] = piece(i < n ? (list != nullptr ? list[i] : i) : 0, i < n);
            }
#pragma unroll
            for (int u = 0; u < kAhead; ++u) {
                float v[NE];
                V::unpack(p[u].raw, v);
                f(p[u], v);
            }
        }
    }
    // f(number without idle bits, weight) of their elements
    template <typename F>
    __device__ __forceinline__ void each(const uint32_t *list, uint32_t n, F &&f) const
    {
        each_piece(list, n, [&](const Piece &p, const float (&v)[NE]) {
#pragma unroll
            for (uint32_t e = 0; e < NE; ++e) {
                if (e >= p.have) continue;
                const uint32_t number = number_of(no_nan(v[e]));
                f(number >> kShift, [&] { return weight(number); });
            }
        });
    }

    // One round of the search: the numbers in the range are counted (and weighed) into S::kBins stretches of it; the range becomes the one in
    // which the running count (BY_WEIGHT: weight) from the top reaches what target() says, given the weight in the range.
    // all(f): f(number, weight) for every number that there is.
    template <bool BY_WEIGHT, typename All, typename Target>
    __device__ __forceinline__ void narrow(Range &r, All &&all, Target &&target)
    {
        const uint32_t width = r.high - r.low;
        constexpr uint32_t kBits = S::kBins == 2048 ? 11 : 10;
        static_assert(S::kBins == 1u << kBits, "");
        const uint32_t shift = width < S::kBins ? 0 : 32 - __clz(width) - kBits;
        for (uint32_t i = threadIdx.x; i < S::kBins; i += NT) {
            s.bins.count[i] = 0;
            if (BY_WEIGHT) s.bins.weight[i] = 0;
        }
        __syncthreads();
        all([&](uint32_t n, auto &&weight) {
            if (n < r.low || n > r.high) return;
            const uint32_t bin = (n - r.low) >> shift;
            atomicAdd(&s.bins.count[bin], 1u);
            if constexpr (BY_WEIGHT) {
                const u64 w = weight();
                if (w != 0) atomicAdd(&s.bins.weight[bin], w);
            }
        });
        __syncthreads();
        // from the top: neighbours per thread
        constexpr uint32_t kMine = S::kBins / NT;
        uint32_t count[kMine];
        u64 weight[kMine];
        uint32_t counts = 0;
        u64 weights = 0;
#pragma unroll
        for (uint32_t i = 0; i < kMine; ++i) {
            const uint32_t bin = S::kBins - 1 - (threadIdx.x * kMine + i);
            counts += count[i] = s.bins.count[bin];
            weights += weight[i] = BY_WEIGHT ? s.bins.weight[bin] : 0;
        }
        uint32_t all_count;
        u64 whole = 0;
        uint32_t c = before(counts, &all_count);
        u64 w = BY_WEIGHT ? before(weights, &whole) : 0;
        const u64 there = BY_WEIGHT ? r.weight_above + whole : r.above + all_count;
        const u64 asked = target(whole);
        const u64 aim = asked < there ? asked : there;   // (all of it, where there is less)
        c += r.above;
        w += r.weight_above;
#pragma unroll
        for (uint32_t i = 0; i < kMine; ++i) {
            const u64 at = BY_WEIGHT ? w : c;
            const u64 add = BY_WEIGHT ? weight[i] : count[i];
            if (at < aim && at + add >= aim) {
                const uint32_t bin = S::kBins - 1 - (threadIdx.x * kMine + i);
                const uint32_t low = r.low + (bin << shift);
                const uint32_t last = low + ((1u << shift) - 1);
                s.range = {low, last < r.high ? last : r.high, c, count[i], w, weight[i]};
            }
            c += count[i];
            w += weight[i];
        }
        __syncthreads();
        r = s.range;
    }

    __device__ __forceinline__ void put(uint32_t at, float l, uint32_t place) const
    {
        if (at < S::kList) s.list.listed[at] = static_cast<u64>(number_of(l)) << 32 | static_cast<uint32_t>(~place);
    }
    // Lists the elements of the groups s.groups[0 .. n) that reach `low`, in the order of the columns; returns how many there are, or a
    // number over S::kList as soon as they are known to be more.
    __device__ __forceinline__ uint32_t list(uint32_t n, uint32_t low)
    {
        constexpr int kAhead = 2;   // turns that are read and counted together, 16 bits of a sum for each
        static_assert(NT * NE < 1 << 16, "");
        // (the least value of the number; the numbers of minus infinity and below are all values')
        const float least = low <= kLeast >> kShift ? minus_infinity() : value_of(low << kShift);
        uint32_t listed = 0;
        for (uint32_t turn = 0; turn < n && listed <= S::kList; turn += kTurn * kAhead) {
            Piece p[kAhead];
#pragma unroll
            for (int u = 0; u < kAhead; ++u) {
                const uint32_t i = turn + u * kTurn + threadIdx.x / kLanes;
                p[u] = piece(i < n ? s.groups[i] : 0, i < n);
            }
            float v[kAhead][NE];
            u64 counts = 0;
#pragma unroll
            for (int u = 0; u < kAhead; ++u) {
                V::unpack(p[u].raw, v[u]);
                uint32_t count = 0;
#pragma unroll
                for (uint32_t j = 0; j < NE; ++j) {
                    v[u][j] = no_nan(v[u][j]);
                    count += j < p[u].have && v[u][j] >= least;
                }
                counts |= static_cast<u64>(count) << (16 * u);
            }
            u64 all;
            u64 mine = before(counts, &all);
#pragma unroll
            for (int u = 0; u < kAhead; ++u) {
                uint32_t at = listed + static_cast<uint32_t>(mine & 0xffffu);
#pragma unroll
                for (uint32_t j = 0; j < NE; ++j) {
                    if (j < p[u].have && v[u][j] >= least) put(at++, v[u][j], p[u].place + j);
                }
                listed += static_cast<uint32_t>(all & 0xffffu);
                mine >>= 16;
                all >>= 16;
            }
        }
        __syncthreads();
        return listed;
    }
    // The same where of the elements that are `low` the first `equal` are wanted: a turn after the other.
    __device__ __forceinline__ uint32_t list_ties(uint32_t n, uint32_t low, uint32_t equal)
    {
        uint32_t over_all = 0, same_all = 0;
        for (uint32_t turn = 0; turn < n; turn += kTurn) {
            const uint32_t i = turn + threadIdx.x / kLanes;
            const Piece p = piece(i < n ? s.groups[i] : 0, i < n);
            float v[NE];
            V::unpack(p.raw, v);
            uint32_t number[NE];
            uint32_t over = 0, same = 0;
#pragma unroll
            for (uint32_t j = 0; j < NE; ++j) {
                number[j] = number_of(no_nan(v[j])) >> kShift;
                over += j < p.have && number[j] > low;
                same += j < p.have && number[j] == low;
            }
            uint32_t all;
            const uint32_t packed = before(over << 16 | same, &all);
            uint32_t same_before = same_all + (packed & 0xffffu);
            uint32_t at = over_all + (packed >> 16) + min(same_before, equal);
#pragma unroll
            for (uint32_t j = 0; j < NE; ++j) {
                if (j >= p.have || number[j] < low) continue;
                if (number[j] == low && same_before++ >= equal) continue;
                put(at++, no_nan(v[j]), p.place + j);
            }
            over_all += all >> 16;
            same_all += all & 0xffffu;
        }
        __syncthreads();
        return over_all + min(same_all, equal);
    }

    // The first `k` (HCCLX_TOP_MAX at most) of the order, and others if that is as easy: s.list.listed holds them in the order of their
    // columns, the number of them is returned.  sure: how many of them are the first of the order.
    __device__ __forceinline__ uint32_t list_first(uint32_t k, uint32_t *sure)
    {
        // Groups: those whose largest reaches `low`.
        Range g = {0, top >> kShift, 0, ngroups, 0, 0};
        uint32_t equal = kNoEnd;   // of the groups whose largest is low, the first so many
        const uint32_t enough = max(k + k / 2 + 32, S::kList / kGroup);
        if (ngroups > enough) {
            g.low = bottom >> kShift;
            do {
                narrow<false>(g, [&](auto &&f) { each_group([&](uint32_t, uint32_t n) { f(n >> kShift, [] { return u64(0); }); }); },
                              [&](u64) { return u64(k); });
            } while (g.above + g.inside > enough && g.low != g.high);
            if (g.above + g.inside > enough) equal = k - g.above;   // (groups left out may hold what is listed of the others)
            if (g.above + g.inside < k) g.low = 0;   // (fewer groups than k: many ranks of few columns)
        }
        uint32_t n = 0;
        {
            uint32_t over = 0, same = 0;
            each_group([&](uint32_t, uint32_t m) {
                over += m != kNone && m >> kShift > g.low;
                same += m != kNone && m >> kShift == g.low;
            });
            // (over: at most `enough`; both fit)
            static_assert(S::kMostGroups < 4096 && HCCLX_LOGITS_MAX_COLUMNS / kGroup + 8 * kMostRanks < 1 << 20, "");
            uint32_t all;
            const uint32_t packed = before(over << 20 | same, &all);
            uint32_t same_before = packed & 0xfffffu;
            uint32_t at = (packed >> 20) + min(same_before, equal);
            n = min((all >> 20) + min(all & 0xfffffu, equal), S::kMostGroups);   // (never more: `enough` and k bound them)
            each_group([&](uint32_t i, uint32_t m) {
                if (m == kNone || m >> kShift < g.low) return;
                if (m >> kShift == g.low && same_before++ >= equal) return;
                if (at < S::kMostGroups) s.groups[at] = i;
                ++at;
            });
            __syncthreads();
        }
        // Elements that reach what all groups reach, if they fit.
        uint32_t listed = kNoEnd;
        uint32_t low = g.low;
        if (low != 0 || n * kGroup <= S::kList) listed = list(n, low);
        if (listed > S::kList) {
            // The same again with the vectors of the groups in the groups' place: where there are k, elements reach the k-th vector's largest.
            Range e = {low, top >> kShift, 0, 0, 0, 0};
            do {
                narrow<false>(e, [&](auto &&f) {
                    each_piece(s.groups, n, [&](const Piece &p, const float (&v)[NE]) {
                        if (p.have == 0) return;
                        float m = minus_infinity();
#pragma unroll
                        for (uint32_t j = 0; j < NE; ++j) m = fmaxf(m, v[j]);
                        f(number_of(m) >> kShift, [] { return u64(0); });
                    });
                }, [&](u64) { return u64(k); });
            } while (e.above + e.inside > k + k / 2 + 32 && e.low != e.high);
            if (e.above + e.inside >= k) listed = list(n, low = e.low);
        }
        if (listed > S::kList) {   // elements themselves
            Range e = {low, top >> kShift, 0, 0, 0, 0};
            do {
                narrow<false>(e, [&](auto &&f) { each(s.groups, n, f); }, [&](u64) { return u64(k); });
            } while (e.above + e.inside > S::kList && e.low != e.high);
            listed = e.above + e.inside > S::kList ? list_ties(n, e.low, k - e.above) : list(n, e.low);
        }
        *sure = equal == kNoEnd ? listed : k;
        return listed;
    }

};

template <int DT, int NT, typename S>
__global__ void __launch_bounds__(NT)
k_top_logits(SelectArgs a)
{
    using D = DTypeOf<DT>;
    __shared__ S s;
    Row<DT, NT, S> r(a, s, blockIdx.x);
    r.c = 1.4426950408889634074;   // (of the sum)
    uint32_t sure;
    const uint32_t n = r.list_first(a.k, &sure);
    auto write = [&](uint32_t place, u64 x) {
        reinterpret_cast<typename D::S *>(a.values)[r.row * a.k + place] = D::narrow(value_of(static_cast<uint32_t>(x >> 32)));
        a.indices[r.row * a.k + place] = static_cast<int32_t>(column_of<DT>(a, x));
    };
    if (n <= kCounted) {
        const uint32_t place = r.template count_before<false>(n, 0, nullptr);
        if (threadIdx.x < n && place < a.k) write(place, s.list.listed[threadIdx.x]);
    } else {
        r.sort(n);
        for (uint32_t i = threadIdx.x; i < a.k; i += NT) write(i, s.list.sorted[i]);
    }
    if (a.lse != nullptr) {
        double sum = 0.0;
        for (uint32_t i = threadIdx.x; i < a.nruns; i += NT) sum += r.run_sum(i);
        sum = r.total(sum);
        if (threadIdx.x == 0) a.lse[r.row] = static_cast<float>(r.top_value + log(sum));
    }
}

typedef unsigned __int128 u128;

// x times whole, for 0 < x < 1, as the whole number below or (UP) above: exactly, from the 24 bits of x and all of the product, which has 100 at
// most.  (In doubles a whole of more than 2^53 was rounded first, and a border that lies at the product was on either side of it.)
template <bool UP, typename W>
__device__ __forceinline__ W share_of(float x, W whole)
{
    const uint32_t bits = __float_as_uint(x), power = max(bits >> 23, 1u);
    const u64 m = (bits & 0x7fffffu) | (bits >> 23 != 0 ? 0x800000u : 0u);
    const uint32_t down = min(150 - power, 127u);   // x = m 2^-down: 24 or more
    if constexpr (sizeof(W) == 8) {   // (half the operations)
        const u64 low = m * whole, high = __umul64hi(m, whole);
        const u64 n = down < 64 ? high << (64 - down) | low >> down : high >> (down - 64);
        const u64 rest = down < 64 ? low << (64 - down) : low | (high & ~(~u64(0) << (down - 64)));
        return n + (UP && rest != 0 ? 1 : 0);
    } else {
        const u128 product = whole * m, n = product >> down;
        return n + (UP && n << down != product ? 1 : 0);
    }
}
// floor(u x whole), inside the whole
template <typename W>
__device__ __forceinline__ W aim_of(float u, W whole)
{
    if (!(u > 0.0f)) return 0;
    return u < 1.0f ? share_of<false>(u, whole) : whole - 1;
}
// What of `whole` top_p asks for.
__device__ __forceinline__ u64 part_of(float p, u64 whole) { return p > 0.0f ? share_of<true>(p, whole) : 0; }

// The same of a sum over a whole row, in multiples of 2^-51, as multiples of 2^-bits.
__device__ __forceinline__ u64 part_of_whole(const SelectArgs &a, float p, u128 whole)
{
    if (!(p > 0.0f)) return 0;
    const u128 n = share_of<true>(p, whole);
    const uint32_t down = kWholeBits - a.bits;
    return static_cast<u64>(n >> down) + ((n >> down) << down != n ? 1 : 0);
}

// What stays of a row that no list holds: numbers over `cut`, the first `equal` of those that are it, and of them all what is `least`
// times as probable as the first.
struct Kept {
    uint32_t cut;   // (without idle bits)
    uint32_t equal;
    double least;
};

// Draws among them: the chunks of the row are weighed, 512 at a time, and the one that the aim lies in is gone through.  A first walk
// finds the whole.
template <int DT, int NT>
__device__ __forceinline__ void draw_kept(const SelectArgs &a, Row<DT, NT> &r, Shared &s, const Kept &kept, float u)
{
    using R = Row<DT, NT>;
    constexpr uint32_t NE = R::NE;
    constexpr uint32_t kShift = kIdle<DT>;
    constexpr uint32_t kWalk = NT < 512 ? NT : 512;
    const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x / 64;
    const bool drop = kept.least > 0.0;
    auto weight = [&](uint32_t number) {
        if (drop && !(r.share(number) >= kept.least)) return u64(0);
        return r.weight(number);
    };
    u64 aim = 0, whole = 0;
    for (int find = 0; find < 2; ++find) {
        u64 weight_before = 0;
        uint32_t equal_before = 0;
        for (uint32_t first = 0; first < a.rows.nchunks; first += kWalk) {
            u64 equal_weight = 0;   // of one element at the cut
            for (uint32_t at = wave; at < kWalk; at += R::kWaves) {
                const uint32_t chunk = first + at;
                u64 sum = 0;
                uint32_t same = 0;
                if (chunk < a.rows.nchunks) {
                    const Stretch t = a.rows.chunks[chunk];
                    const u32x4 raw = load_piece<DT, false>(t.at + r.row * t.step, lane, t.elems);
                    float v[NE];
                    R::V::unpack(raw, v);
#pragma unroll
                    for (uint32_t e = 0; e < NE; ++e) {
                        const uint32_t number = number_of(no_nan(v[e]));
                        if (lane * NE + e >= t.elems || number >> kShift < kept.cut) continue;
                        if (number >> kShift == kept.cut) {
                            ++same;
                            equal_weight = weight(number);
                        } else {
                            sum += weight(number);
                        }
                    }
                }
                sum = wave_total(sum);
                same = wave_total(same);
                if (lane == 0) {
                    s.walk.weight[at] = sum;
                    s.walk.equal[at] = same;
                }
            }
            if (equal_weight != 0) s.one = equal_weight;   // (all that do write the same)
            __syncthreads();
            const u64 one = s.one;
            const u64 sum = threadIdx.x < kWalk ? s.walk.weight[threadIdx.x] : 0;
            const uint32_t same = threadIdx.x < kWalk ? s.walk.equal[threadIdx.x] : 0;
            uint32_t same_all;
            const uint32_t same_before = equal_before + r.before(same, &same_all);
            const uint32_t taken = min(same_before + same, kept.equal) - min(same_before, kept.equal);
            u64 sum_all;
            const u64 mine = sum + taken * one;
            const u64 at = weight_before + r.before(mine, &sum_all);
            if (find == 1 && aim >= at && aim - at < mine) {
                s.word[0] = first + threadIdx.x;   // the chunk
                s.word[1] = same_before;
                s.word64[0] = at;
            }
            weight_before += sum_all;
            equal_before += same_all;
            __syncthreads();
        }
        if (find == 0) {
            whole = weight_before;
            aim = aim_of(u, whole);
        }
    }
    if (wave != 0) return;
    // one wavefront, one chunk
    const Stretch t = a.rows.chunks[s.word[0]];
    const u32x4 raw = load_piece<DT, false>(t.at + r.row * t.step, lane, t.elems);
    float v[NE];
    R::V::unpack(raw, v);
    uint32_t same = 0;
#pragma unroll
    for (uint32_t e = 0; e < NE; ++e) same += lane * NE + e < t.elems && number_of(no_nan(v[e])) >> kShift == kept.cut;
    uint32_t same_before = wave_sums(same) + s.word[1] - same;
    u64 w[NE];
    u64 sum = 0;
#pragma unroll
    for (uint32_t e = 0; e < NE; ++e) {
        const uint32_t number = number_of(no_nan(v[e]));
        bool in = lane * NE + e < t.elems && number >> kShift >= kept.cut;
        if (in && number >> kShift == kept.cut) in = same_before++ < kept.equal;
        sum += w[e] = in ? weight(number) : 0;
    }
    u64 at = wave_sums(sum) + s.word64[0] - sum;
#pragma unroll
    for (uint32_t e = 0; e < NE; ++e) {
        if (aim >= at && aim - at < w[e]) {
            r.write_choice(t.first + lane * NE + e, number_of(no_nan(v[e])), ldexp(static_cast<double>(whole), -static_cast<int>(a.bits)));
        }
        at += w[e];
    }
}

// A walk over the chunks of a row, in their order: f(chunk, what the weights in front of it sum up to, its own).  Weights are multiples of 2^-51, the
// most that the sum of a chunk has room for in 64 bits, and sums over chunks have 128.  Returns that of the row.  AGAIN: the walk before was
// this row's, and what it weighed last is still there.
template <int DT, int NT, bool AGAIN, typename F>
__device__ __forceinline__ u128 walk_whole(const SelectArgs &a, Row<DT, NT> &r, Shared &s, F &&f)
{
    using R = Row<DT, NT>;
    constexpr uint32_t NE = R::NE;
    const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x / 64;
    static_assert(NT == 512, "a thread for each chunk");
    u128 front = 0;
    for (uint32_t first = 0; first < a.rows.nchunks; first += NT) {
        for (uint32_t at = wave; at < NT; at += R::kWaves) {
            if (AGAIN && a.rows.nchunks <= NT) break;
            const uint32_t chunk = first + at;
            u64 sum = 0;
            if (chunk < a.rows.nchunks) {
                const Stretch t = a.rows.chunks[chunk];
                const u32x4 raw = load_piece<DT, false>(t.at + r.row * t.step, lane, t.elems);
                float v[NE];
                R::V::unpack(raw, v);
#pragma unroll
                for (uint32_t e = 0; e < NE; ++e) sum += lane * NE + e < t.elems ? r.weight(no_nan(v[e]), kWholeBits) : 0;
            }
            sum = wave_total(sum);
            if (lane == 0) s.walk.weight[at] = sum;
        }
        __syncthreads();
        const u64 mine = s.walk.weight[threadIdx.x];
        u64 low_all, high_all;
        const u64 low = r.before(mine & 0xffffffffu, &low_all);
        const u64 high = r.before(mine >> 32, &high_all);
        f(first + threadIdx.x, front + (static_cast<u128>(high) << 32) + low, mine);
        front += (static_cast<u128>(high_all) << 32) + low_all;
        __syncthreads();
    }
    return front;
}

// No filter, by the definition: the chunk that the aim lies in is gone through.
template <int DT, int NT>
__device__ __forceinline__ void draw_whole(const SelectArgs &a, Row<DT, NT> &r, Shared &s, float u)
{
    using R = Row<DT, NT>;
    constexpr uint32_t NE = R::NE;
    const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x / 64;
    const u128 whole = walk_whole<DT, NT, false>(a, r, s, [](uint32_t, u128, u64) {});
    const u128 aim = aim_of(u, whole);
    (void)walk_whole<DT, NT, true>(a, r, s, [&](uint32_t chunk, u128 at, u64 mine) {
        if (aim >= at && aim - at < mine) {
            s.word[0] = chunk;
            s.word64[0] = static_cast<u64>(aim - at);
        }
    });
    if (wave != 0) return;
    // one wavefront, one chunk
    const Stretch t = a.rows.chunks[s.word[0]];
    const u32x4 raw = load_piece<DT, false>(t.at + r.row * t.step, lane, t.elems);
    float v[NE];
    R::V::unpack(raw, v);
    u64 w[NE];
    u64 sum = 0;
#pragma unroll
    for (uint32_t e = 0; e < NE; ++e) sum += w[e] = lane * NE + e < t.elems ? r.weight(no_nan(v[e]), kWholeBits) : 0;
    u64 at = wave_sums(sum) - sum;
    const u64 rest = s.word64[0];
#pragma unroll
    for (uint32_t e = 0; e < NE; ++e) {
        if (rest >= at && rest - at < w[e]) {
            const double all = static_cast<double>(static_cast<u64>(whole >> 64)) * 0x1p64 + static_cast<double>(static_cast<u64>(whole));
            r.write_choice(t.first + lane * NE + e, number_of(no_nan(v[e])), ldexp(all, -static_cast<int>(kWholeBits)));
        }
        at += w[e];
    }
}

// How far a sum of doubles over what the first launch's runs hold, whose order goes by the plan (how many chunks a run has), may be from that of the
// multiples of 2^-51, with an error of each of n elements in it.  That is 2^-52 where a number is rounded, and 2^-53 of a run's largest where
// the run leaves it out (taken twice).  In parts of the whole: an exponent of up to 53 powers of two, rounded twice, is good to 2^-46.8 of its
// term; three of them, and 200 additions of doubles one behind the other, make 2^-44.3.
__device__ __forceinline__ double slack(double n, double whole) { return n * 0x1p-51 + whole * 0x1p-43; }

// No filter: the run in which the running sum passes u x the whole, then the element, by such sums.  The whole numbers say the same where both of
// the element's borders are further from the aim than that can matter: with k elements in front of a border, the distance border - u whole
// is off by 1 - u of the error of the first k and u of that of the others.
// Otherwise false is returned, and nothing is drawn (for one row of 131072 columns in some millions, whose chunks are then weighed again: 76 us
// more; 1 row takes 9 us without that).
template <int DT, int NT>
__device__ __forceinline__ bool draw_all(const SelectArgs &a, Row<DT, NT> &r, Shared &s, float u)
{
    using R = Row<DT, NT>;
    constexpr uint32_t NE = R::NE;
    const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x / 64;
    const uint32_t each = (a.nruns + NT - 1) / NT;
    const uint32_t from = min(threadIdx.x * each, a.nruns), to = min(from + each, a.nruns);
    double mine = 0.0;
    for (uint32_t i = from; i < to; ++i) mine += r.run_sum(i);
    if (threadIdx.x == 0) {
        s.word[0] = s.word[1] = 0;
        s.word[2] = 1;   // nothing is drawn
    }
    double whole;
    const double begin = r.before(mine, &whole);
    double at = begin;
    double aim = static_cast<double>(u) * whole;
    if (!(aim > 0.0)) aim = 0.0;
    // the last run that begins at or before the aim and has anything (sums are rounded: the aim may lie behind all)
    uint32_t last = 0;
    for (uint32_t i = from; i < to; ++i) {
        const double w = each == 1 ? mine : r.run_sum(i);
        if (w > 0.0 && at <= aim) last = i + 1;
        at += w;
    }
    last = wave_most(last);
    if (lane == 0 && last != 0) atomicMax(&s.word[0], last);
    __syncthreads();
    const uint32_t run = s.word[0] - 1;
    if (run >= from && run < to) {
        at = begin;
        for (uint32_t i = from; i < run; ++i) at += r.run_sum(i);
        s.word64[0] = __builtin_bit_cast(u64, at);
    }
    // its chunks, one for each wavefront
    const uint32_t chunk = run * a.per_run + wave;
    const bool there = wave < a.per_run && chunk < a.rows.nchunks;
    const Stretch t = a.rows.chunks[there ? chunk : 0];
    const uint32_t elems = there ? t.elems : 0;
    const u32x4 raw = load_piece<DT, false>(t.at + r.row * t.step, lane, elems);
    float v[NE];
    R::V::unpack(raw, v);
    double w[NE];
    double sum = 0.0;
#pragma unroll
    for (uint32_t e = 0; e < NE; ++e) {
        w[e] = lane * NE + e < elems ? r.share(no_nan(v[e]), 0) : 0.0;
        sum += w[e];
    }
    double all;
    at = r.before(sum, &all);
    at += __builtin_bit_cast(double, s.word64[0]);
    const double first = at;
    last = 0;
#pragma unroll
    for (uint32_t e = 0; e < NE; ++e) {
        if (w[e] > 0.0 && at <= aim) last = threadIdx.x * NE + e + 1;
        at += w[e];
    }
    last = wave_most(last);
    if (lane == 0 && last != 0) atomicMax(&s.word[1], last);
    __syncthreads();
    const uint32_t place = s.word[1] - 1;
    if (place / NE == threadIdx.x) {
        float l = 0.0f;
        double its = 0.0, front = 0.0;
        at = first;
#pragma unroll
        for (uint32_t e = 0; e < NE; ++e) {
            if (place % NE == e) {
                l = no_nan(v[e]);
                its = w[e];
                front = at;
            }
            at += w[e];
        }
        const uint32_t column = t.first + (lane * NE + place % NE);
        const double share = fmin(fmax(static_cast<double>(u), 0.0), 1.0);
        const double gap = slack((1.0 - share) * (column + 2) + share * (a.rows.vocab - column + 1), whole);
        // (at 0: nothing in front of it has any weight)
        if ((front == 0.0 || aim - front >= gap) && front + its - aim >= gap) {
            r.write_choice(column, number_of(l), whole);
            s.word[2] = 0;
        }
    }
    __syncthreads();
    return s.word[2] == 0;
}

// The cut is searched by numbers, among all elements, and chunks are weighed: right for every row, but one workgroup goes through all
// of it several times (where top_p is a part of the whole row once more, for the sum of that).
template <int DT, int NT>
__device__ __forceinline__ void draw_by_numbers(const SelectArgs &a, Row<DT, NT> &r, Shared &s, const RowChoice &choice, float u)
{
    constexpr uint32_t kShift = kIdle<DT>;
    Kept stay = {0, kNoEnd, choice.by_min ? choice.least : 0.0};
    auto all = [&](auto &&f) { r.each(nullptr, r.ngroups, f); };
    Range range = {kLeast >> kShift, r.top >> kShift, 0, 0, 0, 0};
    uint32_t cut_count = 0;
    if (choice.by_k) {
        do {
            r.template narrow<false>(range, all, [&](u64) { return u64(choice.k); });
        } while (range.low != range.high);
        stay.cut = range.low;
        stay.equal = choice.k - range.above;
        cut_count = range.inside;
    }
    if (choice.by_p) {
        range = {stay.cut > kLeast >> kShift ? stay.cut : kLeast >> kShift, r.top >> kShift, 0, 0, 0, 0};
        u64 aim = 0;
        if (!choice.by_k) aim = part_of_whole(a, choice.p, walk_whole<DT, NT, false>(a, r, s, [](uint32_t, u128, u64) {}));
        bool first = true;
        // (what is equal to the cut of top_k and does not stay is at the end of the order)
        const u64 over = choice.by_k && cut_count > stay.equal ? (cut_count - stay.equal) * r.weight(stay.cut << kShift | (stay.cut >> (31 - kShift) != 0 ? 0 : (1u << kShift) - 1)) : 0;
        do {
            r.template narrow<true>(range, all, [&](u64 whole) {
                if (first) aim = max(u64(1), min(choice.by_k ? part_of(choice.p, whole - over) : aim, whole));
                return aim;
            });
            first = false;
        } while (range.low != range.high);
        const u64 one = range.inside != 0 ? range.weight_inside / range.inside : 1;
        const u64 need = one != 0 ? (aim - range.weight_above + one - 1) / one : 1;
        const uint32_t equal = static_cast<uint32_t>(min(need, static_cast<u64>(range.inside)));
        stay.equal = stay.cut == range.low && choice.by_k ? min(stay.equal, equal) : equal;
        stay.cut = range.low;
    }
    if (threadIdx.x == 0) s.one = 0;
    __syncthreads();
    draw_kept(a, r, s, stay, u);
}

// Distances from the row's largest in levels.
struct Distance {
    float top;
    float scale;   // 64 log2(e) / T
    bool fits;     // whether a row has levels
    __device__ __forceinline__ Distance(double top_value, double c) : top(static_cast<float>(top_value)), scale(static_cast<float>(64.0 * c))
    {
        fits = top != __builtin_inff() && scale >= 0x1p-80f && scale <= 0x1p80f;
    }
    __device__ __forceinline__ float operator()(float l) const { return (top - l) * scale; }   // (NaN of NaN)
};
// 64 levels to a power of two over 24 of them, and 8 to each of the 64 behind: a top_k may reach that far down.
constexpr uint32_t kNear = 24 * 64;
constexpr uint32_t kStep = 8;
__device__ __forceinline__ uint32_t level_of(float x)   // (minus infinity has the nearest whole number that there is)
{
    const uint32_t at = static_cast<uint32_t>(fminf(x, 65536.0f));
    return at < kNear ? at : min(kNear + (at - kNear) / kStep, kLevels - 1);
}
__device__ __forceinline__ uint32_t level_begin(uint32_t level) { return level < kNear ? level : kNear + (level - kNear) * kStep; }

// What a level holds is one word: its elements, times 2^40, and what they lack of the weight that they would have at the level's upper
// end, in parts of 2^22 of that (2^18 in the wide ones, which have 2^-24 of the largest's weight): 1 - 2^(-f / 64) for an element f 64ths of a power
// of two further down, of which two terms do.  Rounding to such parts costs the sum over a level some 2^-23 of itself at random, so which level
// holds the cut of top_p is known but for one in many thousands of rows; the draw finds out.
__device__ __forceinline__ float lack_of(uint32_t level) { return level < kNear ? 0x1p22f : 0x1p18f; }
__device__ __forceinline__ u64 level_entry(float x, uint32_t level)
{
    const float z = (x - static_cast<float>(level_begin(level))) * static_cast<float>(0.69314718055994530942 / 64);
    return u64(1) << 40 | static_cast<uint32_t>(rintf((z - 0.5f * z * z) * lack_of(level)));
}
__device__ __forceinline__ uint32_t entry_count(u64 e) { return static_cast<uint32_t>(e >> 40); }
__device__ __forceinline__ double entry_weight(u64 e, uint32_t level, double at_end)
{
    return at_end * (entry_count(e) - static_cast<double>(e & ((u64(1) << 40) - 1)) / lack_of(level));
}

// Whether several workgroups can draw from a row: not where the weight that top_p asks for goes by a cut of top_k.
__device__ __forceinline__ bool is_wide(const RowChoice &choice, double top_value)
{
    return !(choice.by_k && choice.by_p) && Distance(top_value, choice.c).fits;
}

// The chunks first .. last - 1 of a part of a row that may be left to several workgroups.
struct WidePart {
    uint32_t slot;
    uint32_t from;   // spans
    uint32_t to;
    __device__ __forceinline__ WidePart(const SelectArgs &a, uint32_t block) : slot(block / a.wide_parts)
    {
        const uint32_t part = block % a.wide_parts;
        from = a.nspans * part / a.wide_parts;
        to = a.nspans * (part + 1) / a.wide_parts;
    }
};

// The elements of a part by levels.  Where there are few rows, by workgroups of the second launch that have no row of their own, before it is
// known whether levels are asked for: by then they are there (37 rows of 50021: 32 us for the draw, 37 with a launch of its own; 256 of 131072
// 73 and 79; 1 row 16 and 17.5).  Where rows fill the device that holds up the others (1024 rows of 131072: 225 us for the draw, 186 with a
// launch of its own, which rows that are not asked leave at once).
template <int DT, int NT>
__device__ __forceinline__ void count_levels(const SelectArgs &a, u64 *mine, uint32_t *most, uint32_t block)
{
    using V = Vec16<DT>;
    constexpr uint32_t NE = V::NE;
    constexpr uint32_t kWaves = NT / 64;
    constexpr int kAhead = 4;
    const WidePart part(a, block);
    const uint64_t row = a.first + part.slot;
    const RowChoice choice(a.choice, row, a.rows.vocab);
    if (!choice.by_levels()) return;
    for (uint32_t i = threadIdx.x; i < kLevels; i += NT) mine[i] = 0;
    const uint32_t ngroups = a.rows.nchunks * (kChunk<DT> / kGroup);
    uint32_t top = 0;
    for (uint32_t i = threadIdx.x * 4; i < ngroups; i += NT * 4) {
        const u32x4 v = *reinterpret_cast<const u32x4 *>(a.most + row * ngroups + i);
        top = max(max(top, max(v.x, v.y)), max(v.z, v.w));
    }
    top = wave_most(top);
    const uint32_t lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
    if (lane == 0) most[wave] = top;
    __syncthreads();
    for (uint32_t w = 0; w < kWaves; ++w) top = max(top, most[w]);
    const Distance distance(value_of(top), choice.c);
    if (top <= kLeast || !distance.fits) return;
    // What is so improbable that even as many as there are columns hold no more than 1 - top_p of the largest's weight alone lies behind the cut.
    float far = __builtin_inff();
    if (!choice.by_k) {
        const double behind = (1.0 - static_cast<double>(choice.p)) / a.rows.vocab;
        if (behind > 0.0) far = static_cast<float>(-64.0 * log2(behind)) + 2.0f;
    }
    const uint32_t to = min(part.to * a.span, a.rows.nchunks);
    for (uint32_t first = part.from * a.span + wave; first < to; first += kWaves * kAhead) {
        u32x4 raw[kAhead];
        uint32_t elems[kAhead];
#pragma unroll
        for (int k = 0; k < kAhead; ++k) {
            const uint32_t i = first + k * kWaves;
            const Stretch t = a.rows.chunks[i < to ? i : first];
            elems[k] = i < to ? t.elems : 0;
            raw[k] = load_piece<DT, false>(t.at + row * t.step, lane, elems[k]);
        }
#pragma unroll
        for (int k = 0; k < kAhead; ++k) {
            float v[NE];
            V::unpack(raw[k], v);
#pragma unroll
            for (uint32_t e = 0; e < NE; ++e) {
                const float x = distance(v[e]);
                if (!(x <= far) || lane * NE + e >= elems[k]) continue;
                const uint32_t level = level_of(x);
                // (what is in the last one is not told apart)
                atomicAdd(&mine[level], level == kLevels - 1 ? u64(1) << 40 : level_entry(x, level));
            }
        }
    }
    __syncthreads();
    u64 *const all = a.levels + static_cast<uint64_t>(part.slot) * kLevels;
    for (uint32_t i = threadIdx.x; i < kLevels; i += NT) {
        if (mine[i] != 0) atomicAdd(&all[i], mine[i]);
    }
}

template <int DT, int NT>
__global__ void __launch_bounds__(NT)
k_sample_levels(SelectArgs a)
{
    __shared__ u64 s_levels[kLevels];
    __shared__ uint32_t s_most[NT / 64];
    if (a.wide[blockIdx.x / a.wide_parts].wide == 1) count_levels<DT, NT>(a, s_levels, s_most, blockIdx.x);
}

template <int NT>
__device__ __forceinline__ Band band_of(const SelectArgs &a, Team<NT> &r, Shared &s, const RowChoice &choice, const Wide &w, const u64 *levels)
{
    constexpr uint32_t kMine = kLevels / NT;
    const Distance distance(r.top_value, r.c);
    Band band = {-1.0f, __builtin_inff(), choice.by_k || choice.by_p, choice.by_min, true};
    if (band.by_level) {
        // levels are as far apart as the rounded scale has them
        const double apart = r.c / static_cast<double>(distance.scale);
        if (threadIdx.x == 0) s.word[0] = kLevels;
        uint32_t counts[kMine];
        double weights[kMine];
        uint32_t count = 0, all;
        double weight = 0.0, whole;
#pragma unroll
        for (uint32_t i = 0; i < kMine; ++i) {
            const uint32_t level = threadIdx.x * kMine + i;
            const u64 e = levels[level];
            count += counts[i] = entry_count(e);
            weight += weights[i] = counts[i] == 0 ? 0.0 : entry_weight(e, level, exp2_exact(-(level_begin(level) * apart)));
        }
        count = r.before(count, &all);
        weight = r.before(weight, &whole);
        const double aim = ldexp(static_cast<double>(w.p_high), -static_cast<int>(a.bits));
#pragma unroll
        for (uint32_t i = 0; i < kMine; ++i) {
            const bool by_k = choice.by_k && count < choice.k && count + counts[i] >= choice.k;
            const bool by_p = !choice.by_k && weight < aim && weight + weights[i] >= aim;
            if (counts[i] != 0 && (by_k || by_p)) s.word[0] = threadIdx.x * kMine + i;
            count += counts[i];
            weight += weights[i];
        }
        __syncthreads();
        const uint32_t level = s.word[0];
        __syncthreads();
        band.known = level < kLevels - 1;
        band.low = static_cast<float>(level_begin(level));
        band.high = static_cast<float>(level_begin(level + 1));
    }
    if (band.by_min && band.known) {
        // (distances are good to 2^-22 of themselves, and none that matters is over 2^14)
        const float at = static_cast<float>(-log2(choice.least) / r.c * static_cast<double>(distance.scale));
        const float low = at - 0.01f, high = at + 0.01f;
        if (!band.by_level || high <= band.low) {   // (the draw finds out whether the cut of top_p is nearer than its level after all)
            band.by_level = false;
            band.low = low;
            band.high = high;
        } else if (low >= band.high) {
            band.by_min = false;
        } else {
            band.low = fminf(low, band.low);
            band.high = fmaxf(high, band.high);
        }
    }
    return band;
}

// Weighs a wavefront's chunk: the elements nearer than the band (their weight is returned in every lane, their number is added to `over`), and
// lists those in it.  Few of many elements may be that near, and a weight takes some thirty instructions of 64 bits: they are
// gathered in LDS, and weighed by all lanes.
template <int DT, int NT>
__device__ __forceinline__ u64 weigh_chunk(const Team<NT> &r, Shared &s, const Distance &distance, const Band &band, uint32_t chunk, u32x4 raw,
                                           uint32_t elems, uint32_t *over)
{
    using V = Vec16<DT>;
    constexpr uint32_t NE = V::NE;
    static_assert(64 * NE <= kQueue, "");
    const uint32_t lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
    float *const queue = s.wide.queue[wave];
    float v[NE];
    V::unpack(raw, v);
    uint32_t near = 0, in = 0;
#pragma unroll
    for (uint32_t e = 0; e < NE; ++e) {
        const float x = distance(v[e]);
        const bool there = lane * NE + e < elems;
        near |= (there && x < band.low ? 1u : 0u) << e;
        in |= (there && x >= band.low && x < band.high ? 1u : 0u) << e;
    }
    if (in != 0) {
        uint32_t at = atomicAdd(&s.word[2], static_cast<uint32_t>(__popc(in)));
#pragma unroll
        for (uint32_t e = 0; e < NE; ++e) {
            if ((in >> e & 1) == 0) continue;
            const uint32_t place = chunk * kChunk<DT> + lane * NE + e;
            if (at < kList) s.wide.listed[at] = static_cast<u64>(number_of(v[e])) << 32 | static_cast<uint32_t>(~place);
            ++at;
        }
    }
    const uint32_t mine = __popc(near);
    const uint32_t sums = wave_sums(mine);
    const uint32_t found = of_last_lane(sums);
    uint32_t at = sums - mine;
#pragma unroll
    for (uint32_t e = 0; e < NE; ++e) {
        if (near >> e & 1) queue[at++] = v[e];
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    u64 sum = 0;
    for (uint32_t i = 0; i < found; i += 128) {
        const uint32_t first = i + lane, second = first + 64;
        const u64 one = r.weight(queue[min(first, found - 1)]), two = r.weight(queue[min(second, found - 1)]);
        sum += (first < found ? one : 0) + (second < found ? two : 0);
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    *over += found;
    return wave_total(sum);
}

// What stays of a list whose elements the threads hold, N each (key 0: none): those from the returned key on.  `stay` of them stay (top_k), or
// those before whose place in the order the weight is less than `aim`; *front is what is before the last of them.  As by Row::narrow: keys are
// counted and weighed into equal stretches of their range, which leaves one of them: two rounds, or three where many numbers are alike.
template <int NT, int N>
__device__ __forceinline__ u64 last_that_stays(Team<NT> &r, Shared &s, const u64 (&key)[N], const u64 (&weight)[N], bool by_count, uint32_t stay, u64 aim, u64 *front)
{
    static_assert(NT == 512, "a stretch for each thread");
    const uint32_t t = threadIdx.x;
    uint32_t most = 0, least = kNoEnd, place = 0;
#pragma unroll
    for (int i = 0; i < N; ++i) {
        if (key[i] == 0) continue;
        most = max(most, static_cast<uint32_t>(key[i] >> 32));
        least = min(least, static_cast<uint32_t>(key[i] >> 32));
        place = max(place, ~static_cast<uint32_t>(key[i]));
    }
    most = wave_most(most);
    least = ~wave_most(~least);
    place = wave_most(place);
    if ((t & 63) == 0) {
        s.most[t / 64] = most;
        s.least[t / 64] = least;
        s.place[t / 64] = place;
    }
    __syncthreads();
#pragma unroll
    for (uint32_t w = 0; w < NT / 64; ++w) {
        most = max(most, s.most[w]);
        least = min(least, s.least[w]);
        place = max(place, s.place[w]);
    }
    u64 low = static_cast<u64>(least) << 32 | static_cast<uint32_t>(~place), high = static_cast<u64>(most) << 32 | kNoEnd;
    uint32_t count_before = 0;
    u64 weight_before = 0;
    while (low != high) {
        const u64 width = high - low;
        const uint32_t shift = width < NT ? 0 : 64 - __clzll(static_cast<long long>(width)) - 9;
        s.bins.count[t] = 0;
        s.bins.weight[t] = 0;
        __syncthreads();
#pragma unroll
        for (int i = 0; i < N; ++i) {
            if (key[i] < low || key[i] > high) continue;
            const uint32_t bin = static_cast<uint32_t>((key[i] - low) >> shift);
            atomicAdd(&s.bins.count[bin], 1u);
            if (weight[i] != 0) atomicAdd(&s.bins.weight[bin], weight[i]);
        }
        __syncthreads();
        const uint32_t bin = NT - 1 - t;   // from the top
        const uint32_t more = s.bins.count[bin];
        const u64 add = s.bins.weight[bin];
        uint32_t all;
        u64 whole;
        const uint32_t c = count_before + r.before(more, &all);
        const u64 w = weight_before + r.before(add, &whole);
        if (more != 0 && (by_count ? c < stay && c + more >= stay : w < aim && w + add >= aim)) s.range = {bin, 0, c, more, w, 0};
        __syncthreads();
        const Range found = s.range;
        count_before = found.above;
        *front = weight_before = found.weight_above;
        const u64 begin = low + (static_cast<u64>(found.low) << shift);
        high = min(high, begin + ((u64(1) << shift) - 1));
        low = begin;
        if (found.inside == 1) {   // its own key
#pragma unroll
            for (int i = 0; i < N; ++i) {
                if (key[i] >= low && key[i] <= high) s.one = key[i];
            }
            __syncthreads();
            return s.one;
        }
    }
    return low;
}

// The third launch: weights of a part's spans, and the list of what the cut lies among.
template <int DT, int NT>
__global__ void __launch_bounds__(NT)
k_sample_weigh(SelectArgs a)
{
    constexpr uint32_t kWaves = NT / 64;
    constexpr uint32_t kAhead = 4;
    static_assert(NT >= kMostSpans, "a thread for each span");
    __shared__ Shared s;
    const WidePart part(a, blockIdx.x);
    const Wide wide = a.wide[part.slot];
    if (wide.wide != 1) return;
    const uint64_t row = a.first + part.slot;
    const uint32_t lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
    const uint32_t first = part.from * a.span, to = min(part.to * a.span, a.rows.nchunks);
    u32x4 raw[kAhead];
    uint32_t elems[kAhead];
    const auto load = [&](uint32_t chunk) {
#pragma unroll
        for (uint32_t k = 0; k < kAhead; ++k) {
            const uint32_t i = chunk + k * kWaves;
            const Stretch t = a.rows.chunks[i < to ? i : first];
            elems[k] = i < to ? t.elems : 0;
            raw[k] = load_piece<DT, false>(t.at + row * t.step, lane, elems[k]);
        }
    };
    load(first + wave);   // (on its way while the band is found)
    const RowChoice choice(a.choice, row, a.rows.vocab);
    Team<NT> r(a, s, row, wide.top, choice.c);
    const Distance distance(r.top_value, r.c);
    if (threadIdx.x < part.to - part.from) s.span_weight[threadIdx.x] = 0;
    if (threadIdx.x == 0) s.word[2] = 0;
    const Band band = band_of(a, r, s, choice, wide, a.levels + static_cast<uint64_t>(part.slot) * kLevels);
    if (blockIdx.x % a.wide_parts == 0 && threadIdx.x == 0) a.bands[part.slot] = band;
    if (!band.known) return;
    __syncthreads();
    u64 weight = 0;
    uint32_t over = 0;
    for (uint32_t chunk = first + wave; chunk < to; chunk += kWaves * kAhead) {
        if (chunk != first + wave) load(chunk);
#pragma unroll
        for (uint32_t k = 0; k < kAhead; ++k) {
            const uint32_t i = chunk + k * kWaves;
            if (i >= to) break;
            const u64 sum = weigh_chunk<DT>(r, s, distance, band, i, raw[k], elems[k], &over);
            weight += sum;
            if (lane == 0 && sum != 0) atomicAdd(&s.span_weight[i / a.span - part.from], sum);
        }
    }
    weight = r.total(lane == 0 ? weight : 0);
    over = r.total(lane == 0 ? over : 0);
    if (threadIdx.x < part.to - part.from) a.spans[static_cast<uint64_t>(part.slot) * kMostSpans + part.from + threadIdx.x] = s.span_weight[threadIdx.x];
    const uint32_t listed = s.word[2];
    for (uint32_t i = threadIdx.x; i < min(listed, a.band_each); i += NT) a.listed[static_cast<uint64_t>(blockIdx.x) * a.band_each + i] = s.wide.listed[i];
    if (threadIdx.x == 0) a.found[blockIdx.x] = {weight, over, listed};
}

// Draws from a row of whose band n elements are listed, N for a thread at most; `over` elements of the weight `above` are nearer.  Returns false,
// and nothing is drawn, where the cut is not among them, or top_p may ask for one more or less.
template <int DT, int NT, int N>
__device__ __forceinline__ bool draw_band(const SelectArgs &a, Team<NT> &r, Shared &s, const RowChoice &choice, const Band &band, float u, const Wide &wide,
                                          uint32_t n, uint32_t over, u64 above)
{
    using V = Vec16<DT>;
    constexpr uint32_t NE = V::NE;
    constexpr uint32_t kWaves = NT / 64;
    const uint32_t lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
    const Distance distance(r.top_value, r.c);
    const uint64_t slot = blockIdx.x;
    u64 key[N], w[N];
    u64 sum = 0;
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const uint32_t place = threadIdx.x + i * NT;
        uint32_t part = 0;
#pragma unroll
        for (uint32_t d = kMostParts / 2; d != 0; d /= 2) part += s.groups[part + d] <= place ? d : 0;
        key[i] = place < n ? a.listed[(slot * a.wide_parts + part) * a.band_each + place - s.groups[part]] : 0;
        sum += w[i] = place < n ? r.weight(static_cast<uint32_t>(key[i] >> 32)) : 0;
    }
    const u64 inside = r.total(sum);
    u64 last = 0;
    if (band.by_level) {
        const bool right = choice.by_k ? over < choice.k && over + n >= choice.k : above < wide.p_low && above + inside >= wide.p_high;
        if (!right) return false;
        u64 front = 0;
        last = last_that_stays(r, s, key, w, choice.by_k, choice.k - over, wide.p_high - above, &front);
        if (!choice.by_k && above + front >= wide.p_low) return false;   // (what top_p asks for may be in front of it)
    }
    const auto stays = [&](u64 x) {
        return x >= last && (!band.by_min || static_cast<uint32_t>(x >> 32) == r.top || r.share(static_cast<uint32_t>(x >> 32)) >= choice.least);
    };
    // the spans' weights, with those of the band that stay
    __syncthreads();
    s.span_weight[threadIdx.x] = threadIdx.x < a.nspans ? a.spans[slot * kMostSpans + threadIdx.x] : 0;
    static_assert(NT == kMostSpans, "a thread for each span");
    __syncthreads();
#pragma unroll
    for (int i = 0; i < N; ++i) {
        if (w[i] != 0 && stays(key[i])) atomicAdd(&s.span_weight[~static_cast<uint32_t>(key[i]) / kChunk<DT> / a.span], w[i]);
    }
    __syncthreads();
    // the span, then the element: a wavefront for each chunk
    sum = s.span_weight[threadIdx.x];
    u64 whole;
    u64 begin = r.before(sum, &whole);
    if (choice.by_p && !band.by_level && whole >= wide.p_low) return false;   // (top_p cuts off some of what min_p leaves)
    const u64 aim = aim_of(u, whole);
    if (aim >= begin && aim - begin < sum) {
        s.word[0] = threadIdx.x;
        s.word64[0] = begin;
    }
    __syncthreads();
    const uint32_t first = s.word[0] * a.span;
    const uint32_t to = min(first + a.span, a.rows.nchunks);
    begin = s.word64[0];
    for (uint32_t turn = first; turn < to; turn += kWaves) {
        const bool there = turn + wave < to;
        const uint32_t chunk = there ? turn + wave : first;
        const Stretch t = a.rows.chunks[chunk];
        const uint32_t elems = there ? t.elems : 0;
        const u32x4 raw = load_piece<DT, false>(t.at + r.row * t.step, lane, elems);
        float v[NE];
        V::unpack(raw, v);
        u64 each[NE];
        sum = 0;
#pragma unroll
        for (uint32_t e = 0; e < NE; ++e) {
            const u64 x = static_cast<u64>(number_of(no_nan(v[e]))) << 32 | static_cast<uint32_t>(~(chunk * kChunk<DT> + lane * NE + e));
            const bool in = lane * NE + e < elems && (distance(v[e]) < band.low || stays(x));
            sum += each[e] = in ? r.weight(v[e]) : 0;
        }
        u64 all;
        u64 at = begin + r.before(sum, &all);
#pragma unroll
        for (uint32_t e = 0; e < NE; ++e) {
            if (aim >= at && aim - at < each[e]) {
                r.write_choice(t.first + lane * NE + e, number_of(v[e]), ldexp(static_cast<double>(whole), -static_cast<int>(a.bits)));
            }
            at += each[e];
        }
        begin += all;
    }
    return true;
}

// The last launch: the cut of rows that are left to it, and the draw.
template <int DT, int NT>
__global__ void __launch_bounds__(NT)
k_sample_wide(SelectArgs a)
{
    __shared__ Shared s;
    const Wide wide = a.wide[blockIdx.x];
    if (wide.wide == 0) return;
    const uint64_t row = a.first + blockIdx.x;
    const RowChoice choice(a.choice, row, a.rows.vocab);
    const float u = a.choice.random[row];
    const uint32_t lane = threadIdx.x & 63;
    if (wide.wide == 1) {
        const Band band = a.bands[blockIdx.x];
        if (band.known) {
            Found f = {0, 0, 0};
            if (lane < a.wide_parts) f = a.found[blockIdx.x * a.wide_parts + lane];
            static_assert(kMostParts <= 64 && (kMostParts & (kMostParts - 1)) == 0, "");
            const uint32_t begin = wave_sums(f.listed) - f.listed;   // of the part's list in that of all
            const uint32_t n = wave_total(f.listed), over = wave_total(f.over);
            const u64 above = wave_total(static_cast<u64>(f.weight));
            if (n <= kBand && wave_most(f.listed) <= a.band_each) {
                if (threadIdx.x < 64) s.groups[lane] = lane < a.wide_parts ? begin : n;
                Team<NT> r(a, s, row, wide.top, choice.c);
                __syncthreads();
                if (n <= kBand / 4 ? draw_band<DT, NT, kBand / 4 / NT>(a, r, s, choice, band, u, wide, n, over, above)
                                   : draw_band<DT, NT, kBand / NT>(a, r, s, choice, band, u, wide, n, over, above)) {
                    return;
                }
            }
        }
    }
    // The cut's level has more elements than are listed, or the cut is in another.  (Or there is no cut, and what is to be drawn is next to a border.)
    __syncthreads();
    Row<DT, NT> r(a, s, row);
    r.c = choice.c;
    if (choice.none()) {
        draw_whole(a, r, s, u);
        return;
    }
    draw_by_numbers(a, r, s, choice, u);
}

// The second launch: rows from a.first on.  ALONE: there are none behind it, since no row has a filter, or none is longer than a list.
// (Otherwise six wavefronts for a SIMD: one register more, and a CU has two workgroups instead of three.)
template <int DT, int NT, bool ALONE>
__global__ void __launch_bounds__(NT, ALONE ? 4 : 6)
k_sample(SelectArgs a, uint32_t rows)
{
    constexpr uint32_t kMine = kList / NT;
    __shared__ Shared s;
    if (!ALONE && blockIdx.x >= rows) {
        static_assert(kList >= kLevels, "");
        count_levels<DT, NT>(a, s.list.listed, s.most, blockIdx.x - rows);
        return;
    }
    const uint64_t row = a.first + blockIdx.x;
    Wide &wide = a.wide[blockIdx.x];
    if (threadIdx.x == 0) wide.wide = 0;
    Row<DT, NT> r(a, s, row);
    const RowChoice choice(a.choice, row, a.rows.vocab);
    const float u = a.choice.random[row];
    r.c = choice.c;
    if (r.top <= kLeast) {   // nothing to choose from
        if (threadIdx.x == 0) {
            a.choice.token[r.row] = -1;
            if (a.choice.logprob != nullptr) a.choice.logprob[r.row] = minus_infinity();
        }
        return;
    }
    if (choice.none()) {
        if (draw_all(a, r, s, u)) return;
        if constexpr (ALONE) {
            draw_whole(a, r, s, u);
        } else if (threadIdx.x == 0) {
            wide = {2, r.top, 0, 0};
        }
        return;
    }
    const double unit = ldexp(1.0, -static_cast<int>(a.bits));
    // The weight that top_p asks for lies between these two.  Of a whole row that comes from sums of doubles; where an element ends between them, the row is
    // left to the launches behind, the last of which adds up whole numbers.
    u64 p_low = 0, p_high = 0;
    if (choice.by_p && !choice.by_k) {
        double mine = 0.0;
        for (uint32_t i = threadIdx.x; i < a.nruns; i += NT) mine += r.run_sum(i);
        mine = r.total(mine);
        const double off = slack(a.rows.vocab, mine);
        p_low = part_of(choice.p, static_cast<u64>(ldexp(fmax(mine - off, 0.0), static_cast<int>(a.bits))));
        p_high = part_of(choice.p, static_cast<u64>(ldexp(mine + off, static_cast<int>(a.bits))) + 1);
    }
    uint32_t sure = 0;
    if (!choice.by_k || choice.k <= HCCLX_TOP_MAX) {
        const uint32_t n = r.list_first(choice.by_k ? choice.k : min(kNucleus, a.rows.vocab), &sure);
        const uint32_t limit = choice.by_k ? choice.k : sure;
        if (n <= kCounted) {
            const u64 x = threadIdx.x < n ? s.list.listed[threadIdx.x] : 0;
            const float l = value_of(static_cast<uint32_t>(x >> 32));
            const u64 w = threadIdx.x < n ? r.weight(l) : 0;
            u64 weight_before;
            const uint32_t place = r.template count_before<true>(n, w, &weight_before);
            const bool first = threadIdx.x < n && place < limit;
            // (where the list holds the whole row, bits is kWholeBits)
            if (choice.by_p && (choice.by_k || n == a.rows.vocab)) p_low = p_high = part_of(choice.p, r.total(first ? w : 0));
            bool in = first;
            if (choice.by_p) in = in && (place == 0 || weight_before < p_high);
            if (choice.by_min) in = in && (place == 0 || r.share(l, 0) >= choice.least);
            const bool unsure = choice.by_p && in && place != 0 && weight_before >= p_low;
            if (choice.by_k || n == a.rows.vocab || r.total(unsure ? kNotSure : static_cast<uint32_t>(in)) < sure) {
                u64 whole;
                const u64 at = r.before(in ? w : 0, &whole);
                const u64 aim = aim_of(u, whole);
                if (in && aim >= at && aim - at < w) r.write_choice(column_of<DT>(a, x), static_cast<uint32_t>(x >> 32), static_cast<double>(whole) * unit);
                return;
            }
        } else {
            r.sort(n);
            u64 w[kMine];
            u64 sum = 0;
#pragma unroll
            for (uint32_t i = 0; i < kMine; ++i) {
                const uint32_t at = threadIdx.x * kMine + i;
                sum += w[i] = at < limit ? r.weight(static_cast<uint32_t>(s.list.sorted[at] >> 32)) : 0;
            }
            u64 whole;
            u64 at = r.before(sum, &whole);
            if (choice.by_p && (choice.by_k || n == a.rows.vocab)) p_low = p_high = part_of(choice.p, whole);
            uint32_t keep = 0;
#pragma unroll
            for (uint32_t i = 0; i < kMine; ++i) {
                const uint32_t place = threadIdx.x * kMine + i;
                bool in = place < limit;
                if (choice.by_p) in = in && (place == 0 || at < p_high);
                if (choice.by_min) in = in && (place == 0 || r.share(static_cast<uint32_t>(s.list.sorted[place] >> 32)) >= choice.least);
                keep += choice.by_p && in && place != 0 && at >= p_low ? kNotSure : in;
                at += w[i];
            }
            const uint32_t kept = r.total(keep);
            if (choice.by_k || kept < sure || n == a.rows.vocab) {
                const u64 last = s.list.sorted[kept - 1];
                sum = 0;
#pragma unroll
                for (uint32_t i = 0; i < kMine; ++i) {
                    const uint32_t place = threadIdx.x * kMine + i;
                    const u64 x = place < n ? s.list.listed[place] : 0;
                    sum += w[i] = place < n && x >= last ? r.weight(static_cast<uint32_t>(x >> 32)) : 0;
                }
                at = r.before(sum, &whole);
                const u64 aim = aim_of(u, whole);
#pragma unroll
                for (uint32_t i = 0; i < kMine; ++i) {
                    if (aim >= at && aim - at < w[i]) {
                        const u64 x = s.list.listed[threadIdx.x * kMine + i];
                        r.write_choice(column_of<DT>(a, x), static_cast<uint32_t>(x >> 32), static_cast<double>(whole) * unit);
                    }
                    at += w[i];
                }
                return;
            }
        }
    }
    // (never where there is no launch for it: the list held all columns)
    if (threadIdx.x == 0) wide = {is_wide(choice, r.top_value) ? 1u : 2u, r.top, p_low, p_high};
}

// ---- host ------------------------------------------------------------------------------------------------------------------

struct SelectWork : PlanWork {
    SelectArgs args{};
    Table table;
    DeviceBlock scratch;   // most, runs
    int dtype = 0;
    bool sample = false;
    uint32_t parts = 1;    // workgroups of the first launch per row
    uint32_t batch = 0;         // rows whose wide ones are drawn from together
    bool small = false;         // whether many rows with short lists have small workgroups
    bool apart = false;         // whether levels are counted in a launch of their own

    template <int DT, int U>
    void runs(const SelectArgs &args, uint32_t rows, hipStream_t st) const
    {
        const dim3 grid(rows * parts), block(kRunWaves * 64);
        if (sample) {
            HCCLX_LAUNCH((k_logit_runs<DT, U, kRunChoice>), grid, block, 0, st, args, parts);
        } else if (args.lse != nullptr) {
            HCCLX_LAUNCH((k_logit_runs<DT, U, kRunSum>), grid, block, 0, st, args, parts);
        } else {
            HCCLX_LAUNCH((k_logit_runs<DT, U, kRunPlain>), grid, block, 0, st, args, parts);
        }
    }
    template <int DT>
    void first_launch(const SelectArgs &a, uint32_t rows, hipStream_t st) const
    {
        switch (a.per_run) {
            case 1: runs<DT, 1>(a, rows, st); break;
            case 2: runs<DT, 2>(a, rows, st); break;
            case 4: runs<DT, 4>(a, rows, st); break;
            default: runs<DT, 8>(a, rows, st); break;
        }
    }
    template <int DT>
    void run(hipStream_t st) const
    {
        constexpr int NT = 512;
        if (!sample) {
            first_launch<DT>(args, args.rows.rows, st);
            if (small) {
                HCCLX_LAUNCH((k_top_logits<DT, NT / 2, SmallShared>), dim3(args.rows.rows), dim3(NT / 2), 0, st, args);
            } else {
                HCCLX_LAUNCH((k_top_logits<DT, NT, Shared>), dim3(args.rows.rows), dim3(NT), 0, st, args);
            }
            return;
        }
        SelectArgs of = args;
        for (uint32_t first = 0; first < args.rows.rows; first += batch) {
            of.first = first;
            const uint32_t rows = std::min(batch, args.rows.rows - first);
            const uint32_t parts_of_all = rows * args.wide_parts;
            first_launch<DT>(of, rows, st);
            if (args.wide_parts == 0) {
                HCCLX_LAUNCH((k_sample<DT, NT, true>), dim3(rows), dim3(NT), 0, st, of, rows);
                continue;
            }
            HCCLX_LAUNCH((k_sample<DT, NT, false>), dim3(rows + (apart ? 0 : parts_of_all)), dim3(NT), 0, st, of, rows);
            if (apart) HCCLX_LAUNCH((k_sample_levels<DT, NT>), dim3(parts_of_all), dim3(NT), 0, st, of);
            HCCLX_LAUNCH((k_sample_weigh<DT, NT>), dim3(parts_of_all), dim3(NT), 0, st, of);
            HCCLX_LAUNCH((k_sample_wide<DT, NT>), dim3(rows), dim3(NT), 0, st, of);
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
        return e == hipSuccess ? HCCL_SUCCESS : fail_hip(e, sample ? "sampling kernels" : "top logits kernels");
    }
};

// The table, the scratch memory and the shape of the first launch.
int finish(const hcclx_logits_t &l, uint32_t vocab, bool sums, std::unique_ptr<SelectWork> w, hcclx_plan_t **plan)
{
    DeviceCtx *ctx = device_ctx();
    if (!ctx) return HCCL_E_RUNTIME;
    int rc = lay_out(l, nullptr, vocab, &w->table);
    if (rc != HCCL_SUCCESS) return rc;
    SelectArgs &a = w->args;
    a.rows = w->table.rows;
    w->dtype = l.dtype;
    // As many chunks per wavefront as leave every CU eight workgroups (64 draws of 131072 40.3 us, with four 39.7, with sixteen 41.0).
    a.per_run = 8;
    auto parts = [&] { return (a.rows.nchunks + a.per_run * kRunWaves - 1) / (a.per_run * kRunWaves); };
    while (a.per_run > 1 && static_cast<uint64_t>(l.rows) * parts() < 8ull * static_cast<uint32_t>(ctx->num_cus)) a.per_run /= 2;
    w->parts = parts();
    if (static_cast<uint64_t>(l.rows) * w->parts * kRunWaves * 64 > 0xffffffffull) return fail(HCCL_E_PARA, "too many rows of so many columns");
    a.nruns = (a.rows.nchunks + a.per_run - 1) / a.per_run;
    a.bits = 51;   // a weight is below 2^52, the sum of all below 2^62
    while (vocab > 1ull << (62 - a.bits)) --a.bits;
    const uint64_t runs = sums ? static_cast<uint64_t>(l.rows) * a.nruns * sizeof(Run) : 0;
    const uint32_t per = 64 * (16 / dtype_size(l.dtype)) / kGroup;
    const uint64_t most = static_cast<uint64_t>(l.rows) * a.rows.nchunks * per * sizeof(uint32_t);
    uint64_t held = runs + most;
    const auto more = [&](uint64_t bytes) {
        const uint64_t at = held = (held + 15) / 16 * 16;
        held += bytes;
        return at;
    };
    // Where rows fill the device more than three times, small workgroups for their lists, of which seven find room on a CU (64 of 4096 rows of
    // 131072 bf16 237 us, by four large ones 249, of 5000 67 and 85; of 1000 rows of 5000 22.7 and 26.1, of 600 19.1 and 18.7).
    w->small = a.k <= kSmallTop && l.rows > 3 * static_cast<uint32_t>(ctx->num_cus);
    uint64_t wide = 0, bands = 0, levels = 0, found = 0, listed = 0, spans = 0;
    if (w->sample && l.rows != 0) {
        // Rows that the list of kNucleus always does for are never wide; nor are those that no filter but a short top_k may shorten, which
        // only the device knows.
        w->batch = std::min(l.rows, kBatch);
        w->apart = w->batch > static_cast<uint32_t>(ctx->num_cus);
        const bool may_be_wide = vocab > kNucleus && (a.choice.top_k != nullptr || a.choice.top_p != nullptr || a.choice.min_p != nullptr);
        a.span = (a.rows.nchunks + kMostSpans - 1) / kMostSpans;
        a.nspans = (a.rows.nchunks + a.span - 1) / a.span;
        // Workgroups for a row that may be wide: most rows are not, and their workgroups only look.  In launches of their own eight for a row
        // (1024 rows of 131072 186 us, with four 200, with two 228, with sixteen 188), of sixteen chunks at least (of 5000 65, with eight 71); next to
        // the lists as many as there is room for (256 rows 73 us with eight, 78 with sixteen, 81 with 32; 1 row 16 with two, eight or 32).
        const uint32_t parts = w->apart ? std::clamp(std::min(8192 / w->batch, (a.rows.nchunks + 15) / 16), 1u, 8u) : std::clamp(2048 / w->batch, 2u, kMostParts);
        a.wide_parts = may_be_wide ? std::min(a.nspans, parts) : 0;
        a.band_each = std::clamp(kBand / std::max(1u, a.wide_parts), 512u, kList);
        wide = more(w->batch * sizeof(Wide));
        levels = more(may_be_wide ? w->batch * sizeof(u64) * kLevels : 0);
        bands = more(w->batch * sizeof(Band));
        found = more(static_cast<uint64_t>(w->batch) * a.wide_parts * sizeof(Found));
        listed = more(static_cast<uint64_t>(w->batch) * a.wide_parts * sizeof(u64) * a.band_each);
        spans = more(may_be_wide ? w->batch * sizeof(u64) * kMostSpans : 0);
    }
    if (held != 0 && (rc = w->scratch.get(held)) != HCCL_SUCCESS) return rc;
    a.runs = reinterpret_cast<Run *>(w->scratch.p);
    a.most = reinterpret_cast<uint32_t *>(w->scratch.p + runs);
    a.wide = reinterpret_cast<Wide *>(w->scratch.p + wide);
    a.levels = reinterpret_cast<u64 *>(w->scratch.p + levels);
    a.bands = reinterpret_cast<Band *>(w->scratch.p + bands);
    a.found = reinterpret_cast<Found *>(w->scratch.p + found);
    a.listed = reinterpret_cast<u64 *>(w->scratch.p + listed);
    a.spans = reinterpret_cast<u64 *>(w->scratch.p + spans);
    const uint64_t all = held + w->table.bytes;
    return plan_of(ctx, std::move(w), static_cast<uint64_t>(l.rows) * vocab * dtype_size(l.dtype), all, plan);
}

struct Out {
    const char *what;
    const void *p;
    uint64_t bytes;
};

int make_top(const hcclx_top_logits_t &t, hcclx_plan_t **plan)
{
    const hcclx_logits_t &l = t.logits;
    uint32_t vocab = 0;
    int rc = logits::check(l, nullptr, &vocab);
    if (rc != HCCL_SUCCESS) return rc;
    if (t.k == 0 || t.k > HCCLX_TOP_MAX || t.k > vocab) {
        return fail(HCCL_E_PARA, "k outside 1.." + std::to_string(std::min<uint32_t>(HCCLX_TOP_MAX, vocab)));
    }
    const bool none = l.rows == 0;
    const uint64_t size = dtype_size(l.dtype), entries = static_cast<uint64_t>(l.rows) * t.k;
    if ((rc = check_array(t.values, size, none, "values")) != HCCL_SUCCESS) return rc;
    if ((rc = check_array(t.indices, 4, none, "indices")) != HCCL_SUCCESS) return rc;
    if ((rc = check_array(t.lse, 4, true, "lse")) != HCCL_SUCCESS) return rc;
    const Out out[3] = {{"values", t.values, entries * size}, {"indices", t.indices, entries * 4}, {"lse", t.lse, l.rows * 4ull}};
    for (uint32_t i = 0; i < 3; ++i) {
        if ((rc = check_apart(l, "logits", l.logits, out[i].what, out[i].p, out[i].bytes)) != HCCL_SUCCESS) return rc;
        for (uint32_t j = 0; j < i; ++j) {
            if ((rc = check_apart(out[i].what, out[i].p, out[i].bytes, out[j].what, out[j].p, out[j].bytes)) != HCCL_SUCCESS) return rc;
        }
    }
    auto w = std::make_unique<SelectWork>();
    w->args.k = t.k;
    w->args.values = static_cast<char *>(t.values);
    w->args.indices = t.indices;
    w->args.lse = t.lse;
    return finish(l, vocab, t.lse != nullptr, std::move(w), plan);
}

int make_sample(const hcclx_sample_t &t, hcclx_plan_t **plan)
{
    const hcclx_logits_t &l = t.logits;
    uint32_t vocab = 0;
    int rc = logits::check(l, nullptr, &vocab);
    if (rc != HCCL_SUCCESS) return rc;
    const bool none = l.rows == 0;
    const uint64_t bytes = l.rows * 4ull;
    const Out in[5] = {{"temperature", t.temperature, bytes}, {"top_k", t.top_k, bytes}, {"top_p", t.top_p, bytes}, {"min_p", t.min_p, bytes},
                       {"random", t.random, bytes}};
    for (uint32_t i = 0; i < 5; ++i) {
        if ((rc = check_array(in[i].p, 4, none || i != 4, in[i].what)) != HCCL_SUCCESS) return rc;
    }
    if ((rc = check_array(t.token, 4, none, "token")) != HCCL_SUCCESS) return rc;
    if ((rc = check_array(t.logprob, 4, true, "logprob")) != HCCL_SUCCESS) return rc;
    const Out out[2] = {{"token", t.token, bytes}, {"logprob", t.logprob, bytes}};
    for (const Out &o : out) {
        if ((rc = check_apart(l, "logits", l.logits, o.what, o.p, o.bytes)) != HCCL_SUCCESS) return rc;
        for (const Out &i : in) {
            if ((rc = check_apart(o.what, o.p, o.bytes, i.what, i.p, i.bytes)) != HCCL_SUCCESS) return rc;
        }
    }
    if ((rc = check_apart("logprob", t.logprob, bytes, "token", t.token, bytes)) != HCCL_SUCCESS) return rc;
    auto w = std::make_unique<SelectWork>();
    w->sample = true;
    w->args.choice = {t.temperature, t.top_k, t.top_p, t.min_p, t.random, t.token, t.logprob};
    return finish(l, vocab, true, std::move(w), plan);
}

}  // namespace

extern "C" {

int hcclx_top_logits_plan_create(const hcclx_top_logits_t *top, hcclx_plan_t **plan)
{
    if (plan == nullptr) return fail(HCCL_E_PTR, "plan is null");
    *plan = nullptr;
    if (top == nullptr) return fail(HCCL_E_PTR, "top is null");
    return guarded([&] { return make_top(*top, plan); });
}

int hcclx_sample_plan_create(const hcclx_sample_t *sample, hcclx_plan_t **plan)
{
    if (plan == nullptr) return fail(HCCL_E_PTR, "plan is null");
    *plan = nullptr;
    if (sample == nullptr) return fail(HCCL_E_PTR, "sample is null");
    return guarded([&] { return make_sample(*sample, plan); });
}

}  // extern "C"
