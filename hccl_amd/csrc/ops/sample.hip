// The largest logits of a row, and the draw of the next token (include/hcclx_ops.h: hcclx_top_logits_*, hcclx_sample_*).
//
// Two launches.  The first reads every logit once and leaves, of every 64 neighbouring columns (a group), the largest, and for runs
// of a few chunks the sum of exp((l - most) / T) where it is wanted.  The second, a workgroup per row, works on what that left:
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
#include "ops/logits.h"

#include <algorithm>

using namespace hcclx;
using namespace hcclx::logits;

namespace {

constexpr uint32_t kGroup = 64;          // columns
constexpr uint32_t kRunWaves = 4;        // of a workgroup of the first launch, a run each
constexpr uint32_t kThreads = 512;       // of the second
constexpr uint32_t kWaves = kThreads / 64;
constexpr uint32_t kBins = 4 * kThreads;
constexpr uint32_t kList = 2048;         // elements that are sorted at once
constexpr uint32_t kMostGroups = HCCLX_TOP_MAX + HCCLX_TOP_MAX / 2 + 32;
constexpr uint32_t kNucleus = 256;       // listed where no top_k bounds the list
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

struct SelectArgs {
    Rows rows;
    uint32_t *most;     // [rows][nchunks * groups of a chunk]: the numbers of the groups' largest
    Run *runs;          // [rows][nruns]
    uint32_t nruns;
    uint32_t per_run;   // chunks
    uint32_t bits;      // s
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

struct RowChoice {
    bool greedy;
    bool by_k;
    bool by_p;
    bool by_min;
    uint32_t k;
    double p;
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
    const uint64_t row = blockIdx.x / parts;
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
    const uint32_t run = blockIdx.x % parts * kRunWaves + wave;
    const uint32_t lane = threadIdx.x & 63;
    const uint32_t from = run * U;
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
        if (most == minus_infinity()) {
        } else if constexpr (KIND == kRunSum) {
            float s = 0.0f;
#pragma unroll
            for (int u = 0; u < U; ++u) {
                float f[NE];
                V::unpack(raw[u], f);
#pragma unroll
                for (int e = 0; e < NE; ++e) s += no_nan(f[e]) == most ? 1.0f : exp2_fast((no_nan(f[e]) - most) * 1.44269504f);
            }
            sum = wave_sum(s);
        } else {
#pragma unroll
            for (int u = 0; u < U; ++u) {
                float f[NE];
                V::unpack(raw[u], f);
#pragma unroll
                for (int e = 0; e < NE; ++e) {
                    const float l = no_nan(f[e]);
                    sum += l == most ? 1.0 : exp2_exact((static_cast<double>(l) - most) * choice.c);
                }
            }
            sum = wave_sum64(sum);
        }
        if (lane == 0) a.runs[row * a.nruns + run] = {sum, most, 0};
    }
}

// ---- the second launch ---------------------------------------------------------------------------------------------------

typedef unsigned long long u64;

struct Range {
    uint32_t low;      // numbers (without their idle bits) that are left, both included
    uint32_t high;
    uint32_t above;    // how many are over them
    uint32_t inside;   // and in them
    u64 weight_above;
    u64 weight_inside;
};

struct Shared {
    union {
        struct {
            uint32_t count[kBins];
            u64 weight[kBins];
        } bins;
        struct {
            u64 listed[kList];   // (number, ~column), in the order of the columns
            u64 sorted[kList];
        } list;
        struct {
            u64 weight[kThreads];   // of the wavefronts' pieces of a row
            uint32_t equal[kThreads];
        } walk;
    };
    uint32_t groups[kMostGroups];
    u64 part[2][kWaves];
    double part64[kWaves];
    uint32_t part32[2][kWaves];
    Range range;
    uint32_t word[4];
    u64 wide;
};

// Sums over the threads before this one, and over all.  (Two barriers; s: kWaves.)
template <typename T>
__device__ __forceinline__ T before(T v, T *s, T *all)
{
    const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x / 64;
    T sum = v;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const T o = __shfl_up(sum, d, 64);
        if (lane >= static_cast<uint32_t>(d)) sum += o;
    }
    if (lane == 63) s[wave] = sum;
    __syncthreads();
    T from = 0, whole = 0;
#pragma unroll
    for (uint32_t w = 0; w < kWaves; ++w) {
        from += w < wave ? s[w] : T(0);
        whole += s[w];
    }
    __syncthreads();
    *all = whole;
    return from + sum - v;
}
__device__ __forceinline__ uint32_t most_of(uint32_t v, uint32_t *s)
{
#pragma unroll
    for (int d = 32; d >= 1; d >>= 1) v = max(v, static_cast<uint32_t>(__shfl_xor(v, d, 64)));
    if ((threadIdx.x & 63) == 0) s[threadIdx.x / 64] = v;
    __syncthreads();
    v = s[0];
#pragma unroll
    for (uint32_t w = 1; w < kWaves; ++w) v = max(v, s[w]);
    __syncthreads();
    return v;
}

// One round of the search: the numbers in the range are counted (and weighed) into kBins stretches of it; the range becomes the one in
// which the running count (BY_WEIGHT: weight) from the top reaches what target() says, given the weight in the range.
// each(f): f(number, weight) for every number that there is.
template <bool BY_WEIGHT, typename Each, typename Target>
__device__ __forceinline__ void narrow(Range &r, Shared &s, Each &&each, Target &&target)
{
    const uint32_t width = r.high - r.low;
    const uint32_t shift = width < kBins ? 0 : 32 - __clz(width) - 11;   // kBins = 2^11
    static_assert(kBins == 2048, "");
    for (uint32_t i = threadIdx.x; i < kBins; i += kThreads) {
        s.bins.count[i] = 0;
        if (BY_WEIGHT) s.bins.weight[i] = 0;
    }
    __syncthreads();
    each([&](uint32_t n, auto &&weight) {
        if (n < r.low || n > r.high) return;
        const uint32_t bin = (n - r.low) >> shift;
        atomicAdd(&s.bins.count[bin], 1u);
        if constexpr (BY_WEIGHT) {
            const u64 w = weight();
            if (w != 0) atomicAdd(&s.bins.weight[bin], w);
        }
    });
    __syncthreads();
    // from the top: thread t has four stretches
    constexpr uint32_t kMine = kBins / kThreads;
    uint32_t count[kMine];
    u64 weight[kMine];
    uint32_t counts = 0;
    u64 weights = 0;
#pragma unroll
    for (uint32_t i = 0; i < kMine; ++i) {
        const uint32_t bin = kBins - 1 - (threadIdx.x * kMine + i);
        counts += count[i] = s.bins.count[bin];
        weights += weight[i] = BY_WEIGHT ? s.bins.weight[bin] : 0;
    }
    uint32_t all;
    u64 whole = 0;
    uint32_t c = before(counts, s.part32[0], &all);
    u64 w = BY_WEIGHT ? before(weights, s.part[0], &whole) : 0;
    const u64 there = BY_WEIGHT ? r.weight_above + whole : r.above + all;
    const u64 asked = target(whole);
    const u64 aim = asked < there ? asked : there;   // (all of it, where there is less)
    c += r.above;
    w += r.weight_above;
#pragma unroll
    for (uint32_t i = 0; i < kMine; ++i) {
        const u64 at = BY_WEIGHT ? w : c;
        const u64 add = BY_WEIGHT ? weight[i] : count[i];
        if (at < aim && at + add >= aim) {
            const uint32_t bin = kBins - 1 - (threadIdx.x * kMine + i);
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

// A lane's vector of a group: lanes kGroup / NE in a row hold one.
struct Piece {
    u32x4 raw;
    uint32_t first;   // column
    uint32_t have;    // elements that exist
};
template <int DT>
__device__ __forceinline__ Piece piece_of(const SelectArgs &a, uint64_t row, uint32_t group, bool there)
{
    constexpr uint32_t NE = Vec16<DT>::NE;
    constexpr uint32_t kPer = kChunk<DT> / kGroup;
    const Stretch t = a.rows.chunks[there ? group / kPer : 0];
    const uint32_t lane = group % kPer * (kGroup / NE) + threadIdx.x % (kGroup / NE);   // of the chunk
    const uint32_t at = lane * NE;
    Piece p;
    p.have = !there || at >= t.elems ? 0 : t.elems - at < NE ? t.elems - at : NE;
    p.first = t.first + at;
    p.raw = load_piece<DT, false>(t.at + row * t.step, lane, there ? t.elems : 0);
    return p;
}

template <int DT>
struct Row {
    using V = Vec16<DT>;
    static constexpr uint32_t NE = V::NE;
    static constexpr uint32_t kPer = kChunk<DT> / kGroup;
    static constexpr uint32_t kTurn = kThreads / (kGroup / NE);   // groups of a turn
    const SelectArgs &a;
    const uint64_t row;
    const uint32_t *most;
    const uint32_t ngroups;
    uint32_t top;      // the largest number of the row
    double top_value;
    double c;          // log2(e) / T

    __device__ __forceinline__ Row(const SelectArgs &args, uint64_t r)
        : a(args), row(r), most(args.most + r * args.rows.nchunks * kPer), ngroups(args.rows.nchunks * kPer)
    {
    }
    __device__ __forceinline__ double share(uint32_t number) const   // exp((l - most) / T)
    {
        return number == top ? 1.0 : exp2_exact((static_cast<double>(value_of(number)) - top_value) * c);
    }
    __device__ __forceinline__ u64 weight(uint32_t number) const { return static_cast<u64>(rint(ldexp(share(number), static_cast<int>(a.bits)))); }

    // f(number, weight) of the elements of n groups: those of the list, or (nullptr) all
    template <typename F>
    __device__ __forceinline__ void each(const uint32_t *list, uint32_t n, F &&f) const
    {
        constexpr int kAhead = 4;
        for (uint32_t g = threadIdx.x / (kGroup / NE); g < n; g += kTurn * kAhead) {
            Piece p[kAhead];
#pragma unroll
            for (int u = 0; u < kAhead; ++u) {
                const uint32_t i = g + u * kTurn;
                p[u] = piece_of<DT>(a, row, i < n ? (list != nullptr ? list[i] : i) : 0, i < n);
            }
#pragma unroll
            for (int u = 0; u < kAhead; ++u) {
                float v[NE];
                V::unpack(p[u].raw, v);
#pragma unroll
                for (uint32_t e = 0; e < NE; ++e) {
                    if (e >= p[u].have) continue;
                    const uint32_t number = number_of(no_nan(v[e]));
                    f(number >> kIdle<DT>, [&] { return weight(number); });
                }
            }
        }
    }
};

// The first `k` (kList at most) of the order, more if that is as easy: s.list.listed holds them in the order of their columns, the
// number of them is returned.
template <int DT>
__device__ __forceinline__ uint32_t list_first(const Row<DT> &r, Shared &s, uint32_t k)
{
    constexpr uint32_t NE = Row<DT>::NE;
    constexpr uint32_t kTurn = Row<DT>::kTurn;
    constexpr uint32_t kShift = kIdle<DT>;
    // Groups: those whose largest reaches `low`.
    Range g = {0, r.top >> kShift, 0, r.ngroups, 0, 0};
    uint32_t equal = 0xffffffffu;   // of the groups whose largest is low, the first so many
    const uint32_t enough = max(k + k / 2 + 32, kList / kGroup);
    if (g.inside > enough) {
        g.low = kLeast >> kShift;
        do {
            narrow<false>(g, s, [&](auto &&f) {
                for (uint32_t i = threadIdx.x; i < r.ngroups; i += kThreads) f(r.most[i] >> kShift, [] { return u64(0); });
            }, [&](u64) { return u64(k); });
        } while (g.above + g.inside > enough && g.low != g.high);
        if (g.above + g.inside > enough) equal = k - g.above;
    }
    // listed in their order: a thread looks at neighbours
    uint32_t ngroups = 0;
    {
        const uint32_t each = (r.ngroups + kThreads - 1) / kThreads;
        const uint32_t from = min(threadIdx.x * each, r.ngroups), to = min(from + each, r.ngroups);
        uint32_t over = 0, same = 0;
        for (uint32_t i = from; i < to; ++i) {
            const uint32_t n = r.most[i];
            const bool there = n != kNone;
            over += there && n >> kShift > g.low;
            same += there && n >> kShift == g.low;
        }
        u64 all;
        const u64 packed = before(static_cast<u64>(over) << 32 | same, s.part[0], &all);
        uint32_t same_before = static_cast<uint32_t>(packed);
        uint32_t at = static_cast<uint32_t>(packed >> 32) + min(same_before, equal);
        ngroups = static_cast<uint32_t>(all >> 32) + min(static_cast<uint32_t>(all), equal);
        for (uint32_t i = from; i < to; ++i) {
            const uint32_t n = r.most[i];
            if (n == kNone || n >> kShift < g.low) continue;
            if (n >> kShift == g.low && same_before++ >= equal) continue;
            if (at < kMostGroups) s.groups[at] = i;
            ++at;
        }
        ngroups = min(ngroups, kMostGroups);   // (never more: `enough` and k bound them)
        __syncthreads();
    }
    // Elements: those that reach low, if they fit; else those of a narrower range.
    Range e = {g.low, r.top >> kShift, 0, 0, 0, 0};
    equal = 0xffffffffu;
    for (;;) {
        uint32_t n = 0, over_all = 0, same_all = 0;
        for (uint32_t turn = 0; turn < ngroups && n <= kList; turn += kTurn) {
            const uint32_t i = turn + threadIdx.x / (kGroup / NE);
            const Piece p = piece_of<DT>(r.a, r.row, i < ngroups ? s.groups[i] : 0, i < ngroups);
            float v[NE];
            Row<DT>::V::unpack(p.raw, v);
            uint32_t number[NE];
            uint32_t over = 0, same = 0;
#pragma unroll
            for (uint32_t j = 0; j < NE; ++j) {
                number[j] = number_of(no_nan(v[j]));
                over += j < p.have && number[j] >> kShift > e.low;
                same += j < p.have && number[j] >> kShift == e.low;
            }
            uint32_t all;
            const uint32_t packed = before(over << 16 | same, s.part32[0], &all);   // (of at most kThreads * NE elements)
            uint32_t same_before = same_all + (packed & 0xffffu);
            uint32_t at = over_all + (packed >> 16) + min(same_before, equal);
#pragma unroll
            for (uint32_t j = 0; j < NE; ++j) {
                if (j >= p.have || number[j] >> kShift < e.low) continue;
                if (number[j] >> kShift == e.low && same_before++ >= equal) continue;
                if (at < kList) s.list.listed[at] = static_cast<u64>(number[j]) << 32 | static_cast<uint32_t>(~(p.first + j));
                ++at;
            }
            over_all += all >> 16;
            same_all += all & 0xffffu;
            n = over_all + min(same_all, equal);
        }
        __syncthreads();
        if (n <= kList) return n;
        e.above = e.inside = 0;
        do {
            narrow<false>(e, s, [&](auto &&f) { r.each(s.groups, ngroups, f); }, [&](u64) { return u64(k); });
        } while (e.above + e.inside > kList && e.low != e.high);
        if (e.above + e.inside > kList) equal = k - e.above;
        e.high = r.top >> kShift;
    }
}

// Sorts s.list.listed[0 .. n) into s.list.sorted, descending.
__device__ __forceinline__ void sort_list(Shared &s, uint32_t n)
{
    uint32_t size = 64;
    while (size < n) size *= 2;
    for (uint32_t i = threadIdx.x; i < size; i += kThreads) s.list.sorted[i] = i < n ? s.list.listed[i] : 0;
    __syncthreads();
    for (uint32_t width = 2; width <= size; width *= 2) {
        for (uint32_t step = width / 2; step >= 1; step /= 2) {
            for (uint32_t t = threadIdx.x; t < size / 2; t += kThreads) {
                const uint32_t i = (t & ~(step - 1)) * 2 + (t & (step - 1));
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

// The row's largest number.
template <int DT>
__device__ __forceinline__ uint32_t top_of(const Row<DT> &r, Shared &s)
{
    uint32_t top = 0;
    for (uint32_t i = threadIdx.x; i < r.ngroups; i += kThreads) top = max(top, r.most[i]);
    return most_of(top, s.part32[0]);
}

template <int DT>
__global__ void __launch_bounds__(kThreads)
k_top_logits(SelectArgs a)
{
    using D = DTypeOf<DT>;
    __shared__ Shared s;
    Row<DT> r(a, blockIdx.x);
    r.top = top_of(r, s);
    const uint32_t n = list_first(r, s, a.k);
    sort_list(s, n);
    for (uint32_t i = threadIdx.x; i < a.k; i += kThreads) {
        const u64 x = s.list.sorted[i];
        reinterpret_cast<typename D::S *>(a.values)[r.row * a.k + i] = D::narrow(value_of(static_cast<uint32_t>(x >> 32)));
        a.indices[r.row * a.k + i] = static_cast<int32_t>(~static_cast<uint32_t>(x));
    }
    if (a.lse != nullptr) {
        const float most = value_of(r.top);
        double sum = 0.0;
        for (uint32_t i = threadIdx.x; i < a.nruns; i += kThreads) {
            const Run run = a.runs[r.row * a.nruns + i];
            sum += run.most == most ? run.sum : run.sum * exp2_exact((static_cast<double>(run.most) - most) * 1.4426950408889634074);
        }
        double all;
        (void)before(sum, s.part64, &all);
        if (threadIdx.x == 0) a.lse[r.row] = static_cast<float>(most + log(all));
    }
}

// whole: the sum of what could have been drawn, of exp((l - most) / T).
template <int DT>
__device__ __forceinline__ void write_choice(const SelectArgs &a, const Row<DT> &r, uint32_t column, uint32_t number, double whole)
{
    a.choice.token[r.row] = static_cast<int32_t>(column);
    if (a.choice.logprob != nullptr) {
        const double x = number == r.top ? 0.0 : (static_cast<double>(value_of(number)) - r.top_value) * r.c * 0.69314718055994530942;
        a.choice.logprob[r.row] = static_cast<float>(x - log(whole));
    }
}

// floor(u x whole), inside the whole
__device__ __forceinline__ u64 aim_of(float u, u64 whole)
{
    const double t = static_cast<double>(u) * static_cast<double>(whole);
    if (!(t > 0.0)) return 0;
    return t >= static_cast<double>(whole) ? whole - 1 : min(static_cast<u64>(t), whole - 1);
}

// What stays of a row that no list holds: numbers over `cut`, the first `equal` of those that are it, and of them all what is `least`
// times as probable as the first.
struct Kept {
    uint32_t cut;   // (without idle bits)
    uint32_t equal;
    double least;
};

// Draws among them: the wavefronts' pieces of the row are weighed, kWalk turns at a time, and the one that the aim lies in is gone
// through.  A first walk finds the whole.
template <int DT>
__device__ __forceinline__ void draw_kept(const SelectArgs &a, const Row<DT> &r, Shared &s, const Kept &kept, float u)
{
    constexpr uint32_t NE = Row<DT>::NE;
    constexpr uint32_t kShift = kIdle<DT>;
    constexpr uint32_t kWalk = kThreads / kWaves;   // turns
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
        for (uint32_t first = 0; first < a.rows.nchunks; first += kThreads) {   // kWalk turns of kWaves chunks
            u64 equal_weight = 0;   // of one element at the cut
            for (uint32_t turn = 0; turn < kWalk; ++turn) {
                const uint32_t chunk = first + turn * kWaves + wave;
                u64 sum = 0;
                uint32_t same = 0;
                if (chunk < a.rows.nchunks) {
                    const Stretch t = a.rows.chunks[chunk];
                    const u32x4 raw = load_piece<DT, false>(t.at + r.row * t.step, lane, t.elems);
                    float v[NE];
                    Row<DT>::V::unpack(raw, v);
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
#pragma unroll
                for (int d = 32; d >= 1; d >>= 1) {
                    sum += __shfl_xor(sum, d, 64);
                    same += __shfl_xor(same, d, 64);
                }
                if (lane == 0) {
                    s.walk.weight[turn * kWaves + wave] = sum;
                    s.walk.equal[turn * kWaves + wave] = same;
                }
            }
            if (equal_weight != 0) s.wide = equal_weight;   // (all that do write the same)
            __syncthreads();
            const u64 one = s.wide;
            const u64 sum = s.walk.weight[threadIdx.x];
            const uint32_t same = s.walk.equal[threadIdx.x];
            uint32_t same_all;
            const uint32_t same_before = equal_before + before(same, s.part32[0], &same_all);
            const uint32_t taken = min(same_before + same, kept.equal) - min(same_before, kept.equal);
            u64 sum_all;
            const u64 mine = sum + taken * one;
            const u64 at = weight_before + before(mine, s.part[0], &sum_all);
            if (find == 1 && aim >= at && aim - at < mine) {
                s.word[0] = first + threadIdx.x;   // the chunk
                s.word[1] = same_before;
                s.part[1][0] = at;
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
    Row<DT>::V::unpack(raw, v);
    uint32_t same = 0;
#pragma unroll
    for (uint32_t e = 0; e < NE; ++e) same += lane * NE + e < t.elems && number_of(no_nan(v[e])) >> kShift == kept.cut;
    uint32_t same_before = same;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const uint32_t o = __shfl_up(same_before, d, 64);
        if (lane >= static_cast<uint32_t>(d)) same_before += o;
    }
    same_before += s.word[1] - same;
    u64 w[NE];
    u64 sum = 0;
#pragma unroll
    for (uint32_t e = 0; e < NE; ++e) {
        const uint32_t number = number_of(no_nan(v[e]));
        bool in = lane * NE + e < t.elems && number >> kShift >= kept.cut;
        if (in && number >> kShift == kept.cut) in = same_before++ < kept.equal;
        sum += w[e] = in ? weight(number) : 0;
    }
    u64 at = sum;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const u64 o = __shfl_up(at, d, 64);
        if (lane >= static_cast<uint32_t>(d)) at += o;
    }
    at += s.part[1][0] - sum;
#pragma unroll
    for (uint32_t e = 0; e < NE; ++e) {
        if (aim >= at && aim - at < w[e]) {
            write_choice(a, r, t.first + lane * NE + e, number_of(no_nan(v[e])), ldexp(static_cast<double>(whole), -static_cast<int>(a.bits)));
        }
        at += w[e];
    }
}

// No filter: the run in which the running sum passes u x the whole, then the element.
template <int DT>
__device__ __forceinline__ void draw_all(const SelectArgs &a, const Row<DT> &r, Shared &s, float u)
{
    constexpr uint32_t NE = Row<DT>::NE;
    const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x / 64;
    const Run *runs = a.runs + r.row * a.nruns;
    const uint32_t each = (a.nruns + kThreads - 1) / kThreads;
    const uint32_t from = min(threadIdx.x * each, a.nruns), to = min(from + each, a.nruns);
    auto sum_of = [&](uint32_t i) {
        const Run run = runs[i];
        return run.most == static_cast<float>(r.top_value) ? run.sum : run.sum * exp2_exact((static_cast<double>(run.most) - r.top_value) * r.c);
    };
    double mine = 0.0;
    for (uint32_t i = from; i < to; ++i) mine += sum_of(i);
    double whole;
    const double begin = before(mine, s.part64, &whole);
    double at = begin;
    double aim = static_cast<double>(u) * whole;
    if (!(aim > 0.0)) aim = 0.0;
    // the last run that begins at or before the aim and has anything (sums are rounded: the aim may lie behind all)
    if (threadIdx.x == 0) s.word[0] = 0;
    __syncthreads();
    for (uint32_t i = from; i < to; ++i) {
        const double w = sum_of(i);
        if (w > 0.0 && at <= aim) atomicMax(&s.word[0], i + 1);
        at += w;
    }
    __syncthreads();
    const uint32_t run = s.word[0] - 1;
    if (run >= from && run < to) {
        at = begin;
        for (uint32_t i = from; i < run; ++i) at += sum_of(i);
        s.part64[0] = at;
    }
    __syncthreads();
    at = s.part64[0];
    __syncthreads();
    // its chunks, one for each wavefront
    const uint32_t chunk = run * a.per_run + wave;
    const bool there = wave < a.per_run && chunk < a.rows.nchunks;
    const Stretch t = a.rows.chunks[there ? chunk : 0];
    const uint32_t elems = there ? t.elems : 0;
    const u32x4 raw = load_piece<DT, false>(t.at + r.row * t.step, lane, elems);
    float v[NE];
    Row<DT>::V::unpack(raw, v);
    double w[NE];
    double sum = 0.0;
#pragma unroll
    for (uint32_t e = 0; e < NE; ++e) {
        w[e] = lane * NE + e < elems ? r.share(number_of(no_nan(v[e]))) : 0.0;
        sum += w[e];
    }
    double all;
    at += before(sum, s.part64, &all);
    if (threadIdx.x == 0) s.word[1] = 0;
    __syncthreads();
#pragma unroll
    for (uint32_t e = 0; e < NE; ++e) {
        if (w[e] > 0.0 && at <= aim) atomicMax(&s.word[1], threadIdx.x * NE + e + 1);
        at += w[e];
    }
    __syncthreads();
    const uint32_t place = s.word[1] - 1;
    if (place / NE != threadIdx.x) return;
#pragma unroll
    for (uint32_t e = 0; e < NE; ++e) {
        if (place % NE == e) write_choice(a, r, t.first + lane * NE + e, number_of(no_nan(v[e])), whole);
    }
}

template <int DT>
__global__ void __launch_bounds__(kThreads)
k_sample(SelectArgs a)
{
    constexpr uint32_t kMine = kList / kThreads;
    constexpr uint32_t kShift = kIdle<DT>;
    __shared__ Shared s;
    Row<DT> r(a, blockIdx.x);
    const RowChoice choice(a.choice, r.row, a.rows.vocab);
    const float u = a.choice.random[r.row];
    r.top = top_of(r, s);
    r.top_value = value_of(r.top);
    r.c = choice.c;
    if (r.top <= kLeast) {   // nothing to choose from
        if (threadIdx.x == 0) {
            a.choice.token[r.row] = -1;
            if (a.choice.logprob != nullptr) a.choice.logprob[r.row] = minus_infinity();
        }
        return;
    }
    if (!choice.by_k && !choice.by_p && !choice.by_min) {
        draw_all(a, r, s, u);
        return;
    }
    u64 p_of_whole = 0;   // the weight that top_p asks for, where it is of the whole row
    if (choice.by_p && !choice.by_k) {
        double mine = 0.0;
        for (uint32_t i = threadIdx.x; i < a.nruns; i += kThreads) {
            const Run run = a.runs[r.row * a.nruns + i];
            mine += run.most == static_cast<float>(r.top_value) ? run.sum : run.sum * exp2_exact((static_cast<double>(run.most) - r.top_value) * r.c);
        }
        double whole;
        (void)before(mine, s.part64, &whole);
        p_of_whole = choice.p > 0.0 ? static_cast<u64>(ceil(ldexp(choice.p * whole, static_cast<int>(a.bits)))) : 0;
    }
    if (!choice.by_k || choice.k <= HCCLX_TOP_MAX) {
        const uint32_t n = list_first(r, s, choice.by_k ? choice.k : min(kNucleus, a.rows.vocab));
        sort_list(s, n);
        const uint32_t limit = choice.by_k ? choice.k : n;
        u64 w[kMine];
        u64 sum = 0;
#pragma unroll
        for (uint32_t i = 0; i < kMine; ++i) {
            const uint32_t at = threadIdx.x * kMine + i;
            sum += w[i] = at < limit ? r.weight(static_cast<uint32_t>(s.list.sorted[at] >> 32)) : 0;
        }
        u64 whole;
        u64 at = before(sum, s.part[0], &whole);
        if (choice.by_k) p_of_whole = choice.p > 0.0 ? static_cast<u64>(ceil(choice.p * static_cast<double>(whole))) : 0;
        uint32_t keep = 0;
#pragma unroll
        for (uint32_t i = 0; i < kMine; ++i) {
            const uint32_t place = threadIdx.x * kMine + i;
            bool in = place < limit;
            if (choice.by_p) in = in && (place == 0 || at < p_of_whole);
            if (choice.by_min) in = in && (place == 0 || r.share(static_cast<uint32_t>(s.list.sorted[place] >> 32)) >= choice.least);
            keep += in;
            at += w[i];
        }
        uint32_t kept;
        (void)before(keep, s.part32[0], &kept);
        if (choice.by_k || kept < n || n == a.rows.vocab) {
            const u64 last = s.list.sorted[kept - 1];
            sum = 0;
#pragma unroll
            for (uint32_t i = 0; i < kMine; ++i) {
                const uint32_t place = threadIdx.x * kMine + i;
                const u64 x = place < n ? s.list.listed[place] : 0;
                sum += w[i] = place < n && x >= last ? r.weight(static_cast<uint32_t>(x >> 32)) : 0;
            }
            at = before(sum, s.part[0], &whole);
            const u64 aim = aim_of(u, whole);
#pragma unroll
            for (uint32_t i = 0; i < kMine; ++i) {
                if (aim >= at && aim - at < w[i]) {
                    const u64 x = s.list.listed[threadIdx.x * kMine + i];
                    write_choice(a, r, ~static_cast<uint32_t>(x), static_cast<uint32_t>(x >> 32), ldexp(static_cast<double>(whole), -static_cast<int>(a.bits)));
                }
                at += w[i];
            }
            return;
        }
        __syncthreads();   // the list makes room
    }
    // More stays than a list holds: the cut is searched among all elements.
    Kept stay = {0, 0xffffffffu, choice.by_min ? choice.least : 0.0};
    auto all = [&](auto &&f) { r.each(nullptr, r.ngroups, f); };
    Range range = {kLeast >> kShift, r.top >> kShift, 0, 0, 0, 0};
    uint32_t cut_count = 0;
    if (choice.by_k) {
        do {
            narrow<false>(range, s, all, [&](u64) { return u64(choice.k); });
        } while (range.low != range.high);
        stay.cut = range.low;
        stay.equal = choice.k - range.above;
        cut_count = range.inside;
    }
    if (choice.by_p) {
        range = {stay.cut > kLeast >> kShift ? stay.cut : kLeast >> kShift, r.top >> kShift, 0, 0, 0, 0};
        u64 aim = 0;
        bool first = true;
        // (what is equal to the cut of top_k and does not stay is at the end of the order)
        const u64 over = choice.by_k && cut_count > stay.equal ? (cut_count - stay.equal) * r.weight(stay.cut << kShift | (stay.cut >> (31 - kShift) != 0 ? 0 : (1u << kShift) - 1)) : 0;
        do {
            narrow<true>(range, s, all, [&](u64 whole) {
                if (first) {
                    aim = choice.by_k && choice.p > 0.0 ? static_cast<u64>(ceil(choice.p * static_cast<double>(whole - over))) : p_of_whole;
                    aim = max(u64(1), min(aim, whole));
                }
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
    if (threadIdx.x == 0) s.wide = 0;
    __syncthreads();
    draw_kept(a, r, s, stay, u);
}

// ---- host ------------------------------------------------------------------------------------------------------------------

struct SelectWork : PlanWork {
    SelectArgs args{};
    Table table;
    DeviceBlock scratch;   // most, runs
    int dtype = 0;
    bool sample = false;
    uint32_t parts = 1;    // workgroups of the first launch per row

    template <int DT, int U>
    void runs(hipStream_t st) const
    {
        const dim3 grid(args.rows.rows * parts), block(kRunWaves * 64);
        if (sample) {
            HCCLX_LAUNCH((k_logit_runs<DT, U, kRunChoice>), grid, block, 0, st, args, parts);
        } else if (args.lse != nullptr) {
            HCCLX_LAUNCH((k_logit_runs<DT, U, kRunSum>), grid, block, 0, st, args, parts);
        } else {
            HCCLX_LAUNCH((k_logit_runs<DT, U, kRunPlain>), grid, block, 0, st, args, parts);
        }
    }
    template <int DT>
    void run(hipStream_t st) const
    {
        switch (args.per_run) {
            case 1: runs<DT, 1>(st); break;
            case 2: runs<DT, 2>(st); break;
            case 4: runs<DT, 4>(st); break;
            default: runs<DT, 8>(st); break;
        }
        if (sample) {
            HCCLX_LAUNCH((k_sample<DT>), dim3(args.rows.rows), dim3(kThreads), 0, st, args);
        } else {
            HCCLX_LAUNCH((k_top_logits<DT>), dim3(args.rows.rows), dim3(kThreads), 0, st, args);
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
    // As many chunks per wavefront as leave every CU four workgroups.
    a.per_run = 8;
    auto parts = [&] { return (a.rows.nchunks + a.per_run * kRunWaves - 1) / (a.per_run * kRunWaves); };
    while (a.per_run > 1 && static_cast<uint64_t>(l.rows) * parts() < 4ull * static_cast<uint32_t>(ctx->num_cus)) a.per_run /= 2;
    w->parts = parts();
    if (static_cast<uint64_t>(l.rows) * w->parts * kRunWaves * 64 > 0xffffffffull) return fail(HCCL_E_PARA, "too many rows of so many columns");
    a.nruns = (a.rows.nchunks + a.per_run - 1) / a.per_run;
    a.bits = 62;
    for (uint64_t n = 1; n < vocab; n *= 2) --a.bits;
    const uint64_t runs = sums ? static_cast<uint64_t>(l.rows) * a.nruns * sizeof(Run) : 0;
    const uint32_t per = 64 * (16 / dtype_size(l.dtype)) / kGroup;
    const uint64_t most = static_cast<uint64_t>(l.rows) * a.rows.nchunks * per * sizeof(uint32_t);
    const uint64_t held = runs + most;
    if (held != 0 && (rc = w->scratch.get(held)) != HCCL_SUCCESS) return rc;
    a.runs = reinterpret_cast<Run *>(w->scratch.p);
    a.most = reinterpret_cast<uint32_t *>(w->scratch.p + runs);
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
