// Root-mean-square norm with the residual's addition, and its gradient (include/hcclx_ops.h: hcclx_rms_norm_*).
//
// Bound: HBM bandwidth.  A row is read into registers once, whatever follows: the total, its mean square, the largest
// result (8-bit rows) and the results all come from there.
#include "hcclx_internal.h"
#include "hcclx_ops.h"
#include "kernels/elem.h"
#include "kernels/fold.h"
#include "ops/lanes.h"

#include <algorithm>
#include <string>

using namespace hcclx;

namespace {

constexpr uint32_t kMostRanks = 64;
constexpr uint32_t kTail = HCCLX_ROW8_TAIL;

struct NormPtrs {
    const char *x[kMostRanks];
    const char *residual[kMostRanks];
    const char *weight[kMostRanks];
    char *total[kMostRanks];
    char *out[kMostRanks];
};
struct GradPtrs {
    const char *dy[kMostRanks];
    const char *total[kMostRanks];
    const char *weight[kMostRanks];
    const char *dtotal[kMostRanks];
    char *dx[kMostRanks];
};
struct OutPtrs {
    char *p[kMostRanks];
};

// A thread holds at most so many vectors of 16 bytes of a row.  (Two: 8 ranks x 4096 x 7168 to 8 bits 351 us instead of 305, in one
// run; 8 x 2048 x 4096 91 instead of 93, 8 x 64 x 7168 the same.)
constexpr uint32_t kMostVectors = 4;
constexpr uint32_t kGroup = 256;   // threads of a workgroup that holds several rows, at most
template <int DT> constexpr int kMostThreads = HCCLX_NORM_MAX_ROW / (Vec16<DT>::NE * kMostVectors);
static_assert(kMostThreads<HCCL_DATA_TYPE_FP32> <= 1024, "a workgroup holds the longest row");

// Vector v of a row of `elems` elements as it lies in memory; zeros behind the row's end.  WARM: it is read again (weights).
template <int DT, bool WARM>
__device__ __forceinline__ u32x4 load_vec(const char *row, uint32_t v, uint32_t elems)
{
    using V = Vec16<DT>;
    using S = typename V::S;
    const uint32_t at = v * V::NE;
    if (at + V::NE <= elems) {
        const char *p = row + static_cast<size_t>(v) * 16;
        return WARM ? ld16_cached(p) : __builtin_nontemporal_load(as_global(p));
    }
    S tmp[V::NE];
#pragma unroll
    for (int e = 0; e < V::NE; ++e) tmp[e] = at + e < elems ? reinterpret_cast<const S *>(row)[at + e] : S(0);
    u32x4 raw;
    __builtin_memcpy(&raw, tmp, 16);
    return raw;
}

template <int DT>
__device__ __forceinline__ void store_vec(char *row, uint32_t v, uint32_t elems, const float (&f)[Vec16<DT>::NE])
{
    using V = Vec16<DT>;
    using S = typename V::S;
    const uint32_t at = v * V::NE;
    if (at + V::NE <= elems) {
        st16(row + static_cast<size_t>(v) * 16, V::pack(f));
    } else {
#pragma unroll
        for (int e = 0; e < V::NE; ++e) {
            if (at + e < elems) reinterpret_cast<S *>(row)[at + e] = V::D::narrow(f[e]);
        }
    }
}

// Sums of N values over the threads of a row (blockDim.x of them, whole wavefronts), or the largest of N magnitudes.  s: N floats per
// wavefront of the workgroup, of which no reader is left.
template <bool MAX, int N>
__device__ __forceinline__ void row_reduce(float (&v)[N], float (*s)[N])
{
#pragma unroll
    for (int k = 0; k < N; ++k) v[k] = MAX ? wave_max(v[k]) : wave_sum(v[k]);
    const uint32_t waves = blockDim.x / 64;
    if (waves == 1) return;
    float(*mine)[N] = s + threadIdx.y * waves;
    if ((threadIdx.x & 63) == 0) {
#pragma unroll
        for (int k = 0; k < N; ++k) mine[threadIdx.x / 64][k] = v[k];
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < N; ++k) v[k] = mine[0][k];
    for (uint32_t w = 1; w < waves; ++w) {
#pragma unroll
        for (int k = 0; k < N; ++k) v[k] = MAX ? fmaxf(v[k], mine[w][k]) : v[k] + mine[w][k];
    }
}

// A row per blockDim.x threads and no second row: what a workgroup waits for, others have on their way.  bf16, 8 ranks x 4096 x 7168
// with residual and 8-bit rows 285 us (5.8 TB/s), 8 x 2048 x 4096 in 16 bits 93 us (5.8).  8 x 64 x 7168 to 8 bits 10 us with the rows
// in the last-level cache, 13 from memory (2.0 TB/s), in 16 bits 10: neither the bytes nor one trip to memory make that up; the chain
// of a rank's addresses, its rows and two reductions has not been taken apart.
template <int DT, bool QUANT, int NV>
__global__ void __launch_bounds__(kMostThreads<DT>)
k_rms_norm(NormPtrs ptrs, uint32_t rows, uint32_t elems, float eps)
{
    using V = Vec16<DT>;
    constexpr int NE = V::NE;
    __shared__ float s_part[2][16][1];
    const uint32_t rank = blockIdx.y;
    const uint32_t row = blockIdx.x * blockDim.y + threadIdx.y;
    const bool live = row < rows;
    const size_t at = static_cast<size_t>(live ? row : rows - 1) * elems * sizeof(typename V::S);   // behind the last: it again, unstored
    const char *x = ptrs.x[rank] + at;
    const char *residual = ptrs.residual[rank];
    char *total = ptrs.total[rank];
    u32x4 w[NV];
    float t[NV][NE];
    float square[1] = {0.0f};
    {   // everything that is read, together: small launches are little more than this round trip
        u32x4 rx[NV], rr[NV];
#pragma unroll
        for (int i = 0; i < NV; ++i) rx[i] = load_vec<DT, false>(x, threadIdx.x + i * blockDim.x, elems);
        if (residual != nullptr) {
#pragma unroll
            for (int i = 0; i < NV; ++i) rr[i] = load_vec<DT, false>(residual + at, threadIdx.x + i * blockDim.x, elems);
        }
#pragma unroll
        for (int i = 0; i < NV; ++i) w[i] = load_vec<DT, true>(ptrs.weight[rank], threadIdx.x + i * blockDim.x, elems);
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            V::unpack(rx[i], t[i]);
            if (residual != nullptr) {
                float r[NE];
                V::unpack(rr[i], r);
#pragma unroll
                for (int e = 0; e < NE; ++e) t[i][e] = V::D::widen(V::D::narrow(t[i][e] + r[e]));
            }
        }
    }
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        if (total != nullptr && live) store_vec<DT>(total + at, threadIdx.x + i * blockDim.x, elems, t[i]);
#pragma unroll
        for (int e = 0; e < NE; ++e) square[0] += t[i][e] * t[i][e];
    }
    row_reduce<false, 1>(square, s_part[0]);
    const float r = 1.0f / sqrtf(square[0] / static_cast<float>(elems) + eps);
    float most[1] = {0.0f};
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        float f[NE];
        V::unpack(w[i], f);
#pragma unroll
        for (int e = 0; e < NE; ++e) {
            t[i][e] = t[i][e] * r * f[e];
            if (QUANT) most[0] = fmaxf(most[0], fabsf(t[i][e]));
        }
    }
    if constexpr (QUANT) {
        row_reduce<true, 1>(most, s_part[1]);
        if (!live) return;
        const CodeScale code(most[0]);
        char *out = ptrs.out[rank] + static_cast<size_t>(row) * (elems + kTail);
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const uint32_t v = threadIdx.x + i * blockDim.x;
            if (v * NE >= elems) continue;   // (elems is a multiple of 16 here: no vector is cut)
#pragma unroll
            for (int q = 0; q < NE / 4; ++q) {
                const uint32_t c = to_e4m3(code(t[i][4 * q]), code(t[i][4 * q + 1]), code(t[i][4 * q + 2]), code(t[i][4 * q + 3]));
                reinterpret_cast<uint32_t *>(out)[v * (NE / 4) + q] = c;
            }
        }
        if (threadIdx.x == 0) {
            const u32x4 tail = {__float_as_uint(code.scale), 0u, 0u, 0u};
            st16(out + elems, tail);
        }
    } else if (live) {
#pragma unroll
        for (int i = 0; i < NV; ++i) store_vec<DT>(ptrs.out[rank] + at, threadIdx.x + i * blockDim.x, elems, t[i]);
    }
}

// Slot s of a rank (threadIdx.y of a workgroup) takes the rows s, s + slots, ...; it adds up its part of dweight in registers
// and the workgroup writes the sum of its slots' to partial[rank][workgroup][elems].  AHEAD: a row is read while the one before it is
// computed (dtotal, which is wanted last, when its turn begins: ahead too it has no registers).  With x = total and
// r = 1 / sqrt(mean x^2 + eps):
// dx = r (dy w - x r^2 mean(x dy w)) + dtotal,  dw = sum over the rows of dy x r.
// Bound: how many rows are on their way, four workgroups of 256 threads per CU at 128 registers.  bf16, 8 ranks x 2048 x 4096 108 us
// (5.0 TB/s; two workgroups per CU 163, three 137; dtotal ahead 123).
template <int DT, int NV, bool AHEAD>
__global__ void __launch_bounds__(AHEAD ? 1024 : kMostThreads<DT>)
k_rms_norm_grad(GradPtrs ptrs, uint32_t rows, uint32_t elems, float eps, float *partial)
{
    using V = Vec16<DT>;
    constexpr int NE = V::NE;
    __shared__ float s_part[2][16][2];   // of the rows in turn
    __shared__ float s_join[NE][kGroup];
    const uint32_t rank = blockIdx.y;
    const uint32_t slots = gridDim.x * blockDim.y;
    const char *dtotal = ptrs.dtotal[rank];
    const char *dys = ptrs.dy[rank];
    const char *totals = ptrs.total[rank];
    float acc[NV][NE];
    u32x4 w[NV], rt[NV], ra[NV];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
#pragma unroll
        for (int e = 0; e < NE; ++e) acc[i][e] = 0.0f;
    }
    auto read = [&](uint32_t row) {   // (behind the last row: it again)
        const size_t at = static_cast<size_t>(row < rows ? row : rows - 1) * elems * sizeof(typename V::S);
#pragma unroll
        for (int i = 0; i < NV; ++i) rt[i] = load_vec<DT, false>(totals + at, threadIdx.x + i * blockDim.x, elems);
#pragma unroll
        for (int i = 0; i < NV; ++i) ra[i] = load_vec<DT, false>(dys + at, threadIdx.x + i * blockDim.x, elems);
    };
    read(blockIdx.x * blockDim.y + threadIdx.y);
#pragma unroll
    for (int i = 0; i < NV; ++i) w[i] = load_vec<DT, true>(ptrs.weight[rank], threadIdx.x + i * blockDim.x, elems);
    uint32_t turn = 0;
    // as many turns for every slot of a workgroup: they meet at barriers
    for (uint32_t first = blockIdx.x * blockDim.y; first < rows; first += slots, turn ^= 1) {
        const uint32_t row = first + threadIdx.y;
        const bool live = row < rows;
        const size_t at = static_cast<size_t>(live ? row : rows - 1) * elems * sizeof(typename V::S);
        // (the row stays as it was read and is widened twice: in 16 bits that is half the registers)
        u32x4 ct[NV], ca[NV], cd[NV];
        float sums[2] = {0.0f, 0.0f};   // of total^2 and of total * dy * weight
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            ct[i] = rt[i];
            ca[i] = ra[i];
        }
        if (dtotal != nullptr) {
#pragma unroll
            for (int i = 0; i < NV; ++i) cd[i] = load_vec<DT, false>(dtotal + at, threadIdx.x + i * blockDim.x, elems);
        }
        if (AHEAD && first + slots < rows) read(row + slots);
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            float f[NE], t[NE], g[NE];
            V::unpack(w[i], f);
            V::unpack(ct[i], t);
            V::unpack(ca[i], g);
#pragma unroll
            for (int e = 0; e < NE; ++e) {
                sums[0] += t[e] * t[e];
                sums[1] += t[e] * (g[e] * f[e]);
            }
        }
        row_reduce<false, 2>(sums, s_part[turn]);
        const float r = 1.0f / sqrtf(sums[0] / static_cast<float>(elems) + eps);
        const float c = (r * r) * (sums[1] / static_cast<float>(elems));
        if (live) {
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                float f[NE], t[NE], g[NE], d[NE];
                asm("" : "+v"(ct[i]), "+v"(ca[i]));   // widened again, not kept
                V::unpack(w[i], f);
                V::unpack(ct[i], t);
                V::unpack(ca[i], g);
                if (dtotal != nullptr) V::unpack(cd[i], d);
#pragma unroll
                for (int e = 0; e < NE; ++e) {
                    acc[i][e] += g[e] * (t[e] * r);
                    const float x = r * (g[e] * f[e] - t[e] * c);
                    d[e] = dtotal != nullptr ? x + d[e] : x;
                }
                store_vec<DT>(ptrs.dx[rank] + at, threadIdx.x + i * blockDim.x, elems, d);
            }
        }
        if (!AHEAD && first + slots < rows) read(row + slots);
    }
    if (partial == nullptr) return;
    if (blockDim.y > 1) {   // the workgroup's slots first, in their order
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            __syncthreads();
#pragma unroll
            for (int e = 0; e < NE; ++e) s_join[e][threadIdx.y * blockDim.x + threadIdx.x] = acc[i][e];
            __syncthreads();
            if (threadIdx.y != 0) continue;
            for (uint32_t y = 1; y < blockDim.y; ++y) {
#pragma unroll
                for (int e = 0; e < NE; ++e) acc[i][e] += s_join[e][y * blockDim.x + threadIdx.x];
            }
        }
        if (threadIdx.y != 0) return;
    }
    float *mine = partial + (static_cast<size_t>(rank) * gridDim.x + blockIdx.x) * elems;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const uint32_t at = (threadIdx.x + i * blockDim.x) * NE;
#pragma unroll
        for (int e = 0; e < NE; ++e) {
            if (at + e < elems) mine[at + e] = acc[i][e];
        }
    }
}

// dweight = the workgroups' parts, added in their order: 64 columns per workgroup, every 16th part per row of threads, then the rows.
template <int DT>
__global__ void __launch_bounds__(1024)
k_rms_norm_join(OutPtrs dweight, uint32_t parts, uint32_t elems, const float *partial)
{
    using D = DTypeOf<DT>;
    __shared__ float s_sum[16][64];
    const uint32_t rank = blockIdx.y;
    const uint32_t col = blockIdx.x * 64 + threadIdx.x;
    float sum = 0.0f;
    if (col < elems) {
        const float *p = partial + static_cast<size_t>(rank) * parts * elems + col;
#pragma unroll 8
        for (uint32_t s = threadIdx.y; s < parts; s += 16) sum += p[static_cast<size_t>(s) * elems];
    }
    s_sum[threadIdx.y][threadIdx.x] = sum;
    __syncthreads();
    if (threadIdx.y != 0 || col >= elems) return;
    for (uint32_t y = 1; y < 16; ++y) sum += s_sum[y][threadIdx.x];
    reinterpret_cast<typename D::S *>(dweight.p[rank])[col] = D::narrow(sum);
}

// Threads per row and vectors per thread: a row is held by as few wavefronts as leave a thread at most so many vectors of it (1024
// threads: more), one, two or a multiple of four of them, one for every SIMD (five: gradient of 8 x 1024 x 4097 bf16 137 us, eight
// 108); workgroups of short rows hold several.  The norm takes four; its gradient, which holds three rows, the next
// ones and a part of dweight, two.
struct RowShape {
    uint32_t threads;
    uint32_t per_group;
    uint32_t vectors;
    uint64_t groups(uint64_t rows) const { return (rows + per_group - 1) / per_group; }
};
RowShape shape_of(uint32_t elems, int ne, uint32_t most_vectors)
{
    const uint32_t vecs = (elems + ne - 1) / ne;
    uint32_t threads = 64;
    while (threads < 1024 && threads * most_vectors < vecs) threads += std::min(threads, kGroup);
    return {threads, std::max(1u, kGroup / threads), (vecs + threads - 1) / threads};
}

template <int DT, bool QUANT>
void launch_norm(const RowShape &s, dim3 grid, hipStream_t st, const NormPtrs &p, uint32_t rows, uint32_t elems, float eps)
{
    const dim3 block(s.threads, s.per_group);
    switch (s.vectors) {
        case 1: HCCLX_LAUNCH((k_rms_norm<DT, QUANT, 1>), grid, block, 0, st, p, rows, elems, eps); break;
        case 2: HCCLX_LAUNCH((k_rms_norm<DT, QUANT, 2>), grid, block, 0, st, p, rows, elems, eps); break;
        case 3: HCCLX_LAUNCH((k_rms_norm<DT, QUANT, 3>), grid, block, 0, st, p, rows, elems, eps); break;
        default: HCCLX_LAUNCH((k_rms_norm<DT, QUANT, 4>), grid, block, 0, st, p, rows, elems, eps); break;
    }
}

template <int DT>
void launch_grad(const RowShape &s, dim3 grid, hipStream_t st, const GradPtrs &p, uint32_t rows, uint32_t elems, float eps, float *partial)
{
    const dim3 block(s.threads, s.per_group);
    if (s.vectors == 1) {
        HCCLX_LAUNCH((k_rms_norm_grad<DT, 1, true>), grid, block, 0, st, p, rows, elems, eps, partial);
    } else if (s.vectors == 2) {
        HCCLX_LAUNCH((k_rms_norm_grad<DT, 2, true>), grid, block, 0, st, p, rows, elems, eps, partial);
    } else if constexpr (Vec16<DT>::NE == 4) {   // 32-bit rows that 1024 threads hold with four vectors each
        HCCLX_LAUNCH((k_rms_norm_grad<DT, 4, false>), grid, block, 0, st, p, rows, elems, eps, partial);
    }
}

struct NormWork : PlanWork {
    NormPtrs ptrs{};
    uint32_t n = 0, rows = 0, elems = 0;
    int dtype = 0;
    bool quant = false;
    float eps = 0.0f;
    RowShape shape{};

    int launch(const DeviceCtx *, hipStream_t st) const override
    {
        if (rows == 0) return HCCL_SUCCESS;
        const dim3 grid(static_cast<uint32_t>(shape.groups(rows)), n);
        if (dtype == HCCL_DATA_TYPE_FP32) {
            quant ? launch_norm<HCCL_DATA_TYPE_FP32, true>(shape, grid, st, ptrs, rows, elems, eps)
                  : launch_norm<HCCL_DATA_TYPE_FP32, false>(shape, grid, st, ptrs, rows, elems, eps);
        } else if (dtype == HCCL_DATA_TYPE_FP16) {
            quant ? launch_norm<HCCL_DATA_TYPE_FP16, true>(shape, grid, st, ptrs, rows, elems, eps)
                  : launch_norm<HCCL_DATA_TYPE_FP16, false>(shape, grid, st, ptrs, rows, elems, eps);
        } else {
            quant ? launch_norm<HCCL_DATA_TYPE_BFP16, true>(shape, grid, st, ptrs, rows, elems, eps)
                  : launch_norm<HCCL_DATA_TYPE_BFP16, false>(shape, grid, st, ptrs, rows, elems, eps);
        }
        const hipError_t e = hipGetLastError();
        return e == hipSuccess ? HCCL_SUCCESS : fail_hip(e, "norm kernel");
    }
};

struct NormGradWork : PlanWork {
    GradPtrs ptrs{};
    OutPtrs dweight{};
    bool want_dweight = false;
    uint32_t n = 0, rows = 0, elems = 0, groups = 0;
    int dtype = 0;
    float eps = 0.0f;
    RowShape shape{};
    DeviceBlock partial;   // float[n][groups][elems]

    template <int DT>
    void run(hipStream_t st) const
    {
        float *part = reinterpret_cast<float *>(partial.p);
        if (rows != 0) launch_grad<DT>(shape, dim3(groups, n), st, ptrs, rows, elems, eps, part);
        if (want_dweight) {
            HCCLX_LAUNCH((k_rms_norm_join<DT>), dim3((elems + 63) / 64, n), dim3(64, 16), 0, st, dweight, rows != 0 ? groups : 0u, elems, part);
        }
    }

    int launch(const DeviceCtx *, hipStream_t st) const override
    {
        if (dtype == HCCL_DATA_TYPE_FP32) {
            run<HCCL_DATA_TYPE_FP32>(st);
        } else if (dtype == HCCL_DATA_TYPE_FP16) {
            run<HCCL_DATA_TYPE_FP16>(st);
        } else {
            run<HCCL_DATA_TYPE_BFP16>(st);
        }
        const hipError_t e = hipGetLastError();
        return e == hipSuccess ? HCCL_SUCCESS : fail_hip(e, "norm gradient kernels");
    }
};

int check_norm(uint32_t n, uint32_t row_elems, int dtype)
{
    if (n == 0 || n > kMostRanks) return fail(HCCL_E_PARA, "rank count outside 1.." + std::to_string(kMostRanks));
    if (row_elems == 0 || row_elems > HCCLX_NORM_MAX_ROW) {
        return fail(HCCL_E_PARA, "row length outside 1.." + std::to_string(HCCLX_NORM_MAX_ROW));
    }
    if (dtype != HCCL_DATA_TYPE_FP32 && dtype != HCCL_DATA_TYPE_FP16 && dtype != HCCL_DATA_TYPE_BFP16) {
        return fail(HCCL_E_NOT_SUPPORT, "the norm takes fp32, fp16 or bf16");
    }
    return HCCL_SUCCESS;
}

// n pointers aligned to `align`; in == nullptr is refused unless `optional`.
template <typename P, typename Q>
int take(P *const *in, uint32_t n, uint64_t align, bool optional, const char *what, Q **out)
{
    if (in == nullptr) return optional ? HCCL_SUCCESS : fail(HCCL_E_PTR, std::string(what) + " pointer array is null");
    for (uint32_t i = 0; i < n; ++i) {
        if (in[i] == nullptr) return fail(HCCL_E_PTR, std::string(what) + "[" + std::to_string(i) + "] is null");
        if (reinterpret_cast<uint64_t>(in[i]) % align != 0) {
            return fail(HCCL_E_PARA, std::string(what) + "[" + std::to_string(i) + "] is not aligned to " + std::to_string(align) + " bytes");
        }
        out[i] = static_cast<Q *>(static_cast<P *>(in[i]));
    }
    return HCCL_SUCCESS;
}

// Rows and ranks run in any order and at once, so what a launch writes may lie on what it reads only where nobody else reads it: `own`
// says whether rank i's may lie on that rank's part, given how far behind it begins.  to: n pointers to `bytes` each, from (may be
// all null): n to `from_bytes`.
template <typename Own>
int check_apart(uint32_t n, const char *to_what, char *const *to, uint64_t bytes, const char *from_what, const char *const *from,
                uint64_t from_bytes, Own &&own)
{
    if (to[0] == nullptr || from[0] == nullptr) return HCCL_SUCCESS;
    for (uint32_t i = 0; i < n; ++i) {
        for (uint32_t j = 0; j < n; ++j) {
            const uint64_t t = reinterpret_cast<uint64_t>(to[i]);
            const uint64_t f = reinterpret_cast<uint64_t>(from[j]);
            if (t >= f + from_bytes || f >= t + bytes || (i == j && own(t - f))) continue;
            return fail(HCCL_E_PARA, std::string(to_what) + "[" + std::to_string(i) + "] overlaps " + from_what + "[" + std::to_string(j) +
                                         "], which others read or write");
        }
    }
    return HCCL_SUCCESS;
}

int make_norm(const hcclx_rms_norm_t &a, hcclx_plan_t **plan)
{
    int rc = check_norm(a.n, a.row_elems, a.dtype);
    if (rc != HCCL_SUCCESS) return rc;
    const bool quant = a.out_dtype == HCCL_DATA_TYPE_FP8E4M3;
    if (!quant && a.out_dtype != a.dtype) return fail(HCCL_E_NOT_SUPPORT, "out has the rows' type or HCCL_DATA_TYPE_FP8E4M3");
    if (quant && a.row_elems % 16 != 0) return fail(HCCL_E_PARA, "8-bit rows are multiples of 16 elements");
    auto w = std::make_unique<NormWork>();
    const uint64_t size = dtype_size(a.dtype);
    w->shape = shape_of(a.row_elems, 16 / static_cast<int>(size), kMostVectors);
    if (w->shape.groups(a.rows) * w->shape.threads > 0xffffffffull) return fail(HCCL_E_PARA, "too many rows");   // of a launch along x
    if ((rc = take(a.x, a.n, size, false, "x", w->ptrs.x)) != HCCL_SUCCESS) return rc;
    if ((rc = take(a.residual, a.n, size, true, "residual", w->ptrs.residual)) != HCCL_SUCCESS) return rc;
    if ((rc = take(a.weight, a.n, size, false, "weight", w->ptrs.weight)) != HCCL_SUCCESS) return rc;
    if ((rc = take(a.total, a.n, size, true, "total", w->ptrs.total)) != HCCL_SUCCESS) return rc;
    if ((rc = take(a.out, a.n, quant ? 16 : size, false, "out", w->ptrs.out)) != HCCL_SUCCESS) return rc;
    DeviceCtx *ctx = device_ctx();
    if (!ctx) return HCCL_E_RUNTIME;
    if (a.rows != 0) {
        const uint64_t row = a.row_elems * size;
        const uint64_t bytes = a.rows * row;
        const uint64_t out_bytes = quant ? static_cast<uint64_t>(a.rows) * (a.row_elems + kTail) : bytes;
        const NormPtrs &p = w->ptrs;
        // a row's threads have read all of it before the first of them writes out, but not before total; rows of out begin where those
        // of x do unless they are of 8 bits
        const bool one = a.rows == 1;
        const auto out_on_rows = [&](uint64_t behind) { return one || (!quant && behind == 0); };
        const auto out_on_total = [&](uint64_t behind) { return !quant && behind == 0; };   // out is what stays
        const auto out_on_weight = [&](uint64_t) { return one; };
        const auto total_on_rows = [](uint64_t behind) { return behind == 0; };
        const auto total_on_weight = [&](uint64_t behind) { return one && behind == 0; };
        if ((rc = check_apart(a.n, "out", p.out, out_bytes, "x", p.x, bytes, out_on_rows)) != HCCL_SUCCESS) return rc;
        if ((rc = check_apart(a.n, "out", p.out, out_bytes, "residual", p.residual, bytes, out_on_rows)) != HCCL_SUCCESS) return rc;
        if ((rc = check_apart(a.n, "out", p.out, out_bytes, "weight", p.weight, row, out_on_weight)) != HCCL_SUCCESS) return rc;
        if ((rc = check_apart(a.n, "out", p.out, out_bytes, "total", p.total, bytes, out_on_total)) != HCCL_SUCCESS) return rc;
        if ((rc = check_apart(a.n, "total", p.total, bytes, "x", p.x, bytes, total_on_rows)) != HCCL_SUCCESS) return rc;
        if ((rc = check_apart(a.n, "total", p.total, bytes, "residual", p.residual, bytes, total_on_rows)) != HCCL_SUCCESS) return rc;
        if ((rc = check_apart(a.n, "total", p.total, bytes, "weight", p.weight, row, total_on_weight)) != HCCL_SUCCESS) return rc;
    }
    w->n = a.n;
    w->rows = a.rows;
    w->elems = a.row_elems;
    w->dtype = a.dtype;
    w->quant = quant;
    w->eps = a.eps;
    const uint64_t elements = static_cast<uint64_t>(a.n) * a.rows * a.row_elems;
    const uint64_t algo = elements * (size * (1 + (a.residual != nullptr) + (a.total != nullptr)) + (quant ? 1 : size));
    return plan_of(ctx, std::move(w), algo, 0, plan);
}

int make_norm_grad(const hcclx_rms_norm_grad_t &a, hcclx_plan_t **plan)
{
    int rc = check_norm(a.n, a.row_elems, a.dtype);
    if (rc != HCCL_SUCCESS) return rc;
    auto w = std::make_unique<NormGradWork>();
    const uint64_t size = dtype_size(a.dtype);
    if ((rc = take(a.dy, a.n, size, false, "dy", w->ptrs.dy)) != HCCL_SUCCESS) return rc;
    if ((rc = take(a.total, a.n, size, false, "total", w->ptrs.total)) != HCCL_SUCCESS) return rc;
    if ((rc = take(a.weight, a.n, size, false, "weight", w->ptrs.weight)) != HCCL_SUCCESS) return rc;
    if ((rc = take(a.dtotal, a.n, size, true, "dtotal", w->ptrs.dtotal)) != HCCL_SUCCESS) return rc;
    if ((rc = take(a.dx, a.n, size, false, "dx", w->ptrs.dx)) != HCCL_SUCCESS) return rc;
    if ((rc = take(a.dweight, a.n, size, true, "dweight", w->dweight.p)) != HCCL_SUCCESS) return rc;
    DeviceCtx *ctx = device_ctx();
    if (!ctx) return HCCL_E_RUNTIME;
    if (a.rows != 0) {
        const uint64_t row = a.row_elems * size;
        const uint64_t bytes = a.rows * row;
        const GradPtrs &p = w->ptrs;
        const auto on_rows = [](uint64_t behind) { return behind == 0; };
        const auto on_weight = [&](uint64_t behind) { return a.rows == 1 && behind == 0; };
        if ((rc = check_apart(a.n, "dx", p.dx, bytes, "dy", p.dy, bytes, on_rows)) != HCCL_SUCCESS) return rc;
        if ((rc = check_apart(a.n, "dx", p.dx, bytes, "total", p.total, bytes, on_rows)) != HCCL_SUCCESS) return rc;
        if ((rc = check_apart(a.n, "dx", p.dx, bytes, "dtotal", p.dtotal, bytes, on_rows)) != HCCL_SUCCESS) return rc;
        if ((rc = check_apart(a.n, "dx", p.dx, bytes, "weight", p.weight, row, on_weight)) != HCCL_SUCCESS) return rc;
    }
    w->want_dweight = a.dweight != nullptr;
    w->n = a.n;
    w->rows = a.rows;
    w->elems = a.row_elems;
    w->dtype = a.dtype;
    w->eps = a.eps;
    w->shape = shape_of(a.row_elems, 16 / static_cast<int>(size), 2);
    const uint32_t most = static_cast<uint32_t>(w->shape.groups(a.rows));
    // A workgroup takes four rows at least, while there are workgroups for every CU: its part of dweight is as long as a row of floats
    // (8 ranks x 256 x 4096 bf16, two rows 32 us, four 25; 3 x 777 x 1001 fp32, two at a time, four 15.7, eight 20.7).  Four workgroups
    // per CU: of 256 threads a CU holds as many; of longer rows' the others follow (8 x 1024 x 8192 118 us, as many as it holds 131).
    w->groups = std::min(std::max(a.rows / 4 + (a.rows % 4 != 0), std::min(most, ctx->num_cus / a.n)), std::max(1u, 4u * ctx->num_cus / a.n));
    if (a.rows > 0xffffffffu - w->groups * w->shape.per_group) return fail(HCCL_E_PARA, "too many rows");   // a slot's next row has 32 bits
    uint64_t held = 0;
    if (w->want_dweight && a.rows != 0) {
        held = static_cast<uint64_t>(a.n) * w->groups * a.row_elems * sizeof(float);
        if ((rc = w->partial.get(held)) != HCCL_SUCCESS) return rc;
    }
    const uint64_t elements = static_cast<uint64_t>(a.n) * a.rows * a.row_elems;
    return plan_of(ctx, std::move(w), elements * size * (3 + (a.dtotal != nullptr)), held, plan);
}

}  // namespace

extern "C" {

int hcclx_rms_norm_plan_create(const hcclx_rms_norm_t *norm, hcclx_plan_t **plan)
{
    if (plan == nullptr) return fail(HCCL_E_PTR, "plan is null");
    *plan = nullptr;
    if (norm == nullptr) return fail(HCCL_E_PTR, "norm is null");
    return guarded([&] { return make_norm(*norm, plan); });
}

int hcclx_rms_norm_grad_plan_create(const hcclx_rms_norm_grad_t *norm, hcclx_plan_t **plan)
{
    if (plan == nullptr) return fail(HCCL_E_PTR, "plan is null");
    *plan = nullptr;
    if (norm == nullptr) return fail(HCCL_E_PTR, "norm is null");
    return guarded([&] { return make_norm_grad(*norm, plan); });
}

}  // extern "C"
