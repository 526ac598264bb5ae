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

// A thread holds at most so many vectors of 16 bytes of a row.
constexpr uint32_t kMostVectors = 4;
template <int DT> constexpr int kMostThreads = HCCLX_NORM_MAX_ROW / (Vec16<DT>::NE * kMostVectors);
static_assert(kMostThreads<HCCL_DATA_TYPE_FP32> <= 1024, "a workgroup holds the longest row");

// Vector v of a row of `elems` elements as 32-bit floats; zeros behind the row's end.
template <int DT>
__device__ __forceinline__ void load_vec(const char *row, uint32_t v, uint32_t elems, float (&f)[Vec16<DT>::NE])
{
    using V = Vec16<DT>;
    using S = typename V::S;
    const uint32_t at = v * V::NE;
    if (at + V::NE <= elems) {
        V::unpack(ld16_cached(row + static_cast<size_t>(v) * 16), f);
    } else {
#pragma unroll
        for (int e = 0; e < V::NE; ++e) f[e] = at + e < elems ? V::D::widen(reinterpret_cast<const S *>(row)[at + e]) : 0.0f;
    }
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

// Sum / maximum over the threads of a row (blockDim.x of them, whole wavefronts).  s: one float per wavefront of the workgroup.
template <bool MAX>
__device__ __forceinline__ float row_reduce(float v, float *s)
{
    v = MAX ? wave_max(v) : wave_sum(v);
    const uint32_t waves = blockDim.x / 64;
    if (waves == 1) return v;
    float *mine = s + threadIdx.y * waves;
    __syncthreads();   // the last reduction's values have been read
    if ((threadIdx.x & 63) == 0) mine[threadIdx.x / 64] = v;
    __syncthreads();
    v = mine[0];
    for (uint32_t w = 1; w < waves; ++w) v = MAX ? fmaxf(v, mine[w]) : v + mine[w];
    return v;
}

template <int DT, bool QUANT, int NV>
__global__ void __launch_bounds__(kMostThreads<DT>)
k_rms_norm(NormPtrs ptrs, uint32_t rows, uint32_t elems, float eps)
{
    using V = Vec16<DT>;
    constexpr int NE = V::NE;
    __shared__ float s_part[16];
    const uint32_t rank = blockIdx.y;
    const uint32_t row = blockIdx.x * blockDim.y + threadIdx.y;
    const bool live = row < rows;
    const size_t at = static_cast<size_t>(live ? row : rows - 1) * elems * sizeof(typename V::S);   // behind the last: it again, unstored
    const char *x = ptrs.x[rank] + at;
    const char *residual = ptrs.residual[rank];
    char *total = ptrs.total[rank];
    float t[NV][NE];
    float square = 0.0f;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const uint32_t v = threadIdx.x + i * blockDim.x;
        load_vec<DT>(x, v, elems, t[i]);
        if (residual != nullptr) {
            float r[NE];
            load_vec<DT>(residual + at, v, elems, r);
#pragma unroll
            for (int e = 0; e < NE; ++e) t[i][e] = V::D::widen(V::D::narrow(t[i][e] + r[e]));
        }
    }
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        if (total != nullptr && live) store_vec<DT>(total + at, threadIdx.x + i * blockDim.x, elems, t[i]);
#pragma unroll
        for (int e = 0; e < NE; ++e) square += t[i][e] * t[i][e];
    }
    square = row_reduce<false>(square, s_part);
    const float r = 1.0f / sqrtf(square / static_cast<float>(elems) + eps);
    float most = 0.0f;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        float w[NE];
        load_vec<DT>(ptrs.weight[rank], threadIdx.x + i * blockDim.x, elems, w);
#pragma unroll
        for (int e = 0; e < NE; ++e) {
            t[i][e] = t[i][e] * r * w[e];
            if (QUANT) most = fmaxf(most, fabsf(t[i][e]));
        }
    }
    if constexpr (QUANT) {
        most = row_reduce<true>(most, s_part);
        if (!live) return;
        const CodeScale code(most);
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
// and writes it to partial[rank][slot][elems].
template <int DT, int NV>
__global__ void __launch_bounds__(kMostThreads<DT>)
k_rms_norm_grad(GradPtrs ptrs, uint32_t rows, uint32_t elems, float eps, float *partial)
{
    using V = Vec16<DT>;
    constexpr int NE = V::NE;
    __shared__ float s_part[2][16];
    const uint32_t rank = blockIdx.y;
    const uint32_t slots = gridDim.x * blockDim.y;
    const uint32_t slot = blockIdx.x * blockDim.y + threadIdx.y;
    const char *dtotal = ptrs.dtotal[rank];
    float acc[NV][NE];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
#pragma unroll
        for (int e = 0; e < NE; ++e) acc[i][e] = 0.0f;
    }
    // as many turns for every slot of a workgroup: they meet at barriers
    for (uint32_t first = blockIdx.x * blockDim.y; first < rows; first += slots) {
        const uint32_t row = first + threadIdx.y;
        const bool live = row < rows;
        const size_t at = static_cast<size_t>(live ? row : rows - 1) * elems * sizeof(typename V::S);
        float t[NV][NE];
        float a[NV][NE];
        float square = 0.0f;
        float dot = 0.0f;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            load_vec<DT>(ptrs.total[rank] + at, threadIdx.x + i * blockDim.x, elems, t[i]);
            load_vec<DT>(ptrs.dy[rank] + at, threadIdx.x + i * blockDim.x, elems, a[i]);
        }
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            float w[NE];
            load_vec<DT>(ptrs.weight[rank], threadIdx.x + i * blockDim.x, elems, w);
#pragma unroll
            for (int e = 0; e < NE; ++e) {
                square += t[i][e] * t[i][e];
                dot += t[i][e] * (a[i][e] * w[e]);
            }
        }
        square = row_reduce<false>(square, s_part[0]);
        dot = row_reduce<false>(dot, s_part[1]);
        const float r = 1.0f / sqrtf(square / static_cast<float>(elems) + eps);
        const float c = (r * r) * (dot / static_cast<float>(elems));
        if (!live) continue;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const uint32_t v = threadIdx.x + i * blockDim.x;
            float w[NE];
            load_vec<DT>(ptrs.weight[rank], v, elems, w);
            float d[NE];
#pragma unroll
            for (int e = 0; e < NE; ++e) {
                acc[i][e] += a[i][e] * (t[i][e] * r);
                d[e] = r * (a[i][e] * w[e] - t[i][e] * c);
            }
            if (dtotal != nullptr) {
                float more[NE];
                load_vec<DT>(dtotal + at, v, elems, more);
#pragma unroll
                for (int e = 0; e < NE; ++e) d[e] += more[e];
            }
            store_vec<DT>(ptrs.dx[rank] + at, v, elems, d);
        }
    }
    if (partial == nullptr) return;
    char *mine = reinterpret_cast<char *>(partial + (static_cast<size_t>(rank) * slots + slot) * elems);
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const uint32_t at = (threadIdx.x + i * blockDim.x) * NE;
#pragma unroll
        for (int e = 0; e < NE; ++e) {
            if (at + e < elems) reinterpret_cast<float *>(mine)[at + e] = acc[i][e];
        }
    }
}

// dweight = the slots' parts, added in their order: 64 columns per workgroup, every 16th slot per row of threads, then the rows.
template <int DT>
__global__ void __launch_bounds__(1024)
k_rms_norm_join(OutPtrs dweight, uint32_t slots, uint32_t elems, const float *partial)
{
    using D = DTypeOf<DT>;
    __shared__ float s_sum[16][64];
    const uint32_t rank = blockIdx.y;
    const uint32_t col = blockIdx.x * 64 + threadIdx.x;
    float sum = 0.0f;
    if (col < elems) {
        const float *p = partial + static_cast<size_t>(rank) * slots * elems + col;
#pragma unroll 4
        for (uint32_t s = threadIdx.y; s < slots; s += 16) sum += p[static_cast<size_t>(s) * elems];
    }
    s_sum[threadIdx.y][threadIdx.x] = sum;
    __syncthreads();
    if (threadIdx.y != 0 || col >= elems) return;
    for (uint32_t y = 1; y < 16; ++y) sum += s_sum[y][threadIdx.x];
    reinterpret_cast<typename D::S *>(dweight.p[rank])[col] = D::narrow(sum);
}

// Threads per row and vectors per thread: a row is held by as few wavefronts as leave a thread at most four vectors of it;
// workgroups of short rows hold several.
struct RowShape {
    uint32_t threads;
    uint32_t per_group;
    uint32_t vectors;
};
RowShape shape_of(uint32_t elems, int ne)
{
    const uint32_t vecs = (elems + ne - 1) / ne;
    uint32_t threads = 64;
    while (threads * kMostVectors < vecs) threads *= 2;
    return {threads, std::max(1u, 256u / threads), (vecs + threads - 1) / threads};
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
    switch (s.vectors) {
        case 1: HCCLX_LAUNCH((k_rms_norm_grad<DT, 1>), grid, block, 0, st, p, rows, elems, eps, partial); break;
        case 2: HCCLX_LAUNCH((k_rms_norm_grad<DT, 2>), grid, block, 0, st, p, rows, elems, eps, partial); break;
        case 3: HCCLX_LAUNCH((k_rms_norm_grad<DT, 3>), grid, block, 0, st, p, rows, elems, eps, partial); break;
        default: HCCLX_LAUNCH((k_rms_norm_grad<DT, 4>), grid, block, 0, st, p, rows, elems, eps, partial); break;
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
        const dim3 grid((rows + shape.per_group - 1) / shape.per_group, n);
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
    DeviceBlock partial;   // float[n][slots][elems]

    template <int DT>
    void run(hipStream_t st) const
    {
        float *part = reinterpret_cast<float *>(partial.p);
        const uint32_t slots = groups * shape.per_group;
        if (rows != 0) launch_grad<DT>(shape, dim3(groups, n), st, ptrs, rows, elems, eps, part);
        if (want_dweight) {
            HCCLX_LAUNCH((k_rms_norm_join<DT>), dim3((elems + 63) / 64, n), dim3(64, 16), 0, st, dweight, rows != 0 ? slots : 0u, elems, part);
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

int make_norm(const hcclx_rms_norm_t &a, hcclx_plan_t **plan)
{
    int rc = check_norm(a.n, a.row_elems, a.dtype);
    if (rc != HCCL_SUCCESS) return rc;
    const bool quant = a.out_dtype == HCCL_DATA_TYPE_FP8E4M3;
    if (!quant && a.out_dtype != a.dtype) return fail(HCCL_E_NOT_SUPPORT, "out has the rows' type or HCCL_DATA_TYPE_FP8E4M3");
    if (quant && a.row_elems % 16 != 0) return fail(HCCL_E_PARA, "8-bit rows are multiples of 16 elements");
    auto w = std::make_unique<NormWork>();
    const uint64_t size = dtype_size(a.dtype);
    if ((rc = take(a.x, a.n, size, false, "x", w->ptrs.x)) != HCCL_SUCCESS) return rc;
    if ((rc = take(a.residual, a.n, size, true, "residual", w->ptrs.residual)) != HCCL_SUCCESS) return rc;
    if ((rc = take(a.weight, a.n, size, false, "weight", w->ptrs.weight)) != HCCL_SUCCESS) return rc;
    if ((rc = take(a.total, a.n, size, true, "total", w->ptrs.total)) != HCCL_SUCCESS) return rc;
    if ((rc = take(a.out, a.n, quant ? 16 : size, false, "out", w->ptrs.out)) != HCCL_SUCCESS) return rc;
    DeviceCtx *ctx = device_ctx();
    if (!ctx) return HCCL_E_RUNTIME;
    w->n = a.n;
    w->rows = a.rows;
    w->elems = a.row_elems;
    w->dtype = a.dtype;
    w->quant = quant;
    w->eps = a.eps;
    w->shape = shape_of(a.row_elems, 16 / static_cast<int>(size));
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
    w->want_dweight = a.dweight != nullptr;
    w->n = a.n;
    w->rows = a.rows;
    w->elems = a.row_elems;
    w->dtype = a.dtype;
    w->eps = a.eps;
    w->shape = shape_of(a.row_elems, 16 / static_cast<int>(size));
    const uint32_t most = (a.rows + w->shape.per_group - 1) / w->shape.per_group;
    w->groups = std::min(most, std::max(1u, 4u * ctx->num_cus / a.n));
    uint64_t held = 0;
    if (w->want_dweight && a.rows != 0) {
        held = static_cast<uint64_t>(a.n) * w->groups * w->shape.per_group * a.row_elems * sizeof(float);
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
