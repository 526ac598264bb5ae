// The AdamW step over many tensors in one launch (include/hcclx_ops.h: hcclx_adamw_*).
//
// Bound: HBM bandwidth: 28 bytes per element with 16-bit gradients, states in 32 bits and a 16-bit copy, 16 with states in 8 bits.
// A workgroup takes a tile of one tensor; a wavefront takes 256 elements of it, a lane four neighbouring ones, so that every access
// of a wavefront is one run of memory and a block's scale is a reduction in registers.  (Two such blocks per wavefront, which ends
// later and holds more registers: 100 M elements 632 us, one 522.)
#include "hcclx_internal.h"
#include "hcclx_ops.h"
#include "kernels/elem.h"
#include "kernels/fold.h"
#include "ops/lanes.h"

#include <cmath>
#include <string>
#include <vector>

using namespace hcclx;

namespace {

constexpr uint32_t kBlock = HCCLX_ADAMW_BLOCK;
constexpr uint32_t kThreads256 = 256;
constexpr uint32_t kTile = kBlock * (kThreads256 / 64);   // elements per workgroup
static_assert(kBlock == 64 * 4, "a lane holds four elements of a block");

struct TensorDev {
    uint64_t count;
    float *param;
    const char *grad;
    char *m;
    char *v;
    float *m_scale;
    float *v_scale;
    char *copy;
    uint64_t first_tile;
    float weight_decay;
    uint32_t index;
};

struct StepArgs {
    float lr, beta1, rest1, beta2, rest2, eps, unbias1, root2;   // rest = 1 - beta, unbias = 1 / (1 - beta^step), root2 = sqrt(unbias2)
    uint32_t seed;
    const float *grad_scale;
};

// (shifts and factors: of C. Wellons' published search for 32-bit mixers whose output bits depend on all input bits alike)
__device__ __forceinline__ uint32_t mix(uint32_t x)
{
    x ^= x >> 16;
    x *= 0x7FEB352Du;
    x ^= x >> 15;
    x *= 0x846CA68Bu;
    x ^= x >> 16;
    return x;
}

// |x| as the e4m3 value below it or the one above (which u in [0, 1) decides), with x's sign.  The values lie a power of two
// apart: of the magnitude's own power 2^-3, 2^-9 at least.  NaN stays NaN.
__device__ __forceinline__ float round_by(float x, float u)
{
    const float a = fabsf(x);
    uint32_t power = __float_as_uint(a) & 0x7f800000u;                       // 2^floor(log2 a)
    power = power < 0x3c800000u ? 0x3c800000u : power;                       // 2^-6 at least
    const float gap = __uint_as_float(power - 0x01800000u);                  // / 8
    const float inverse = __uint_as_float(0x7f000000u - (power - 0x01800000u));
    float q = floorf(a * inverse + u) * gap;
    q = q > kE4m3Most ? kE4m3Most : q;   // the largest magnitude of a block may come out of its scale a rounding above 448
    return copysignf(q, x);
}

typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef u32x2 u32x2_u __attribute__((aligned(1)));
typedef uint32_t u32_u __attribute__((aligned(1)));
typedef float f32x4v __attribute__((ext_vector_type(4)));
typedef f32x4v f32x4_u __attribute__((aligned(4)));

// The tensors' addresses come out of a table, which does not say that they are in global memory.
template <typename T>
using Global = __attribute__((address_space(1))) T *;
template <typename T>
__device__ __forceinline__ Global<T> global(const void *p)
{
    return reinterpret_cast<Global<T>>(reinterpret_cast<uint64_t>(p));
}

__device__ __forceinline__ uint32_t pack2(float a, float b, HcclDataType dt)
{
    if (dt == HCCL_DATA_TYPE_BFP16) {
        typedef __bf16 B2 __attribute__((ext_vector_type(2)));
        return __builtin_bit_cast(uint32_t, B2{static_cast<__bf16>(a), static_cast<__bf16>(b)});
    }
    typedef _Float16 H2 __attribute__((ext_vector_type(2)));
    return __builtin_bit_cast(uint32_t, H2{static_cast<_Float16>(a), static_cast<_Float16>(b)});
}

// Four elements at `at` as floats; only the first `have` exist.
template <int DT>
__device__ __forceinline__ void load4(const void *base, uint64_t at, uint32_t have, float (&f)[4])
{
    using D = DTypeOf<DT>;
    using S = typename D::S;
    const Global<const S> p = global<const S>(base) + at;
    if (have >= 4) {
        if constexpr (sizeof(S) == 4) {
            const f32x4v x = *reinterpret_cast<Global<const f32x4_u>>(p);
#pragma unroll
            for (int e = 0; e < 4; ++e) f[e] = x[e];
        } else {
            const u32x2 x = *reinterpret_cast<Global<const u32x2_u>>(p);
#pragma unroll
            for (int e = 0; e < 4; ++e) f[e] = D::widen(static_cast<S>(x[e / 2] >> (16 * (e & 1))));
        }
    } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) f[e] = static_cast<uint32_t>(e) < have ? D::widen(p[e]) : 0.0f;
    }
}
template <int DT>
__device__ __forceinline__ void store4(void *base, uint64_t at, uint32_t have, const float (&f)[4])
{
    using D = DTypeOf<DT>;
    using S = typename D::S;
    const Global<S> p = global<S>(base) + at;
    if (have >= 4) {
        if constexpr (sizeof(S) == 4) {
            __builtin_nontemporal_store(f32x4v{f[0], f[1], f[2], f[3]}, reinterpret_cast<Global<f32x4_u>>(p));
        } else {
            constexpr HcclDataType kDt = static_cast<HcclDataType>(DT);
            __builtin_nontemporal_store(u32x2{pack2(f[0], f[1], kDt), pack2(f[2], f[3], kDt)}, reinterpret_cast<Global<u32x2_u>>(p));
        }
    } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            if (static_cast<uint32_t>(e) < have) p[e] = D::narrow(f[e]);
        }
    }
}
__device__ __forceinline__ uint32_t load_codes(const void *base, uint64_t at, uint32_t have)
{
    const Global<const uint8_t> p = global<const uint8_t>(base) + at;
    if (have >= 4) return *reinterpret_cast<Global<const u32_u>>(p);
    uint32_t c = 0;
#pragma unroll
    for (uint32_t e = 0; e < 3; ++e) {
        if (e < have) c |= static_cast<uint32_t>(p[e]) << (8 * e);
    }
    return c;
}
__device__ __forceinline__ void store_codes(void *base, uint64_t at, uint32_t have, uint32_t c)
{
    const Global<uint8_t> p = global<uint8_t>(base) + at;
    if (have >= 4) {
        __builtin_nontemporal_store(c, reinterpret_cast<Global<u32_u>>(p));
    } else {
#pragma unroll
        for (uint32_t e = 0; e < 3; ++e) {
            if (e < have) p[e] = static_cast<uint8_t>(c >> (8 * e));
        }
    }
}

// x / scale, rounded as a division is, for a whole block: with the scale's inverse, one step of the quotient's remainder gives the
// nearest float (Markstein).  Where the products would leave the range of normal floats it is a division.
struct Quotient {
    float by;
    float inverse;
    bool plain;
    __device__ __forceinline__ explicit Quotient(float scale)
    {
        by = scale > 0.0f ? scale : 1.0f;
        inverse = 1.0f / by;
        plain = !(by > 0x1p-90f && by < 0x1p90f);
    }
    __device__ __forceinline__ float operator()(float x) const
    {
        if (plain) return x / by;
        const float q = x * inverse;
        return __builtin_fmaf(__builtin_fmaf(-q, by, x), inverse, q);
    }
};

// The eight XCDs take workgroups in turn: every XCD gets an eighth of the tiles that lie next to each other.  (100 M elements with 32-bit
// states 523 us, tiles in the workgroups' order 537; with 8-bit states 319 and 310, so those keep that order.)
__device__ __forceinline__ uint32_t of_xcd(uint32_t group, uint32_t groups)
{
    const uint32_t xcd = group % 8;
    const uint32_t more = groups % 8;   // XCDs with a tile more than the others
    return xcd * (groups / 8) + (xcd < more ? xcd : more) + group / 8;
}

template <int GRAD, bool SMALL, int COPY>   // COPY: a 16-bit type, or fp32 for none
__global__ void __launch_bounds__(kThreads256)
k_adamw(const TensorDev *tensors, const uint32_t *tensor_of_tile, StepArgs a)
{
    const uint32_t tile = SMALL ? blockIdx.x : of_xcd(blockIdx.x, gridDim.x);
    const TensorDev t = tensors[tensor_of_tile[tile]];
    const uint32_t lane = threadIdx.x & 63;
    const uint64_t start = (tile - t.first_tile) * kTile + static_cast<uint64_t>(threadIdx.x / 64) * kBlock;
    const float scale = a.grad_scale != nullptr ? *a.grad_scale : 1.0f;
    const uint32_t key = mix(a.seed + (t.index + 1) * 0x9E3779B9u);
    const uint64_t at = start + lane * 4;
    const uint32_t have = at >= t.count ? 0u : t.count - at >= 4 ? 4u : static_cast<uint32_t>(t.count - at);
    if (start >= t.count) return;   // the wavefront's whole block is behind the end
    const uint64_t block = start / kBlock;
    float g[4], p[4], m[4], v[4];
    load4<GRAD>(t.grad, at, have, g);
    load4<HCCL_DATA_TYPE_FP32>(t.param, at, have, p);
    if constexpr (SMALL) {
        const uint32_t cm = load_codes(t.m, at, have);
        const uint32_t cv = load_codes(t.v, at, have);
        const float ms = global<const float>(t.m_scale)[block];
        const float vs = global<const float>(t.v_scale)[block];
        from_e4m3(cm, m);
        from_e4m3(cv, v);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            m[e] *= ms;
            v[e] *= vs;
            v[e] *= v[e];
        }
    } else {
        load4<HCCL_DATA_TYPE_FP32>(t.m, at, have, m);
        load4<HCCL_DATA_TYPE_FP32>(t.v, at, have, v);
    }
    float r[4];   // sqrt(v)
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        const float x = g[e] * scale;
        m[e] = a.beta1 * m[e] + a.rest1 * x;
        v[e] = a.beta2 * v[e] + a.rest2 * x * x;
        r[e] = sqrtf(v[e]);
        // (the hardware's reciprocal is good to a rounding, of an update that is small against the parameter)
        const float update = (m[e] * a.unbias1) * __builtin_amdgcn_rcpf(r[e] * a.root2 + a.eps);
        p[e] = p[e] - a.lr * (t.weight_decay * p[e] + update);
    }
    store4<HCCL_DATA_TYPE_FP32>(t.param, at, have, p);
    if constexpr (COPY != HCCL_DATA_TYPE_FP32) store4<COPY>(t.copy, at, have, p);
    if constexpr (SMALL) {
        float most_m = 0.0f;
        float most_r = 0.0f;
#pragma unroll
        for (int e = 0; e < 4; ++e) {   // (elements behind the end are zeros throughout)
            most_m = fmaxf(most_m, fabsf(m[e]));
            most_r = fmaxf(most_r, r[e]);
        }
        const float scale_m = wave_max(most_m) * (1.0f / kE4m3Most);
        const float scale_r = wave_max(most_r) * (1.0f / kE4m3Most);
        const Quotient of_m(scale_m);
        const Quotient of_r(scale_r);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const uint32_t word = mix(static_cast<uint32_t>(at) + e + key);
            m[e] = round_by(of_m(m[e]), static_cast<float>(word & 0xffffu) * 0x1p-16f);
            v[e] = round_by(of_r(r[e]), static_cast<float>(word >> 16) * 0x1p-16f);
        }
        store_codes(t.m, at, have, to_e4m3(m[0], m[1], m[2], m[3]));
        store_codes(t.v, at, have, to_e4m3(v[0], v[1], v[2], v[3]));
        if (lane == 0) {
            global<float>(t.m_scale)[block] = scale_m;
            global<float>(t.v_scale)[block] = scale_r;
        }
    } else {
        store4<HCCL_DATA_TYPE_FP32>(t.m, at, have, m);
        store4<HCCL_DATA_TYPE_FP32>(t.v, at, have, v);
    }
}

struct AdamWWork : PlanWork {
    DeviceBlock table;   // TensorDev[], uint32_t[tiles]
    size_t tiles_at = 0;
    uint32_t tiles = 0;
    int grad = 0, copy = HCCL_DATA_TYPE_FP32;
    bool small = false;

    int launch(const DeviceCtx *, hipStream_t) const override
    {
        return fail(HCCL_E_PARA, "an AdamW plan is launched by hcclx_adamw_step");
    }

    template <int GRAD, bool SMALL>
    void run(const StepArgs &a, hipStream_t st) const
    {
        const TensorDev *t = reinterpret_cast<const TensorDev *>(table.p);
        const uint32_t *of = reinterpret_cast<const uint32_t *>(table.p + tiles_at);
        if (copy == HCCL_DATA_TYPE_BFP16) {
            HCCLX_LAUNCH((k_adamw<GRAD, SMALL, HCCL_DATA_TYPE_BFP16>), dim3(tiles), dim3(kThreads256), 0, st, t, of, a);
        } else if (copy == HCCL_DATA_TYPE_FP16) {
            HCCLX_LAUNCH((k_adamw<GRAD, SMALL, HCCL_DATA_TYPE_FP16>), dim3(tiles), dim3(kThreads256), 0, st, t, of, a);
        } else {
            HCCLX_LAUNCH((k_adamw<GRAD, SMALL, HCCL_DATA_TYPE_FP32>), dim3(tiles), dim3(kThreads256), 0, st, t, of, a);
        }
    }

    int step(const StepArgs &a, hipStream_t st) const
    {
        if (tiles == 0) return HCCL_SUCCESS;
        if (grad == HCCL_DATA_TYPE_FP32) {
            small ? run<HCCL_DATA_TYPE_FP32, true>(a, st) : run<HCCL_DATA_TYPE_FP32, false>(a, st);
        } else if (grad == HCCL_DATA_TYPE_FP16) {
            small ? run<HCCL_DATA_TYPE_FP16, true>(a, st) : run<HCCL_DATA_TYPE_FP16, false>(a, st);
        } else {
            small ? run<HCCL_DATA_TYPE_BFP16, true>(a, st) : run<HCCL_DATA_TYPE_BFP16, false>(a, st);
        }
        const hipError_t e = hipGetLastError();
        return e == hipSuccess ? HCCL_SUCCESS : fail_hip(e, "AdamW kernel");
    }
};

int check_pointer(const void *p, uint64_t align, uint32_t i, const char *what)
{
    if (p == nullptr) return fail(HCCL_E_PTR, std::string(what) + " of tensor " + std::to_string(i) + " is null");
    if (reinterpret_cast<uint64_t>(p) % align != 0) {
        return fail(HCCL_E_PARA, std::string(what) + " of tensor " + std::to_string(i) + " is not aligned to its elements");
    }
    return HCCL_SUCCESS;
}

int make_adamw(const hcclx_adamw_tensor_t *tensors, uint32_t n, int grad, int state, int copy, hcclx_plan_t **plan)
{
    if (grad != HCCL_DATA_TYPE_FP32 && grad != HCCL_DATA_TYPE_FP16 && grad != HCCL_DATA_TYPE_BFP16) {
        return fail(HCCL_E_NOT_SUPPORT, "gradients are fp32, fp16 or bf16");
    }
    if (state != HCCL_DATA_TYPE_FP32 && state != HCCL_DATA_TYPE_FP8E4M3) return fail(HCCL_E_NOT_SUPPORT, "states are fp32 or HCCL_DATA_TYPE_FP8E4M3");
    if (n != 0 && tensors == nullptr) return fail(HCCL_E_PTR, "tensors is null");
    const bool small = state == HCCL_DATA_TYPE_FP8E4M3;
    const bool copies = n != 0 && tensors[0].copy != nullptr;
    if (copies && copy != HCCL_DATA_TYPE_FP16 && copy != HCCL_DATA_TYPE_BFP16) return fail(HCCL_E_NOT_SUPPORT, "the copy is fp16 or bf16");
    const uint64_t gsize = dtype_size(grad);
    std::vector<TensorDev> devs;
    uint64_t tiles = 0;
    uint64_t elements = 0;
    for (uint32_t i = 0; i < n; ++i) {
        const hcclx_adamw_tensor_t &t = tensors[i];
        if ((t.copy != nullptr) != copies) return fail(HCCL_E_PTR, "all tensors have a copy, or none");
        if (t.count == 0) continue;
        int rc = check_pointer(t.param, 4, i, "param");
        if (rc == HCCL_SUCCESS) rc = check_pointer(t.grad, gsize, i, "grad");
        if (rc == HCCL_SUCCESS) rc = check_pointer(t.m, small ? 1 : 4, i, "m");
        if (rc == HCCL_SUCCESS) rc = check_pointer(t.v, small ? 1 : 4, i, "v");
        if (rc == HCCL_SUCCESS && small) rc = check_pointer(t.m_scale, 4, i, "m_scale");
        if (rc == HCCL_SUCCESS && small) rc = check_pointer(t.v_scale, 4, i, "v_scale");
        if (rc == HCCL_SUCCESS && copies) rc = check_pointer(t.copy, 2, i, "copy");
        if (rc != HCCL_SUCCESS) return rc;
        const uint64_t more = t.count / kTile + (t.count % kTile != 0);
        if (more > kMostBlocksX - tiles) return fail(HCCL_E_PARA, "too many elements for one launch");
        devs.push_back({t.count, t.param, static_cast<const char *>(t.grad), static_cast<char *>(t.m), static_cast<char *>(t.v), t.m_scale,
                        t.v_scale, static_cast<char *>(t.copy), tiles, t.weight_decay, i});
        tiles += more;
        elements += t.count;
    }
    DeviceCtx *ctx = device_ctx();
    if (!ctx) return HCCL_E_RUNTIME;
    auto w = std::make_unique<AdamWWork>();
    w->grad = grad;
    w->copy = copies ? copy : HCCL_DATA_TYPE_FP32;
    w->small = small;
    w->tiles = static_cast<uint32_t>(tiles);
    uint64_t held = 0;
    if (tiles != 0) {
        w->tiles_at = (devs.size() * sizeof(TensorDev) + 255) / 256 * 256;
        held = w->tiles_at + tiles * sizeof(uint32_t);
        std::vector<uint32_t> of(tiles);
        for (size_t i = 0; i < devs.size(); ++i) {
            const uint64_t end = i + 1 < devs.size() ? devs[i + 1].first_tile : tiles;
            for (uint64_t k = devs[i].first_tile; k < end; ++k) of[k] = static_cast<uint32_t>(i);
        }
        const int rc = w->table.get(held);
        if (rc != HCCL_SUCCESS) return rc;
        HCCLX_HIP(hipMemcpy(w->table.p, devs.data(), devs.size() * sizeof(TensorDev), hipMemcpyHostToDevice));
        HCCLX_HIP(hipMemcpy(w->table.p + w->tiles_at, of.data(), tiles * sizeof(uint32_t), hipMemcpyHostToDevice));
    }
    const uint64_t each = 8 + (small ? 4 : 16) + gsize + (copies ? 2 : 0);
    return plan_of(ctx, std::move(w), elements * each, held, plan);
}

}  // namespace

extern "C" {

int hcclx_adamw_plan_create(const hcclx_adamw_tensor_t *tensors, uint32_t ntensors, int grad_dtype, int state_dtype, int copy_dtype,
                            hcclx_plan_t **plan)
{
    if (plan == nullptr) return fail(HCCL_E_PTR, "plan is null");
    *plan = nullptr;
    return guarded([&] { return make_adamw(tensors, ntensors, grad_dtype, state_dtype, copy_dtype, plan); });
}

int hcclx_adamw_step(const hcclx_plan_t *plan, const hcclx_adamw_step_t *step, void *stream)
{
    if (plan == nullptr) return fail(HCCL_E_PTR, "plan is null");
    if (step == nullptr) return fail(HCCL_E_PTR, "step is null");
    const AdamWWork *work = dynamic_cast<const AdamWWork *>(work_of(plan));
    if (work == nullptr) return fail(HCCL_E_PARA, "not an AdamW plan");
    if (step->step == 0) return fail(HCCL_E_PARA, "steps are counted from 1");
    if (!(step->beta1 >= 0.0 && step->beta1 < 1.0 && step->beta2 >= 0.0 && step->beta2 < 1.0)) return fail(HCCL_E_PARA, "beta outside [0, 1)");
    if (!(step->eps >= 0.0)) return fail(HCCL_E_PARA, "eps is negative");
    if (reinterpret_cast<uint64_t>(step->grad_scale) % 4 != 0) return fail(HCCL_E_PARA, "grad_scale is not aligned");
    DeviceCtx *ctx = device_ctx();
    if (!ctx) return HCCL_E_RUNTIME;
    if (ctx->device != plan_device(plan)) return fail(HCCL_E_PARA, "plan belongs to another device");
    StepArgs a;
    a.lr = static_cast<float>(step->lr);
    a.beta1 = static_cast<float>(step->beta1);
    a.rest1 = static_cast<float>(1.0 - step->beta1);
    a.beta2 = static_cast<float>(step->beta2);
    a.rest2 = static_cast<float>(1.0 - step->beta2);
    a.eps = static_cast<float>(step->eps);
    a.unbias1 = static_cast<float>(1.0 / (1.0 - std::pow(step->beta1, step->step)));
    a.root2 = static_cast<float>(std::sqrt(1.0 / (1.0 - std::pow(step->beta2, step->step))));
    a.seed = step->seed;
    a.grad_scale = step->grad_scale;
    return work->step(a, static_cast<hipStream_t>(stream));
}

}  // extern "C"
