// C entry points of the experts' gated feed-forward block (include/hcclx_ops.h: hcclx_gated_ffn_*): checks, the plans' scratch
// memory and the order of the products.
//
// Forward: two launches (three where 8-bit rows are widened first).  Gradient: three; with T rows in all, the products of the
// forward pass are 6 T dim hidden operations, those of the gradient twice as many.
#include "hcclx_internal.h"
#include "hcclx_ops.h"
#include "ops/ffn.h"

#include <algorithm>
#include <string>

using namespace hcclx;

namespace {

int check_shape(const hcclx_ffn_shape_t &s, FfnRows *out)
{
    if (s.n == 0 || s.n > kFfnRanks) return fail(HCCL_E_PARA, "rank count outside 1.." + std::to_string(kFfnRanks));
    if (s.dtype != HCCL_DATA_TYPE_FP16 && s.dtype != HCCL_DATA_TYPE_BFP16) return fail(HCCL_E_NOT_SUPPORT, "the feed-forward block takes fp16 or bf16");
    if (s.activation != HCCLX_ACT_SILU && s.activation != HCCLX_ACT_GELU_TANH) return fail(HCCL_E_NOT_SUPPORT, "unknown activation");
    if (s.dim == 0 || s.dim % 8 != 0 || s.dim > HCCLX_FFN_MAX_DIM || s.hidden == 0 || s.hidden % 8 != 0 || s.hidden > HCCLX_FFN_MAX_DIM) {
        return fail(HCCL_E_PARA, "dim and hidden are multiples of 8, at most " + std::to_string(HCCLX_FFN_MAX_DIM));
    }
    const uint64_t all = static_cast<uint64_t>(s.n) * s.capacity;
    const uint64_t most = s.rows == 0 || s.rows > all ? all : s.rows;
    if (most > 0xffffffffull / 256) return fail(HCCL_E_PARA, "too many rows");   // a workgroup of 256 for each, in one launch
    if (s.counts != nullptr && (s.counts_per_rank == 0 || s.counts_per_rank > kFfnRanks)) {
        return fail(HCCL_E_PARA, "counts per rank outside 1.." + std::to_string(kFfnRanks));
    }
    if (s.counts != nullptr && s.count_unit == 0) return fail(HCCL_E_PARA, "count_unit is zero");
    if (reinterpret_cast<uint64_t>(s.counts) % 8 != 0) return fail(HCCL_E_PARA, "counts is not aligned to 8 bytes");
    *out = {s.counts, s.counts_per_rank, s.count_unit, s.n, s.capacity, static_cast<uint32_t>(most), s.dim, s.hidden};
    return HCCL_SUCCESS;
}

int take(const void *const *in, uint32_t n, const char *what, const char **out)
{
    if (in == nullptr) return fail(HCCL_E_PTR, std::string(what) + " pointer array is null");
    for (uint32_t i = 0; i < n; ++i) {
        if (in[i] == nullptr) return fail(HCCL_E_PTR, std::string(what) + "[" + std::to_string(i) + "] is null");
        if ((reinterpret_cast<uint64_t>(in[i]) & 15) != 0) {
            return fail(HCCL_E_PARA, std::string(what) + "[" + std::to_string(i) + "] is not 16-byte aligned");
        }
        out[i] = static_cast<const char *>(in[i]);
    }
    return HCCL_SUCCESS;
}

hipError_t product(int dtype, FfnKind kind, const FfnArgs &a, uint32_t cus, hipStream_t st)
{
    return dtype == HCCL_DATA_TYPE_FP16 ? launch_ffn<HCCL_DATA_TYPE_FP16>(kind, a, cus, st) : launch_ffn<HCCL_DATA_TYPE_BFP16>(kind, a, cus, st);
}

struct FfnWork : PlanWork {
    int dtype = 0;
    FfnArgs up{};     // gate and up products
    FfnArgs down{};
    DeviceBlock scratch;   // h, x16

    int launch(const DeviceCtx *ctx, hipStream_t st) const override
    {
        hipError_t e = product(dtype, kFfnGateUp, up, ctx->num_cus, st);
        if (e == hipSuccess) e = product(dtype, kFfnDown, down, ctx->num_cus, st);
        return e == hipSuccess ? HCCL_SUCCESS : fail_hip(e, "feed-forward kernels");
    }
};

struct FfnGradWork : PlanWork {
    int dtype = 0;
    FfnArgs hidden{};
    FfnArgs input{};
    FfnArgs weights{};
    bool weights_first = false;   // dx lies on what the weights' products read
    DeviceBlock scratch;          // h, dproj

    int launch(const DeviceCtx *ctx, hipStream_t st) const override
    {
        hipError_t e = product(dtype, kFfnGradHidden, hidden, ctx->num_cus, st);
        if (e == hipSuccess && weights_first) e = product(dtype, kFfnGradWeights, weights, ctx->num_cus, st);
        if (e == hipSuccess) e = product(dtype, kFfnGradInput, input, ctx->num_cus, st);
        if (e == hipSuccess && !weights_first) e = product(dtype, kFfnGradWeights, weights, ctx->num_cus, st);
        return e == hipSuccess ? HCCL_SUCCESS : fail_hip(e, "feed-forward gradient kernels");
    }
};

uint64_t round256(uint64_t x) { return (x + 255) & ~255ull; }

int make_ffn(const hcclx_gated_ffn_t &f, hcclx_plan_t **plan)
{
    FfnRows rows;
    int rc = check_shape(f.shape, &rows);
    if (rc != HCCL_SUCCESS) return rc;
    const bool small = f.x_dtype == HCCL_DATA_TYPE_FP8E4M3;
    if (!small && f.x_dtype != f.shape.dtype) return fail(HCCL_E_NOT_SUPPORT, "x has the weights' type or HCCL_DATA_TYPE_FP8E4M3");
    if (small && rows.dim % 16 != 0) return fail(HCCL_E_PARA, "8-bit rows are multiples of 16 elements");
    if (small && f.saved != nullptr) return fail(HCCL_E_NOT_SUPPORT, "the gradient takes rows of the weights' type");
    if ((reinterpret_cast<uint64_t>(f.saved) & 15) != 0) return fail(HCCL_E_PARA, "saved is not 16-byte aligned");
    auto w = std::make_unique<FfnWork>();
    w->dtype = f.shape.dtype;
    w->up.rows = w->down.rows = rows;
    w->up.act = f.shape.activation;
    w->up.saved = static_cast<float *>(f.saved);
    if ((rc = take(f.x, rows.n, "x", w->up.p[0])) != HCCL_SUCCESS) return rc;
    if ((rc = take(f.w_gate, rows.n, "w_gate", w->up.p[1])) != HCCL_SUCCESS) return rc;
    if ((rc = take(f.w_up, rows.n, "w_up", w->up.p[2])) != HCCL_SUCCESS) return rc;
    if ((rc = take(f.w_down, rows.n, "w_down", w->down.p[0])) != HCCL_SUCCESS) return rc;
    if ((rc = take(const_cast<const void *const *>(f.out), rows.n, "out", w->down.p[1])) != HCCL_SUCCESS) return rc;
    DeviceCtx *ctx = device_ctx();
    if (!ctx) return HCCL_E_RUNTIME;
    const uint64_t h_bytes = round256(static_cast<uint64_t>(rows.most) * rows.hidden * 2);
    const uint64_t held = h_bytes + (small ? round256(static_cast<uint64_t>(rows.most) * rows.dim * 2) : 0);
    if (held != 0 && (rc = w->scratch.get(held)) != HCCL_SUCCESS) return rc;
    w->up.h = w->down.h = w->scratch.p;
    w->up.x8 = small;
    if (small) w->up.x16 = w->scratch.p + h_bytes;
    const uint64_t weights = 3ull * rows.n * rows.dim * rows.hidden * 2;
    return plan_of(ctx, std::move(w), weights + static_cast<uint64_t>(rows.most) * rows.dim * (small ? 3 : 4), held, plan);
}

// How many of n pointers are among n others.
uint32_t among(uint32_t n, const char *const *a, const char *const *b)
{
    return static_cast<uint32_t>(std::count_if(a, a + n, [&](const char *p) { return std::find(b, b + n, p) != b + n; }));
}

int make_ffn_grad(const hcclx_gated_ffn_grad_t &f, hcclx_plan_t **plan)
{
    FfnRows rows;
    int rc = check_shape(f.shape, &rows);
    if (rc != HCCL_SUCCESS) return rc;
    if (f.saved == nullptr) return fail(HCCL_E_PTR, "saved is null");
    if ((reinterpret_cast<uint64_t>(f.saved) & 15) != 0) return fail(HCCL_E_PARA, "saved is not 16-byte aligned");
    auto w = std::make_unique<FfnGradWork>();
    w->dtype = f.shape.dtype;
    w->hidden.rows = w->input.rows = w->weights.rows = rows;
    w->hidden.act = f.shape.activation;
    w->hidden.saved = static_cast<float *>(const_cast<void *>(f.saved));
    if ((rc = take(f.dy, rows.n, "dy", w->hidden.p[0])) != HCCL_SUCCESS) return rc;
    if ((rc = take(f.w_down, rows.n, "w_down", w->hidden.p[1])) != HCCL_SUCCESS) return rc;
    if ((rc = take(f.w_gate, rows.n, "w_gate", w->input.p[0])) != HCCL_SUCCESS) return rc;
    if ((rc = take(f.w_up, rows.n, "w_up", w->input.p[1])) != HCCL_SUCCESS) return rc;
    if ((rc = take(const_cast<const void *const *>(f.dx), rows.n, "dx", w->input.p[2])) != HCCL_SUCCESS) return rc;
    if ((rc = take(f.x, rows.n, "x", w->weights.p[0])) != HCCL_SUCCESS) return rc;
    if ((rc = take(f.dy, rows.n, "dy", w->weights.p[1])) != HCCL_SUCCESS) return rc;
    if ((rc = take(const_cast<const void *const *>(f.dw_gate), rows.n, "dw_gate", w->weights.p[2])) != HCCL_SUCCESS) return rc;
    if ((rc = take(const_cast<const void *const *>(f.dw_up), rows.n, "dw_up", w->weights.p[3])) != HCCL_SUCCESS) return rc;
    if ((rc = take(const_cast<const void *const *>(f.dw_down), rows.n, "dw_down", w->weights.p[4])) != HCCL_SUCCESS) return rc;
    // What a product writes may lie on what only products before it read.  How many rows a buffer has is known on the device only, and
    // one without rows may begin where another ends, so nothing is refused for a single rank's address.
    const uint32_t n = rows.n;
    const char *const *x = w->weights.p[0], *const *dy = w->weights.p[1], *const *dx = w->input.p[2];
    const char *const *w_gate = w->input.p[0], *const *w_up = w->input.p[1];
    const uint32_t dx_on_x = among(n, dx, x), dx_on_dy = among(n, dx, dy);
    w->weights_first = dx_on_x != 0 || dx_on_dy != 0;
    if (rows.most != 0 && (among(n, dx, w_gate) == n || among(n, dx, w_up) == n)) return fail(HCCL_E_PARA, "dx on w_gate or w_up");
    for (uint32_t k = 2; k < 5 && rows.most != 0; ++k) {
        const char *const *dw = w->weights.p[k];
        if (among(n, dw, x) == n || among(n, dw, dy) == n) return fail(HCCL_E_PARA, "the gradient of a weight on x or dy");
        if ((dx_on_x == n || dx_on_dy == n) && among(n, dw, w_gate) + among(n, dw, w_up) != 0) {
            return fail(HCCL_E_PARA, "dx on x or dy and the gradient of a weight on w_gate or w_up at once");
        }
    }
    DeviceCtx *ctx = device_ctx();
    if (!ctx) return HCCL_E_RUNTIME;
    const uint64_t h_bytes = round256(static_cast<uint64_t>(rows.most) * rows.hidden * 2);
    const uint64_t held = 3 * h_bytes;
    if (held != 0 && (rc = w->scratch.get(held)) != HCCL_SUCCESS) return rc;
    w->hidden.h = w->weights.h = w->scratch.p;
    w->hidden.dproj = w->input.dproj = w->weights.dproj = w->scratch.p + h_bytes;
    const uint64_t weights = 6ull * rows.n * rows.dim * rows.hidden * 2;
    const uint64_t per_row = 6ull * rows.dim + 8ull * rows.hidden;
    return plan_of(ctx, std::move(w), weights + rows.most * per_row, held, plan);
}

}  // namespace

extern "C" {

uint64_t hcclx_gated_ffn_saved_bytes(uint64_t rows, uint32_t hidden) { return rows * hidden * 2 * sizeof(float); }

int hcclx_gated_ffn_plan_create(const hcclx_gated_ffn_t *ffn, hcclx_plan_t **plan)
{
    if (plan == nullptr) return fail(HCCL_E_PTR, "plan is null");
    *plan = nullptr;
    if (ffn == nullptr) return fail(HCCL_E_PTR, "ffn is null");
    return guarded([&] { return make_ffn(*ffn, plan); });
}

int hcclx_gated_ffn_grad_plan_create(const hcclx_gated_ffn_grad_t *ffn, hcclx_plan_t **plan)
{
    if (plan == nullptr) return fail(HCCL_E_PTR, "plan is null");
    *plan = nullptr;
    if (ffn == nullptr) return fail(HCCL_E_PTR, "ffn is null");
    return guarded([&] { return make_ffn_grad(*ffn, plan); });
}

}  // extern "C"
