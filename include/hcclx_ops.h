/*
 * hcclx_ops.h -- operators that stand next to the collectives of a training or serving step, for n virtual ranks whose
 * buffers live in one GPU's HBM: the norm in front of an MoE exchange, the experts' feed-forward block behind it, and the
 * AdamW step on a shard of reduced gradients.  No counterpart in the reference, whose callers bring these themselves.
 *
 * Every operator is a plan (hcclx.h): created once from shapes and device pointers, launched any number of times on any
 * stream, also into a HIP graph that is being captured, destroyed with hcclx_plan_destroy.  Arrays of pointers are host
 * arrays and are copied; what they point to has to outlive the plan.  A plan that has device memory of its own (the
 * experts' block, the norm's gradient) has one copy of it: two launches of such a plan must not overlap in time.
 * Elements lie back to back; a buffer is aligned to its element where nothing else is said.  Refusals: HCCL_E_PTR for a
 * missing pointer, HCCL_E_PARA for a size or alignment, HCCL_E_NOT_SUPPORT for a type.
 */
#ifndef HCCL_AMD_HCCLX_OPS_H_
#define HCCL_AMD_HCCLX_OPS_H_

#include "hcclx.h"

#ifdef __cplusplus
extern "C" {
#endif

/* ---- Root-mean-square norm, with the residual's addition ---------------------------------------------------------
 * For every row of every rank:
 *     total = x + residual, rounded to dtype                (without residual: total = x)
 *     out   = total * weight / sqrt(mean(total^2) + eps),   of the total as it is stored, in 32 bits, rounded once
 * Types: fp32, fp16, bf16.  With out_dtype HCCL_DATA_TYPE_FP8E4M3 a row of out is row_elems codes, followed by
 * HCCLX_ROW8_TAIL bytes: the row's scale (float), max|out| / 448, and zeros.  An element is code * scale, the code rounded to
 * nearest; a row of zeros has scale 0.  Such rows are multiples of 16 bytes (row_elems has to be one), so that an MoE
 * dispatch of row_elems + HCCLX_ROW8_TAIL elements of HCCL_DATA_TYPE_FP8E4M3 carries codes and scale, and the experts' block
 * reads them where they arrive.
 * x, residual and weight have one pointer per rank (several may be the same).  Where no other rank reads them, total may be x or
 * residual, and out may be the one of them that total is not; not so 8-bit rows, which lie at other places than those of x (a single
 * row may).  Results that overlap anything else the launch reads or writes are refused (HCCL_E_PARA). */
#define HCCLX_ROW8_TAIL 16
#define HCCLX_NORM_MAX_ROW 16384
typedef struct {
    uint32_t n;         /* ranks, 1 .. 64 */
    uint32_t rows;      /* of each rank, as many as fit a launch (2^22 - 1 of any length, 2^28 - 4 of the shortest); 0: nothing to do */
    uint32_t row_elems; /* 1 .. HCCLX_NORM_MAX_ROW */
    int dtype;          /* of x, residual, weight and total */
    int out_dtype;      /* dtype or HCCL_DATA_TYPE_FP8E4M3 */
    float eps;
    const void *const *x;
    const void *const *residual; /* NULL: none */
    const void *const *weight;
    void *const *total;          /* NULL: not stored */
    void *const *out;
} hcclx_rms_norm_t;
int hcclx_rms_norm_plan_create(const hcclx_rms_norm_t *norm, hcclx_plan_t **plan);

/* Its gradient.  total is what the norm stored (or x, without a residual); r = 1 / sqrt(mean(total^2) + eps):
 *     dx      = r * (dy * weight - total * r^2 * mean(dy * weight * total)) + dtotal
 *     dweight = sum over the rank's rows of dy * total * r
 * dx is the gradient of x and of residual alike; dtotal is what reaches total from elsewhere (NULL: nothing).  Sums are held
 * in 32 bits and added in a fixed order.  dx may be its rank's dy, total or dtotal where no other rank reads it; on top of anything
 * else that is read it is refused (HCCL_E_PARA).  dweight, which is written when all has been read, may be weight; NULL: not
 * wanted. */
typedef struct {
    uint32_t n;
    uint32_t rows; /* 0: dweight becomes zeros */
    uint32_t row_elems;
    int dtype;
    float eps;
    const void *const *dy;
    const void *const *total;
    const void *const *weight;
    const void *const *dtotal;
    void *const *dx;
    void *const *dweight;
} hcclx_rms_norm_grad_t;
int hcclx_rms_norm_grad_plan_create(const hcclx_rms_norm_grad_t *norm, hcclx_plan_t **plan);

/* ---- Gated feed-forward block, one expert per rank ----------------------------------------------------------------
 * For every row x of rank j, with that rank's weights (row-major, w_gate and w_up hidden x dim, w_down dim x hidden):
 *     h = act(x w_gate^T) * (x w_up^T),     out = h w_down^T
 * Types: fp16, bf16.  Products accumulate in 32 bits; h, the operand of the second product, is rounded to dtype.
 *
 * How many rows rank j has is read on the device when the plan is launched:
 *     rows_j = (counts[j * counts_per_rank + 0] + ... + counts[j * counts_per_rank + counts_per_rank - 1]) / count_unit
 * With counts = recv_counts of hcclx_moe_route, counts_per_rank = n and count_unit = its row_elems these are the rows that
 * hcclx_moe_dispatch left in recv[j].  counts NULL: capacity rows each.  Rows beyond capacity, and beyond `rows` in all ranks
 * together, are not read and not written.
 *
 * x_dtype HCCL_DATA_TYPE_FP8E4M3: x holds rows of codes and a scale as the norm writes them (dim a multiple of 16).
 * dim and hidden are multiples of 8, at most HCCLX_FFN_MAX_DIM; rows, weights and out are 16-byte aligned.  out overlaps no input.
 * saved: for the gradient, hcclx_gated_ffn_saved_bytes(rows, hidden) bytes, 16-byte aligned: both products in 32 bits (so that the
 * gradient is that of the values the forward pass had).  NULL when only out is wanted. */
#define HCCLX_FFN_MAX_DIM 262144
typedef enum {
    HCCLX_ACT_SILU = 0,     /* a / (1 + exp(-a)) */
    HCCLX_ACT_GELU_TANH = 1 /* a / 2 * (1 + tanh(sqrt(2 / pi) * (a + 0.044715 a^3))) */
} hcclx_act_t;
typedef struct {
    uint32_t n;        /* ranks, 1 .. 64 */
    uint32_t capacity; /* rows that fit a rank's buffers */
    uint32_t dim;
    uint32_t hidden;
    uint64_t rows;     /* at most so many in all ranks together; 0: n * capacity.  Scratch memory is sized by it, and kernels are
                          chosen by it: a decoding step's plan should say how many rows it has at most */
    int dtype;
    int activation;    /* hcclx_act_t */
    const uint64_t *counts; /* device */
    uint32_t counts_per_rank;
    uint32_t count_unit;
} hcclx_ffn_shape_t;
typedef struct {
    hcclx_ffn_shape_t shape;
    int x_dtype;       /* shape.dtype or HCCL_DATA_TYPE_FP8E4M3 */
    const void *const *x;
    const void *const *w_gate;
    const void *const *w_up;
    const void *const *w_down;
    void *const *out;
    void *saved;
} hcclx_gated_ffn_t;
uint64_t hcclx_gated_ffn_saved_bytes(uint64_t rows, uint32_t hidden);
int hcclx_gated_ffn_plan_create(const hcclx_gated_ffn_t *ffn, hcclx_plan_t **plan);

/* Its gradients, from dy of out and what the forward pass saved for the same shape and counts.  The gradients of the weights
 * are sums over the rank's rows (zeros where it has none), rounded once; the operands of their products are rounded to dtype
 * (the gradients of both products of the forward pass, and h).  The buffers of dx may be those of dy or of x, and
 * those of dw_gate, dw_up and dw_down the weights', but not both at once (w_down's always); what is written on other inputs is refused
 * where an address says so (HCCL_E_PARA). */
typedef struct {
    hcclx_ffn_shape_t shape;
    const void *const *dy;
    const void *const *x;
    const void *const *w_gate;
    const void *const *w_up;
    const void *const *w_down;
    const void *saved;
    void *const *dx;
    void *const *dw_gate;
    void *const *dw_up;
    void *const *dw_down;
} hcclx_gated_ffn_grad_t;
int hcclx_gated_ffn_grad_plan_create(const hcclx_gated_ffn_grad_t *ffn, hcclx_plan_t **plan);

/* ---- AdamW over many tensors at once --------------------------------------------------------------------------------
 *     g = grad * grad_scale
 *     m = beta1 m + (1 - beta1) g,   v = beta2 v + (1 - beta2) g^2
 *     param = param - lr (weight_decay param + (m / (1 - beta1^step)) / (sqrt(v / (1 - beta2^step)) + eps))
 * param is fp32; grad is fp32, fp16 or bf16; copy (optional) receives the new param rounded to fp16 or bf16, for the
 * AllGather that follows.  One launch for all tensors.
 *
 * state_dtype fp32: m and v are floats.  state_dtype HCCL_DATA_TYPE_FP8E4M3: m and v are one code per element; every
 * HCCLX_ADAMW_BLOCK elements of a tensor (the last block may be shorter) have a scale each in m_scale and v_scale, the largest
 * magnitude of the block / 448.  m = code * scale; sqrt(v) = code * scale: of the square root, 8 bits hold twice the range.  The
 * new states are rounded stochastically: up to the next code with the probability of the distance from the one below.  (To
 * nearest, a moving average that moves by less than half a code per step would stand still.)  The random number of element k
 * of tensor t is  mix(k + mix(seed + (t + 1) * 0x9E3779B9)),  in 32-bit arithmetic, its low half for m and its high half for
 * sqrt(v), with
 *     mix(x):  x ^= x >> 16;  x *= 0x7FEB352D;  x ^= x >> 15;  x *= 0x846CA68B;  x ^= x >> 16
 * (its shifts and factors are those of C. Wellons' published search for such mixers), so that a step is a function of its arguments;
 * give every step another seed.  Magnitudes below 2^-9 codes, 4.4e-6 of the largest of their block, are held as zero or as 2^-9 of a
 * code: where sqrt(v) is held as zero and m is not, what is left of the update's denominator is the new gradient's part and eps, so
 * eps is to be chosen with that in mind. */
#define HCCLX_ADAMW_BLOCK 256
typedef struct {
    uint64_t count;
    float *param;
    const void *grad;
    void *m;
    void *v;
    float *m_scale; /* 8-bit states only */
    float *v_scale;
    void *copy;     /* all tensors have one, or none */
    float weight_decay;
} hcclx_adamw_tensor_t;
typedef struct {
    double lr;
    double beta1;
    double beta2;
    double eps;
    uint32_t step; /* 1, 2, ... */
    uint32_t seed;
    const float *grad_scale; /* device; NULL: 1 */
} hcclx_adamw_step_t;
/* copy_dtype: fp16 or bf16, when the tensors have a copy. */
int hcclx_adamw_plan_create(const hcclx_adamw_tensor_t *tensors, uint32_t ntensors, int grad_dtype, int state_dtype,
                            int copy_dtype, hcclx_plan_t **plan);
/* Launches a plan made by hcclx_adamw_plan_create (hcclx_plan_launch refuses it: it has no step).  Captured into a HIP graph,
 * the values of *step are those of the capture. */
int hcclx_adamw_step(const hcclx_plan_t *plan, const hcclx_adamw_step_t *step, void *stream);

#ifdef __cplusplus
}
#endif
#endif /* HCCL_AMD_HCCLX_OPS_H_ */
