/*
 * hcclx_ops.h -- operators that stand next to the collectives of a training or serving step, for n virtual ranks whose
 * buffers live in one GPU's HBM: the norm in front of an MoE exchange, the experts' feed-forward block behind it, the
 * AdamW step on a shard of reduced gradients, and the output layer whose columns the ranks share: its largest logits, a loss
 * against a teacher's, and the draw of the next token.  No counterpart in the reference, whose callers bring these themselves.
 *
 * Every operator is a plan (hcclx.h): created once from shapes and device pointers, launched any number of times on any
 * stream, also into a HIP graph that is being captured, destroyed with hcclx_plan_destroy.  Arrays of pointers are host
 * arrays and are copied; what they point to has to outlive the plan.  A plan that has device memory of its own (the
 * experts' block, the norm's gradient, the operators of the output layer) has one copy of it: two launches of such a plan must not
 * overlap in time.
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

/* ---- Logits whose columns are split over the ranks --------------------------------------------------------------------
 * Every rank holds some columns of all rows: row r of the output layer is row r of rank 0, of rank 1 and so on, side by side, and its
 * columns are numbered through.  Types: fp32, fp16, bf16.  What lies between a rank's rows is neither read nor written, so ranks may
 * hold columns of one matrix.  What the operators below write may not overlap what they read, or each other (HCCL_E_PARA), but where
 * it is said. */
#define HCCLX_LOGITS_MAX_COLUMNS (1u << 24) /* of all ranks together */
#define HCCLX_TOP_MAX 1024                  /* entries of a list of largest logits */
typedef struct {
    uint32_t n;                 /* ranks, 1 .. 64 */
    uint32_t rows;              /* up to 2^22 - 1, of very many columns fewer; 0: nothing to do */
    int dtype;
    const void *const *logits;  /* aligned to their element; not looked at where a rank has no columns */
    const uint32_t *columns;    /* host: columns of each rank */
    const uint64_t *row_stride; /* host: elements from one row of a rank to the next, below 2^32; NULL: its columns */
} hcclx_logits_t;

/* The k largest logits of every row, in descending order, of equal ones the first; NaN counts as -infinity, -0 as 0.
 *     lse = log sum exp(logit) of the row, so that value - lse is the logarithm of a probability.  Summed in 32 bits, joined in 64. */
typedef struct {
    hcclx_logits_t logits;
    uint32_t k;       /* 1 .. HCCLX_TOP_MAX, no more than there are columns */
    void *values;     /* rows x k, of the logits' type */
    int32_t *indices; /* rows x k: numbers of the columns */
    float *lse;       /* rows; NULL: not wanted */
} hcclx_top_logits_t;
int hcclx_top_logits_plan_create(const hcclx_top_logits_t *top, hcclx_plan_t **plan);

/* Distillation from a teacher's largest logits.  For every row, with T the temperature:
 *     p = softmax(teacher / T) over the row's k entries,   q = softmax(logits / T) over all columns
 *     loss    = weight T^2 sum over the entries of p (log p - log q[indices])
 *     dlogits = weight T (q - the sum of p over the entries that name the column)
 * Entries whose index is no column's (-1, say) are left out, and a row without any entry but those, or but logits of -infinity, has
 * loss 0 and gradients 0; a column may be named by several entries.  A row of weight 0 (a masked token) is not read, whatever it holds:
 * loss 0, gradients 0.  NaN and +infinity in a row that counts, the teacher's or the student's, make its loss and gradients NaN.  A column
 * whose logit is -infinity has q = 0, and so has every column of a row of nothing else: with an entry of p > 0 there the loss is infinite, and its
 * gradient - weight T p.  The sum over the row's columns is held in 32 bits, what concerns the entries alone in 64; where several name a column, the
 * sum of their p is one of multiples of 2^-62.  So a loss is good to some 2^-20 weight T^2 beside its own last bits.  At columns that no entry names,
 * what is below 2^-126 of the row's largest weight is 0.
 *
 * stats: two floats per row for hcclx_distill_grad_plan_create, 8-byte aligned.  dlogits: one pointer per rank, rows as far apart as
 * the logits', and each may be that rank's logits.  A program that knows the weights before the loss gets the gradients in the same
 * launch that way, without another pass over the logits. */
typedef struct {
    uint32_t k;             /* 1 .. HCCLX_TOP_MAX */
    int dtype;              /* fp32, fp16 or bf16 */
    const void *logits;     /* rows x k */
    const int32_t *indices; /* rows x k */
    float temperature;      /* 1e-6 .. 1e6 */
} hcclx_teacher_t;
typedef struct {
    hcclx_logits_t logits;
    hcclx_teacher_t teacher;
    const float *weight;   /* rows; NULL: 1 */
    float *loss;           /* rows; NULL: not wanted */
    float *stats;          /* rows x 2; NULL: not wanted */
    void *const *dlogits;  /* NULL: not wanted */
} hcclx_distill_t;
int hcclx_distill_plan_create(const hcclx_distill_t *distill, hcclx_plan_t **plan);

/* Its gradient alone, from what the loss left in stats for the same logits and teacher.  weight: what the row's gradient is
 * multiplied with, the loss's weight times what reaches the loss.  A row that the loss passed over for its weight of 0 has
 * gradients 0 whatever its weight is here. */
typedef struct {
    hcclx_logits_t logits;
    hcclx_teacher_t teacher;
    const float *weight;
    const float *stats;
    void *const *dlogits;
} hcclx_distill_grad_t;
int hcclx_distill_grad_plan_create(const hcclx_distill_grad_t *distill, hcclx_plan_t **plan);

/* Draws a token for every row.  With w = exp((logit - the row's largest) / temperature), what stays of a row is
 *     of the order of hcclx_top_logits_t (descending, of equal logits the first)   the first top_k,
 *     of those the shortest beginning whose w are top_p of theirs or more          (one token at least),
 *     of those the ones with w >= min_p                                            (the first always);
 * and the token is the first, in order of the columns, at which the running sum of the w that stay is more than random times all of
 * them.  Settings are read on the device, one per row:
 *     temperature  0, negative or NaN: the row's first largest logit; NULL: 1
 *     top_k        0 or less, or as many as there are columns: all; NULL: all
 *     top_p        1 or more, or NaN: all; 0 or less: one; NULL: all
 *     min_p        0 or less, or NaN: all; more than 1 counts as 1; NULL: all
 *     random       in [0, 1) from the caller's generator, so that a draw is a function of its arguments (outside: the nearest end; NaN: 0)
 * NaN counts as -infinity and is never drawn; a row of nothing else gets token -1 and logprob -infinity.  Of +infinities one is drawn.
 * w are computed in 64 bits and summed as whole multiples, so that sums, and the token, do not go by their order or by the other rows of the plan:
 * of 2^-51 where all columns count (in a row without a filter, and for what top_p is a part of where there is no top_k), otherwise of 2^-38 or
 * less (2^-45 for 131072 columns).  What is less than half of that is never drawn. */
typedef struct {
    hcclx_logits_t logits;
    const float *temperature;
    const int32_t *top_k;
    const float *top_p;
    const float *min_p;
    const float *random;
    int32_t *token;  /* rows */
    float *logprob;  /* rows: log(w / the sum of what stays), of the token; NULL: not wanted */
} hcclx_sample_t;
int hcclx_sample_plan_create(const hcclx_sample_t *sample, hcclx_plan_t **plan);

#ifdef __cplusplus
}
#endif
#endif /* HCCL_AMD_HCCLX_OPS_H_ */
