/*
 * trident_b200 - C ABI of the query-encoder operators (sm_100a): embedding lookup and its gradient,
 * layer norm and its gradient, and an AdamW step over many tensors. They train and run a token-embedding
 * encoder in front of an index; the search itself is in trident_b200.h. The reference has no counterpart:
 * it takes its vectors as given.
 *
 * The conventions are those of trident_b200.h: status codes and trident_last_error(), work queued on
 * `stream`, every buffer owned by the caller, no device memory allocated. Row-major matrices take a row
 * stride `ld_*` in elements (>= D); pointers need the alignment of their type only (wider alignment makes
 * wider loads possible). All sums are held in 32 bits; results depend on the inputs and sizes alone, not
 * on the order in which blocks run.
 */
#ifndef TRIDENT_B200_ENCODER_H
#define TRIDENT_B200_ENCODER_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* Element types of the operators. */
enum trident_dtype { TRIDENT_F32 = 0, TRIDENT_F16 = 1, TRIDENT_BF16 = 2 };

/* Bit set in a `dev_status` word by an id that is neither -1 nor in [0, V). */
#define TRIDENT_STATUS_BAD_ID 4

/* out[t, :] = scale * table[ids[t], :], the product rounded once to the table's type.
 *   table [V, D] of `dtype`; ids [T] int32 or int64 (id_bits 32 or 64); out [T, D] of `dtype`.
 * An id of -1 (a padded token, or a missing search result) gives a row of zeros. Any other id outside
 * [0, V) gives a row of NaN and sets TRIDENT_STATUS_BAD_ID in *dev_status (one device int32, or NULL).
 * out must not overlap the table. */
int trident_embed_lookup(const void* table, int32_t dtype, int64_t V, int32_t D, int64_t ld_table, const void* ids,
                         int32_t id_bits, int64_t T, float scale, void* out, int64_t ld_out, int32_t* dev_status,
                         void* stream);

/* Workspace bytes of trident_embed_grad. */
int trident_embed_grad_workspace_size(int64_t T, int64_t V, int32_t D, size_t* bytes);

/* The lookup's gradient: out[v, :] = scale * sum over t with ids[t] = v of grad[t, :], or that sum added
 * to out[v, :] (accumulate = 1; rows that no id names are then not touched). Ids outside [0, V) give
 * nothing (-1 silently, others set TRIDENT_STATUS_BAD_ID). Each row's sum is taken in an order that the
 * ids alone fix, in 32 bits, and rounded once.
 *   grad [T, D] of `dtype`; out [V, D] of out_dtype (`dtype` or TRIDENT_F32); T, V < 2^31; the workspace
 *   is 256-byte aligned. */
int trident_embed_grad(const void* grad, int32_t dtype, int64_t ld_grad, const void* ids, int32_t id_bits, int64_t T,
                       int64_t V, int32_t D, float scale, int32_t accumulate, void* out, int32_t out_dtype,
                       int64_t ld_out, void* workspace, size_t workspace_bytes, int32_t* dev_status, void* stream);

/* Layer norm of each row: mean = sum x / D, rstd = 1 / sqrt(sum (x - mean)^2 / D + eps),
 * y = (x - mean) rstd weight + bias.
 *   x [rows, D], y [rows, D] of `dtype` (y may be x); weight, bias [D] of param_dtype (`dtype` or
 *   TRIDENT_F32; NULL: 1 and 0); mean, rstd [rows] float32 (both may be NULL). */
int trident_layer_norm(const void* x, int32_t dtype, int64_t rows, int32_t D, int64_t ld_x, const void* weight,
                       const void* bias, int32_t param_dtype, float eps, void* y, int64_t ld_y, float* mean,
                       float* rstd, void* stream);

/* Workspace bytes of trident_layer_norm_grad. */
int trident_layer_norm_grad_workspace_size(int64_t rows, int32_t D, size_t* bytes);

/* Layer norm's backward pass. With xh = (x - mean) rstd and g = dy weight:
 *   dx = rstd (g - sum g / D - xh sum(g xh) / D), dweight = sum over rows of dy xh, dbias = of dy.
 * dx [rows, D] of `dtype` (may be dy); dweight, dbias [D] of param_dtype (either may be NULL); rows = 0
 * writes zeros to both. The workspace is 256-byte aligned. */
int trident_layer_norm_grad(const void* dy, int64_t ld_dy, const void* x, int64_t ld_x, int32_t dtype, int64_t rows,
                            int32_t D, const void* weight, int32_t param_dtype, const float* mean, const float* rstd,
                            void* dx, int64_t ld_dx, void* dweight, void* dbias, void* workspace,
                            size_t workspace_bytes, void* stream);

/* Elements that share the scales of an 8-bit state. */
#define TRIDENT_ADAMW_BLOCK 256

/* One tensor of an AdamW step: n elements each of
 *   param    param_dtype, updated;
 *   grad     grad_dtype, read;
 *   master   float32 or NULL: the parameter in 32 bits, updated in its place, param then being its rounding;
 *   m, v     the states: float32 m and v (state_bits = 32), or 8-bit e4m3 values (state_bits = 8) with
 *   m_scale, v_scale  float32, one for each TRIDENT_ADAMW_BLOCK elements: the state is
 *            m = e4m3(m) * m_scale and sqrt(v) = e4m3(v) * v_scale (the root, so that the 8 bits span
 *            twice as many octaves of v). */
typedef struct trident_adamw_tensor {
    void* param;
    const void* grad;
    float* master;
    void* m;
    void* v;
    float* m_scale;
    float* v_scale;
    int64_t n;
} trident_adamw_tensor;

typedef struct trident_adamw_config {
    int32_t param_dtype;
    int32_t grad_dtype;         /* param_dtype or TRIDENT_F32                             */
    int32_t state_bits;         /* 32 or 8                                                */
    uint32_t rounding_seed;     /* random bits of this step's 8-bit rounding              */
    int64_t step;               /* t >= 1, this step's number                             */
    double lr, beta1, beta2, eps, weight_decay;
    const float* grad_scale;    /* device float that multiplies every gradient, or NULL   */
} trident_adamw_config;

/* One AdamW step (decoupled weight decay) over `count` tensors in as few launches as their descriptors
 * fit (they travel as kernel arguments: `tensors` is read before the call returns):
 *   g = grad * grad_scale;  m = beta1 m + (1 - beta1) g;  v = beta2 v + (1 - beta2) g^2;
 *   p = p (1 - lr weight_decay) - lr / (1 - beta1^t) * m / (sqrt(v) / sqrt(1 - beta2^t) + eps),
 * in 32 bits. 8-bit states are decoded, updated and used in 32 bits, then encoded again with the scale
 * max / 448 of their block: m to the nearest value; sqrt(v) at random to one of its two neighbours so
 * that its mean is kept (to the nearest, the 1 - beta2 of a typical step would always round away), and
 * never to 0 unless v is 0. The random bits are a hash of rounding_seed and the element's place, counted
 * in whole blocks over the tensors in order. A block with a NaN or infinite state has a scale that is
 * not finite. Tensors must not overlap; n = 0 is allowed. */
int trident_adamw_step(const trident_adamw_tensor* tensors, int32_t count, const trident_adamw_config* config,
                       void* stream);

#ifdef __cplusplus
}
#endif

#endif /* TRIDENT_B200_ENCODER_H */
