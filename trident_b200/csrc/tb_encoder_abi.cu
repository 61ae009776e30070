// C ABI of the query-encoder operators (trident_b200_encoder.h): argument checks and launches.
#include <stdarg.h>
#include <stdio.h>

#include "tb_encoder.h"

using namespace tb;

namespace {

int fail(int code, const char* fmt, ...) {
    char buf[512];
    va_list ap;
    va_start(ap, fmt);
    vsnprintf(buf, sizeof(buf), fmt, ap);
    va_end(ap);
    return record_error(code, buf);
}

int elem_size(int dtype) { return dtype == TRIDENT_F32 ? 4 : 2; }

int check_dtype(const char* what, int32_t dtype) {
    if (dtype != TRIDENT_F32 && dtype != TRIDENT_F16 && dtype != TRIDENT_BF16)
        return fail(TRIDENT_ERR_UNSUPPORTED, "%s=%d (supported: 0 f32, 1 f16, 2 bf16)", what, dtype);
    return TRIDENT_OK;
}

// A matrix of `rows` rows: there if it has any element, aligned to its type, its stride at least D.
int check_matrix(const char* what, const void* p, int size, int64_t rows, int64_t D, int64_t ld) {
    if (rows == 0) return TRIDENT_OK;
    if (!p) return fail(TRIDENT_ERR_INVALID, "%s is NULL", what);
    if ((uintptr_t)p % size) return fail(TRIDENT_ERR_INVALID, "%s is not aligned to its type", what);
    if (ld < D) return fail(TRIDENT_ERR_INVALID, "row stride %lld of %s < D=%lld", (long long)ld, what, (long long)D);
    if (ld > ((int64_t)1 << 60) / size / (rows > 0 ? rows : 1))
        return fail(TRIDENT_ERR_UNSUPPORTED, "%s spans too many bytes", what);
    return TRIDENT_OK;
}

int check_vector(const char* what, const void* p, int size, bool needed) {
    if (!p && needed) return fail(TRIDENT_ERR_INVALID, "%s is NULL", what);
    if ((uintptr_t)p % size) return fail(TRIDENT_ERR_INVALID, "%s is not aligned to its type", what);
    return TRIDENT_OK;
}

int check_workspace(const void* ws, size_t bytes, size_t need) {
    if (need == 0) return TRIDENT_OK;
    if (!ws || bytes < need) return fail(TRIDENT_ERR_WORKSPACE, "workspace of %zu bytes < %zu needed", ws ? bytes : 0, need);
    if ((uintptr_t)ws & 255) return fail(TRIDENT_ERR_INVALID, "workspace must be 256-byte aligned");
    return TRIDENT_OK;
}

int check_ids(const void* ids, int32_t id_bits, int64_t T, int64_t V, int32_t D, const int32_t* status) {
    constexpr int64_t kMost = ((int64_t)1 << 31) - 1;
    if (id_bits != 32 && id_bits != 64) return fail(TRIDENT_ERR_UNSUPPORTED, "id_bits=%d (supported: 32, 64)", id_bits);
    if (T < 0 || T > kMost - 4096) return fail(TRIDENT_ERR_UNSUPPORTED, "T=%lld outside [0, 2^31 - 4096)", (long long)T);
    if (V < 0 || V > kMost) return fail(TRIDENT_ERR_UNSUPPORTED, "V=%lld outside [0, 2^31)", (long long)V);
    if (D < 1) return fail(TRIDENT_ERR_INVALID, "D=%d", D);
    int rc = check_vector("ids", ids, id_bits / 8, T > 0);
    return rc ? rc : check_vector("dev_status", status, 4, false);
}

#define TB_CHECK(expr)              \
    do {                            \
        const int _rc = (expr);     \
        if (_rc) return _rc;        \
    } while (0)

}  // namespace

extern "C" {

int trident_embed_lookup(const void* table, int32_t dtype, int64_t V, int32_t D, int64_t ld_table, const void* ids,
                         int32_t id_bits, int64_t T, float scale, void* out, int64_t ld_out, int32_t* dev_status,
                         void* stream) {
    TB_CHECK(check_dtype("dtype", dtype));
    TB_CHECK(check_ids(ids, id_bits, T, V, D, dev_status));
    TB_CHECK(check_matrix("table", table, elem_size(dtype), V, D, ld_table));
    TB_CHECK(check_matrix("out", out, elem_size(dtype), T, D, ld_out));
    if (T == 0) return TRIDENT_OK;
    count_launches(1);
    return cuda_status(launch_embed_lookup(table, dtype, V, D, ld_table, ids, id_bits == 64, T, scale, out, ld_out,
                                           dev_status, (cudaStream_t)stream),
                       "embed_lookup");
}

int trident_embed_grad_workspace_size(int64_t T, int64_t V, int32_t D, size_t* bytes) {
    TB_CHECK(check_ids(reinterpret_cast<const void*>(16), 32, T, V, D, nullptr));
    if (!bytes) return fail(TRIDENT_ERR_INVALID, "bytes is NULL");
    *bytes = embed_grad_workspace(T, D);
    return TRIDENT_OK;
}

int trident_embed_grad(const void* grad, int32_t dtype, int64_t ld_grad, const void* ids, int32_t id_bits, int64_t T,
                       int64_t V, int32_t D, float scale, int32_t accumulate, void* out, int32_t out_dtype, int64_t ld_out,
                       void* workspace, size_t workspace_bytes, int32_t* dev_status, void* stream) {
    TB_CHECK(check_dtype("dtype", dtype));
    if (out_dtype != dtype && out_dtype != TRIDENT_F32)
        return fail(TRIDENT_ERR_UNSUPPORTED, "out_dtype=%d (supported: dtype=%d, 0 f32)", out_dtype, dtype);
    if (accumulate != 0 && accumulate != 1) return fail(TRIDENT_ERR_INVALID, "accumulate=%d", accumulate);
    TB_CHECK(check_ids(ids, id_bits, T, V, D, dev_status));
    TB_CHECK(check_matrix("grad", grad, elem_size(dtype), T, D, ld_grad));
    TB_CHECK(check_matrix("out", out, elem_size(out_dtype), V, D, ld_out));
    TB_CHECK(check_workspace(workspace, workspace_bytes, embed_grad_workspace(T, D)));
    if (V == 0 && T == 0) return TRIDENT_OK;
    int launches = 0;
    const cudaError_t e = launch_embed_grad(grad, dtype, ld_grad, ids, id_bits == 64, T, V, D, scale, accumulate, out,
                                            out_dtype, ld_out, workspace, dev_status, &launches, (cudaStream_t)stream);
    count_launches(launches);
    if (e == cudaErrorInvalidConfiguration) return fail(TRIDENT_ERR_UNSUPPORTED, "T=%lld rows of D=%d are too many", (long long)T, D);
    return cuda_status(e, "embed_grad");
}

static int check_norm(int32_t dtype, int32_t param_dtype, int64_t rows, int32_t D) {
    TB_CHECK(check_dtype("dtype", dtype));
    if (param_dtype != dtype && param_dtype != TRIDENT_F32)
        return fail(TRIDENT_ERR_UNSUPPORTED, "param_dtype=%d (supported: dtype=%d, 0 f32)", param_dtype, dtype);
    if (rows < 0 || rows >= (int64_t)1 << 31) return fail(TRIDENT_ERR_UNSUPPORTED, "rows=%lld outside [0, 2^31)", (long long)rows);
    if (D < 1) return fail(TRIDENT_ERR_INVALID, "D=%d", D);
    return TRIDENT_OK;
}

int trident_layer_norm(const void* x, int32_t dtype, int64_t rows, int32_t D, int64_t ld_x, const void* weight,
                       const void* bias, int32_t param_dtype, float eps, void* y, int64_t ld_y, float* mean, float* rstd,
                       void* stream) {
    TB_CHECK(check_norm(dtype, param_dtype, rows, D));
    TB_CHECK(check_matrix("x", x, elem_size(dtype), rows, D, ld_x));
    TB_CHECK(check_matrix("y", y, elem_size(dtype), rows, D, ld_y));
    TB_CHECK(check_vector("weight", weight, elem_size(param_dtype), false));
    TB_CHECK(check_vector("bias", bias, elem_size(param_dtype), false));
    TB_CHECK(check_vector("mean", mean, 4, false));
    TB_CHECK(check_vector("rstd", rstd, 4, false));
    if (!(eps >= 0.0f)) return fail(TRIDENT_ERR_INVALID, "eps=%g", (double)eps);
    if (rows == 0) return TRIDENT_OK;
    count_launches(1);
    return cuda_status(launch_layer_norm(x, dtype, rows, D, ld_x, weight, bias, param_dtype, eps, y, ld_y, mean, rstd,
                                         (cudaStream_t)stream),
                       "layer_norm");
}

int trident_layer_norm_grad_workspace_size(int64_t rows, int32_t D, size_t* bytes) {
    TB_CHECK(check_norm(TRIDENT_F32, TRIDENT_F32, rows, D));
    if (!bytes) return fail(TRIDENT_ERR_INVALID, "bytes is NULL");
    *bytes = layer_norm_grad_workspace(rows, D);
    return TRIDENT_OK;
}

int trident_layer_norm_grad(const void* dy, int64_t ld_dy, const void* x, int64_t ld_x, int32_t dtype, int64_t rows, int32_t D,
                            const void* weight, int32_t param_dtype, const float* mean, const float* rstd, void* dx,
                            int64_t ld_dx, void* dweight, void* dbias, void* workspace, size_t workspace_bytes, void* stream) {
    TB_CHECK(check_norm(dtype, param_dtype, rows, D));
    TB_CHECK(check_matrix("dy", dy, elem_size(dtype), rows, D, ld_dy));
    TB_CHECK(check_matrix("x", x, elem_size(dtype), rows, D, ld_x));
    TB_CHECK(check_matrix("dx", dx, elem_size(dtype), rows, D, ld_dx));
    TB_CHECK(check_vector("weight", weight, elem_size(param_dtype), false));
    TB_CHECK(check_vector("mean", mean, 4, rows > 0));
    TB_CHECK(check_vector("rstd", rstd, 4, rows > 0));
    TB_CHECK(check_vector("dweight", dweight, elem_size(param_dtype), false));
    TB_CHECK(check_vector("dbias", dbias, elem_size(param_dtype), false));
    TB_CHECK(check_workspace(workspace, workspace_bytes, layer_norm_grad_workspace(rows, D)));
    int launches = 0;
    const cudaError_t e = launch_layer_norm_grad(dy, ld_dy, x, ld_x, dtype, rows, D, weight, param_dtype, mean, rstd, dx, ld_dx,
                                                 dweight, dbias, workspace, &launches, (cudaStream_t)stream);
    count_launches(launches);
    return cuda_status(e, "layer_norm_grad");
}

int trident_adamw_step(const trident_adamw_tensor* tensors, int32_t count, const trident_adamw_config* c, void* stream) {
    if (!c) return fail(TRIDENT_ERR_INVALID, "config is NULL");
    TB_CHECK(check_dtype("param_dtype", c->param_dtype));
    if (c->grad_dtype != c->param_dtype && c->grad_dtype != TRIDENT_F32)
        return fail(TRIDENT_ERR_UNSUPPORTED, "grad_dtype=%d (supported: param_dtype=%d, 0 f32)", c->grad_dtype, c->param_dtype);
    if (c->state_bits != 32 && c->state_bits != 8)
        return fail(TRIDENT_ERR_UNSUPPORTED, "state_bits=%d (supported: 32, 8)", c->state_bits);
    if (c->step < 1) return fail(TRIDENT_ERR_INVALID, "step=%lld", (long long)c->step);
    if (!(c->beta1 >= 0.0 && c->beta1 < 1.0) || !(c->beta2 >= 0.0 && c->beta2 < 1.0))
        return fail(TRIDENT_ERR_INVALID, "beta1=%g beta2=%g outside [0, 1)", c->beta1, c->beta2);
    if (!(c->eps >= 0.0) || !(c->weight_decay >= 0.0) || !(c->lr >= 0.0))
        return fail(TRIDENT_ERR_INVALID, "lr=%g eps=%g weight_decay=%g", c->lr, c->eps, c->weight_decay);
    TB_CHECK(check_vector("grad_scale", c->grad_scale, 4, false));
    if (count < 0) return fail(TRIDENT_ERR_INVALID, "count=%d", count);
    if (count == 0) return TRIDENT_OK;
    if (!tensors) return fail(TRIDENT_ERR_INVALID, "tensors is NULL");
    const bool bits8 = c->state_bits == 8;
    const int state = bits8 ? 1 : 4;
    bool master = false;
    for (int32_t i = 0; i < count; ++i) master = master || (tensors[i].n > 0 && tensors[i].master);
    if (master && c->param_dtype == TRIDENT_F32) return fail(TRIDENT_ERR_INVALID, "a float32 parameter has no master copy");
    uint64_t blocks = 0;
    for (int32_t i = 0; i < count; ++i) {
        const trident_adamw_tensor& t = tensors[i];
        if (t.n < 0) return fail(TRIDENT_ERR_INVALID, "tensor %d: n=%lld", i, (long long)t.n);
        if (t.n > 0 && (t.master != nullptr) != master) return fail(TRIDENT_ERR_INVALID, "tensor %d: master copies for all tensors or none", i);
        blocks += ((uint64_t)t.n + TRIDENT_ADAMW_BLOCK - 1) / TRIDENT_ADAMW_BLOCK;
        if (blocks >= (uint64_t)1 << 31) return fail(TRIDENT_ERR_UNSUPPORTED, "more than 2^31 blocks of %d values", TRIDENT_ADAMW_BLOCK);
        if (t.n == 0) continue;
        const void* ptrs[] = {t.param, t.grad, t.m, t.v, bits8 ? t.m_scale : t.m, bits8 ? t.v_scale : t.v};
        const int sizes[] = {elem_size(c->param_dtype), elem_size(c->grad_dtype), state, state, 4, 4};
        const char* names[] = {"param", "grad", "m", "v", "m_scale", "v_scale"};
        for (int k = 0; k < 6; ++k) {
            if (!ptrs[k]) return fail(TRIDENT_ERR_INVALID, "tensor %d: %s is NULL", i, names[k]);
            if ((uintptr_t)ptrs[k] % sizes[k]) return fail(TRIDENT_ERR_INVALID, "tensor %d: %s is not aligned to its type", i, names[k]);
        }
        if ((uintptr_t)t.master % 4) return fail(TRIDENT_ERR_INVALID, "tensor %d: master is not aligned to its type", i);
    }
    int launches = 0;
    const cudaError_t e = launch_adamw(tensors, count, *c, master, &launches, (cudaStream_t)stream);
    count_launches(launches);
    return cuda_status(e, "adamw_step");
}

}  // extern "C"
