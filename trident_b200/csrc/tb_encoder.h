// Host-side launchers of the query-encoder operators, and the helpers that pick their instances.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stddef.h>
#include <stdint.h>

#include <atomic>
#include <initializer_list>
#include <type_traits>

#include "tb_internal.h"
#include "trident_b200_encoder.h"

namespace tb {

template <class T> struct TypeIs { using type = T; };

// f(TypeIs<T>{}) for the element type `dtype`, checked by the caller.
template <class F>
cudaError_t with_type(int dtype, F&& f) {
    if (dtype == TRIDENT_F32) return f(TypeIs<float>{});
    if (dtype == TRIDENT_F16) return f(TypeIs<__half>{});
    return f(TypeIs<__nv_bfloat16>{});
}

// A matrix as its accesses see it.
struct Operand {
    const void* p;
    int64_t ld;
    int size;
};

// The widest access, in elements (a power of two <= most), that every row of every operand allows: the
// base, the row stride and D are whole multiples of it (of 16 bytes where it is wider than that).
inline int wide_elements(std::initializer_list<Operand> ops, int64_t D, int most) {
    int v = most;
    for (; v > 1; v /= 2) {
        bool ok = D % v == 0;
        for (const Operand& o : ops) {
            const int64_t bytes = v * o.size < 16 ? v * o.size : 16;
            ok = ok && ((uintptr_t)o.p % bytes) == 0 && (o.ld * o.size) % bytes == 0;
        }
        if (ok) break;
    }
    return v;
}

// f(integral_constant<vec>) for vec in {1, 2, 4, 8} up to MOST.
template <int MOST, class F>
void with_vec(int vec, F&& f) {
    if constexpr (MOST >= 8)
        if (vec == 8) return f(std::integral_constant<int, 8>{});
    if (vec == 4) return f(std::integral_constant<int, 4>{});
    if (vec == 2) return f(std::integral_constant<int, 2>{});
    f(std::integral_constant<int, 1>{});
}

// Lets KERNEL have `bytes` of dynamic shared memory on the current device (48 KB in all, its own static
// memory among them, need no leave). What it was last given on a device is remembered.
template <auto KERNEL>
cudaError_t allow_smem(size_t bytes) {
    if (bytes <= 40 * 1024) return cudaSuccess;
    static std::atomic<size_t> given[64];
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    const bool known = dev >= 0 && dev < 64;
    if (known && given[dev].load(std::memory_order_relaxed) >= bytes) return cudaSuccess;
    e = cudaFuncSetAttribute(KERNEL, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes);
    if (e == cudaSuccess && known) given[dev].store(bytes, std::memory_order_relaxed);
    return e;
}

// Launches a kernel that may come onto the GPU before the one before it on the stream has ended (it waits for
// that end itself, wait_for_previous(), before it touches memory): the gap between two launches is hidden.
template <class... P, class... A>
cudaError_t launch_chained(void (*kernel)(P...), int64_t grid, int block, size_t smem, cudaStream_t st, A... args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)grid);
    cfg.blockDim = dim3(block);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute attr;
    attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr.val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, kernel, P(args)...);
}

cudaError_t launch_embed_lookup(const void* table, int dtype, int64_t V, int D, int64_t ld, const void* ids, int id64,
                                int64_t count, float scale, void* out, int64_t ld_out, int32_t* status, cudaStream_t st);
size_t embed_grad_workspace(int64_t T, int D);
cudaError_t launch_embed_grad(const void* grad, int dtype, int64_t ld, const void* ids, int id64, int64_t count, int64_t V,
                              int D, float scale, int accumulate, void* out, int out_dtype, int64_t ld_out,
                              void* workspace, int32_t* status, int* launches, cudaStream_t st);

cudaError_t launch_layer_norm(const void* x, int dtype, int64_t rows, int D, int64_t ld_x, const void* weight,
                              const void* bias, int param_dtype, float eps, void* y, int64_t ld_y, float* mean,
                              float* rstd, cudaStream_t st);
size_t layer_norm_grad_workspace(int64_t rows, int D);
cudaError_t launch_layer_norm_grad(const void* dy, int64_t ld_dy, const void* x, int64_t ld_x, int dtype, int64_t rows,
                                   int D, const void* weight, int param_dtype, const float* mean, const float* rstd,
                                   void* dx, int64_t ld_dx, void* dweight, void* dbias, void* workspace, int* launches,
                                   cudaStream_t st);

cudaError_t launch_adamw(const trident_adamw_tensor* tensors, int count, const trident_adamw_config& cfg, bool master,
                         int* launches, cudaStream_t st);

// Counts kernel launches for trident_launch_count, and turns a CUDA error into a status (tb_abi.cu).
void count_launches(int n);
int cuda_status(cudaError_t e, const char* where);

}  // namespace tb
