// Layer norm and its backward pass.
//
// Forward: mean = sum x / D, rstd = 1 / sqrt(sum (x - mean)^2 / D + eps), y = (x - mean) rstd w + b. A row
// stays in the registers of its warps (32 columns a lane), so the centred second moment costs no second
// read and loses nothing to cancellation.
//
// Backward: xh = (x - mean) rstd, g = dy w; dx = rstd (g - sum g / D - xh sum(g xh) / D); dw = sum_rows dy xh,
// db = sum_rows dy. A thread owns 8 columns for all the rows that its group of warps takes, so that the
// columns' sums stay in registers; each group leaves one partial row and a second kernel adds the partials
// in order.
#include "tb_encoder.h"
#include "tb_vec.cuh"

namespace tb {

namespace {

constexpr int kLaneCols = 32;     // forward: columns of a row that a lane holds
constexpr int kFwdMaxWarps = 8;   // ... up to 8 warps a row: D <= 8192
constexpr int kGradCols = 8;      // backward: columns that a thread owns
constexpr int kGradRows = 4;      // rows in flight in a group
constexpr int kGradMaxWarps = 16; // D <= 4096

int pow2_at_least(int64_t x) {
    int p = 1;
    while (p < x) p *= 2;
    return p;
}

// Sum of v over the `warps` warps of this thread's row (slot: their shared words; every thread of the
// block calls).
__device__ __forceinline__ float row_sum(float v, float* slot, int warps, int warp_in_row) {
    v = warp_sum(v);
    if (warps == 1) return v;
    if ((threadIdx.x & 31) == 0) slot[warp_in_row] = v;
    __syncthreads();
    float s = 0.0f;
    for (int w = 0; w < warps; ++w) s += slot[w];
    __syncthreads();
    return s;
}

// ---- forward

// NV wide columns of VEC elements a lane; `warps` warps a row, 8 warps a block.
template <class T, class P, int VEC, int NV>
__global__ void __launch_bounds__(256) norm_kernel(const T* x, int64_t rows, int D, int64_t ld_x, const P* __restrict__ w,
                                                   const P* __restrict__ b, float eps, T* y, int64_t ld_y, float* mean,
                                                   float* rstd, int warps) {
    __shared__ float slots[2][8];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int in_row = warp % warps, group = warp / warps;
    const int cols = D / VEC;
    const int64_t row = (int64_t)blockIdx.x * (8 / warps) + group;
    const bool live = row < rows;
    const float inv_d = 1.0f / (float)D;
    float f[NV * VEC];
    float s = 0.0f;
    Pack<T, VEC> p[NV];
#pragma unroll
    for (int k = 0; k < NV; ++k) {
        const int c = (k * warps + in_row) * 32 + lane;
        if (live && c < cols) p[k] = Pack<T, VEC>::load(x + row * ld_x + (int64_t)c * VEC);
    }
#pragma unroll
    for (int k = 0; k < NV; ++k) {
        const int c = (k * warps + in_row) * 32 + lane;
        if (live && c < cols) {
            p[k].get(f + k * VEC);
#pragma unroll
            for (int i = 0; i < VEC; ++i) s += f[k * VEC + i];
        }
    }
    const float mu = row_sum(s, slots[0] + group * warps, warps, in_row) * inv_d;
    s = 0.0f;
#pragma unroll
    for (int k = 0; k < NV; ++k) {
        const int c = (k * warps + in_row) * 32 + lane;
        if (live && c < cols) {
#pragma unroll
            for (int i = 0; i < VEC; ++i) {
                f[k * VEC + i] -= mu;
                s = fmaf(f[k * VEC + i], f[k * VEC + i], s);
            }
        }
    }
    const float r = 1.0f / sqrtf(row_sum(s, slots[1] + group * warps, warps, in_row) * inv_d + eps);
    if (!live) return;
#pragma unroll
    for (int k = 0; k < NV; ++k) {
        const int c = (k * warps + in_row) * 32 + lane;
        if (c >= cols) continue;
        float wf[VEC], bf[VEC];
        if (w) load_n<P, VEC>(w + (int64_t)c * VEC, wf);
        if (b) load_n<P, VEC>(b + (int64_t)c * VEC, bf);
        float* g = f + k * VEC;
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
            g[i] *= r;
            if (w) g[i] *= wf[i];
            if (b) g[i] += bf[i];
        }
        Pack<T, VEC>::of(g).store(y + row * ld_y + (int64_t)c * VEC);
    }
    if (in_row == 0 && lane == 0) {
        if (mean) mean[row] = mu;
        if (rstd) rstd[row] = r;
    }
}

// Any D: one block a row, the row read once for each of the three steps (from L2 after the first).
template <class T, class P>
__global__ void __launch_bounds__(1024) norm_long_kernel(const T* x, int64_t rows, int D, int64_t ld_x, const P* __restrict__ w,
                                                         const P* __restrict__ b, float eps, T* y, int64_t ld_y, float* mean,
                                                         float* rstd) {
    __shared__ float slots[32];
    const int warp = threadIdx.x >> 5;
    const float inv_d = 1.0f / (float)D;
    for (int64_t row = blockIdx.x; row < rows; row += gridDim.x) {
        const T* xr = x + row * ld_x;
        float s = 0.0f;
        for (int c = threadIdx.x; c < D; c += 1024) s += to_float(xr[c]);
        const float mu = row_sum(s, slots, 32, warp) * inv_d;
        s = 0.0f;
        for (int c = threadIdx.x; c < D; c += 1024) {
            const float d = to_float(xr[c]) - mu;
            s = fmaf(d, d, s);
        }
        const float r = 1.0f / sqrtf(row_sum(s, slots, 32, warp) * inv_d + eps);
        for (int c = threadIdx.x; c < D; c += 1024) {
            float v = (to_float(xr[c]) - mu) * r;
            if (w) v *= to_float(w[c]);
            if (b) v += to_float(b[c]);
            y[row * ld_y + c] = from_float<T>(v);
        }
        if (threadIdx.x == 0) {
            if (mean) mean[row] = mu;
            if (rstd) rstd[row] = r;
        }
    }
}

template <class T, class P>
cudaError_t norm_typed(const T* x, int64_t rows, int D, int64_t ld_x, const P* w, const P* b, float eps, T* y, int64_t ld_y,
                       float* mean, float* rstd, cudaStream_t st) {
    if (D > kLaneCols * 32 * kFwdMaxWarps) {
        const int64_t grid = rows < 65536 ? rows : 65536;
        norm_long_kernel<T, P><<<(unsigned)grid, 1024, 0, st>>>(x, rows, D, ld_x, w, b, eps, y, ld_y, mean, rstd);
        return cudaGetLastError();
    }
    constexpr int kVec = 16 / (int)sizeof(T);
    int vec = wide_elements({{x, ld_x, (int)sizeof(T)}, {y, ld_y, (int)sizeof(T)}, {w, 0, (int)sizeof(P)}, {b, 0, (int)sizeof(P)}},
                            D, kVec);
    if (vec < kVec) vec = 1;
    const int per_warp = kLaneCols * 32;
    const int warps = pow2_at_least((D + per_warp - 1) / per_warp);
    const int64_t per_block = 8 / warps;
    const int64_t grid = (rows + per_block - 1) / per_block;
    if (grid > 0x7fffffff) return cudaErrorInvalidConfiguration;
    const int nv = (D / vec + 32 * warps - 1) / (32 * warps);
    auto go = [&](auto v, auto k) {
        constexpr int VEC = decltype(v)::value, NV = decltype(k)::value;
        norm_kernel<T, P, VEC, NV><<<(unsigned)grid, 256, 0, st>>>(x, rows, D, ld_x, w, b, eps, y, ld_y, mean, rstd, warps);
    };
    auto pick = [&](auto v) {
        constexpr int VEC = decltype(v)::value;
        constexpr int MAX = kLaneCols / VEC;
        if constexpr (MAX >= 32)
            if (nv > 16) return go(v, std::integral_constant<int, 32>{});
        if constexpr (MAX >= 16)
            if (nv > 8) return go(v, std::integral_constant<int, 16>{});
        if constexpr (MAX >= 8)
            if (nv > 4) return go(v, std::integral_constant<int, 8>{});
        if (nv > 2) return go(v, std::integral_constant<int, 4>{});
        if (nv > 1) return go(v, std::integral_constant<int, 2>{});
        go(v, std::integral_constant<int, 1>{});
    };
    if (vec == kVec) pick(std::integral_constant<int, kVec>{});
    else pick(std::integral_constant<int, 1>{});
    return cudaGetLastError();
}

// ---- backward

// Groups of `warps` warps take turns of kGradRows rows; NV * VEC = kGradCols columns a thread.
template <class T, class P, int VEC>
__global__ void __launch_bounds__(32 * kGradMaxWarps) norm_grad_kernel(const T* dy, int64_t ld_dy, const T* __restrict__ x, int64_t ld_x, int64_t rows, int D,
                                 const P* __restrict__ w, const float* __restrict__ mean, const float* __restrict__ rstd,
                                 T* dx, int64_t ld_dx, float* __restrict__ part, int64_t ld_part, int warps) {
    constexpr int NV = kGradCols / VEC;
    __shared__ float2 slots[2][kGradMaxWarps][kGradRows];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int in_row = warp % warps, group = warp / warps;
    const int groups_here = blockDim.x / 32 / warps;
    const int64_t groups = (int64_t)gridDim.x * groups_here, me = (int64_t)blockIdx.x * groups_here + group;
    const int cols = D / VEC;
    const float inv_d = 1.0f / (float)D;
    int col[NV];
    float wf[kGradCols], dw[kGradCols] = {}, db[kGradCols] = {};
#pragma unroll
    for (int k = 0; k < NV; ++k) {
        col[k] = (k * warps + in_row) * 32 + lane;
#pragma unroll
        for (int i = 0; i < VEC; ++i) wf[k * VEC + i] = 1.0f;
        if (w && col[k] < cols) load_n<P, VEC>(w + (int64_t)col[k] * VEC, wf + k * VEC);
    }
    const int64_t steps = (rows + groups * kGradRows - 1) / (groups * kGradRows);  // the same for every group
    for (int64_t t = 0; t < steps; ++t) {
        const int64_t r0 = (t * groups + me) * kGradRows;
        Pack<T, VEC> px[kGradRows][NV], pg[kGradRows][NV];
        float mu[kGradRows], rs[kGradRows];
#pragma unroll
        for (int r = 0; r < kGradRows; ++r) {
            if (r0 + r >= rows) continue;
            mu[r] = mean[r0 + r];
            rs[r] = rstd[r0 + r];
#pragma unroll
            for (int k = 0; k < NV; ++k) {
                if (col[k] >= cols) continue;
                px[r][k] = Pack<T, VEC>::load(x + (r0 + r) * ld_x + (int64_t)col[k] * VEC);
                pg[r][k] = Pack<T, VEC>::load(dy + (r0 + r) * ld_dy + (int64_t)col[k] * VEC);
            }
        }
        float s1[kGradRows], s2[kGradRows];
#pragma unroll
        for (int r = 0; r < kGradRows; ++r) {
            s1[r] = s2[r] = 0.0f;
            if (r0 + r >= rows) continue;
#pragma unroll
            for (int k = 0; k < NV; ++k) {
                if (col[k] >= cols) continue;
                float xf[VEC], gf[VEC];
                px[r][k].get(xf);
                pg[r][k].get(gf);
#pragma unroll
                for (int i = 0; i < VEC; ++i) {
                    const float xh = (xf[i] - mu[r]) * rs[r];
                    const float g = gf[i] * wf[k * VEC + i];
                    dw[k * VEC + i] = fmaf(gf[i], xh, dw[k * VEC + i]);
                    db[k * VEC + i] += gf[i];
                    s1[r] += g;
                    s2[r] = fmaf(g, xh, s2[r]);
                }
            }
        }
#pragma unroll
        for (int r = 0; r < kGradRows; ++r) {
            s1[r] = warp_sum(s1[r]);
            s2[r] = warp_sum(s2[r]);
        }
        if (warps > 1) {  // two sets of slots in turn: one barrier a step
            if (lane == 0) {
#pragma unroll
                for (int r = 0; r < kGradRows; ++r) slots[t & 1][warp][r] = make_float2(s1[r], s2[r]);
            }
            __syncthreads();
#pragma unroll
            for (int r = 0; r < kGradRows; ++r) {
                s1[r] = s2[r] = 0.0f;
                for (int q = 0; q < warps; ++q) {
                    const float2 v = slots[t & 1][group * warps + q][r];
                    s1[r] += v.x;
                    s2[r] += v.y;
                }
            }
        }
#pragma unroll
        for (int r = 0; r < kGradRows; ++r) {
            if (r0 + r >= rows) continue;
            const float c1 = s1[r] * inv_d, c2 = s2[r] * inv_d;
#pragma unroll
            for (int k = 0; k < NV; ++k) {
                if (col[k] >= cols) continue;
                float xf[VEC], gf[VEC];
                px[r][k].get(xf);
                pg[r][k].get(gf);
#pragma unroll
                for (int i = 0; i < VEC; ++i) {
                    const float xh = (xf[i] - mu[r]) * rs[r];
                    gf[i] = rs[r] * (gf[i] * wf[k * VEC + i] - c1 - xh * c2);
                }
                Pack<T, VEC>::of(gf).store(dx + (r0 + r) * ld_dx + (int64_t)col[k] * VEC);
            }
        }
    }
    float* pw = part + me * 2 * ld_part;
#pragma unroll
    for (int k = 0; k < NV; ++k) {
        if (col[k] >= cols) continue;
        store_n<float, VEC>(pw + (int64_t)col[k] * VEC, dw + k * VEC);
        store_n<float, VEC>(pw + ld_part + (int64_t)col[k] * VEC, db + k * VEC);
    }
}

// dw and db (blockIdx.y) of 32 columns a block: 32 lanes of partial rows each, added in order.
template <class P>
__global__ void __launch_bounds__(1024) norm_grad_sum_kernel(const float* __restrict__ part, int64_t parts, int64_t ld_part,
                                                             int D, P* dw, P* db) {
    __shared__ float s[32][33];
    P* out = blockIdx.y ? db : dw;
    if (!out) return;
    const int tx = threadIdx.x & 31, ty = threadIdx.x >> 5;
    const int c = blockIdx.x * 32 + tx;
    float acc = 0.0f;
    if (c < D) {
        const float* p = part + blockIdx.y * ld_part + c;
#pragma unroll 8
        for (int64_t q = ty; q < parts; q += 32) acc += p[q * 2 * ld_part];
    }
    s[ty][tx] = acc;
    __syncthreads();
    acc = warp_sum(s[tx][ty]);  // column ty of the block
    const int cc = blockIdx.x * 32 + ty;
    if (tx == 0 && cc < D) out[cc] = from_float<P>(acc);
}

// Any D: the row's sums first, then dx; the columns' sums by norm_grad_columns_kernel.
template <class T, class P>
__global__ void __launch_bounds__(1024) norm_grad_long_kernel(const T* dy, int64_t ld_dy, const T* __restrict__ x, int64_t ld_x,
                                                              int64_t rows, int D, const P* __restrict__ w,
                                                              const float* __restrict__ mean, const float* __restrict__ rstd,
                                                              T* dx, int64_t ld_dx) {
    __shared__ float slots[2][32];
    const int warp = threadIdx.x >> 5;
    for (int64_t row = blockIdx.x; row < rows; row += gridDim.x) {
        const float mu = mean[row], rs = rstd[row];
        float s1 = 0.0f, s2 = 0.0f;
        for (int c = threadIdx.x; c < D; c += 1024) {
            const float g = to_float(dy[row * ld_dy + c]) * (w ? to_float(w[c]) : 1.0f);
            s1 += g;
            s2 = fmaf(g, (to_float(x[row * ld_x + c]) - mu) * rs, s2);
        }
        const float c1 = row_sum(s1, slots[0], 32, warp) / (float)D, c2 = row_sum(s2, slots[1], 32, warp) / (float)D;
        for (int c = threadIdx.x; c < D; c += 1024) {
            const float g = to_float(dy[row * ld_dy + c]) * (w ? to_float(w[c]) : 1.0f);
            dx[row * ld_dx + c] = from_float<T>(rs * (g - c1 - (to_float(x[row * ld_x + c]) - mu) * rs * c2));
        }
    }
}

// The partial column sums of the rows that block row blockIdx.y takes.
template <class T>
__global__ void __launch_bounds__(256) norm_grad_columns_kernel(const T* __restrict__ dy, int64_t ld_dy, const T* __restrict__ x,
                                                                int64_t ld_x, int64_t rows, int D, const float* __restrict__ mean,
                                                                const float* __restrict__ rstd, float* __restrict__ part,
                                                                int64_t ld_part) {
    const int c = blockIdx.x * 256 + threadIdx.x;
    if (c >= D) return;
    const int64_t lo = rows * blockIdx.y / gridDim.y, hi = rows * (blockIdx.y + 1) / gridDim.y;
    float dw = 0.0f, db = 0.0f;
#pragma unroll 4
    for (int64_t r = lo; r < hi; ++r) {
        const float g = to_float(dy[r * ld_dy + c]);
        dw = fmaf(g, (to_float(x[r * ld_x + c]) - mean[r]) * rstd[r], dw);
        db += g;
    }
    part[blockIdx.y * 2 * ld_part + c] = dw;
    part[(blockIdx.y * 2 + 1) * ld_part + c] = db;
}

constexpr int kLongParts = 64;  // partial rows of the any-D path

struct GradShape {
    int warps;         // warps a row; 0: the any-D path
    int threads;
    int blocks;
    int64_t parts;     // partial rows
    int64_t ld_part;
};

GradShape grad_shape(int64_t rows, int D) {
    GradShape g;
    g.ld_part = (D + 3) / 4 * 4;
    const int per_warp = 32 * kGradCols;
    if (D > per_warp * kGradMaxWarps) {
        g.warps = g.threads = g.blocks = 0;
        g.parts = rows < kLongParts ? rows : kLongParts;
        return g;
    }
    g.warps = pow2_at_least((D + per_warp - 1) / per_warp);
    g.threads = g.warps * 32 < 128 ? 128 : g.warps * 32;
    const int groups = g.threads / 32 / g.warps;
    // four 128-thread blocks an SM at this kernel's registers; one step of kGradRows rows a group at least
    const int64_t most = (int64_t)num_sms() * (512 / g.threads > 0 ? 512 / g.threads : 1);
    const int64_t need = (rows + (int64_t)groups * kGradRows - 1) / ((int64_t)groups * kGradRows);
    g.blocks = (int)(need < most ? need : most);
    g.parts = (int64_t)g.blocks * groups;
    return g;
}

template <class T, class P>
cudaError_t grad_typed(const T* dy, int64_t ld_dy, const T* x, int64_t ld_x, int64_t rows, int D, const P* w, const float* mean,
                       const float* rstd, T* dx, int64_t ld_dx, P* dw, P* db, float* part, int* launches, cudaStream_t st) {
    const GradShape g = grad_shape(rows, D);
    if (rows > 0 && g.warps == 0) {
        norm_grad_columns_kernel<T><<<dim3((D + 255) / 256, (unsigned)g.parts), 256, 0, st>>>(dy, ld_dy, x, ld_x, rows, D, mean, rstd,
                                                                                             part, g.ld_part);
        const int64_t grid = rows < 65536 ? rows : 65536;
        norm_grad_long_kernel<T, P><<<(unsigned)grid, 1024, 0, st>>>(dy, ld_dy, x, ld_x, rows, D, w, mean, rstd, dx, ld_dx);
        *launches += 2;
    } else if (rows > 0) {
        constexpr int kVec = 16 / (int)sizeof(T) < kGradCols ? 16 / (int)sizeof(T) : kGradCols;
        const int es = (int)sizeof(T);
        const int vec = wide_elements({{x, ld_x, es}, {dy, ld_dy, es}, {dx, ld_dx, es}, {w, 0, (int)sizeof(P)}}, D, kVec);
        if (vec == kVec)
            norm_grad_kernel<T, P, kVec><<<g.blocks, g.threads, 0, st>>>(dy, ld_dy, x, ld_x, rows, D, w, mean, rstd, dx, ld_dx,
                                                                        part, g.ld_part, g.warps);
        else
            norm_grad_kernel<T, P, 1><<<g.blocks, g.threads, 0, st>>>(dy, ld_dy, x, ld_x, rows, D, w, mean, rstd, dx, ld_dx,
                                                                     part, g.ld_part, g.warps);
        *launches += 1;
    }
    if (dw || db) {
        norm_grad_sum_kernel<P><<<dim3((D + 31) / 32, 2), 1024, 0, st>>>(part, rows > 0 ? g.parts : 0, g.ld_part, D, dw, db);
        *launches += 1;
    }
    return cudaGetLastError();
}

}  // namespace

cudaError_t launch_layer_norm(const void* x, int dtype, int64_t rows, int D, int64_t ld_x, const void* weight, const void* bias,
                              int param_dtype, float eps, void* y, int64_t ld_y, float* mean, float* rstd, cudaStream_t st) {
    return with_type(dtype, [&](auto t) {
        using T = typename decltype(t)::type;
        const T* xt = static_cast<const T*>(x);
        T* yt = static_cast<T*>(y);
        if (param_dtype == TRIDENT_F32)
            return norm_typed<T, float>(xt, rows, D, ld_x, static_cast<const float*>(weight), static_cast<const float*>(bias), eps,
                                        yt, ld_y, mean, rstd, st);
        return norm_typed<T, T>(xt, rows, D, ld_x, static_cast<const T*>(weight), static_cast<const T*>(bias), eps, yt, ld_y, mean,
                                rstd, st);
    });
}

size_t layer_norm_grad_workspace(int64_t rows, int D) {
    const GradShape g = grad_shape(rows, D);
    return (size_t)(g.parts > 0 ? g.parts : 1) * 2 * g.ld_part * sizeof(float);
}

cudaError_t launch_layer_norm_grad(const void* dy, int64_t ld_dy, const void* x, int64_t ld_x, int dtype, int64_t rows, int D,
                                   const void* weight, int param_dtype, const float* mean, const float* rstd, void* dx,
                                   int64_t ld_dx, void* dweight, void* dbias, void* workspace, int* launches, cudaStream_t st) {
    return with_type(dtype, [&](auto t) {
        using T = typename decltype(t)::type;
        const T *dyt = static_cast<const T*>(dy), *xt = static_cast<const T*>(x);
        float* part = static_cast<float*>(workspace);
        if (param_dtype == TRIDENT_F32)
            return grad_typed<T, float>(dyt, ld_dy, xt, ld_x, rows, D, static_cast<const float*>(weight), mean, rstd,
                                        static_cast<T*>(dx), ld_dx, static_cast<float*>(dweight), static_cast<float*>(dbias), part,
                                        launches, st);
        return grad_typed<T, T>(dyt, ld_dy, xt, ld_x, rows, D, static_cast<const T*>(weight), mean, rstd, static_cast<T*>(dx), ld_dx,
                                static_cast<T*>(dweight), static_cast<T*>(dbias), part, launches, st);
    });
}

}  // namespace tb
