// Layer norm and its backward pass.
//
// Forward: mean = sum x / D, rstd = 1 / sqrt(sum (x - mean)^2 / D + eps), y = (x - mean) rstd w + b. A row
// stays in the registers of its warps (at most 32 columns a lane), so the centred second moment costs no second
// read and loses nothing to cancellation. Few rows take norm_kernel (one row a warp, the least latency), many
// rows norm_rows_kernel; rows that start at no 16-byte place norm_ragged_kernel (100,000 rows of 1,001 bf16
// columns took 576 us by 2-byte loads, 106 us by it).
//
// Backward: xh = (x - mean) rstd, g = dy w; dx = rstd (g - sum g / D - xh sum(g xh) / D); dw = sum_rows dy xh,
// db = sum_rows dy. A thread owns 8 columns for all the rows that its group of warps takes, so that the
// columns' sums stay in registers; each block leaves one partial row and a second kernel adds the partials
// in order.
//
// Both read and write each element once and are bound by those bytes, the 16-bit types also by instructions: a
// row of 960 takes about 340 (forward, one warp) and 670 (backward, four warps). On a B200, of its measured copy
// bandwidth of 6.45 TB/s: 320,000 x 960 bf16 forward 197-210 us (91-97%), backward 321-347 us (82-89%); 100,000 x 960
// float32 backward 177 us (101%); 50,000 x 1001 float32 forward 78 us (80%), backward 123 us (76%); 100,000 x 1001
// bf16 106 us (58%) and 181 us (52%), where every element is a 2-byte access to shared memory. One warp a row in
// the backward pass, without barriers, spilled its 64 column sums a lane and took 574 us at 320,000 x 960.

#include "tb_encoder.h"
#include "tb_vec.cuh"

namespace tb {

namespace {

constexpr int kLaneCols = 32;     // forward: columns of a row that a lane holds
constexpr int kFwdMaxWarps = 8;   // ... up to 8 warps a row: D <= 8192
constexpr int kGradCols = 8;      // backward: columns that a thread owns
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

// A row of D elements at `row` into shared memory, as the 16-byte pieces that hold it: its first element ends
// up at to + (row & 15). Pieces reach into what lies around the row, but not beyond the `span` bytes from
// `base` that are the caller's; a piece that would is copied by elements. Thread `i` of `n`.
template <class T>
__device__ __forceinline__ void copy_pieces(char* to, const T* row, int D, const T* base, int64_t span, int i, int n) {
    const char* p = reinterpret_cast<const char*>(reinterpret_cast<uintptr_t>(row) & ~(uintptr_t)15);
    const char* b = reinterpret_cast<const char*>(base);
    const char* end = reinterpret_cast<const char*>(row + D);
    const int pieces = (int)((end - p + 15) >> 4);
    for (; i < pieces; i += n) {
        const char* q = p + i * 16;
        if (q >= b && q + 16 <= b + span) {
            copy16_async(to + i * 16, q);
        } else {
            for (int k = 0; k < 16; k += (int)sizeof(T))
                if (q + k >= reinterpret_cast<const char*>(row) && q + k < end)
                    *reinterpret_cast<T*>(to + i * 16 + k) = *reinterpret_cast<const T*>(q + k);
        }
    }
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

// Many rows of 16-byte columns. Warps stay and take turns of ROWS rows; the next rows are on their way into
// shared memory (each lane copies the columns that it will use, so no barrier is needed) while some are
// computed, and weight and bias wait in shared memory as float, read once for ROWS rows. LANES lanes a row
// for narrow rows, else `warps` warps.
constexpr int kStages = 3;
constexpr int kRowWarps = 16;  // warps of a block

template <int NV> constexpr int kRowsAtOnce = NV >= 4 ? 1 : NV == 2 ? 2 : 4;

template <class T, class P, int NV, int LANES>
__global__ void __launch_bounds__(32 * kRowWarps) norm_rows_kernel(const T* x, int64_t rows, int D, int64_t ld_x,
                                                                   const P* __restrict__ w, const P* __restrict__ b,
                                                                   float eps, T* y, int64_t ld_y, float* mean, float* rstd,
                                                                   int warps) {
    constexpr int VEC = 16 / (int)sizeof(T), H = VEC / 2, ROWS = kRowsAtOnce<NV>;
    extern __shared__ __align__(16) uint4 smem[];
    __shared__ float slots[2][kRowWarps][ROWS];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int in_row = LANES < 32 ? 0 : warp % warps;
    const int group = LANES < 32 ? threadIdx.x / LANES : warp / warps;
    const int groups = LANES < 32 ? kRowWarps * (32 / LANES) : kRowWarps / warps;
    const int sub = lane & (LANES - 1);
    const int cols = D / VEC;
    const float inv_d = 1.0f / (float)D;
    uint4* ring = smem + warp * (kStages * ROWS * NV * 32) + lane;  // [stage][row][k][lane of the warp]
    float4* pw = reinterpret_cast<float4*>(smem + kRowWarps * kStages * ROWS * NV * 32);  // [half][column] of 4 floats
    float4* pb = pw + (VEC / 4) * cols;
    for (int i = threadIdx.x; i < (VEC / 4) * cols; i += blockDim.x) {
        const int h = i / cols, c = i - h * cols;
        float f[4] = {1.0f, 1.0f, 1.0f, 1.0f}, g[4] = {};
        if (w) load_n<P, 4>(w + (int64_t)c * VEC + h * 4, f);
        if (b) load_n<P, 4>(b + (int64_t)c * VEC + h * 4, g);
        pw[i] = make_float4(f[0], f[1], f[2], f[3]);
        pb[i] = make_float4(g[0], g[1], g[2], g[3]);
    }
    const int col0 = in_row * LANES + sub, col_step = warps * LANES;
    bool on[NV];  // columns past the end read as 0 and are kept 0
#pragma unroll
    for (int k = 0; k < NV; ++k) on[k] = col0 + k * col_step < cols;
    const int64_t stride = (int64_t)gridDim.x * groups * ROWS;
    const int steps = (int)((rows + stride - 1) / stride);  // the same for every group
    int64_t row = ((int64_t)blockIdx.x * groups + group) * ROWS;
    int64_t ahead = row;                       // first row of the next copy
    const T* src = x + row * ld_x + (int64_t)col0 * VEC;
    int fetch_at = 0, take_at = 0;             // stages
    auto fetch = [&]() {
        const int64_t left = rows - ahead;
        uint4* to = ring + fetch_at * (ROWS * NV * 32);
        const T* p = src;
#pragma unroll
        for (int r = 0; r < ROWS; ++r) {
#pragma unroll
            for (int k = 0; k < NV; ++k)
                copy16_async_or_zero(to + (r * NV + k) * 32, r < left && on[k] ? p + k * col_step * VEC : x, r < left && on[k]);
            p += ld_x;
        }
        copy_commit();
        ahead += stride;
        src += stride * ld_x;
        fetch_at = fetch_at + 1 == kStages ? 0 : fetch_at + 1;
    };
#pragma unroll
    for (int t = 0; t < kStages - 1; ++t) fetch();
    __syncthreads();  // weight and bias
    auto sums = [&](float* v, int which) {  // over the row, of ROWS values
#pragma unroll
        for (int r = 0; r < ROWS; ++r) {
#pragma unroll
            for (int o = LANES / 2; o > 0; o >>= 1) v[r] += __shfl_xor_sync(0xffffffffu, v[r], o);
        }
        if (LANES < 32 || warps == 1) return;
        if (lane == 0) {
#pragma unroll
            for (int r = 0; r < ROWS; ++r) slots[which][warp][r] = v[r];
        }
        asm volatile("bar.sync %0, %1;" ::"r"(1 + group), "r"(warps * 32) : "memory");
#pragma unroll
        for (int r = 0; r < ROWS; ++r) v[r] = 0.0f;
        for (int q = 0; q < warps; ++q) {
#pragma unroll
            for (int r = 0; r < ROWS; ++r) v[r] += slots[which][group * warps + q][r];
        }
    };
    T* dst = y + row * ld_y + (int64_t)col0 * VEC;
    for (int t = 0; t < steps; ++t) {
        fetch();
        copy_wait<kStages - 1>();
        const uint4* from = ring + take_at * (ROWS * NV * 32);
        const int64_t left = rows - row;  // rows past the end compute on old copies and are not stored
        float2 f[ROWS][NV][H];
        float v[ROWS], mu[ROWS];
#pragma unroll
        for (int r = 0; r < ROWS; ++r) {
            float2 s = splat(0.0f);
#pragma unroll
            for (int k = 0; k < NV; ++k) {
                unpack16<T>(from[(r * NV + k) * 32], f[r][k]);
#pragma unroll
                for (int i = 0; i < H; ++i) s = __fadd2_rn(s, f[r][k][i]);
            }
            v[r] = s.x + s.y;
        }
        sums(v, 0);
#pragma unroll
        for (int r = 0; r < ROWS; ++r) {
            mu[r] = v[r] * inv_d;
            float2 s = splat(0.0f);
#pragma unroll
            for (int k = 0; k < NV; ++k) {
                const float2 shift = splat(on[k] ? -mu[r] : 0.0f);
#pragma unroll
                for (int i = 0; i < H; ++i) {
                    f[r][k][i] = __fadd2_rn(f[r][k][i], shift);
                    s = __ffma2_rn(f[r][k][i], f[r][k][i], s);
                }
            }
            v[r] = s.x + s.y;
        }
        sums(v, 1);
#pragma unroll
        for (int r = 0; r < ROWS; ++r) v[r] = rsqrtf(fmaf(v[r], inv_d, eps));
#pragma unroll
        for (int k = 0; k < NV; ++k) {
            const int c = on[k] ? col0 + k * col_step : 0;
#pragma unroll
            for (int h = 0; h < VEC / 4; ++h) {
                const float4 wv = pw[h * cols + c], bv = pb[h * cols + c];
#pragma unroll
                for (int r = 0; r < ROWS; ++r) {
                    float2* g = f[r][k] + 2 * h;
                    g[0] = __ffma2_rn(__fmul2_rn(g[0], splat(v[r])), make_float2(wv.x, wv.y), make_float2(bv.x, bv.y));
                    g[1] = __ffma2_rn(__fmul2_rn(g[1], splat(v[r])), make_float2(wv.z, wv.w), make_float2(bv.z, bv.w));
                }
            }
        }
        T* q = dst;
#pragma unroll
        for (int r = 0; r < ROWS; ++r) {
            if (r < left) {
#pragma unroll
                for (int k = 0; k < NV; ++k)
                    if (on[k]) __stcs(reinterpret_cast<uint4*>(q + k * col_step * VEC), pack16<T>(f[r][k]));
                if (in_row == 0 && sub == 0) {
                    if (mean) mean[row + r] = mu[r];
                    if (rstd) rstd[row + r] = v[r];
                }
            }
            q += ld_y;
        }
        row += stride;
        dst += stride * ld_y;
        take_at = take_at + 1 == kStages ? 0 : take_at + 1;
    }
}

// Rows that start anywhere: as norm_rows_kernel, but the warps of a row copy the 16-byte pieces that hold it and
// read their columns E at a time (2 where rows of a 16-bit type start at 4-byte places). NV such reads a lane.
template <class T, class P, int E, int NV, int S>
__global__ void __launch_bounds__(32 * kRowWarps) norm_ragged_kernel(const T* x, int64_t rows, int D, int64_t ld_x,
                                                                     const P* __restrict__ w, const P* __restrict__ b,
                                                                     float eps, T* y, int64_t ld_y, float* mean, float* rstd,
                                                                     int warps, int slot_bytes) {
    constexpr int N = E * NV, H = N / 2;  // columns and pairs of columns of a lane
    extern __shared__ __align__(16) uint4 smem[];
    __shared__ float slots[2][kRowWarps];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, in_row = warp % warps, group = warp / warps;
    const int groups = kRowWarps / warps;
    const float inv_d = 1.0f / (float)D;
    char* ring = reinterpret_cast<char*>(smem) + group * S * slot_bytes;
    float* pw = reinterpret_cast<float*>(reinterpret_cast<char*>(smem) + groups * S * slot_bytes);
    float* pb = pw + D;
    for (int i = threadIdx.x; i < D; i += blockDim.x) {
        pw[i] = w ? to_float(w[i]) : 1.0f;
        pb[i] = b ? to_float(b[i]) : 0.0f;
    }
    const int col0 = in_row * 32 * N + lane * E;  // a lane's column j: col0 + j / E * 32 * E + j % E
    const bool full = (in_row + 1) * 32 * N <= D;
    auto on = [&](int j) { return col0 + j / E * 32 * E + j % E < D; };
    const int64_t stride = (int64_t)gridDim.x * groups;
    const int steps = (int)((rows + stride - 1) / stride);  // the same for every group
    int64_t row = (int64_t)blockIdx.x * groups + group, ahead = row;
    const int64_t span = ((rows - 1) * ld_x + D) * (int64_t)sizeof(T);
    int fetch_at = 0, take_at = 0;
    auto fetch = [&]() {
        if (ahead < rows) copy_pieces(ring + fetch_at * slot_bytes, x + ahead * ld_x, D, x, span, in_row * 32 + lane, warps * 32);
        copy_commit();
        ahead += stride;
        fetch_at = fetch_at + 1 == S ? 0 : fetch_at + 1;
    };
    auto barrier = [&]() {
        if (warps > 1) asm volatile("bar.sync %0, %1;" ::"r"(1 + group), "r"(warps * 32) : "memory");
        else __syncwarp();
    };
    auto sum = [&](float v, int which) {
        v = warp_sum(v);
        if (warps == 1) return v;
        if (lane == 0) slots[which][warp] = v;
        barrier();
        float r = 0.0f;
        for (int q = 0; q < warps; ++q) r += slots[which][group * warps + q];
        return r;
    };
#pragma unroll
    for (int t = 0; t < S - 1; ++t) fetch();
    __syncthreads();  // weight and bias
    for (int t = 0; t < steps; ++t) {
        copy_wait<S - 2>();
        barrier();  // the row is there for all its warps, and the stage before is free
        fetch();
        auto compute = [&](auto mask) {
            constexpr bool MASK = decltype(mask)::value;
            const T* q = reinterpret_cast<const T*>(ring + take_at * slot_bytes + (reinterpret_cast<uintptr_t>(x + row * ld_x) & 15)) + col0;
            float2 f[H];
            float2 s = splat(0.0f);
#pragma unroll
            for (int i = 0; i < H; ++i) {
                if constexpr (E == 2) {
                    f[i] = !MASK || on(2 * i) ? unpack2<T>(*reinterpret_cast<const uint32_t*>(q + 64 * i)) : splat(0.0f);
                } else {
                    f[i].x = !MASK || on(2 * i) ? to_float(q[64 * i]) : 0.0f;
                    f[i].y = !MASK || on(2 * i + 1) ? to_float(q[64 * i + 32]) : 0.0f;
                }
                s = __fadd2_rn(s, f[i]);
            }
            const float mu = sum(s.x + s.y, 0) * inv_d;
            s = splat(0.0f);
#pragma unroll
            for (int i = 0; i < H; ++i) {
                f[i] = __fadd2_rn(f[i], MASK ? make_float2(on(2 * i) ? -mu : 0.0f, on(2 * i + 1) ? -mu : 0.0f) : splat(-mu));
                s = __ffma2_rn(f[i], f[i], s);
            }
            const float r = rsqrtf(fmaf(sum(s.x + s.y, 1), inv_d, eps));
            T* o = y + row * ld_y + col0;
            if (row < rows) {
#pragma unroll
                for (int i = 0; i < H; ++i) {
                    const int a = 64 * i, c = E == 2 ? a + 1 : a + 32;
                    const bool oa = !MASK || on(2 * i), ob = !MASK || on(2 * i + 1);
                    const float2 wv = make_float2(oa ? pw[col0 + a] : 0.0f, ob ? pw[col0 + c] : 0.0f);
                    const float2 bv = make_float2(oa ? pb[col0 + a] : 0.0f, ob ? pb[col0 + c] : 0.0f);
                    f[i] = __ffma2_rn(__fmul2_rn(f[i], splat(r)), wv, bv);
                    if constexpr (E == 2) {
                        if (oa) *reinterpret_cast<uint32_t*>(o + a) = pack2<T>(f[i].x, f[i].y);
                    } else {
                        if (oa) o[a] = from_float<T>(f[i].x);
                        if (ob) o[c] = from_float<T>(f[i].y);
                    }
                }
                if (in_row == 0 && lane == 0) {
                    if (mean) mean[row] = mu;
                    if (rstd) rstd[row] = r;
                }
            }
        };
        if (full) compute(std::false_type{});
        else compute(std::true_type{});
        row += stride;
        take_at = take_at + 1 == S ? 0 : take_at + 1;
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
    const int vec = wide_elements({{x, ld_x, (int)sizeof(T)}, {y, ld_y, (int)sizeof(T)}, {w, 0, (int)sizeof(P)}, {b, 0, (int)sizeof(P)}},
                            D, kVec);
    const int per_warp = kLaneCols * 32;
    const int warps = pow2_at_least((D + per_warp - 1) / per_warp);
    // resident warps from eight rows a warp on: 960 bf16 columns, 4,096 rows 8.6 us (one row a warp 7.4), 16,384 rows
    // 16.3 (15.2), 32,768 rows 24.5 (34.4)
    if (vec == kVec && rows * warps >= (int64_t)num_sms() * kRowWarps * 8) {
        // 32 columns a lane (16 of a float32 row that takes more than one warp, for shared memory)
        const int wide = D <= per_warp || sizeof(T) == 2 ? per_warp : per_warp / 2;
        const int row_warps = pow2_at_least((D + wide - 1) / wide);
        auto stream = [&](auto k, auto l) {
            constexpr int NV = decltype(k)::value, LANES = decltype(l)::value;
            const size_t bytes = (size_t)kRowWarps * kStages * kRowsAtOnce<NV> * NV * 32 * 16 + (size_t)D * 8;
            const cudaError_t e = allow_smem<norm_rows_kernel<T, P, NV, LANES>>(bytes);
            if (e != cudaSuccess) return e;
            const int per_sm = bytes <= 112 * 1024 ? 2 : 1;  // of 227 KB, 1 KB a block the system's
            norm_rows_kernel<T, P, NV, LANES><<<num_sms() * per_sm, 32 * kRowWarps, bytes, st>>>(x, rows, D, ld_x, w, b, eps, y,
                                                                                               ld_y, mean, rstd, row_warps);
            return cudaGetLastError();
        };
        const int cols = D / kVec, n = (cols + 32 * row_warps - 1) / (32 * row_warps);
        const std::integral_constant<int, 32> all;
        if (cols <= 8) return stream(std::integral_constant<int, 1>{}, std::integral_constant<int, 8>{});
        if (cols <= 16) return stream(std::integral_constant<int, 1>{}, std::integral_constant<int, 16>{});
        if (n == 1) return stream(std::integral_constant<int, 1>{}, all);
        if (n == 2) return stream(std::integral_constant<int, 2>{}, all);
        if constexpr (kVec == 4)
            if (n > 4) return stream(std::integral_constant<int, 8>{}, all);
        return stream(std::integral_constant<int, 4>{}, all);
    }
    if (vec < kVec) {
        const int es = (int)sizeof(T), slot = (D * es / 16 + 2) * 16;
        auto stream = [&](auto e_, auto k, auto s_) {
            constexpr int E = decltype(e_)::value, NV = decltype(k)::value, S = decltype(s_)::value;
            const size_t bytes = (size_t)(kRowWarps / warps) * S * slot + (size_t)D * 8;
            const cudaError_t e = allow_smem<norm_ragged_kernel<T, P, E, NV, S>>(bytes);
            if (e != cudaSuccess) return e;
            const int64_t resident = (int64_t)num_sms() * (bytes <= 112 * 1024 ? 2 : 1), groups = kRowWarps / warps;
            const int64_t need = (rows + groups - 1) / groups;
            norm_ragged_kernel<T, P, E, NV, S><<<(unsigned)(need < resident ? need : resident), 32 * kRowWarps, bytes, st>>>(
                x, rows, D, ld_x, w, b, eps, y, ld_y, mean, rstd, warps, slot);
            return cudaGetLastError();
        };
        const int lane_cols = (D + 32 * warps - 1) / (32 * warps);
        auto pick = [&](auto e_) {
            constexpr int E = decltype(e_)::value;
            const std::integral_constant<int, 3> s3;
            if (lane_cols <= 4) return stream(e_, std::integral_constant<int, 4 / E>{}, s3);
            if (lane_cols <= 8) return stream(e_, std::integral_constant<int, 8 / E>{}, s3);
            if (lane_cols <= 16) return stream(e_, std::integral_constant<int, 16 / E>{}, s3);
            if constexpr (sizeof(T) == 4)  // the widest rows and their weights leave room for two stages
                if (D > 4096) return stream(e_, std::integral_constant<int, 32 / E>{}, std::integral_constant<int, 2>{});
            return stream(e_, std::integral_constant<int, 32 / E>{}, s3);
        };
        if constexpr (sizeof(T) == 2) {
            const int pair = wide_elements({{x, ld_x, 2}, {y, ld_y, 2}}, D, 2);
            if (pair == 2) return pick(std::integral_constant<int, 2>{});
        }
        return pick(std::integral_constant<int, 1>{});
    }
    const int64_t per_block = 8 / warps;
    const int64_t grid = (rows + per_block - 1) / per_block;
    if (grid > 0x7fffffff) return cudaErrorInvalidConfiguration;
    const int nv = (D / kVec + 32 * warps - 1) / (32 * warps);
    auto go = [&](auto k) {
        constexpr int NV = decltype(k)::value;
        norm_kernel<T, P, kVec, NV><<<(unsigned)grid, 256, 0, st>>>(x, rows, D, ld_x, w, b, eps, y, ld_y, mean, rstd, warps);
    };
    if (nv == 1) go(std::integral_constant<int, 1>{});
    else if (nv == 2) go(std::integral_constant<int, 2>{});
    else if (kVec == 4 && nv > 4) go(std::integral_constant<int, kVec == 4 ? 8 : 4>{});
    else go(std::integral_constant<int, 4>{});
    return cudaGetLastError();
}

// ---- backward

// One pass over x and dy: groups of LANES lanes (a narrow row) or of `warps` warps take turns of R rows.
// A thread owns kGradCols columns for all rows of its group. The next rows are on their way into shared
// memory while one set is computed, so that the loads in flight take no registers:
//   E = 0: rows of whole 16-byte columns; each thread copies its own columns and needs no barrier for them;
//   E = 1, 2: rows that start anywhere; the group copies the 16-byte pieces that hold them, and a thread's
//          columns are read E at a time (2 where rows of a 16-bit type start at 4-byte places).
template <class T, class P, int R, int LANES, int E, int S>
__global__ void __launch_bounds__(32 * kGradMaxWarps)
    norm_grad_rows_kernel(const T* dy, int64_t ld_dy, const T* x, int64_t ld_x, int64_t rows, int D, const P* __restrict__ w,
                          const float* __restrict__ mean, const float* __restrict__ rstd, T* dx, int64_t ld_dx,
                          float* __restrict__ part, int64_t ld_part, int warps, int slot_bytes) {
    constexpr int VEC = 16 / (int)sizeof(T), NV = kGradCols / VEC, N = kGradCols / 2;  // N pairs of columns
    constexpr int PER = 32 / LANES;
    extern __shared__ __align__(16) uint4 smem[];
    __shared__ __align__(16) float slots[2][kGradMaxWarps * PER][2 * R];
    wait_for_previous();
    const int tid = threadIdx.x, threads = blockDim.x, lane = tid & 31, warp = tid >> 5, sub = lane & (LANES - 1);
    const int in_row = warp % warps, warp_group = warp / warps;
    const int group = LANES < 32 ? tid / LANES : warp_group;
    const int groups_here = threads / 32 / warps * PER;
    const float inv_d = 1.0f / (float)D;
    // column of element j of this thread
    auto column = [&](int j) {
        if constexpr (E == 0) return ((j / VEC * warps + in_row) * LANES + sub) * VEC + j % VEC;
        if constexpr (E == 2) return ((in_row * N + j / 2) * 32 + lane) * 2 + j % 2;
        return (in_row * kGradCols + j) * 32 + lane;
    };
    const bool full = (in_row + 1) * 32 * kGradCols <= D;   // E != 0: no column of this warp is past the end
    const bool flat = ld_x == D && ld_dy == D;              // the rows of a step are one piece of memory
    float2 wf[N], dw[N], db[N];
    bool on[kGradCols];
#pragma unroll
    for (int i = 0; i < N; ++i) {
        float f[2];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int c = column(2 * i + h);
            on[2 * i + h] = c < D;
            f[h] = w && c < D ? to_float(w[c]) : 1.0f;
        }
        wf[i] = make_float2(f[0], f[1]);
        dw[i] = db[i] = splat(0.0f);
    }
    const int64_t stride = (int64_t)gridDim.x * groups_here * R;
    const int steps = (int)((rows + stride - 1) / stride);  // the same for every group
    int64_t row = ((int64_t)blockIdx.x * groups_here + group) * R, ahead = row;
    const T *px = x + row * ld_x, *pg = dy + row * ld_dy;   // of the next copy
    const int64_t span_x = ((rows - 1) * ld_x + D) * (int64_t)sizeof(T), span_g = ((rows - 1) * ld_dy + D) * (int64_t)sizeof(T);
    constexpr int kStage = R * 2 * NV;  // E = 0: [row][x, dy][k] of [thread]
    int fetch_at = 0, take_at = 0;
    auto fetch = [&]() {
        const int64_t left = rows - ahead;
        const T *qx = px, *qg = pg;
        char* slot = reinterpret_cast<char*>(smem) + (fetch_at * groups_here + group) * R * 2 * slot_bytes;
        if (E != 0 && flat && left > 0) {
            const int n = (int)(left < R ? left : R) * D;
            copy_pieces(slot, qx, n, x, span_x, in_row * 32 + lane, warps * 32);
            copy_pieces(slot + R * slot_bytes, qg, n, dy, span_g, in_row * 32 + lane, warps * 32);
        }
#pragma unroll
        for (int r = 0; r < R; ++r) {
            if constexpr (E == 0) {
                uint4* to = smem + fetch_at * kStage * threads + tid;
#pragma unroll
                for (int k = 0; k < NV; ++k) {  // 0 in columns and rows past the end: they add nothing
                    const bool there = r < left && on[k * VEC];
                    copy16_async_or_zero(to + ((r * 2) * NV + k) * threads, there ? qx + column(k * VEC) : x, there);
                    copy16_async_or_zero(to + ((r * 2 + 1) * NV + k) * threads, there ? qg + column(k * VEC) : dy, there);
                }
            } else if (r < left && !flat) {
                copy_pieces(slot + r * slot_bytes, qx, D, x, span_x, in_row * 32 + lane, warps * 32);
                copy_pieces(slot + (R + r) * slot_bytes, qg, D, dy, span_g, in_row * 32 + lane, warps * 32);
            }
            qx += ld_x;
            qg += ld_dy;
        }
        copy_commit();
        ahead += stride;
        px += stride * ld_x;
        pg += stride * ld_dy;
        fetch_at = fetch_at + 1 == S ? 0 : fetch_at + 1;
    };
    auto group_barrier = [&]() {
        if (warps > 1) asm volatile("bar.sync %0, %1;" ::"r"(1 + warp_group), "r"(warps * 32) : "memory");
        else __syncwarp();
    };
    // this thread's columns of row r of the stage in hand; `at`: where the row (flat: the step's first row)
    // lies in memory. With MASK 0 past the end.
    auto take = [&](int r, bool is_dy, const T* at, float2* f, auto mask) {
        [[maybe_unused]] constexpr bool MASK = decltype(mask)::value;
        if constexpr (E == 0) {
            const uint4* from = smem + take_at * kStage * threads + tid;
#pragma unroll
            for (int k = 0; k < NV; ++k) unpack16<T>(from[((r * 2 + is_dy) * NV + k) * threads], f + k * (VEC / 2));
        } else {
            const char* slot = reinterpret_cast<const char*>(smem) + ((take_at * groups_here + group) * 2 + is_dy) * R * slot_bytes;
            const T* q = reinterpret_cast<const T*>(slot + (reinterpret_cast<uintptr_t>(at) & 15) + (flat ? r * D * (int)sizeof(T) : r * slot_bytes)) + column(0);
#pragma unroll
            for (int i = 0; i < N; ++i) {
                if constexpr (E == 2) {
                    f[i] = !MASK || on[2 * i] ? unpack2<T>(*reinterpret_cast<const uint32_t*>(q + 64 * i)) : splat(0.0f);
                } else {
                    f[i].x = !MASK || on[2 * i] ? to_float(q[64 * i]) : 0.0f;
                    f[i].y = !MASK || on[2 * i + 1] ? to_float(q[64 * i + 32]) : 0.0f;
                }
            }
        }
    };
#pragma unroll
    for (int t = 0; t < S - 1; ++t) fetch();
    const bool wide = ((reinterpret_cast<uintptr_t>(mean) | reinterpret_cast<uintptr_t>(rstd)) & (4 * R - 1)) == 0;
    float rs_next[R], mu_next[R];  // the statistics of the step after
    auto stats = [&](int64_t at) {
        if (wide && at + R <= rows) {
            Pack<float, R>::load(rstd + at).get(rs_next);
            Pack<float, R>::load(mean + at).get(mu_next);
        } else {
#pragma unroll
            for (int r = 0; r < R; ++r) {
                rs_next[r] = at + r < rows ? rstd[at + r] : 0.0f;
                mu_next[r] = at + r < rows ? mean[at + r] : 0.0f;
            }
        }
    };
    stats(row);
    T* out = dx + row * ld_dx;
    const T *xr = x + row * ld_x, *gr = dy + row * ld_dy;
    for (int t = 0; t < steps; ++t) {
        copy_wait<S - 2>();
        if constexpr (E != 0) group_barrier();  // the rows are there for all, and the stage before is free
        fetch();
        const int left = (int)min(rows - row, (int64_t)R);  // may be negative
        float rs[R], mu[R];
#pragma unroll
        for (int r = 0; r < R; ++r) {
            rs[r] = rs_next[r];
            mu[r] = -mu_next[r];
        }
        stats(row + stride);
        float v[2 * R];  // sums of g, then of g (x - mean), over this thread's columns
        auto first = [&](auto mask) {
#pragma unroll
            for (int r = 0; r < R; ++r) {
                float2 s1 = splat(0.0f), s2 = splat(0.0f);
                if (E == 0 || r < left) {
                    float2 xf[N], gf[N];
                    take(r, false, flat ? xr : xr + r * ld_x, xf, mask);
                    take(r, true, flat ? gr : gr + r * ld_dy, gf, mask);
#pragma unroll
                    for (int i = 0; i < N; ++i) {
                        const float2 d = __fadd2_rn(xf[i], splat(mu[r]));
                        const float2 g = __fmul2_rn(gf[i], wf[i]);
                        dw[i] = __ffma2_rn(__fmul2_rn(gf[i], splat(rs[r])), d, dw[i]);
                        db[i] = __fadd2_rn(db[i], gf[i]);
                        s1 = __fadd2_rn(s1, g);
                        s2 = __ffma2_rn(g, d, s2);
                    }
                }
                v[r] = s1.x + s1.y;
                v[R + r] = s2.x + s2.y;
            }
        };
        if (E == 0 || full) first(std::false_type{});
        else first(std::true_type{});
        // 2 R sums over the lanes together: each step halves the sums that a lane holds, or adds a pair of lanes
        int mine = 0;
#pragma unroll
        for (int o = LANES / 2, m = 2 * R; o > 0; o >>= 1) {
            if (m > 1) {
                m /= 2;
                const bool up = lane & o;
#pragma unroll
                for (int i = 0; i < m; ++i) {
                    const float keep = up ? v[i + m] : v[i], give = up ? v[i] : v[i + m];
                    v[i] = keep + __shfl_xor_sync(0xffffffffu, give, o);
                }
                mine = mine * 2 + (up ? 1 : 0);
            } else {
                v[0] += __shfl_xor_sync(0xffffffffu, v[0], o);
            }
        }
        // two sets of slots in turn: one barrier a step
        if ((lane & (LANES / (2 * R) - 1)) == 0) slots[t & 1][LANES < 32 ? group : warp][mine] = v[0];
        group_barrier();
#pragma unroll
        for (int i = 0; i < 2 * R; ++i) v[i] = 0.0f;
        for (int q = 0; q < warps; ++q) {
            const float4* sq = reinterpret_cast<const float4*>(slots[t & 1][LANES < 32 ? group : warp_group * warps + q]);
#pragma unroll
            for (int i = 0; i < R / 2; ++i) {
                const float4 f = sq[i];
                v[4 * i] += f.x;
                v[4 * i + 1] += f.y;
                v[4 * i + 2] += f.z;
                v[4 * i + 3] += f.w;
            }
        }
        T* q = out;
#pragma unroll
        for (int r = 0; r < R; ++r) {
            const float c1 = -v[r] * inv_d * rs[r], c2 = -v[R + r] * inv_d * rs[r] * rs[r] * rs[r];
            if (E == 0 || r < left) {
                float2 xf[N], gf[N];
                take(r, false, flat ? xr : xr + r * ld_x, xf, std::false_type{});  // columns past the end are not stored
                take(r, true, flat ? gr : gr + r * ld_dy, gf, std::false_type{});
#pragma unroll
                for (int i = 0; i < N; ++i) {
                    const float2 d = __fadd2_rn(xf[i], splat(mu[r]));
                    const float2 g = __fmul2_rn(gf[i], wf[i]);
                    gf[i] = __ffma2_rn(d, splat(c2), __ffma2_rn(g, splat(rs[r]), splat(c1)));
                }
                if constexpr (E == 0) {
#pragma unroll
                    for (int k = 0; k < NV; ++k)
                        if (r < left && on[k * VEC]) __stcs(reinterpret_cast<uint4*>(q + column(k * VEC)), pack16<T>(gf + k * (VEC / 2)));
                } else {
#pragma unroll
                    for (int i = 0; i < N; ++i) {
                        if constexpr (E == 2) {
                            if (on[2 * i]) *reinterpret_cast<uint32_t*>(q + column(2 * i)) = pack2<T>(gf[i].x, gf[i].y);
                        } else {
                            if (on[2 * i]) q[column(2 * i)] = from_float<T>(gf[i].x);
                            if (on[2 * i + 1]) q[column(2 * i + 1)] = from_float<T>(gf[i].y);
                        }
                    }
                }
            }
            q += ld_dx;
        }
        row += stride;
        out += stride * ld_dx;
        xr += stride * ld_x;
        gr += stride * ld_dy;
        take_at = take_at + 1 == S ? 0 : take_at + 1;
    }
    // one partial row a block: the lanes with the same columns, then the block's groups in order
#pragma unroll
    for (int o = LANES; o < 32; o <<= 1) {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            dw[i].x += __shfl_xor_sync(0xffffffffu, dw[i].x, o);
            dw[i].y += __shfl_xor_sync(0xffffffffu, dw[i].y, o);
            db[i].x += __shfl_xor_sync(0xffffffffu, db[i].x, o);
            db[i].y += __shfl_xor_sync(0xffffffffu, db[i].y, o);
        }
    }
    const int sets = threads / 32 / warps;
    float* to = part + (int64_t)blockIdx.x * 2 * ld_part;
    if (sets > 1) {
        copy_wait<0>();
        __syncthreads();  // the copies' memory is free
        to = reinterpret_cast<float*>(smem) + warp_group * 2 * D;
    }
    const int64_t second = sets > 1 ? D : ld_part;
    if (lane < LANES) {
#pragma unroll
        for (int j = 0; j < kGradCols; ++j) {
            if (!on[j]) continue;
            to[column(j)] = j % 2 ? dw[j / 2].y : dw[j / 2].x;
            to[second + column(j)] = j % 2 ? db[j / 2].y : db[j / 2].x;
        }
    }
    if (sets == 1) return;
    __syncthreads();
    for (int i = tid; i < 2 * D; i += threads) {
        float a = 0.0f;
        for (int g = 0; g < sets; ++g) a += reinterpret_cast<const float*>(smem)[g * 2 * D + i];
        part[((int64_t)blockIdx.x * 2 + (i >= D)) * ld_part + (i >= D ? i - D : i)] = a;
    }
}

// dw (the first half of the blocks) and db of 32 columns a block: 32 sets of partial rows each, added in order.
template <class P>
__global__ void __launch_bounds__(1024) norm_grad_sum_kernel(const float* __restrict__ part, int64_t parts, int64_t ld_part,
                                                             int D, P* dw, P* db) {
    __shared__ float s[32][33];
    wait_for_previous();
    const bool second = blockIdx.x >= gridDim.x / 2;
    P* out = second ? db : dw;
    if (!out) return;
    const int tx = threadIdx.x & 31, ty = threadIdx.x >> 5;
    const int c0 = (second ? blockIdx.x - gridDim.x / 2 : blockIdx.x) * 32, c = c0 + tx;
    float acc = 0.0f;
    if (c < D) {
        const float* p = part + (second ? ld_part : 0) + c;
#pragma unroll 8
        for (int64_t q = ty; q < parts; q += 32) acc += p[q * 2 * ld_part];
    }
    s[ty][tx] = acc;
    __syncthreads();
    acc = warp_sum(s[tx][ty]);  // column ty of the block
    const int cc = c0 + ty;
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
    int64_t parts;     // partial rows, one a block, at most
    int64_t ld_part;
};

GradShape grad_shape(int64_t rows, int D) {
    GradShape g;
    g.ld_part = (D + 3) / 4 * 4;
    const int per_warp = 32 * kGradCols;
    if (D > per_warp * kGradMaxWarps) {
        g.warps = g.threads = 0;
        g.parts = rows < kLongParts ? rows : kLongParts;
        return g;
    }
    g.warps = pow2_at_least((D + per_warp - 1) / per_warp);
    g.threads = g.warps <= 8 ? 256 : g.warps * 32;
    // 512 threads an SM at this kernel's registers; a row of its own for each block at least
    const int64_t most = (int64_t)num_sms() * (512 / g.threads);
    g.parts = rows < most ? rows : most;
    return g;
}

template <class T, class P>
cudaError_t grad_typed(const T* dy, int64_t ld_dy, const T* x, int64_t ld_x, int64_t rows, int D, const P* w, const float* mean,
                       const float* rstd, T* dx, int64_t ld_dx, P* dw, P* db, float* part, int* launches, cudaStream_t st) {
    GradShape g = grad_shape(rows, D);
    if (rows > 0 && g.warps == 0) {
        norm_grad_columns_kernel<T><<<dim3((D + 255) / 256, (unsigned)g.parts), 256, 0, st>>>(dy, ld_dy, x, ld_x, rows, D, mean, rstd,
                                                                                             part, g.ld_part);
        const int64_t grid = rows < 65536 ? rows : 65536;
        norm_grad_long_kernel<T, P><<<(unsigned)grid, 1024, 0, st>>>(dy, ld_dy, x, ld_x, rows, D, w, mean, rstd, dx, ld_dx);
        *launches += 2;
    } else if (rows > 0) {
        const int es = (int)sizeof(T), cols = D * es / 16;
        const int vec = wide_elements({{x, ld_x, es}, {dy, ld_dy, es}, {dx, ld_dx, es}}, D, 16 / es);
        const int slot = (D * es / 16 + 2) * 16;  // of a row that starts anywhere
        auto go = [&](auto r_, auto lanes_, auto e_, auto s_) {
            constexpr int R = decltype(r_)::value, LANES = decltype(lanes_)::value, E = decltype(e_)::value, S = decltype(s_)::value;
            constexpr auto kernel = norm_grad_rows_kernel<T, P, R, LANES, E, S>;
            const int groups = g.threads / 32 / g.warps * (32 / LANES);
            const size_t bytes = E == 0 ? (size_t)S * R * 2 * kGradCols * es * g.threads : (size_t)S * groups * R * 2 * slot + (size_t)g.warps * 32 * kGradCols * es;  // room past the last row
            const cudaError_t e = allow_smem<kernel>(bytes);
            if (e != cudaSuccess) return e;
            // no more blocks than are resident: each has its share of the rows from the start
            const int64_t resident = (int64_t)num_sms() * (g.threads == 256 && bytes <= 108 * 1024 ? 2 : 1);
            const int64_t need = (rows + groups * R - 1) / (groups * R);
            g.parts = need < resident ? need : resident;
            kernel<<<(unsigned)g.parts, g.threads, bytes, st>>>(dy, ld_dy, x, ld_x, rows, D, w, mean, rstd, dx, ld_dx, part, g.ld_part,
                                                              g.warps, slot);
            return cudaGetLastError();
        };
        const std::integral_constant<int, 0> i0;
        const std::integral_constant<int, 1> i1;
        const std::integral_constant<int, 2> i2;
        const std::integral_constant<int, 3> i3;
        const std::integral_constant<int, 4> i4;
        const std::integral_constant<int, 32> all;
        // four rows at a time where two blocks an SM have room for three stages of them, else two (50,000 x 1001
        // float32: 145 us with four rows and one block, 123 us with two and two)
        auto ragged = [&](auto e_) {
            const size_t stage = (size_t)(g.threads / 32 / g.warps) * 4 * 2 * slot;
            return 3 * stage <= 104 * 1024 ? go(i4, all, e_, i3) : go(i2, all, e_, i3);
        };
        cudaError_t e;
        if (vec * es == 16) {
            if (cols * (16 / es) <= 8 * kGradCols) e = go(i4, std::integral_constant<int, 8>{}, i0, i3);
            else if (cols * (16 / es) <= 16 * kGradCols) e = go(i4, std::integral_constant<int, 16>{}, i0, i3);
            else e = g.threads * es > 1024 ? go(i2, all, i0, i3) : go(i4, all, i0, i3);
        } else if constexpr (sizeof(T) == 2) {
            e = vec >= 2 ? ragged(i2) : ragged(i1);
        } else {
            e = ragged(i1);
        }
        if (e != cudaSuccess) return e;
        *launches += 1;
    }
    if (dw || db) {
        const cudaError_t e = launch_chained(norm_grad_sum_kernel<P>, (D + 31) / 32 * 2, 1024, 0, st, part, rows > 0 ? g.parts : 0,
                                             g.ld_part, D, dw, db);
        if (e != cudaSuccess) return e;
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
