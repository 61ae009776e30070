// One AdamW step over many tensors.
//
// The step reads and writes each value's parameter, gradient and states once and computes a few dozen
// operations on them, so it is bound by those bytes. A warp takes one block of 256 values (8 a lane), which
// is also the block that shares the scales of 8-bit states: its maxima are warp reductions. The tensors'
// descriptors travel as kernel arguments, so a step is one launch without copies for up to kMaxTensors
// tensors, and a captured graph replays it.
#include <cuda_fp8.h>
#include <math.h>

#include "tb_encoder.h"
#include "tb_vec.cuh"

namespace tb {

namespace {

constexpr int kBlock = TRIDENT_ADAMW_BLOCK;
constexpr int kLane = kBlock / 32;  // values of a lane
constexpr int kMaxTensors = 440;    // descriptors in 32,764 bytes of kernel arguments
constexpr float kE4m3Max = 448.0f, kE4m3Min = 1.0f / 512.0f;
constexpr float kTiny = 1e-30f;     // a block maximum below this counts as 0 (its reciprocal would overflow)

struct Scalars {
    float decay;        // 1 - lr weight_decay
    float step_size;    // lr / (1 - beta1^t)
    float inv_root;     // 1 / sqrt(1 - beta2^t)
    float beta1, beta2, keep1, keep2;  // keep = 1 - beta
    float eps;
    uint32_t seed;
    uint32_t pair0;     // pairs of values in the launches before this one
    const float* grad_scale;
};

template <int CAP>
struct Tensors {
    trident_adamw_tensor t[CAP];
    uint32_t first[CAP + 1];  // blocks before each tensor
    int32_t count;
    Scalars s;
};

__device__ __forceinline__ float e4m3_value(uint32_t byte) {
    const __half_raw h = __nv_cvt_fp8_to_halfraw((__nv_fp8_storage_t)byte, __NV_E4M3);
    return __half2float(__half(h));
}

__device__ __forceinline__ uint32_t e4m3_pair(float a, float b) {
    return (uint32_t)__nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E4M3);
}

// 32 random bits for a pair of values: two rounds of xor-shift and multiplication by odd constants (the
// fractional bits of the golden ratio and of sqrt(2)).
__device__ __forceinline__ uint32_t random_bits(uint32_t pair, uint32_t seed) {
    uint32_t h = pair * 0x9E3779B9u + seed;
    h = (h ^ (h >> 16)) * 0x6A09E667u;
    return (h ^ (h >> 15)) * 0x9E3779B9u;
}

// The maximum of |x| over a warp's values as float bits: as integers a NaN is above infinity, so it stays.
__device__ __forceinline__ float warp_absmax(const float* x) {
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < kLane; ++i) m = max(m, __float_as_uint(x[i]) & 0x7fffffffu);
    return __uint_as_float(__reduce_max_sync(0xffffffffu, m));
}

template <class T>
__device__ __forceinline__ void load_lane(const T* p, int64_t n, bool whole, float* f) {
    if (whole) {
        load_n<T, kLane>(p, f);
    } else {
#pragma unroll
        for (int i = 0; i < kLane; ++i) f[i] = i < n ? to_float(p[i]) : 0.0f;
    }
}
template <class T>
__device__ __forceinline__ void store_lane(T* p, int64_t n, bool whole, const float* f) {
    if (whole) {
        store_n<T, kLane>(p, f);
    } else {
#pragma unroll
        for (int i = 0; i < kLane; ++i)
            if (i < n) p[i] = from_float<T>(f[i]);
    }
}

// Eight e4m3 bytes of a lane.
__device__ __forceinline__ void load_bytes(const uint8_t* p, int64_t n, bool whole, uint32_t* w) {
    if (whole) {
        const uint2 v = *reinterpret_cast<const uint2*>(p);
        w[0] = v.x;
        w[1] = v.y;
    } else {
        w[0] = w[1] = 0;
#pragma unroll
        for (int i = 0; i < kLane; ++i)
            if (i < n) w[i / 4] |= (uint32_t)p[i] << (8 * (i & 3));
    }
}
__device__ __forceinline__ void store_bytes(uint8_t* p, int64_t n, bool whole, const uint32_t* w) {
    if (whole) {
        *reinterpret_cast<uint2*>(p) = make_uint2(w[0], w[1]);
    } else {
#pragma unroll
        for (int i = 0; i < kLane; ++i)
            if (i < n) p[i] = (uint8_t)(w[i / 4] >> (8 * (i & 3)));
    }
}

template <class P, class G, bool MASTER, bool BITS8, int CAP>
__global__ void __launch_bounds__(256) adamw_kernel(const __grid_constant__ Tensors<CAP> a) {
    const int lane = threadIdx.x & 31;
    const uint32_t blocks = a.first[a.count];
    const float gs = a.s.grad_scale ? *a.s.grad_scale : 1.0f;
    for (uint32_t u = blockIdx.x * 8 + (threadIdx.x >> 5); u < blocks; u += gridDim.x * 8) {
        int lo = 0, hi = a.count;  // the tensor of block u: the last whose first block is not after it
        while (hi - lo > 1) {
            const int mid = (lo + hi) >> 1;
            if (a.first[mid] <= u) lo = mid; else hi = mid;
        }
        const trident_adamw_tensor& t = a.t[lo];
        const uint32_t block = u - a.first[lo];
        const int64_t at = (int64_t)block * kBlock + lane * kLane;
        const int64_t n = t.n - at;  // values from this lane's first on
        P* pp = static_cast<P*>(t.param) + at;
        const G* gp = static_cast<const G*>(t.grad) + at;
        float* mp = MASTER ? t.master + at : nullptr;
        uintptr_t bits = reinterpret_cast<uintptr_t>(pp) | reinterpret_cast<uintptr_t>(gp) | reinterpret_cast<uintptr_t>(mp);
        if constexpr (BITS8) {
            bits |= (reinterpret_cast<uintptr_t>(t.m) | reinterpret_cast<uintptr_t>(t.v)) & 7 ? 1 : 0;
        } else {
            bits |= reinterpret_cast<uintptr_t>(t.m) | reinterpret_cast<uintptr_t>(t.v);
        }
        const bool whole = n >= kLane && (bits & 15) == 0;
        float p[kLane], g[kLane], m[kLane], v[kLane];
        if constexpr (MASTER) load_lane<float>(mp, n, whole, p); else load_lane<P>(pp, n, whole, p);
        load_lane<G>(gp, n, whole, g);
        if constexpr (BITS8) {
            uint32_t mb[2], vb[2];
            load_bytes(static_cast<const uint8_t*>(t.m) + at, n, whole, mb);
            load_bytes(static_cast<const uint8_t*>(t.v) + at, n, whole, vb);
            const float ms = t.m_scale[block], vs = t.v_scale[block];
#pragma unroll
            for (int i = 0; i < kLane; ++i) {
                m[i] = e4m3_value((mb[i / 4] >> (8 * (i & 3))) & 0xff) * ms;
                const float root = e4m3_value((vb[i / 4] >> (8 * (i & 3))) & 0xff) * vs;
                v[i] = root * root;
            }
        } else {
            load_lane<float>(static_cast<const float*>(t.m) + at, n, whole, m);
            load_lane<float>(static_cast<const float*>(t.v) + at, n, whole, v);
        }
        float root[kLane];
#pragma unroll
        for (int i = 0; i < kLane; ++i) {
            const float gi = g[i] * gs;
            m[i] = fmaf(a.s.keep1, gi, a.s.beta1 * m[i]);
            v[i] = fmaf(a.s.keep2, gi * gi, a.s.beta2 * v[i]);
            root[i] = sqrtf(v[i]);
            const float denom = fmaf(root[i], a.s.inv_root, a.s.eps);
            p[i] = p[i] * a.s.decay - a.s.step_size * m[i] / denom;
        }
        store_lane<P>(pp, n, whole, p);
        if constexpr (MASTER) store_lane<float>(mp, n, whole, p);
        if constexpr (BITS8) {
#pragma unroll
            for (int i = 0; i < kLane; ++i)  // values past the end take no part in the maxima
                if (i >= n) m[i] = root[i] = 0.0f;
            const float mt = warp_absmax(m), vt = warp_absmax(root);
            const bool mlive = !(mt < kTiny), vlive = !(vt < kTiny);  // true for NaN
            const float mi = mlive ? kE4m3Max / mt : 0.0f, vi = vlive ? kE4m3Max / vt : 0.0f;
            uint32_t mb[2] = {0, 0}, vb[2] = {0, 0};
            const uint32_t pair = a.s.pair0 + u * (kBlock / 2) + lane * (kLane / 2);
#pragma unroll
            for (int i = 0; i < kLane; i += 2) {
                mb[i / 4] |= e4m3_pair(m[i] * mi, m[i + 1] * mi) << (8 * (i & 3));
                const uint32_t r = random_bits(pair + i / 2, a.s.seed);
                float q[2];
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                    // e4m3 keeps 3 of the 23 mantissa bits: 20 random bits below them, then cut
                    const float x = fminf(root[i + k] * vi, kE4m3Max);
                    const uint32_t rnd = ((k ? r >> 16 : r & 0xffffu)) << 4;
                    const float y = __uint_as_float((__float_as_uint(x) + rnd) & 0xfff00000u);
                    q[k] = x > 0.0f ? fminf(fmaxf(y, kE4m3Min), kE4m3Max) : 0.0f;
                }
                vb[i / 4] |= e4m3_pair(q[0], q[1]) << (8 * (i & 3));
            }
            store_bytes(static_cast<uint8_t*>(t.m) + at, n, whole, mb);
            store_bytes(static_cast<uint8_t*>(t.v) + at, n, whole, vb);
            if (lane == 0) {
                t.m_scale[block] = mlive ? mt / kE4m3Max : 0.0f;
                t.v_scale[block] = vlive ? vt / kE4m3Max : 0.0f;
            }
        } else {
            store_lane<float>(static_cast<float*>(t.m) + at, n, whole, m);
            store_lane<float>(static_cast<float*>(t.v) + at, n, whole, v);
        }
    }
}

template <class P, class G, bool MASTER, bool BITS8>
cudaError_t run(const trident_adamw_tensor* tensors, int count, Scalars s, int* launches, cudaStream_t st) {
    auto go = [&](auto cap, int lo, int n, uint32_t* blocks) {
        constexpr int CAP = decltype(cap)::value;
        static thread_local Tensors<CAP> a;
        a.count = n;
        a.s = s;
        uint64_t at = 0;
        for (int i = 0; i < n; ++i) {
            a.t[i] = tensors[lo + i];
            a.first[i] = (uint32_t)at;
            at += (uint64_t)(a.t[i].n + kBlock - 1) / kBlock;
        }
        a.first[n] = (uint32_t)at;
        *blocks = (uint32_t)at;
        if (at == 0) return cudaSuccess;
        const uint64_t need = (at + 7) / 8, most = (uint64_t)num_sms() * 8;
        adamw_kernel<P, G, MASTER, BITS8, CAP><<<(unsigned)(need < most ? need : most), 256, 0, st>>>(a);
        *launches += 1;
        return cudaGetLastError();
    };
    for (int lo = 0; lo < count; lo += kMaxTensors) {
        const int n = count - lo < kMaxTensors ? count - lo : kMaxTensors;
        uint32_t blocks = 0;
        cudaError_t e = n <= 16 ? go(std::integral_constant<int, 16>{}, lo, n, &blocks)
                                : go(std::integral_constant<int, kMaxTensors>{}, lo, n, &blocks);
        if (e != cudaSuccess) return e;
        s.pair0 += blocks * (kBlock / 2);
    }
    return cudaSuccess;
}

template <class P, class G>
cudaError_t pick(const trident_adamw_tensor* tensors, int count, const Scalars& s, bool master, bool bits8, int* launches,
                 cudaStream_t st) {
    if constexpr (!std::is_same<P, float>::value) {
        if (master)
            return bits8 ? run<P, G, true, true>(tensors, count, s, launches, st) : run<P, G, true, false>(tensors, count, s, launches, st);
    }
    return bits8 ? run<P, G, false, true>(tensors, count, s, launches, st) : run<P, G, false, false>(tensors, count, s, launches, st);
}

}  // namespace

cudaError_t launch_adamw(const trident_adamw_tensor* tensors, int count, const trident_adamw_config& c, bool master,
                         int* launches, cudaStream_t st) {
    Scalars s;
    s.decay = (float)(1.0 - c.lr * c.weight_decay);
    s.step_size = (float)(c.lr / (1.0 - pow(c.beta1, (double)c.step)));
    s.inv_root = (float)(1.0 / sqrt(1.0 - pow(c.beta2, (double)c.step)));
    s.beta1 = (float)c.beta1;
    s.beta2 = (float)c.beta2;
    s.keep1 = (float)(1.0 - c.beta1);
    s.keep2 = (float)(1.0 - c.beta2);
    s.eps = (float)c.eps;
    s.seed = c.rounding_seed;
    s.pair0 = 0;
    s.grad_scale = c.grad_scale;
    const bool bits8 = c.state_bits == 8;
    return with_type(c.param_dtype, [&](auto t) {
        using P = typename decltype(t)::type;
        return c.grad_dtype == TRIDENT_F32 ? pick<P, float>(tensors, count, s, master, bits8, launches, st)
                                           : pick<P, P>(tensors, count, s, master, bits8, launches, st);
    });
}

}  // namespace tb
