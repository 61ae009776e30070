// One AdamW step over many tensors.
//
// The step reads and writes each value's parameter, gradient and states once and computes a few dozen
// operations on them. A warp takes one block of 256 values at a time (8 a lane), which is also the block that
// shares the scales of 8-bit states: its maxima are warp reductions. The tensors' descriptors travel as
// kernel arguments, so a step is one launch without copies for up to kMaxTensors tensors, and a captured
// graph replays it.
//
// 32-bit states are bound by their bytes: 40M bf16 values with master copies (28 bytes a value) take 169 us on
// a B200, 6.6 TB/s. Thread blocks come in order and none stays: a resident grid that strides over the tensors
// took 206 us. 8-bit states (10 bytes a value) are bound by instructions, some 380 for a lane's 8 values: 100M
// bf16 values take 223 us, 4.5 TB/s. Packed float pairs brought 382 us to 213, the scales' lines of their own
// that to 188; the moments' separate roundings and the exact square root, without which the 8-bit values of two
// machines part in a few places of a million, cost 35 us of it.
#include <cuda_fp8.h>
#include <math.h>

#include "tb_encoder.h"
#include "tb_vec.cuh"

namespace tb {

namespace {

constexpr int kBlock = TRIDENT_ADAMW_BLOCK;
constexpr int kLane = kBlock / 32;  // values of a lane
// Consecutive blocks that a thread block takes. The scales of 8-bit states are 4 bytes a block: 32 blocks fill
// a line of memory, which one thread block then reads and writes alone.
template <bool BITS8> constexpr int kUnit = BITS8 ? 32 : 8;
constexpr int kMaxTensors = 440;    // descriptors in 32,764 bytes of kernel arguments
constexpr float kE4m3Max = 448.0f, kE4m3Min = 1.0f / 512.0f;
constexpr float kTiny = 1e-30f;     // a block maximum below this counts as 0 (its reciprocal would overflow)

struct Scalars {
    float decay;        // 1 - lr weight_decay
    float step_size;    // -lr / (1 - beta1^t)
    float inv_root;     // 1 / sqrt(1 - beta2^t)
    float beta1, beta2, keep1, keep2;  // keep = 1 - beta
    float eps;
    uint32_t seed;
    uint32_t block0;    // blocks in the launches before this one
    const float* grad_scale;
};

template <int CAP>
struct Tensors {
    trident_adamw_tensor t[CAP];
    uint32_t first_unit[CAP + 1];  // units of blocks before each tensor
    uint32_t first_block[CAP];     // blocks before each tensor
    int32_t count;
    Scalars s;
};

// Two e4m3 bytes (the low half of `pair`) as floats, and two floats as e4m3 bytes, to nearest.
__device__ __forceinline__ float2 e4m3_values(uint32_t pair) {
    const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)pair, __NV_E4M3);
    return __half22float2(__half2(h));
}
__device__ __forceinline__ uint32_t e4m3_pair(float2 f) {
    return (uint32_t)__nv_cvt_float2_to_fp8x2(f, __NV_SATFINITE, __NV_E4M3);
}

// 32 random bits for a pair of values: two rounds of xor-shift and multiplication by odd constants (the
// fractional bits of the golden ratio and of sqrt(2)).
__device__ __forceinline__ uint32_t random_bits(uint32_t pair, uint32_t seed) {
    uint32_t h = pair * 0x9E3779B9u + seed;
    h = (h ^ (h >> 16)) * 0x6A09E667u;
    return (h ^ (h >> 15)) * 0x9E3779B9u;
}

// The largest |value| of a warp's pairs; NaN if one is (as float bits a NaN is above infinity).
__device__ __forceinline__ float absmax3(float a, float b, float c) {
    float r;
    asm("max.NaN.abs.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}
__device__ __forceinline__ float warp_absmax(const float2* v) {
    float m = absmax3(v[0].x, v[0].y, 0.0f);
#pragma unroll
    for (int i = 1; i < 4; ++i) m = absmax3(v[i].x, v[i].y, m);
    return __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(m)));
}
// The smallest of a warp's pairs of values >= 0.
__device__ __forceinline__ float warp_min(const float2* v) {
    uint32_t m = __float_as_uint(v[0].x);
#pragma unroll
    for (int i = 0; i < 4; ++i) m = min(min(__float_as_uint(v[i].x), __float_as_uint(v[i].y)), m);
    return __uint_as_float(__reduce_min_sync(0xffffffffu, m));
}

// The lane's 8 values as pairs: 16-byte accesses (WHOLE), else the n that there are.
template <class T, bool WHOLE>
__device__ __forceinline__ void load_lane(const T* p, int n, float2* f) {
    if constexpr (WHOLE) {
        constexpr int K = kPairs16<T>;
#pragma unroll
        for (int i = 0; i < kLane / 2; i += K) unpack16<T>(__ldcs(reinterpret_cast<const uint4*>(p + 2 * i)), f + i);
    } else {
#pragma unroll
        for (int i = 0; i < kLane / 2; ++i) {
            f[i].x = 2 * i < n ? to_float(p[2 * i]) : 0.0f;
            f[i].y = 2 * i + 1 < n ? to_float(p[2 * i + 1]) : 0.0f;
        }
    }
}
template <class T, bool WHOLE>
__device__ __forceinline__ void store_lane(T* p, int n, const float2* f) {
    if constexpr (WHOLE) {
        constexpr int K = kPairs16<T>;
#pragma unroll
        for (int i = 0; i < kLane / 2; i += K) __stcs(reinterpret_cast<uint4*>(p + 2 * i), pack16<T>(f + i));
    } else {
#pragma unroll
        for (int i = 0; i < kLane / 2; ++i) {
            if (2 * i < n) p[2 * i] = from_float<T>(f[i].x);
            if (2 * i + 1 < n) p[2 * i + 1] = from_float<T>(f[i].y);
        }
    }
}

// Eight e4m3 bytes of a lane.
template <bool WHOLE>
__device__ __forceinline__ uint2 load_bytes(const uint8_t* p, int n) {
    if constexpr (WHOLE) return __ldcs(reinterpret_cast<const uint2*>(p));
    uint32_t w[2] = {0, 0};
#pragma unroll
    for (int i = 0; i < kLane; ++i)
        if (i < n) w[i / 4] |= (uint32_t)p[i] << (8 * (i & 3));
    return make_uint2(w[0], w[1]);
}
template <bool WHOLE>
__device__ __forceinline__ void store_bytes(uint8_t* p, int n, uint2 w) {
    if constexpr (WHOLE) {
        __stcs(reinterpret_cast<uint2*>(p), w);
    } else {
#pragma unroll
        for (int i = 0; i < kLane; ++i)
            if (i < n) p[i] = (uint8_t)((i < 4 ? w.x : w.y) >> (8 * (i & 3)));
    }
}

// What a block of maximum `top` is multiplied by before its encoding, and its scale. A maximum below kTiny
// counts as 0, as its reciprocal would overflow.
__device__ __forceinline__ float encoding_factor(float top) { return top < kTiny ? 0.0f : __fdiv_rn(kE4m3Max, top); }
__device__ __forceinline__ float block_scale(float top) { return top < kTiny ? 0.0f : __fdiv_rn(top, kE4m3Max); }

// An 8-bit state's encoding: scaled by mul to the block's maximum. m: to nearest.
__device__ __forceinline__ uint2 encode_nearest(const float2* v, float mul) {
    uint32_t b[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) b[i] = e4m3_pair(__fmul2_rn(v[i], splat(mul)));
    return make_uint2(__byte_perm(b[0], b[1], 0x5410), __byte_perm(b[2], b[3], 0x5410));
}
// The root (>= 0): e4m3 keeps 3 of the 23 mantissa bits; 20 random bits are added below them and what is
// below is cut, so that each neighbour comes with the chance that keeps the mean. SMALL: the block has values
// that e4m3 would round to 0; only 0 itself becomes 0.
template <bool SMALL>
__device__ __forceinline__ uint2 encode_random(const float2* v, float mul, uint32_t pair, uint32_t seed) {
    uint32_t b[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const uint32_t r = random_bits(pair + i, seed);
        const float2 x = __fmul2_rn(v[i], splat(mul));
        float2 y;  // above the largest value the conversion saturates
        y.x = __uint_as_float((__float_as_uint(x.x) + ((r & 0xffffu) << 4)) & 0xfff00000u);
        y.y = __uint_as_float((__float_as_uint(x.y) + ((r >> 16) << 4)) & 0xfff00000u);
        if constexpr (SMALL) {
            y.x = x.x > 0.0f ? fmaxf(y.x, kE4m3Min) : 0.0f;
            y.y = x.y > 0.0f ? fmaxf(y.y, kE4m3Min) : 0.0f;
        }
        b[i] = e4m3_pair(y);
    }
    return make_uint2(__byte_perm(b[0], b[1], 0x5410), __byte_perm(b[2], b[3], 0x5410));
}

template <class P, class G, bool MASTER, bool BITS8, int CAP>
__global__ void __launch_bounds__(256, 4) adamw_kernel(const __grid_constant__ Tensors<CAP> a) {
    constexpr int UNIT = kUnit<BITS8>;
    __shared__ float scales[2][UNIT];  // of m and of v's root: the old scales, then the new maxima
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const uint32_t u = blockIdx.x;
    const float gs = a.s.grad_scale ? *a.s.grad_scale : 1.0f;
    int lo = 0, hi = a.count;  // the tensor of unit u: the last whose first unit is not after it
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (a.first_unit[mid] <= u) lo = mid; else hi = mid;
    }
    const trident_adamw_tensor& t = a.t[lo];
    const uint32_t block0 = (u - a.first_unit[lo]) * UNIT;
    // every array of the tensor starts at a 16-byte place (an 8-byte one for 8-bit states)
    uintptr_t bits = reinterpret_cast<uintptr_t>(t.param) | reinterpret_cast<uintptr_t>(t.grad);
    if constexpr (MASTER) bits |= reinterpret_cast<uintptr_t>(t.master);
    const uintptr_t states = reinterpret_cast<uintptr_t>(t.m) | reinterpret_cast<uintptr_t>(t.v);
    const bool wide = (bits & 15) == 0 && (states & (BITS8 ? 7 : 15)) == 0;
    // values from the unit's first on, as far as they matter
    const int left = (int)min(t.n - (int64_t)block0 * kBlock, (int64_t)UNIT * kBlock);
    const int there = (left + kBlock - 1) / kBlock;  // blocks
    if constexpr (BITS8) {
        if (threadIdx.x < 2 * UNIT && (threadIdx.x & (UNIT - 1)) < there) {
            const int i = threadIdx.x & (UNIT - 1);
            scales[threadIdx.x / UNIT][i] = (threadIdx.x < UNIT ? t.m_scale : t.v_scale)[block0 + i];
        }
        __syncthreads();
    }
    // one block; WHOLE (the same for the warp): all its values are there and their arrays allow wide accesses
    auto step = [&](int k, auto whole_) {
        constexpr bool WHOLE = decltype(whole_)::value;
        const uint32_t block = block0 + k;
        const int64_t at = (int64_t)block * kBlock + lane * kLane;
        const int n = WHOLE ? kLane : min(max(left - k * kBlock - lane * kLane, 0), kLane);  // values of this lane
        P* pp = static_cast<P*>(t.param) + at;
        float2 p[4], g[4], m[4], v[4];
        if constexpr (MASTER) load_lane<float, WHOLE>(t.master + at, n, p); else load_lane<P, WHOLE>(pp, n, p);
        load_lane<G, WHOLE>(static_cast<const G*>(t.grad) + at, n, g);
        if constexpr (BITS8) {
            const uint2 mb = load_bytes<WHOLE>(static_cast<const uint8_t*>(t.m) + at, n);
            const uint2 vb = load_bytes<WHOLE>(static_cast<const uint8_t*>(t.v) + at, n);
            const float ms = scales[0][k], vs = scales[1][k];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int sh = 16 * (i & 1);
                m[i] = __fmul2_rn(e4m3_values((i < 2 ? mb.x : mb.y) >> sh), splat(ms));
                v[i] = __fmul2_rn(e4m3_values((i < 2 ? vb.x : vb.y) >> sh), splat(vs));
                v[i] = __fmul2_rn(v[i], v[i]);
            }
        } else {
            load_lane<float, WHOLE>(static_cast<const float*>(t.m) + at, n, m);
            load_lane<float, WHOLE>(static_cast<const float*>(t.v) + at, n, v);
        }
        float2 root[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float2 gi = __fmul2_rn(g[i], splat(gs));
            // each operation rounded by itself: what is encoded in 8 bits is the formula's, to the last bit
            m[i] = add2_apart(__fmul2_rn(m[i], splat(a.s.beta1)), __fmul2_rn(gi, splat(a.s.keep1)));
            v[i] = add2_apart(__fmul2_rn(v[i], splat(a.s.beta2)), __fmul2_rn(__fmul2_rn(gi, gi), splat(a.s.keep2)));
            root[i] = BITS8 ? make_float2(__fsqrt_rn(v[i].x), __fsqrt_rn(v[i].y)) : make_float2(sqrt_approx(v[i].x), sqrt_approx(v[i].y));
            const float2 denom = __ffma2_rn(root[i], splat(a.s.inv_root), splat(a.s.eps));
            const float2 upd = __fmul2_rn(__fmul2_rn(m[i], splat(a.s.step_size)), make_float2(rcp_approx(denom.x), rcp_approx(denom.y)));
            p[i] = __ffma2_rn(p[i], splat(a.s.decay), upd);
        }
        store_lane<P, WHOLE>(pp, n, p);
        if constexpr (MASTER) store_lane<float, WHOLE>(t.master + at, n, p);
        if constexpr (BITS8) {
            if constexpr (!WHOLE) {  // values past the end take no part in the maxima
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    if (2 * i >= n) m[i].x = root[i].x = 0.0f;
                    if (2 * i + 1 >= n) m[i].y = root[i].y = 0.0f;
                }
            }
            const float mt = warp_absmax(m), vt = warp_absmax(root);
            store_bytes<WHOLE>(static_cast<uint8_t*>(t.m) + at, n, encode_nearest(m, encoding_factor(mt)));
            const float mul = encoding_factor(vt);
            const uint32_t pair = (a.s.block0 + a.first_block[lo] + block) * (kBlock / 2) + lane * (kLane / 2);
            const bool small = !(warp_min(root) * mul >= kE4m3Min);
            store_bytes<WHOLE>(static_cast<uint8_t*>(t.v) + at, n,
                               small ? encode_random<true>(root, mul, pair, a.s.seed) : encode_random<false>(root, mul, pair, a.s.seed));
            if (lane < 2) scales[lane][k] = lane ? vt : mt;
        } else {
            store_lane<float, WHOLE>(static_cast<float*>(t.m) + at, n, m);
            store_lane<float, WHOLE>(static_cast<float*>(t.v) + at, n, v);
        }
    };
#pragma unroll 1
    for (int k = warp; k < there; k += 8) {
        if (wide && left >= (k + 1) * kBlock) step(k, std::true_type{});
        else step(k, std::false_type{});
    }
    if constexpr (BITS8) {
        __syncthreads();
        if (threadIdx.x < 2 * UNIT && (threadIdx.x & (UNIT - 1)) < there) {
            const int i = threadIdx.x & (UNIT - 1);
            (threadIdx.x < UNIT ? t.m_scale : t.v_scale)[block0 + i] = block_scale(scales[threadIdx.x / UNIT][i]);
        }
    }
}

template <class P, class G, bool MASTER, bool BITS8>
cudaError_t run(const trident_adamw_tensor* tensors, int count, Scalars s, int* launches, cudaStream_t st) {
    auto go = [&](auto cap, int lo, int n, uint32_t* blocks) {
        constexpr int CAP = decltype(cap)::value;
        Tensors<CAP> a;
        a.count = n;
        a.s = s;
        uint32_t at = 0, unit = 0;
        for (int i = 0; i < n; ++i) {
            a.t[i] = tensors[lo + i];
            a.first_block[i] = at;
            a.first_unit[i] = unit;
            const uint32_t b = (uint32_t)((a.t[i].n + kBlock - 1) / kBlock);
            at += b;
            unit += (b + kUnit<BITS8> - 1) / kUnit<BITS8>;
        }
        a.first_unit[n] = unit;
        *blocks = at;
        if (unit == 0) return cudaSuccess;
        adamw_kernel<P, G, MASTER, BITS8, CAP><<<unit, 256, 0, st>>>(a);
        *launches += 1;
        return cudaGetLastError();
    };
    for (int lo = 0; lo < count; lo += kMaxTensors) {
        const int n = count - lo < kMaxTensors ? count - lo : kMaxTensors;
        uint32_t blocks = 0;
        // a small step has small arguments: 6 tensors 10.6 us, with room for kMaxTensors 14.7 us
        cudaError_t e = n <= 16   ? go(std::integral_constant<int, 16>{}, lo, n, &blocks)
                        : n <= 64 ? go(std::integral_constant<int, 64>{}, lo, n, &blocks)
                                  : go(std::integral_constant<int, kMaxTensors>{}, lo, n, &blocks);
        if (e != cudaSuccess) return e;
        s.block0 += blocks;
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
    s.step_size = (float)(-c.lr / (1.0 - pow(c.beta1, (double)c.step)));
    s.inv_root = (float)(1.0 / sqrt(1.0 - pow(c.beta2, (double)c.step)));
    s.beta1 = (float)c.beta1;
    s.beta2 = (float)c.beta2;
    s.keep1 = (float)(1.0 - c.beta1);
    s.keep2 = (float)(1.0 - c.beta2);
    s.eps = (float)c.eps;
    s.seed = c.rounding_seed;
    s.block0 = 0;
    s.grad_scale = c.grad_scale;
    const bool bits8 = c.state_bits == 8;
    return with_type(c.param_dtype, [&](auto t) {
        using P = typename decltype(t)::type;
        return c.grad_dtype == TRIDENT_F32 ? pick<P, float>(tensors, count, s, master, bits8, launches, st)
                                           : pick<P, P>(tensors, count, s, master, bits8, launches, st);
    });
}

}  // namespace tb
