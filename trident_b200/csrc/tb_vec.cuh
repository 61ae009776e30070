// Typed wide loads and stores of the encoder operators: N elements of T moved as one 2- to 16-byte
// access, computed on as float.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

namespace tb {

template <int BYTES> struct RawOf;
template <> struct RawOf<16> { using type = uint4; };
template <> struct RawOf<8> { using type = uint2; };
template <> struct RawOf<4> { using type = uint32_t; };
template <> struct RawOf<2> { using type = uint16_t; };

__device__ __forceinline__ float to_float(float x) { return x; }
__device__ __forceinline__ float to_float(__half x) { return __half2float(x); }
__device__ __forceinline__ float to_float(__nv_bfloat16 x) { return __bfloat162float(x); }
template <class T> __device__ __forceinline__ T from_float(float x);
template <> __device__ __forceinline__ float from_float<float>(float x) { return x; }
template <> __device__ __forceinline__ __half from_float<__half>(float x) { return __float2half_rn(x); }
template <> __device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }

// Two packed 16-bit elements <-> two floats.
template <class T> __device__ __forceinline__ float2 unpack2(uint32_t w);
template <> __device__ __forceinline__ float2 unpack2<__nv_bfloat16>(uint32_t w) {
    return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
}
template <> __device__ __forceinline__ float2 unpack2<__half>(uint32_t w) {
    return __half22float2(*reinterpret_cast<const __half2*>(&w));
}
template <class T> __device__ __forceinline__ uint32_t pack2(float a, float b);
template <> __device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float a, float b) {
    const __nv_bfloat162 p = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&p);
}
template <> __device__ __forceinline__ uint32_t pack2<__half>(float a, float b) {
    const __half2 p = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&p);
}

// N elements of T as raw bits. N * sizeof(T) is 2, 4, 8 or 16; addresses are aligned to it.
template <class T, int N>
struct Pack {
    using Raw = typename RawOf<(int)sizeof(T) * N>::type;
    Raw raw;

    __device__ __forceinline__ static Pack load(const T* p) {
        Pack r;
        r.raw = *reinterpret_cast<const Raw*>(p);
        return r;
    }
    // read once: evict first
    __device__ __forceinline__ static Pack load_stream(const T* p) {
        Pack r;
        r.raw = __ldcs(reinterpret_cast<const Raw*>(p));
        return r;
    }
    __device__ __forceinline__ void store(T* p) const { *reinterpret_cast<Raw*>(p) = raw; }

    __device__ __forceinline__ void get(float* f) const {
        if constexpr (N == 1) {
            f[0] = to_float(*reinterpret_cast<const T*>(&raw));
        } else if constexpr (sizeof(T) == 4) {
            const float* s = reinterpret_cast<const float*>(&raw);
#pragma unroll
            for (int i = 0; i < N; ++i) f[i] = s[i];
        } else {
            const uint32_t* w = reinterpret_cast<const uint32_t*>(&raw);
#pragma unroll
            for (int i = 0; i < N / 2; ++i) {
                const float2 t = unpack2<T>(w[i]);
                f[2 * i] = t.x;
                f[2 * i + 1] = t.y;
            }
        }
    }
    __device__ __forceinline__ static Pack of(const float* f) {
        Pack r;
        if constexpr (N == 1) {
            *reinterpret_cast<T*>(&r.raw) = from_float<T>(f[0]);
        } else if constexpr (sizeof(T) == 4) {
            float* s = reinterpret_cast<float*>(&r.raw);
#pragma unroll
            for (int i = 0; i < N; ++i) s[i] = f[i];
        } else {
            uint32_t* w = reinterpret_cast<uint32_t*>(&r.raw);
#pragma unroll
            for (int i = 0; i < N / 2; ++i) w[i] = pack2<T>(f[2 * i], f[2 * i + 1]);
        }
        return r;
    }
};

// Packed pairs of floats: one instruction for two operations.
__device__ __forceinline__ float2 splat(float x) { return make_float2(x, x); }

// The sum of two products of pairs with each product rounded. (Packed, the compiler joins a product and a sum
// into one fused operation, whatever rounding they name; single sums of packed products stay apart.)
__device__ __forceinline__ float2 add2_apart(float2 a, float2 b) { return make_float2(__fadd_rn(a.x, b.x), __fadd_rn(a.y, b.y)); }

// The 16 bytes at p as pairs of floats (4 of float32, 8 of a 16-bit type), and back.
template <class T> constexpr int kPairs16 = 8 / (int)sizeof(T);
template <class T>
__device__ __forceinline__ void unpack16(const uint4& raw, float2* f) {
    if constexpr (sizeof(T) == 4) {
        f[0] = make_float2(__uint_as_float(raw.x), __uint_as_float(raw.y));
        f[1] = make_float2(__uint_as_float(raw.z), __uint_as_float(raw.w));
    } else {
        f[0] = unpack2<T>(raw.x);
        f[1] = unpack2<T>(raw.y);
        f[2] = unpack2<T>(raw.z);
        f[3] = unpack2<T>(raw.w);
    }
}
template <class T>
__device__ __forceinline__ uint4 pack16(const float2* f) {
    if constexpr (sizeof(T) == 4)
        return make_uint4(__float_as_uint(f[0].x), __float_as_uint(f[0].y), __float_as_uint(f[1].x), __float_as_uint(f[1].y));
    else
        return make_uint4(pack2<T>(f[0].x, f[0].y), pack2<T>(f[1].x, f[1].y), pack2<T>(f[2].x, f[2].y), pack2<T>(f[3].x, f[3].y));
}

// sqrt(x) to a few units in the last place; values below 2^-126 count as 0.
__device__ __forceinline__ float sqrt_approx(float x) {
    float r;
    asm("sqrt.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}

// 1 / x to a unit in the last place for 2^-126 <= x <= 2^126; infinite below.
__device__ __forceinline__ float rcp_approx(float x) {
    float r;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}

// 16 bytes from global to shared memory without a register, in groups that are waited for by count.
__device__ __forceinline__ void copy16_async(void* smem, const void* gmem) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"((uint32_t)__cvta_generic_to_shared(smem)), "l"(gmem) : "memory");
}
// The same, or 16 bytes of zeros where !on (p is then not read, but is an address all the same).
__device__ __forceinline__ void copy16_async_or_zero(void* smem, const void* p, bool on) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"((uint32_t)__cvta_generic_to_shared(smem)), "l"(p),
                 "r"(on ? 16 : 0)
                 : "memory");
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copy_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

// N floats to or from memory of type T, in accesses of at most 16 bytes.
template <class T, int N>
__device__ __forceinline__ void load_n(const T* p, float* f) {
    constexpr int M = (int)sizeof(T) * N > 16 ? 16 / (int)sizeof(T) : N;
#pragma unroll
    for (int i = 0; i < N; i += M) Pack<T, M>::load(p + i).get(f + i);
}
template <class T, int N>
__device__ __forceinline__ void store_n(T* p, const float* f) {
    constexpr int M = (int)sizeof(T) * N > 16 ? 16 / (int)sizeof(T) : N;
#pragma unroll
    for (int i = 0; i < N; i += M) Pack<T, M>::of(f + i).store(p + i);
}

// For kernels of launch_chained: waits for the end of the kernel before (at once after any other launch), then
// lets the one after come onto the GPU.
__device__ __forceinline__ void wait_for_previous() {
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
}

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

}  // namespace tb
