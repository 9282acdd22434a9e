// Shared pieces of the mixed-precision network operators (norm.cu, linear.cu): typed
// access, activations for 16-bit results, host-side argument checks.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include <initializer_list>
#include <new>
#include <type_traits>

#include "common.cuh"

namespace rune {
namespace ops {

constexpr float kE4m3Max = 448.0f;

// ----------------------------------------------------------------------------- host side
// Runs fn on device `device` and maps every exception to a status; the caller's current device
// is restored. Nothing throws through the C boundary.
template <typename Fn>
int guarded(int device, Fn&& fn) {
    int before = -1;
    int code = RUNE_OK;
    try {
        RUNE_CUDA_TRY(cudaGetDevice(&before));
        // also where it is current already: a new thread has no context before this call, and the
        // driver's tensor-map encoder needs one
        RUNE_CUDA_TRY(cudaSetDevice(device));
        fn();
    } catch (const Error& e) {
        set_error(e.message);
        code = e.code;
        if (code == RUNE_ERR_CUDA) cudaGetLastError();  // reported here: not again by a later call
    } catch (const std::bad_alloc&) {
        set_error("out of host memory");
        code = RUNE_ERR_OOM;
    } catch (const std::exception& e) {
        set_error(e.what());
        code = RUNE_ERR_INVALID;
    } catch (...) {
        set_error("unknown failure");
        code = RUNE_ERR_INVALID;
    }
    if (before >= 0 && before != device) cudaSetDevice(before);
    return code;
}

inline void require(bool ok, const char* message) {
    if (!ok) throw Error(RUNE_ERR_INVALID, message);
}

inline int dtype_bytes(int dtype) { return dtype == RUNE_F32 ? 4 : dtype == RUNE_E4M3 ? 1 : 2; }

inline bool aligned(const void* p, size_t bytes) { return (uintptr_t)p % bytes == 0; }

// every array starts on a multiple of `bytes`, its values' size (or more, where the header asks)
inline void require_aligned(std::initializer_list<const void*> arrays, size_t bytes) {
    for (const void* p : arrays)
        require(aligned(p, bytes), "an array does not start on a multiple of its values' size");
}

int sm_count(int device);

// Throws, once, if a wait of an operator's kernel on the device gave up. Every entry calls it.
void check_waits(int device);

// Launches an operator's kernel so that it may begin while the one before it in the stream ends
// (programmatic dependent launch): its prologue and the launch itself are hidden, and follow_on()
// in the kernel holds back everything that touches memory. cluster: blocks of one, or 0.
template <typename... Params, typename... Args>
void launch(void (*kernel)(Params...), dim3 grid, dim3 block, size_t smem, int cluster,
            cudaStream_t stream, Args&&... args) {
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = grid;
    cfg.blockDim = block;
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute at[2];
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    at[1].id = cudaLaunchAttributeClusterDimension;
    at[1].val.clusterDim = {(unsigned)cluster, 1, 1};
    cfg.attrs = at;
    cfg.numAttrs = cluster > 0 ? 2 : 1;
    RUNE_CUDA_TRY(cudaLaunchKernelEx(&cfg, kernel, std::forward<Args>(args)...));
}

// Sums the float32 partials [parts][width] over parts into out[width] of type dtype. Many parts
// are summed in two steps, through partial_scratch(parts) further rows of `width` floats.
int64_t partial_scratch(int64_t parts);
void sum_partials(const float* partials, int64_t parts, int64_t width, void* out, int dtype,
                  float* scratch, cudaStream_t stream);

// ----------------------------------------------------------------------------- launches
// Every thread calls it before its first access to global memory and, in kernels that hold TMEM,
// after the block has its TMEM: waits until the kernel before in the stream is complete and its
// writes are visible, and lets the next one begin its own prologue. A kernel whose blocks wait
// here needs nothing of the next one, and all its blocks are resident by then, so the next one's
// waiting for shared memory or TMEM ends. What the kernel before wrote is not constant for the
// life of this one: no read-only (non-coherent) loads of it, which could be moved ahead of here.
__device__ __forceinline__ void follow_on() {
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
}

// ----------------------------------------------------------------------------- typed access
__device__ __forceinline__ float to_float(float v) { return v; }
__device__ __forceinline__ float to_float(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_float(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T>
__device__ __forceinline__ T from_float(float v);
template <>
__device__ __forceinline__ float from_float<float>(float v) { return v; }
template <>
__device__ __forceinline__ __half from_float<__half>(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float v) {
    return __float2bfloat16_rn(v);
}

// two floats rounded to a packed pair (a in the low half)
template <typename T>
__device__ __forceinline__ uint32_t pack2(float a, float b);
template <>
__device__ __forceinline__ uint32_t pack2<__half>(float a, float b) {
    __half2 v = __floats2half2_rn(a, b);
    return *reinterpret_cast<uint32_t*>(&v);
}
template <>
__device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float a, float b) {
    __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<uint32_t*>(&v);
}
template <typename T>
__device__ __forceinline__ float2 unpack2(uint32_t w);
template <>
__device__ __forceinline__ float2 unpack2<__half>(uint32_t w) {
    return __half22float2(*reinterpret_cast<__half2*>(&w));
}
template <>
__device__ __forceinline__ float2 unpack2<__nv_bfloat16>(uint32_t w) {
    return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
}

// maximum that keeps a NaN
__device__ __forceinline__ float max_nan(float a, float b) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}

// ----------------------------------------------------------------------------- activations
// For results that are rounded to 16 bits (2^-8 or 2^-11 relative): few instructions without a
// branch. Values are off by 2e-6 of themselves, at |x| = 10 by 5e-6 (the exponentials' arguments
// are float32); derivatives by as much of their terms. Exponentials below 2^-126 are 0.
__device__ __forceinline__ float rcp_fast(float x) {
    float r;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}

// Two float32 values in one 64-bit register: Blackwell adds, multiplies and fuses them in one
// instruction, which halves the arithmetic of the epilogues.
struct Two {
    uint64_t v;
};
__device__ __forceinline__ Two two(float a, float b) {
    Two t;
    asm("mov.b64 %0, {%1, %2};" : "=l"(t.v) : "f"(a), "f"(b));
    return t;
}
__device__ __forceinline__ Two two(float a) { return two(a, a); }
__device__ __forceinline__ void split(Two t, float& a, float& b) {
    asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(t.v));
}
__device__ __forceinline__ Two operator+(Two a, Two b) {
    Two t;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(t.v) : "l"(a.v), "l"(b.v));
    return t;
}
__device__ __forceinline__ Two operator*(Two a, Two b) {
    Two t;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(t.v) : "l"(a.v), "l"(b.v));
    return t;
}
__device__ __forceinline__ Two fma(Two a, Two b, Two c) {
    Two t;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(t.v) : "l"(a.v), "l"(b.v), "l"(c.v));
    return t;
}
template <typename Fn>
__device__ __forceinline__ Two each(Two t, Fn&& fn) {
    float a, b;
    split(t, a, b);
    return two(fn(a), fn(b));
}
__device__ __forceinline__ Two ex2(Two t) {  // 2^t
    return each(t, [](float x) {
        float r;
        asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
        return r;
    });
}
__device__ __forceinline__ Two rcp(Two t) {
    return each(t, [](float x) { return rcp_fast(x); });
}
// a where the sign of s is clear, b where it is set
__device__ __forceinline__ Two by_sign(Two s, Two a, Two b) {
    float s0, s1, a0, a1, b0, b1;
    split(s, s0, s1);
    split(a, a0, a1);
    split(b, b0, b1);
    return two(s0 < 0.0f ? b0 : a0, s1 < 0.0f ? b1 : a1);
}

constexpr float kLog2E = 1.44269504088896f;

// tanh |x| = 1 - 2 E / (1 + E) with E = e^(-2 |x|); near zero, where that cancels, its Taylor series
// to x^7 (next term 62/2835 x^9: 3e-7 of the value at 1/4). Its derivative is 4 E / (1 + E)^2, which
// keeps its digits where 1 - tanh^2 cancels.
__device__ __forceinline__ Two tanh_two(Two x, Two& d) {
    Two e = ex2(each(x, [](float v) { return fabsf(v); }) * two(-2.0f * kLog2E));
    Two r = rcp(e + two(1.0f)), er = e * r;
    Two t = fma(er, two(-2.0f), two(1.0f));
    d = er * r * two(4.0f);
    Two q = x * x;
    Two s = fma(fma(fma(q, two(-17.0f / 315.0f), two(2.0f / 15.0f)), q, two(-1.0f / 3.0f)) * q, x,
                x);
    float x0, x1, q0, q1, t0, t1, s0, s1;
    split(x, x0, x1);
    split(q, q0, q1);
    split(t, t0, t1);
    split(s, s0, s1);
    return two(q0 < 0.0625f ? s0 : copysignf(t0, x0), q1 < 0.0625f ? s1 : copysignf(t1, x1));
}

// Upper tail Q(|x|) = 1 - Phi(|x|) of the normal distribution and e^(-x^2 / 2). Q e^(x^2 / 2) falls
// as 1 / |x|, so it is t P(t) / 2 with t = 1 / (1 + 0.264 |x|): P of degree 6 fitted to the smallest
// relative error for |x| <= 14, where the exponential leaves the normal numbers (6e-7; 2.4e-6 with
// float32's roundings to |x| = 8, 8e-6 to 13).
__device__ __forceinline__ Two normal_tail(Two x, Two& e) {
    Two a = each(x, [](float v) { return fabsf(v); });
    e = ex2(x * x * two(-0.5f * kLog2E));
    Two t = rcp(fma(a, two(0.264f), two(1.0f)));
    Two p = fma(t, two(-0.138046006f), two(0.405043842f));
    p = fma(t, p, two(-0.150011193f));
    p = fma(t, p, two(0.295525210f));
    p = fma(t, p, two(0.161625310f));
    p = fma(t, p, two(0.215504562f));
    p = fma(t, p, two(0.210358062f));
    return p * t * e * two(0.5f);
}

template <int ACT>
__device__ __forceinline__ Two act_value(Two x) {
    if constexpr (ACT == RUNE_ACT_TANH) {
        Two d;
        return tanh_two(x, d);
    } else if constexpr (ACT == RUNE_ACT_SILU) {
        return x * rcp(ex2(x * two(-kLog2E)) + two(1.0f));
    } else if constexpr (ACT == RUNE_ACT_GELU) {
        Two e, q = normal_tail(x, e);
        return x * by_sign(x, fma(q, two(-1.0f), two(1.0f)), q);
    } else {
        return x;
    }
}

// value y and derivative dy of the activation
template <int ACT>
__device__ __forceinline__ void act_both(Two x, Two& y, Two& dy) {
    if constexpr (ACT == RUNE_ACT_TANH) {
        y = tanh_two(x, dy);
    } else if constexpr (ACT == RUNE_ACT_SILU) {
        Two s = rcp(ex2(x * two(-kLog2E)) + two(1.0f));
        y = x * s;
        // s (1 + x (1 - s)), as a product: where s is 0 and x is infinite both forms are NaN
        dy = s * fma(x, fma(s, two(-1.0f), two(1.0f)), two(1.0f));
    } else if constexpr (ACT == RUNE_ACT_GELU) {
        Two e, q = normal_tail(x, e);
        Two cdf = by_sign(x, fma(q, two(-1.0f), two(1.0f)), q);
        y = x * cdf;
        dy = fma(x * e, two(0.39894228040143268f), cdf);
    } else {
        y = x;
        dy = two(1.0f);
    }
}

template <int ACT>
__device__ __forceinline__ float act_value(float x) {
    float a, b;
    split(act_value<ACT>(two(x)), a, b);
    return a;
}

// fn(std::integral_constant<int, ACT>) for the activation code `act`
template <typename Fn>
__host__ __device__ __forceinline__ void with_activation(int act, Fn&& fn) {
    switch (act) {
        case RUNE_ACT_TANH: fn(std::integral_constant<int, RUNE_ACT_TANH>()); break;
        case RUNE_ACT_SILU: fn(std::integral_constant<int, RUNE_ACT_SILU>()); break;
        case RUNE_ACT_GELU: fn(std::integral_constant<int, RUNE_ACT_GELU>()); break;
        default: fn(std::integral_constant<int, RUNE_ACT_NONE>()); break;
    }
}

}  // namespace ops
}  // namespace rune
