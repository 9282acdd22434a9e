// dz = dy act'(z) of the linear layers from a saved float32 z, elementwise, and the sums of dz's
// columns: one layer (linear.cu), rows by group (grouped.cu).
#pragma once

#include "ops.cuh"

namespace rune {
namespace ops {

namespace {

// A block works on strips of rows x kColumns columns: a thread has four columns and every fourth
// row of the strip, and the four threads of a column join their sums in order.
constexpr int kColumns = 256;

// four values at p: by one access, or the `count` of them that are inside
template <typename T, bool WHOLE>
__device__ __forceinline__ void get4(const T* p, int count, float (&v)[4]) {
    if constexpr (WHOLE) {
        const uint2 q = *reinterpret_cast<const uint2*>(p);
        const float2 a = unpack2<T>(q.x), b = unpack2<T>(q.y);
        v[0] = a.x, v[1] = a.y, v[2] = b.x, v[3] = b.y;
    } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) v[j] = j < count ? to_float(p[j]) : 0.0f;
    }
}
template <typename T, bool WHOLE>
__device__ __forceinline__ void set4(T* p, int count, const float (&v)[4]) {
    if constexpr (WHOLE) {
        *reinterpret_cast<uint2*>(p) = make_uint2(pack2<T>(v[0], v[1]), pack2<T>(v[2], v[3]));
    } else {
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (j < count) p[j] = from_float<T>(v[j]);
    }
}
// joins the four threads' sums of a column and writes them
__device__ __forceinline__ void join4(const float (&s)[4], float* sums, int count) {
    __shared__ float joined[4][kColumns];
    const int quad = threadIdx.x & 63, part = threadIdx.x >> 6;
    __syncthreads();
#pragma unroll
    for (int j = 0; j < 4; ++j) joined[part][quad * 4 + j] = s[j];
    __syncthreads();
    if (part == 0) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int c = quad * 4 + j;
            if (j < count) sums[j] = joined[0][c] + joined[1][c] + joined[2][c] + joined[3][c];
        }
    }
}

// dz of rows r0 .. r1 - 1 in the block's columns (blockIdx.x), and their sums
template <bool GATED, typename T>
__device__ __forceinline__ void act_grad_rows(int64_t r0, int64_t r1, int64_t n, const float* z,
                                              int64_t ld_part, const T* dy, int64_t ld_dy,
                                              bool wide_dy, T* dz, int64_t ld_dz, int act,
                                              float* sums) {
    const int64_t col = (int64_t)blockIdx.x * kColumns + (threadIdx.x & 63) * 4;
    const int count = (int)max((int64_t)0, min((int64_t)4, n - col)), part = threadIdx.x >> 6;
    const int64_t ld_z = GATED ? 2 * ld_part : ld_part;
    const bool whole = wide_dy && count == 4 && (!GATED || n % 4 == 0);
    float s0[4] = {}, s1[4] = {};
    auto rows = [&](auto a, auto whole_c) {
        constexpr int ACT = decltype(a)::value;
        constexpr bool WHOLE = decltype(whole_c)::value;  // no branch among the loads
#pragma unroll 2
        for (int64_t r = r0 + part; r < r1; r += 4) {
            const float4 q = *reinterpret_cast<const float4*>(z + r * ld_z + col);
            float4 up = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            if (GATED) up = *reinterpret_cast<const float4*>(z + r * ld_z + ld_part + col);
            float d[4], g[4];
            get4<T, WHOLE>(dy + r * ld_dy + col, count, d);
            Two y0, y1, a0, a1;
            act_both<ACT>(two(q.x, q.y), y0, a0);
            act_both<ACT>(two(q.z, q.w), y1, a1);
            Two g0 = two(d[0], d[1]) * a0, g1 = two(d[2], d[3]) * a1;
            if constexpr (GATED) {
                float u[4];
                g0 = g0 * two(up.x, up.y), g1 = g1 * two(up.z, up.w);
                split(two(d[0], d[1]) * y0, u[0], u[1]);
                split(two(d[2], d[3]) * y1, u[2], u[3]);
                set4<T, WHOLE>(dz + r * ld_dz + n + col, count, u);
#pragma unroll
                for (int j = 0; j < 4; ++j) s1[j] += u[j];
            }
            split(g0, g[0], g[1]);
            split(g1, g[2], g[3]);
            set4<T, WHOLE>(dz + r * ld_dz + col, count, g);
#pragma unroll
            for (int j = 0; j < 4; ++j) s0[j] += g[j];
        }
    };
    if (count > 0)
        with_activation(act, [&](auto a) {
            if (whole) rows(a, std::true_type());
            else rows(a, std::false_type());
        });
    if (sums) {
        join4(s0, sums + col, count);
        if (GATED) join4(s1, sums + n + col, count);
    }
}

}  // namespace
}  // namespace ops
}  // namespace rune
