// Root-mean-square normalisation with the residual's addition (rune/mobius/layers.py:26-44),
//   h = x + residual,  r = 1 / sqrt(mean(h^2) + eps),  y = h r w,
// with y in the inputs' type or in 8 bits (e4m3) with a scale per row, and its backward pass
//   dx = dresidual = r (dy w - n mean(dy w n)) + dh,  n = h r,   dw = sum_rows dy n.
//
// A row stays in registers between the sum of its squares and its output, so every value is read
// once and written once: memory bandwidth bounds the kernels, launch latency the shortest calls.
// B200, of the measured copy's 6.5 TB/s: 373248 x 256 bf16 with residual 123 us, 6.2 TB/s;
// 16384 x 4096 to e4m3 80 us, 5.9; backward 143 us (6.7, five arrays) and 16384 x 4096 112 us
// (6.0); one row of 4096 2.2 us.
//
// A warp takes a row of up to 256 values (forward 512), a block of width / 8 threads (forward
// width / 16) one of up to 8192 (16384); longer rows are read twice, the second time from L2.
//
// Accesses are 16 bytes. Rows whose width or stride leaves them off 16 bytes, but all arrays by
// the same amount (contiguous arrays of an odd width), are taken from the 16-byte boundary before
// their start (kShifted): the two ends of a row are single values, the rest is whole. Only rows
// that lie differently in the arrays are read value by value.

#include <algorithm>
#include <atomic>

#include "ops.cuh"

namespace rune {
namespace ops {

namespace {

constexpr int kEpt = 8;              // values of a row per thread (forward, block: twice that)
constexpr int kLongThreads = 1024;

enum Access { kWhole, kShifted, kSingle };

// 16 bytes of a row, or one value of it
template <typename T, Access ACC>
struct alignas(ACC == kSingle ? sizeof(T) : 16) Piece {
    static constexpr int N = ACC == kSingle ? 1 : 16 / (int)sizeof(T);
    T v[N];

    // values col .. col + N - 1 of the row at p, zeros outside [0, width)
    __device__ __forceinline__ void load(const T* p, int col, int width) {
        if constexpr (ACC == kSingle) {
            v[0] = col < width ? p[col] : from_float<T>(0.0f);
        } else {
            if (ACC == kWhole ? col < width : col >= 0 && col + N <= width) {
                *reinterpret_cast<uint4*>(v) = *reinterpret_cast<const uint4*>(p + col);
            } else {
                *reinterpret_cast<uint4*>(v) = make_uint4(0, 0, 0, 0);
                if constexpr (ACC == kShifted) {
#pragma unroll
                    for (int i = 0; i < N; ++i)
                        if (col + i >= 0 && col + i < width) v[i] = p[col + i];
                }
            }
        }
    }
    __device__ __forceinline__ void store(T* p, int col, int width) const {
        if constexpr (ACC == kSingle) {
            if (col < width) p[col] = v[0];
        } else {
            if (ACC == kWhole ? col < width : col >= 0 && col + N <= width) {
                *reinterpret_cast<uint4*>(p + col) = *reinterpret_cast<const uint4*>(v);
            } else if constexpr (ACC == kShifted) {
#pragma unroll
                for (int i = 0; i < N; ++i)
                    if (col + i >= 0 && col + i < width) p[col + i] = v[i];
            }
        }
    }
    __device__ __forceinline__ void get(float* f) const {
#pragma unroll
        for (int i = 0; i < N; ++i) f[i] = to_float(v[i]);
    }
    __device__ __forceinline__ void set(const float* f) {
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] = from_float<T>(f[i]);
    }
};

// how many values the row at p starts after a 16-byte boundary
template <typename T, Access ACC>
__device__ __forceinline__ int shift_of(const T* p) {
    return ACC == kShifted ? (int)((uintptr_t)p % 16 / sizeof(T)) : 0;
}

// weights of a piece: in the rows' type or float32
template <typename T, Access ACC>
__device__ __forceinline__ void load_weight(const void* w, bool w32, int col, int width,
                                            float* v) {
    constexpr int N = Piece<T, ACC>::N;
    if (!w32 && ACC == kWhole) {
        Piece<T, ACC> q;
        q.load(static_cast<const T*>(w), col, width);
        q.get(v);
        return;
    }
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const bool in = col + i >= 0 && col + i < width;
        v[i] = !in ? 0.0f : w32 ? static_cast<const float*>(w)[col + i]
                                : to_float(static_cast<const T*>(w)[col + i]);
    }
}

// sum (or NaN-keeping maximum) over the threads of a row: the warp, or the block
template <bool BLOCK, bool MAX>
__device__ __forceinline__ float row_reduce(float v, float* shared) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        float u = __shfl_xor_sync(0xffffffffu, v, o);
        v = MAX ? max_nan(v, u) : v + u;
    }
    if constexpr (BLOCK) {
        const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, warps = blockDim.x >> 5;
        if (lane == 0) shared[warp] = v;
        __syncthreads();
        v = lane < warps ? shared[lane] : 0.0f;  // every warp repeats the same short tree
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
            float u = __shfl_xor_sync(0xffffffffu, v, o);
            v = MAX ? max_nan(v, u) : v + u;
        }
        __syncthreads();
    }
    return v;
}

// sum and, where MAX, maximum over the threads of a row in one meeting; `shared` is used once
template <bool BLOCK, bool MAX>
__device__ __forceinline__ void row_join(float& sum, float& amax, float2* shared) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        sum += __shfl_xor_sync(0xffffffffu, sum, o);
        if constexpr (MAX) amax = max_nan(amax, __shfl_xor_sync(0xffffffffu, amax, o));
    }
    if constexpr (BLOCK) {
        const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, warps = blockDim.x >> 5;
        if (lane == 0) shared[warp] = make_float2(sum, amax);
        __syncthreads();
        const float2 v = lane < warps ? shared[lane] : make_float2(0.0f, 0.0f);
        sum = v.x, amax = v.y;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {  // every warp repeats the same short tree
            sum += __shfl_xor_sync(0xffffffffu, sum, o);
            if constexpr (MAX) amax = max_nan(amax, __shfl_xor_sync(0xffffffffu, amax, o));
        }
    }
}

// values col .. of a row in e4m3: four at a time where the row allows, else one by one
template <int N, bool WHOLE>
__device__ __forceinline__ void store_e4m3(void* row, int col, int width, const float* v) {
    auto* p = static_cast<__nv_fp8_storage_t*>(row) + col;
    if constexpr (WHOLE) {
        if (col >= width) return;
#pragma unroll
        for (int i = 0; i < N; i += 4) {
            uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(v[i], v[i + 1]), __NV_SATFINITE,
                                                   __NV_E4M3);
            uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(v[i + 2], v[i + 3]),
                                                   __NV_SATFINITE, __NV_E4M3);
            *reinterpret_cast<uint32_t*>(p + i) = lo | hi << 16;
        }
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i)
            if (col + i >= 0 && col + i < width)
                p[i] = __nv_cvt_float_to_fp8(v[i], __NV_SATFINITE, __NV_E4M3);
    }
}

// Scale of a row whose largest magnitude is amax: 448 stands for amax; an all-zero row takes 1.
// Never below the smallest normal float, whose reciprocal is finite.
__device__ __forceinline__ float row_scale(float amax) {
    return amax == 0.0f ? 1.0f : max_nan(amax * (1.0f / kE4m3Max), 0x1p-126f);
}

// ----------------------------------------------------------------------------- forward
// EPT values of a row per thread. The 8-bit output's scale needs max |y| = r max |h w|, which is
// found together with the sum of squares: one meeting of the threads a row.
template <typename T, Access ACC, int EPT, int THREADS, bool BLOCK, bool Q8>
__global__ void
__launch_bounds__(THREADS, ACC == kWhole && sizeof(T) == 2 && BLOCK ? 1536 / THREADS : 1) k_norm(const rune_norm_args p) {
    using P = Piece<T, ACC>;
    constexpr int N = P::N, NC = EPT / N;
    follow_on();
    __shared__ float2 shared[32];
    const int width = (int)p.width;
    const int t = BLOCK ? threadIdx.x : threadIdx.x & 31, tpr = BLOCK ? blockDim.x : 32;
    const bool w32 = p.weight_dtype == RUNE_F32;
    const int64_t row = BLOCK ? (int64_t)blockIdx.x
                              : (int64_t)blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5);
    if (row >= p.rows) return;  // a whole warp, which meets no other
    const T* x = static_cast<const T*>(p.x) + row * p.x_stride;
    const int first = t * N - shift_of<T, ACC>(x), step = tpr * N;
    P px[NC], pr[NC];
#pragma unroll
    for (int c = 0; c < NC; ++c) px[c].load(x, first + c * step, width);
    float h[EPT];
    if (p.residual) {
        const T* res = static_cast<const T*>(p.residual) + row * p.residual_stride;
#pragma unroll
        for (int c = 0; c < NC; ++c) pr[c].load(res, first + c * step, width);
#pragma unroll
        for (int c = 0; c < NC; ++c) {
            float f[N];
            px[c].get(h + c * N);
            pr[c].get(f);
#pragma unroll
            for (int i = 0; i < N; ++i) h[c * N + i] += f[i];
            if (p.h) {
                P q;
                q.set(h + c * N);
                q.store(static_cast<T*>(p.h) + row * p.width, first + c * step, width);
            }
        }
    } else {
#pragma unroll
        for (int c = 0; c < NC; ++c) px[c].get(h + c * N);
    }
    float sum = 0.0f, amax = 0.0f;
#pragma unroll
    for (int i = 0; i < EPT; ++i) sum += h[i] * h[i];
    if (p.weight) {
#pragma unroll
        for (int c = 0; c < NC; ++c) {
            float w[N];
            load_weight<T, ACC>(p.weight, w32, first + c * step, width, w);
#pragma unroll
            for (int i = 0; i < N; ++i) h[c * N + i] *= w[i];
        }
    }
    if constexpr (Q8) {
#pragma unroll
        for (int i = 0; i < EPT; ++i) amax = max_nan(amax, fabsf(h[i]));
    }
    row_join<BLOCK, Q8>(sum, amax, shared);
    const float r = p.weight ? 1.0f / sqrtf(sum / (float)width + p.eps) : 1.0f;
    if (t == 0 && p.rstd) p.rstd[row] = r;
#pragma unroll
    for (int i = 0; i < EPT; ++i) h[i] *= r;
    if constexpr (Q8) {
        const float scale = row_scale(r * amax), inv = 1.0f / scale;
        if (t == 0) p.scale[row] = scale;
        // after r and not with it: r / scale of a row of tiny values can pass float32's range
#pragma unroll
        for (int i = 0; i < EPT; ++i) h[i] *= inv;
    }
#pragma unroll
    for (int c = 0; c < NC; ++c) {
        if constexpr (Q8) {
            store_e4m3<N, ACC == kWhole>(static_cast<char*>(p.y) + row * p.width,
                                         first + c * step, width, h + c * N);
        } else {
            P q;
            q.set(h + c * N);
            q.store(static_cast<T*>(p.y) + row * p.width, first + c * step, width);
        }
    }
}

// Rows longer than a block's registers: a block reads the row for the sum (writing h), again for the
// largest magnitude (8 bits only) and again for the output; the repeats come from L2.
template <typename T, bool Q8>
__global__ void __launch_bounds__(kLongThreads) k_norm_long(const rune_norm_args p) {
    follow_on();
    __shared__ float shared[32];
    const bool w32 = p.weight_dtype == RUNE_F32;
    const int t = threadIdx.x;
    for (int64_t row = blockIdx.x; row < p.rows; row += gridDim.x) {
        const T* x = static_cast<const T*>(p.x) + row * p.x_stride;
        const T* res = p.residual
                           ? static_cast<const T*>(p.residual) + row * p.residual_stride
                           : nullptr;
        auto at = [&](int64_t i) { return to_float(x[i]) + (res ? to_float(res[i]) : 0.0f); };
        auto weight = [&](int64_t i) {
            if (!p.weight) return 1.0f;
            return w32 ? static_cast<const float*>(p.weight)[i]
                       : to_float(static_cast<const T*>(p.weight)[i]);
        };
        float r = 1.0f;
        float sum = 0.0f;
        for (int64_t i = t; i < p.width; i += blockDim.x) {
            float h = at(i);
            sum += h * h;
            if (res && p.h) static_cast<T*>(p.h)[row * p.width + i] = from_float<T>(h);
        }
        if (p.weight) {
            sum = row_reduce<true, false>(sum, shared);
            r = 1.0f / sqrtf(sum / (float)p.width + p.eps);
            if (p.rstd && t == 0) p.rstd[row] = r;
        }
        float inv = 1.0f;
        if constexpr (Q8) {
            float amax = 0.0f;
            for (int64_t i = t; i < p.width; i += blockDim.x)
                amax = max_nan(amax, fabsf(at(i) * r * weight(i)));
            const float scale = row_scale(row_reduce<true, true>(amax, shared));
            if (t == 0) p.scale[row] = scale;
            inv = 1.0f / scale;
        }
        for (int64_t i = t; i < p.width; i += blockDim.x) {
            float y = at(i) * r * weight(i);
            if constexpr (Q8) {
                y *= inv;
                store_e4m3<1, false>(static_cast<char*>(p.y) + row * p.width + i, 0, 1, &y);
            } else {
                static_cast<T*>(p.y)[row * p.width + i] = from_float<T>(y);
            }
        }
    }
}

// ----------------------------------------------------------------------------- backward
// Each block keeps the sums of its rows for dweight in registers (a thread's columns are the same
// for every row that it takes: the grid is a multiple of eight rows, after which a shift recurs)
// and writes one row of partials. Where rows are whole, each thread copies its pieces of the next
// AHEAD rows into shared memory slots of its own (cp.async: bytes in flight without registers,
// and nobody else reads them, so no barrier); else (AHEAD = 0) it loads them as it needs them.
__device__ __forceinline__ void copy16(uint32_t dst, const void* src) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}

template <typename T, Access ACC, bool BLOCK, int AHEAD>
__global__ void __launch_bounds__(BLOCK ? 1024 : 256, BLOCK || ACC != kWhole ? 1 : 3)
k_norm_bwd(const rune_norm_grad_args p, float* partials) {
    using P = Piece<T, ACC>;
    constexpr int N = P::N, NC = kEpt / N;
    follow_on();
    __shared__ float shared[32];
    extern __shared__ __align__(16) unsigned char dynamic[];
    const int width = (int)p.width;
    const int t = BLOCK ? threadIdx.x : threadIdx.x & 31, tpr = BLOCK ? blockDim.x : 32;
    const int rpb = BLOCK ? 1 : blockDim.x >> 5, warp = threadIdx.x >> 5;
    const float inv_width = 1.0f / (float)width;
    int64_t row = (int64_t)blockIdx.x * rpb + (BLOCK ? 0 : warp);
    const int64_t stride = (int64_t)gridDim.x * rpb;
    const int first = t * N - shift_of<T, ACC>(static_cast<const T*>(p.x) + row * p.x_stride);
    const int step = tpr * N;
    float w[kEpt], dw[kEpt];
#pragma unroll
    for (int i = 0; i < kEpt; ++i) dw[i] = 0.0f;
#pragma unroll
    for (int c = 0; c < NC; ++c)
        load_weight<T, ACC>(p.weight, p.weight_dtype == RUNE_F32, first + c * step, width,
                            w + c * N);
    // slots [stage][array][piece][thread] of 16 bytes
    auto slot = [&](int stage, int array, int c) {
        return dynamic + ((((stage * 4 + array) * NC + c) * blockDim.x + threadIdx.x) << 4);
    };
    auto fetch = [&](int64_t at, int stage) {
        if (at < p.rows) {
#pragma unroll
            for (int c = 0; c < NC; ++c) {
                const int col = first + c * step;
                if (col >= width) continue;
                auto copy = [&](int array, const void* base, int64_t ld) {
                    copy16((uint32_t)__cvta_generic_to_shared(slot(stage, array, c)),
                           static_cast<const T*>(base) + at * ld + col);
                };
                copy(0, p.x, p.x_stride);
                if (p.residual) copy(1, p.residual, p.residual_stride);
                copy(2, p.dy, p.dy_stride);
                if (p.dh) copy(3, p.dh, p.dh_stride);
            }
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
    // the thread's values of array `array` in row `at`
    auto take = [&](int array, const void* base, int64_t ld, int64_t at, int stage, int c,
                    float* f) {
        const int col = first + c * step;
        P q;
        if constexpr (AHEAD > 0) {
            *reinterpret_cast<uint4*>(q.v) = col < width
                                                 ? *reinterpret_cast<uint4*>(slot(stage, array, c))
                                                 : make_uint4(0, 0, 0, 0);
        } else {
            q.load(static_cast<const T*>(base) + at * ld, col, width);
        }
        q.get(f);
    };
    if constexpr (AHEAD > 0) {
        for (int s = 0; s < AHEAD; ++s) fetch(row + s * stride, s);
    }
    float r = row < p.rows ? p.rstd[row] : 0.0f;
    int stage = 0;
    for (; row < p.rows; row += stride) {
        const float r_next = row + stride < p.rows ? p.rstd[row + stride] : 0.0f;
        if constexpr (AHEAD > 0)
            asm volatile("cp.async.wait_group %0;" ::"n"(AHEAD > 0 ? AHEAD - 1 : 0) : "memory");
        float n[kEpt], dy[kEpt], dh[kEpt], dot = 0.0f;
#pragma unroll
        for (int c = 0; c < NC; ++c) {
            take(0, p.x, p.x_stride, row, stage, c, n + c * N);
            take(2, p.dy, p.dy_stride, row, stage, c, dy + c * N);
            if (p.residual) {
                float f[N];
                take(1, p.residual, p.residual_stride, row, stage, c, f);
#pragma unroll
                for (int i = 0; i < N; ++i) n[c * N + i] += f[i];
            }
            if (p.dh) {
                take(3, p.dh, p.dh_stride, row, stage, c, dh + c * N);
            } else {
#pragma unroll
                for (int i = 0; i < N; ++i) dh[c * N + i] = 0.0f;
            }
        }
        if constexpr (AHEAD > 0) {
            fetch(row + AHEAD * stride, stage);
            if (++stage == AHEAD) stage = 0;
        }
#pragma unroll
        for (int i = 0; i < kEpt; ++i) {
            n[i] *= r;
            dw[i] += dy[i] * n[i];
            dy[i] *= w[i];
            dot += dy[i] * n[i];
        }
        dot = row_reduce<BLOCK, false>(dot, shared) * inv_width;
#pragma unroll
        for (int c = 0; c < NC; ++c) {
            float dx[N];
#pragma unroll
            for (int i = 0; i < N; ++i) {
                const int j = c * N + i;
                dx[i] = r * (dy[j] - n[j] * dot) + dh[j];
            }
            P q;
            q.set(dx);
            q.store(static_cast<T*>(p.dx) + row * p.width, first + c * step, width);
        }
        r = r_next;
    }
    if constexpr (AHEAD > 0) asm volatile("cp.async.wait_all;" ::: "memory");
    if (!partials) return;
    if constexpr (BLOCK) {
#pragma unroll
        for (int i = 0; i < kEpt; ++i) {
            const int col = first + i / N * step + i % N;
            if (col >= 0 && col < width) partials[(int64_t)blockIdx.x * width + col] = dw[i];
        }
    } else {
        float* columns = reinterpret_cast<float*>(dynamic);  // warps x width, over the slots
        __syncthreads();
#pragma unroll
        for (int i = 0; i < kEpt; ++i) {
            const int col = first + i / N * step + i % N;
            if (col >= 0 && col < width) columns[warp * width + col] = dw[i];
        }
        __syncthreads();
        for (int col = threadIdx.x; col < width; col += blockDim.x) {
            float s = 0.0f;
            for (int k = 0; k < rpb; ++k) s += columns[k * width + col];
            partials[(int64_t)blockIdx.x * width + col] = s;
        }
    }
}

// Rows longer than a block's registers: the row is read twice and the block's partials are accumulated in
// its own row of the workspace (each column always by the same thread).
template <typename T>
__global__ void __launch_bounds__(kLongThreads)
k_norm_bwd_long(const rune_norm_grad_args p, float* partials) {
    follow_on();
    __shared__ float shared[32];
    const bool w32 = p.weight_dtype == RUNE_F32;
    const int t = threadIdx.x;
    bool first = true;
    for (int64_t row = blockIdx.x; row < p.rows; row += gridDim.x, first = false) {
        const T* xp = static_cast<const T*>(p.x) + row * p.x_stride;
        const T* rp = p.residual
                          ? static_cast<const T*>(p.residual) + row * p.residual_stride
                          : nullptr;
        auto h = [&](int64_t i) { return to_float(xp[i]) + (rp ? to_float(rp[i]) : 0.0f); };
        auto weight = [&](int64_t i) {
            return w32 ? static_cast<const float*>(p.weight)[i]
                       : to_float(static_cast<const T*>(p.weight)[i]);
        };
        const T* dyp = static_cast<const T*>(p.dy) + row * p.dy_stride;
        const T* dhp = p.dh ? static_cast<const T*>(p.dh) + row * p.dh_stride : nullptr;
        const float r = p.rstd[row];
        float dot = 0.0f;
        for (int64_t i = t; i < p.width; i += blockDim.x) {
            float w = weight(i), n = h(i) * r, dy = to_float(dyp[i]);
            dot += dy * w * n;
            if (partials) {
                float* at = partials + (int64_t)blockIdx.x * p.width + i;
                *at = (first ? 0.0f : *at) + dy * n;
            }
        }
        dot = row_reduce<true, false>(dot, shared) / (float)p.width;
        for (int64_t i = t; i < p.width; i += blockDim.x) {
            float w = weight(i), n = h(i) * r;
            float dx = r * (to_float(dyp[i]) * w - n * dot) + (dhp ? to_float(dhp[i]) : 0.0f);
            static_cast<T*>(p.dx)[row * p.width + i] = from_float<T>(dx);
        }
    }
}

// Columns of float32 partials [parts][width]: a block sums 32 columns of kPartRows parts with 32
// threads each, then joins their sums in order; block row y writes row y of out.
constexpr int kPartRows = 512;

template <typename T>
__global__ void __launch_bounds__(1024)
k_sum_partials(const float* partials, int64_t parts, int64_t width, T* out) {
    follow_on();
    __shared__ float s[32][33];
    const int64_t col = (int64_t)blockIdx.x * 32 + threadIdx.x;
    const int64_t end = min(parts, ((int64_t)blockIdx.y + 1) * kPartRows);
    float v = 0.0f;
    if (col < width) {
#pragma unroll 8
        for (int64_t r = (int64_t)blockIdx.y * kPartRows + threadIdx.y; r < end; r += 32)
            v += partials[r * width + col];
    }
    s[threadIdx.y][threadIdx.x] = v;
    __syncthreads();
    if (threadIdx.y < 8) {
        for (int k = threadIdx.y + 8; k < 32; k += 8) v += s[k][threadIdx.x];
        s[threadIdx.y][threadIdx.x] = v;
    }
    __syncthreads();
    if (threadIdx.y == 0 && col < width) {
        float sum = 0.0f;
        for (int k = 0; k < 8; ++k) sum += s[k][threadIdx.x];
        out[blockIdx.y * width + col] = from_float<T>(sum);
    }
}

// ----------------------------------------------------------------------------- host
// threads for a row of `width` values, `ept` each, wherever its first 16-byte boundary lies
int threads_for(int64_t width, int ept, Access acc, int n) {
    const int64_t need = width + (acc == kShifted ? n - 1 : 0);
    return (int)((need + ept * 32 - 1) / (ept * 32)) * 32;
}

// Blocks of the backward: as many as are resident at once (a second wave would double the time:
// 373248 x 256 with four blocks too many 317 against 282 us), each leaving one row of partials. A
// multiple of eight, except where a row is read twice (every block has a row there). kWarpBlocks
// and kBlockThreads an SM are what registers and slots allow, kWarpBlocks - 1 without slots.
constexpr int kWarpBlocks = 3, kBlockThreads = 1024;

int64_t backward_blocks(const rune_norm_grad_args& a, Access acc, int threads) {
    const int64_t sms = sm_count(a.device);
    if (threads > 1024) return std::min(a.rows, sms * 2);
    int64_t most = sms * (acc == kWhole ? kWarpBlocks : kWarpBlocks - 1), rows = (a.rows + 7) / 8;
    if (threads > 32) most = sms * std::max(1, kBlockThreads / threads), rows = a.rows;
    most = std::max<int64_t>(8, most);
    return rows < most ? (rows + 7) / 8 * 8 : most / 8 * 8;
}

// Arrays of type-`es` rows: how all of them can be accessed.
struct Layout {
    int es;
    bool whole = true, alike = true, any = false;
    uintptr_t base = 0;
    int64_t step = 0;
    void add(const void* p, int64_t ld, int64_t width) {
        if (!p) return;
        const uintptr_t b = (uintptr_t)p % 16;
        const int64_t st = ld * es % 16;
        whole = whole && b == 0 && st == 0 && width * es % 16 == 0;
        alike = alike && b % es == 0 && (!any || (b == base && st == step));
        base = b, step = st, any = true;
    }
    Access access() const { return whole ? kWhole : alike ? kShifted : kSingle; }
};

bool known_norm_type(int dtype) {
    return dtype == RUNE_F32 || dtype == RUNE_F16 || dtype == RUNE_BF16;
}

// fn(integral_constant<Access>) for `acc`
template <typename Fn>
void with_access(Access acc, Fn&& fn) {
    if (acc == kWhole) fn(std::integral_constant<Access, kWhole>());
    else if (acc == kShifted) fn(std::integral_constant<Access, kShifted>());
    else fn(std::integral_constant<Access, kSingle>());
}

template <typename T>
void launch_norm(const rune_norm_args& a, cudaStream_t stream) {
    const bool q8 = a.out_dtype == RUNE_E4M3;
    Layout l{(int)sizeof(T)};
    l.add(a.x, a.x_stride, a.width);
    l.add(a.residual, a.residual_stride, a.width);
    l.add(a.h, a.width, a.width);
    if (!q8) l.add(a.y, a.width, a.width);
    if (q8) l.whole = l.whole && aligned(a.y, 4);
    if (a.weight) l.whole = l.whole && aligned(a.weight, 16);
    with_access(l.access(), [&](auto acc_c) {
        constexpr Access ACC = decltype(acc_c)::value;
        constexpr int N = Piece<T, ACC>::N;
        const int wide = threads_for(a.width, 2 * kEpt, ACC, N);
        if (wide > 1024) {
            const int grid = (int)std::min<int64_t>(a.rows, 1 << 20);
            if (q8) launch(k_norm_long<T, true>, grid, kLongThreads, 0, 0, stream, a);
            else launch(k_norm_long<T, false>, grid, kLongThreads, 0, 0, stream, a);
            return;
        }
        auto go = [&](auto ept_c, auto threads_c, auto block_c) {
            constexpr int EPT = decltype(ept_c)::value, THREADS = decltype(threads_c)::value;
            constexpr bool BLOCK = decltype(block_c)::value;
            const int threads = BLOCK ? wide : THREADS;
            const int64_t grid = BLOCK ? a.rows : (a.rows + 7) / 8;
            require(grid <= INT32_MAX, "too many rows");
            if (q8)
                launch(k_norm<T, ACC, EPT, THREADS, BLOCK, true>, (int)grid, threads, 0, 0, stream, a);
            else
                launch(k_norm<T, ACC, EPT, THREADS, BLOCK, false>, (int)grid, threads, 0, 0, stream,
                       a);
        };
        using std::integral_constant;
        if (threads_for(a.width, kEpt, ACC, N) == 32)
            go(integral_constant<int, kEpt>(), integral_constant<int, 256>(), std::false_type());
        else if (wide == 32)
            go(integral_constant<int, 2 * kEpt>(), integral_constant<int, 256>(),
               std::false_type());
        else if (wide <= 512)
            go(integral_constant<int, 2 * kEpt>(), integral_constant<int, 512>(),
               std::true_type());
        else
            go(integral_constant<int, 2 * kEpt>(), integral_constant<int, 1024>(),
               std::true_type());
    });
}

// shared memory of the backward's slots for one row ahead
template <typename T>
constexpr size_t slots_bytes(int threads) { return (size_t)threads * 4 * kEpt * sizeof(T); }

// rows of partials for dweight
template <typename T>
int64_t launch_norm_bwd(const rune_norm_grad_args& a, float* partials, cudaStream_t stream) {
    Layout l{(int)sizeof(T)};
    l.add(a.x, a.x_stride, a.width);
    l.add(a.residual, a.residual_stride, a.width);
    l.add(a.dy, a.dy_stride, a.width);
    l.add(a.dh, a.dh_stride, a.width);
    l.add(a.dx, a.width, a.width);
    l.whole = l.whole && aligned(a.weight, 16);
    int64_t blocks = 0;
    with_access(l.access(), [&](auto acc_c) {
        constexpr Access ACC = decltype(acc_c)::value;
        const int threads = threads_for(a.width, kEpt, ACC, Piece<T, ACC>::N);
        blocks = backward_blocks(a, ACC, threads);
        if (threads > 1024) {
            launch(k_norm_bwd_long<T>, (int)blocks, kLongThreads, 0, 0, stream, a, partials);
        } else {
            const bool block = threads > 32;
            const int n = block ? threads : 256;
            // rows ahead: kBlockThreads threads' slots have to fit an SM
            constexpr int kAheadBlock = sizeof(T) == 2 ? 3 : 1;
            constexpr int kAheadWarp = sizeof(T) == 2 ? 4 : 2;
            auto go = [&](auto block_c, auto ahead_c) {
                constexpr bool BLOCK = decltype(block_c)::value;
                constexpr int AHEAD = decltype(ahead_c)::value;
                constexpr auto kernel = k_norm_bwd<T, ACC, BLOCK, AHEAD>;
                const size_t smem = std::max(AHEAD * slots_bytes<T>(n),
                                             BLOCK ? 0 : 8 * a.width * sizeof(float));
                constexpr size_t kMost = AHEAD * slots_bytes<T>(BLOCK ? 1024 : 256);
                if constexpr (kMost > 48 * 1024) {
                    // the largest that any width takes, once: a limit of this call's own size could
                    // be lowered by another thread's narrower call before this one's launch
                    static std::atomic<uint64_t> allowed{0};  // devices whose limit is raised
                    if (a.device >= 64 ||
                        !(allowed.load(std::memory_order_relaxed) >> a.device & 1)) {
                        RUNE_CUDA_TRY(cudaFuncSetAttribute(
                            kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kMost));
                        if (a.device < 64)
                            allowed.fetch_or(uint64_t(1) << a.device, std::memory_order_relaxed);
                    }
                }
                launch(kernel, (int)blocks, n, smem, 0, stream, a, partials);
            };
            using std::integral_constant;
            constexpr bool kSlots = ACC == kWhole;
            if (block)
                go(std::true_type(), integral_constant<int, kSlots ? kAheadBlock : 0>());
            else
                go(std::false_type(), integral_constant<int, kSlots ? kAheadWarp : 0>());
        }
    });
    return blocks;
}

int64_t norm_grad_workspace(const rune_norm_grad_args& a) {
    if (!a.dweight || a.rows <= 0) return 0;
    // enough for every way that the arrays can lie
    int64_t blocks = 0;
    for (Access acc : {kWhole, kShifted, kSingle})
        for (int n : {1, 4, 8})
            blocks = std::max(blocks, backward_blocks(a, acc, threads_for(a.width, kEpt, acc, n)));
    return (blocks + partial_scratch(blocks)) * a.width * (int64_t)sizeof(float);
}

}  // namespace

int sm_count(int device) {
    constexpr int kMax = 64;
    static std::atomic<int> known[kMax];
    int n = device >= 0 && device < kMax ? known[device].load(std::memory_order_relaxed) : 0;
    if (n == 0) {
        RUNE_CUDA_TRY(cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, device));
        if (device >= 0 && device < kMax) known[device].store(n, std::memory_order_relaxed);
    }
    return n;
}

int64_t partial_scratch(int64_t parts) {
    int64_t rows = 0;
    while (parts > kPartRows) rows += parts = (parts + kPartRows - 1) / kPartRows;
    return rows;
}

void sum_partials(const float* partials, int64_t parts, int64_t width, void* out, int dtype,
                  float* scratch, cudaStream_t stream) {
    const dim3 block(32, 32);
    dim3 grid((unsigned)((width + 31) / 32));
    while (parts > kPartRows) {
        const int64_t sets = (parts + kPartRows - 1) / kPartRows;
        require(sets <= 65535, "too many rows");
        grid.y = (unsigned)sets;
        launch(k_sum_partials<float>, grid, block, 0, 0, stream, partials, parts, width, scratch);
        partials = scratch, parts = sets, grid.y = 1;
        scratch += sets * width;
    }
    if (dtype == RUNE_F32)
        launch(k_sum_partials<float>, grid, block, 0, 0, stream, partials, parts, width, (float*)out);
    else if (dtype == RUNE_F16)
        launch(k_sum_partials<__half>, grid, block, 0, 0, stream, partials, parts, width,
               (__half*)out);
    else
        launch(k_sum_partials<__nv_bfloat16>, grid, block, 0, 0, stream, partials, parts, width,
               (__nv_bfloat16*)out);
}

}  // namespace ops
}  // namespace rune

using namespace rune;
using namespace rune::ops;

extern "C" {

int rune_rms_norm(const rune_norm_args* args, void* stream_) {
    if (!args) {
        set_error("null argument");
        return RUNE_ERR_INVALID;
    }
    const rune_norm_args a = *args;
    auto stream = static_cast<cudaStream_t>(stream_);
    return guarded(a.device, [&] {
        require(a.rows >= 0 && a.width >= 1 && a.width <= INT32_MAX, "rows or width out of range");
        require(known_norm_type(a.dtype), "rms_norm takes float32, float16 or bfloat16 rows");
        require(a.weight_dtype == a.dtype || a.weight_dtype == RUNE_F32,
                "the weight has the rows' type or float32");
        require(a.out_dtype == a.dtype || (a.out_dtype == RUNE_E4M3 && a.scale),
                "the output has the rows' type, or is e4m3 with a scale array");
        check_waits(a.device);
        if (a.rows == 0) return;
        require(a.x && a.y, "null argument");
        require_aligned({a.x, a.residual, a.h}, dtype_bytes(a.dtype));
        require_aligned({a.y}, dtype_bytes(a.out_dtype));
        require_aligned({a.weight}, dtype_bytes(a.weight_dtype));
        require_aligned({a.scale, a.rstd}, sizeof(float));
        if (a.dtype == RUNE_F32) launch_norm<float>(a, stream);
        else if (a.dtype == RUNE_F16) launch_norm<__half>(a, stream);
        else launch_norm<__nv_bfloat16>(a, stream);
        RUNE_LAUNCH_CHECK();
    });
}

static void check_norm_grad(const rune_norm_grad_args& a) {
    require(a.rows >= 0 && a.width >= 1 && a.width <= INT32_MAX, "rows or width out of range");
    require(known_norm_type(a.dtype), "rms_norm takes float32, float16 or bfloat16 rows");
    require(a.weight_dtype == a.dtype || a.weight_dtype == RUNE_F32,
            "the weight has the rows' type or float32");
    require_aligned({a.x, a.residual, a.dy, a.dh, a.dx}, dtype_bytes(a.dtype));
    require_aligned({a.weight, a.dweight}, dtype_bytes(a.weight_dtype));
    require_aligned({a.rstd}, sizeof(float));
}

int rune_rms_norm_backward_workspace(const rune_norm_grad_args* args, int64_t* bytes) {
    if (!args || !bytes) {
        set_error("null argument");
        return RUNE_ERR_INVALID;
    }
    const rune_norm_grad_args a = *args;
    return guarded(a.device, [&] {
        check_norm_grad(a);
        *bytes = norm_grad_workspace(a);
    });
}

int rune_rms_norm_backward(const rune_norm_grad_args* args, void* stream_) {
    if (!args) {
        set_error("null argument");
        return RUNE_ERR_INVALID;
    }
    const rune_norm_grad_args a = *args;
    auto stream = static_cast<cudaStream_t>(stream_);
    return guarded(a.device, [&] {
        check_norm_grad(a);
        check_waits(a.device);
        const int64_t need = norm_grad_workspace(a);
        require(a.workspace_bytes >= need && (need == 0 || aligned(a.workspace, 256)),
                "the workspace is too small or not 256-byte aligned");
        if (a.rows == 0) {
            if (a.dweight)
                RUNE_CUDA_TRY(cudaMemsetAsync(
                    a.dweight, 0, (size_t)a.width * dtype_bytes(a.weight_dtype), stream));
            return;
        }
        require(a.x && a.weight && a.rstd && a.dy && a.dx, "null argument");
        float* partials = a.dweight ? static_cast<float*>(a.workspace) : nullptr;
        int64_t parts;
        if (a.dtype == RUNE_F32) parts = launch_norm_bwd<float>(a, partials, stream);
        else if (a.dtype == RUNE_F16) parts = launch_norm_bwd<__half>(a, partials, stream);
        else parts = launch_norm_bwd<__nv_bfloat16>(a, partials, stream);
        RUNE_LAUNCH_CHECK();
        if (partials)
            sum_partials(partials, parts, a.width, a.dweight, a.weight_dtype,
                         partials + parts * a.width, stream);
    });
}

}  // extern "C"
