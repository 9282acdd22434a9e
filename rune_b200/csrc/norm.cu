// Root-mean-square normalisation with the residual's addition (rune/mobius/layers.py:26-44),
//   h = x + residual,  r = 1 / sqrt(mean(h^2) + eps),  y = h r w,
// with y in the inputs' type or in 8 bits (e4m3) with a scale per row, and its backward pass
//   dx = dresidual = r (dy w - n mean(dy w n)) + dh,  n = h r,   dw = sum_rows dy n.
//
// A row stays in registers between the sum of its squares and its output, so every value is read
// once and written once: memory bandwidth bounds the kernels, launch latency the shortest calls.
// A warp takes a row of up to kWarpMax values, a block of width / 8 threads one of up to
// kBlockMax; longer rows are read twice (the second time from L2). Accesses are 16 bytes where
// addresses and strides allow, else single values of consecutive lanes.

#include <algorithm>
#include <atomic>

#include "ops.cuh"

namespace rune {
namespace ops {

namespace {

constexpr int kEpt = 8;              // values of a row per thread
constexpr int kWarpMax = 32 * kEpt;  // 256
constexpr int kWarpWide = 32 * 32;   // a warp with 32 values per lane (forward only)
constexpr int kBlockMax = 1024 * kEpt;
constexpr int kLongThreads = 1024;

// weight value: in the rows' type or float32
template <typename T, int VEC>
__device__ __forceinline__ void load_weight(const void* w, bool w32, int64_t at, float* v) {
    if (w32) {
#pragma unroll
        for (int i = 0; i < VEC; ++i) v[i] = __ldg(static_cast<const float*>(w) + at + i);
    } else {
        load_vec<T, VEC>(static_cast<const T*>(w) + at, v);
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

template <int VEC>
__device__ __forceinline__ void store_e4m3(void* y, int64_t at, const float* v) {
    auto* p = static_cast<__nv_fp8_storage_t*>(y) + at;
    if constexpr (VEC == 1) {
        *p = __nv_cvt_float_to_fp8(v[0], __NV_SATFINITE, __NV_E4M3);
    } else {
#pragma unroll
        for (int i = 0; i < VEC; i += 4) {
            uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(v[i], v[i + 1]), __NV_SATFINITE,
                                                   __NV_E4M3);
            uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(v[i + 2], v[i + 3]),
                                                   __NV_SATFINITE, __NV_E4M3);
            *reinterpret_cast<uint32_t*>(p + i) = lo | hi << 16;
        }
    }
}

// scale of a row whose largest magnitude is amax: 448 stands for amax; an all-zero row takes 1
__device__ __forceinline__ float row_scale(float amax) {
    return amax == 0.0f ? 1.0f : amax * (1.0f / kE4m3Max);
}

// ----------------------------------------------------------------------------- forward
template <typename T, int VEC, int EPT, bool BLOCK, bool Q8>
__global__ void __launch_bounds__(BLOCK ? 1024 : 256) k_norm(const rune_norm_args p) {
    constexpr int NC = EPT / VEC;
    __shared__ float shared[32];
    const int width = (int)p.width;
    const int t = BLOCK ? threadIdx.x : threadIdx.x & 31, tpr = BLOCK ? blockDim.x : 32;
    const int rpb = BLOCK ? 1 : blockDim.x >> 5;
    const bool w32 = p.weight_dtype == RUNE_F32;
    const float inv_width = 1.0f / (float)width;
    for (int64_t row = (int64_t)blockIdx.x * rpb + (BLOCK ? 0 : threadIdx.x >> 5); row < p.rows;
         row += (int64_t)gridDim.x * rpb) {
        float h[EPT], r2[EPT];
#pragma unroll
        for (int c = 0; c < NC; ++c) {
            const int col = (c * tpr + t) * VEC;
            if (col < width)
                load_vec<T, VEC>(static_cast<const T*>(p.x) + row * p.x_stride + col, h + c * VEC);
            else
                for (int i = 0; i < VEC; ++i) h[c * VEC + i] = 0.0f;
        }
        if (p.residual) {
#pragma unroll
            for (int c = 0; c < NC; ++c) {
                const int col = (c * tpr + t) * VEC;
                if (col < width)
                    load_vec<T, VEC>(
                        static_cast<const T*>(p.residual) + row * p.residual_stride + col,
                        r2 + c * VEC);
                else
                    for (int i = 0; i < VEC; ++i) r2[c * VEC + i] = 0.0f;
            }
#pragma unroll
            for (int i = 0; i < EPT; ++i) h[i] += r2[i];
            if (p.h) {
#pragma unroll
                for (int c = 0; c < NC; ++c) {
                    const int col = (c * tpr + t) * VEC;
                    if (col < width)
                        store_vec<T, VEC>(static_cast<T*>(p.h) + row * p.width + col,
                                          h + c * VEC);
                }
            }
        }
        float y[EPT];
        if (p.weight) {
            float sum = 0.0f;
#pragma unroll
            for (int i = 0; i < EPT; ++i) sum += h[i] * h[i];
            sum = row_reduce<BLOCK, false>(sum, shared);
            const float r = 1.0f / sqrtf(sum * inv_width + p.eps);
            if (p.rstd && t == 0) p.rstd[row] = r;
#pragma unroll
            for (int c = 0; c < NC; ++c) {
                const int col = (c * tpr + t) * VEC;
                float w[VEC];
                if (col < width) load_weight<T, VEC>(p.weight, w32, col, w);
#pragma unroll
                for (int i = 0; i < VEC; ++i)
                    y[c * VEC + i] = col < width ? h[c * VEC + i] * r * w[i] : 0.0f;
            }
        } else {
#pragma unroll
            for (int i = 0; i < EPT; ++i) y[i] = h[i];
        }
        float inv = 1.0f;
        if constexpr (Q8) {
            float amax = 0.0f;
#pragma unroll
            for (int i = 0; i < EPT; ++i) amax = max_nan(amax, fabsf(y[i]));
            const float scale = row_scale(row_reduce<BLOCK, true>(amax, shared));
            if (t == 0) p.scale[row] = scale;
            inv = 1.0f / scale;
        }
#pragma unroll
        for (int c = 0; c < NC; ++c) {
            const int col = (c * tpr + t) * VEC;
            if (col >= width) continue;
            if constexpr (Q8) {
                float q[VEC];
#pragma unroll
                for (int i = 0; i < VEC; ++i) q[i] = y[c * VEC + i] * inv;
                store_e4m3<VEC>(p.y, row * p.width + col, q);
            } else {
                store_vec<T, VEC>(static_cast<T*>(p.y) + row * p.width + col, y + c * VEC);
            }
        }
    }
}

// Rows longer than kBlockMax: a block reads the row for the sum (writing h), again for the
// largest magnitude (8 bits only) and again for the output; the repeats come from L2.
template <typename T, bool Q8>
__global__ void __launch_bounds__(kLongThreads) k_norm_long(const rune_norm_args p) {
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
            float w;
            load_weight<T, 1>(p.weight, w32, i, &w);
            return w;
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
                store_e4m3<1>(p.y, row * p.width + i, &y);
            } else {
                static_cast<T*>(p.y)[row * p.width + i] = from_float<T>(y);
            }
        }
    }
}

// ----------------------------------------------------------------------------- backward
// Each block keeps the sums of its rows for dweight in registers (a warp's or a block's columns
// are the same for every row that it takes) and writes one row of partials.
template <typename T, int VEC, bool BLOCK>
__global__ void __launch_bounds__(BLOCK ? 1024 : 256)
k_norm_bwd(const rune_norm_grad_args p, float* __restrict__ partials) {
    constexpr int NC = kEpt / VEC;
    __shared__ float shared[32];
    extern __shared__ float columns[];  // warps x width, when a warp takes a row
    const int width = (int)p.width;
    const int t = BLOCK ? threadIdx.x : threadIdx.x & 31, tpr = BLOCK ? blockDim.x : 32;
    const int rpb = BLOCK ? 1 : blockDim.x >> 5, warp = threadIdx.x >> 5;
    const float inv_width = 1.0f / (float)width;
    float w[kEpt], dw[kEpt];
#pragma unroll
    for (int i = 0; i < kEpt; ++i) w[i] = dw[i] = 0.0f;
#pragma unroll
    for (int c = 0; c < NC; ++c) {
        const int col = (c * tpr + t) * VEC;
        if (col < width)
            load_weight<T, VEC>(p.weight, p.weight_dtype == RUNE_F32, col, w + c * VEC);
    }
    for (int64_t row = (int64_t)blockIdx.x * rpb + (BLOCK ? 0 : warp); row < p.rows;
         row += (int64_t)gridDim.x * rpb) {
        float h[kEpt], dy[kEpt], dh[kEpt];
        const float r = p.rstd[row];
#pragma unroll
        for (int i = 0; i < kEpt; ++i) h[i] = dy[i] = dh[i] = 0.0f;
#pragma unroll
        for (int c = 0; c < NC; ++c) {
            const int col = (c * tpr + t) * VEC;
            if (col >= width) continue;
            load_vec<T, VEC>(static_cast<const T*>(p.h) + row * p.h_stride + col, h + c * VEC);
            load_vec<T, VEC>(static_cast<const T*>(p.dy) + row * p.dy_stride + col, dy + c * VEC);
            if (p.dh)
                load_vec<T, VEC>(static_cast<const T*>(p.dh) + row * p.dh_stride + col,
                                 dh + c * VEC);
        }
        float dot = 0.0f;
#pragma unroll
        for (int i = 0; i < kEpt; ++i) {
            h[i] *= r;  // n
            dw[i] += dy[i] * h[i];
            dy[i] *= w[i];
            dot += dy[i] * h[i];
        }
        dot = row_reduce<BLOCK, false>(dot, shared) * inv_width;
#pragma unroll
        for (int c = 0; c < NC; ++c) {
            const int col = (c * tpr + t) * VEC;
            if (col >= width) continue;
            float dx[VEC];
#pragma unroll
            for (int i = 0; i < VEC; ++i) {
                const int j = c * VEC + i;
                dx[i] = r * (dy[j] - h[j] * dot) + dh[j];
            }
            store_vec<T, VEC>(static_cast<T*>(p.dx) + row * p.width + col, dx);
        }
    }
    if (!partials) return;
    if constexpr (BLOCK) {
#pragma unroll
        for (int c = 0; c < NC; ++c) {
            const int col = (c * tpr + t) * VEC;
            if (col >= width) continue;
#pragma unroll
            for (int i = 0; i < VEC; ++i)
                partials[(int64_t)blockIdx.x * width + col + i] = dw[c * VEC + i];
        }
    } else {
#pragma unroll
        for (int c = 0; c < NC; ++c) {
            const int col = (c * tpr + t) * VEC;
            if (col >= width) continue;
#pragma unroll
            for (int i = 0; i < VEC; ++i) columns[warp * width + col + i] = dw[c * VEC + i];
        }
        __syncthreads();
        for (int col = threadIdx.x; col < width; col += blockDim.x) {
            float s = 0.0f;
            for (int k = 0; k < rpb; ++k) s += columns[k * width + col];
            partials[(int64_t)blockIdx.x * width + col] = s;
        }
    }
}

// Rows longer than kBlockMax: the row is read twice and the block's partials are accumulated in
// its own row of the workspace (each column always by the same thread).
template <typename T>
__global__ void __launch_bounds__(kLongThreads)
k_norm_bwd_long(const rune_norm_grad_args p, float* __restrict__ partials) {
    __shared__ float shared[32];
    const bool w32 = p.weight_dtype == RUNE_F32;
    const int t = threadIdx.x;
    bool first = true;
    for (int64_t row = blockIdx.x; row < p.rows; row += gridDim.x, first = false) {
        const T* hp = static_cast<const T*>(p.h) + row * p.h_stride;
        const T* dyp = static_cast<const T*>(p.dy) + row * p.dy_stride;
        const T* dhp = p.dh ? static_cast<const T*>(p.dh) + row * p.dh_stride : nullptr;
        const float r = p.rstd[row];
        float dot = 0.0f;
        for (int64_t i = t; i < p.width; i += blockDim.x) {
            float w, n = to_float(hp[i]) * r, dy = to_float(dyp[i]);
            load_weight<T, 1>(p.weight, w32, i, &w);
            dot += dy * w * n;
            if (partials) {
                float* at = partials + (int64_t)blockIdx.x * p.width + i;
                *at = (first ? 0.0f : *at) + dy * n;
            }
        }
        dot = row_reduce<true, false>(dot, shared) / (float)p.width;
        for (int64_t i = t; i < p.width; i += blockDim.x) {
            float w, n = to_float(hp[i]) * r;
            load_weight<T, 1>(p.weight, w32, i, &w);
            float dx = r * (to_float(dyp[i]) * w - n * dot) + (dhp ? to_float(dhp[i]) : 0.0f);
            static_cast<T*>(p.dx)[row * p.width + i] = from_float<T>(dx);
        }
    }
}

// Columns of float32 partials [parts][width]: a block sums 32 columns with 32 threads each, then
// joins the 32 sums in order.
template <typename T>
__global__ void __launch_bounds__(1024)
k_sum_partials(const float* __restrict__ partials, int64_t parts, int64_t width, T* out) {
    __shared__ float s[32][33];
    const int64_t col = (int64_t)blockIdx.x * 32 + threadIdx.x;
    float v = 0.0f;
    if (col < width)
        for (int64_t r = threadIdx.y; r < parts; r += 32) v += partials[r * width + col];
    s[threadIdx.y][threadIdx.x] = v;
    __syncthreads();
    if (threadIdx.y == 0 && col < width) {
        float sum = 0.0f;
        for (int k = 0; k < 32; ++k) sum += s[k][threadIdx.x];
        out[col] = from_float<T>(sum);
    }
}

// ----------------------------------------------------------------------------- host
int threads_for(int64_t width) { return (int)((width + kEpt * 32 - 1) / (kEpt * 32)) * 32; }

// Blocks of the backward: enough to fill the GPU; each leaves one row of partials.
int64_t backward_blocks(const rune_norm_grad_args& a) {
    const int64_t sms = sm_count(a.device);
    if (a.width <= kWarpMax) return std::min((a.rows + 7) / 8, sms * 6);
    if (a.width > kBlockMax) return std::min(a.rows, sms * 2);
    return std::min(a.rows, sms * std::max<int64_t>(1, 1024 / threads_for(a.width)));
}

bool known_norm_type(int dtype) {
    return dtype == RUNE_F32 || dtype == RUNE_F16 || dtype == RUNE_BF16;
}

template <typename T>
void launch_norm(const rune_norm_args& a, cudaStream_t stream) {
    constexpr int V = 16 / sizeof(T);
    const bool q8 = a.out_dtype == RUNE_E4M3;
    bool vec = a.width % V == 0 && a.x_stride % V == 0 && aligned(a.x, 16) && aligned(a.y, 16) &&
               (!a.weight || aligned(a.weight, 16)) &&
               (!a.residual || (aligned(a.residual, 16) && a.residual_stride % V == 0)) &&
               (!a.h || aligned(a.h, 16));
    if (a.width > kBlockMax) {
        int grid = (int)std::min<int64_t>(a.rows, 1 << 20);
        if (q8) k_norm_long<T, true><<<grid, kLongThreads, 0, stream>>>(a);
        else k_norm_long<T, false><<<grid, kLongThreads, 0, stream>>>(a);
        return;
    }
    auto go = [&](auto vec_c, auto ept_c, auto block_c) {
        constexpr int VEC = decltype(vec_c)::value, EPT = decltype(ept_c)::value;
        constexpr bool BLOCK = decltype(block_c)::value;
        const int64_t rpb = BLOCK ? 1 : 8;
        const int threads = BLOCK ? threads_for(a.width) : 256;
        const int grid = (int)std::min<int64_t>((a.rows + rpb - 1) / rpb, 1 << 20);
        if (q8) k_norm<T, VEC, EPT, BLOCK, true><<<grid, threads, 0, stream>>>(a);
        else k_norm<T, VEC, EPT, BLOCK, false><<<grid, threads, 0, stream>>>(a);
    };
    using std::integral_constant;
    auto shape = [&](auto vec_c) {
        if (a.width <= kWarpMax)
            go(vec_c, integral_constant<int, kEpt>(), std::false_type());
        else if (a.width <= kWarpWide)
            go(vec_c, integral_constant<int, 32>(), std::false_type());
        else
            go(vec_c, integral_constant<int, kEpt>(), std::true_type());
    };
    if (vec) shape(integral_constant<int, V>());
    else shape(integral_constant<int, 1>());
}

template <typename T>
void launch_norm_bwd(const rune_norm_grad_args& a, float* partials, cudaStream_t stream) {
    constexpr int V = 16 / sizeof(T);
    const int grid = (int)backward_blocks(a);
    if (a.width > kBlockMax) {
        k_norm_bwd_long<T><<<grid, kLongThreads, 0, stream>>>(a, partials);
        return;
    }
    bool vec = a.width % V == 0 && a.h_stride % V == 0 && a.dy_stride % V == 0 &&
               aligned(a.h, 16) && aligned(a.dy, 16) && aligned(a.weight, 16) &&
               aligned(a.dx, 16) && (!a.dh || (aligned(a.dh, 16) && a.dh_stride % V == 0));
    const bool block = a.width > kWarpMax;
    const int threads = block ? threads_for(a.width) : 256;
    const size_t smem = block ? 0 : 8 * (size_t)a.width * sizeof(float);
    if (vec && block) k_norm_bwd<T, V, true><<<grid, threads, smem, stream>>>(a, partials);
    else if (vec) k_norm_bwd<T, V, false><<<grid, threads, smem, stream>>>(a, partials);
    else if (block) k_norm_bwd<T, 1, true><<<grid, threads, smem, stream>>>(a, partials);
    else k_norm_bwd<T, 1, false><<<grid, threads, smem, stream>>>(a, partials);
}

int64_t norm_grad_workspace(const rune_norm_grad_args& a) {
    if (!a.dweight || a.rows <= 0) return 0;
    return backward_blocks(a) * a.width * (int64_t)sizeof(float);
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

void sum_partials(const float* partials, int64_t parts, int64_t width, void* out, int dtype,
                  cudaStream_t stream) {
    dim3 block(32, 32);
    int grid = (int)((width + 31) / 32);
    if (dtype == RUNE_F32)
        k_sum_partials<<<grid, block, 0, stream>>>(partials, parts, width, (float*)out);
    else if (dtype == RUNE_F16)
        k_sum_partials<<<grid, block, 0, stream>>>(partials, parts, width, (__half*)out);
    else
        k_sum_partials<<<grid, block, 0, stream>>>(partials, parts, width, (__nv_bfloat16*)out);
    RUNE_LAUNCH_CHECK();
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
        if (a.rows == 0) return;
        require(a.x && a.y, "null argument");
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
        const int64_t need = norm_grad_workspace(a);
        require(a.workspace_bytes >= need && (need == 0 || aligned(a.workspace, 256)),
                "the workspace is too small or not 256-byte aligned");
        if (a.rows == 0) {
            if (a.dweight)
                RUNE_CUDA_TRY(cudaMemsetAsync(
                    a.dweight, 0, (size_t)a.width * dtype_bytes(a.weight_dtype), stream));
            return;
        }
        require(a.h && a.weight && a.rstd && a.dy && a.dx, "null argument");
        float* partials = a.dweight ? static_cast<float*>(a.workspace) : nullptr;
        if (a.dtype == RUNE_F32) launch_norm_bwd<float>(a, partials, stream);
        else if (a.dtype == RUNE_F16) launch_norm_bwd<__half>(a, partials, stream);
        else launch_norm_bwd<__nv_bfloat16>(a, partials, stream);
        RUNE_LAUNCH_CHECK();
        if (partials)
            sum_partials(partials, backward_blocks(a), a.width, a.dweight, a.weight_dtype,
                         stream);
    });
}

}  // extern "C"
