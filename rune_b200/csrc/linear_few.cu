// Linear and gated layers for few rows (decoding, single structures): the weights are read once
// and bound the time, so the product is turned round, D[feature, row] = sum_k W[feature, k] x[row, k]:
// a block takes 128 weight rows (gated: 64 gate rows and their 64 partners) as the tensor core's
// M and all rows of x, at most kFewRows, as its N. The range of k is split over the blocks of a
// cluster, whose sums meet in distributed shared memory, each block finishing its share of the
// features: one launch, no scratch, the same order of additions every time.
//
// B200, bf16: 1 x 4096 -> 8192 13.8 us, 4.9 TB/s of weights (the 128-row tiles: 44 us); gated
// 5 x 4096 -> 2 x 8192 24.2 us, 5.6 TB/s. Some 3 us are launch, first copies and the join; a third
// of them hides behind the kernel before.
//
// Warp 4 streams W and x by TMA through a ring, warp 5 issues the products, warps 0-3 read the
// accumulator (a lane holds a feature) into the ring's memory, free by then, for the join.

#include <algorithm>
#include <atomic>

#include "linear.cuh"

namespace rune {
namespace ops {

namespace {

constexpr int kThreads = 192;
constexpr int kPrefetchWarp = 4;  // the TMA warp
constexpr int kFeatures = 128;
constexpr uint32_t kWLine = kFeatures * kLineBytes;  // 16 KB
// 128-byte lines of k in a stage: the loop over stages costs some 0.3 us a turn, which the four
// small products of one line do not fill (1 x 8192 -> 1024 with one line 8.5 us)
constexpr int kLines = 2;
constexpr int kMaxStages = 12;
constexpr uint32_t kRingBytes = 108 * 1024;           // two blocks an SM
constexpr uint32_t kSmemMax = kRingBytes + 1024;

struct FewParams {
    int rows, rows_pad;      // rows of x, and rounded up to the tensor core's 16
    int64_t n;               // outputs
    int kblocks;             // stages of k
    int stages, act, gated;
    uint32_t idesc, tmem_cols, ring_bytes;
    int64_t ld_res;
    const void* bias;
    const void* res;
    const float* x_scale;
    const float* w_scale;
    void* out;
    float* z;
    unsigned* flag;
    unsigned polls;          // bound of every wait
};

struct FewShared {
    unsigned long long full[kMaxStages], empty[kMaxStages], done;
    uint32_t tmem;
    int fail;
    int issued;
};

template <typename T, bool FP8>
__global__ void __launch_bounds__(kThreads)
k_few(const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_x,
      const FewParams p) {
    using namespace tc;
    extern __shared__ __align__(1024) unsigned char smem[];
    const int tid = threadIdx.x, lane = tid & 31;
    const int warp = __shfl_sync(0xffffffffu, tid >> 5, 0);
    constexpr int kLine = FP8 ? 128 : 64;  // values
    const uint32_t x_line = (uint32_t)p.rows_pad * kLineBytes;
    const uint32_t stage_bytes = kLines * (kWLine + x_line);
    FewShared& sh = *reinterpret_cast<FewShared*>(smem + p.ring_bytes);
    const uint32_t splits = cluster_size(), rank = cluster_rank();
    const int width = p.gated ? kFeatures / 2 : kFeatures;  // features of y in this tile
    const int64_t f0 = (int64_t)(blockIdx.x / splits) * width;
    const int kb0 = p.kblocks * (int)rank / (int)splits;
    const int kb1 = p.kblocks * ((int)rank + 1) / (int)splits;
    volatile int* fail = &sh.fail;

    if (tid == 0) {
        for (int s = 0; s < p.stages; ++s) {
            mbar_init(smem_u32(&sh.full[s]), 1);
            mbar_init(smem_u32(&sh.empty[s]), 1);
        }
        mbar_init(smem_u32(&sh.done), 1);
        sh.fail = 0;
        sh.issued = 0;
        asm volatile("fence.mbarrier_init.release.cluster;");
    }
    if (tid == 128) {
        prefetch_map(&map_w);
        prefetch_map(&map_x);
    }
    if (warp == 5) tmem_alloc(&sh.tmem, p.tmem_cols);
    fence_before_sync();
    __syncthreads();
    fence_after_sync();
    const uint32_t tmem = __shfl_sync(0xffffffffu, sh.tmem, 0);
    if (warp == kPrefetchWarp && kb1 - kb0 > p.stages) {
        // the first weights on their way to L2, where a write by the kernel before would still be
        // seen, while that kernel ends (5 x 4096 -> 2 x 8192 25.0 -> 24.4 us); not where the ring
        // takes them all at once (1 x 1024 -> 1024 4.1 -> 4.4)
        const int kb = kb0 * kLines + lane;
        if (lane < p.stages * kLines && kb < kb1 * kLines) {
            prefetch_tile(&map_w, kb * kLine, (int)f0);
            if (p.gated) prefetch_tile(&map_w, kb * kLine, (int)(p.n + f0));
        }
        __syncwarp();
    }
    follow_on();

    if (warp == 4) {
        const bool one = elect_one();
        int st = 0, issued = 0;
        uint32_t parity = 1;
        bool ok = true;
        for (int kb = kb0; kb < kb1; ++kb) {
            ok = mbar_wait(smem_u32(&sh.empty[st]), parity, p.polls) && !*fail;
            if (!__all_sync(0xffffffffu, ok)) {
                ok = false;
                break;
            }
            const uint32_t bar = smem_u32(&sh.full[st]);
            const uint32_t a = smem_u32(smem) + (uint32_t)st * stage_bytes;
            if (one) {
                mbar_expect_tx(bar, stage_bytes);
#pragma unroll
                for (int l = 0; l < kLines; ++l) {
                    const int x = (kb * kLines + l) * kLine;
                    tma_load(a + l * kWLine, &map_w, x, (int)f0, bar);
                    if (p.gated)
                        tma_load(a + l * kWLine + kWLine / 2, &map_w, x, (int)(p.n + f0), bar);
                    tma_load(a + kLines * kWLine + l * x_line, &map_x, x, 0, bar);
                }
            }
            __syncwarp();  // the other lanes' polling must not hold up the copies' issue
            ++issued;
            if (++st == p.stages) st = 0, parity ^= 1;
        }
        if (!ok) *fail = 1;
        if (one) sh.issued = issued;
    } else if (warp == 5) {
        const bool one = elect_one();
        const uint64_t desc_w = operand_desc(smem_u32(smem), false);
        const uint64_t desc_x = operand_desc(smem_u32(smem) + kLines * kWLine, false);
        int st = 0;
        uint32_t parity = 0;
        bool ok = true;
        for (int kb = kb0; kb < kb1; ++kb) {
            ok = mbar_wait(smem_u32(&sh.full[st]), parity, p.polls) && !*fail;
            if (!__all_sync(0xffffffffu, ok)) {
                ok = false;
                break;
            }
            fence_after_sync();
            const uint64_t at = (uint64_t)((uint32_t)st * (stage_bytes >> 4));
            if (one) {
#pragma unroll
                for (int l = 0; l < kLines; ++l)
#pragma unroll
                    for (int k = 0; k < 4; ++k)
                        mma<FP8, false>(tmem, desc_w + at + l * (kWLine >> 4) + 2 * k,
                                        desc_x + at + l * (x_line >> 4) + 2 * k, p.idesc,
                                        kb > kb0 || l > 0 || k > 0);
                mma_commit(smem_u32(&sh.empty[st]));
            }
            __syncwarp();
            if (++st == p.stages) st = 0, parity ^= 1;
        }
        if (one) mma_commit(smem_u32(&sh.done));
        __syncwarp();
        if (!ok) *fail = 1;
    }
    // every warp meets here, also after a failure; the products are done before the ring is reused
    __syncthreads();
    if (!mbar_wait(smem_u32(&sh.done), 0, p.polls)) *fail = 1;
    __syncthreads();
    const bool failed = *fail;
    if (failed) {
        // what is in flight lands, by waits of the full bound, before the ring takes the sums and
        // TMEM goes: the copies first, then the products (warp 5 commits `done` in any case)
        if (tid == 0) {
            atomicExch_system(p.flag, 1u);
            for (int i = max(0, sh.issued - p.stages); i < sh.issued; ++i)
                mbar_wait(smem_u32(&sh.full[i % p.stages]), (i / p.stages) & 1);
        }
        mbar_wait(smem_u32(&sh.done), 0);
        __syncthreads();
    }
    fence_after_sync();
    float* sums = reinterpret_cast<float*>(smem);  // [rows_pad][128]
    if (warp < 4 && !failed) {
        for (int c = 0; c < p.rows; c += 16) {
            float v[16];
            tmem_ld16(tmem + ((uint32_t)(warp * 32) << 16) + c, v);
#pragma unroll
            for (int j = 0; j < 16; ++j) sums[(c + j) * kFeatures + tid] = v[j];
        }
    }
    fence_before_sync();
    __syncwarp();
    if (splits > 1) cluster_sync();
    else __syncthreads();
    // This block's share: `per` features of the tile, all rows, the blocks' sums in their order.
    // A thread keeps one feature, so its bias and scale are read once and neighbouring lanes
    // write neighbouring outputs.
    const int per = width / (int)splits, f = (int)rank * per + tid % per;
    const int64_t col = f0 + f;
    if (warp < 4 && col < p.n && !failed) {
        const uint32_t base = smem_u32(sums);
        const int step = 128 / per;
        const int64_t up = p.n + col;
        float bias[2] = {0.0f, 0.0f}, scale[2] = {1.0f, 1.0f};
        if (p.bias) {
            bias[0] = to_float(static_cast<const T*>(p.bias)[col]);
            if (p.gated) bias[1] = to_float(static_cast<const T*>(p.bias)[up]);
        }
        if (p.w_scale) {
            scale[0] = p.w_scale[col];
            if (p.gated) scale[1] = p.w_scale[up];
        }
        // kRows rows at a time: their remote loads are all in flight before the first is used
        constexpr int kRows = 4;
        auto sums_of = [&](int row, int feature, float (&s)[kRows]) {
            float v[kRows][8];
#pragma unroll
            for (int i = 0; i < kRows; ++i) {
                const int at = min(row + i * step, p.rows - 1) * kFeatures + feature;
                if (splits == 1) {
                    v[i][0] = sums[at];
                } else {
#pragma unroll
                    for (int r = 0; r < 8; ++r)
                        if (r < (int)splits) v[i][r] = peer_float(peer_address(base + at * 4, r));
                }
            }
#pragma unroll
            for (int i = 0; i < kRows; ++i) {
                s[i] = v[i][0];
#pragma unroll
                for (int r = 1; r < 8; ++r)
                    if (r < (int)splits) s[i] += v[i][r];
            }
        };
        with_activation(p.act, [&](auto a) {
            for (int row0 = tid / per; row0 < p.rows; row0 += step * kRows) {
                float z[kRows], u[kRows];
                sums_of(row0, f, z);
                if (p.gated) sums_of(row0, f + width, u);
#pragma unroll
                for (int i = 0; i < kRows; ++i) {
                    const int row = min(row0 + i * step, p.rows - 1);  // the last one repeats
                    const float xs = p.x_scale ? p.x_scale[row] : 1.0f;
                    z[i] = z[i] * (xs * scale[0]) + bias[0];
                    if (p.gated) u[i] = u[i] * (xs * scale[1]) + bias[1];
                    if (p.z) {
                        const int64_t line = (p.n + 3) / 4 * 4;
                        float* at = p.z + row * (p.gated ? 2 * line : line) + col;
                        at[0] = z[i];
                        if (p.gated) at[line] = u[i];
                    }
                    float v = act_value<decltype(a)::value>(z[i]);
                    if (p.gated) v *= u[i];
                    else if (p.res)
                        v += to_float(static_cast<const T*>(p.res)[row * p.ld_res + col]);
                    static_cast<T*>(p.out)[row * p.n + col] = from_float<T>(v);
                }
            }
        });
    }
    // the blocks of the cluster stay until all have read; then TMEM goes
    __syncwarp();
    if (splits > 1) cluster_sync();
    else __syncthreads();
    if (warp == 5) {
        fence_after_sync();
        tmem_dealloc(tmem, p.tmem_cols);
    }
}

template <typename T, bool FP8>
void launch_few(const CUtensorMap& mw, const CUtensorMap& mx, const FewParams& p, int tiles,
                int splits, int device, cudaStream_t stream) {
    static std::atomic<uint64_t> allowed{0};
    if (device >= 64 || !(allowed.load(std::memory_order_relaxed) >> device & 1)) {
        RUNE_CUDA_TRY(cudaFuncSetAttribute(k_few<T, FP8>,
                                           cudaFuncAttributeMaxDynamicSharedMemorySize,
                                           (int)kSmemMax));
        if (device < 64) allowed.fetch_or(uint64_t(1) << device, std::memory_order_relaxed);
    }
    launch(k_few<T, FP8>, (unsigned)(tiles * splits), kThreads, p.ring_bytes + sizeof(FewShared),
           splits, stream, mw, mx, p);
}

}  // namespace

// The layer of `a` with operands x and w that TMA can read; a.rows at most kFewRows.
void linear_few(const rune_linear_args& a, const Matrix& x, const Matrix& w, cudaStream_t stream) {
    const bool fp8 = a.dtype == RUNE_E4M3;
    const int eb = fp8 ? 1 : 2, line = kLines * (int)kLineBytes / eb, sms = sm_count(a.device);
    FewParams p{};
    p.rows = (int)a.rows;
    p.rows_pad = (p.rows + 15) / 16 * 16;
    p.n = a.outputs;
    p.gated = a.gated;
    p.act = a.activation;
    p.kblocks = (int)((a.inputs + line - 1) / line);
    const int width = a.gated ? kFeatures / 2 : kFeatures;
    const int64_t tiles = (a.outputs + width - 1) / width;
    // as many blocks as two an SM, with a stage of k each at least
    int splits = 1;
    while (splits < 8 && tiles * splits * 2 <= 2 * sms && p.kblocks >= splits * 2)
        splits *= 2;
    const uint32_t stage = kLines * (kWLine + (uint32_t)p.rows_pad * kLineBytes);
    p.stages = (int)std::min<uint32_t>(kMaxStages, kRingBytes / stage);
    p.ring_bytes = std::max(p.stages * stage, p.rows_pad * kFeatures * (uint32_t)sizeof(float));
    p.tmem_cols = p.rows_pad <= 32 ? 32 : p.rows_pad <= 64 ? 64 : 128;
    p.idesc = operand_idesc(!fp8 && a.dtype == RUNE_BF16 ? 1 : 0, false, false, kFeatures,
                            p.rows_pad);
    p.bias = a.bias;
    p.res = a.residual, p.ld_res = a.residual_stride;
    p.x_scale = a.x_scale, p.w_scale = a.weight_scale;
    p.out = a.y;
    p.z = a.saved;
    p.flag = wait_flag(a.device);
    p.polls = wait_polls();
    const CUtensorMap mw = make_map(w, eb, width), mx = make_map(x, eb, p.rows_pad);
    const bool half = a.out_dtype == RUNE_F16;
    auto go = [&](auto t) {
        using T = decltype(t);
        if (fp8) launch_few<T, true>(mw, mx, p, (int)tiles, splits, a.device, stream);
        else launch_few<T, false>(mw, mx, p, (int)tiles, splits, a.device, stream);
    };
    if (half) go(__half());
    else go(__nv_bfloat16());
}

}  // namespace ops
}  // namespace rune
