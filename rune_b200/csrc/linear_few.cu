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
// Rows by group (grouped_few): the same for each group that has rows, of which there are no more than
// rows; the blocks find theirs in the offsets. Gated 10 x 4096 -> 2 x 2048, six of 16 groups met: 37 us,
// 5.4 TB/s of weights (the tiles: 60 us).
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
    int tiles, groups;       // GROUPED: tiles of a group's outputs
    const int32_t* offsets;
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

// The want-th group that has rows; false if there are fewer. By all threads, with room for the groups'
// first rows at `first`.
__device__ __forceinline__ bool find_group(const FewParams& p, int want, int* first, int& group,
                                           int& row0, int& rows) {
    for (int g = threadIdx.x; g <= p.groups; g += kThreads)
        first[g] = min(max(p.offsets[g], 0), p.rows);
    __syncthreads();
    const int lane = threadIdx.x & 31;
    bool found = false;
    for (int g0 = 0; g0 < p.groups && !found; g0 += 32) {
        const int g = min(g0 + lane, p.groups - 1);
        const unsigned some =
            __ballot_sync(0xffffffffu, g0 + lane < p.groups && first[g + 1] > first[g]);
        const int n = __popc(some);
        if (want < n) {
            group = g0 + (int)__fns(some, 0, want + 1);
            row0 = first[group], rows = first[group + 1] - row0;
            found = true;
        }
        want -= n;
    }
    tc::fence_async_smem();  // copies come here next
    __syncthreads();
    return found;
}

template <typename T, bool FP8, bool GROUPED>
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
    const int tile = (int)(blockIdx.x / splits);
    const int64_t f0 = (int64_t)(GROUPED ? tile % p.tiles : tile) * width;
    int group = 0, row0 = 0, rows = p.rows;
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
    if (!GROUPED && warp == kPrefetchWarp && kb1 - kb0 > p.stages) {
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
    bool work = true;
    if constexpr (GROUPED) {
        int* first = reinterpret_cast<int*>(smem);  // the ring's memory, before it is in use
        work = find_group(p, tile / p.tiles, first, group, row0, rows);
        // the rows that no group has
        const int end = min(max(p.offsets[p.groups], 0), p.rows);
        const int64_t n = (int64_t)(p.rows - end) * p.n;
        for (int64_t i = (int64_t)blockIdx.x * kThreads + tid; i < n;
             i += (int64_t)gridDim.x * kThreads)
            static_cast<T*>(p.out)[end * p.n + i] = from_float<T>(0.0f);
        if (!work) {  // and so for the whole cluster
            if (warp == 5) tmem_dealloc(tmem, p.tmem_cols);
            return;
        }
    }
    const int64_t bias_at = GROUPED ? (int64_t)group * (p.gated ? 2 * p.n : p.n) : 0;

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
                    auto load_w = [&](uint32_t to, int64_t feature) {
                        if constexpr (GROUPED) tma_load3(to, &map_w, x, (int)feature, group, bar);
                        else tma_load(to, &map_w, x, (int)feature, bar);
                    };
                    load_w(a + l * kWLine, f0);
                    if (p.gated) load_w(a + l * kWLine + kWLine / 2, p.n + f0);
                    tma_load(a + kLines * kWLine + l * x_line, &map_x, x, row0, bar);
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
        for (int c = 0; c < rows; c += 16) {
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
            bias[0] = to_float(static_cast<const T*>(p.bias)[bias_at + col]);
            if (p.gated) bias[1] = to_float(static_cast<const T*>(p.bias)[bias_at + up]);
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
                const int at = min(row + i * step, rows - 1) * kFeatures + feature;
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
            for (int r0 = tid / per; r0 < rows; r0 += step * kRows) {
                float z[kRows], u[kRows];
                sums_of(r0, f, z);
                if (p.gated) sums_of(r0, f + width, u);
#pragma unroll
                for (int i = 0; i < kRows; ++i) {
                    const int row = row0 + min(r0 + i * step, rows - 1);  // the last one repeats
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

template <typename T, bool FP8, bool GROUPED>
void launch_few(const CUtensorMap& mw, const CUtensorMap& mx, const FewParams& p, int tiles,
                int splits, int device, cudaStream_t stream) {
    static std::atomic<uint64_t> allowed{0};
    if (device >= 64 || !(allowed.load(std::memory_order_relaxed) >> device & 1)) {
        RUNE_CUDA_TRY(cudaFuncSetAttribute(k_few<T, FP8, GROUPED>,
                                           cudaFuncAttributeMaxDynamicSharedMemorySize,
                                           (int)kSmemMax));
        if (device < 64) allowed.fetch_or(uint64_t(1) << device, std::memory_order_relaxed);
    }
    launch(k_few<T, FP8, GROUPED>, (unsigned)(tiles * splits), kThreads, p.ring_bytes + sizeof(FewShared),
           splits, stream, mw, mx, p);
}

// What both calls share: blocks, ring and product of `count` layers of at most p.rows rows each.
// Returns the range of k's splits.
int plan_few(FewParams& p, int64_t inputs, int64_t count, int dtype, int device) {
    const bool fp8 = dtype == RUNE_E4M3;
    const int line = kLines * (int)kLineBytes / (fp8 ? 1 : 2), sms = sm_count(device);
    p.rows_pad = (p.rows + 15) / 16 * 16;
    p.kblocks = (int)((inputs + line - 1) / line);
    const int width = p.gated ? kFeatures / 2 : kFeatures;
    p.tiles = (int)((p.n + width - 1) / width);
    // as many blocks as two an SM, with a stage of k each at least
    int splits = 1;
    while (splits < 8 && p.tiles * count * splits * 2 <= 2 * sms && p.kblocks >= splits * 2)
        splits *= 2;
    const uint32_t stage = kLines * (kWLine + (uint32_t)p.rows_pad * kLineBytes);
    p.stages = (int)std::min<uint32_t>(kMaxStages, kRingBytes / stage);
    p.ring_bytes = std::max(p.stages * stage, p.rows_pad * kFeatures * (uint32_t)sizeof(float));
    p.tmem_cols = p.rows_pad <= 32 ? 32 : p.rows_pad <= 64 ? 64 : 128;
    p.idesc = operand_idesc(!fp8 && dtype == RUNE_BF16 ? 1 : 0, false, false, kFeatures, p.rows_pad);
    p.flag = wait_flag(device);
    p.polls = wait_polls();
    return splits;
}

}  // namespace

// The layer of `a` with operands x and w that TMA can read; a.rows at most kFewRows.
void linear_few(const rune_linear_args& a, const Matrix& x, const Matrix& w, cudaStream_t stream) {
    const bool fp8 = a.dtype == RUNE_E4M3;
    const int eb = fp8 ? 1 : 2, width = a.gated ? kFeatures / 2 : kFeatures;
    FewParams p{};
    p.rows = (int)a.rows;
    p.n = a.outputs;
    p.gated = a.gated;
    p.act = a.activation;
    const int splits = plan_few(p, a.inputs, 1, a.dtype, a.device);
    p.bias = a.bias;
    p.res = a.residual, p.ld_res = a.residual_stride;
    p.x_scale = a.x_scale, p.w_scale = a.weight_scale;
    p.out = a.y;
    p.z = a.saved;
    const CUtensorMap mw = make_map(w, eb, width), mx = make_map(x, eb, p.rows_pad);
    const bool half = a.out_dtype == RUNE_F16;
    auto go = [&](auto t) {
        using T = decltype(t);
        if (fp8)
            launch_few<T, true, false>(mw, mx, p, p.tiles, splits, a.device, stream);
        else
            launch_few<T, false, false>(mw, mx, p, p.tiles, splits, a.device, stream);
    };
    if (half) go(__half());
    else go(__nv_bfloat16());
}

// The grouped layer of `a` likewise; w: the groups' matrices one below the other.
void grouped_few(const rune_grouped_linear_args& a, const Matrix& x, const Matrix& w,
                 cudaStream_t stream) {
    const int64_t n_all = a.gated ? 2 * a.outputs : a.outputs, met = std::min(a.groups, a.rows);
    FewParams p{};
    p.rows = (int)a.rows;
    p.groups = (int)a.groups;
    p.offsets = a.offsets;
    p.n = a.outputs;
    p.gated = a.gated;
    p.act = a.activation;
    const int splits = plan_few(p, a.inputs, met, a.dtype, a.device);
    p.bias = a.bias;
    p.out = a.y;
    p.z = a.saved;
    Matrix one = w;
    one.rows = n_all;
    const CUtensorMap mw = make_map3(one, a.groups, n_all * w.ld, 2,
                                     a.gated ? kFeatures / 2 : kFeatures);
    const CUtensorMap mx = make_map(x, 2, p.rows_pad);
    require(p.tiles * met * splits < (1LL << 31), "too many tiles");
    auto go = [&](auto t) {
        using T = decltype(t);
        launch_few<T, false, true>(mw, mx, p, (int)(p.tiles * met), splits, a.device, stream);
    };
    if (a.dtype == RUNE_F16) go(__half());
    else go(__nv_bfloat16());
}

}  // namespace ops
}  // namespace rune
