// Newton-Schulz orthogonalisation of a stack of matrices (orthogonalize): from X = x / (|x|_F + eps),
// `steps` times
//   A = X X^T,   B = b A + c A A,   X <- a X + B X
// (with more rows than columns A = X^T X and X <- a X + X B: the tensor core reads X in its other
// order, nothing is transposed). With a, b, c of a steep odd polynomial the singular values of X
// approach 1.
//
// Three products a step on the tile kernel, over all matrices of the stack at once; A and B are
// symmetric, so only the tiles on and below the diagonal are computed, and each leaves twice.
//
// Operands are float16, scaled by 2^10: |x|_F <= 1 leaves values of X near 1 / sqrt(rows columns),
// and of A and B at most a few units, and 2^10 keeps both clear of float16's smallest normal
// numbers (2^-24 after scaling) and of its largest (64). bfloat16 would need no scale, but every
// step rounds X, A and B, and 8 bits instead of 11 cost eight times the error of the result.
// The norm is summed in float64, products in float32.
//
// Small matrices spend a product's time between launches (5.5 us each for 256 x 512), so k_small
// takes one matrix through all steps in a cluster of eight blocks, which meet between products:
// 8 x 256 x 512, five steps, 95 us as a chain of launches, @@ us so.

#include <cmath>

#include "tile.cuh"

namespace rune {
namespace ops {

namespace {

constexpr float kScale = 1024.0f;  // of X, A and B
constexpr int kNormThreads = 256;

struct NormParams {
    int64_t rows, cols, step, row, col;  // of x, strides in elements
    int64_t ld, out_step;                // of the scaled copy
    int blocks;                          // that share a matrix
    float eps;
    const void* x;
    double* sums;                        // [count][blocks]
    __half* out;
    __nv_bfloat16* final;                // the result itself where there are no steps
};

template <typename T>
__device__ __forceinline__ float value_at(const NormParams& p, int64_t z, int64_t r, int64_t c) {
    return to_float(static_cast<const T*>(p.x)[z * p.step + r * p.row + c * p.col]);
}

// squares of a block's share of a matrix: rows blockIdx.x, + blocks, ...
template <typename T>
__global__ void __launch_bounds__(kNormThreads) k_squares(const NormParams p) {
    follow_on();
    const int64_t z = blockIdx.y;
    double sum = 0.0;
    for (int64_t r = blockIdx.x; r < p.rows; r += p.blocks)
        for (int64_t c = threadIdx.x; c < p.cols; c += kNormThreads) {
            const double v = value_at<T>(p, z, r, c);
            sum += v * v;
        }
    sum = warp_sum(sum);
    __shared__ double joined[kNormThreads / 32];
    if ((threadIdx.x & 31) == 0) joined[threadIdx.x >> 5] = sum;
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int i = 1; i < kNormThreads / 32; ++i) sum += joined[i];
        p.sums[z * p.blocks + blockIdx.x] = sum;
    }
}

template <typename T>
__global__ void __launch_bounds__(kNormThreads) k_scale(const NormParams p) {
    follow_on();
    const int64_t z = blockIdx.y;
    __shared__ double factor;
    if (threadIdx.x < 32) {
        double sum = 0.0;
        for (int i = threadIdx.x; i < p.blocks; i += 32) sum += p.sums[z * p.blocks + i];
        sum = warp_sum(sum);
        if (threadIdx.x == 0) factor = 1.0 / (sqrt(sum) + (double)p.eps);
    }
    __syncthreads();
    const double f = factor;
    for (int64_t r = blockIdx.x; r < p.rows; r += p.blocks)
        for (int64_t c = threadIdx.x; c < p.cols; c += kNormThreads) {
            const double v = value_at<T>(p, z, r, c) * f;
            if (p.final)
                p.final[(z * p.rows + r) * p.cols + c] = __float2bfloat16_rn((float)v);
            else
                p.out[z * p.out_step + r * p.ld + c] = __float2half_rn((float)(v * kScale));
        }
}

// ----------------------------------------------------------------------------- small matrices
// All steps of one matrix in a cluster of kCluster blocks. Each product's tiles of 128 x bn go round
// the blocks; X, A and B stay in scratch, that is in L2. Every block runs every cluster barrier
// whatever failed in it, so none waits for another that has left.
constexpr int kCluster = 8, kSmallEpi = 8, kSmallTma = 8, kSmallMma = 9;
constexpr int kSmallThreads = 32 * 10, kSmallStages = 5;
constexpr uint32_t kBox = 64 * kLineBytes;                     // 64 lines
constexpr uint32_t kSmallStage = 4 * kBox;                     // 128 x 64 of A, up to 128 x 64 of B
constexpr uint32_t kSmallBufs = kSmallEpi * 2 * kWarpBuf;

struct SmallProduct {
    int m, n, kblocks, bn, tiles;
    int symmetric;
};
struct SmallParams {
    CUtensorMap x[2], g, h;                     // boxes of 64 x 64: operands in either order
    CUtensorMap x_out[2], g_out, h_out, y_out;  // boxes of 32 x 32
    SmallProduct gram, poly, next;
    const __half* in_x[2];
    const __half* in_g;
    int64_t ld_x, step_x, ld_g, step_g;
    __nv_bfloat16* y;
    int rows, cols, steps, tall, tma_y;
    float a, b, c;
    unsigned* flag;
    unsigned polls;
};
struct SmallShared {
    unsigned long long full[kSmallStages], empty[kSmallStages], acc_full[2], acc_empty[2], drained;
    uint32_t tmem;
    int fail, issued;
};

__device__ __forceinline__ void bulk_store_done() {
    asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
}
// between what other threads wrote and this thread's copies of it, either way
__device__ __forceinline__ void fence_async_all() {
    asm volatile("fence.proxy.async;" ::: "memory");
}

// tile w of a product: rows mt * 128, columns nt * bn. Symmetric ones have the tiles that begin on or
// left of the diagonal: mt + 1 lots of 128 / bn in line mt.
__device__ __forceinline__ void small_tile(const SmallProduct& q, int w, int& mt, int& nt) {
    if (q.symmetric) {
        const int each = 128 / q.bn;
        mt = 0;
        while (w >= (mt + 1) * each) w -= (mt + 1) * each, ++mt;
        nt = w;
    } else {
        const int across = (q.n + q.bn - 1) / q.bn;
        mt = w / across, nt = w - mt * across;
    }
}

__global__ void __launch_bounds__(kSmallThreads, 1)
k_small(const __grid_constant__ SmallParams p) {
    using namespace tc;
    extern __shared__ __align__(1024) unsigned char smem[];
    unsigned char* bufs = smem + kSmallStages * kSmallStage;
    auto* sh = reinterpret_cast<SmallShared*>(bufs + kSmallBufs);
    const int tid = threadIdx.x, lane = tid & 31;
    const int warp = __shfl_sync(0xffffffffu, tid >> 5, 0);
    const int rank = (int)cluster_rank(), z = blockIdx.x / kCluster;
    if (tid == 0) {
        for (int i = 0; i < kSmallStages; ++i) {
            mbar_init(smem_u32(&sh->full[i]), 1);
            mbar_init(smem_u32(&sh->empty[i]), 1);
        }
        for (int i = 0; i < 2; ++i) {
            mbar_init(smem_u32(&sh->acc_full[i]), 1);
            mbar_init(smem_u32(&sh->acc_empty[i]), kSmallEpi);
        }
        mbar_init(smem_u32(&sh->drained), 1);
        sh->fail = 0;
        sh->issued = 0;
        asm volatile("fence.mbarrier_init.release.cluster;");
    }
    if (warp == kSmallMma) tmem_alloc(&sh->tmem, 256);
    fence_before_sync();
    __syncthreads();
    fence_after_sync();
    const uint32_t tmem = __shfl_sync(0xffffffffu, sh->tmem, 0);
    volatile int* fail = &sh->fail;
    follow_on();

    const bool one = elect_one();
    int st = 0, issued = 0, buf = 0;
    uint32_t parity = warp == kSmallTma ? 1 : 0;         // of the stage's next wait
    uint32_t acc_parity = warp == kSmallMma ? 1 : 0;     // of the accumulator's
    const Stage s0(smem_u32(bufs) + warp * 2 * kWarpBuf, lane);
    const Stage s1(smem_u32(bufs) + (warp * 2 + 1) * kWarpBuf, lane);

    for (int phase = 0; phase < 3 * p.steps; ++phase) {
        const int step = phase / 3, kind = phase - 3 * step;
        const bool last = phase + 1 == 3 * p.steps;
        const SmallProduct& q = kind == 0 ? p.gram : kind == 1 ? p.poly : p.next;
        const int from = step & 1;
        // gram: A and B are X; poly: A; next: B X, or X B of tall ones
        const bool a_mn = kind == 0 && p.tall, b_mn = kind == 0 ? p.tall : kind == 2 && !p.tall;
        if (warp == kSmallTma) {
            const CUtensorMap* x = &p.x[from];
            const CUtensorMap* am = kind == 0 ? x : kind == 1 ? &p.g : p.tall ? x : &p.h;
            const CUtensorMap* bm = kind == 0 ? x : kind == 1 ? &p.g : p.tall ? &p.h : x;
            fence_async_all();
            bool ok = !*fail;
            for (int w = rank; w < q.tiles && ok; w += kCluster) {
                int mt, nt;
                small_tile(q, w, mt, nt);
                for (int kb = 0; kb < q.kblocks; ++kb) {
                    ok = mbar_wait(smem_u32(&sh->empty[st]), parity, p.polls) && !*fail;
                    if (!__all_sync(0xffffffffu, ok)) {
                        ok = false;
                        break;
                    }
                    const uint32_t bar = smem_u32(&sh->full[st]);
                    const uint32_t a = smem_u32(smem) + (uint32_t)st * kSmallStage;
                    if (one) {
                        mbar_expect_tx(bar, (2 + q.bn / 64) * kBox);
                        for (int i = 0; i < 2 + q.bn / 64; ++i) {
                            const bool is_b = i >= 2;
                            const int line = is_b ? nt * q.bn + (i - 2) * 64 : mt * 128 + i * 64;
                            const bool mn = is_b ? b_mn : a_mn;
                            tma_load3(a + i * kBox, is_b ? bm : am, mn ? line : kb * 64,
                                      mn ? kb * 64 : line, z, bar);
                        }
                    }
                    __syncwarp();
                    ++issued;
                    if (++st == kSmallStages) st = 0, parity ^= 1;
                }
            }
            if (!ok && !*fail) *fail = 1;
            if (one) sh->issued = issued;
            __syncwarp();
        } else if (warp == kSmallMma) {
            const uint64_t step_a = a_mn ? 2048 >> 4 : 32 >> 4, step_b = b_mn ? 2048 >> 4 : 32 >> 4;
            const uint64_t desc_a = operand_desc(smem_u32(smem), a_mn);
            const uint64_t desc_b = operand_desc(smem_u32(smem) + 2 * kBox, b_mn);
            const uint32_t idesc = operand_idesc(0, a_mn, b_mn, 128, q.bn);
            bool ok = !*fail;
            for (int w = rank; w < q.tiles && ok; w += kCluster) {
                ok = mbar_wait(smem_u32(&sh->acc_empty[buf]), acc_parity, p.polls) && !*fail;
                if (!__all_sync(0xffffffffu, ok)) {
                    ok = false;
                    break;
                }
                fence_after_sync();
                const uint32_t acc = tmem + buf * 128;
                for (int kb = 0; kb < q.kblocks; ++kb) {
                    ok = mbar_wait(smem_u32(&sh->full[st]), parity, p.polls) && !*fail;
                    if (!__all_sync(0xffffffffu, ok)) {
                        ok = false;
                        break;
                    }
                    fence_after_sync();
                    const uint64_t at = (uint64_t)((uint32_t)st * (kSmallStage >> 4));
                    if (one) {
#pragma unroll
                        for (int k = 0; k < 4; ++k)
                            mma<false, false>(acc, desc_a + at + k * step_a,
                                              desc_b + at + k * step_b, idesc, kb > 0 || k > 0);
                        mma_commit(smem_u32(&sh->empty[st]));
                    }
                    __syncwarp();
                    if (++st == kSmallStages) st = 0, parity ^= 1;
                }
                if (one) mma_commit(smem_u32(&sh->acc_full[buf]));
                __syncwarp();
                buf ^= 1;
                if (buf == 0) acc_parity ^= 1;
            }
            if (!ok && !*fail) *fail = 2;
        } else {
            // sums are of scaled values, 2^20 of the products'; the last result leaves without scale
            const float unit = last ? 1.0f / kScale : 1.0f;
            const float alpha = kind == 0 ? 1.0f / kScale : kind == 1 ? p.c / kScale : unit / kScale;
            const float beta = kind == 1 ? p.b : p.a * unit;
            const CUtensorMap* out = kind == 0 ? &p.g_out : kind == 1 ? &p.h_out
                                     : last   ? &p.y_out : &p.x_out[from ^ 1];
            const __half* in = kind == 0 ? nullptr
                               : kind == 1 ? p.in_g + z * p.step_g : p.in_x[from] + z * p.step_x;
            const int64_t ld = kind == 1 ? p.ld_g : p.ld_x;
            const bool tma = !last || p.tma_y;
            const int quarter = warp & 3, share = warp >> 2;
            bool ok = !*fail;
            for (int w = rank; w < q.tiles && ok; w += kCluster) {
                int mt, nt;
                small_tile(q, w, mt, nt);
                const int row0 = mt * 128 + quarter * 32, rows = max(0, min(32, q.m - row0));
                const uint32_t acc = tmem + buf * 128 + ((uint32_t)(quarter * 32) << 16);
                const bool mirror = q.symmetric && nt * q.bn + q.bn <= mt * 128;
                for (int c = share * 32; c < q.bn; c += 64) {
                    const int col = nt * q.bn + c;
                    if (lane == 0) bulk_store_read();
                    __syncwarp();
                    if (in) {
                        // past L1, which may hold these lines as they were a step before
                        const int r0 = lane >> 2, cc = (lane & 3) * 8;
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            uint4 v = make_uint4(0, 0, 0, 0);
                            if (r0 + 8 * i < rows && col + cc < q.n)
                                v = __ldcg(reinterpret_cast<const uint4*>(
                                    in + (int64_t)(row0 + r0 + 8 * i) * ld + col + cc));
                            put16(s0.turn(i), v);
                        }
                        __syncwarp();
                    }
                    if (c == share * 32) {
                        ok = mbar_wait(smem_u32(&sh->acc_full[buf]), acc_parity, p.polls) && !*fail;
                        ok = __all_sync(0xffffffffu, ok);
                        if (!ok) break;
                        fence_after_sync();
                    }
#pragma unroll
                    for (int half = 0; half < 2; ++half) {
                        float v[16];
                        Two t[8], u[8];
                        tmem_ld16(acc + c + half * 16, v);
                        if (in) get_row<__half>(s0, half, u);
#pragma unroll
                        for (int j = 0; j < 8; ++j) {
                            t[j] = two(v[2 * j], v[2 * j + 1]) * two(alpha);
                            if (in) t[j] = fma(u[j], two(beta), t[j]);
                        }
                        if (mirror) put_column<__half>(s1, half, t);
                        if (last) put_row<__nv_bfloat16>(s0, half, t);
                        else put_row<__half>(s0, half, t);
                    }
                    if (tma) fence_async_smem();
                    __syncwarp();
                    if (tma) {
                        if (lane == 0 && rows > 0 && col < q.n) {
                            bulk_store3(out, s0.base, col, row0, z);
                            if (mirror) bulk_store3(out, s1.base, row0, col, z);
                            bulk_store_commit();
                        }
                    } else {
                        store_rows<__nv_bfloat16>(
                            s0, p.y + ((int64_t)z * p.rows + row0) * p.cols + col, p.cols, rows,
                            q.n - col);
                    }
                    __syncwarp();
                }
                if (!ok) break;
                fence_before_sync();
                __syncwarp();
                if (lane == 0) mbar_arrive(smem_u32(&sh->acc_empty[buf]));
                __syncwarp();
                buf ^= 1;
                if (buf == 0) acc_parity ^= 1;
            }
            if (!ok && !*fail) *fail = 4;
            if (lane == 0) {  // the results are in L2
                bulk_store_done();
                fence_async_all();
            }
        }
        __syncwarp();
        cluster_sync();
    }
    // what is in flight after a wait that gave up lands before the block's memory goes
    __syncthreads();
    if (*fail) {
        if (tid == 0) {
            atomicExch_system(p.flag, (unsigned)*fail);
            for (int i = max(0, sh->issued - kSmallStages); i < sh->issued; ++i)
                mbar_wait(smem_u32(&sh->full[i % kSmallStages]), (i / kSmallStages) & 1);
        }
        __syncwarp();
        if (warp == kSmallMma) {
            if (one) mma_commit(smem_u32(&sh->drained));
            __syncwarp();
            mbar_wait(smem_u32(&sh->drained), 0);
        }
        __syncwarp();
    }
    fence_before_sync();
    __syncthreads();
    if (warp == kSmallMma) {
        fence_after_sync();
        tmem_dealloc(tmem, 256);
    }
}

// A stack of matrices in scratch or of results.
struct Stack {
    void* p;
    int64_t rows, cols, ld, step;
    Matrix matrix() const { return {p, rows, cols, ld}; }
    CUtensorMap map(int64_t count, int box) const {
        return make_map3(matrix(), count, step, 2, box);
    }
};

struct Step {
    Stack a, b, out;
    bool a_mn, b_mn, symmetric, bf16;  // bf16: type of the result
    const Stack* in;                   // beta in, or null
    float alpha, beta;
    int64_t k, count;
    int device;
};

template <typename T>
void run_step(const Step& s, cudaStream_t stream) {
    const int sms = sm_count(s.device);
    const uint32_t fixed = kFixedSmem<kUpdate>;
    const int64_t m = s.out.rows, n = s.out.cols;
    const int kblocks = (int)((s.k + 63) / 64);
    // square tiles of a symmetric product; else the cheapest by the time of the tiles
    Plan plan{};
    double best = 0.0;
    for (int pair = 1; pair >= 0; --pair)
        for (int bn : {256, 128, 64}) {
            if (pair && bn == 64) continue;
            const int high = pair ? 2 * kBM : kBM, units = pair ? sms / 2 : sms;
            if (s.symmetric && bn != high) continue;
            const int64_t tm = (m + high - 1) / high, tn = (n + bn - 1) / bn;
            const int64_t tiles = (s.symmetric ? tm * (tm + 1) / 2 : tm * tn) * s.count;
            const double main = kblocks * block_cycles(pair, bn);
            const double epi = 1000.0 + (s.symmetric ? 24.0 : 16.0) * bn;
            const double cost =
                (double)((tiles + units - 1) / units) * std::max(main, epi) + std::min(main, epi);
            if (plan.bn == 0 || cost < best) {
                best = cost;
                plan = {bn, 1, kblocks, ring_stages(pair, bn, fixed), pair == 1};
            }
        }
    const int high = plan.pair ? 2 * kBM : kBM;
    TileParams p{};
    p.m = m, p.n = n;
    p.act = RUNE_ACT_NONE;
    p.kblocks = p.kb_per_split = kblocks, p.splits = 1;
    p.bn = plan.bn, p.stages = plan.stages;
    p.tiles_m = (int)((m + high - 1) / high), p.tiles_n = (int)((n + p.bn - 1) / p.bn);
    p.by_tiles = make_divisor((unsigned)p.tiles_m * p.tiles_n);
    p.by_group = make_divisor(kGroup * (unsigned)p.tiles_n);
    p.by_last = make_divisor(std::max(1u, (unsigned)p.tiles_m % kGroup));
    p.a_mn = s.a_mn, p.b_mn = s.b_mn;
    p.idesc = operand_idesc(0, s.a_mn, s.b_mn, high, p.bn);
    p.groups = (int)s.count;
    p.symmetric = s.symmetric;
    p.alpha = s.alpha, p.beta = s.beta;
    p.out = s.out.p, p.ld_out = s.out.ld, p.out_step = s.out.step;
    p.tma_out = wide16(s.out.p, s.out.ld, s.out.ld) && s.out.step % 8 == 0;
    if (s.in) {
        p.in = s.in->p, p.ld_in = s.in->ld, p.in_step = s.in->step;
        p.vec_in = 1;  // lines are padded to 16 bytes
    }
    p.flag = wait_flag(s.device);
    p.polls = wait_polls();
    const CUtensorMap a = s.a.map(s.count, s.a_mn ? 64 : kBM);
    const CUtensorMap b = s.b.map(s.count, s.b_mn ? 64 : plan.pair ? p.bn / 2 : p.bn);
    const CUtensorMap o =
        p.tma_out ? make_out_map3(s.out.p, m, n, s.out.ld, s.count, s.out.step) : a;
    const int64_t work = (s.symmetric ? (int64_t)p.tiles_m * (p.tiles_m + 1) / 2
                                      : (int64_t)p.tiles_m * p.tiles_n) * s.count;
    require(work < (1LL << 31) - 1024, "too many tiles");
    if (plan.pair)
        launch_blocks<kUpdate, kBatch, T, false, true>(a, b, o, o, p, work, fixed, sms, s.device,
                                                       stream);
    else
        launch_blocks<kUpdate, kBatch, T, false, false>(a, b, o, o, p, work, fixed, sms, s.device,
                                                        stream);
}

// The products of a matrix of rows x cols in tiles of 128 x 64 or 128 x 128, whichever takes the
// blocks of a cluster less time, and the cycles that a step takes.
struct SmallPlan {
    SmallProduct gram, poly, next;
    double cycles;
};
SmallPlan plan_small(int64_t rows, int64_t cols) {
    SmallPlan plan{};
    const int64_t small = std::min(rows, cols), large = std::max(rows, cols);
    auto product = [&](int64_t m, int64_t n, int64_t k, bool symmetric) {
        SmallProduct best{};
        double best_cost = 0.0;
        for (int bn : {128, 64}) {
            const int64_t tm = (m + 127) / 128, tn = (n + bn - 1) / bn;
            const int64_t tiles = symmetric ? tm * (tm + 1) / 2 * (128 / bn) : tm * tn;
            const int kblocks = (int)((k + 63) / 64);
            const double main = kblocks * block_cycles(false, bn), epi = 600.0 + 16.0 * bn;
            const double turns = (double)((tiles + kCluster - 1) / kCluster);
            const double cost = 3000.0 + turns * std::max(main, epi) + std::min(main, epi);
            if (best.bn == 0 || cost < best_cost) {
                best_cost = cost;
                best = {(int)m, (int)n, kblocks, bn, (int)tiles, symmetric};
            }
        }
        plan.cycles += best_cost;
        return best;
    };
    plan.gram = product(small, small, large, true);
    plan.poly = product(small, small, small, true);
    plan.next = product(rows, cols, small, false);
    return plan;
}

void run_small(const rune_orthogonalize_args& a, const SmallPlan& plan, const Stack (&x)[2],
               const Stack& g, const Stack& h, cudaStream_t stream) {
    SmallParams p{};
    const Stack y{a.y, a.rows, a.cols, a.cols, a.rows * a.cols};
    auto out = [&](const Stack& t) {
        return make_out_map3(t.p, t.rows, t.cols, t.ld, a.count, t.step);
    };
    for (int i = 0; i < 2; ++i) {
        const Stack& t = a.steps > 1 ? x[i] : x[0];
        p.x[i] = t.map(a.count, 64), p.x_out[i] = out(t);
        p.in_x[i] = static_cast<const __half*>(t.p);
    }
    p.g = g.map(a.count, 64), p.g_out = out(g);
    p.h = h.map(a.count, 64), p.h_out = out(h);
    p.tma_y = wide16(a.y, a.cols, a.cols);
    p.y_out = p.tma_y ? out(y) : p.g_out;
    p.gram = plan.gram, p.poly = plan.poly, p.next = plan.next;
    p.in_g = static_cast<const __half*>(g.p);
    p.ld_x = x[0].ld, p.step_x = x[0].step, p.ld_g = g.ld, p.step_g = g.step;
    p.y = static_cast<__nv_bfloat16*>(a.y);
    p.rows = (int)a.rows, p.cols = (int)a.cols;
    p.steps = a.steps, p.tall = a.rows > a.cols;
    p.a = a.a, p.b = a.b, p.c = a.c;
    p.flag = wait_flag(a.device);
    p.polls = wait_polls();
    const size_t smem = kSmallStages * kSmallStage + kSmallBufs + sizeof(SmallShared);
    static std::atomic<uint64_t> allowed{0};  // devices whose limit is raised
    if (a.device >= 64 || !(allowed.load(std::memory_order_relaxed) >> a.device & 1)) {
        RUNE_CUDA_TRY(cudaFuncSetAttribute(k_small, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                           (int)smem));
        if (a.device < 64) allowed.fetch_or(uint64_t(1) << a.device, std::memory_order_relaxed);
    }
    launch(k_small, (unsigned)(a.count * kCluster), kSmallThreads, smem, kCluster, stream, p);
}

// Whether the clusters take less time than a chain of launches, of 10000 cycles a product at least
// and then at the tensor cores' rate of all SMs.
bool use_small(const rune_orthogonalize_args& a, const SmallPlan& plan) {
    const int64_t small = std::min(a.rows, a.cols), large = std::max(a.rows, a.cols);
    if (a.steps == 0 || large > (1 << 20) || a.count > (1 << 16)) return false;
    const int sms = sm_count(a.device);
    // clusters at once: blocks of one lie in one group of SMs, so not all SMs find a place
    const double waves = std::ceil((double)a.count * kCluster / (sms * 0.85));
    const double kb = (double)a.count * ((small + 127) / 128) * ((large + 63) / 64) / sms;
    const double chain = 3.0 * std::max(10000.0, 3000.0 + kb * ((small + 127) / 128) * 350.0);
    return waves * plan.cycles < chain;
}

int norm_blocks(const rune_orthogonalize_args& a) {
    const int64_t most = std::max<int64_t>(1, (int64_t)sm_count(a.device) * 8 / a.count);
    return (int)std::min<int64_t>(a.rows, most);
}

void orthogonalize(const rune_orthogonalize_args& a, Scratch& ws, cudaStream_t stream) {
    const bool tall = a.rows > a.cols;
    const int64_t small = tall ? a.cols : a.rows;
    const int64_t ld = pad16(a.cols, 2), lds = pad16(small, 2);
    NormParams n{};
    n.rows = a.rows, n.cols = a.cols;
    n.step = a.x_step, n.row = a.x_row, n.col = a.x_col;
    n.ld = ld, n.out_step = a.rows * ld;
    n.blocks = norm_blocks(a);
    n.eps = a.eps;
    n.x = a.x;
    n.sums = ws.take<double>(a.count * n.blocks);
    Stack x[2], g{}, h{};
    if (a.steps > 0) {
        for (int i = 0; i < (a.steps > 1 ? 2 : 1); ++i)
            x[i] = {ws.take<__half>(a.count * a.rows * ld), a.rows, a.cols, ld, a.rows * ld};
        g = {ws.take<__half>(a.count * small * lds), small, small, lds, small * lds};
        h = {ws.take<__half>(a.count * small * lds), small, small, lds, small * lds};
    }
    if (ws.sizing()) return;
    n.out = static_cast<__half*>(x[0].p);
    n.final = a.steps == 0 ? static_cast<__nv_bfloat16*>(a.y) : nullptr;
    const dim3 grid((unsigned)n.blocks, (unsigned)a.count);
    const SmallPlan plan = plan_small(a.rows, a.cols);
    auto prepare = [&](auto t) {
        using T = decltype(t);
        launch(k_squares<T>, grid, kNormThreads, 0, 0, stream, n);
        launch(k_scale<T>, grid, kNormThreads, 0, 0, stream, n);
    };
    if (a.dtype == RUNE_F16) prepare(__half());
    else if (a.dtype == RUNE_BF16) prepare(__nv_bfloat16());
    else prepare(float());
    if (use_small(a, plan)) {
        run_small(a, plan, x, g, h, stream);
        return;
    }
    for (int i = 0; i < a.steps; ++i) {
        const Stack from = x[i & 1];
        const bool last = i + 1 == a.steps;
        const Stack to = last ? Stack{a.y, a.rows, a.cols, a.cols, a.rows * a.cols}
                              : x[(i + 1) & 1];
        // sums are of scaled values: 2^20 of the products'
        const Step gram{from, from, g, tall, tall, true, false, nullptr, 1.0f / kScale, 0.0f,
                        tall ? a.rows : a.cols, a.count, a.device};
        run_step<__half>(gram, stream);
        const Step poly{g, g, h, false, false, true, false, &g, a.c / kScale, a.b, small, a.count,
                        a.device};
        run_step<__half>(poly, stream);
        // the last one leaves without the scale
        const float unit = last ? 1.0f / kScale : 1.0f;
        Step next{tall ? from : h, tall ? h : from, to, false, !tall, false, last, &from,
                  unit / kScale, a.a * unit, small, a.count, a.device};
        if (last) run_step<__nv_bfloat16>(next, stream);
        else run_step<__half>(next, stream);
    }
}

void check_args(const rune_orthogonalize_args& a) {
    constexpr int64_t most = INT32_MAX / 4;
    require(a.count >= 0 && a.count <= 65535, "count out of range: 0 to 65535");
    require(a.rows >= 0 && a.rows <= most && a.cols >= 0 && a.cols <= most,
            "rows or columns out of range");
    require(a.dtype == RUNE_F32 || a.dtype == RUNE_F16 || a.dtype == RUNE_BF16,
            "x is float32, float16 or bfloat16");
    require(a.steps >= 0 && a.steps <= 64, "steps out of range: 0 to 64");
    require(a.eps >= 0.0f, "eps cannot be negative");
    require(a.count * a.rows * a.cols == 0 || (a.x && a.y), "null argument");
    require_aligned({a.x}, dtype_bytes(a.dtype));
    require_aligned({a.y}, 2);
}

}  // namespace
}  // namespace ops
}  // namespace rune

using namespace rune;
using namespace rune::ops;

extern "C" {

int rune_orthogonalize_workspace(const rune_orthogonalize_args* args, int64_t* bytes) {
    if (!args || !bytes) {
        set_error("null argument");
        return RUNE_ERR_INVALID;
    }
    const rune_orthogonalize_args a = *args;
    return guarded(a.device, [&] {
        check_args(a);
        Scratch ws{nullptr};
        if (a.count > 0 && a.rows > 0 && a.cols > 0) orthogonalize(a, ws, nullptr);
        *bytes = ws.off;
    });
}

int rune_orthogonalize(const rune_orthogonalize_args* args, void* stream_) {
    if (!args) {
        set_error("null argument");
        return RUNE_ERR_INVALID;
    }
    const rune_orthogonalize_args a = *args;
    auto stream = static_cast<cudaStream_t>(stream_);
    return guarded(a.device, [&] {
        check_args(a);
        check_waits(a.device);
        if (a.count == 0 || a.rows == 0 || a.cols == 0) return;
        Scratch need{nullptr};
        orthogonalize(a, need, stream);
        require(a.workspace && aligned(a.workspace, 256) && a.workspace_bytes >= need.off,
                "the workspace is too small or not 256-byte aligned");
        Scratch ws{static_cast<char*>(a.workspace)};
        orthogonalize(a, ws, stream);
        RUNE_LAUNCH_CHECK();
    });
}

}  // extern "C"
