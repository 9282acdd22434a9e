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
// 8 x 256 x 512, five steps, 96 us as a chain of launches, 75 us so.

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

// fn(r, c, values of columns c, c + 32, ...) for a lane's part of the rows `row`, + every, ... of which
// a warp has each: enough under way at once
constexpr int kAhead = 8;
template <typename T, typename Fn>
__device__ __forceinline__ void values_of(const NormParams& p, int64_t z, int64_t row, int64_t every,
                                          Fn&& fn) {
    for (int64_t r = row; r < p.rows; r += every)
        for (int64_t c = threadIdx.x & 31; c < p.cols; c += 32 * kAhead) {
            float v[kAhead];
#pragma unroll
            for (int i = 0; i < kAhead; ++i)
                v[i] = c + 32 * i < p.cols ? value_at<T>(p, z, r, c + 32 * i) : 0.0f;
            fn(r, c, v);
        }
}

// sum of a few squares, in float64 where float32 would leave its range
__device__ __forceinline__ double squares(const float (&v)[kAhead]) {
    float s = 0.0f;
#pragma unroll
    for (int i = 0; i < kAhead; ++i) s = fmaf(v[i], v[i], s);
    if (s > 1.0e-25f && s < 1.0e35f) return s;
    double d = 0.0;
#pragma unroll
    for (int i = 0; i < kAhead; ++i) d += (double)v[i] * v[i];
    return d;
}

// v f for any float64 f > 0 in three float32 products, of which the outer ones are exact: a power of
// two, f's fraction, and the rest of the power (float64 products of all values took as long as reading
// them three times)
struct Factor {
    float first, fraction, last;
    __device__ __forceinline__ explicit Factor(double f) {
        int e = 0;
        fraction = (float)frexp(f, &e);
        e = max(-250, min(250, e));
        first = exp2f((float)(e / 2)), last = exp2f((float)(e - e / 2));
    }
    __device__ __forceinline__ float times(float v) const { return v * first * fraction * last; }
};

// squares of a block's share of a matrix
template <typename T>
__global__ void __launch_bounds__(kNormThreads) k_squares(const NormParams p) {
    follow_on();
    const int64_t z = blockIdx.y;
    double sum = 0.0;
    constexpr int kWarps = kNormThreads / 32;
    values_of<T>(p, z, blockIdx.x * kWarps + (threadIdx.x >> 5), p.blocks * kWarps,
                 [&](int64_t, int64_t, const float(&v)[kAhead]) { sum += squares(v); });
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
    const Factor f(p.final ? factor : factor * kScale);
    constexpr int kWarps = kNormThreads / 32;
    values_of<T>(p, z, blockIdx.x * kWarps + (threadIdx.x >> 5), p.blocks * kWarps,
                 [&](int64_t r, int64_t c, const float(&v)[kAhead]) {
#pragma unroll
                     for (int i = 0; i < kAhead; ++i) {
                         const int64_t at = c + 32 * i;
                         if (at >= p.cols) break;
                         const float x = f.times(v[i]);
                         if (p.final)
                             p.final[(z * p.rows + r) * p.cols + at] = __float2bfloat16_rn(x);
                         else
                             p.out[z * p.out_step + r * p.ld + at] = __float2half_rn(x);
                     }
                 });
}

// ----------------------------------------------------------------------------- small matrices
// All steps of one matrix in a cluster of kCluster blocks. Each product's tiles of 128 x bn go round
// the blocks; X, A and B stay in scratch, that is in L2. With a tile or two a block there is nothing
// to gain from symmetry, and the lanes write their rows' values themselves: what counts is the time
// from one product's last value to the next one's first. Every block runs every cluster barrier
// whatever failed in it, so none waits for another that has left.
// 8 x 256 x 512: 7800 to 9000 cycles a product, of which 2300 pass before the first copies land, 450
// are a k-block's (an SM's share of L2 for 24 to 32 KB), 1500 the epilogue's and 1000 the barrier's.
constexpr int kCluster = 8, kSmallStages = 6;
constexpr uint32_t kBox = 64 * kLineBytes;                     // 64 lines
constexpr uint32_t kSmallStage = 4 * kBox;                     // 128 x 64 of A, up to 128 x 64 of B

struct SmallProduct {
    int m, n, kblocks, bn, tiles;
};
struct SmallParams {
    CUtensorMap map_x[2], map_g, map_h;  // boxes of 64 x 64: operands in either order
    SmallProduct gram, poly, next;
    __half *x[2], *g, *h;
    int64_t ld_x, step_x, ld_g, step_g;
    NormParams norm;                     // of the matrices as they come
    __nv_bfloat16* y;
    int rows, cols, steps, tall, wide_y;
    float a, b, c;
    unsigned* flag;
    unsigned polls;
};
struct SmallShared {
    unsigned long long full[kSmallStages], empty[kSmallStages], acc_full[2], acc_empty[2], drained;
    uint32_t tmem;
    int fail, issued;
    double squares[kEpiWarps + 3];  // of the warps, and the block's
};

__device__ __forceinline__ double peer_double(uint32_t addr) {
    double v;
    asm volatile("ld.shared::cluster.f64 %0, [%1];" : "=d"(v) : "r"(addr));
    return v;
}
// between accesses to global memory by threads and by copies
__device__ __forceinline__ void fence_async_global() {
    asm volatile("fence.proxy.async.global;" ::: "memory");
}

// tile w of a product: rows mt * 128, columns nt * bn
__device__ __forceinline__ void small_tile(const SmallProduct& q, int w, int& mt, int& nt) {
    const int across = (q.n + q.bn - 1) / q.bn;
    mt = w / across, nt = w - mt * across;
}

template <typename T>
__global__ void __launch_bounds__(kThreads, 1) k_small(const __grid_constant__ SmallParams p) {
    using namespace tc;
    extern __shared__ __align__(1024) unsigned char smem[];
    auto* sh = reinterpret_cast<SmallShared*>(smem + kSmallStages * kSmallStage);
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
            mbar_init(smem_u32(&sh->acc_empty[i]), kEpiWarps);
        }
        mbar_init(smem_u32(&sh->drained), 1);
        sh->fail = 0;
        sh->issued = 0;
        asm volatile("fence.mbarrier_init.release.cluster;");
    }
    if (warp == kMmaWarp) tmem_alloc(&sh->tmem, 256);
    if (warp == kTmaWarp && lane < 4) prefetch_map(&p.map_x[0] + lane);  // all of them
    fence_before_sync();
    __syncthreads();
    fence_after_sync();
    const uint32_t tmem = __shfl_sync(0xffffffffu, sh->tmem, 0);
    volatile int* fail = &sh->fail;
    follow_on();

    // X = x / (|x|_F + eps): a row a warp, every kCluster-th block's; the rows come again from L2
    {
        const NormParams& n = p.norm;
        const int first = rank * kThreads / 32 + warp, every = kCluster * kThreads / 32;
        double sum = 0.0;
        values_of<T>(n, z, first, every,
                     [&](int64_t, int64_t, const float(&v)[kAhead]) { sum += squares(v); });
        sum = warp_sum(sum);
        if (lane == 0) sh->squares[warp] = sum;
        __syncthreads();
        if (tid == 0) {
            sum = 0.0;
            for (int i = 0; i < kThreads / 32; ++i) sum += sh->squares[i];
            sh->squares[kThreads / 32] = sum;
        }
        __syncthreads();
        cluster_sync();
        sum = 0.0;
        for (int i = 0; i < kCluster; ++i)
            sum += peer_double(peer_address(smem_u32(&sh->squares[kThreads / 32]), i));
        const Factor f(kScale / (sqrt(sum) + (double)n.eps));
        values_of<T>(n, z, first, every, [&](int64_t r, int64_t c, const float(&v)[kAhead]) {
            __half* to = p.x[0] + z * p.step_x + r * p.ld_x;
#pragma unroll
            for (int i = 0; i < kAhead; ++i)
                if (c + 32 * i < p.cols) to[c + 32 * i] = __float2half_rn(f.times(v[i]));
        });
        fence_async_global();
        __syncwarp();
        cluster_sync();
    }

    const bool one = elect_one();
    int st = 0, issued = 0, buf = 0;
    uint32_t parity = warp == kTmaWarp ? 1 : 0;         // of the stage's next wait
    uint32_t acc_parity = warp == kMmaWarp ? 1 : 0;     // of the accumulator's

    // `boxes` of a stage from its box `at` on: 64 lines each from `line` on, k-block kb
    auto load = [&](int line, int boxes, const CUtensorMap* map, bool mn, int stage, int at,
                    int kb) {
        const uint32_t to = smem_u32(smem) + (uint32_t)stage * kSmallStage + at * kBox;
        for (int i = 0; i < boxes; ++i)
            tma_load3(to + i * kBox, map, mn ? line + i * 64 : kb * 64,
                      mn ? kb * 64 : line + i * 64, z, smem_u32(&sh->full[stage]));
    };

    for (int phase = 0; phase < 3 * p.steps; ++phase) {
        const int step = phase / 3, kind = phase - 3 * step;
        const bool last = phase + 1 == 3 * p.steps;
        const SmallProduct& q = kind == 0 ? p.gram : kind == 1 ? p.poly : p.next;
        const int from = step & 1;
        // gram: A and B are X; poly: A; next: B X, or X B of tall ones
        const bool a_mn = kind == 0 && p.tall, b_mn = kind == 0 ? p.tall : kind == 2 && !p.tall;
        if (warp == kTmaWarp) {
            const CUtensorMap* x = &p.map_x[from];
            const CUtensorMap* am = kind == 0 ? x : kind == 1 ? &p.map_g : p.tall ? x : &p.map_h;
            const CUtensorMap* bm = kind == 0 ? x : kind == 1 ? &p.map_g : p.tall ? &p.map_h : x;
            fence_async_global();
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
                    if (one) {
                        mbar_expect_tx(smem_u32(&sh->full[st]), (2 + q.bn / 64) * kBox);
                        load(mt * 128, 2, am, a_mn, st, 0, kb);
                        load(nt * q.bn, q.bn / 64, bm, b_mn, st, 2, kb);
                    }
                    __syncwarp();
                    ++issued;
                    if (++st == kSmallStages) st = 0, parity ^= 1;
                }
            }
            if (!ok && !*fail) *fail = 1;
            if (one) sh->issued = issued;
            __syncwarp();
        } else if (warp == kMmaWarp) {
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
            const __half* in = kind == 0 ? nullptr
                               : kind == 1 ? p.g + z * p.step_g : p.x[from] + z * p.step_x;
            const int64_t ld_in = kind == 1 ? p.ld_g : p.ld_x;
            __half* out = kind == 0 ? p.g + z * p.step_g
                          : kind == 1 ? p.h + z * p.step_g : p.x[from ^ 1] + z * p.step_x;
            const int64_t ld_out = kind < 2 ? p.ld_g : p.ld_x;
            const int quarter = warp & 3, share = warp >> 2;
            bool ok = !*fail;
            for (int w = rank; w < q.tiles && ok; w += kCluster) {
                int mt, nt;
                small_tile(q, w, mt, nt);
                const int row = mt * 128 + quarter * 32 + lane;
                const uint32_t acc = tmem + buf * 128 + ((uint32_t)(quarter * 32) << 16);
                // the lane's 16 values in two pieces of 16 bytes; lines are padded to these
                auto pieces = [&](int col, auto&& fn) {
#pragma unroll
                    for (int i = 0; i < 2; ++i)
                        if (row < q.m && col + 8 * i < q.n) fn(i, col + 8 * i);
                };
                uint4 given[2][2] = {};
#pragma unroll
                for (int t = 0; t < 2; ++t)
                    if (in && share * 16 + t * 64 < q.bn)
                        pieces(nt * q.bn + share * 16 + t * 64, [&](int i, int col) {
                            // past L1, which may hold these lines as they were a step before
                            given[t][i] =
                                __ldcg(reinterpret_cast<const uint4*>(in + row * ld_in + col));
                        });
                ok = mbar_wait(smem_u32(&sh->acc_full[buf]), acc_parity, p.polls) && !*fail;
                ok = __all_sync(0xffffffffu, ok);
                if (!ok) break;
                fence_after_sync();
#pragma unroll
                for (int t = 0; t < 2; ++t) {
                    const int c = share * 16 + t * 64, col0 = nt * q.bn + c;
                    if (c >= q.bn) break;
                    float v[16];
                    tmem_ld16(acc + c, v);
#pragma unroll
                    for (int j = 0; j < 16; ++j) v[j] *= alpha;
                    if (in) {
#pragma unroll
                        for (int j = 0; j < 8; ++j) {
                            const uint4& g = given[t][j / 4];
                            const uint32_t word = j % 4 == 0 ? g.x : j % 4 == 1 ? g.y
                                                  : j % 4 == 2 ? g.z : g.w;
                            const float2 f = unpack2<__half>(word);
                            v[2 * j] = fmaf(f.x, beta, v[2 * j]);
                            v[2 * j + 1] = fmaf(f.y, beta, v[2 * j + 1]);
                        }
                    }
                    auto packed = [&](auto type, int i) {
                        using O = decltype(type);
                        const float* f = v + 8 * i;
                        return make_uint4(pack2<O>(f[0], f[1]), pack2<O>(f[2], f[3]),
                                          pack2<O>(f[4], f[5]), pack2<O>(f[6], f[7]));
                    };
                    if (!last) {
                        pieces(col0, [&](int i, int col) {
                            *reinterpret_cast<uint4*>(out + row * ld_out + col) =
                                packed(__half(), i);
                        });
                    } else {
                        __nv_bfloat16* to = p.y + ((int64_t)z * p.rows + row) * p.cols;
                        if (p.wide_y) {
                            pieces(col0, [&](int i, int col) {
                                *reinterpret_cast<uint4*>(to + col) = packed(__nv_bfloat16(), i);
                            });
                        } else if (row < q.m) {
#pragma unroll
                            for (int j = 0; j < 16; ++j)
                                if (col0 + j < q.n) to[col0 + j] = __float2bfloat16_rn(v[j]);
                        }
                    }
                }
                fence_before_sync();
                __syncwarp();
                if (lane == 0) mbar_arrive(smem_u32(&sh->acc_empty[buf]));
                __syncwarp();
                buf ^= 1;
                if (buf == 0) acc_parity ^= 1;
            }
            if (!ok && !*fail) *fail = 4;
            fence_async_global();  // copies will read what was written
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
        if (warp == kMmaWarp) {
            if (one) mma_commit(smem_u32(&sh->drained));
            __syncwarp();
            mbar_wait(smem_u32(&sh->drained), 0);
        }
        __syncwarp();
    }
    fence_before_sync();
    __syncthreads();
    if (warp == kMmaWarp) {
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
// blocks of a cluster less time, and the cycles that a step takes (the figures beside k_small).
struct SmallPlan {
    SmallProduct gram, poly, next;
    double cycles;
};
SmallPlan plan_small(int64_t rows, int64_t cols) {
    SmallPlan plan{};
    const int64_t small = std::min(rows, cols), large = std::max(rows, cols);
    auto product = [&](int64_t m, int64_t n, int64_t k) {
        SmallProduct best{};
        double best_cost = 0.0;
        for (int bn : {128, 64}) {
            const int64_t tm = (m + 127) / 128, tn = (n + bn - 1) / bn;
            const int kblocks = (int)((k + 63) / 64);
            const double turns = (double)((tm * tn + kCluster - 1) / kCluster);
            const double cost = 6800.0 + (turns - 1.0) * 1500.0 +
                                turns * kblocks * (bn == 64 ? 250.0 : 500.0);
            if (best.bn == 0 || cost < best_cost) {
                best_cost = cost;
                best = {(int)m, (int)n, kblocks, bn, (int)(tm * tn)};
            }
        }
        plan.cycles += best_cost;
        return best;
    };
    plan.gram = product(small, small, large);
    plan.poly = product(small, small, small);
    plan.next = product(rows, cols, small);
    return plan;
}

void run_small(const rune_orthogonalize_args& a, const SmallPlan& plan, const Stack (&x)[2],
               const Stack& g, const Stack& h, const NormParams& norm, cudaStream_t stream) {
    SmallParams p{};
    p.norm = norm;
    for (int i = 0; i < 2; ++i) {
        const Stack& t = a.steps > 1 ? x[i] : x[0];
        p.map_x[i] = t.map(a.count, 64);
        p.x[i] = static_cast<__half*>(t.p);
    }
    p.map_g = g.map(a.count, 64), p.g = static_cast<__half*>(g.p);
    p.map_h = h.map(a.count, 64), p.h = static_cast<__half*>(h.p);
    p.wide_y = wide16(a.y, a.cols, a.cols);
    p.gram = plan.gram, p.poly = plan.poly, p.next = plan.next;
    p.ld_x = x[0].ld, p.step_x = x[0].step, p.ld_g = g.ld, p.step_g = g.step;
    p.y = static_cast<__nv_bfloat16*>(a.y);
    p.rows = (int)a.rows, p.cols = (int)a.cols;
    p.steps = a.steps, p.tall = a.rows > a.cols;
    p.a = a.a, p.b = a.b, p.c = a.c;
    p.flag = wait_flag(a.device);
    p.polls = wait_polls();
    const size_t smem = kSmallStages * kSmallStage + sizeof(SmallShared);
    auto typed = [&](auto t) {
        using T = decltype(t);
        static std::atomic<uint64_t> allowed{0};  // devices whose limit is raised
        if (a.device >= 64 || !(allowed.load(std::memory_order_relaxed) >> a.device & 1)) {
            RUNE_CUDA_TRY(cudaFuncSetAttribute(
                k_small<T>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
            if (a.device < 64) allowed.fetch_or(uint64_t(1) << a.device, std::memory_order_relaxed);
        }
        launch(k_small<T>, (unsigned)(a.count * kCluster), kThreads, smem, kCluster, stream, p);
    };
    if (a.dtype == RUNE_F16) typed(__half());
    else if (a.dtype == RUNE_BF16) typed(__nv_bfloat16());
    else typed(float());
}

// Whether the clusters take less time than a chain of launches, of 11500 cycles a product at least
// and then at the tensor cores' rate of all SMs. B200, five steps, clusters / chain, us: 1 x 256 x 256
// 59 / 80, 15 x 256 x 512 76 / 113, 12 x 128 x 1024 78 / 97; 16 x 256 x 512, in two waves, 150 / 110.
bool use_small(const rune_orthogonalize_args& a, const SmallPlan& plan) {
    const int64_t small = std::min(a.rows, a.cols), large = std::max(a.rows, a.cols);
    if (a.steps == 0 || large > (1 << 20) || a.count > (1 << 16)) return false;
    const int sms = sm_count(a.device);
    // clusters at once: blocks of one lie in one group of SMs, so not all SMs find a place
    const double waves = std::ceil((double)a.count * kCluster / (sms * 0.85));
    const double kb = (double)a.count * ((small + 127) / 128) * ((large + 63) / 64) / sms;
    const double chain = 3.0 * std::max(11500.0, 5000.0 + kb * ((small + 127) / 128) * 350.0);
    return waves * plan.cycles < chain;
}

int norm_blocks(const rune_orthogonalize_args& a) {
    const int64_t most = std::max<int64_t>(1, (int64_t)sm_count(a.device) * 8 / a.count);
    return (int)std::min<int64_t>((a.rows + 7) / 8, most);  // eight rows a block at once
}

void orthogonalize(const rune_orthogonalize_args& a, Scratch& ws, cudaStream_t stream) {
    const bool tall = a.rows > a.cols;
    const int64_t small = tall ? a.cols : a.rows;
    const int64_t ld = pad_line(a.cols, 2), lds = pad_line(small, 2);
    NormParams n{};
    n.rows = a.rows, n.cols = a.cols;
    n.step = a.x_step, n.row = a.x_row, n.col = a.x_col;
    n.ld = ld, n.out_step = a.rows * ld;
    n.blocks = norm_blocks(a);
    n.eps = a.eps;
    n.x = a.x;
    n.sums = ws.take<double>(a.count * n.blocks);
    Stack x[2]{}, g{}, h{};
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
    if (use_small(a, plan)) {
        run_small(a, plan, x, g, h, n, stream);
        return;
    }
    auto prepare = [&](auto t) {
        using T = decltype(t);
        launch(k_squares<T>, grid, kNormThreads, 0, 0, stream, n);
        launch(k_scale<T>, grid, kNormThreads, 0, 0, stream, n);
    };
    if (a.dtype == RUNE_F16) prepare(__half());
    else if (a.dtype == RUNE_BF16) prepare(__nv_bfloat16());
    else prepare(float());
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
