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
