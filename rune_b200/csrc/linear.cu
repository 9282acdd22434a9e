// Linear layers on the tensor cores (tcgen05): the matrix product with scales, bias, activation
// and residual in its epilogue, the gated pair act(x Wg^T) * (x Wu^T), and their gradients
// (rune/mobius/layers.py:47-67 trains the same layer by automatic differentiation).
//
// One persistent kernel serves every product D[m, n] = sum_k A[m, k] B[n, k]:
//   forward      A = x   [rows, inputs]  (K-major)    B = W  [outputs, inputs] (K-major)
//   dx = dz W    A = dz  [rows, outputs] (K-major)    B = W  read MN-major
//   dW = dz^T x  A = dz  read MN-major                B = x  read MN-major
// so no operand is ever transposed in memory: the tensor core reads either order from the
// swizzled tiles that TMA writes. Tails of every size are zeros that TMA fills in.
//
// A block works on tiles of 128 rows x bn accumulator columns (bn = 64, 128 or 256), or a pair of
// blocks on 256 x bn (cta_group::2):
//   warp 16    one lane streams tiles of A and B (64 values of k; 128 for e4m3) by TMA into a ring
//              of as many stages as fit;
//   warp 17    one lane issues the products into one of two TMEM accumulators;
//   warps 0-15 the epilogue of the other accumulator: a lane holds a row; groups of 32 x 32 values
//              pass through swizzled buffers that TMA stores from.
// Every wait is bounded; one that gives up raises the device's wait flag and ends the block.
//
// What bounds it (B200, bf16): the tensor cores at wide layers - 8192 x 4096 -> 4096 179 us, 1535
// TFLOP/s; gated 4096 x 4096 -> 2 x 8192 338 us, 1624 TFLOP/s, the rate of a library product, and
// under long load the power limit (390 us). Narrow layers of many rows are bound by the epilogue:
// 110592 x 256 -> 512 35 us without activation (4.9 TB/s), 51 with silu, whose two special
// functions a value take 27; gated 64. What it took to get there, each at the size named:
//   tensor-core instructions issued by a converged warp, one kind a kernel   8192 x 4096 -> 4096
//     518 -> 232 us (from a divergent thread with both kinds they came at a third of the rate)
//   pairs of blocks, half of B's shared-memory traffic                        232 -> 182 us
//   sixteen epilogue warps for eight (every instruction waits some cycles for the one before)
//     and two values an instruction                       gated 110592 x 256 -> 512 101 -> 71 us
//   outputs by TMA for 16-byte stores of the lanes                            76 -> 63 us

#include <algorithm>
#include <atomic>
#include <mutex>

#include "act_grad.cuh"
#include "tile.cuh"

namespace rune {
namespace ops {

namespace {

// ----------------------------------------------------------------------------- joins
// y (and z) from the float32 sums of `splits` ranges of k, added in order. Four columns a
// thread; the sums' lines are padded to four values.
template <int MODE, typename T>
__global__ void __launch_bounds__(256) k_join(const TileParams p, const float* part) {
    follow_on();
    constexpr bool kPair = MODE == kGated;
    const int64_t groups = (p.n + 3) / 4, total = p.m * groups;
    const int64_t lds = ((kPair ? 2 * p.n : p.n) + 3) / 4 * 4;
    for (int64_t i = blockIdx.x * (int64_t)blockDim.x + threadIdx.x; i < total;
         i += (int64_t)gridDim.x * blockDim.x) {
        const int64_t row = i / groups, col = (i % groups) * 4;
        const float xs = p.x_scale ? p.x_scale[row] : 1.0f;
        auto sum = [&](int64_t c0, float (&v)[4]) {
#pragma unroll
            for (int j = 0; j < 4; ++j) v[j] = 0.0f;
            for (int s = 0; s < p.splits; ++s) {
                const float* at = part + ((int64_t)s * p.m + row) * lds + c0;
                if (!kPair || p.n % 4 == 0) {
                    float4 q = *reinterpret_cast<const float4*>(at);
                    v[0] += q.x, v[1] += q.y, v[2] += q.z, v[3] += q.w;
                } else {
                    for (int j = 0; j < 4 && col + j < p.n; ++j) v[j] += at[j];
                }
            }
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                if (col + j >= p.n) continue;
                if (p.w_scale) v[j] *= xs * p.w_scale[c0 + j];
                if (p.bias) v[j] += to_float(static_cast<const T*>(p.bias)[c0 + j]);
                if (p.z) p.z[row * p.ld_z + (c0 >= p.n ? p.ld_part + c0 - p.n : c0) + j] = v[j];
            }
        };
        float v[4], u[4];
        sum(col, v);
        if constexpr (kPair) sum(p.n + col, u);
        with_activation(p.act, [&](auto a) {
#pragma unroll
            for (int j = 0; j < 4; ++j) v[j] = act_value<decltype(a)::value>(v[j]);
        });
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            if (col + j >= p.n) continue;
            if constexpr (kPair) v[j] *= u[j];
            else if (p.in) v[j] += to_float(static_cast<const T*>(p.in)[row * p.ld_in + col + j]);
        }
        T* out = static_cast<T*>(p.out) + row * p.ld_out + col;
        if (p.tma_out && col + 4 <= p.n)
            *reinterpret_cast<uint2*>(out) = make_uint2(pack2<T>(v[0], v[1]), pack2<T>(v[2], v[3]));
        else
            for (int j = 0; j < 4 && col + j < p.n; ++j) out[j] = from_float<T>(v[j]);
    }
}

// ----------------------------------------------------------------------------- elementwise
// rows of a strip: fewer where 64 would leave the GPU short of blocks
int strip_rows(int64_t m, int64_t n, int sms) {
    const int64_t across = (n + kColumns - 1) / kColumns;
    int rows = 64;
    while (rows > 8 && (m + rows - 1) / rows * across < 4 * sms) rows /= 2;
    return rows;
}

// dz from a saved float32 z and dy, and the sums of each strip's columns
template <bool GATED, typename T>
__global__ void __launch_bounds__(256, 5)
k_act_grad(int64_t m, int64_t n, const float* z, int64_t ld_part,
           const T* dy, int64_t ld_dy, bool wide_dy, T* dz,
           int64_t ld_dz, int act, int strip, float* sums) {
    follow_on();
    const int64_t nz = GATED ? 2 * n : n, strips = (m + strip - 1) / strip;
    for (int64_t k = blockIdx.y; k < strips; k += gridDim.y)
        act_grad_rows<GATED, T>(k * strip, min(m, (k + 1) * strip), n, z, ld_part, dy, ld_dy,
                                wide_dy, dz, ld_dz, act, sums ? sums + k * nz : nullptr);
}

// the sums of each strip's columns
template <typename T>
__global__ void __launch_bounds__(256)
k_column_sums(int64_t m, int64_t n, const T* x, int64_t ld, bool wide, int strip,
              float* sums) {
    follow_on();
    const int64_t col = (int64_t)blockIdx.x * kColumns + (threadIdx.x & 63) * 4;
    const int count = (int)max((int64_t)0, min((int64_t)4, n - col)), part = threadIdx.x >> 6;
    const int64_t strips = (m + strip - 1) / strip;
    for (int64_t k = blockIdx.y; k < strips; k += gridDim.y) {
        const int64_t r1 = min(m, (k + 1) * strip);
        float s[4] = {};
        auto rows = [&](auto whole_c) {
#pragma unroll 8
            for (int64_t r = k * strip + part; r < r1; r += 4) {
                float v[4];
                get4<T, decltype(whole_c)::value>(x + r * ld + col, count, v);
#pragma unroll
                for (int j = 0; j < 4; ++j) s[j] += v[j];
            }
        };
        if (wide && count == 4) rows(std::true_type());
        else if (count > 0) rows(std::false_type());
        join4(s, sums + k * n + col, count);
    }
}

// Copies lines of `bytes` bytes, `ld` apart, to lines padded to 16 bytes (ld_dst), for operands
// that TMA cannot read in place; the padding is never read. A thread writes 16 bytes from the two
// aligned 16-byte words that hold them, shifted together; where such a word is not inside the
// matrix (its first and last lines), byte by byte.
__global__ void __launch_bounds__(256)
k_pack(const uint8_t* src, int64_t rows, int64_t bytes, int64_t ld,
       uint8_t* dst, int64_t ld_dst) {
    follow_on();
    const int64_t pieces = ld_dst / 16, total = rows * pieces;
    const uint8_t* const end = src + (rows - 1) * ld + bytes;
    const bool small = total <= INT32_MAX;  // quotients of 32 bits are a few instructions
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total;
         i += (int64_t)gridDim.x * 256) {
        const int64_t r = small ? (int64_t)((unsigned)i / (unsigned)pieces) : i / pieces;
        const int64_t at = (i - r * pieces) * 16;
        const uint8_t* from = src + r * ld + at;
        const unsigned off = (unsigned)((uintptr_t)from & 15);
        const uint8_t* word = from - off;
        uint4 out;
        if (word >= src && word + (off ? 32 : 16) <= end) {
            const uint4 a = *reinterpret_cast<const uint4*>(word);
            const uint4 b = off ? reinterpret_cast<const uint4*>(word)[1] : a;
            uint32_t w[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
            // by whole words in two steps, then by the bits that are left
            if (off & 8) {
#pragma unroll
                for (int i = 0; i < 6; ++i) w[i] = w[i + 2];
            }
            if (off & 4) {
#pragma unroll
                for (int i = 0; i < 5; ++i) w[i] = w[i + 1];
            }
            const unsigned bits = (off & 3) * 8;
            out.x = __funnelshift_r(w[0], w[1], bits);
            out.y = __funnelshift_r(w[1], w[2], bits);
            out.z = __funnelshift_r(w[2], w[3], bits);
            out.w = __funnelshift_r(w[3], w[4], bits);
        } else {
            uint32_t w[4] = {};
            for (int i = 0; i < 16; ++i)
                if (at + i < bytes) w[i / 4] |= (uint32_t)from[i] << (i % 4 * 8);
            out = make_uint4(w[0], w[1], w[2], w[3]);
        }
        *reinterpret_cast<uint4*>(dst + r * ld_dst + at) = out;
    }
}

// ----------------------------------------------------------------------------- host
// Tile, range of k and pairing of one product, by a model of its time in cycles: the k-blocks, an
// epilogue (16 cycles a column, 25 with an activation: measured at 110592 x 256 -> 512, 35 and
// 51 us), hidden behind the next tile's products, and for ranges of k the launch and the traffic of
// their join.
Plan plan_product(int64_t m, int64_t n_cols, int kblocks, bool can_split, bool gate, bool act,
                  int sms, uint32_t fixed) {
    Plan best{};
    double best_cost = 0.0;
    for (int pair = 1; pair >= 0; --pair) {
        for (int bn : {256, 128, 64}) {
            if ((gate || pair) && bn == 64) continue;  // halves of at least 64 columns
            const int rows = pair ? 2 * kBM : kBM, units = pair ? sms / 2 : sms;
            const int64_t tiles = ((m + rows - 1) / rows) * ((n_cols + bn - 1) / bn);
            const int most = can_split ? (int)std::min<int64_t>(std::max(1, kblocks / 4),
                                                                std::max<int64_t>(1, units / tiles))
                                       : 1;
            for (int s = 1; s <= most; ++s) {
                const int per = (kblocks + s - 1) / s;
                const int splits = (kblocks + per - 1) / per;
                const double waves = (double)((tiles * splits + units - 1) / units);
                const double main = per * block_cycles(pair, bn);
                const double epi = 1000.0 + (act ? (gate ? 15.0 : 25.0) : 16.0) * bn;
                double cost = 2000.0 + waves * std::max(main, epi) + std::min(main, epi);
                if (splits > 1)
                    cost += 5000.0 + (double)m * n_cols * (splits + 1) * 4.0 / 3000.0;
                if (best.bn == 0 || cost < best_cost) {
                    best_cost = cost;
                    best = {bn, splits, per, 0, pair == 1};
                }
            }
        }
    }
    best.stages = ring_stages(best.pair, best.bn, fixed);
    return best;
}

template <int MODE, typename T, bool FP8, bool PAIR>
void launch_tile(const CUtensorMap& a, const CUtensorMap& b, TileParams p, int sms, int device,
                 cudaStream_t stream) {
    CUtensorMap o = a, o2 = a;  // unused unless the output goes by TMA
    if (MODE != kPartial && p.tma_out) {
        o = make_out_map(p.out, p.m, p.n, p.ld_out);
        if (MODE == kGatedGrad)
            o2 = make_out_map(static_cast<T*>(p.out) + p.n, p.m, p.n, p.ld_out);
    }
    const int64_t work = (int64_t)p.tiles_m * p.tiles_n * p.splits;
    require(work < (1LL << 31) - 1024, "too many tiles");
    p.by_tiles = make_divisor((unsigned)p.tiles_m * p.tiles_n);
    p.by_group = make_divisor(kGroup * p.tiles_n);
    p.by_last = make_divisor(std::max(1u, (unsigned)p.tiles_m % kGroup));
    launch_blocks<MODE, kWhole, T, FP8, PAIR>(a, b, o, o2, p, work, kFixedSmem<MODE>, sms, device,
                                              stream);
}

// One product D[m, n] = A B^T: operands, epilogue (in p) and scratch for a split.
struct Product {
    Matrix a, b;             // K-major: [m, k], [n, k]; MN-major: [k, m], [k, n]
    bool a_mn = false, b_mn = false;
    int mode = kForward;
    int dtype = RUNE_BF16;   // of the operands
    int out_type = RUNE_BF16;
    int64_t k = 0;
};

template <int MODE, typename T>
void run_mode(const Product& g, TileParams p, Scratch& ws, int device, cudaStream_t stream) {
    const int sms = sm_count(device);
    const bool fp8 = g.dtype == RUNE_E4M3, pair = MODE == kGated || MODE == kGatedGrad;
    const int eb = fp8 ? 1 : 2, line = (int)kLineBytes / eb;
    const int64_t n_cols = pair ? 2 * p.n : p.n;
    p.kblocks = (int)((g.k + line - 1) / line);
    const bool can_split = MODE == kForward || MODE == kGated;
    Plan plan = plan_product(p.m, n_cols, p.kblocks, can_split, pair,
                             p.act != RUNE_ACT_NONE, sms, kFixedSmem<MODE>);
    float* part = nullptr;
    const int64_t ld_part = (n_cols + 3) / 4 * 4;
    if (plan.splits > 1) part = ws.take<float>(plan.splits * p.m * ld_part);
    if (ws.sizing()) return;
    p.bn = plan.bn;
    p.splits = plan.splits;
    p.kb_per_split = plan.kb_per_split;
    p.stages = plan.stages;
    const int tile_rows = plan.pair ? 2 * kBM : kBM;
    p.tiles_m = (int)((p.m + tile_rows - 1) / tile_rows);
    p.a_mn = g.a_mn, p.b_mn = g.b_mn;
    p.idesc = operand_idesc(fp8 ? 0 : g.dtype == RUNE_BF16 ? 1 : 0, g.a_mn, g.b_mn, tile_rows,
                            p.bn);
    const int b_box = plan.pair || pair ? p.bn / 2 : p.bn;  // lines of B in one copy
    p.flag = wait_flag(device);
    p.polls = wait_polls();
    const CUtensorMap ma = make_map(g.a, eb, g.a_mn ? 64 : kBM);
    if (plan.splits == 1) {
        const int width = pair ? p.bn / 2 : p.bn;
        p.tiles_n = (int)((p.n + width - 1) / width);
        const CUtensorMap mb = make_map(g.b, eb, g.b_mn ? 64 : b_box);
        auto go = [&](auto fp8_c) {
            constexpr bool FP8 = decltype(fp8_c)::value;
            if (plan.pair) launch_tile<MODE, T, FP8, true>(ma, mb, p, sms, device, stream);
            else launch_tile<MODE, T, FP8, false>(ma, mb, p, sms, device, stream);
        };
        if constexpr (MODE == kForward || MODE == kGated) {
            if (fp8) {
                go(std::true_type());
                return;
            }
        }
        go(std::false_type());
        return;
    }
    if constexpr (MODE == kForward || MODE == kGated) {
        TileParams q = p;  // plain sums over all rows of B, gate and up alike
        q.n = n_cols;
        q.tiles_n = (int)((n_cols + p.bn - 1) / p.bn);
        q.z = part;
        q.ld_z = ld_part;
        const CUtensorMap mb = make_map(g.b, eb, g.b_mn ? 64 : plan.pair ? p.bn / 2 : p.bn);
        auto go = [&](auto fp8_c) {
            constexpr bool FP8 = decltype(fp8_c)::value;
            if (plan.pair)
                launch_tile<kPartial, __half, FP8, true>(ma, mb, q, sms, device, stream);
            else
                launch_tile<kPartial, __half, FP8, false>(ma, mb, q, sms, device, stream);
        };
        if (fp8) go(std::true_type());
        else go(std::false_type());
        const int64_t items = p.m * ((p.n + 3) / 4);
        const int grid = (int)std::min<int64_t>((items + 255) / 256, (int64_t)sms * 16);
        launch(k_join<MODE, T>, grid, 256, 0, 0, stream, p, part);
        RUNE_LAUNCH_CHECK();
    }
}

void run_product(const Product& g, const TileParams& p, Scratch& ws, int device,
                 cudaStream_t stream) {
    auto typed = [&](auto t) {
        using T = decltype(t);
        switch (g.mode) {
            case kForward: run_mode<kForward, T>(g, p, ws, device, stream); break;
            case kGated: run_mode<kGated, T>(g, p, ws, device, stream); break;
            case kGrad: run_mode<kGrad, T>(g, p, ws, device, stream); break;
            default: run_mode<kGatedGrad, T>(g, p, ws, device, stream); break;
        }
    };
    if (g.out_type == RUNE_F16) typed(__half());
    else typed(__nv_bfloat16());
}

void pad_rows(const void* src, int64_t rows, int64_t bytes, int64_t ld, void* dst, int64_t ld_dst,
              cudaStream_t stream) {
    const int64_t blocks = (rows * (ld_dst / 16) + 255) / 256;
    launch(k_pack, (unsigned)std::min<int64_t>(blocks, 1 << 20), 256, 0, 0, stream, static_cast<const uint8_t*>(src), rows, bytes,
           ld, static_cast<uint8_t*>(dst), ld_dst);
}

// values of a row of the saved z for `outputs` columns (each of gate and up)
int64_t saved_line(int64_t outputs) { return (outputs + 3) / 4 * 4; }

void forward(const rune_linear_args& a, Scratch& ws, cudaStream_t stream) {
    const int eb = dtype_bytes(a.dtype);
    const int64_t n_all = a.gated ? 2 * a.outputs : a.outputs;
    Product g;
    g.a = readable({a.x, a.rows, a.inputs, a.x_stride}, eb, ws, stream);
    g.b = readable({a.weight, n_all, a.inputs, a.weight_stride}, eb, ws, stream);
    if (a.rows <= kFewRows) {
        if (!ws.sizing()) linear_few(a, g.a, g.b, stream);
        return;
    }
    g.mode = a.gated ? kGated : kForward;
    g.dtype = a.dtype;
    g.out_type = a.out_dtype;
    g.k = a.inputs;
    TileParams p{};
    p.m = a.rows, p.n = a.outputs;
    p.act = a.activation;
    p.out = a.y, p.ld_out = a.outputs;
    p.tma_out = wide16(a.y, a.outputs, a.outputs);
    p.in = a.residual, p.ld_in = a.residual_stride;
    p.vec_in = a.residual && wide16(a.residual, a.residual_stride, a.outputs);
    p.bias = a.bias;
    p.vec_bias = aligned(a.bias, 16) && a.outputs % 8 == 0;
    p.x_scale = a.x_scale, p.w_scale = a.weight_scale;
    p.z = a.saved, p.ld_part = saved_line(a.outputs);
    p.ld_z = (a.gated ? 2 : 1) * p.ld_part;
    run_product(g, p, ws, a.device, stream);
}

// rows of float32 for the parts of dbias (the tiles of a pair write whole eights) and their sums
int64_t round8(int64_t n) { return (n + 7) / 8 * 8; }
int64_t sum_rows(int64_t parts) { return round8(parts) + partial_scratch(parts); }

void backward(const rune_linear_grad_args& a, Scratch& ws, cudaStream_t stream) {
    const int64_t n_all = a.gated ? 2 * a.outputs : a.outputs;
    const bool plain = !a.gated && a.activation == RUNE_ACT_NONE;
    const bool half = a.dtype == RUNE_F16, want_dz = a.dx || a.dweight;
    // the operands that more than one product reads, readable by TMA
    Matrix x{a.x, a.rows, a.inputs, a.x_stride}, w{a.weight, n_all, a.inputs, a.weight_stride};
    const bool recompute = !plain && !a.saved;
    if (recompute || a.dweight) x = readable(x, 2, ws, stream);
    if (recompute || a.dx) w = readable(w, 2, ws, stream);
    // dz and the parts of dbias
    Matrix dz{a.dy, a.rows, n_all, a.dy_stride};
    float* sums = nullptr;
    int64_t parts = 0;
    const int strip = strip_rows(a.rows, a.outputs, sm_count(a.device));
    const int64_t strips = (a.rows + strip - 1) / strip;
    const bool wide_dy = aligned(a.dy, 8) && a.dy_stride % 4 == 0;
    if (plain) {
        if (want_dz) dz = readable(dz, 2, ws, stream);
        if (a.dbias) {
            parts = strips;
            sums = ws.take<float>(sum_rows(parts) * n_all);
            if (!ws.sizing()) {
                dim3 grid((unsigned)((n_all + kColumns - 1) / kColumns),
                          (unsigned)std::min<int64_t>(strips, 65535));
                if (half)
                    launch(k_column_sums<__half>, grid, 256, 0, 0, stream, a.rows, n_all,
                           static_cast<const __half*>(a.dy), a.dy_stride, wide_dy, strip, sums);
                else
                    launch(k_column_sums<__nv_bfloat16>, grid, 256, 0, 0, stream, a.rows, n_all,
                           static_cast<const __nv_bfloat16*>(a.dy), a.dy_stride, wide_dy, strip,
                           sums);
                RUNE_LAUNCH_CHECK();
            }
        }
    } else {
        dz.ld = pad_line(n_all, 2);
        uint16_t* to = ws.take<uint16_t>(a.rows * dz.ld);
        dz.p = to;
        if (a.saved) {
            parts = strips;
            if (a.dbias) sums = ws.take<float>(sum_rows(parts) * n_all);
            if (!ws.sizing()) {
                dim3 grid((unsigned)((a.outputs + kColumns - 1) / kColumns),
                          (unsigned)std::min<int64_t>(strips, 65535));
                auto go = [&](auto t) {
                    using T = decltype(t);
                    auto* dy = static_cast<const T*>(a.dy);
                    auto* out = reinterpret_cast<T*>(to);
                    if (a.gated)
                        launch(k_act_grad<true, T>, grid, 256, 0, 0, stream, a.rows, a.outputs,
                               a.saved, saved_line(a.outputs), dy, a.dy_stride, wide_dy, out,
                               dz.ld, a.activation, strip, sums);
                    else
                        launch(k_act_grad<false, T>, grid, 256, 0, 0, stream, a.rows, a.outputs,
                               a.saved, saved_line(a.outputs), dy, a.dy_stride, wide_dy, out,
                               dz.ld, a.activation, strip, sums);
                };
                if (half) go(__half());
                else go(__nv_bfloat16());
                RUNE_LAUNCH_CHECK();
            }
        } else {
            parts = (a.rows + 31) / 32;  // one a warp; the last tile (of a pair) has more warps
            if (a.dbias) sums = ws.take<float>(sum_rows(parts) * n_all);
            Product g;
            g.a = x, g.b = w;
            g.mode = a.gated ? kGatedGrad : kGrad;
            g.dtype = g.out_type = a.dtype;
            g.k = a.inputs;
            TileParams p{};
            p.m = a.rows, p.n = a.outputs;
            p.act = a.activation;
            p.out = to, p.ld_out = dz.ld;
            p.tma_out = !a.gated || a.outputs % 8 == 0;
            p.in = a.dy, p.ld_in = a.dy_stride;
            p.vec_in = wide16(a.dy, a.dy_stride, a.outputs);
            p.bias = a.bias;
            p.vec_bias = aligned(a.bias, 16) && a.outputs % 8 == 0;
            p.colsum = sums;
            run_product(g, p, ws, a.device, stream);
        }
        if (ws.sizing()) dz.p = reinterpret_cast<const void*>(256);
    }
    if (a.dbias && !ws.sizing())
        sum_partials(sums, parts, n_all, a.dbias, a.dtype, sums + round8(parts) * n_all,
                     stream);
    if (a.dx) {
        Product g;
        g.a = dz, g.b = w;
        g.b_mn = true;
        g.dtype = g.out_type = a.dtype;
        g.k = n_all;
        TileParams p{};
        p.m = a.rows, p.n = a.inputs;
        p.act = RUNE_ACT_NONE;
        p.out = a.dx, p.ld_out = a.inputs;
        p.tma_out = wide16(a.dx, a.inputs, a.inputs);
        run_product(g, p, ws, a.device, stream);
    }
    if (a.dweight) {
        Product g;
        g.a = dz, g.b = x;
        g.a_mn = g.b_mn = true;
        g.dtype = g.out_type = a.dtype;
        g.k = a.rows;
        TileParams p{};
        p.m = n_all, p.n = a.inputs;
        p.act = RUNE_ACT_NONE;
        p.out = a.dweight, p.ld_out = a.inputs;
        p.tma_out = wide16(a.dweight, a.inputs, a.inputs);
        run_product(g, p, ws, a.device, stream);
    }
}

constexpr int64_t kMaxSize = INT32_MAX - 512;  // tile coordinates are 32-bit

void check_sizes(int64_t rows, int64_t inputs, int64_t outputs, int gated, int act) {
    require(rows >= 0 && rows <= kMaxSize, "rows out of range");
    require(inputs >= 1 && inputs <= kMaxSize && outputs >= 1 && outputs <= kMaxSize / 2,
            "inputs or outputs out of range");
    require(act == RUNE_ACT_NONE || act == RUNE_ACT_TANH || act == RUNE_ACT_SILU ||
                act == RUNE_ACT_GELU,
            "unknown activation");
    require(!gated || act != RUNE_ACT_NONE, "a gated layer needs an activation");
}

void check_linear(const rune_linear_args& a) {
    check_sizes(a.rows, a.inputs, a.outputs, a.gated, a.activation);
    const bool fp8 = a.dtype == RUNE_E4M3;
    require(fp8 || a.dtype == RUNE_F16 || a.dtype == RUNE_BF16,
            "a linear layer takes float16, bfloat16 or e4m3 operands");
    require(fp8 ? a.out_dtype == RUNE_F16 || a.out_dtype == RUNE_BF16 : a.out_dtype == a.dtype,
            "the output has the operands' 16-bit type, or is 16-bit for e4m3");
    require(!!a.x_scale == fp8 && !!a.weight_scale == fp8,
            "x_scale and weight_scale go with e4m3 operands, both of them");
    require(!(a.gated && a.residual), "a gated layer takes no residual");
    require(a.rows == 0 || (a.x && a.weight && a.y), "null argument");
    require_aligned({a.x, a.weight}, dtype_bytes(a.dtype));
    require_aligned({a.bias, a.residual, a.y}, dtype_bytes(a.out_dtype));
    require_aligned({a.x_scale, a.weight_scale}, sizeof(float));
    require(aligned(a.saved, 16), "saved is not 16-byte aligned");
}

void check_grad(const rune_linear_grad_args& a) {
    check_sizes(a.rows, a.inputs, a.outputs, a.gated, a.activation);
    require(a.dtype == RUNE_F16 || a.dtype == RUNE_BF16,
            "gradients take float16 or bfloat16 operands");
    require(a.rows == 0 || (a.x && a.weight && a.dy), "null argument");
    require_aligned({a.x, a.weight, a.bias, a.dy, a.dx, a.dweight, a.dbias},
                    dtype_bytes(a.dtype));
    require(aligned(a.saved, 16), "saved is not 16-byte aligned");
}

using EncodeTiled = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*,
                                 const cuuint64_t*, const cuuint64_t*, const cuuint32_t*,
                                 const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                                 CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

EncodeTiled encode_tiled() {
    static EncodeTiled fn = [] {
        void* p = nullptr;
        cudaDriverEntryPointQueryResult found{};
        if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &p, 12000,
                                             cudaEnableDefault, &found) != cudaSuccess ||
            found != cudaDriverEntryPointSuccess)
            p = nullptr;
        return reinterpret_cast<EncodeTiled>(p);
    }();
    if (!fn) throw Error(RUNE_ERR_CUDA, "the CUDA driver has no cuTensorMapEncodeTiled");
    return fn;
}

std::atomic<unsigned> g_polls{RUNE_DEFAULT_WAIT_POLLS};
std::mutex g_flag_mutex;
constexpr int kMaxDevices = 64;
std::atomic<unsigned*> g_flag_host[kMaxDevices];
unsigned* g_flag_dev[kMaxDevices];

}  // namespace

Matrix readable(Matrix m, int elem_bytes, Scratch& ws, cudaStream_t stream) {
    if (m.rows == 1) m.ld = pad16(m.cols, elem_bytes);  // no second line to reach
    if (tma_ready(m, elem_bytes)) return m;
    Matrix d = m;
    d.ld = pad_line(m.cols, elem_bytes);
    void* to = ws.take<char>(m.rows * d.ld * elem_bytes);
    d.p = to;
    if (ws.sizing()) {
        d.p = reinterpret_cast<const void*>(256);  // any aligned address: only sizes are asked
        return d;
    }
    pad_rows(m.p, m.rows, m.cols * elem_bytes, m.ld * elem_bytes, to, d.ld * elem_bytes, stream);
    return d;
}

CUtensorMap make_map(const Matrix& m, int elem_bytes, int box_rows) {
    CUtensorMap map;
    const cuuint64_t dims[2] = {(cuuint64_t)m.cols, (cuuint64_t)m.rows};
    const cuuint64_t strides[1] = {(cuuint64_t)(m.ld * elem_bytes)};
    const cuuint32_t box[2] = {kLineBytes / (cuuint32_t)elem_bytes, (cuuint32_t)box_rows};
    const cuuint32_t step[2] = {1, 1};
    CUresult r = encode_tiled()(
        &map, elem_bytes == 1 ? CU_TENSOR_MAP_DATA_TYPE_UINT8 : CU_TENSOR_MAP_DATA_TYPE_UINT16, 2,
        const_cast<void*>(m.p), dims, strides, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE,
        CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
        CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS)
        throw Error(RUNE_ERR_INVALID,
                    "an operand cannot be described to TMA (status " + std::to_string(r) + ")");
    return map;
}

CUtensorMap make_map3(const Matrix& m, int64_t count, int64_t step, int elem_bytes, int box_rows) {
    CUtensorMap map;
    const cuuint64_t dims[3] = {(cuuint64_t)m.cols, (cuuint64_t)m.rows, (cuuint64_t)count};
    const cuuint64_t strides[2] = {(cuuint64_t)(m.ld * elem_bytes), (cuuint64_t)(step * elem_bytes)};
    const cuuint32_t box[3] = {kLineBytes / (cuuint32_t)elem_bytes, (cuuint32_t)box_rows, 1};
    const cuuint32_t each[3] = {1, 1, 1};
    CUresult r = encode_tiled()(
        &map, elem_bytes == 1 ? CU_TENSOR_MAP_DATA_TYPE_UINT8 : CU_TENSOR_MAP_DATA_TYPE_UINT16, 3,
        const_cast<void*>(m.p), dims, strides, box, each, CU_TENSOR_MAP_INTERLEAVE_NONE,
        CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
        CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS)
        throw Error(RUNE_ERR_INVALID,
                    "an operand cannot be described to TMA (status " + std::to_string(r) + ")");
    return map;
}

CUtensorMap make_out_map(const void* p, int64_t rows, int64_t cols, int64_t ld) {
    CUtensorMap map;
    const cuuint64_t dims[2] = {(cuuint64_t)cols, (cuuint64_t)rows};
    const cuuint64_t strides[1] = {(cuuint64_t)(ld * 2)};
    const cuuint32_t box[2] = {32, 32}, step[2] = {1, 1};
    CUresult r = encode_tiled()(&map, CU_TENSOR_MAP_DATA_TYPE_UINT16, 2, const_cast<void*>(p),
                                dims, strides, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE,
                                CU_TENSOR_MAP_SWIZZLE_64B, CU_TENSOR_MAP_L2_PROMOTION_NONE,
                                CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS)
        throw Error(RUNE_ERR_INVALID,
                    "an output cannot be described to TMA (status " + std::to_string(r) + ")");
    return map;
}

CUtensorMap make_out_map3(const void* p, int64_t rows, int64_t cols, int64_t ld, int64_t count,
                          int64_t step) {
    CUtensorMap map;
    const cuuint64_t dims[3] = {(cuuint64_t)cols, (cuuint64_t)rows, (cuuint64_t)count};
    const cuuint64_t strides[2] = {(cuuint64_t)(ld * 2), (cuuint64_t)(step * 2)};
    const cuuint32_t box[3] = {32, 32, 1}, each[3] = {1, 1, 1};
    CUresult r = encode_tiled()(&map, CU_TENSOR_MAP_DATA_TYPE_UINT16, 3, const_cast<void*>(p),
                                dims, strides, box, each, CU_TENSOR_MAP_INTERLEAVE_NONE,
                                CU_TENSOR_MAP_SWIZZLE_64B, CU_TENSOR_MAP_L2_PROMOTION_NONE,
                                CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS)
        throw Error(RUNE_ERR_INVALID,
                    "an output cannot be described to TMA (status " + std::to_string(r) + ")");
    return map;
}

unsigned wait_polls() { return g_polls.load(std::memory_order_relaxed); }

unsigned* wait_flag(int device) {
    if (device < 0 || device >= kMaxDevices)
        throw Error(RUNE_ERR_INVALID, "device index out of range");
    if (!g_flag_host[device].load(std::memory_order_acquire)) {
        std::lock_guard<std::mutex> lock(g_flag_mutex);
        if (!g_flag_host[device].load(std::memory_order_relaxed)) {
            // allowed while another thread, or this one, captures a graph
            cudaStreamCaptureMode mode = cudaStreamCaptureModeRelaxed;
            RUNE_CUDA_TRY(cudaThreadExchangeStreamCaptureMode(&mode));
            unsigned* host = nullptr;
            cudaError_t e = cudaHostAlloc(&host, sizeof(unsigned),
                                          cudaHostAllocMapped | cudaHostAllocPortable);
            if (e == cudaSuccess) {
                *host = 0;
                e = cudaHostGetDevicePointer(&g_flag_dev[device], host, 0);
            }
            cudaThreadExchangeStreamCaptureMode(&mode);
            RUNE_CUDA_TRY(e);
            g_flag_host[device].store(host, std::memory_order_release);
        }
    }
    return g_flag_dev[device];
}

void check_waits(int device) {
    if (device < 0 || device >= kMaxDevices) return;
    unsigned* host = g_flag_host[device].load(std::memory_order_acquire);
    if (!host || !*static_cast<volatile unsigned*>(host)) return;
    if (const unsigned where = __atomic_exchange_n(host, 0u, __ATOMIC_ACQ_REL))
        throw Error(RUNE_ERR_CUDA,
                    "A device-side copy of an earlier linear operator did not complete in time "
                    "(wait " + std::to_string(where) + "); the results of that call are invalid.");
}

}  // namespace ops
}  // namespace rune

using namespace rune;
using namespace rune::ops;

extern "C" {

int rune_linear_set_wait_polls(uint32_t polls) {
    g_polls.store(polls, std::memory_order_relaxed);
    return RUNE_OK;
}

int rune_linear_check_waits(int32_t device) {
    return guarded(device, [&] { check_waits(device); });
}

int rune_pad_rows(int32_t device, int64_t rows, int64_t bytes, int64_t stride, const void* src,
                  int64_t padded_stride, void* dst, void* stream) {
    return guarded(device, [&] {
        require(rows >= 0 && bytes >= 1 && padded_stride >= bytes && padded_stride % 16 == 0 &&
                    padded_stride / 16 <= INT32_MAX,
                "rows, bytes or padded_stride out of range");
        check_waits(device);
        if (rows == 0) return;
        require(src && dst && aligned(dst, 16), "null argument, or dst not 16-byte aligned");
        pad_rows(src, rows, bytes, stride, dst, padded_stride, static_cast<cudaStream_t>(stream));
    });
}

int rune_linear_workspace(const rune_linear_args* args, int64_t* bytes) {
    if (!args || !bytes) {
        set_error("null argument");
        return RUNE_ERR_INVALID;
    }
    const rune_linear_args a = *args;
    return guarded(a.device, [&] {
        check_linear(a);
        Scratch ws{nullptr};
        if (a.rows > 0) forward(a, ws, nullptr);
        *bytes = ws.off;
    });
}

int rune_linear(const rune_linear_args* args, void* stream_) {
    if (!args) {
        set_error("null argument");
        return RUNE_ERR_INVALID;
    }
    const rune_linear_args a = *args;
    auto stream = static_cast<cudaStream_t>(stream_);
    return guarded(a.device, [&] {
        check_linear(a);
        check_waits(a.device);
        if (a.rows == 0) return;
        Scratch need{nullptr};
        forward(a, need, stream);
        if (need.off > 0 && !a.workspace)
            throw Error(RUNE_ERR_RETRY, "the call needs a workspace");
        require(need.off == 0 || (a.workspace && aligned(a.workspace, 256) &&
                                  a.workspace_bytes >= need.off),
                "the workspace is too small or not 256-byte aligned");
        Scratch ws{need.off ? static_cast<char*>(a.workspace) : reinterpret_cast<char*>(256)};
        forward(a, ws, stream);
    });
}

int rune_linear_backward_workspace(const rune_linear_grad_args* args, int64_t* bytes) {
    if (!args || !bytes) {
        set_error("null argument");
        return RUNE_ERR_INVALID;
    }
    const rune_linear_grad_args a = *args;
    return guarded(a.device, [&] {
        check_grad(a);
        Scratch ws{nullptr};
        if (a.rows > 0) backward(a, ws, nullptr);
        *bytes = ws.off;
    });
}

int rune_linear_backward(const rune_linear_grad_args* args, void* stream_) {
    if (!args) {
        set_error("null argument");
        return RUNE_ERR_INVALID;
    }
    const rune_linear_grad_args a = *args;
    auto stream = static_cast<cudaStream_t>(stream_);
    return guarded(a.device, [&] {
        check_grad(a);
        check_waits(a.device);
        const int64_t n_all = a.gated ? 2 * a.outputs : a.outputs;
        if (a.rows == 0) {
            if (a.dweight)
                RUNE_CUDA_TRY(cudaMemsetAsync(a.dweight, 0, (size_t)(n_all * a.inputs * 2),
                                              stream));
            if (a.dbias)
                RUNE_CUDA_TRY(cudaMemsetAsync(a.dbias, 0, (size_t)(n_all * 2), stream));
            return;
        }
        Scratch need{nullptr};
        backward(a, need, stream);
        require(need.off == 0 || (a.workspace && aligned(a.workspace, 256) &&
                                  a.workspace_bytes >= need.off),
                "the workspace is too small or not 256-byte aligned");
        Scratch ws{need.off ? static_cast<char*>(a.workspace) : reinterpret_cast<char*>(256)};
        backward(a, ws, stream);
    });
}

}  // extern "C"
