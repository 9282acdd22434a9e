// Linear and gated layers whose rows come in groups, each with its own weights, and their gradients:
//   y[p] = act(x[p] W_g^T + b_g),   gated: act(x[p] Wg_g^T + bg_g) * (x[p] Wu_g^T + bu_g),
//   dx[p] = dz[p] W_g,  dW_g = sum over p in g of dz[p]^T x[p],  db_g = sum over p in g of dz[p],
// for the places p of group g that the sort left in offsets[g] .. offsets[g + 1] - 1.
//
// The tile kernel of the linear layers runs them in one launch each. The groups' sizes are known on
// the GPU alone, so a block works its tiles out from the offsets:
//   forward, dz, dx   tiles of the rows of each group. A tile that reaches past its group's end
//                     reads rows of the next, whose results no one stores: boxes of whole rows leave
//                     by TMA, the last ones by the lanes. Weights are a 3-D map, zeros beyond a
//                     group's matrix, since dx contracts over its rows. Or, turned round, tiles of
//                     outputs by as many rows as there are, which wastes less at the groups' ends.
//   dW                a product per group over its rows. What lies behind the last row must be
//                     zeros in both operands (the next group's row may hold an infinity), so what a
//                     group has behind its whole blocks of 64 rows is copied to lines of its own
//                     first (k_group_tails). Tensor maps of each group's rows, written by the GPU,
//                     would save the copy; tests with them ended in memory faults.
// z of an activated layer is computed again in the backward pass or read from a float32 copy that the
// forward saved: the caller's choice, by what each costs.
//
// What bounds it (B200): wide layers the tensor cores under the power limit - 32768 x 2048 -> 4096 in
// 64 groups 520 us among other passes, 1.06 PFLOP/s (after a rest 465, 1.18); narrow ones of many rows
// the epilogue - gated 221184 x 256 -> 2 x 512 in 8 groups 135 us forward, 240 dz with recomputed z, 98
// dx (5.5 TB/s), 95 + 16 dW; small groups the weights - 8001 rows in 61 groups of 1024 -> 2 x 1408 86 us
// forward (5.2 TB/s), 73 dx, 83 dW (353 MB written; a write alone takes 92).

#include <cmath>

#include "act_grad.cuh"
#include "tile.cuh"

namespace rune {
namespace ops {

namespace {

constexpr int64_t kMaxSize = INT32_MAX - 512;  // tile coordinates are 32-bit
constexpr int64_t kMaxGroups = 1024;

// ----------------------------------------------------------------------------- kernels
// The last rows of each group behind its whole blocks of 64, of two matrices: 64 lines a group that has
// rows, zeros behind its end (those that have whole blocks alone are not written, and not read). Memory
// bounds it: 61 groups of 2816 and 1024 columns 16 us, 45 MB.
struct TailParams {
    const int32_t* offsets;
    int64_t rows;
    const uint16_t* from[2];
    uint16_t* to[2];
    int64_t ld_from[2], cols[2], ld_to[2];
};
__global__ void __launch_bounds__(256) k_group_tails(const TailParams p) {
    follow_on();
    const int g = blockIdx.y, which = blockIdx.z;
    const int64_t first = min((int64_t)max(p.offsets[g], 0), p.rows);
    const int64_t end = min((int64_t)max(p.offsets[g + 1], 0), p.rows);
    const int n = first < end ? (int)((end - first) & 63) : 0;
    if (n == 0) return;
    const int64_t ld = p.ld_from[which], cols = p.cols[which], ld_to = p.ld_to[which];
    const uint16_t* from = p.from[which] + (end - n) * ld;
    uint16_t* to = p.to[which] + (int64_t)tail_place(g, (int)first) * 64 * ld_to;
    const unsigned pieces = (unsigned)(ld_to / 8);
    for (unsigned i = blockIdx.x * 256 + threadIdx.x; i < 64 * pieces; i += gridDim.x * 256) {
        const int r = (int)(i / pieces);
        const int64_t c = (int64_t)(i - r * pieces) * 8;
        uint4 v = make_uint4(0, 0, 0, 0);
        if (r < n && c + 8 <= cols) {
            v = *reinterpret_cast<const uint4*>(from + r * ld + c);
        } else if (r < n) {
            uint32_t w[4] = {};
            for (int j = 0; j < 8; ++j)
                if (c + j < cols) w[j / 2] |= (uint32_t)from[r * ld + c + j] << (j % 2 * 16);
            v = make_uint4(w[0], w[1], w[2], w[3]);
        }
        *reinterpret_cast<uint4*>(to + r * ld_to + c) = v;
    }
}

// Number of lines of `high` rows that the groups before g fill, up to g and all; like the tile
// kernel's no more than offsets in order lead to, which the parts are sized for.
struct LineCount {
    int before, with, all;
};
__device__ __forceinline__ int group_lines(const int32_t* offsets, int64_t rows, int g, int high) {
    const int64_t a = min((int64_t)max(offsets[g], 0), rows);
    const int64_t b = min((int64_t)max(offsets[g + 1], 0), rows);
    return (int)((max((int64_t)0, b - a) + high - 1) / high);
}
__device__ __forceinline__ LineCount count_lines(const int32_t* offsets, int64_t rows, int groups,
                                                 int g, int high) {
    __shared__ int sums[2][32];
    const int most = (int)most_lines(rows, groups, high);
    int before = 0, all = 0;
    for (int i = threadIdx.x; i < groups; i += blockDim.x) {
        const int n = group_lines(offsets, rows, i, high);
        all = min(all + n, most);
        before = min(before + (i < g ? n : 0), most);
    }
    all = (int)__reduce_add_sync(0xffffffffu, (unsigned)all);
    before = (int)__reduce_add_sync(0xffffffffu, (unsigned)before);
    if ((threadIdx.x & 31) == 0) sums[0][threadIdx.x >> 5] = before, sums[1][threadIdx.x >> 5] = all;
    __syncthreads();
    before = all = 0;
    for (int w = 0; w < (int)blockDim.x / 32; ++w) {
        before = min(before + sums[0][w], most);
        all = min(all + sums[1][w], most);
    }
    return {before, min(before + group_lines(offsets, rows, g, high), most), all};
}

struct SumParams {
    const int32_t* offsets;
    int64_t rows, n;
    int groups, high, each;  // rows of a line of tiles, parts that each line left
    int64_t ld;              // k_group_columns: of x
    const void* x;
    float* parts;            // [lines * each][n]
    void* out;               // [groups][n]
    int ranges;              // of a group's rows or parts, summed apart
    int64_t line;
    float* sums;             // [ranges][groups][line]
};

// sums (p.sums) of the columns of a range of a group's rows: kColumns a block, four rows at a time
template <typename T>
__global__ void __launch_bounds__(256)
k_group_columns(const SumParams p, bool wide) {
    follow_on();
    const int64_t col = (int64_t)blockIdx.x * kColumns + (threadIdx.x & 63) * 4;
    const int count = (int)max((int64_t)0, min((int64_t)4, p.n - col)), part = threadIdx.x >> 6;
    const int g = blockIdx.y, range = blockIdx.z;
    const int64_t a = min((int64_t)max(p.offsets[g], 0), p.rows);
    const int64_t n = max((int64_t)0, min((int64_t)max(p.offsets[g + 1], 0), p.rows) - a);
    const int64_t r0 = a + n * range / p.ranges, r1 = a + n * (range + 1) / p.ranges;
    float s[4] = {};
    auto rows = [&](auto whole) {
        const T* x = static_cast<const T*>(p.x) + col;
#pragma unroll 8
        for (int64_t r = r0 + part; r < r1; r += 4) {
            float v[4];
            get4<T, decltype(whole)::value>(x + r * p.ld, count, v);
#pragma unroll
            for (int j = 0; j < 4; ++j) s[j] += v[j];
        }
    };
    if (wide && count == 4) rows(std::true_type());
    else if (count > 0) rows(std::false_type());
    join4(s, p.sums + ((int64_t)range * p.groups + g) * p.line + col, count);
}

// sums of a range of the parts that a group's lines of tiles left: 64 columns a block
template <typename T>
__global__ void __launch_bounds__(256)
k_group_sums(const SumParams p) {
    follow_on();
    __shared__ float joined[4][64];
    const int c = threadIdx.x & 63, turn = threadIdx.x >> 6;
    const int64_t col = (int64_t)blockIdx.x * 64 + c;
    const int g = blockIdx.y, range = blockIdx.z;
    const LineCount lines = count_lines(p.offsets, p.rows, p.groups, g, p.high);
    const int64_t n = (int64_t)(lines.with - lines.before) * p.each;
    const int64_t first = (int64_t)lines.before * p.each;
    const int64_t from = first + n * range / p.ranges, to = first + n * (range + 1) / p.ranges;
    float s = 0.0f;
    if (col < p.n) {
#pragma unroll 8
        for (int64_t i = from + turn; i < to; i += 4) s += p.parts[i * p.n + col];
    }
    joined[turn][c] = s;
    __syncthreads();
    if (turn != 0 || col >= p.n) return;
    const float sum = joined[0][c] + joined[1][c] + joined[2][c] + joined[3][c];
    if (p.ranges == 1) static_cast<T*>(p.out)[g * p.n + col] = from_float<T>(sum);
    else p.sums[((int64_t)range * p.groups + g) * p.line + col] = sum;
}

// dz of a range of a group's rows from a saved z, and its columns' sums (in p.sums); p.ld and p.x are
// of dy. Memory bounds it, and the largest group's last range: 8001 x 2816 in 61 groups 45 us, of 25.
struct SavedParams {
    const float* z;
    int64_t outputs, ld_part, ld_dz;
    void* dz;
    int act;
    bool wide_dy;
};
template <bool GATED, typename T>
__global__ void __launch_bounds__(256, 3)
k_group_act_grad(const SavedParams q, const SumParams p) {
    follow_on();
    const int g = blockIdx.y, range = blockIdx.z;
    const int64_t a = min((int64_t)max(p.offsets[g], 0), p.rows);
    const int64_t n = max((int64_t)0, min((int64_t)max(p.offsets[g + 1], 0), p.rows) - a);
    act_grad_rows<GATED, T>(
        a + n * range / p.ranges, a + n * (range + 1) / p.ranges, q.outputs, q.z, q.ld_part,
        static_cast<const T*>(p.x), p.ld, q.wide_dy, static_cast<T*>(q.dz), q.ld_dz, q.act,
        p.sums ? p.sums + ((int64_t)range * p.groups + g) * p.line : nullptr);
}

// value i of dbias from the sums of the ranges, in order
template <typename T>
__device__ __forceinline__ void join_sums(const SumParams& p, int64_t i) {
    if (i >= p.groups * p.n) return;
    const int64_t g = i / p.n, col = i - g * p.n;
    float s = 0.0f;
#pragma unroll 8
    for (int r = 0; r < p.ranges; ++r) s += p.sums[((int64_t)r * p.groups + g) * p.line + col];
    static_cast<T*>(p.out)[i] = from_float<T>(s);
}
template <typename T>
__global__ void __launch_bounds__(256) k_join_sums(const SumParams p) {
    follow_on();
    join_sums<T>(p, (int64_t)blockIdx.x * 256 + threadIdx.x);
}

// dW from the parts of its tiles (kDepthRanges), added in the order of k: a block has 1024 / `lanes`
// values of a tile, four a thread; `lanes` threads share the parts and join their sums in order. The
// blocks behind the tiles' finish dbias.
struct JoinParams {
    const int32_t* offsets;
    int64_t rows, m, n;
    int groups, tiles_m, tiles_n, high, bn, ranges, lanes;  // ranges: planned
    bool wide;         // rows of the output on 8 bytes
    const float* parts;
    void* out;         // [groups][m][n]
};
constexpr int kJoinThreads = 256;
template <typename T>
__global__ void __launch_bounds__(kJoinThreads)
k_join_parts(const JoinParams p, const SumParams sum) {
    follow_on();
    __shared__ float4 joined[kJoinThreads];
    const int tiles = p.tiles_m * p.tiles_n, g = blockIdx.x / tiles, at = blockIdx.x - g * tiles;
    if (g >= p.groups) {
        const int64_t block = (int64_t)(blockIdx.x - p.groups * tiles) * gridDim.y + blockIdx.y;
        join_sums<T>(sum, block * kJoinThreads + threadIdx.x);
        return;
    }
    const LineCount lines = count_lines(p.offsets, p.rows, p.groups, g, 64);
    // the ranges in which the group's first and last k-blocks lie
    int r0 = 0, r1 = -1;
    if (lines.with > lines.before) {
        const unsigned ranges = range_count(p.ranges, lines.all);
        r0 = (int)range_at(lines.before, ranges, lines.all);
        r1 = (int)range_at(lines.with - 1, ranges, lines.all);
    }
    const int each = kJoinThreads / p.lanes;
    const int item = threadIdx.x % each, lane = threadIdx.x / each;
    const int i = (blockIdx.y * each + item) * 4, row = i / p.bn, col = i - row * p.bn;
    const int64_t out_row = (int64_t)(at / p.tiles_n) * p.high + row;
    const int64_t out_col = (int64_t)(at % p.tiles_n) * p.bn + col;
    const bool in = out_row < p.m && out_col < p.n;
    float v[4] = {};
    if (in) {
        const int64_t size = (int64_t)p.high * p.bn;
        const float* part = p.parts + ((int64_t)g * tiles + at) * size + i;
#pragma unroll 4
        for (int r = r0 + lane; r <= r1; r += p.lanes) {
            const float4 q = *reinterpret_cast<const float4*>(part + r * tiles * size);
            v[0] += q.x, v[1] += q.y, v[2] += q.z, v[3] += q.w;
        }
    }
    if (p.lanes > 1) {
        joined[threadIdx.x] = make_float4(v[0], v[1], v[2], v[3]);
        __syncthreads();
        if (lane > 0) return;
        for (int s = 1; s < p.lanes; ++s) {
            const float4 q = joined[s * each + item];
            v[0] += q.x, v[1] += q.y, v[2] += q.z, v[3] += q.w;
        }
    }
    if (!in) return;
    T* to = static_cast<T*>(p.out) + (g * p.m + out_row) * p.n + out_col;
    if (p.wide)
        *reinterpret_cast<uint2*>(to) = make_uint2(pack2<T>(v[0], v[1]), pack2<T>(v[2], v[3]));
    else
        for (int j = 0; j < 4 && out_col + j < p.n; ++j) to[j] = from_float<T>(v[j]);
}

// ----------------------------------------------------------------------------- host
uint32_t table_bytes(int64_t groups) {
    return (uint32_t)((2 * groups + 2) * 4 + 127) / 128 * 128;
}

// Tile and pairing of a product of rows by group, by the time of the whole product's model. Each
// group that has rows ends inside a line of tiles.
Plan plan_rows(int64_t rows, int64_t groups, int64_t n_cols, int kblocks, bool gate, bool act,
               int sms, uint32_t fixed) {
    Plan best{};
    double best_cost = 0.0;
    const double met = (double)std::min(rows, groups);
    for (int pair = 1; pair >= 0; --pair) {
        for (int bn : {256, 128, 64}) {
            if ((gate || pair) && bn == 64) continue;  // halves of at least 64 columns
            const int high = pair ? 2 * kBM : kBM, units = pair ? sms / 2 : sms;
            const double lines = std::max(met, rows / (double)high + 0.5 * met);
            const double tiles = lines * ((n_cols + bn - 1) / bn);
            const double waves = std::max(1.0, tiles / units + (tiles > units ? 0.5 : 0.0));
            const double main = kblocks * block_cycles(pair, bn);
            const double epi = 1000.0 + (act ? (gate ? 15.0 : 25.0) : 16.0) * bn;
            const double cost = waves * std::max(main, epi) + std::min(main, epi);
            if (best.bn == 0 || cost < best_cost) {
                best_cost = cost;
                best = {bn, 1, kblocks, 0, pair == 1};
            }
        }
    }
    best.stages = ring_stages(best.pair, best.bn, fixed);
    return best;
}

// Whether a product of rows by group is sooner done turned round (kRowsAcross), where the lines that
// the groups' ends leave part empty count: contractions that hide the epilogue, groups of some rows
// but not of very many, outputs that fill their tiles. B200, pass after pass (under the power limit),
// kRowGroups / kRowsAcross, us:
//   32768 x 2048 -> 4096, 64 groups, gelu 555 / 520    16000 x 512 -> 512, 16 groups 15.0 / 12.2
//   20000 x 4096 -> 1024, 128 groups      300 / 236    200000 x 1024 -> 256, 8 groups  96 /  97
//   2000 x 2816 -> 1024, 61 groups       61.7 / 65.2   100 x 4096 -> 4096, 16 groups 90.7 / 92.4
bool across_pays(int64_t rows, int64_t groups, int64_t n, int kblocks) {
    const int64_t met = std::min(rows, groups);
    return kblocks >= 8 && rows >= 96 * met && rows <= 4096 * met &&
           (n + 255) / 256 * 256 * 4 <= n * 5;
}

// Tile and pairing of the groups' products over their rows. Either a tile is a block's own (splits
// 1), and the last block's tiles, of a group of perhaps three times the mean, end late; or the
// k-blocks of all groups divide into `splits` equal ranges, for the traffic and the launch of a join.
Plan plan_depth(int64_t rows, int64_t groups, int64_t m, int64_t n, int sms, uint32_t fixed) {
    Plan best{};
    double best_cost = 0.0;
    const double depth = std::max(1.0, rows / 64.0 / groups + 0.5);  // k-blocks of a group
    for (int pair = 1; pair >= 0; --pair) {
        for (int bn : {256, 128, 64}) {
            if (pair && bn == 64) continue;
            const int high = pair ? 2 * kBM : kBM, units = pair ? sms / 2 : sms;
            const double tiles = (double)((m + high - 1) / high) * ((n + bn - 1) / bn);
            const double epi = 1000.0 + 16.0 * bn, block = block_cycles(pair, bn);
            auto offer = [&](double cost, int splits) {
                if (best.bn == 0 || cost < best_cost) {
                    best_cost = cost;
                    best = {bn, splits, 0, 0, pair == 1};
                }
            };
            offer(std::max(1.0, tiles * groups / units) * std::max(depth * block, epi) +
                      2.0 * depth * block + epi, 1);
            if (tiles * (rows / 64.0 + groups) > 1.0e9) continue;  // its counter has 32 bits
            for (int waves = 1; waves <= 4; ++waves) {
                // one to four items a block, of four k-blocks at least
                const int ranges = (int)std::min(std::floor(waves * units / tiles),
                                                 depth * groups / 4.0);
                if (ranges < 2) continue;
                const double items = std::ceil(ranges * tiles / units);
                const double each = depth * groups / ranges * block;
                offer(items * (each + (1.0 + (double)groups / ranges) * epi) + 6000.0 +
                          (ranges + groups) * tiles * high * bn * 8.0 / 3000.0, ranges);
            }
        }
    }
    best.stages = ring_stages(best.pair, best.bn, fixed);
    return best;
}

// A stack of `groups` matrices, rows and matrices alike `ld` values apart.
struct Weights {
    Matrix all;
    int64_t rows;  // of each
    CUtensorMap map(int64_t groups, int box_rows) const {
        Matrix one = all;
        one.rows = rows;
        return make_map3(one, groups, rows * all.ld, 2, box_rows);
    }
};

template <int MODE, int KIND, typename T>
void launch_kind(bool pair, const CUtensorMap& a, const CUtensorMap& b, const CUtensorMap& o,
                 const CUtensorMap& o2, const TileParams& p, int64_t work, uint32_t fixed, int sms,
                 int device, cudaStream_t stream, const CUtensorMap* tail = nullptr) {
    require(work < (1LL << 31) - 1024, "too many tiles");
    if (pair)
        launch_blocks<MODE, KIND, T, false, true>(a, b, o, o2, p, work, fixed, sms, device, stream,
                                                  tail);
    else
        launch_blocks<MODE, KIND, T, false, false>(a, b, o, o2, p, work, fixed, sms, device,
                                                   stream, tail);
}

// Rows of A by group, each with its matrix of w (K-major, or MN-major for dx).
struct RowProduct {
    Matrix a;
    Weights w;
    bool w_mn = false;
    int64_t k = 0, groups = 0;
    const int32_t* offsets = nullptr;
    int device = 0, dtype = 0;
};

// Height of the tiles' lines: dbias needs it for its parts.
template <int MODE, typename T>
int run_rows(const RowProduct& g, TileParams p, bool launch_it, cudaStream_t stream) {
    constexpr bool kGate = MODE == kGated || MODE == kGatedGrad;
    const int sms = sm_count(g.device);
    const int64_t n_cols = kGate ? 2 * p.n : p.n;
    const uint32_t fixed = kFixedSmem<MODE> + table_bytes(g.groups);
    p.kblocks = (int)((g.k + 63) / 64);
    const Plan plan = plan_rows(g.a.rows, g.groups, n_cols, p.kblocks, kGate,
                                p.act != RUNE_ACT_NONE, sms, fixed);
    const int high = plan.pair ? 2 * kBM : kBM;
    if (!launch_it) return high;
    p.m = p.m_all = g.a.rows;
    p.groups = (int)g.groups;
    p.offsets = g.offsets;
    p.bias_step = n_cols;
    p.bn = plan.bn, p.stages = plan.stages;
    p.splits = 1, p.kb_per_split = p.kblocks;
    const int width = kGate ? p.bn / 2 : p.bn;
    p.tiles_n = (int)((p.n + width - 1) / width);
    p.by_tiles = make_divisor((unsigned)p.tiles_n);
    p.by_group = make_divisor(kGroup * (unsigned)p.tiles_n);
    p.b_mn = g.w_mn;
    p.idesc = operand_idesc(g.dtype == RUNE_BF16 ? 1 : 0, false, g.w_mn, high, p.bn);
    p.flag = wait_flag(g.device);
    p.polls = wait_polls();
    const CUtensorMap a = make_map(g.a, 2, kBM);
    const CUtensorMap b =
        g.w.map(g.groups, g.w_mn ? 64 : plan.pair || kGate ? p.bn / 2 : p.bn);
    CUtensorMap o = a, o2 = a;  // unused unless the output goes by TMA
    if (p.tma_out) {
        o = make_out_map(p.out, p.m_all, p.n, p.ld_out);
        if (MODE == kGatedGrad)
            o2 = make_out_map(static_cast<T*>(p.out) + p.n, p.m_all, p.n, p.ld_out);
    }
    launch_kind<MODE, kRowGroups, T>(plan.pair, a, b, o, o2, p,
                                     most_lines(p.m_all, g.groups, high) * p.tiles_n, fixed, sms,
                                     g.device, stream);
    return high;
}

// The same turned round, for kForward and kPlain.
template <int MODE, typename T>
void run_across(const RowProduct& g, TileParams p, cudaStream_t stream) {
    const int sms = sm_count(g.device);
    const uint32_t fixed = kFixedSmem<MODE> + table_bytes(g.groups);
    p.kblocks = p.kb_per_split = (int)((g.k + 63) / 64), p.splits = 1;
    p.m = p.m_all = g.a.rows;
    p.groups = (int)g.groups;
    p.offsets = g.offsets;
    p.bias_step = p.n;
    p.bn = 2 * kBM, p.stages = ring_stages(true, p.bn, fixed);
    p.tiles_n = (int)((p.n + 2 * kBM - 1) / (2 * kBM));
    p.by_tiles = make_divisor((unsigned)p.tiles_n);
    p.by_group = make_divisor(kGroup * (unsigned)p.tiles_n);
    p.a_mn = g.w_mn;
    p.idesc = operand_idesc(g.dtype == RUNE_BF16 ? 1 : 0, g.w_mn, false, 2 * kBM, 0);  // and N
    p.flag = wait_flag(g.device);
    p.polls = wait_polls();
    const CUtensorMap a = g.w.map(g.groups, g.w_mn ? 64 : kBM);
    const CUtensorMap b = make_map(g.a, 2, 16), whole = make_map(g.a, 2, kBM);
    const CUtensorMap o = p.tma_out ? make_out_map(p.out, p.m_all, p.n, p.ld_out) : a;
    const int64_t work = most_lines(p.m_all, g.groups, 2 * kBM) * p.tiles_n;
    require(work < (1LL << 31) - 1024, "too many tiles");
    launch_blocks<MODE, kRowsAcross, T, false, true>(a, b, o, whole, p, work, fixed, sms, g.device,
                                                     stream);
}

int run_rows(int mode, const RowProduct& g, const TileParams& p, bool launch_it,
             cudaStream_t stream) {
    const int kblocks = (int)((g.k + 63) / 64);
    if (launch_it && (mode == kForward || mode == kPlain) &&
        across_pays(g.a.rows, g.groups, p.n, kblocks)) {
        auto go = [&](auto t) {
            using T = decltype(t);
            if (mode == kPlain) run_across<kPlain, T>(g, p, stream);
            else run_across<kForward, T>(g, p, stream);
        };
        if (g.dtype == RUNE_F16) go(__half());
        else go(__nv_bfloat16());
        return 0;
    }
    auto typed = [&](auto t) {
        using T = decltype(t);
        switch (mode) {
            case kForward: return run_rows<kForward, T>(g, p, launch_it, stream);
            case kGated: return run_rows<kGated, T>(g, p, launch_it, stream);
            case kGrad: return run_rows<kGrad, T>(g, p, launch_it, stream);
            case kPlain: return run_rows<kPlain, T>(g, p, launch_it, stream);
            default: return run_rows<kGatedGrad, T>(g, p, launch_it, stream);
        }
    };
    return g.dtype == RUNE_F16 ? typed(__half()) : typed(__nv_bfloat16());
}

void forward(const rune_grouped_linear_args& a, Scratch& ws, cudaStream_t stream) {
    const int64_t n_all = a.gated ? 2 * a.outputs : a.outputs;
    RowProduct g;
    g.a = readable({a.x, a.rows, a.inputs, a.x_stride}, 2, ws, stream);
    g.w = {readable({a.weight, a.groups * n_all, a.inputs, a.weight_stride}, 2, ws, stream), n_all};
    if (ws.sizing()) return;
    if (a.rows <= kFewRows) {
        grouped_few(a, g.a, g.w.all, stream);
        return;
    }
    g.k = a.inputs, g.groups = a.groups;
    g.offsets = a.offsets;
    g.device = a.device, g.dtype = a.dtype;
    TileParams p{};
    p.n = a.outputs;
    p.act = a.activation;
    p.out = a.y, p.ld_out = a.outputs;
    p.tma_out = wide16(a.y, a.outputs, a.outputs);
    p.zero_tail = 1;
    p.bias = a.bias;
    p.vec_bias = aligned(a.bias, 16) && a.outputs % 8 == 0;
    p.z = a.saved, p.ld_part = (a.outputs + 3) / 4 * 4;
    p.ld_z = (a.gated ? 2 : 1) * p.ld_part;
    const bool plain = a.activation == RUNE_ACT_NONE && !a.bias && !a.saved;
    run_rows(a.gated ? kGated : plain ? kPlain : kForward, g, p, true, stream);
}

// The groups' products dW = dz^T x: plan, scratch and the last rows to copy.
struct Depth {
    Plan plan{};
    uint32_t fixed = 0;
    int high = 0, tiles_m = 0, tiles_n = 0;
    float* parts = nullptr;
    TailParams tails{};
};

Depth plan_weights(const rune_grouped_linear_grad_args& a, const Matrix& dz, const Matrix& x,
                   Scratch& ws) {
    Depth d;
    const int64_t m = dz.cols, n = x.cols;
    d.fixed = std::max(kFixedSmem<kPlain>, kFixedSmem<kPartial>) + table_bytes(a.groups);
    d.plan = plan_depth(a.rows, a.groups, m, n, sm_count(a.device), d.fixed);
    d.high = d.plan.pair ? 2 * kBM : kBM;
    d.tiles_m = (int)((m + d.high - 1) / d.high);
    d.tiles_n = (int)((n + d.plan.bn - 1) / d.plan.bn);
    for (int i = 0; i < 2; ++i) {
        const Matrix& from = i ? x : dz;
        d.tails.from[i] = static_cast<const uint16_t*>(from.p), d.tails.ld_from[i] = from.ld;
        d.tails.cols[i] = from.cols, d.tails.ld_to[i] = pad_line(from.cols, 2);
        // k_group_tails counts the pieces of 64 lines in 32 bits, and one line is half a GB here
        require(d.tails.ld_to[i] <= 1LL << 28, "inputs or outputs out of range for weight gradients: "
                                               "2^28 at most");
        d.tails.to[i] = ws.take<uint16_t>(std::min(a.groups, a.rows) * 64 * d.tails.ld_to[i]);
    }
    d.tails.offsets = a.offsets, d.tails.rows = a.rows;
    if (d.plan.splits > 1)
        d.parts = ws.take<float>((a.groups + d.plan.splits) * d.tiles_m * d.tiles_n * d.high *
                                 d.plan.bn);
    return d;
}

// sum: of dbias, whose ranges this call's last kernel joins; true if it did
template <typename T>
bool run_weights(const rune_grouped_linear_grad_args& a, const Matrix& dz, const Matrix& x,
                 const Depth& d, const SumParams& sum, cudaStream_t stream) {
    const int64_t m = dz.cols, n = x.cols, each = (int64_t)d.tiles_m * d.tiles_n;
    const int sms = sm_count(a.device);
    const CUtensorMap ma = make_map(dz, 2, 64), mb = make_map(x, 2, 64);
    auto tail = [&](int i) {
        return make_map({d.tails.to[i], std::min(a.groups, a.rows) * 64, d.tails.cols[i],
                         d.tails.ld_to[i]}, 2, 64);
    };
    const CUtensorMap ta = tail(0), tb = tail(1);
    TileParams p{};
    p.m = m, p.n = n;
    p.act = RUNE_ACT_NONE;
    p.m_all = a.rows, p.groups = (int)a.groups, p.offsets = a.offsets;
    p.bn = d.plan.bn, p.stages = d.plan.stages, p.splits = 1;
    p.tiles_m = d.tiles_m, p.tiles_n = d.tiles_n;
    p.by_tiles = make_divisor((unsigned)each);
    p.by_group = make_divisor(kGroup * (unsigned)d.tiles_n);
    p.by_last = make_divisor(std::max(1u, (unsigned)d.tiles_m % kGroup));
    p.a_mn = p.b_mn = 1;
    p.idesc = operand_idesc(a.dtype == RUNE_BF16 ? 1 : 0, true, true, d.high, p.bn);
    p.flag = wait_flag(a.device);
    p.polls = wait_polls();
    if (d.plan.splits == 1) {
        p.out = a.dweight, p.ld_out = n, p.out_step = m * n;
        p.tma_out = wide16(a.dweight, n, n);
        const CUtensorMap o =
            p.tma_out ? make_out_map3(a.dweight, m, n, n, a.groups, m * n) : ma;
        launch_kind<kPlain, kDepthGroups, T>(d.plan.pair, ma, mb, o, ta, p, each * a.groups, d.fixed,
                                             sms, a.device, stream, &tb);
        return false;
    }
    p.ranges = d.plan.splits;
    p.z = d.parts, p.ld_part = d.high;
    launch_kind<kPartial, kDepthRanges, __half>(d.plan.pair, ma, mb, ma, ta, p, p.ranges * each,
                                                d.fixed, sms, a.device, stream, &tb);
    // sixteen threads share the parts of a tile where these are many
    const int lanes = p.ranges >= 16 * a.groups ? 16 : 1;
    const JoinParams j{a.offsets, a.rows, m, n, (int)a.groups, d.tiles_m, d.tiles_n, d.high, p.bn,
                       p.ranges, lanes, n % 4 == 0 && aligned(a.dweight, 8), d.parts, a.dweight};
    const int64_t rows_y = d.high * p.bn / 4 * lanes / kJoinThreads;
    const int64_t more = sum.sums ? (a.groups * sum.n + rows_y * kJoinThreads - 1) /
                                              (rows_y * kJoinThreads) : 0;
    launch(k_join_parts<T>, dim3((unsigned)(each * a.groups + more), (unsigned)rows_y),
           kJoinThreads, 0, 0, stream, j, sum);
    return true;
}

void backward(const rune_grouped_linear_grad_args& a, Scratch& ws, cudaStream_t stream) {
    const int64_t n_all = a.gated ? 2 * a.outputs : a.outputs;
    const bool plain = !a.gated && a.activation == RUNE_ACT_NONE;
    const bool half = a.dtype == RUNE_F16;
    Matrix x{a.x, a.rows, a.inputs, a.x_stride};
    Weights w{{a.weight, a.groups * n_all, a.inputs, a.weight_stride}, n_all};
    const bool recompute = !plain && !a.saved;
    if (recompute || a.dweight) x = readable(x, 2, ws, stream);
    if (recompute || a.dx) w.all = readable(w.all, 2, ws, stream);
    RowProduct g;
    g.groups = a.groups, g.offsets = a.offsets;
    g.device = a.device, g.dtype = a.dtype;
    Matrix dz{a.dy, a.rows, n_all, a.dy_stride};
    SumParams sum{a.offsets, a.rows, n_all, (int)a.groups, 0, 0, a.dy_stride, a.dy, nullptr,
                  a.dbias, 1, 0, nullptr};
    TileParams p{};
    const int mode = a.gated ? kGatedGrad : kGrad;
    if (plain) {
        if (a.dx || a.dweight) dz = readable(dz, 2, ws, stream);
    } else {
        dz.ld = pad_line(n_all, 2);
        dz.p = ws.take<uint16_t>(a.rows * dz.ld);
    }
    if (recompute) {
        g.a = x, g.w = w, g.k = a.inputs;
        p.n = a.outputs;
        p.act = a.activation;
        p.out = const_cast<void*>(dz.p), p.ld_out = dz.ld;
        p.tma_out = !a.gated || a.outputs % 8 == 0;
        p.in = a.dy, p.ld_in = a.dy_stride;
        p.vec_in = wide16(a.dy, a.dy_stride, a.outputs);
        p.bias = a.bias;
        p.vec_bias = aligned(a.bias, 16) && a.outputs % 8 == 0;
        sum.high = run_rows(mode, g, p, false, stream);
        sum.each = sum.high / 32;  // one a warp
    }
    if (a.dbias || (!plain && a.saved)) {
        const int64_t parts =
            recompute ? most_lines(a.rows, a.groups, sum.high) * sum.each : a.rows;
        if (recompute) sum.parts = ws.take<float>(parts * n_all);
        // parts or rows of a range where groups are alike: few enough that the largest group's ranges do
        // not end last, and enough to make up for a block's start
        const int64_t mean = parts / a.groups, each = recompute ? 64 : plain ? 40 : 16;
        sum.ranges = mean < 4 * each ? 1 : (int)std::min<int64_t>(256, mean / each);
        sum.line = (n_all + 3) / 4 * 4;
        if (a.dbias && (sum.ranges > 1 || !recompute))
            sum.sums = ws.take<float>(sum.ranges * a.groups * sum.line);
    }
    Depth depth;
    if (a.dweight) depth = plan_weights(a, dz, x, ws);
    if (ws.sizing()) return;
    if (recompute) {
        p.colsum = sum.parts;
        run_rows(mode, g, p, true, stream);
    }
    auto typed = [&](auto t) {
        using T = decltype(t);
        const unsigned slices = sum.ranges;
        const bool wide_dy = aligned(a.dy, 8) && a.dy_stride % 4 == 0;
        if (!plain && a.saved) {
            const SavedParams q{a.saved, a.outputs, (a.outputs + 3) / 4 * 4, dz.ld,
                                const_cast<void*>(dz.p), a.activation, wide_dy};
            const dim3 grid((unsigned)((a.outputs + kColumns - 1) / kColumns), (unsigned)a.groups,
                            slices);
            if (a.gated)
                launch(k_group_act_grad<true, T>, grid, 256, 0, 0, stream, q, sum);
            else
                launch(k_group_act_grad<false, T>, grid, 256, 0, 0, stream, q, sum);
        } else if (a.dbias) {
            const int64_t columns = plain ? kColumns : 64;
            const dim3 grid((unsigned)((n_all + columns - 1) / columns), (unsigned)a.groups,
                            slices);
            if (plain)
                launch(k_group_columns<T>, grid, 256, 0, 0, stream, sum, wide_dy);
            else
                launch(k_group_sums<T>, grid, 256, 0, 0, stream, sum);
        }
        if (a.dweight) {
            const int64_t wide = std::max(depth.tails.ld_to[0], depth.tails.ld_to[1]) * 8;
            const dim3 grid((unsigned)std::min<int64_t>((wide + 1023) / 1024, 256),
                            (unsigned)a.groups, 2);
            launch(k_group_tails, grid, 256, 0, 0, stream, depth.tails);
        }
        if (a.dx) {
            RowProduct d = g;
            d.a = dz, d.w = w, d.w_mn = true;
            d.k = n_all;
            TileParams q{};
            q.n = a.inputs;
            q.act = RUNE_ACT_NONE;
            q.out = a.dx, q.ld_out = a.inputs;
            q.tma_out = wide16(a.dx, a.inputs, a.inputs);
            q.zero_tail = 1;
            run_rows(kPlain, d, q, true, stream);
        }
        const bool joined = a.dweight && run_weights<T>(a, dz, x, depth, sum, stream);
        if (sum.sums && !joined)
            launch(k_join_sums<T>, (unsigned)((a.groups * n_all + 255) / 256), 256, 0, 0, stream,
                   sum);
    };
    if (half) typed(__half());
    else typed(__nv_bfloat16());
}

template <typename Args>
void check_args(const Args& a) {
    require(a.rows >= 0 && a.rows <= kMaxSize, "rows out of range");
    require(a.groups >= 1 && a.groups <= kMaxGroups, "groups out of range: 1 to 1024");
    require(a.inputs >= 1 && a.inputs <= kMaxSize && a.outputs >= 1 && a.outputs <= kMaxSize / 2,
            "inputs or outputs out of range");
    require(a.outputs * 2 <= kMaxSize / a.groups, "groups times outputs out of range");
    require(a.activation == RUNE_ACT_NONE || a.activation == RUNE_ACT_TANH ||
                a.activation == RUNE_ACT_SILU || a.activation == RUNE_ACT_GELU,
            "unknown activation");
    require(!a.gated || a.activation != RUNE_ACT_NONE, "a gated layer needs an activation");
    require(a.dtype == RUNE_F16 || a.dtype == RUNE_BF16,
            "a grouped layer takes float16 or bfloat16 operands");
    require(a.rows == 0 || (a.x && a.weight && a.offsets), "null argument");
    require_aligned({a.x, a.weight, a.bias}, 2);
    require_aligned({a.offsets}, 4);
    require(aligned(a.saved, 16), "saved is not 16-byte aligned");
}

template <typename Args>
Scratch carve(const Args& a, int64_t need) {
    require(need == 0 || (a.workspace && aligned(a.workspace, 256) && a.workspace_bytes >= need),
            "the workspace is too small or not 256-byte aligned");
    return {need ? static_cast<char*>(a.workspace) : reinterpret_cast<char*>(256)};
}

}  // namespace
}  // namespace ops
}  // namespace rune

using namespace rune;
using namespace rune::ops;

extern "C" {

int rune_grouped_linear_workspace(const rune_grouped_linear_args* args, int64_t* bytes) {
    if (!args || !bytes) {
        set_error("null argument");
        return RUNE_ERR_INVALID;
    }
    const rune_grouped_linear_args a = *args;
    return guarded(a.device, [&] {
        check_args(a);
        Scratch ws{nullptr};
        if (a.rows > 0) forward(a, ws, nullptr);
        *bytes = ws.off;
    });
}

int rune_grouped_linear(const rune_grouped_linear_args* args, void* stream_) {
    if (!args) {
        set_error("null argument");
        return RUNE_ERR_INVALID;
    }
    const rune_grouped_linear_args a = *args;
    auto stream = static_cast<cudaStream_t>(stream_);
    return guarded(a.device, [&] {
        check_args(a);
        require_aligned({a.y}, 2);
        check_waits(a.device);
        if (a.rows == 0) return;
        require(a.y, "null argument");
        Scratch need{nullptr};
        forward(a, need, stream);
        if (need.off > 0 && !a.workspace)
            throw Error(RUNE_ERR_RETRY, "the call needs a workspace");
        Scratch ws = carve(a, need.off);
        forward(a, ws, stream);
        RUNE_LAUNCH_CHECK();
    });
}

int rune_grouped_linear_backward_workspace(const rune_grouped_linear_grad_args* args,
                                           int64_t* bytes) {
    if (!args || !bytes) {
        set_error("null argument");
        return RUNE_ERR_INVALID;
    }
    const rune_grouped_linear_grad_args a = *args;
    return guarded(a.device, [&] {
        check_args(a);
        Scratch ws{nullptr};
        if (a.rows > 0) backward(a, ws, nullptr);
        *bytes = ws.off;
    });
}

int rune_grouped_linear_backward(const rune_grouped_linear_grad_args* args, void* stream_) {
    if (!args) {
        set_error("null argument");
        return RUNE_ERR_INVALID;
    }
    const rune_grouped_linear_grad_args a = *args;
    auto stream = static_cast<cudaStream_t>(stream_);
    return guarded(a.device, [&] {
        check_args(a);
        require_aligned({a.dy, a.dx, a.dweight, a.dbias}, 2);
        check_waits(a.device);
        const int64_t n_all = a.gated ? 2 * a.outputs : a.outputs;
        if (a.rows == 0) {
            if (a.dweight)
                RUNE_CUDA_TRY(cudaMemsetAsync(
                    a.dweight, 0, (size_t)(a.groups * n_all * a.inputs * 2), stream));
            if (a.dbias)
                RUNE_CUDA_TRY(
                    cudaMemsetAsync(a.dbias, 0, (size_t)(a.groups * n_all * 2), stream));
            return;
        }
        require(a.dy, "null argument");
        Scratch need{nullptr};
        backward(a, need, stream);
        Scratch ws = carve(a, need.off);
        backward(a, ws, stream);
        RUNE_LAUNCH_CHECK();
    });
}

}  // extern "C"
