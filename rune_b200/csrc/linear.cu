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

#include "linear.cuh"

namespace rune {
namespace ops {

namespace {

enum Mode {
    kForward,    // y = act(acc + bias) + residual, z saved on request
    kGated,      // y = act(gate) * up; the tile's columns are half gate, half up
    kGrad,       // dz = dy act'(acc + bias), column sums of dz
    kGatedGrad,  // d gate = dy up act'(gate), d up = dy act(gate), column sums
    kPartial     // float32 sums of one range of k
};

constexpr int kBM = 128;
constexpr int kEpiWarps = 16, kTmaWarp = 16, kMmaWarp = 17;
constexpr int kThreads = 32 * 18;
constexpr uint32_t kAStage = kBM * kLineBytes;  // 16 KB
constexpr uint32_t kRowBytes = 64;               // of a warp's buffer: 32 16-bit or 16 float values
constexpr uint32_t kWarpBuf = 32 * kRowBytes;    // 2 KB
constexpr int kMaxStages = 8;
constexpr uint32_t kSmemMax = 227 * 1024;

// Exact quotient of n < 2^31 by a divisor fixed for the launch: n * mul >> shift.
struct Divisor {
    unsigned by, mul, shift;
    __device__ __forceinline__ unsigned quotient(unsigned n) const {
        return (unsigned)(((uint64_t)n * mul) >> shift);
    }
};
Divisor make_divisor(unsigned by) {
    // with 2^L >= by, mul = ceil(2^(31 + L) / by) < 2^32 errs by less than n / 2^31 of a unit
    unsigned l = 0;
    while ((1ull << l) < by) ++l;
    return {by, (unsigned)(((1ull << (31 + l)) + by - 1) / by), 31 + l};
}

struct TileParams {
    int64_t m, n;           // rows and columns of the output (gated: columns of y)
    int64_t ld_out, ld_in;
    int64_t ld_z, ld_part;  // of z: rows, and within a row the parts (gate, up)
    int kblocks, kb_per_split, splits;
    int tiles_m, tiles_n, bn, stages;
    Divisor by_tiles, by_group, by_last;  // tile_of's: all tiles, a group's, the last group's rows
    int a_mn, b_mn, act;
    int tma_out, vec_in, vec_bias;  // rows on 16 bytes: copies by TMA, 16-byte accesses
    uint32_t idesc;
    void* out;
    const void* in;         // residual, or dy
    const void* bias;
    const float* x_scale;
    const float* w_scale;
    float* z;               // saved z, or the partial sums
    float* colsum;          // [tiles_m * 4][n or 2n]
    unsigned* flag;
    unsigned polls;         // bound of every wait
};

struct TileShared {
    unsigned long long full[kMaxStages], empty[kMaxStages];
    unsigned long long acc_full[2], acc_empty[2], drained;
    uint32_t tmem;
    int fail;
    int issued;             // stages whose copies were issued
};

// buffers of kWarpBuf per epilogue warp, and all shared memory beside the ring
template <int MODE>
constexpr uint32_t kWarpBufs = MODE == kGatedGrad ? 2 : 1;
template <int MODE>
constexpr uint32_t kFixedSmem =
    kEpiWarps * kWarpBufs<MODE> * kWarpBuf + (uint32_t)((sizeof(TileShared) + 127) / 128 * 128);

struct Tile {
    int mt, nt, split;
};

// Tiles in groups of 16 tile rows, column by column, so that the blocks at work share a few
// lines of both operands in L2; the ranges of k of one tile come last.
constexpr unsigned kGroup = 16;
__device__ __forceinline__ Tile tile_of(const TileParams& p, unsigned w) {
    Tile t{0, 0, 0};
    if (p.splits > 1) {
        t.split = p.by_tiles.quotient(w);
        w -= t.split * p.by_tiles.by;
    }
    const unsigned g = p.by_group.quotient(w), in = w - g * p.by_group.by;
    const unsigned left = p.tiles_m - g * kGroup, rows = min(kGroup, left);
    t.nt = left >= kGroup ? in / kGroup : p.by_last.quotient(in);
    t.mt = g * kGroup + (in - t.nt * rows);
    return t;
}

// ---- a warp's 32 rows x 32 columns of 16-bit values between global memory and its buffer.
// Rows are four pieces of 16 bytes, piece c of row r at c ^ (r / 2 & 3), so that both the row-wise
// accesses of the lanes and the coalesced ones (lane l: piece l & 3 of row 8 i + l / 4) spread
// over the banks.
struct Stage {
    uint32_t row, swizzle;  // of the lane's own row
    uint32_t coalesced;     // the lane's piece of rows 0 .. 7
    uint32_t base;
    int lane;
    __device__ __forceinline__ Stage(uint32_t buf, int l) : base(buf), lane(l) {
        row = buf + l * kRowBytes;
        swizzle = ((l >> 1) & 3) << 4;
        coalesced = buf + (l >> 2) * kRowBytes + (((l & 3) ^ ((l >> 3) & 3)) << 4);
    }
    __device__ __forceinline__ uint32_t own(int c) const {  // piece c of the lane's row
        return row + (uint32_t(c << 4) ^ swizzle);
    }
    __device__ __forceinline__ uint32_t turn(int i) const {  // coalesced, row 8 i + lane / 4
        return coalesced + i * 8 * kRowBytes;
    }
    __device__ __forceinline__ uint32_t at(int r, int byte) const {
        return base + r * kRowBytes + ((byte & ~15) ^ (((r >> 1) & 3) << 4)) + (byte & 15);
    }
};
__device__ __forceinline__ void put16(uint32_t addr, uint4 v) {
    asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "r"(v.x), "r"(v.y),
                 "r"(v.z), "r"(v.w)
                 : "memory");
}
__device__ __forceinline__ uint4 get16(uint32_t addr) {
    uint4 v;
    asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];"
                 : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
                 : "r"(addr)
                 : "memory");
    return v;
}
__device__ __forceinline__ void put_half(uint32_t addr, uint16_t v) {
    asm volatile("st.shared.u16 [%0], %1;" ::"r"(addr), "h"(v) : "memory");
}
__device__ __forceinline__ uint16_t get_half(uint32_t addr) {
    uint16_t v;
    asm volatile("ld.shared.u16 %0, [%1];" : "=h"(v) : "r"(addr) : "memory");
    return v;
}
// rows x cols (of 32 x 32, zeros beyond) from src into the buffer
template <typename T>
__device__ __forceinline__ void load_rows(const Stage& st, const T* src, int64_t ld, int rows,
                                          int64_t cols, bool vec) {
    if (vec) {
        const int r0 = st.lane >> 2, c = (st.lane & 3) * 8;
        const T* p = src + r0 * ld + c;
        const bool in = c < cols;
        uint4 v[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            v[i] = make_uint4(0, 0, 0, 0);
            if (in && r0 + 8 * i < rows)
                v[i] = *reinterpret_cast<const uint4*>(p + i * 8 * ld);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) put16(st.turn(i), v[i]);
    } else {
#pragma unroll 8
        for (int r = 0; r < 32; ++r) {
            uint16_t v = 0;
            if (r < rows && st.lane < cols)
                v = reinterpret_cast<const uint16_t*>(src)[(int64_t)r * ld + st.lane];
            put_half(st.at(r, st.lane * 2), v);
        }
    }
}

// sums over the warp's rows of 16 columns that each lane holds of its own row, before they are
// rounded. Every step halves the columns that a lane keeps; then two lanes have one column.
__device__ __forceinline__ void column_sums(const Two (&z)[8], int lane, int64_t cols,
                                            float* sums) {
    float a[16];
#pragma unroll
    for (int j = 0; j < 8; ++j) split(z[j], a[2 * j], a[2 * j + 1]);
    int column = 0;
#pragma unroll
    for (int n = 8; n > 0; n >>= 1) {
        const bool upper = lane & (2 * n);
#pragma unroll
        for (int j = 0; j < n; ++j) {
            const float give = upper ? a[j] : a[n + j];
            a[j] = (upper ? a[n + j] : a[j]) + __shfl_xor_sync(0xffffffffu, give, 2 * n);
        }
        column += upper ? n : 0;
    }
    a[0] += __shfl_xor_sync(0xffffffffu, a[0], 1);
    if (!(lane & 1) && column < cols) sums[column] = a[0];
}

// the buffer's rows x cols to dst, value by value: outputs whose rows are off 16 bytes
template <typename T>
__device__ __forceinline__ void store_rows(const Stage& st, T* dst, int64_t ld, int rows,
                                           int64_t cols) {
#pragma unroll 8
    for (int r = 0; r < 32; ++r) {
        const uint16_t h = get_half(st.at(r, st.lane * 2));
        if (r < rows && st.lane < cols)
            reinterpret_cast<uint16_t*>(dst)[(int64_t)r * ld + st.lane] = h;
    }
}

// a warp's 32 rows x 16 columns of float32, each lane its row, through the buffer to memory whose
// rows are padded to 16 bytes
__device__ __forceinline__ void store_rows32(const Stage& st, const float (&v)[16], float* dst,
                                             int64_t ld, int rows, int64_t cols) {
    __syncwarp();
#pragma unroll
    for (int c = 0; c < 4; ++c)
        put16(st.own(c), make_uint4(__float_as_uint(v[4 * c]), __float_as_uint(v[4 * c + 1]),
                                    __float_as_uint(v[4 * c + 2]), __float_as_uint(v[4 * c + 3])));
    __syncwarp();
    const int r0 = st.lane >> 2, c = (st.lane & 3) * 4;
    float* p = dst + r0 * ld + c;
#pragma unroll
    for (int i = 0; i < 4; ++i)
        if (c < cols && r0 + 8 * i < rows)
            *reinterpret_cast<uint4*>(p + i * 8 * ld) = get16(st.turn(i));
    __syncwarp();
}

// Bias of 16 columns from `col` (left of them inside), read by all lanes at once and before the
// accumulator, so that the two waits overlap.
template <typename T>
struct Bias {
    uint32_t w[8];
    __device__ __forceinline__ void load(const TileParams& p, int64_t col, int64_t left) {
        const T* bias = static_cast<const T*>(p.bias) + col;
        if (!p.bias) return;
        if (p.vec_bias) {
#pragma unroll
            for (int g = 0; g < 2; ++g) {
                uint4 q = make_uint4(0, 0, 0, 0);
                if (g * 8 < left) q = reinterpret_cast<const uint4*>(bias)[g];
                w[4 * g] = q.x, w[4 * g + 1] = q.y, w[4 * g + 2] = q.z, w[4 * g + 3] = q.w;
            }
        } else {
#pragma unroll
            for (int j = 0; j < 8; ++j)
                w[j] = pack2<T>(2 * j < left ? to_float(bias[2 * j]) : 0.0f,
                                2 * j + 1 < left ? to_float(bias[2 * j + 1]) : 0.0f);
        }
    }
};

// acc -> z: scales of e4m3 operands and bias
template <typename T, bool FP8>
__device__ __forceinline__ void finish_z(const float (&v)[16], Two (&z)[8], const Bias<T>& bias,
                                         const TileParams& p, int64_t col, int64_t left,
                                         float x_scale) {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        z[j] = two(v[2 * j], v[2 * j + 1]);
        if constexpr (FP8) {
            const float s0 = 2 * j < left ? p.w_scale[col + 2 * j] : 0.0f;
            const float s1 = 2 * j + 1 < left ? p.w_scale[col + 2 * j + 1] : 0.0f;
            z[j] = z[j] * (two(x_scale) * two(s0, s1));
        }
        if (p.bias) {
            const float2 f = unpack2<T>(bias.w[j]);
            z[j] = z[j] + two(f.x, f.y);
        }
    }
}

// 16 values of a lane's row to and from pieces 2 half, 2 half + 1 of its line
template <typename T>
__device__ __forceinline__ void put_row(const Stage& st, int half, const Two (&v)[8]) {
    uint32_t w[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        float a, b;
        split(v[j], a, b);
        w[j] = pack2<T>(a, b);
    }
#pragma unroll
    for (int c = 0; c < 2; ++c)
        put16(st.own(half * 2 + c), make_uint4(w[4 * c], w[4 * c + 1], w[4 * c + 2], w[4 * c + 3]));
}

template <typename T>
__device__ __forceinline__ void get_row(const Stage& st, int half, Two (&v)[8]) {
#pragma unroll
    for (int c = 0; c < 2; ++c) {
        const uint4 q = get16(st.own(half * 2 + c));
        const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const float2 f = unpack2<T>(w[j]);
            v[4 * c + j] = two(f.x, f.y);
        }
    }
}

// One warp's part of a finished tile: 32 rows (a warp reads the quarter of TMEM's lanes that its
// number gives) and every fourth group of 32 columns, the rest being its three partners'. `release` is
// called when the accumulator has been read. `wait` comes back when the accumulator is complete;
// what the first group reads from memory is asked for before.
template <int MODE, typename T, bool FP8, typename Wait, typename Release>
__device__ __forceinline__ void epilogue(const TileParams& p, const Tile& t, uint32_t acc,
                                         const Stage& st, const Stage& st2, int warp,
                                         const CUtensorMap* out_map, const CUtensorMap* out2_map,
                                         Wait&& wait, Release&& release) {
    const int quarter = warp & 3, share = warp >> 2;
    const int row0 = t.mt * kBM + quarter * 32;
    const int rows = (int)max((int64_t)0, min((int64_t)32, p.m - row0));
    constexpr bool kGate = MODE == kGated || MODE == kGatedGrad;
    const int width = kGate ? p.bn / 2 : p.bn;  // output columns of the tile
    const int64_t col0 = (int64_t)t.nt * width;
    const int end = (int)min((int64_t)width, p.n - col0);
    const int lane = st.lane;
    constexpr bool kReads = MODE == kGrad || MODE == kGatedGrad;
    const bool reads = kReads || (MODE == kForward && p.in);
    auto read_in = [&](int c) {  // residual or dy of the group
        load_rows(st, static_cast<const T*>(p.in) + (int64_t)row0 * p.ld_in + col0 + c, p.ld_in,
                  rows, end - c, p.vec_in);
    };
    // the buffers are free again when the last copy out has read them
    auto reuse = [&] {
        if (lane == 0) bulk_store_read();
        __syncwarp();
    };
    const bool ahead = reads && !(MODE == kForward && p.z) && share * 32 < end;
    if (ahead) {
        reuse();
        read_in(share * 32);
    }
    if (!wait()) return;
    if constexpr (MODE == kPartial) {
        for (int c = share * 16; c < end; c += 64) {
            float v[16];
            tc::tmem_ld16(acc + c, v);
            store_rows32(st, v, p.z + ((int64_t)t.split * p.m + row0) * p.ld_z + col0 + c,
                         p.ld_z, rows, end - c);
        }
        release();
        return;
    }
    float* sums = nullptr;  // this warp's row of the parts of dbias
    if (kReads && p.colsum)
        sums = p.colsum + ((int64_t)t.mt * 4 + quarter) * (kGate ? 2 * p.n : p.n);
    const float xs = FP8 && lane < rows ? p.x_scale[row0 + lane] : 0.0f;
    for (int c = share * 32; c < end; c += 128) {
        const int64_t col = col0 + c, left = p.n - col;
        if constexpr (MODE == kForward || MODE == kGated) {
            if (p.z) {  // the pre-activations, in float32
                reuse();
                for (int part = 0; part < (kGate ? 2 : 1); ++part) {
                    for (int half = 0; half < 2 && half * 16 < left; ++half) {
                        const int64_t at = part * p.n + col + half * 16;
                        float v[16];
                        Two z[8];
                        Bias<T> bias;
                        bias.load(p, at, left - half * 16);
                        tc::tmem_ld16(acc + c + part * width + half * 16, v);
                        finish_z<T, FP8>(v, z, bias, p, at, left - half * 16, xs);
#pragma unroll
                        for (int j = 0; j < 8; ++j) split(z[j], v[2 * j], v[2 * j + 1]);
                        store_rows32(st, v,
                                     p.z + (int64_t)row0 * p.ld_z + part * p.ld_part + col +
                                         half * 16,
                                     p.ld_z, rows, left - half * 16);
                    }
                }
            }
        }
        if (!ahead || c != share * 32) {
            reuse();
            if (reads) read_in(c);
        }
        __syncwarp();
#pragma unroll 1
        for (int half = 0; half < 2; ++half) {
            const int at = c + half * 16;
            const int64_t zcol = col + half * 16, zleft = left - half * 16;
            Two z[8], u[8];
            {
                float v[16], w[16];
                Bias<T> bias, bias_up;
                bias.load(p, zcol, zleft);
                if constexpr (kGate) {
                    bias_up.load(p, p.n + zcol, zleft);
                    tmem_ld16x2(acc + at, acc + at + width, v, w);
                } else {
                    tc::tmem_ld16(acc + at, v);
                }
                if (half == 1 && c + 128 >= end) release();
                finish_z<T, FP8>(v, z, bias, p, zcol, zleft, xs);
                if constexpr (kGate) finish_z<T, FP8>(w, u, bias_up, p, p.n + zcol, zleft, xs);
            }
            if constexpr (MODE == kForward) {
                with_activation(p.act, [&](auto a) {
#pragma unroll
                    for (int j = 0; j < 8; ++j) z[j] = act_value<decltype(a)::value>(z[j]);
                });
                if (p.in) {
                    get_row<T>(st, half, u);
#pragma unroll
                    for (int j = 0; j < 8; ++j) z[j] = z[j] + u[j];
                }
            } else if constexpr (MODE == kGrad) {
                get_row<T>(st, half, u);
                with_activation(p.act, [&](auto a) {
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        Two y, da;
                        act_both<decltype(a)::value>(z[j], y, da);
                        z[j] = u[j] * da;
                    }
                });
            } else if constexpr (MODE == kGated) {
                with_activation(p.act, [&](auto a) {
#pragma unroll
                    for (int j = 0; j < 8; ++j)
                        z[j] = act_value<decltype(a)::value>(z[j]) * u[j];
                });
            } else {
                Two d[8];
                get_row<T>(st, half, d);
                with_activation(p.act, [&](auto a) {
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        Two y, da;
                        act_both<decltype(a)::value>(z[j], y, da);
                        z[j] = d[j] * u[j] * da;
                        u[j] = d[j] * y;
                    }
                });
                put_row<T>(st2, half, u);
            }
            if constexpr (kReads) {
                if (sums) {
                    if (lane >= rows) {  // beyond the last row: nothing, whatever the bias is
#pragma unroll
                        for (int j = 0; j < 8; ++j) z[j] = u[j] = two(0.0f);
                    }
                    column_sums(z, lane, zleft, sums + zcol);
                    if constexpr (kGate) column_sums(u, lane, zleft, sums + p.n + zcol);
                }
            }
            put_row<T>(st, half, z);
        }
        if (p.tma_out) tc::fence_async_smem();
        __syncwarp();
        if (p.tma_out) {
            if (lane == 0 && rows > 0) {
                bulk_store(out_map, st.base, (int)col, row0);
                if constexpr (MODE == kGatedGrad) bulk_store(out2_map, st2.base, (int)col, row0);
                bulk_store_commit();
            }
        } else {
            T* out = static_cast<T*>(p.out) + (int64_t)row0 * p.ld_out + col;
            store_rows<T>(st, out, p.ld_out, rows, left);
            if constexpr (MODE == kGatedGrad)
                store_rows<T>(st2, out + p.n, p.ld_out, rows, left);
        }
        __syncwarp();
    }
    if (share * 32 >= end) release();  // no columns here
}

// After a wait gave up: lets what is in flight land (bounded) before the blocks' memory goes. The
// copies of both blocks count on the even one's barriers; a stage that only one of them had filled
// when the other gave up gets the other's part from here. Not inlined: among the kernels' own code
// it cost the gated forward 3 % (110592 x 256 -> 512 65.6 against 63.7 us).
template <bool PAIR>
__device__ __noinline__ void drain(TileShared* sh, unsigned* flag, int stages,
                                   uint32_t stage_bytes) {
    using namespace tc;
    const int rank = PAIR ? (int)cluster_rank() : 0, warp = threadIdx.x >> 5;
    const volatile int* fail = &sh->fail;
    if (threadIdx.x == 0 && *fail) atomicExch_system(flag, (unsigned)*fail);
    if (threadIdx.x == 0 && rank == 0) {
        const int mine = sh->issued;
        const int theirs = PAIR ? (int)peer_word(peer_address(smem_u32(&sh->issued), 1)) : mine;
        const int issued = max(mine, theirs);
        for (int i = max(0, issued - stages); i < issued; ++i) {
            const uint32_t bar = smem_u32(&sh->full[i % stages]);
            if (i >= theirs) mbar_complete_tx(bar, stage_bytes);
            if (i >= mine) mbar_expect_tx(bar, stage_bytes);
            mbar_wait(bar, (i / stages) & 1);
        }
    }
    __syncwarp();
    // the products, and on the odd block the arrivals that their completion sends there
    if (warp == kMmaWarp) {
        if (rank == 0 && elect_one()) {
            if constexpr (PAIR) mma_commit_pair(smem_u32(&sh->drained));
            else mma_commit(smem_u32(&sh->drained));
        }
        __syncwarp();
        mbar_wait(smem_u32(&sh->drained), 0);
    }
    __syncwarp();
}

// PAIR: two blocks of a cluster (the two SMs of a TPC) work on one tile of 256 rows. Each holds its
// 128 rows of A and of the accumulator and half of the tile's B, which the tensor cores of both
// read: half the shared-memory traffic and half the copies for B. The even block issues the
// products; copies of both count on its barriers, completed products on both blocks'.
template <int MODE, typename T, bool FP8, bool PAIR>
__global__ void __launch_bounds__(kThreads, 1)
k_tile(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b,
       const __grid_constant__ CUtensorMap map_o, const __grid_constant__ CUtensorMap map_o2,
       const TileParams p) {
    using namespace tc;
    extern __shared__ __align__(1024) unsigned char smem[];
    const int b_rows = PAIR ? p.bn / 2 : p.bn;  // of B in this block's stages
    const uint32_t stage_bytes = kAStage + (uint32_t)b_rows * kLineBytes;
    unsigned char* bufs = smem + (size_t)p.stages * stage_bytes;
    auto* sh = reinterpret_cast<TileShared*>(bufs + kEpiWarps * kWarpBufs<MODE> * kWarpBuf);
    const int tid = threadIdx.x, lane = tid & 31;
    const int warp = __shfl_sync(0xffffffffu, tid >> 5, 0);  // uniform, and known to be
    constexpr bool kGate = MODE == kGated || MODE == kGatedGrad;
    const unsigned tiles = (unsigned)p.tiles_m * p.tiles_n, work = tiles * p.splits;
    const int rank = PAIR ? (int)cluster_rank() : 0;
    const unsigned first = PAIR ? blockIdx.x >> 1 : blockIdx.x;
    const unsigned stride = PAIR ? gridDim.x >> 1 : gridDim.x;

    if (tid == 0) {
        for (int s = 0; s < p.stages; ++s) {
            mbar_init(smem_u32(&sh->full[s]), 1);
            mbar_init(smem_u32(&sh->empty[s]), 1);
        }
        for (int b = 0; b < 2; ++b) {
            mbar_init(smem_u32(&sh->acc_full[b]), 1);
            mbar_init(smem_u32(&sh->acc_empty[b]), kEpiWarps * (PAIR ? 2 : 1));
        }
        mbar_init(smem_u32(&sh->drained), 1);
        sh->fail = 0;
        sh->issued = 0;
        asm volatile("fence.mbarrier_init.release.cluster;");
    }
    if (warp == kTmaWarp && elect_one()) {
        prefetch_map(&map_a);
        prefetch_map(&map_b);
    }
    if (warp == kMmaWarp) {
        if constexpr (PAIR) tmem_alloc_pair(&sh->tmem, 512);
        else tmem_alloc(&sh->tmem, 512);
    }
    fence_before_sync();
    __syncwarp();
    if constexpr (PAIR) cluster_sync();
    else __syncthreads();
    fence_after_sync();
    const uint32_t tmem = __shfl_sync(0xffffffffu, sh->tmem, 0);
    volatile int* fail = &sh->fail;
    follow_on();

    if (warp == kTmaWarp) {
        // ---- TMA producer
        const bool one = elect_one();
        const int bw = kGate ? p.bn / 2 : p.bn;
        // barriers of the pair: the even block's
        const uint32_t full0 = PAIR ? peer_address(smem_u32(sh->full), 0) : smem_u32(sh->full);
        auto load = [&](uint32_t dst, const CUtensorMap* map, int x, int y, uint32_t bar) {
            if constexpr (PAIR) tma_load_pair(dst, map, x, y, bar);
            else tma_load(dst, map, x, y, bar);
        };
        int st = 0, issued = 0;
        uint32_t parity = 1;  // of the stage's last release; a fresh barrier passes for 1
        bool ok = true;
        for (unsigned w = first; w < work && ok; w += stride) {
            const Tile t = tile_of(p, w);
            const int kb0 = t.split * p.kb_per_split;
            const int kb1 = min(p.kblocks, kb0 + p.kb_per_split);
            const int m0 = (PAIR ? t.mt * 2 + rank : t.mt) * kBM;
            // first row of B here: a pair's blocks take halves of the tile, gate and up or not
            int n0 = t.nt * bw;
            if (PAIR && rank) n0 += kGate ? (int)p.n : b_rows;
            for (int kb = kb0; kb < kb1; ++kb) {
                ok = mbar_wait(smem_u32(&sh->empty[st]), parity, p.polls) && !*fail;
                if (!__all_sync(0xffffffffu, ok)) {
                    ok = false;
                    break;
                }
                const uint32_t bar = full0 + (uint32_t)st * 8;
                const uint32_t a = smem_u32(smem) + (uint32_t)st * stage_bytes, b = a + kAStage;
                if (one) {
                    if (!PAIR || rank == 0)
                        mbar_expect_tx(smem_u32(&sh->full[st]), (PAIR ? 2 : 1) * stage_bytes);
                    const int x = kb * (FP8 ? 128 : 64);
                    if (p.a_mn) {
                        load(a, &map_a, m0, kb * 64, bar);
                        load(a + kMnChunk, &map_a, m0 + 64, kb * 64, bar);
                    } else {
                        load(a, &map_a, x, m0, bar);
                    }
                    if (p.b_mn) {
                        for (int i = 0; i < b_rows / 64; ++i)
                            load(b + i * kMnChunk, &map_b, n0 + i * 64, kb * 64, bar);
                    } else {
                        load(b, &map_b, x, n0, bar);
                        if (kGate && !PAIR)
                            load(b + bw * kLineBytes, &map_b, x, (int)p.n + n0, bar);
                    }
                }
                __syncwarp();  // the other lanes' polling must not hold up the copies' issue
                ++issued;
                if (++st == p.stages) st = 0, parity ^= 1;
            }
        }
        // the last releases of every stage arrive here (a pair's from the even block) before this
        // block's memory may go
        for (int i = max(0, issued - p.stages); i < issued && ok; ++i) {
            ok = mbar_wait(smem_u32(&sh->empty[i % p.stages]), (i / p.stages) & 1, p.polls) && !*fail;
            ok = __all_sync(0xffffffffu, ok);
        }
        if (!ok && !*fail) *fail = 1;
        if (one) sh->issued = issued;
    } else if (warp == kMmaWarp && rank == 0) {
        // ---- MMA issuer. The whole warp runs the loop and one elected lane issues: control flow
        // and descriptors are uniform then, and stay in the uniform registers that the tensor
        // core instructions take (issued from a divergent thread they came too slowly).
        const bool one = elect_one();
        const uint64_t step_a = p.a_mn ? 2048 >> 4 : 32 >> 4;
        const uint64_t step_b = p.b_mn ? 2048 >> 4 : 32 >> 4;
        const uint64_t desc_a = operand_desc(smem_u32(smem), p.a_mn);
        const uint64_t desc_b = operand_desc(smem_u32(smem) + kAStage, p.b_mn);
        auto commit = [&](unsigned long long* bar) {
            if constexpr (PAIR) mma_commit_pair(smem_u32(bar));
            else mma_commit(smem_u32(bar));
        };
        int st = 0, buf = 0;
        uint32_t parity = 0, acc_parity = 1;
        bool ok = true;
        for (unsigned w = first; w < work && ok; w += stride) {
            const int split = p.splits > 1 ? (int)p.by_tiles.quotient(w) : 0;
            const int kb0 = split * p.kb_per_split;
            const int kb1 = min(p.kblocks, kb0 + p.kb_per_split);
            ok = mbar_wait(smem_u32(&sh->acc_empty[buf]), acc_parity, p.polls) && !*fail;
            if (!__all_sync(0xffffffffu, ok)) {
                if (!*fail) *fail = 2;
                ok = false;
                break;
            }
            fence_after_sync();
            const uint32_t acc = tmem + buf * 256;
            for (int kb = kb0; kb < kb1; ++kb) {
                ok = mbar_wait(smem_u32(&sh->full[st]), parity, p.polls) && !*fail;
                if (!__all_sync(0xffffffffu, ok)) {
                    ok = false;
                    break;
                }
                fence_after_sync();
                const uint64_t at = (uint64_t)((uint32_t)st * (stage_bytes >> 4));
                if (one) {
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        const bool more = kb > kb0 || k > 0;
                        mma<FP8, PAIR>(acc, desc_a + at + k * step_a, desc_b + at + k * step_b,
                                       p.idesc, more);
                    }
                    commit(&sh->empty[st]);
                }
                __syncwarp();
                if (++st == p.stages) st = 0, parity ^= 1;
            }
            if (one) commit(&sh->acc_full[buf]);
            __syncwarp();
            buf ^= 1;
            if (buf == 0) acc_parity ^= 1;
        }
        if (!ok && !*fail) *fail = 3;
        // and the last arrivals of the epilogues (both blocks')
        for (int i = 0; i < 2 && ok; ++i) {
            ok = mbar_wait(smem_u32(&sh->acc_empty[buf]), acc_parity, p.polls) && !*fail;
            ok = __all_sync(0xffffffffu, ok);
            if (!ok && !*fail) *fail = 2;
            buf ^= 1;
            if (buf == 0) acc_parity ^= 1;
        }
    } else if (warp < kEpiWarps) {
        // ---- epilogue
        int n_tile = 0;
        const uint32_t buf = smem_u32(bufs) + warp * kWarpBufs<MODE> * kWarpBuf;
        const Stage st(buf, lane), st2(buf + (kWarpBufs<MODE> - 1) * kWarpBuf, lane);
        const uint32_t quarter = (uint32_t)((warp & 3) * 32) << 16;
        bool ok = true;
        for (unsigned w = first; w < work && ok; w += stride, ++n_tile) {
            Tile t = tile_of(p, w);
            if (PAIR) t.mt = t.mt * 2 + rank;
            const int b = n_tile & 1, round = n_tile >> 1;
            epilogue<MODE, T, FP8>(
                p, t, tmem + b * 256 + quarter, st, st2, warp, &map_o, &map_o2,
                [&] {
                    ok = mbar_wait(smem_u32(&sh->acc_full[b]), round & 1, p.polls) && !*fail;
                    ok = __all_sync(0xffffffffu, ok);
                    fence_after_sync();
                    return ok;
                },
                [&] {
                    fence_before_sync();
                    __syncwarp();
                    if (lane == 0) {
                        if constexpr (PAIR)
                            mbar_arrive_peer(peer_address(smem_u32(&sh->acc_empty[b]), 0));
                        else
                            mbar_arrive(smem_u32(&sh->acc_empty[b]));
                    }
                    __syncwarp();
                });
        }
        if (lane == 0) bulk_store_read();  // the copies out have read the buffers
        if (!ok && !*fail) *fail = 4;
    }
    __syncwarp();
    if constexpr (PAIR) cluster_sync();
    else __syncthreads();
    bool failed = *fail;
    if constexpr (PAIR)
        failed = failed || peer_word(peer_address(smem_u32(&sh->fail), rank ^ 1)) != 0;
    if (failed) {
        drain<PAIR>(sh, p.flag, p.stages, stage_bytes);
    }
    fence_before_sync();
    if constexpr (PAIR) cluster_sync();
    else __syncthreads();
    if (warp == kMmaWarp) {
        fence_after_sync();
        if constexpr (PAIR) tmem_dealloc_pair(tmem, 512);
        else tmem_dealloc(tmem, 512);
    }
}

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
// A block works on strips of rows x kColumns columns: a thread has four columns and every fourth
// row of the strip, and the four threads of a column join their sums in order.
constexpr int kColumns = 256;

// rows of a strip: fewer where 64 would leave the GPU short of blocks
int strip_rows(int64_t m, int64_t n, int sms) {
    const int64_t across = (n + kColumns - 1) / kColumns;
    int rows = 64;
    while (rows > 8 && (m + rows - 1) / rows * across < 4 * sms) rows /= 2;
    return rows;
}

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

// dz from a saved float32 z and dy, and the sums of each strip's columns
template <bool GATED, typename T>
__global__ void __launch_bounds__(256, 5)
k_act_grad(int64_t m, int64_t n, const float* z, int64_t ld_part,
           const T* dy, int64_t ld_dy, bool wide_dy, T* dz,
           int64_t ld_dz, int act, int strip, float* sums) {
    follow_on();
    const int64_t col = (int64_t)blockIdx.x * kColumns + (threadIdx.x & 63) * 4;
    const int count = (int)max((int64_t)0, min((int64_t)4, n - col)), part = threadIdx.x >> 6;
    const int64_t nz = GATED ? 2 * n : n, ld_z = GATED ? 2 * ld_part : ld_part;
    const int64_t strips = (m + strip - 1) / strip;
    const bool whole = wide_dy && count == 4 && (!GATED || n % 4 == 0);
    for (int64_t k = blockIdx.y; k < strips; k += gridDim.y) {
        const int64_t r1 = min(m, (k + 1) * strip);
        float s0[4] = {}, s1[4] = {};
        auto rows = [&](auto a, auto whole_c) {
            constexpr int ACT = decltype(a)::value;
            constexpr bool WHOLE = decltype(whole_c)::value;  // no branch among the loads
#pragma unroll 2
            for (int64_t r = k * strip + part; r < r1; r += 4) {
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
            join4(s0, sums + k * nz + col, count);
            if (GATED) join4(s1, sums + k * nz + n + col, count);
        }
    }
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
    const int64_t pieces = ld_dst / 16;
    const uint8_t* const end = src + (rows - 1) * ld + bytes;
    const int64_t piece = (int64_t)blockIdx.x * 32 + threadIdx.x, at = piece * 16;
    if (piece >= pieces) return;
    for (int64_t r = (int64_t)blockIdx.y * 8 + threadIdx.y; r < rows; r += (int64_t)gridDim.y * 8) {
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
// Scratch carved from the caller's workspace; with a null base it only adds up the bytes.
struct Scratch {
    char* base;
    int64_t off = 0;
    template <typename T>
    T* take(int64_t n) {
        char* p = base ? base + off : nullptr;
        off += (n * (int64_t)sizeof(T) + 255) / 256 * 256;
        return reinterpret_cast<T*>(p);
    }
    bool sizing() const { return base == nullptr; }
};

struct Plan {
    int bn, splits, kb_per_split, stages;
    bool pair;
};

// Cycles that a k-block of 64 takes (measured on B200 at sizes that fill it): the tensor cores'
// 2 cycles a column for the widest tile of a pair, more for the others, which read more shared
// memory for a product.
double block_cycles(bool pair, int bn) {
    return pair ? (bn == 256 ? 520.0 : 370.0) : bn == 256 ? 660.0 : bn == 128 ? 400.0 : 300.0;
}

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
    const uint32_t stage =
        kAStage + (uint32_t)(best.pair ? best.bn / 2 : best.bn) * kLineBytes;
    best.stages = (int)std::min<uint32_t>(kMaxStages, (kSmemMax - fixed) / stage);
    return best;
}

CUtensorMap make_out_map(const void* p, int64_t rows, int64_t cols, int64_t ld);

template <int MODE, typename T, bool FP8, bool PAIR>
void launch_tile(const CUtensorMap& a, const CUtensorMap& b, TileParams p, int sms, int device,
                 cudaStream_t stream) {
    CUtensorMap o = a, o2 = a;  // unused unless the output goes by TMA
    if (MODE != kPartial && p.tma_out) {
        o = make_out_map(p.out, p.m, p.n, p.ld_out);
        if (MODE == kGatedGrad)
            o2 = make_out_map(static_cast<T*>(p.out) + p.n, p.m, p.n, p.ld_out);
    }
    static std::atomic<uint64_t> allowed{0};  // devices whose limit is raised
    if (device >= 64 || !(allowed.load(std::memory_order_relaxed) >> device & 1)) {
        RUNE_CUDA_TRY(cudaFuncSetAttribute(k_tile<MODE, T, FP8, PAIR>,
                                           cudaFuncAttributeMaxDynamicSharedMemorySize,
                                           (int)kSmemMax));
        if (device < 64) allowed.fetch_or(uint64_t(1) << device, std::memory_order_relaxed);
    }
    const int64_t work = (int64_t)p.tiles_m * p.tiles_n * p.splits;
    require(work < (1LL << 31) - 1024, "too many tiles");
    p.by_tiles = make_divisor((unsigned)p.tiles_m * p.tiles_n);
    p.by_group = make_divisor(kGroup * p.tiles_n);
    p.by_last = make_divisor(std::max(1u, (unsigned)p.tiles_m % kGroup));
    const int b_rows = PAIR ? p.bn / 2 : p.bn;
    const unsigned grid = PAIR ? 2 * (unsigned)std::min<int64_t>(work, sms / 2)
                               : (unsigned)std::min<int64_t>(work, sms);
    const size_t smem = (size_t)p.stages * (kAStage + (size_t)b_rows * kLineBytes) + kFixedSmem<MODE>;
    launch(k_tile<MODE, T, FP8, PAIR>, grid, kThreads, smem, PAIR ? 2 : 0, stream, a, b, o, o2, p);
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

int64_t pad16(int64_t cols, int elem_bytes) {
    const int64_t v = 16 / elem_bytes;
    return (cols + v - 1) / v * v;
}

void pad_rows(const void* src, int64_t rows, int64_t bytes, int64_t ld, void* dst, int64_t ld_dst,
              cudaStream_t stream) {
    const dim3 grid((unsigned)((ld_dst / 16 + 31) / 32),
                    (unsigned)std::min<int64_t>((rows + 7) / 8, 65535));
    launch(k_pack, grid, dim3(32, 8), 0, 0, stream, static_cast<const uint8_t*>(src), rows, bytes,
           ld, static_cast<uint8_t*>(dst), ld_dst);
}

// the operand itself, or its padded copy in the scratch
Matrix readable(Matrix m, int elem_bytes, Scratch& ws, cudaStream_t stream) {
    if (m.rows == 1) m.ld = pad16(m.cols, elem_bytes);  // no second line to reach
    if (tma_ready(m, elem_bytes)) return m;
    Matrix d = m;
    d.ld = pad16(m.cols, elem_bytes);
    void* to = ws.take<char>(m.rows * d.ld * elem_bytes);
    d.p = to;
    if (ws.sizing()) {
        d.p = reinterpret_cast<const void*>(256);  // any aligned address: only sizes are asked
        return d;
    }
    pad_rows(m.p, m.rows, m.cols * elem_bytes, m.ld * elem_bytes, to, d.ld * elem_bytes, stream);
    return d;
}

bool wide16(const void* p, int64_t ld, int64_t cols) {
    return aligned(p, 16) && ld % 8 == 0 && cols % 8 == 0;
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
        dz.ld = pad16(n_all, 2);
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

namespace {

// 32 x 32 boxes of a 16-bit output with the 64-byte swizzle, which is the buffers' own
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

}  // namespace

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
