// The tile kernel of the tensor-core products, D[m, n] = sum_k A[m, k] B[n, k]: one product (linear.cu),
// products by group of rows (grouped.cu), stacks of products (orthogonal.cu). What it does and
// measures stands with those; the kinds differ in the tiles' order, the maps and the outputs' ends,
// at compile time.
#pragma once

#include <algorithm>
#include <atomic>

#include "linear.cuh"

namespace rune {
namespace ops {

namespace {

enum Mode {
    kForward,    // y = act(acc + bias) + residual, z saved on request
    kGated,      // y = act(gate) * up; the tile's columns are half gate, half up
    kGrad,       // dz = dy act'(acc + bias), column sums of dz
    kGatedGrad,  // d gate = dy up act'(gate), d up = dy act(gate), column sums
    kPlain,      // y = acc: weight gradients and dx, whose epilogue bounds short contractions
    kPartial,    // float32 sums of one range of k
    kUpdate      // alpha acc + beta in; of a symmetric product the tiles below the diagonal, twice
};

// What the tiles cover:
enum Kind {
    kWhole,        // one product
    kRowGroups,    // the rows of A by group, each with its own matrix B (and bias)
    kRowsAcross,   // the same turned round: the group's matrix is A, its rows are B
    kDepthGroups,  // the contraction by group: a product of its own for the rows of each
    kDepthRanges,  // the same in parts: the k-blocks of all groups in equal ranges
    kBatch         // a stack of products
};
__host__ __device__ constexpr bool by_depth(int kind) {
    return kind == kDepthGroups || kind == kDepthRanges;
}

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
    // groups: row g of `offsets` to row g + 1 are group g's, [0, m_all) holds all of them
    const int32_t* offsets;
    int64_t m_all, bias_step;
    int groups, zero_tail;  // zero_tail: rows of the output behind the last group are cleared
    int ranges;                     // kDepthRanges: planned
    // batches, and kUpdate
    int64_t in_step, out_step;
    float alpha, beta;
    int symmetric;
};

struct TileShared {
    unsigned long long full[kMaxStages], empty[kMaxStages];
    unsigned bytes[kMaxStages];  // that this block's copies into the stage bring
    unsigned long long acc_full[2], acc_empty[2], drained;
    uint32_t tmem;
    int fail;
    int issued;             // stages whose copies were issued
};

// buffers of kWarpBuf per epilogue warp, and all shared memory beside the ring
template <int MODE>
constexpr uint32_t kWarpBufs = MODE == kGatedGrad || MODE == kUpdate ? 2 : 1;
template <int MODE>
constexpr uint32_t kFixedSmem =
    kEpiWarps * kWarpBufs<MODE> * kWarpBuf + (uint32_t)((sizeof(TileShared) + 127) / 128 * 128);

struct Tile {
    int mt, nt;
    int split;          // range of k; kDepthRanges: the part that it leaves
    int z;              // group, or product of the batch
    int row0, row_end;  // of the block's rows of the output: the first, and where they end
    bool empty;         // nothing to add up
};

// Tiles in groups of 16 tile rows, column by column, so that the blocks at work share a few
// lines of both operands in L2; the ranges of k of one tile come last.
constexpr unsigned kGroup = 16;
__device__ __forceinline__ Tile tile_of(const TileParams& p, unsigned w) {
    Tile t{0, 0, 0, 0, 0, 0, false};
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

// rows of a kRowsAcross tile as the tensor core's N: halves of sixteens
__device__ __forceinline__ int rows_across(const Tile& t) {
    return min(2 * kBM, (t.row_end - t.row0 + 31) / 32 * 32);
}

// A value that all lanes of a converged warp have, in a uniform register, where a reduction leaves
// it: what comes from shared memory would stay in every lane's registers, and the epilogues have none
// left (gated 221184 x 256 -> 2 x 512, dz: 330 us with 124 bytes spilled).
__device__ __forceinline__ int uniform(int v) { return (int)__reduce_or_sync(0xffffffffu, (unsigned)v); }

// Lines of `high` rows that groups with offsets in order can fill: each that has rows ends inside one.
__host__ __device__ constexpr int64_t most_lines(int64_t rows, int64_t groups, int high) {
    return rows / high + (rows < groups ? rows : groups);
}

// Place of the lines that hold the last rows of group g (kDepthGroups, kDepthRanges): of groups that have
// rows, with offsets in order, both g and the first row grow, so no two have one place; and there are no
// more places than groups, or rows.
__device__ __forceinline__ int tail_place(int g, int first) { return min(g, first); }

// The tiles of one launch in the order in which a block (or pair) takes them, and the range of k of
// each. Of groups, whose sizes only the GPU knows, a table in shared memory: rows[g], the groups'
// first rows, and lines[g], before group g the number of lines of tiles (by rows) or of k-blocks
// (kDepthRanges).
//   kRowsAcross    tiles of 256 outputs and up to 256 of a group's rows, rounded up to 32: a line's
//                  cost goes with its rows, where kRowGroups' last line of a group costs a whole
//                  one.
//   kDepthRanges   the k-blocks of all groups, one after the other, in equal ranges. An item is a
//                  range of one tile of every group, and leaves a part for each group that it
//                  meets: part (range + group) tiles + tile, since along the k-blocks each part
//                  begins with the next range or the next group. Blocks at work at one time have
//                  the tiles of few ranges, whose operands they share in L2 (110592 x 1024 x 256 in
//                  8 groups, all tiles one after the other instead: 121 us, so 97). Its counter w is
//                  k-block * tiles + tile. Where most rows are in no group there are fewer k-blocks
//                  than the host planned ranges: range_count() of them, so that none is empty and
//                  the join finds every part between a group's first and last written.
__host__ __device__ constexpr unsigned range_count(int planned, unsigned kblocks) {
    return (unsigned)planned < kblocks ? (unsigned)planned : kblocks;
}
__host__ __device__ constexpr unsigned range_at(unsigned x, unsigned ranges, unsigned kblocks) {
    return (unsigned)((((uint64_t)x + 1) * ranges - 1) / kblocks);  // of k-block x
}
template <int KIND, bool PAIR>
struct Schedule {
    static constexpr int kTileRows = PAIR ? 2 * kBM : kBM;
    const TileParams& p;
    int32_t* rows;
    int32_t* lines;
    int rank;
    unsigned unit, step;     // this block (or pair) among how many
    unsigned begin, end;     // of the counter of work
    unsigned ranges;         // kDepthRanges

    __device__ __forceinline__ Schedule(const TileParams& params, int32_t* table, int r)
        : p(params), rows(table), lines(table + params.groups + 1), rank(r),
          unit(PAIR ? blockIdx.x >> 1 : blockIdx.x), step(PAIR ? gridDim.x >> 1 : gridDim.x),
          begin(unit) {}

    // all threads, once the offsets may be read
    __device__ __forceinline__ void fill() {
        const unsigned tiles = (unsigned)p.tiles_m * p.tiles_n;
        if constexpr (KIND == kWhole) {
            end = tiles * p.splits;
        } else if constexpr (KIND == kBatch) {
            // symmetric: of square tiles those on and below the diagonal
            end = (p.symmetric ? (unsigned)p.tiles_m * (p.tiles_m + 1) / 2 : tiles) * p.groups;
        } else {
            for (int g = threadIdx.x; g <= p.groups; g += kThreads)
                rows[g] = (int)min((int64_t)max(p.offsets[g], 0), p.m_all);
            __syncthreads();
            if constexpr (KIND == kDepthGroups) {
                // lines: the groups' order, those of several times the mean first, so that their tiles
                // do not end last (65536 x 368 -> 560 in 46 groups, the largest of a tenth of the
                // rows, training 278 -> 270 us); of many groups, whose ranks would take longer, as
                // they come
                const int large =
                    p.groups <= 256 ? (int)min((int64_t)INT32_MAX - 1, 3 * p.m_all / p.groups)
                                    : INT32_MAX;
                for (int g = threadIdx.x; g < p.groups; g += kThreads) {
                    const bool mine = rows[g + 1] - rows[g] > large;
                    int rank = large == INT32_MAX ? g : 0;
                    // the groups of g's kind before it, and all large ones
                    for (int i = 0; i < p.groups && large != INT32_MAX; ++i) {
                        const bool other = rows[i + 1] - rows[i] > large;
                        rank += other == mine ? i < g : other;
                    }
                    lines[rank] = g;
                }
                __syncthreads();
                end = tiles * p.groups;
            } else {
                if (threadIdx.x < 32) {
                    constexpr int kLine = by_depth(KIND) ? 64 : kTileRows;
                    // no more than offsets in order lead to, which the grids and the parts
                    // are sized for
                    const int most = (int)most_lines(p.m_all, p.groups, kLine);
                    int before = 0;
                    for (int g0 = 0; g0 < p.groups; g0 += 32) {
                        const int g = g0 + threadIdx.x;
                        int n = 0;
                        if (g < p.groups)
                            n = (max(0, rows[g + 1] - rows[g]) + kLine - 1) / kLine;
                        int sum = n;
#pragma unroll
                        for (int o = 1; o < 32; o *= 2) {
                            const int other = __shfl_up_sync(0xffffffffu, sum, o);
                            sum += (int)threadIdx.x >= o ? other : 0;
                        }
                        if (g < p.groups) lines[g] = min(before + sum - n, most);
                        before = min(before + __shfl_sync(0xffffffffu, sum, 31), most);
                    }
                    if (threadIdx.x == 0) lines[p.groups] = before;
                }
                __syncthreads();
                const unsigned all = (unsigned)uniform(lines[p.groups]);
                if constexpr (KIND == kRowGroups || KIND == kRowsAcross) {
                    end = all * p.tiles_n;
                } else {
                    end = all * tiles;
                    ranges = range_count(p.ranges, all);
                    begin = item(unit);
                }
            }
        }
    }

    // the group g with lines[g] <= line < lines[g + 1]
    __device__ __forceinline__ int group_at(int line) const {
        int g = 0, above = p.groups;
        while (above - g > 1) {
            const int mid = (g + above) >> 1;
            if (lines[mid] <= line) g = mid;
            else above = mid;
        }
        return uniform(g);
    }

    // kDepthRanges: the range of k-block x; where range r begins; and the counter at which item i
    // begins (the end behind the last)
    __device__ __forceinline__ unsigned range_of(unsigned x) const {
        return range_at(x, ranges, (unsigned)uniform(lines[p.groups]));
    }
    __device__ __forceinline__ unsigned start(unsigned r) const {
        return (unsigned)((uint64_t)(unsigned)uniform(lines[p.groups]) * r / ranges);
    }
    __device__ __forceinline__ unsigned item(unsigned i) const {
        const unsigned tiles = p.by_tiles.by;
        if (i >= ranges * tiles) return end;
        const unsigned r = p.by_tiles.quotient(i);
        return start(r) * tiles + i - r * tiles;
    }

    __device__ __forceinline__ unsigned next(unsigned w) const {
        if constexpr (KIND == kDepthRanges) {
            const unsigned tiles = p.by_tiles.by, x = p.by_tiles.quotient(w), r = range_of(x);
            int kb0, kb1;
            range(w, kb0, kb1);
            const unsigned on = x + kb1 - kb0;
            return on < start(r + 1) ? w + (kb1 - kb0) * tiles
                                     : item(r * tiles + (w - x * tiles) + step);
        }
        return w + step;
    }

    __device__ __forceinline__ Tile tile(unsigned w) const {
        Tile t;
        if constexpr (KIND == kWhole) {
            t = tile_of(p, w);
            t.row_end = (int)p.m;
        } else if constexpr (KIND == kRowGroups || KIND == kRowsAcross) {
            const int line = (int)p.by_tiles.quotient(w);  // by the tiles of a line
            const int g = group_at(line);
            const unsigned first = uniform(lines[g]), n = uniform(lines[g + 1]) - first;
            const unsigned at = w - first * p.tiles_n, part = p.by_group.quotient(at);
            const unsigned in = at - part * p.by_group.by, high = min(kGroup, n - part * kGroup);
            t.nt = in / high;
            const int mt = part * kGroup + (in - t.nt * high);
            t.split = 0, t.z = g, t.empty = false;
            t.row0 = uniform(rows[g]) + mt * kTileRows + (KIND == kRowGroups ? rank * kBM : 0);
            t.row_end = uniform(rows[g + 1]);
            t.mt = ((int)first + mt) * (kTileRows / kBM) + rank;
            return t;
        } else if constexpr (KIND == kDepthGroups) {
            const unsigned at = p.by_tiles.quotient(w);
            t = tile_of(p, w - at * p.by_tiles.by);
            t.z = uniform(lines[at]);
            t.empty = uniform(rows[t.z + 1] - rows[t.z]) <= 0;
            t.row_end = (int)p.m;
        } else if constexpr (KIND == kDepthRanges) {
            const unsigned x = p.by_tiles.quotient(w), at = w - x * p.by_tiles.by;
            const int g = group_at((int)x), mt = at / p.tiles_n;
            t = Tile{mt, (int)(at - mt * p.tiles_n),
                     (int)((range_of(x) + g) * p.by_tiles.by + at), g, 0, (int)p.m, false};
        } else {
            if (p.symmetric) {
                const unsigned each = (unsigned)p.tiles_m * (p.tiles_m + 1) / 2, in = w % each;
                int mt = (int)((sqrtf(8.0f * in + 1.0f) - 1.0f) * 0.5f);
                while (mt * (mt + 1) / 2 > (int)in) --mt;
                while ((mt + 1) * (mt + 2) / 2 <= (int)in) ++mt;
                t = Tile{mt, (int)in - mt * (mt + 1) / 2, 0, (int)(w / each), 0, 0, false};
            } else {
                const unsigned z = p.by_tiles.quotient(w);
                t = tile_of(p, w - z * p.by_tiles.by);
                t.z = z;
            }
            t.row_end = (int)p.m;
        }
        if (PAIR) t.mt = t.mt * 2 + rank;
        t.row0 = t.mt * kBM;
        return t;
    }

    // lines of k of work item w: [kb0, kb1)
    __device__ __forceinline__ void range(unsigned w, int& kb0, int& kb1) const {
        if constexpr (KIND == kDepthGroups) {
            const int z = uniform(lines[p.by_tiles.quotient(w)]);
            kb0 = 0;
            kb1 = (max(0, uniform(rows[z + 1] - rows[z])) + 63) / 64;
        } else if constexpr (KIND == kDepthRanges) {
            const unsigned x = p.by_tiles.quotient(w);
            const int g = group_at((int)x);
            kb0 = (int)x - uniform(lines[g]);
            kb1 = min(uniform(lines[g + 1]), (int)start(range_of(x) + 1)) - uniform(lines[g]);
        } else {
            const int split =
                KIND == kWhole && p.splits > 1 ? (int)p.by_tiles.quotient(w) : 0;
            kb0 = split * p.kb_per_split;
            kb1 = min(p.kblocks, kb0 + p.kb_per_split);
        }
    }
};

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
__device__ __forceinline__ void rows_loaded() {
    asm volatile("cp.async.wait_all;" ::: "memory");
    __syncwarp();
}
// rows x cols (of 32 x 32, zeros beyond) from src into the buffer; there after rows_loaded()
template <typename T>
__device__ __forceinline__ void load_rows(const Stage& st, const T* start, const T* src, int64_t ld,
                                          int rows, int64_t cols, bool vec) {
    if (vec) {
        const int r0 = st.lane >> 2, c = (st.lane & 3) * 8;
        const T* p = src + r0 * ld + c;
        const bool in = c < cols;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            // else zeros: nothing is read, and the address is `start`, of the matrix
            const bool some = in && r0 + 8 * i < rows;
            asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(st.turn(i)),
                         "l"(some ? p + i * 8 * ld : start), "r"(some ? 16 : 0)
                         : "memory");
        }
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

// the same of a part of a box, where rows are on 16 bytes
template <typename T>
__device__ __forceinline__ void store_rows16(const Stage& st, T* dst, int64_t ld, int rows,
                                             int64_t cols) {
    const int r0 = st.lane >> 2, c = (st.lane & 3) * 8;
    T* p = dst + r0 * ld + c;
#pragma unroll
    for (int i = 0; i < 4; ++i)
        if (c < cols && r0 + 8 * i < rows)
            *reinterpret_cast<uint4*>(p + i * 8 * ld) = get16(st.turn(i));
}

// The box's part of a group's last rows. Not inlined: it is rare, and among the gradients' code it
// took registers that they have not (gated 221184 x 256 -> 2 x 512, dz 330 -> 250 us).
template <typename T>
__device__ __noinline__ void store_part(uint32_t buf, T* dst, int64_t ld, int rows, int cols,
                                        bool wide) {
    const Stage st(buf, threadIdx.x & 31);
    if (wide) store_rows16<T>(st, dst, ld, rows, cols);
    else store_rows<T>(st, dst, ld, rows, cols);
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
    __device__ __forceinline__ void load(const TileParams& p, int64_t col, int64_t left,
                                         int at = 0) {
        const T* bias = static_cast<const T*>(p.bias) + at + col;
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

// the same values as a column of the transposed box: lane's value j is at (16 half + j, lane)
template <typename T>
__device__ __forceinline__ void put_column(const Stage& st, int half, const Two (&v)[8]) {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        float a, b;
        split(v[j], a, b);
        const uint32_t w = pack2<T>(a, b);
        put_half(st.at(half * 16 + 2 * j, st.lane * 2), (uint16_t)w);
        put_half(st.at(half * 16 + 2 * j + 1, st.lane * 2), (uint16_t)(w >> 16));
    }
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
template <int MODE, int KIND, typename T, bool FP8, typename Wait, typename Release>
__device__ __forceinline__ void epilogue(const TileParams& p, const Tile& t, uint32_t acc,
                                         const Stage& st, const Stage& st2, int warp,
                                         const CUtensorMap* out_map, const CUtensorMap* out2_map,
                                         Wait&& wait, Release&& release) {
    const int quarter = warp & 3, share = warp >> 2;
    const int row0 = t.row0 + quarter * 32;
    const int rows = max(0, min(32, t.row_end - row0));
    constexpr bool kGate = MODE == kGated || MODE == kGatedGrad;
    const int width = kGate ? p.bn / 2 : p.bn;  // output columns of the tile
    const int64_t col0 = (int64_t)t.nt * width;
    const int end = (int)min((int64_t)width, p.n - col0);
    const int lane = st.lane;
    constexpr bool kReads = MODE == kGrad || MODE == kGatedGrad;
    const bool reads = kReads || ((MODE == kForward || MODE == kUpdate) && p.in);
    const int bias_at = KIND == kRowGroups ? uniform(t.z * (int)p.bias_step) : 0;
    auto read_in = [&](int c) {  // residual or dy of the group
        const T* in = static_cast<const T*>(p.in);
        if constexpr (KIND == kBatch) in += t.z * p.in_step;
        load_rows(st, in, in + (int64_t)row0 * p.ld_in + col0 + c, p.ld_in, rows, end - c, p.vec_in);
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
    if (!wait()) {
        rows_loaded();
        return;
    }
    if constexpr (MODE == kPartial) {
        for (int c = share * 16; c < end; c += 64) {
            float v[16];
            tc::tmem_ld16(acc + c, v);
            // kDepthRanges: parts of whole tiles, this block's half of a pair's second
            float* to = KIND == kDepthRanges
                            ? p.z + ((int64_t)t.split * p.ld_part + row0 % p.ld_part) * p.bn + c
                            : p.z + ((int64_t)t.split * p.m + row0) * p.ld_z + col0 + c;
            store_rows32(st, v, to, KIND == kDepthRanges ? p.bn : p.ld_z, rows, end - c);
        }
        release();
        return;
    }
    if constexpr (MODE == kPlain) {
        // 32 columns at a time, in a fifth of the instructions that kForward takes for nothing
        for (int c = share * 32; c < end; c += 128) {
            float v[32];
            tc::tmem_ld32(acc + c, v);
            if (c + 128 >= end) release();
            if (KIND == kDepthGroups && t.empty) {
#pragma unroll
                for (int j = 0; j < 32; ++j) v[j] = 0.0f;
            }
            reuse();
#pragma unroll
            for (int q = 0; q < 4; ++q)
                put16(st.own(q), make_uint4(pack2<T>(v[8 * q], v[8 * q + 1]),
                                            pack2<T>(v[8 * q + 2], v[8 * q + 3]),
                                            pack2<T>(v[8 * q + 4], v[8 * q + 5]),
                                            pack2<T>(v[8 * q + 6], v[8 * q + 7])));
            const bool tma = p.tma_out && (KIND != kRowGroups || rows == 32);
            if (tma) tc::fence_async_smem();
            __syncwarp();
            const int64_t col = col0 + c;
            if (!tma) {
                T* out = static_cast<T*>(p.out) + (int64_t)row0 * p.ld_out + col;
                if constexpr (KIND == kDepthGroups) out += t.z * p.out_step;
                store_part<T>(st.base, out, p.ld_out, rows, (int)(p.n - col), p.tma_out);
            } else if (lane == 0 && rows > 0) {
                if constexpr (KIND == kDepthGroups) bulk_store3(out_map, st.base, (int)col, row0, t.z);
                else bulk_store(out_map, st.base, (int)col, row0);
                bulk_store_commit();
            }
            __syncwarp();
        }
        if (share * 32 >= end) release();
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
                        bias.load(p, at, left - half * 16, bias_at);
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
#pragma unroll 1
        for (int half = 0; half < 2; ++half) {
            const int at = c + half * 16;
            const int64_t zcol = col + half * 16, zleft = left - half * 16;
            Two z[8], u[8];
            {
                float v[16], w[16];
                Bias<T> bias, bias_up;
                bias.load(p, zcol, zleft, bias_at);
                if constexpr (kGate) {
                    bias_up.load(p, p.n + zcol, zleft, bias_at);
                    tmem_ld16x2(acc + at, acc + at + width, v, w);
                } else {
                    tc::tmem_ld16(acc + at, v);
                }
                if (half == 1 && c + 128 >= end) release();
                finish_z<T, FP8>(v, z, bias, p, zcol, zleft, xs);
                if constexpr (kGate) finish_z<T, FP8>(w, u, bias_up, p, p.n + zcol, zleft, xs);
            }
            if (reads && half == 0) rows_loaded();
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
            } else if constexpr (MODE == kUpdate) {
                if (p.in) {
                    get_row<__half>(st, half, u);
#pragma unroll
                    for (int j = 0; j < 8; ++j)
                        z[j] = fma(z[j], two(p.alpha), u[j] * two(p.beta));
                } else {
#pragma unroll
                    for (int j = 0; j < 8; ++j) z[j] = z[j] * two(p.alpha);
                }
                if (p.symmetric) put_column<T>(st2, half, z);
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
        // by TMA; the last rows of a group, behind which another's begin, by the lanes
        const bool tma = p.tma_out && (KIND != kRowGroups || rows == 32);
        if (tma) tc::fence_async_smem();
        __syncwarp();
        if (tma) {
            if (lane == 0 && rows > 0) {
                if constexpr (KIND == kBatch) {
                    bulk_store3(out_map, st.base, (int)col, row0, t.z);
                    if constexpr (MODE == kUpdate) {
                        // and its mirror image, left of the diagonal's tiles
                        if (p.symmetric && row0 >= col0 + p.bn)
                            bulk_store3(out_map, st2.base, row0, (int)col, t.z);
                    }
                } else {
                    bulk_store(out_map, st.base, (int)col, row0);
                    if constexpr (MODE == kGatedGrad)
                        bulk_store(out2_map, st2.base, (int)col, row0);
                }
                bulk_store_commit();
            }
        } else {
            T* out = static_cast<T*>(p.out) + (int64_t)row0 * p.ld_out + col;
            if constexpr (KIND == kRowGroups) {
                store_part<T>(st.base, out, p.ld_out, rows, (int)left, p.tma_out);
                if constexpr (MODE == kGatedGrad)
                    store_part<T>(st2.base, out + p.n, p.ld_out, rows, (int)left, p.tma_out);
            } else {
                if constexpr (KIND == kBatch) out += t.z * p.out_step;
                store_rows<T>(st, out, p.ld_out, rows, left);
                if constexpr (MODE == kGatedGrad)
                    store_rows<T>(st2, out + p.n, p.ld_out, rows, left);
            }
        }
        __syncwarp();
    }
    if (share * 32 >= end) release();  // no columns here
}

// The same of kRowsAcross: a lane holds an output, and its columns are rows of the group. Values turn
// as they enter the buffer, column by column.
template <int MODE, typename T, typename Wait, typename Release>
__device__ __forceinline__ void epilogue_across(const TileParams& p, const Tile& t, int rank,
                                                uint32_t acc, const Stage& st, int warp,
                                                const CUtensorMap* out_map, Wait&& wait,
                                                Release&& release) {
    const int quarter = warp & 3, share = warp >> 2, lane = st.lane;
    const int f0 = t.nt * 2 * kBM + rank * kBM + quarter * 32;
    const int rows = min(2 * kBM, t.row_end - t.row0), left = (int)p.n - f0;
    float bias = 0.0f;
    if (MODE == kForward && p.bias && lane < left)
        bias = to_float(static_cast<const T*>(p.bias)[t.z * (int)p.bias_step + f0 + lane]);
    if (!wait()) return;
    for (int c = share * 32; c < rows; c += 128) {
        if (lane == 0) bulk_store_read();
        __syncwarp();
#pragma unroll 1
        for (int half = 0; half < 2; ++half) {
            float v[16];
            Two z[8];
            tc::tmem_ld16(acc + c + half * 16, v);
            if (half == 1 && c + 128 >= rows) release();
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                z[j] = two(v[2 * j], v[2 * j + 1]);
                if (MODE == kForward) z[j] = z[j] + two(bias);
            }
            if constexpr (MODE == kForward) {
                if (p.z && lane < left) {
                    float* to = p.z + (int64_t)(t.row0 + c + half * 16) * p.ld_z + f0 + lane;
#pragma unroll
                    for (int j = 0; j < 16; ++j) {
                        float a, b;
                        split(z[j / 2], a, b);
                        if (c + half * 16 + j < rows) to[j * p.ld_z] = j % 2 ? b : a;
                    }
                }
                with_activation(p.act, [&](auto a) {
#pragma unroll
                    for (int j = 0; j < 8; ++j) z[j] = act_value<decltype(a)::value>(z[j]);
                });
            }
            put_column<T>(st, half, z);
        }
        const int part = min(32, rows - c);
        const bool tma = p.tma_out && part == 32;
        if (tma) tc::fence_async_smem();
        __syncwarp();
        if (!tma) {
            store_part<T>(st.base, static_cast<T*>(p.out) + (int64_t)(t.row0 + c) * p.ld_out + f0,
                          p.ld_out, part, left, p.tma_out);
        } else if (lane == 0 && left > 0) {
            bulk_store(out_map, st.base, f0, t.row0 + c);
            bulk_store_commit();
        }
        __syncwarp();
    }
    if (share * 32 >= rows) release();  // no rows here
}

// After a wait gave up: lets what is in flight land (bounded) before the blocks' memory goes. The
// copies of both blocks count on the even one's barriers; a stage that only one of them had filled
// when the other gave up gets the other's part from here. Not inlined: among the kernels' own code
// it cost the gated forward 3 % (110592 x 256 -> 512 65.6 against 63.7 us).
template <bool PAIR>
__device__ __noinline__ void drain(TileShared* sh, unsigned* flag, int stages) {
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
            if (i >= theirs) mbar_complete_tx(bar, sh->bytes[i % stages]);
            if (i >= mine)
                mbar_expect_tx(bar, peer_word(peer_address(smem_u32(&sh->bytes[i % stages]), 1)));
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

// This block's rows of dy of a tile on their way to L2, by a warp that is a tile ahead of those that
// read them (gated 221184 x 256 -> 2 x 512 in 8 groups, training 627 -> 618 us; with the copies of
// load_rows 604, waited for at their first use 598).
template <typename T, bool GATE>
__device__ __forceinline__ void prefetch_rows(const TileParams& p, const Tile& t, int lane) {
    const int width = GATE ? p.bn / 2 : p.bn;
    const int64_t col0 = (int64_t)t.nt * width;
    const int cols = (int)min((int64_t)width, p.n - col0), rows = min(kBM, t.row_end - t.row0);
    const T* in = static_cast<const T*>(p.in) + (int64_t)t.row0 * p.ld_in + col0;
    for (int c = 0; c < cols; c += 64)
        for (int r = lane; r < rows; r += 32)
            asm volatile("prefetch.global.L2 [%0];" ::"l"(in + r * p.ld_in + c));
}

// PAIR: two blocks of a cluster (the two SMs of a TPC) work on one tile of 256 rows. Each holds its
// 128 rows of A and of the accumulator and half of the tile's B, which the tensor cores of both
// read: half the shared-memory traffic and half the copies for B. The even block issues the
// products; copies of both count on its barriers, completed products on both blocks'.
template <int MODE, int KIND, typename T, bool FP8, bool PAIR>
__global__ void __launch_bounds__(kThreads, 1)
k_tile(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b,
       const __grid_constant__ CUtensorMap map_o, const __grid_constant__ CUtensorMap map_o2,
       const __grid_constant__ CUtensorMap map_t, const TileParams p) {
    using namespace tc;
    extern __shared__ __align__(1024) unsigned char smem[];
    const int b_rows = PAIR ? p.bn / 2 : p.bn;  // of B in this block's stages
    const uint32_t stage_bytes = kAStage + (uint32_t)b_rows * kLineBytes;
    unsigned char* bufs = smem + (size_t)p.stages * stage_bytes;
    auto* sh = reinterpret_cast<TileShared*>(bufs + kEpiWarps * kWarpBufs<MODE> * kWarpBuf);
    const int tid = threadIdx.x, lane = tid & 31;
    const int warp = __shfl_sync(0xffffffffu, tid >> 5, 0);  // uniform, and known to be
    constexpr bool kGate = MODE == kGated || MODE == kGatedGrad;
    constexpr bool kReads = MODE == kGrad || MODE == kGatedGrad;
    const int rank = PAIR ? (int)cluster_rank() : 0;
    Schedule<KIND, PAIR> plan(p, reinterpret_cast<int32_t*>(sh + 1), rank);

    if (tid == 0) {
        for (int s = 0; s < p.stages; ++s) {
            mbar_init(smem_u32(&sh->full[s]), 1);
            mbar_init(smem_u32(&sh->empty[s]), 1);
            sh->bytes[s] = stage_bytes;
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
    plan.fill();

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
        auto load3 = [&](uint32_t dst, const CUtensorMap* map, int x, int y, int z, uint32_t bar) {
            if constexpr (PAIR) tma_load3_pair(dst, map, x, y, z, bar);
            else tma_load3(dst, map, x, y, z, bar);
        };
        auto load_a = [&](uint32_t dst, const CUtensorMap* map, int x, int y, int z, uint32_t bar) {
            if constexpr (KIND == kBatch) load3(dst, map, x, y, z, bar);
            else load(dst, map, x, y, bar);
        };
        auto load_b = [&](uint32_t dst, const CUtensorMap* map, int x, int y, int z, uint32_t bar) {
            if constexpr (KIND == kBatch || KIND == kRowGroups) load3(dst, map, x, y, z, bar);
            else load(dst, map, x, y, bar);
        };
        int st = 0, issued = 0;
        uint32_t parity = 1;  // of the stage's last release; a fresh barrier passes for 1
        bool ok = true;
        for (unsigned w = plan.begin; w < plan.end && ok; w = plan.next(w)) {
            const Tile t = plan.tile(w);
            int kb0, kb1;
            plan.range(w, kb0, kb1);
            const int m0 = t.row0;
            // by depth: the group's rows, and how many k-blocks of them are whole; what is left of
            // them lies in lines of its own, zeros behind the group's end
            int k0 = 0, whole = INT32_MAX;
            if constexpr (by_depth(KIND)) {
                k0 = uniform(plan.rows[t.z]);
                whole = (uniform(plan.rows[t.z + 1]) - k0) / 64;
            }
            // first row of B here: a pair's blocks take halves of the tile, gate and up or not
            int n0 = t.nt * bw;
            if (PAIR && rank) n0 += kGate ? (int)p.n : b_rows;
            if constexpr (kReads) prefetch_rows<T, kGate>(p, t, lane);
            for (int kb = kb0; kb < kb1; ++kb) {
                ok = mbar_wait(smem_u32(&sh->empty[st]), parity, p.polls) && !*fail;
                if (!__all_sync(0xffffffffu, ok)) {
                    ok = false;
                    break;
                }
                const uint32_t bar = full0 + (uint32_t)st * 8;
                const uint32_t a = smem_u32(smem) + (uint32_t)st * stage_bytes, b = a + kAStage;
                const bool in = !by_depth(KIND) || kb < whole;
                const CUtensorMap *a_map = in ? &map_a : &map_o2, *b_map = in ? &map_b : &map_t;
                const int y = in ? k0 + kb * 64 : tail_place(t.z, k0) * 64;
                if constexpr (KIND == kRowsAcross) {
                    // this block's outputs of the matrix, and its half of the rows
                    const int f0 = t.nt * 2 * kBM + rank * kBM;
                    const int half = rows_across(t) / 2, r0 = t.row0 + rank * half;
                    if (one) {
                        sh->bytes[st] = kAStage + half * kLineBytes;
                        if (rank == 0) mbar_expect_tx(smem_u32(&sh->full[st]), 2 * sh->bytes[st]);
                        if (p.a_mn) {
                            load3(a, &map_a, f0, kb * 64, t.z, bar);
                            load3(a + kMnChunk, &map_a, f0 + 64, kb * 64, t.z, bar);
                        } else {
                            load3(a, &map_a, kb * 64, f0, t.z, bar);
                        }
                        if (half == kBM) {
                            load(b, &map_o2, kb * 64, r0, bar);  // in one box
                        } else {
                            for (int i = 0; i < half; i += 16)
                                load(b + i * kLineBytes, &map_b, kb * 64, r0 + i, bar);
                        }
                    }
                } else if (one) {
                    if (!PAIR || rank == 0)
                        mbar_expect_tx(smem_u32(&sh->full[st]), (PAIR ? 2 : 1) * stage_bytes);
                    const int x = kb * (FP8 ? 128 : 64);
                    if (p.a_mn) {
                        load_a(a, a_map, m0, y, t.z, bar);
                        load_a(a + kMnChunk, a_map, m0 + 64, y, t.z, bar);
                    } else {
                        load_a(a, a_map, x, m0, t.z, bar);
                    }
                    if (p.b_mn) {
                        for (int i = 0; i < b_rows / 64; ++i)
                            load_b(b + i * kMnChunk, b_map, n0 + i * 64, y, t.z, bar);
                    } else {
                        load_b(b, b_map, x, n0, t.z, bar);
                        if (kGate && !PAIR)
                            load_b(b + bw * kLineBytes, b_map, x, (int)p.n + n0, t.z, bar);
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
        for (unsigned w = plan.begin; w < plan.end && ok; w = plan.next(w)) {
            int kb0, kb1;
            plan.range(w, kb0, kb1);
            ok = mbar_wait(smem_u32(&sh->acc_empty[buf]), acc_parity, p.polls) && !*fail;
            if (!__all_sync(0xffffffffu, ok)) {
                if (!*fail) *fail = 2;
                ok = false;
                break;
            }
            fence_after_sync();
            const uint32_t acc = tmem + buf * 256;
            uint32_t idesc = p.idesc;
            if constexpr (KIND == kRowsAcross)
                idesc |= (uint32_t)(rows_across(plan.tile(w)) >> 3) << 17;
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
                                       idesc, more);
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
        for (unsigned w = plan.begin; w < plan.end && ok; w = plan.next(w), ++n_tile) {
            const Tile t = plan.tile(w);
            const int b = n_tile & 1, round = n_tile >> 1;
            auto wait = [&] {
                ok = mbar_wait(smem_u32(&sh->acc_full[b]), round & 1, p.polls) && !*fail;
                ok = __all_sync(0xffffffffu, ok);
                fence_after_sync();
                return ok;
            };
            auto release = [&] {
                fence_before_sync();
                __syncwarp();
                if (lane == 0) {
                    if constexpr (PAIR)
                        mbar_arrive_peer(peer_address(smem_u32(&sh->acc_empty[b]), 0));
                    else
                        mbar_arrive(smem_u32(&sh->acc_empty[b]));
                }
                __syncwarp();
            };
            if constexpr (KIND == kRowsAcross)
                epilogue_across<MODE, T>(p, t, rank, tmem + b * 256 + quarter, st, warp, &map_o,
                                         wait, release);
            else
                epilogue<MODE, KIND, T, FP8>(p, t, tmem + b * 256 + quarter, st, st2, warp, &map_o,
                                             &map_o2, wait, release);
        }
        if constexpr ((KIND == kRowGroups || KIND == kRowsAcross) &&
                      (MODE == kForward || MODE == kGated || MODE == kPlain)) {
            // the rows that no group has
            if (p.zero_tail && ok) {
                const int64_t from = plan.rows[p.groups], n = (p.m_all - from) * p.n;
                T* out = static_cast<T*>(p.out) + from * p.n;
                for (int64_t i = (int64_t)blockIdx.x * (kEpiWarps * 32) + tid; i < n;
                     i += (int64_t)gridDim.x * (kEpiWarps * 32))
                    out[i] = from_float<T>(0.0f);
            }
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
        drain<PAIR>(sh, p.flag, p.stages);
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

// ----------------------------------------------------------------------------- host
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

// stages of the ring beside `fixed` bytes of other shared memory
int ring_stages(bool pair, int bn, uint32_t fixed) {
    const uint32_t stage = kAStage + (uint32_t)(pair ? bn / 2 : bn) * kLineBytes;
    return (int)std::min<uint32_t>(kMaxStages, (kSmemMax - fixed) / stage);
}

// the kernel with `fixed` bytes beside the ring
template <int MODE, int KIND, typename T, bool FP8, bool PAIR>
void launch_blocks(const CUtensorMap& a, const CUtensorMap& b, const CUtensorMap& o,
                   const CUtensorMap& o2, const TileParams& p, int64_t work, uint32_t fixed, int sms,
                   int device, cudaStream_t stream, const CUtensorMap* tail = nullptr) {
    static std::atomic<uint64_t> allowed{0};  // devices whose limit is raised
    if (device >= 64 || !(allowed.load(std::memory_order_relaxed) >> device & 1)) {
        RUNE_CUDA_TRY(cudaFuncSetAttribute(k_tile<MODE, KIND, T, FP8, PAIR>,
                                           cudaFuncAttributeMaxDynamicSharedMemorySize,
                                           (int)kSmemMax));
        if (device < 64) allowed.fetch_or(uint64_t(1) << device, std::memory_order_relaxed);
    }
    const int b_rows = PAIR ? p.bn / 2 : p.bn;
    const unsigned grid = PAIR ? 2 * (unsigned)std::min<int64_t>(work, sms / 2)
                               : (unsigned)std::min<int64_t>(work, sms);
    const size_t smem = (size_t)p.stages * (kAStage + (size_t)b_rows * kLineBytes) + fixed;
    launch(k_tile<MODE, KIND, T, FP8, PAIR>, grid, kThreads, smem, PAIR ? 2 : 0, stream, a, b, o,
           o2, tail ? *tail : a, p);
}

}  // namespace
}  // namespace ops
}  // namespace rune
