// Rows by group: the choice of groups (route), the stable sort of rows by group (row_groups), and the
// moves of rows into that order and back (to_groups, from_groups) with their gradients. Groups are
// elements with a network each (rune/nep/model.py:157-170 loops over them) or experts.
//
//   route        the k largest of a row's logits, ties to the lowest index, and their softmax
//                w_j = e^(l_j - l_0) / sum_i e^(l_i - l_0);   dl_j = w_j (dw_j - sum_i w_i dw_i)
//   row_groups   slot s = (row, choice) of group g(s) goes to place(s) = #{t: g(t) < g(s)} +
//                #{t < s: g(t) = g(s)}; order is the inverse, offsets the groups' first places
//   to_groups    xs[p] = x[order(p) / k];                 dx[r] = sum_j dxs[place(r, j)]
//   from_groups  out[r] = sum_j w[r, j] y[place(r, j)];   dy[p] = w[order(p)] dout[order(p) / k],
//                dw[r, j] = <dout[r], y[place(r, j)]>
//
// All are bound by memory or, small, by latency. Every gradient of a move is the other move read by
// its own index, so nothing is added by atomics and equal inputs give equal bits. Slots without a
// group have place -1; the places behind the last group have order -1 and rows of zeros. Indexes
// are checked where they are used: a wrong order or place selects nothing and reads nothing.

#include <algorithm>
#include <atomic>

#include "ops.cuh"

namespace rune {
namespace ops {

namespace {

constexpr int kMaxGroups = 1024, kMaxChoices = 32;
// Rows above which few groups' logits go a thread per row: below, a warp per row is sooner done.
constexpr int64_t kRouteRows = 4096;

// ------------------------------------------------------------------------------------ route
// Orders as the values do: NaN above all, -0 as 0.
__device__ __forceinline__ uint32_t order_key(float v) {
    const uint32_t u = __float_as_uint(v + 0.0f);
    if (v != v) return 0xffffffffu;
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}
constexpr uint32_t kKeyMasked = 0x007fffffu;  // of -inf
__device__ __forceinline__ float key_value(uint32_t key) {
    return key == 0xffffffffu ? __uint_as_float(0x7fc00000u)
                              : __uint_as_float(key & 0x80000000u ? key ^ 0x80000000u : ~key);
}

template <typename T>
struct RouteParams {
    int64_t rows, ld;
    int groups, k;
    const T* logits;
    int32_t* index;
    float* weights;
};

// The softmax over the choices, of which lane j has the j-th: its logit and its group (-1: none).
template <typename T>
__device__ __forceinline__ void finish_route(const RouteParams<T>& p, int64_t row, float value,
                                             int chosen) {
    const int lane = threadIdx.x & 31;
    const float largest = __shfl_sync(0xffffffffu, value, 0);
    const float e = chosen >= 0 ? expf(value - largest) : 0.0f;
    const float sum = warp_sum(e);
    if (lane < p.k) {
        p.index[row * p.k + lane] = chosen;
        p.weights[row * p.k + lane] = chosen >= 0 ? e / sum : 0.0f;
    }
}

// 16-bit logits as words, the order of the value above the index's complement: one comparison
// settles ties too. A lane sorts its PER words (Batcher's network), and each round of the selection
// is the maximum of the lanes' first words, whose lane moves on to its next.
template <typename T>
__device__ __forceinline__ uint32_t short_key(T v) {
    const uint32_t u = *reinterpret_cast<const uint16_t*>(&v);
    if (to_float(v) != to_float(v)) return 0xffffu;
    return u == 0x8000u ? 0x8000u : u & 0x8000u ? u ^ 0xffffu : u | 0x8000u;
}
template <int PER>
__device__ __forceinline__ void sort_down(uint32_t (&w)[PER]) {
#pragma unroll
    for (int size = 1; size < PER; size *= 2)
#pragma unroll
        for (int k = size; k >= 1; k /= 2)
#pragma unroll
            for (int j = k % size; j + k < PER; j += 2 * k)
#pragma unroll
                for (int i = 0; i < k; ++i)
                    if (i + j + k < PER && (i + j) / (2 * size) == (i + j + k) / (2 * size)) {
                        const uint32_t a = w[i + j], b = w[i + j + k];
                        w[i + j] = max(a, b), w[i + j + k] = min(a, b);
                    }
}
template <typename T, int PER>
__global__ void __launch_bounds__(256) k_route_short(const RouteParams<T> p) {
    follow_on();
    const int lane = threadIdx.x & 31;
    for (int64_t row = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5); row < p.rows;
         row += (int64_t)gridDim.x * 8) {
        const T* at = p.logits + row * p.ld;
        uint32_t word[PER];
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            const int g = lane + 32 * i;
            word[i] = g < p.groups ? short_key(at[g]) << 16 | (0xffffu - g) : 0u;
        }
        sort_down(word);
        uint32_t mine = 0;
        for (int j = 0; j < p.k; ++j) {
            const uint32_t top = __reduce_max_sync(0xffffffffu, word[0]);
            if (lane == j) mine = top;
            if (word[0] == top) {
#pragma unroll
                for (int i = 0; i + 1 < PER; ++i) word[i] = word[i + 1];
                word[PER - 1] = 0u;
            }
        }
        const uint32_t key = mine >> 16;
        const uint16_t bits = (uint16_t)(key & 0x8000u ? key ^ 0x8000u : key ^ 0xffffu);
        const float value = key == 0xffffu ? __uint_as_float(0x7fc00000u)
                                           : to_float(*reinterpret_cast<const T*>(&bits));
        const bool some = lane < p.k && value != -INFINITY;  // -inf: not to be chosen
        finish_route(p, row, value, some ? (int)(0xffffu - (mine & 0xffffu)) : -1);
    }
}

// A warp per row; a lane has the values lane, lane + 32, ... A round of the selection is a maximum
// over the warp and the lowest index that has it, both by one reduction instruction. 16384 x 256, 8
// choices: 17 us, and 16-bit ones by their words 10; 16384 x 1000 70 us by either.
template <typename T, int PER>
__global__ void __launch_bounds__(256) k_route(const RouteParams<T> p) {
    follow_on();
    const int lane = threadIdx.x & 31;
    for (int64_t row = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5); row < p.rows;
         row += (int64_t)gridDim.x * 8) {
        const T* at = p.logits + row * p.ld;
        uint32_t key[PER];
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            const int g = lane + 32 * i;
            key[i] = g < p.groups ? order_key(to_float(at[g])) : 0u;
        }
        uint32_t mine = 0;
        int chosen = -1;
        for (int j = 0; j < p.k; ++j) {
            uint32_t top = key[0];
#pragma unroll
            for (int i = 1; i < PER; ++i) top = max(top, key[i]);
            top = __reduce_max_sync(0xffffffffu, top);
            uint32_t first = 0xffffffffu;
#pragma unroll
            for (int i = PER - 1; i >= 0; --i)
                if (key[i] == top) first = lane + 32 * i;
            first = __reduce_min_sync(0xffffffffu, first);
#pragma unroll
            for (int i = 0; i < PER; ++i)
                if (first == lane + 32 * i) key[i] = 0u;
            if (lane == j) mine = top, chosen = (int)first;
        }
        const float value = key_value(mine);
        const bool some = lane < p.k && mine != kKeyMasked;  // -inf: not to be chosen
        finish_route(p, row, value, some ? chosen : -1);
    }
}

// Few groups: a thread per row, of which it holds all logits (131072 x 8, 2 choices: 22 -> 4 us).
template <typename T, int PER>
__global__ void __launch_bounds__(128) k_route_rows(const RouteParams<T> p) {
    follow_on();
    for (int64_t row = (int64_t)blockIdx.x * 128 + threadIdx.x; row < p.rows;
         row += (int64_t)gridDim.x * 128) {
        const T* at = p.logits + row * p.ld;
        uint32_t key[PER];
#pragma unroll
        for (int i = 0; i < PER; ++i) key[i] = i < p.groups ? order_key(to_float(at[i])) : 0u;
        int32_t* index = p.index + row * p.k;
        float* weights = p.weights + row * p.k;
        float largest = 0.0f, sum = 0.0f;
        for (int j = 0; j < p.k; ++j) {
            uint32_t top = key[0];
            int first = 0;
#pragma unroll
            for (int i = 1; i < PER; ++i)
                if (key[i] > top) top = key[i], first = i;
#pragma unroll
            for (int i = 0; i < PER; ++i)
                if (i == first) key[i] = 0u;
            const float value = key_value(top);
            if (j == 0) largest = value;
            const float e = top != kKeyMasked ? expf(value - largest) : 0.0f;
            index[j] = top != kKeyMasked ? first : -1;
            weights[j] = e;  // divided by the sum below
            sum += e;
        }
        if (sum != 0.0f)  // NaN too
            for (int j = 0; j < p.k; ++j) weights[j] = index[j] >= 0 ? weights[j] / sum : 0.0f;
    }
}

template <typename T>
struct RouteGradParams {
    int64_t rows;
    int groups, k;
    bool wide;  // rows of dlogits on 16 bytes
    const int32_t* index;
    const float* weights;
    const float* dweights;
    T* dlogits;
};

// A warp per row: zeros, then the chosen ones' gradients over them.
template <typename T>
__global__ void __launch_bounds__(256) k_route_grad(const RouteGradParams<T> p) {
    follow_on();
    const int lane = threadIdx.x & 31;
    for (int64_t row = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5); row < p.rows;
         row += (int64_t)gridDim.x * 8) {
        int g = -1;
        float w = 0.0f, d = 0.0f;
        if (lane < p.k) {
            g = p.index[row * p.k + lane];
            w = p.weights[row * p.k + lane];
            d = p.dweights[row * p.k + lane];
        }
        const float dot = warp_sum(g >= 0 ? w * d : 0.0f);
        T* out = p.dlogits + row * p.groups;
        if (p.wide) {
            const int pieces = p.groups * (int)sizeof(T) / 16;
            for (int i = lane; i < pieces; i += 32)
                reinterpret_cast<uint4*>(out)[i] = make_uint4(0, 0, 0, 0);
        } else {
            for (int i = lane; i < p.groups; i += 32) out[i] = from_float<T>(0.0f);
        }
        __syncwarp();
        if (g >= 0 && g < p.groups) out[g] = from_float<T>(w * (d - dot));
    }
}

// ------------------------------------------------------------------------------------ sort
// Each warp of each block owns a range of slots, in order. k_count leaves the blocks' counts of
// each group; k_place adds up those before its own, then walks its slots again: a slot's rank
// among the warp's 32 comes from the lanes that match it. One block alone needs no first kernel.
constexpr int kSortWarps = 16, kSortThreads = 32 * kSortWarps;
// groups from which counting takes shared memory's atomics, whose conflicts are few then, for the
// matching of lanes (1048576 slots in 256 groups 41 -> 25 us)
constexpr int kAtomicGroups = 32;
constexpr int64_t kSortAlone = 2048;  // slots that one block sorts by itself

struct SortParams {
    int64_t slots, per_warp;
    int groups, blocks;
    const void* index;
    int32_t* counts;  // [blocks][groups]
    int32_t *offsets, *order, *place;
};

// group of a slot, or -1
template <typename I>
__device__ __forceinline__ int group_of(const SortParams& p, int64_t slot) {
    const I g = static_cast<const I*>(p.index)[slot];
    return g >= 0 && g < p.groups ? (int)g : -1;
}

// this warp's counts into hist[warp][groups] and the block's sums into total[groups]
template <typename I>
__device__ __forceinline__ void count_slots(const SortParams& p, int32_t* hist, int32_t* total) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    int32_t* own = hist + warp * p.groups;
    for (int i = lane; i < p.groups; i += 32) own[i] = 0;
    __syncwarp();
    const int64_t first = ((int64_t)blockIdx.x * kSortWarps + warp) * p.per_warp;
    const int64_t last = min(first + p.per_warp, p.slots);
    constexpr int kAhead = 4;
    for (int64_t s = first; s < last; s += 32 * kAhead) {
        int g[kAhead];
#pragma unroll
        for (int i = 0; i < kAhead; ++i) {
            const int64_t slot = s + 32 * i + lane;
            g[i] = slot < last ? group_of<I>(p, slot) : -1;
        }
#pragma unroll
        for (int i = 0; i < kAhead; ++i) {
            if (p.groups >= kAtomicGroups) {  // whole numbers: their order does not matter
                if (g[i] >= 0) atomicAdd(&own[g[i]], 1);
                continue;
            }
            const unsigned same = __match_any_sync(0xffffffffu, g[i]);
            if (g[i] >= 0 && lane == __ffs(same) - 1) own[g[i]] += __popc(same);
            __syncwarp();
        }
    }
    __syncthreads();
    for (int i = threadIdx.x; i < p.groups; i += kSortThreads) {
        int sum = 0;
#pragma unroll
        for (int w = 0; w < kSortWarps; ++w) sum += hist[w * p.groups + i];
        total[i] = sum;
    }
}

template <typename I>
__global__ void __launch_bounds__(kSortThreads) k_count(const SortParams p) {
    follow_on();
    extern __shared__ int32_t words[];
    count_slots<I>(p, words, p.counts + (int64_t)blockIdx.x * p.groups);
}

template <typename I>
__global__ void __launch_bounds__(kSortThreads) k_place(const SortParams p) {
    follow_on();
    extern __shared__ int32_t words[];
    int32_t* hist = words;                           // [warps][groups]
    int32_t* base = hist + kSortWarps * p.groups;    // [groups]: first place of this block's slots
    int32_t* total = base + p.groups;                // [groups]
    __shared__ int32_t sums[kSortWarps + 1];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    count_slots<I>(p, hist, base);
    __syncthreads();
    if (p.blocks == 1) {
        for (int i = tid; i < p.groups; i += kSortThreads) total[i] = base[i], base[i] = 0;
    } else {
        // `parts` threads add up a group's counts, in ranges of blocks
        for (int i = tid; i < p.groups; i += kSortThreads) total[i] = 0, base[i] = 0;
        __syncthreads();
        int width = 1;
        while (width < p.groups) width *= 2;
        const int parts = max(1, kSortThreads / width), step = kSortThreads / parts;
        for (int g = tid % step; g < p.groups; g += step) {
            int before = 0, all = 0;
#pragma unroll 16
            for (int b = tid / step; b < p.blocks; b += parts) {
                const int c = p.counts[(int64_t)b * p.groups + g];
                all += c;
                before += b < (int)blockIdx.x ? c : 0;
            }
            atomicAdd(&total[g], all);  // whole numbers: their order does not matter
            atomicAdd(&base[g], before);
        }
    }
    __syncthreads();
    // exclusive sums over the groups: two of them a thread
    const int g0 = 2 * tid, a = g0 < p.groups ? total[g0] : 0;
    const int b = g0 + 1 < p.groups ? total[g0 + 1] : 0;
    int sum = a + b;
#pragma unroll
    for (int o = 1; o < 32; o *= 2) {
        const int other = __shfl_up_sync(0xffffffffu, sum, o);
        sum += lane >= o ? other : 0;
    }
    if (lane == 31) sums[warp] = sum;
    __syncthreads();
    if (warp == 0) {
        int s = lane < kSortWarps ? sums[lane] : 0;
        const int own = s;
#pragma unroll
        for (int o = 1; o < kSortWarps; o *= 2) {
            const int other = __shfl_up_sync(0xffffffffu, s, o);
            s += lane >= o ? other : 0;
        }
        if (lane < kSortWarps) sums[lane] = s - own;
        if (lane == kSortWarps - 1) sums[kSortWarps] = s;
    }
    __syncthreads();
    const int before = sums[warp] + sum - a - b;
    if (g0 < p.groups) base[g0] += before;
    if (g0 + 1 < p.groups) base[g0 + 1] += before + a;
    if (blockIdx.x == 0) {
        if (g0 < p.groups) p.offsets[g0] = before;
        if (g0 + 1 < p.groups) p.offsets[g0 + 1] = before + a;
        if (tid == 0) p.offsets[p.groups] = sums[kSortWarps];
    }
    __syncthreads();
    for (int i = tid; i < p.groups; i += kSortThreads) {  // counts to first places of the warps
        int at = base[i];
#pragma unroll
        for (int w = 0; w < kSortWarps; ++w) {
            const int c = hist[w * p.groups + i];
            hist[w * p.groups + i] = at;
            at += c;
        }
    }
    __syncthreads();
    int32_t* own = hist + warp * p.groups;
    const int64_t first = ((int64_t)blockIdx.x * kSortWarps + warp) * p.per_warp;
    const int64_t last = min(first + p.per_warp, p.slots);
    constexpr int kAhead = 4;
    for (int64_t s = first; s < last; s += 32 * kAhead) {
        int g[kAhead];
#pragma unroll
        for (int i = 0; i < kAhead; ++i) {
            const int64_t slot = s + 32 * i + lane;
            g[i] = slot < last ? group_of<I>(p, slot) : -1;
        }
#pragma unroll
        for (int i = 0; i < kAhead; ++i) {
            const int64_t slot = s + 32 * i + lane;
            const unsigned same = __match_any_sync(0xffffffffu, g[i]);
            int at = -1;
            if (g[i] >= 0) at = own[g[i]] + __popc(same & ((1u << lane) - 1));
            __syncwarp();
            if (g[i] >= 0 && lane == __ffs(same) - 1) own[g[i]] += __popc(same);
            __syncwarp();
            if (slot < last) p.place[slot] = at;
            if (at >= 0) p.order[at] = (int32_t)slot;
        }
    }
    // the places behind the last group
    for (int64_t at = sums[kSortWarps] + (int64_t)blockIdx.x * kSortThreads + tid; at < p.slots;
         at += (int64_t)gridDim.x * kSortThreads)
        p.order[at] = -1;
}

// ------------------------------------------------------------------------------------ moves
// N values of T in one access of N * sizeof(T) bytes.
template <typename T, int N>
struct Piece {
    static constexpr int kBytes = N * (int)sizeof(T);
    static_assert(kBytes == 2 || kBytes == 4 || kBytes == 8 || kBytes == 16, "one access");
    using Raw = std::conditional_t<
        kBytes == 16, uint4,
        std::conditional_t<kBytes == 8, uint2,
                           std::conditional_t<kBytes == 4, uint32_t, uint16_t>>>;
    union {
        Raw raw;
        uint16_t half[kBytes / 2];
        uint32_t word[kBytes / 4 ? kBytes / 4 : 1];
    };
    __device__ __forceinline__ void load(const T* p) { raw = *reinterpret_cast<const Raw*>(p); }
    __device__ __forceinline__ void store(T* p) const { *reinterpret_cast<Raw*>(p) = raw; }
    __device__ __forceinline__ void clear() { raw = Raw{}; }
    __device__ __forceinline__ void get(float (&v)[N]) const {
        if constexpr (sizeof(T) == 4) {
#pragma unroll
            for (int i = 0; i < N; ++i) v[i] = __uint_as_float(word[i]);
        } else if constexpr (N == 1) {
            v[0] = to_float(*reinterpret_cast<const T*>(&half[0]));
        } else {
#pragma unroll
            for (int i = 0; i < N / 2; ++i) {
                const float2 f = unpack2<T>(word[i]);
                v[2 * i] = f.x, v[2 * i + 1] = f.y;
            }
        }
    }
    __device__ __forceinline__ void set(const float (&v)[N]) {
        if constexpr (sizeof(T) == 4) {
#pragma unroll
            for (int i = 0; i < N; ++i) word[i] = __float_as_uint(v[i]);
        } else if constexpr (N == 1) {
            const T t = from_float<T>(v[0]);
            half[0] = *reinterpret_cast<const uint16_t*>(&t);
        } else {
#pragma unroll
            for (int i = 0; i < N / 2; ++i) word[i] = pack2<T>(v[2 * i], v[2 * i + 1]);
        }
    }
};

struct MoveParams {
    int64_t rows, slots;       // slots = rows * k
    int64_t ld_in, ld_more;
    int width, k;
    int lanes;                 // of a team, which has a row (or a part of it) to itself
    const void* in;            // to_groups: x; from_groups: y; its gradient: dout
    const void* more;          // the gradient's y
    const int32_t *order, *place;
    const float* weights;      // [slots] or null
    void* out;                 // contiguous
    float* dweights;           // [slots]
};

// A team of lanes moves R rows at a time, C pieces of each a lane, so that enough is under way while
// the rows' indexes, and then their pieces, arrive: narrow rows two at a time, wide ones in parts of
// four pieces a lane, the parts of a row along the grid's y. B200, 110592 x 256 bf16 to two groups
// each and back with gradients: one row a team 223 us, two 176, four (fewer threads an SM) 204.
constexpr int kMoveThreads = 256;
template <int R_, int C_>
struct Shape {
    static constexpr int R = R_, C = C_;
};

struct Team {
    int index, at, count;
    __device__ __forceinline__ explicit Team(int lanes)
        : index(threadIdx.x / lanes), at(threadIdx.x % lanes), count(kMoveThreads / lanes) {}
};

template <typename T, int N, int R, int C, bool SCALED>
__global__ void __launch_bounds__(kMoveThreads) k_to_groups(const MoveParams p) {
    follow_on();
    const Team t(p.lanes);
    const int col0 = ((int)blockIdx.y * C * p.lanes + t.at) * N, step = p.lanes * N;
    for (int64_t r0 = (int64_t)blockIdx.x * t.count * R + t.index; r0 < p.slots;
         r0 += (int64_t)gridDim.x * t.count * R) {
        int slot[R];
        float w[R];
#pragma unroll
        for (int i = 0; i < R; ++i) {
            const int64_t row = r0 + i * t.count;
            slot[i] = row < p.slots ? p.order[row] : -1;
            if (slot[i] >= p.slots) slot[i] = -1;
        }
#pragma unroll
        for (int i = 0; i < R; ++i) w[i] = SCALED && slot[i] >= 0 ? p.weights[slot[i]] : 0.0f;
        Piece<T, N> v[R][C];
#pragma unroll
        for (int i = 0; i < R; ++i) {
            const T* from = static_cast<const T*>(p.in) + (int64_t)(slot[i] / p.k) * p.ld_in;
#pragma unroll
            for (int c = 0; c < C; ++c) {
                v[i][c].clear();
                if (slot[i] >= 0 && col0 + c * step < p.width) v[i][c].load(from + col0 + c * step);
            }
        }
#pragma unroll
        for (int i = 0; i < R; ++i) {
            const int64_t row = r0 + i * t.count;
            T* to = static_cast<T*>(p.out) + row * p.width;
#pragma unroll
            for (int c = 0; c < C; ++c) {
                if constexpr (SCALED) {
                    float f[N];
                    v[i][c].get(f);
#pragma unroll
                    for (int j = 0; j < N; ++j) f[j] = slot[i] >= 0 ? f[j] * w[i] : 0.0f;
                    v[i][c].set(f);
                }
                if (row < p.slots && col0 + c * step < p.width) v[i][c].store(to + col0 + c * step);
            }
        }
    }
}

// kAhead: choices whose pieces are under way at once
template <typename T, int N, int R, int C, int kAhead>
__global__ void __launch_bounds__(kMoveThreads) k_from_groups(const MoveParams p) {
    follow_on();
    const Team t(p.lanes);
    const int col0 = ((int)blockIdx.y * C * p.lanes + t.at) * N, step = p.lanes * N;
    for (int64_t r0 = (int64_t)blockIdx.x * t.count * R + t.index; r0 < p.rows;
         r0 += (int64_t)gridDim.x * t.count * R) {
        float sum[R][C][N] = {};
        for (int j0 = 0; j0 < p.k; j0 += kAhead) {
            int place[R][kAhead];
            float w[R][kAhead];
#pragma unroll
            for (int i = 0; i < R; ++i)
#pragma unroll
                for (int j = 0; j < kAhead; ++j) {
                    const int64_t row = r0 + i * t.count;
                    const bool in = row < p.rows && j0 + j < p.k;
                    place[i][j] = in ? p.place[row * p.k + j0 + j] : -1;
                    w[i][j] = in && p.weights ? p.weights[row * p.k + j0 + j] : 1.0f;
                    if (place[i][j] >= p.slots) place[i][j] = -1;
                }
            Piece<T, N> v[R][C][kAhead];
#pragma unroll
            for (int i = 0; i < R; ++i)
#pragma unroll
                for (int j = 0; j < kAhead; ++j) {
                    const T* from = static_cast<const T*>(p.in) + place[i][j] * p.ld_in;
#pragma unroll
                    for (int c = 0; c < C; ++c)
                        if (place[i][j] >= 0 && col0 + c * step < p.width)
                            v[i][c][j].load(from + col0 + c * step);
                }
#pragma unroll
            for (int i = 0; i < R; ++i)
#pragma unroll
                for (int j = 0; j < kAhead; ++j) {
                    if (place[i][j] < 0) continue;
#pragma unroll
                    for (int c = 0; c < C; ++c) {
                        float f[N];
                        v[i][c][j].get(f);
#pragma unroll
                        for (int n = 0; n < N; ++n)
                            sum[i][c][n] = fmaf(f[n], w[i][j], sum[i][c][n]);
                    }
                }
        }
#pragma unroll
        for (int i = 0; i < R; ++i) {
            const int64_t row = r0 + i * t.count;
            T* to = static_cast<T*>(p.out) + row * p.width;
#pragma unroll
            for (int c = 0; c < C; ++c) {
                Piece<T, N> o;
                o.set(sum[i][c]);
                if (row < p.rows && col0 + c * step < p.width) o.store(to + col0 + c * step);
            }
        }
    }
}

// A team per slot: dy of its place and the weight's gradient, over the whole row; the slots of one
// row are neighbours, so that dout comes from L1 after the first. The team also clears the row of
// dy that is nobody's place.
template <typename T, int N, int R, int C>
__global__ void __launch_bounds__(kMoveThreads) k_from_groups_grad(const MoveParams p) {
    follow_on();
    const Team t(p.lanes);
    const int step = p.lanes * N;
    T* dy = static_cast<T*>(p.out);
    for (int64_t b0 = (int64_t)blockIdx.x * t.count * R; b0 < p.slots;
         b0 += (int64_t)gridDim.x * t.count * R) {  // all teams, for the sums
        const int64_t s0 = b0 + t.index;
        int place[R], owner[R];
        float w[R], dot[R];
#pragma unroll
        for (int i = 0; i < R; ++i) {
            const int64_t slot = s0 + i * t.count;
            place[i] = slot < p.slots ? p.place[slot] : -1;
            owner[i] = slot < p.slots ? p.order[slot] : 0;
            w[i] = slot < p.slots ? p.weights[slot] : 0.0f;
            if (place[i] >= p.slots) place[i] = -1;
            dot[i] = 0.0f;
        }
        for (int col0 = t.at * N; col0 < p.width; col0 += C * step) {
            Piece<T, N> a[R][C], b[R][C];
#pragma unroll
            for (int i = 0; i < R; ++i) {
                const int64_t slot = s0 + i * t.count;
                const T* dout = static_cast<const T*>(p.in) + slot / p.k * p.ld_in;
                const T* y = static_cast<const T*>(p.more) + place[i] * p.ld_more;
#pragma unroll
                for (int c = 0; c < C; ++c) {
                    a[i][c].clear(), b[i][c].clear();
                    if (place[i] < 0 || col0 + c * step >= p.width) continue;
                    a[i][c].load(dout + col0 + c * step);
                    if (p.dweights) b[i][c].load(y + col0 + c * step);
                }
            }
#pragma unroll
            for (int i = 0; i < R; ++i)
#pragma unroll
                for (int c = 0; c < C; ++c) {
                    float f[N], h[N];
                    a[i][c].get(f), b[i][c].get(h);
#pragma unroll
                    for (int n = 0; n < N; ++n) {
                        dot[i] = fmaf(f[n], h[n], dot[i]);
                        f[n] *= w[i];
                    }
                    if (!dy || col0 + c * step >= p.width) continue;
                    a[i][c].set(f);
                    if (place[i] >= 0)
                        a[i][c].store(dy + (int64_t)place[i] * p.width + col0 + c * step);
                    if (owner[i] < 0 || owner[i] >= p.slots) {
                        Piece<T, N> zero;
                        zero.clear();
                        zero.store(dy + (s0 + i * t.count) * p.width + col0 + c * step);
                    }
                }
        }
        if (!p.dweights) continue;
#pragma unroll
        for (int i = 0; i < R; ++i) {
            for (int o = p.lanes / 2; o > 0; o >>= 1)
                dot[i] += __shfl_xor_sync(0xffffffffu, dot[i], o);
            const int64_t slot = s0 + i * t.count;
            if (t.at == 0 && slot < p.slots) p.dweights[slot] = place[i] >= 0 ? dot[i] : 0.0f;
        }
    }
}

// ------------------------------------------------------------------------------------ host
// values in one access: as many as divide every row's start and its width, 16 bytes at most
int piece_values(int elem_bytes, int64_t width,
                 std::initializer_list<std::pair<const void*, int64_t>> rows) {
    int n = 16 / elem_bytes;
    for (auto [p, ld] : rows)
        while (n > 1 && p &&
               ((uintptr_t)p % (n * elem_bytes) != 0 || ld % n != 0 || width % n != 0))
            n /= 2;
    return n;
}

// fn(T(), std::integral_constant<int, N>) for the type and the piece
template <typename Fn>
void with_piece(int dtype, int n, Fn&& fn) {
    auto narrow = [&](auto t) {
        switch (n) {
            case 8: fn(t, std::integral_constant<int, 8>()); break;
            case 4: fn(t, std::integral_constant<int, 4>()); break;
            case 2: fn(t, std::integral_constant<int, 2>()); break;
            default: fn(t, std::integral_constant<int, 1>()); break;
        }
    };
    if (dtype == RUNE_F16) narrow(__half());
    else if (dtype == RUNE_BF16) narrow(__nv_bfloat16());
    else if (n == 4) fn(float(), std::integral_constant<int, 4>());
    else if (n == 2) fn(float(), std::integral_constant<int, 2>());
    else fn(float(), std::integral_constant<int, 1>());
}

template <typename Fn>
void with_type(int dtype, Fn&& fn) {
    if (dtype == RUNE_F16) fn(__half());
    else if (dtype == RUNE_BF16) fn(__nv_bfloat16());
    else fn(float());
}

// fn(Shape<R, C>()) and the grid for `rows` rows of `pieces`; sets p.lanes. parts: whether the parts
// of wide rows lie along the grid's y.
template <typename Fn>
void with_shape(MoveParams& p, int64_t rows, int pieces, bool parts, int device, Fn&& fn) {
    p.lanes = 1;
    while (p.lanes < 32 && p.lanes < pieces) p.lanes *= 2;
    auto go = [&](auto shape) {
        constexpr int R = decltype(shape)::R, C = decltype(shape)::C;
        const int64_t teams = kMoveThreads / p.lanes * R;
        const unsigned y = parts ? (unsigned)((pieces + 32 * C - 1) / (32 * C)) : 1u;
        require(y <= 65535, "width out of range");
        const int64_t most = std::max<int64_t>(1, (int64_t)sm_count(device) * 32 / y);
        fn(shape, dim3((unsigned)std::min<int64_t>((rows + teams - 1) / teams, most), y));
    };
    if (pieces <= 32) go(Shape<2, 1>());
    else if (pieces <= 64) go(Shape<2, 2>());
    else go(Shape<1, 4>());
}

bool value_type(int dtype) {
    return dtype == RUNE_F32 || dtype == RUNE_F16 || dtype == RUNE_BF16;
}

void check_move(const rune_group_move_args& a) {
    require(a.rows >= 0 && a.k >= 1 && a.rows <= (INT32_MAX - 1024) / a.k,
            "rows or k out of range");
    require(a.width >= 1 && a.width <= INT32_MAX / 2, "width out of range");
    require(value_type(a.dtype), "rows are float32, float16 or bfloat16");
    require_aligned({a.order, a.place, a.weights, a.dweights}, 4);
    require_aligned({a.in, a.y, a.out}, dtype_bytes(a.dtype));
}

MoveParams move_params(const rune_group_move_args& a) {
    MoveParams p{};
    p.rows = a.rows, p.slots = a.rows * a.k;
    p.ld_in = a.in_stride, p.ld_more = a.y_stride;
    p.width = (int)a.width, p.k = (int)a.k;
    p.in = a.in, p.more = a.y;
    p.order = a.order, p.place = a.place;
    p.weights = a.weights;
    p.out = a.out, p.dweights = a.dweights;
    return p;
}

int sort_blocks(const rune_row_groups_args& a) {
    const int64_t slots = a.rows * a.k;
    if (slots <= kSortAlone) return 1;
    // a block for 1024 slots at least, and no more counts than every block can add up
    return (int)std::max<int64_t>(
        2, std::min({(slots + 1023) / 1024, (int64_t)sm_count(a.device),
                     (int64_t)65536 / a.groups}));
}

void check_sort(const rune_row_groups_args& a) {
    require(a.rows >= 0 && a.k >= 1 && a.rows <= (INT32_MAX - 1024) / a.k,
            "rows or k out of range");
    require(a.groups >= 1 && a.groups <= kMaxGroups, "groups out of range: 1 to 1024");
    require(a.index_bytes == 4 || a.index_bytes == 8, "an index is int32 or int64");
    require(a.offsets && (a.rows == 0 || (a.index && a.order && a.place)), "null argument");
    require(aligned(a.index, a.index_bytes), "index does not start on a multiple of its size");
    require_aligned({a.offsets, a.order, a.place}, 4);
}

void check_route(const rune_route_args& a) {
    require(a.rows >= 0, "rows out of range");
    require(a.groups >= 1 && a.groups <= kMaxGroups, "groups out of range: 1 to 1024");
    require(a.k >= 1 && a.k <= kMaxChoices && a.k <= a.groups,
            "k out of range: 1 to 32, and no more than there are groups");
    require(a.rows <= (INT32_MAX - 1024) / a.k, "rows out of range");
    require(value_type(a.dtype), "logits are float32, float16 or bfloat16");
    require_aligned({a.logits, a.dlogits}, dtype_bytes(a.dtype));
    require_aligned({a.index, a.weights, a.dweights}, 4);
    require(a.rows == 0 || (a.index && a.weights), "null argument");
}

}  // namespace
}  // namespace ops
}  // namespace rune

using namespace rune;
using namespace rune::ops;

extern "C" {

int rune_route(const rune_route_args* args, void* stream_) {
    if (!args) {
        set_error("null argument");
        return RUNE_ERR_INVALID;
    }
    const rune_route_args a = *args;
    auto stream = static_cast<cudaStream_t>(stream_);
    return guarded(a.device, [&] {
        check_route(a);
        check_waits(a.device);
        if (a.rows == 0) return;
        require(a.logits, "null argument");
        const unsigned grid =
            (unsigned)std::min<int64_t>((a.rows + 7) / 8, (int64_t)sm_count(a.device) * 16);
        with_type(a.dtype, [&](auto t) {
            using T = decltype(t);
            const RouteParams<T> p{a.rows,   a.logits_stride,
                                   (int)a.groups, (int)a.k,
                                   static_cast<const T*>(a.logits), a.index, a.weights};
            auto go = [&](auto per) {
                constexpr int PER = decltype(per)::value;
                if constexpr (sizeof(T) == 2 && PER <= 16)
                    launch(k_route_short<T, PER>, grid, 256, 0, 0, stream, p);
                else
                    launch(k_route<T, PER>, grid, 256, 0, 0, stream, p);
            };
            const int per = (int)((a.groups + 31) / 32);
            auto rows = [&](auto per_c) {
                const int64_t blocks = (a.rows + 127) / 128;
                launch(k_route_rows<T, decltype(per_c)::value>,
                       (unsigned)std::min<int64_t>(blocks, (int64_t)sm_count(a.device) * 16), 128,
                       0, 0, stream, p);
            };
            if (a.groups <= 8 && a.rows > kRouteRows) rows(std::integral_constant<int, 8>());
            else if (a.groups <= 16 && a.rows > kRouteRows)
                rows(std::integral_constant<int, 16>());
            else if (per <= 1) go(std::integral_constant<int, 1>());
            else if (per <= 2) go(std::integral_constant<int, 2>());
            else if (per <= 4) go(std::integral_constant<int, 4>());
            else if (per <= 8) go(std::integral_constant<int, 8>());
            else if (per <= 16) go(std::integral_constant<int, 16>());
            else go(std::integral_constant<int, 32>());
        });
        RUNE_LAUNCH_CHECK();
    });
}

int rune_route_backward(const rune_route_args* args, void* stream_) {
    if (!args) {
        set_error("null argument");
        return RUNE_ERR_INVALID;
    }
    const rune_route_args a = *args;
    auto stream = static_cast<cudaStream_t>(stream_);
    return guarded(a.device, [&] {
        check_route(a);
        check_waits(a.device);
        if (a.rows == 0) return;
        require(a.dweights && a.dlogits, "null argument");
        const unsigned grid =
            (unsigned)std::min<int64_t>((a.rows + 7) / 8, (int64_t)sm_count(a.device) * 16);
        with_type(a.dtype, [&](auto t) {
            using T = decltype(t);
            const RouteGradParams<T> p{a.rows, (int)a.groups, (int)a.k,
                                       aligned(a.dlogits, 16) && a.groups * sizeof(T) % 16 == 0,
                                       a.index, a.weights, a.dweights,
                                       static_cast<T*>(a.dlogits)};
            launch(k_route_grad<T>, grid, 256, 0, 0, stream, p);
        });
        RUNE_LAUNCH_CHECK();
    });
}

int rune_row_groups_workspace(const rune_row_groups_args* args, int64_t* bytes) {
    if (!args || !bytes) {
        set_error("null argument");
        return RUNE_ERR_INVALID;
    }
    const rune_row_groups_args a = *args;
    return guarded(a.device, [&] {
        check_sort(a);
        const int blocks = sort_blocks(a);
        *bytes = blocks > 1 ? (int64_t)blocks * a.groups * 4 : 0;
    });
}

int rune_row_groups(const rune_row_groups_args* args, void* stream_) {
    if (!args) {
        set_error("null argument");
        return RUNE_ERR_INVALID;
    }
    const rune_row_groups_args a = *args;
    auto stream = static_cast<cudaStream_t>(stream_);
    return guarded(a.device, [&] {
        check_sort(a);
        check_waits(a.device);
        SortParams p{};
        p.slots = a.rows * a.k;
        p.groups = (int)a.groups;
        p.blocks = sort_blocks(a);
        const int64_t warps = (int64_t)p.blocks * kSortWarps;
        p.per_warp = ((p.slots + warps - 1) / warps + 31) / 32 * 32;
        p.index = a.index;
        p.offsets = a.offsets, p.order = a.order, p.place = a.place;
        if (p.blocks > 1) {
            require(a.workspace && aligned(a.workspace, 256) &&
                        a.workspace_bytes >= (int64_t)p.blocks * p.groups * 4,
                    "the workspace is too small or not 256-byte aligned");
            p.counts = static_cast<int32_t*>(a.workspace);
        }
        const size_t count_smem = (size_t)kSortWarps * p.groups * 4;
        const size_t place_smem = count_smem + (size_t)p.groups * 8;
        auto go = [&](auto i) {
            using I = decltype(i);
            static std::atomic<uint64_t> allowed{0};  // devices whose limit is raised
            if (a.device >= 64 || !(allowed.load(std::memory_order_relaxed) >> a.device & 1)) {
                constexpr int most = (kSortWarps + 2) * kMaxGroups * 4;
                for (auto kernel : {k_count<I>, k_place<I>})
                    RUNE_CUDA_TRY(cudaFuncSetAttribute(
                        kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, most));
                if (a.device < 64)
                    allowed.fetch_or(uint64_t(1) << a.device, std::memory_order_relaxed);
            }
            if (p.blocks > 1)
                launch(k_count<I>, p.blocks, kSortThreads, count_smem, 0, stream, p);
            launch(k_place<I>, p.blocks, kSortThreads, place_smem, 0, stream, p);
        };
        if (a.index_bytes == 8) go(int64_t());
        else go(int32_t());
        RUNE_LAUNCH_CHECK();
    });
}

int rune_to_groups(const rune_group_move_args* args, void* stream_) {
    if (!args) {
        set_error("null argument");
        return RUNE_ERR_INVALID;
    }
    const rune_group_move_args a = *args;
    auto stream = static_cast<cudaStream_t>(stream_);
    return guarded(a.device, [&] {
        check_move(a);
        check_waits(a.device);
        if (a.rows == 0) return;
        require(a.in && a.order && a.out, "null argument");
        MoveParams p = move_params(a);
        const int n = piece_values(dtype_bytes(a.dtype), a.width,
                                   {{a.in, a.rows > 1 ? a.in_stride : a.width}, {a.out, a.width}});
        with_piece(a.dtype, n, [&](auto t, auto n_c) {
            using T = decltype(t);
            constexpr int N = decltype(n_c)::value;
            with_shape(p, p.slots, (int)(a.width / N), true, a.device, [&](auto shape, dim3 grid) {
                constexpr int R = decltype(shape)::R, C = decltype(shape)::C;
                if (a.weights)
                    launch(k_to_groups<T, N, R, C, true>, grid, kMoveThreads, 0, 0, stream, p);
                else
                    launch(k_to_groups<T, N, R, C, false>, grid, kMoveThreads, 0, 0, stream, p);
            });
        });
        RUNE_LAUNCH_CHECK();
    });
}

int rune_from_groups(const rune_group_move_args* args, void* stream_) {
    if (!args) {
        set_error("null argument");
        return RUNE_ERR_INVALID;
    }
    const rune_group_move_args a = *args;
    auto stream = static_cast<cudaStream_t>(stream_);
    return guarded(a.device, [&] {
        check_move(a);
        check_waits(a.device);
        if (a.rows == 0) return;
        require(a.in && a.place && a.out, "null argument");
        MoveParams p = move_params(a);
        if (a.k == 1) p.order = p.place;
        const int n = piece_values(
            dtype_bytes(a.dtype), a.width,
            {{a.in, a.rows * a.k > 1 ? a.in_stride : a.width}, {a.out, a.width}});
        with_piece(a.dtype, n, [&](auto t, auto n_c) {
            using T = decltype(t);
            constexpr int N = decltype(n_c)::value;
            with_shape(p, p.rows, (int)(a.width / N), true, a.device, [&](auto shape, dim3 grid) {
                constexpr int R = decltype(shape)::R, C = decltype(shape)::C;
                if (p.k > 1)
                    launch(k_from_groups<T, N, R, C, 2>, grid, kMoveThreads, 0, 0, stream, p);
                else if (p.weights)
                    launch(k_from_groups<T, N, R, C, 1>, grid, kMoveThreads, 0, 0, stream, p);
                else  // one choice: the rows in another order, and no sum
                    launch(k_to_groups<T, N, R, C, false>, grid, kMoveThreads, 0, 0, stream, p);
            });
        });
        RUNE_LAUNCH_CHECK();
    });
}

int rune_from_groups_backward(const rune_group_move_args* args, void* stream_) {
    if (!args) {
        set_error("null argument");
        return RUNE_ERR_INVALID;
    }
    const rune_group_move_args a = *args;
    auto stream = static_cast<cudaStream_t>(stream_);
    return guarded(a.device, [&] {
        check_move(a);
        check_waits(a.device);
        if (a.rows == 0) return;
        require(a.in && a.order && a.place && a.weights && (a.out || a.dweights) &&
                    (a.y || !a.dweights),
                "null argument");
        MoveParams p = move_params(a);
        const int n = piece_values(dtype_bytes(a.dtype), a.width,
                                   {{a.in, a.rows > 1 ? a.in_stride : a.width},
                                    {a.y, a.rows * a.k > 1 ? a.y_stride : a.width},
                                    {a.out, a.width}});
        with_piece(a.dtype, n, [&](auto t, auto n_c) {
            using T = decltype(t);
            constexpr int N = decltype(n_c)::value;
            with_shape(p, p.slots, (int)(a.width / N), false, a.device, [&](auto shape, dim3 grid) {
                constexpr int R = decltype(shape)::R, C = decltype(shape)::C;
                launch(k_from_groups_grad<T, N, R, C>, grid, kMoveThreads, 0, 0, stream, p);
            });
        });
        RUNE_LAUNCH_CHECK();
    });
}

}  // extern "C"
