// Pieces shared by the linear-layer kernels: tiled TMA copies, 128-byte-swizzled operand
// descriptors, 16-bit and e4m3 tensor-core products, and the host's plan of one product.
#pragma once

#include <cuda.h>

#include "ops.cuh"
#include "umma.cuh"

namespace rune {
namespace ops {

// ----------------------------------------------------------------------------- device
// Shared-memory operand tiles are written by TMA with the 128-byte swizzle: lines of 128 bytes,
// eight lines (1 KB) a swizzle atom.
//   K-major (the contraction runs along a line): line = row of the operand, 64 values of k
//     (128 for e4m3); stride byte offset 1024 between groups of eight rows.
//   MN-major (the contraction runs across lines): line = one k, 64 rows of the operand; chunks
//     of 64 rows lie kMnChunk bytes apart (leading byte offset), groups of eight k 1024 bytes.
constexpr uint32_t kLineBytes = 128;
constexpr uint32_t kMnChunk = 64 * kLineBytes;

// 64-bit shared-memory descriptor: address, leading and stride offsets in 16-byte units,
// version 1 (bits 46-47), 128-byte swizzle (2 in bits 61-63).
__device__ __forceinline__ uint64_t operand_desc(uint32_t addr, bool mn) {
    uint64_t d = (uint64_t)((addr >> 4) & 0x3FFFu);
    d |= (uint64_t)(mn ? kMnChunk >> 4 : 1) << 16;
    d |= (uint64_t)(1024 >> 4) << 32;
    d |= (uint64_t)1 << 46;
    d |= (uint64_t)2 << 61;
    return d;
}

// Instruction descriptor: float32 accumulator (bit 4), operand types in bits 7-9 and 10-12
// (kind::f16: 0 half, 1 bfloat16; kind::f8f6f4: 0 e4m3), MN-major flags in bits 15 and 16,
// N / 8 in bits 17-22, M / 16 in bits 24-28.
__host__ __device__ constexpr uint32_t operand_idesc(int type, bool a_mn, bool b_mn, int m,
                                                     int n) {
    return (1u << 4) | ((uint32_t)type << 7) | ((uint32_t)type << 10) |
           ((uint32_t)a_mn << 15) | ((uint32_t)b_mn << 16) | ((uint32_t)(n >> 3) << 17) |
           ((uint32_t)(m >> 4) << 24);
}

// D[tmem] (+)= A B^T on f16 / bf16 or e4m3 operands; PAIR: by the tensor cores of two blocks,
// issued by the even one. One thread issues.
template <bool FP8, bool PAIR>
__device__ __forceinline__ void mma(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc,
                                    bool accumulate) {
    const uint32_t acc = accumulate;
#define RUNE_MMA(group, kind)                                                       \
    asm volatile("{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"                      \
                 " tcgen05.mma.cta_group::" group ".kind::" kind                    \
                 " [%0], %1, %2, %3, p;\n}\n" ::"r"(d), "l"(a), "l"(b), "r"(idesc), \
                 "r"(acc)                                                           \
                 : "memory")
    if constexpr (FP8 && PAIR) RUNE_MMA("2", "f8f6f4");
    else if constexpr (FP8) RUNE_MMA("1", "f8f6f4");
    else if constexpr (PAIR) RUNE_MMA("2", "f16");
    else RUNE_MMA("1", "f16");
#undef RUNE_MMA
}

// tc::tmem_ld16 of two groups of columns at once
__device__ __forceinline__ void tmem_ld16x2(uint32_t a0, uint32_t a1, float (&v)[16],
                                            float (&u)[16]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
        "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%32];\n"
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
        "{%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%33];\n"
        "tcgen05.wait::ld.sync.aligned;"
        : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]), "=f"(v[4]), "=f"(v[5]), "=f"(v[6]),
          "=f"(v[7]), "=f"(v[8]), "=f"(v[9]), "=f"(v[10]), "=f"(v[11]), "=f"(v[12]),
          "=f"(v[13]), "=f"(v[14]), "=f"(v[15]), "=f"(u[0]), "=f"(u[1]), "=f"(u[2]),
          "=f"(u[3]), "=f"(u[4]), "=f"(u[5]), "=f"(u[6]), "=f"(u[7]), "=f"(u[8]), "=f"(u[9]),
          "=f"(u[10]), "=f"(u[11]), "=f"(u[12]), "=f"(u[13]), "=f"(u[14]), "=f"(u[15])
        : "r"(a0), "r"(a1)
        : "memory");
}

// ---- clusters
__device__ __forceinline__ uint32_t cluster_rank() {
    uint32_t r;
    asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ uint32_t cluster_size() {
    uint32_t r;
    asm("mov.u32 %0, %%cluster_nctarank;" : "=r"(r));
    return r;
}
// every thread of every block of the cluster (converged warps)
__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;\nbarrier.cluster.wait.acquire.aligned;"
                 ::: "memory");
}
// this block's shared address `addr` in the cluster's block `rank`
__device__ __forceinline__ uint32_t peer_address(uint32_t addr, uint32_t rank) {
    uint32_t a;
    asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(addr), "r"(rank));
    return a;
}
// loads from a peer's shared memory; volatile keeps them between the cluster's barriers
__device__ __forceinline__ float peer_float(uint32_t addr) {
    float v;
    asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(addr));
    return v;
}
__device__ __forceinline__ uint32_t peer_word(uint32_t addr) {
    uint32_t v;
    asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(addr));
    return v;
}
// Relaxed: it tells that TMEM has been read (ordered by the tcgen05 fence before it), and does
// not wait for this thread's global stores as a release would.
__device__ __forceinline__ void mbar_arrive_peer(uint32_t bar) {
    asm volatile("mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [%0];" ::"r"(bar)
                 : "memory");
}

// ---- pairs of blocks on one tile
__device__ __forceinline__ void tmem_alloc_pair(uint32_t* dst, uint32_t cols) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;"
                 ::"r"(tc::smem_u32(dst)), "r"(cols));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;");
}
__device__ __forceinline__ void tmem_dealloc_pair(uint32_t taddr, uint32_t cols) {
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(taddr), "r"(cols));
}
// the barrier at `bar` in both blocks receives an arrival when every product issued so far by
// this thread is complete
__device__ __forceinline__ void mma_commit_pair(uint32_t bar) {
    asm volatile(
        "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64"
        " [%0], %1;" ::"r"(bar), "h"((uint16_t)3)
        : "memory");
}
// a tile into this block's memory, counted on barrier `bar` (cluster address) of the even block
__device__ __forceinline__ void tma_load_pair(uint32_t dst, const CUtensorMap* map, int x, int y,
                                              uint32_t bar) {
    asm volatile(
        "cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes"
        ".cta_group::2 [%0], [%1, {%2, %3}], [%4];"
        ::"r"(dst), "l"(map), "r"(x), "r"(y), "r"(bar)
        : "memory");
}

// one tile of a 2-D tensor map, innermost coordinate x, into shared memory (no multicast)
__device__ __forceinline__ void tma_load(uint32_t dst, const CUtensorMap* map, int x, int y,
                                         uint32_t bar) {
    asm volatile(
        "cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes "
        "[%0], [%1, {%2, %3}], [%4];"
        ::"r"(dst), "l"(map), "r"(x), "r"(y), "r"(bar)
        : "memory");
}

// the same of 3-D maps (a stack of matrices)
__device__ __forceinline__ void tma_load3(uint32_t dst, const CUtensorMap* map, int x, int y, int z,
                                          uint32_t bar) {
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes "
        "[%0], [%1, {%2, %3, %4}], [%5];"
        ::"r"(dst), "l"(map), "r"(x), "r"(y), "r"(z), "r"(bar)
        : "memory");
}
__device__ __forceinline__ void tma_load3_pair(uint32_t dst, const CUtensorMap* map, int x, int y,
                                               int z, uint32_t bar) {
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes"
        ".cta_group::2 [%0], [%1, {%2, %3, %4}], [%5];"
        ::"r"(dst), "l"(map), "r"(x), "r"(y), "r"(z), "r"(bar)
        : "memory");
}
__device__ __forceinline__ void bulk_store3(const CUtensorMap* map, uint32_t src, int x, int y,
                                            int z) {
    asm volatile("cp.async.bulk.tensor.3d.global.shared::cta.bulk_group [%0, {%1, %2, %3}], [%4];"
                 ::"l"(map), "r"(x), "r"(y), "r"(z), "r"(src)
                 : "memory");
}

// the same tile as far as L2
__device__ __forceinline__ void prefetch_tile(const CUtensorMap* map, int x, int y) {
    asm volatile("cp.async.bulk.prefetch.tensor.2d.L2.global [%0, {%1, %2}];"
                 ::"l"(map), "r"(x), "r"(y)
                 : "memory");
}

// one lane of a converged warp
__device__ __forceinline__ bool elect_one() {
    uint32_t r;
    asm volatile("{\n .reg .pred p;\n elect.sync _|p, 0xffffffff;\n selp.u32 %0, 1, 0, p;\n}\n"
                 : "=r"(r));
    return r != 0;
}

__device__ __forceinline__ void prefetch_map(const CUtensorMap* map) {
    asm volatile("prefetch.tensormap [%0];" ::"l"(map) : "memory");
}

// a box from shared memory to the tensor at (x, y); lines and values outside it are left out
__device__ __forceinline__ void bulk_store(const CUtensorMap* map, uint32_t src, int x, int y) {
    asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.bulk_group [%0, {%1, %2}], [%3];"
                 ::"l"(map), "r"(x), "r"(y), "r"(src)
                 : "memory");
}
__device__ __forceinline__ void bulk_store_commit() {
    asm volatile("cp.async.bulk.commit_group;" ::: "memory");
}
// until this thread's copies out have read their shared memory
__device__ __forceinline__ void bulk_store_read() {
    asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
}

// `bytes` that no copy will bring count as arrived
__device__ __forceinline__ void mbar_complete_tx(uint32_t bar, uint32_t bytes) {
    asm volatile("mbarrier.complete_tx.relaxed.cta.shared::cta.b64 [%0], %1;" ::"r"(bar),
                 "r"(bytes)
                 : "memory");
}

__device__ __forceinline__ void mbar_arrive(uint32_t bar) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory");
}

// ----------------------------------------------------------------------------- host
// A matrix operand in device memory: `rows` lines of `cols` values, `ld` values apart.
struct Matrix {
    const void* p = nullptr;
    int64_t rows = 0, cols = 0, ld = 0;
};

// Whether TMA can read it in place: 16-byte base and line stride, lines that do not overlap.
inline bool tma_ready(const Matrix& m, int elem_bytes) {
    return aligned(m.p, 16) && m.ld * elem_bytes % 16 == 0 && m.ld >= m.cols;
}

// Tensor map of `m` with boxes of one 128-byte line x box_rows lines, zeros outside.
CUtensorMap make_map(const Matrix& m, int elem_bytes, int box_rows);
// The same of a stack of `count` matrices, the first of which is `m`, `step` values apart.
CUtensorMap make_map3(const Matrix& m, int64_t count, int64_t step, int elem_bytes, int box_rows);
// 32 x 32 boxes of a 16-bit output with the 64-byte swizzle, which is the warps' buffers' own
CUtensorMap make_out_map(const void* p, int64_t rows, int64_t cols, int64_t ld);
CUtensorMap make_out_map3(const void* p, int64_t rows, int64_t cols, int64_t ld, int64_t count,
                          int64_t step);

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

inline int64_t pad16(int64_t cols, int elem_bytes) {
    const int64_t v = 16 / elem_bytes;
    return (cols + v - 1) / v * v;
}

// Values of a line of scratch that TMA reads: whole 128-byte lines where that adds little. A copied
// line of a tile that starts off 128 bytes touches two (20 x 1384 x 1778, X X^T: 97 against 68 us).
inline int64_t pad_line(int64_t cols, int elem_bytes) {
    if (cols * elem_bytes < 512) return pad16(cols, elem_bytes);
    const int64_t v = kLineBytes / elem_bytes;
    return (cols + v - 1) / v * v;
}

inline bool wide16(const void* p, int64_t ld, int64_t cols) {
    return aligned(p, 16) && ld % 8 == 0 && cols % 8 == 0;
}

// the operand itself, or its padded copy in the scratch
Matrix readable(Matrix m, int elem_bytes, Scratch& ws, cudaStream_t stream);

// Largest number of rows of x that linear_few takes. B200, bf16, us on the GPU with the weights in
// L2, few rows / tiles at 1, 16, 32 and 48 rows:
//   4096 -> 8192   9.6 / 31.2    9.3 / 16.3   10.6 / 16.4   11.8 / 16.4
//   1024 -> 1024   4.0 / 6.5     4.2 / 6.6     4.3 / 6.6     5.4 / 6.6
//    512 -> 256    3.8 / 4.9     3.8 / 5.0     4.8 / 5.0     5.7 / 5.0
//    256 -> 512    3.6 / 3.9     4.8 / 4.0     6.4 / 4.0     8.1 / 4.0
//   gated 4096 -> 2 x 8192  23.3 / 36.6  23.8 / 26.2  26.2 / 26.3  27.9 / 26.3
//   gated  256 -> 2 x 512    4.6 / 4.7    4.7 / 4.8    6.4 / 4.9    8.0 / 4.9
// The rule looks at rows alone: narrow layers of 16 to 48 rows lose by it, up to half.
constexpr int kFewRows = 48;
void linear_few(const rune_linear_args& a, const Matrix& x, const Matrix& w, cudaStream_t stream);
void grouped_few(const rune_grouped_linear_args& a, const Matrix& x, const Matrix& w,
                 cudaStream_t stream);

// Host-mapped word that a kernel sets when a wait gave up (ops::check_waits reads it).
unsigned* wait_flag(int device);
unsigned wait_polls();

}  // namespace ops
}  // namespace rune
