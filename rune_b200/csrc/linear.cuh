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

__device__ __forceinline__ void mma_f16(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc,
                                        bool accumulate) {
    asm volatile(
        "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
        " tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}\n"
        ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"((uint32_t)accumulate)
        : "memory");
}

__device__ __forceinline__ void mma_f8(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc,
                                       bool accumulate) {
    asm volatile(
        "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
        " tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n}\n"
        ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"((uint32_t)accumulate)
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

// Largest number of rows of x that linear_few takes. Measured on B200, bf16, against the 128-row
// tiles: 16 rows x 4096 -> 8192 15.8 against 19.3 us, x 1024 -> 1024 5.3 against 8.0; 64 rows
// 19.2 against 19.3 and 6.5 against 8.0, but x 256 -> 512 10.9 against 5.8.
constexpr int kFewRows = 48;
void linear_few(const rune_linear_args& a, const Matrix& x, const Matrix& w, cudaStream_t stream);

// Host-mapped word that a kernel sets when a wait gave up; check_waits throws if it is set.
unsigned* wait_flag(int device);
void check_waits(int device);

}  // namespace ops
}  // namespace rune
