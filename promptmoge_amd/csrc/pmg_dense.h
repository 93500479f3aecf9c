// Element types, matrix instructions and conversions shared by the dense operators (linear, norm + rotation, attention).
#pragma once
#include "pmg_common.h"

namespace pmg {

typedef float v16f __attribute__((ext_vector_type(16)));
typedef int v16i __attribute__((ext_vector_type(16)));
typedef float v8f __attribute__((ext_vector_type(8)));

// A 16-byte operand chunk of one matrix row, and the product of two such chunks per lane. In the 32 x 32 form lane l
// holds row l & 31 and chunk 2 s + (l >> 5) of step s; in the 16 x 16 form row l & 15 and chunk 4 s + (l >> 4). The
// instruction's own order of k inside a step is the same for both operands, so any assignment of k to (lane, element)
// gives the same sum of products: fp32 spends a chunk's four values on four instructions.
// Output: 32 x 32: column l & 31, row (e & 3) + 8 (e >> 2) + 4 (l >> 5) of element e; 16 x 16: column l & 15, row
// 4 (l >> 4) + e. Sums are held in fp32, or exactly in int32 for int8.
template <class T>
struct Mat;

template <>
struct Mat<_Float16> {
    typedef v8h chunk;
    typedef v16f acc32;
    typedef v4f acc16;
    static constexpr int kPer = 8;  // elements a chunk
    __device__ static inline acc32 mma32(chunk a, chunk b, acc32 c) { return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0); }
    __device__ static inline acc16 mma16(chunk a, chunk b, acc16 c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }
};
template <>
struct Mat<__bf16> {
    typedef v8bf chunk;
    typedef v16f acc32;
    typedef v4f acc16;
    static constexpr int kPer = 8;
    __device__ static inline acc32 mma32(chunk a, chunk b, acc32 c) { return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0); }
    __device__ static inline acc16 mma16(chunk a, chunk b, acc16 c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }
};
template <>
struct Mat<int8_t> {
    typedef v4i chunk;
    typedef v16i acc32;
    typedef v4i acc16;
    static constexpr int kPer = 16;
    __device__ static inline acc32 mma32(chunk a, chunk b, acc32 c) { return __builtin_amdgcn_mfma_i32_32x32x32_i8(a, b, c, 0, 0, 0); }
    __device__ static inline acc16 mma16(chunk a, chunk b, acc16 c) { return __builtin_amdgcn_mfma_i32_16x16x64_i8(a, b, c, 0, 0, 0); }
};
template <>
struct Mat<float> {
    typedef v4f chunk;
    typedef v16f acc32;
    typedef v4f acc16;
    static constexpr int kPer = 4;
    __device__ static inline acc32 mma32(chunk a, chunk b, acc32 c) {
#pragma unroll
        for (int i = 0; i < 4; ++i) c = __builtin_amdgcn_mfma_f32_32x32x2f32(a[i], b[i], c, 0, 0, 0);
        return c;
    }
    __device__ static inline acc16 mma16(chunk a, chunk b, acc16 c) {
#pragma unroll
        for (int i = 0; i < 4; ++i) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a[i], b[i], c, 0, 0, 0);
        return c;
    }
};

// A grid's threads are counted in 32 bits (a larger launch is cut off without an error): blocks of `threads` it may have.
constexpr int64_t grid_blocks(int threads) { return 0xffffffffll / threads; }

// The XCD a block runs on is its index modulo 8: blocks of one XCD take consecutive tiles, which share operands in
// that XCD's L2. Tile of block `id` of n (a permutation of 0 .. n - 1).
__device__ inline uint32_t xcd_tile(uint32_t id, uint32_t n) {
    const uint32_t x = id & 7u, i = id >> 3, q = n >> 3, r = n & 7u;
    return x * q + (x < r ? x : r) + i;
}

// Which 16-byte slot of its LDS row (of `CPR` 16-byte chunks) chunk c of row `row` is kept in. The rows that a 16-byte read of
// 32 rows at one chunk index serves at a time (0-3, 12-15, 20-23, 24-27 and the other half) lie in different banks;
// rows 32 apart are kept alike.
template <int CPR>
__device__ inline int swizzle(int row, int c) {
    if constexpr (CPR == 4) return c ^ ((row >> 2) & 3);
    else if constexpr (CPR == 8) return c ^ ((row ^ ((row >> 3) & 3)) & 7);
    else return c ^ (row & 15);
}

// 16 bytes a lane from memory to LDS, lane after lane from `to` (the same in every lane) on. Written out, for the compiler
// would wait for these loads before the next LDS read of any kind; loads_landed() waits until at most N of the wave's
// loads are still on their way (they land in order).
__device__ inline uint32_t lds_address(const void* to) {
    return __builtin_amdgcn_readfirstlane((uint32_t)(uintptr_t)(__attribute__((address_space(3))) const void*)to);
}
__device__ inline void load_to_lds(const void* from, uint32_t to) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" : : "s"(to), "v"(from) : "memory", "m0");
}
// The same from a buffer: at byte `off` (a lane's) + `more` (the wave's); zeros from its end on.
__device__ inline void buffer_to_lds(v4i rsrc, uint32_t off, uint32_t more, uint32_t to) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, %3 offen lds" : : "s"(to), "v"(off), "s"(rsrc), "s"(more) : "memory", "m0");
}
__device__ inline v4i buffer_of(const void* base, uint32_t bytes) {
    const uint64_t p = (uint64_t)base;
    return v4i{(int)(uint32_t)p, (int)(uint32_t)(p >> 32), (int)bytes, 0x00027000};
}
template <int N>
__device__ inline void loads_landed() {
    asm volatile("s_waitcnt vmcnt(%0)" : : "n"(N) : "memory");
}

// A barrier of the block behind which every wave's loads to LDS but its last N, and every LDS access before, are done.
template <int N>
__device__ inline void landed_barrier() {
    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" : : "n"(N) : "memory");
}

}  // namespace pmg
