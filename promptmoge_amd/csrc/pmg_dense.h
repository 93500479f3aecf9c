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

// The XCD a block runs on is its index modulo 8: blocks of one XCD take consecutive tiles, which share operands in
// that XCD's L2. Tile of block `id` of n (a permutation of 0 .. n - 1).
__device__ inline uint32_t xcd_tile(uint32_t id, uint32_t n) {
    const uint32_t x = id & 7u, i = id >> 3, q = n >> 3, r = n & 7u;
    return x * q + (x < r ? x : r) + i;
}

// Which 16-byte slot of its LDS row chunk `c` of row `row` is kept in (an exclusive or within the row's 8 slots):
// 8, and 16, consecutive rows read at one chunk index lie in different banks.
__device__ inline int swz8(int row, int c) { return c ^ ((row ^ (row >> 3)) & 7); }

}  // namespace pmg
