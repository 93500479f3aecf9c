// Products whose rows are grouped by segments: experts' products (each segment has a w of its own) and a shared projection
// with low-rank adapters (each segment has an adapter). Segment s of S holds the positions offsets[s] .. offsets[s + 1] - 1.
#pragma once
#include "pmg_epilogue.h"

namespace pmg {

struct GroupArgs : Epilogue {
    const void* x;            // [x_rows] rows of ldx
    const void* w;            // [N][K], the next segment's w_next elements on
    const float* bias;        // [N] or NULL, the next segment's b_next elements on
    const int64_t* offsets;   // [S + 1]; adapters may have none: a row a segment
    const int32_t* index;     // row of x of each position, or NULL
    const int32_t* out_index; // row of the result of each position, or NULL
    int64_t x_rows, out_rows, S, ldx, w_next, b_next;
    int P, K, N;
    int fresh;                // rows that no position names are set to 0
    // adapters: scale[i] (x down[i]^T) of each row, as the kernel that uses it reads it, then up [adapters][N][r]
    const void* low;
    float* low_factor;        // fp16 parts: what a row's sums of parts are multiplied by
    int32_t* row_adapter;     // each row's adapter, or -1
    const void* down;         // [adapters][r][K]
    const void* up;
    const float* scale;       // [adapters] or NULL
    const int32_t* adapter;   // [S]
    int r, adapters, vec_up;
    uint32_t tiles_n, tiles, id0;
};

// Positions [0, P) fall into S + 2 pieces: those in front of segment 0, the segments, those behind the last. Piece j starts at
// bound(j). Tiles of BM positions start where a piece starts; piece j's have the numbers bound(j) / BM + j and up, so that a
// tile's piece is found without a sum over the pieces (a piece may have a number more than it has tiles): P / BM + S + 2 in all.
__device__ inline int piece_bound(const GroupArgs& a, int64_t j) {
    if (j <= 0) return 0;
    if (j > a.S + 1) return a.P;
    const int64_t o = a.offsets[j - 1];
    return o < 0 ? 0 : o > a.P ? a.P : (int)o;
}
struct Piece {
    int first, n, s;  // positions first .. first + n - 1 (n < 1: none) of segment s (-1: of none)
};
// A wave looks at 64 pieces at a time; all lanes return the same. Where offsets fall, some tile within [0, P).
template <int BM>
__device__ inline Piece piece_of(const GroupArgs& a, uint32_t id) {
    const int lane = threadIdx.x & 63;
    int64_t lo = 0, n = a.S + 2;
    while (n > 1) {
        const int64_t step = (n + 63) >> 6, c = lo + lane * step;
        const bool in = lane * step < n && (int64_t)((uint32_t)piece_bound(a, c) / BM) + c <= (int64_t)id;
        const uint64_t not_in = ~__ballot(in);
        int64_t cnt = not_in ? __builtin_ctzll(not_in) : 64;
        cnt = cnt < 1 ? 0 : cnt - 1;
        lo += cnt * step;
        n = n - cnt * step < step ? n - cnt * step : step;
    }
    const int p0 = piece_bound(a, lo), p1 = piece_bound(a, lo + 1);
    const int64_t first = p0 + ((int64_t)id - ((int64_t)((uint32_t)p0 / BM) + lo)) * BM;
    Piece p;
    p.n = first < p0 || first >= p1 ? 0 : p1 - first < BM ? (int)(p1 - first) : BM;
    p.first = p.n ? (int)first : 0;
    p.s = lo >= 1 && lo <= a.S ? (int)(lo - 1) : -1;
    p.first = __builtin_amdgcn_readfirstlane(p.first);
    p.n = __builtin_amdgcn_readfirstlane(p.n);
    p.s = __builtin_amdgcn_readfirstlane(p.s);
    return p;
}
inline uint32_t piece_tiles(int64_t P, int64_t S, int BM) { return (uint32_t)(P / BM + S + 2); }

// The row of x that position p reads, or -1 (absent).
__device__ inline int64_t row_in(const GroupArgs& a, int p) {
    if (!a.index) return p;
    const int32_t i = a.index[p];
    return i >= 0 && i < a.x_rows ? i : -1;
}
// Where position p's result goes: a row of the result, -1 (nowhere), or -2 - row: a row that is set to 0.
__device__ inline int row_out(const GroupArgs& a, int p) {
    const bool there = row_in(a, p) >= 0;
    if (!a.out_index) return there ? p : a.fresh ? -2 - p : -1;
    const int32_t o = a.out_index[p];
    return there && o >= 0 && o < a.out_rows ? o : -1;
}
__device__ inline int adapter_of(const GroupArgs& a, int s) {
    if (s < 0) return -1;
    const int i = a.adapter[s];
    return i >= 0 && i < a.adapters ? i : -1;
}

// Bias of columns n .. n + 7 of segment s (0 behind N).
__device__ inline void bias8(const GroupArgs& a, int s, int n, float (&b)[8]) {
    const float* p = a.bias ? a.bias + (int64_t)s * a.b_next : nullptr;
#pragma unroll
    for (int i = 0; i < 8; ++i) b[i] = p && n + i < a.N ? p[n + i] : 0.0f;
}

// n <= 8 zeros in row m of the result from column n0 on.
__device__ inline void zero8(const GroupArgs& a, int64_t m, int n0, int n) {
    const float v[8] = {};
    const int64_t o = m * a.ldo + n0;
    if (a.out_type == PMG_TYPE_F32) store8((float*)a.out + o, n, a.vec_out, v);
    else store8((_Float16*)a.out + o, n, a.vec_out, v);  // (0 is the same in both 16-bit types)
}

// v += low[m] up[row m's adapter]^T for columns n0 .. n0 + n - 1, in fp32: r products a value, one behind the other.
template <class T>
__device__ inline void add_low(const GroupArgs& a, int64_t m, int n0, int n, float (&v)[8]) {
    const int ad = a.row_adapter[m];
    if ((uint32_t)ad >= (uint32_t)a.adapters) return;  // (none; or where offsets fall and nothing wrote it)
    const float* h = (const float*)a.low + m * a.r;
    const T* u = (const T*)a.up + ((int64_t)ad * a.N + n0) * a.r;
    typedef typename Mat<T>::chunk chunk;
    typedef T vec_t __attribute__((ext_vector_type(Mat<T>::kPer)));
    constexpr int PER = Mat<T>::kPer;
    if (a.vec_up && n == 8) {
        for (int j = 0; j < a.r; j += PER) {
            vec_t c[8];
#pragma unroll
            for (int q = 0; q < 8; ++q) c[q] = __builtin_bit_cast(vec_t, *(const chunk*)(u + q * a.r + j));
#pragma unroll
            for (int i = 0; i < PER; ++i) {
                const float t = h[j + i];
#pragma unroll
                for (int q = 0; q < 8; ++q) v[q] = __builtin_fmaf(t, (float)c[q][i], v[q]);
            }
        }
    } else {
        for (int j = 0; j < a.r; ++j) {
            const float t = h[j];
#pragma unroll
            for (int q = 0; q < 8; ++q)
                if (q < n) v[q] = __builtin_fmaf(t, (float)u[q * a.r + j], v[q]);
        }
    }
}

// Parts that a type's low products are carried in: their sum is fp32's value to 2^-24 of it (fp16: of the row's largest).
template <class T>
constexpr int kParts = sizeof(T) == 4 ? 1 : __is_same(T, __bf16) ? 3 : 2;

enum { kExperts = 0, kAdapters = 1, kRowAdapters = 2 };

template <class T>
int launch_experts(GroupArgs& a, bool vec, hipStream_t s);
template <class T>
int launch_lora(GroupArgs& a, bool vec, bool by_segment, hipStream_t s);

}  // namespace pmg
