// Products whose rows are grouped by segments: experts' products (each segment has a w of its own) and a shared projection
// with low-rank adapters (each segment has an adapter). Segment s of S holds the positions offsets[s] .. offsets[s + 1] - 1.
#pragma once
#include "pmg_epilogue.h"
#include "pmg_pieces.h"

namespace pmg {

struct GroupArgs : Epilogue, Pieces {  // (tag: the segments' adapters, which may have no offsets: a row a segment)
    const void* x;            // [x_rows] rows of ldx
    const void* w;            // [N][K], the next segment's w_next elements on
    const float* bias;        // [N] or NULL, the next segment's b_next elements on
    const int32_t* index;     // row of x of each position, or NULL
    const int32_t* out_index; // row of the result of each position, or NULL
    int64_t x_rows, out_rows, ldx, w_next, b_next;
    int K, N;
    int fresh;                // rows that no position names are set to 0
    // adapters: scale[i] (x down[i]^T) of each row, as the kernel that uses it reads it, then up [adapters][N][r]
    const void* low;          // NULL: lora_few_k forms them itself
    float* low_factor;        // fp16 parts: what a row's sums of parts are multiplied by
    int32_t* row_adapter;     // each row's adapter, or -1
    const void* down;         // [adapters][r][K]
    const void* up;
    const float* scale;       // [adapters] or NULL
    int r, adapters, vec_up;
    uint32_t tiles_n, tiles, id0;
};

// The row of x that position p reads (any value where there is none), and whether it is one.
__device__ inline int row_in(const GroupArgs& a, int p) { return a.index ? a.index[p] : p; }
__device__ inline bool in_x(const GroupArgs& a, int row) { return row >= 0 && row < a.x_rows; }
// Where position p's result goes, `from` its row of x: a row of the result, -1 (nowhere), or -2 - row: a row that is set to 0.
__device__ inline int row_out(const GroupArgs& a, int p, int from) {
    const int o = a.out_index ? a.out_index[p] : p;
    if (!a.out_index) return in_x(a, from) ? p : a.fresh ? -2 - p : -1;
    return in_x(a, from) && o >= 0 && o < a.out_rows ? o : -1;
}
__device__ inline int adapter_of(const GroupArgs& a, int tag) { return tag >= 0 && tag < a.adapters ? tag : -1; }

// Bias of columns n .. n + 7 of segment s (0 behind N).
__device__ inline void bias8(const GroupArgs& a, int s, int n, float (&b)[8]) {
#pragma unroll
    for (int i = 0; i < 8; ++i) b[i] = 0.0f;
    if (!a.bias) return;
    const float* p = a.bias + (int64_t)s * a.b_next + n;
    if (n + 8 <= a.N) {
#pragma unroll
        for (int i = 0; i < 8; ++i) b[i] = p[i];
    } else {
        for (int i = 0; i < a.N - n; ++i) {
            const float v = p[i];
#pragma unroll
            for (int q = 0; q < 8; ++q) b[q] = q == i ? v : b[q];
        }
    }
}

// n <= 8 zeros in row m of the result from column n0 on.
__device__ inline void zero8(const GroupArgs& a, int64_t m, int n0, int n) {
    const float v[8] = {};
    const int64_t o = m * a.ldo + n0;
    if (a.out_type == PMG_TYPE_F32) store8((float*)a.out + o, n, a.vec_out, v);
    else store8((_Float16*)a.out + o, n, a.vec_out, v);  // (0 is the same in both 16-bit types)
}

// v += h up[ad]^T for columns n0 .. n0 + n - 1, in fp32: r products a value, one behind the other.
template <class T>
__device__ inline void add_low8(const GroupArgs& a, int ad, const float* h, int n0, int n, float (&v)[8]) {
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
// The same of row m's low products and adapter, as lora_low_k wrote them.
template <class T>
__device__ inline void add_low(const GroupArgs& a, int64_t m, int n0, int n, float (&v)[8]) {
    const int ad = a.row_adapter[m];
    if ((uint32_t)ad >= (uint32_t)a.adapters) return;  // (none; or where offsets fall and nothing wrote it)
    add_low8<T>(a, ad, (const float*)a.low + m * a.r, n0, n, v);
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
