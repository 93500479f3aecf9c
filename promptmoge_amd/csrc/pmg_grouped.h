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

enum { kExperts = 0, kAdapters = 1, kRowAdapters = 2, kFewRows = 3 };

// ------------------------------------------------------------------------------------------------- which kernel takes a call
// Tiles by what a CU's share of them costs, in microseconds, k in units of 128 bytes, fitted to the times of 400 (16 bits) and 250
// (fp32) products of random sizes: 2 % and 0.6 % above the best shape's by the mean, a third and 7 % at the most (uneven segments may
// end in one tile more than the chip holds at a time). Measured, us, rows gathered, 8 segments or as many as said:
//   bf16                       64 x 64, 2 places   3 places   64 x 128   128 x 128   128 x 256   192 x 128
//   300 x 1024 to 1024                9.6             9.9       10.7        13.6        21.4        16.6
//   1000 x 1024 to 1024              13.0            12.0       13.8        14.3        22.0        17.5
//   4800 x 1024 to 1024, by 4        26.2            23.9       22.3        21.5        25.2        20.2
//   9600 x 1024 to 4096, gelu       185             187        163         122         117         147
//   9600 x 4096 to 1024             135             140        111         110         125         109
//   76800 x 128 to 512, by 4, gelu   55.4            54.9       45.9        45.1        40.9        60.6
//   600 x 4096 to 512, by 16         34.2            24.2       39.2        43.2        63.9        47.5
//   fp32                       64 x 64, 2 places   3 of 64 bytes   64 x 128
//   600 x 512 to 512                 15.6            16.8           22.7
//   2048 x 2048 to 512, by 1         48.3            52.8           73.3
//   9600 x 256 to 1024               61.8            58.2           55.5
//   76800 x 64 to 128, by 4          24.7            22.4           23.4
// A library's product of 9600 x 1024 bf16 by one matrix to 4096 without an epilogue takes 97, of 2048 x 2048 fp32 to 512 35. Rows of
// any alignment take 64 x 64.
inline int tile_shape(bool fp32, bool vec, int kind, int64_t P, int64_t S, int K, int N) {
    if (!vec) return 0;
    const double k = (double)(((int64_t)K * (fp32 ? 4 : 2) + 127) / 128);
    const double ends = kind == kRowAdapters ? 0.0 : (double)(S - 1);  // as many segments may end inside a tile
    const auto rounds = [&](int bm, int bn, double least) {
        // fp32: the mean if none do, half, and all; else if a quarter and if three do. Fewer than `whole` are counted whole.
        const int n = fp32 ? 3 : 2;
        const double whole = fp32 ? 2.0 : 6.0;
        double sum = 0.0;
        for (int i = 0; i < n; ++i) {
            const double some = fp32 ? 0.5 * i : 0.25 + 0.5 * i;
            const double q = (__builtin_ceil((double)P / bm) + some * ends) * ((N + bn - 1) / bn) / 256.0;
            sum += q < whole ? __builtin_ceil(q) : q + 0.5;
        }
        return sum < n * least ? least : sum / n;
    };
    const double f[3] = {5.5 + 0.129 * k + rounds(64, 64, 1.0) * (0.489 * k + 1.5), 5.4 + 0.263 * k + rounds(64, 64, 1.0) * (0.477 * k + 0.8),
                         5.2 + 0.097 * k + rounds(64, 128, 1.0) * (k + 1.7)};
    const double h[6] = {1.7 + rounds(64, 64, 2.0) * (0.21 * k + 1.19), 3.2 + rounds(64, 64, 2.0) * (0.17 * k + 1.02),
                         1.1 + rounds(64, 128, 2.0) * (0.331 * k + 1.72), 4.3 + rounds(128, 128, 1.0) * (0.545 * k + 1.95),
                         6.1 + rounds(128, 256, 1.0) * (0.868 * k + 3.2), 1.5 + rounds(192, 128, 1.0) * (0.78 * k + 6.1)};
    const double* c = fp32 ? f : h;
    int best = 0;
    for (int i = 1; i < (fp32 ? 3 : 6); ++i)
        if (c[i] < c[best]) best = i;
    return best;
}
// Rows, columns and LDS places of each.
constexpr int kShapes32[6][3] = {{64, 64, 2}, {64, 64, 3}, {64, 128, 2}};
constexpr int kShapes16[6][3] = {{64, 64, 2}, {64, 64, 3}, {64, 128, 2}, {128, 128, 2}, {128, 256, 3}, {192, 128, 3}};

// Experts: 16 positions a block (grouped_rows_k) where segments have no more by the mean. Row adapters: where that is 512 blocks or fewer.
inline bool few_a_segment(int64_t P, int64_t S) { return P <= 16 * S; }
constexpr int kFew = 8;  // rows that lora_few_k takes at the most
inline bool few_outputs(int64_t P, int N) { return (P + 15) / 16 * ((N + 15) / 16) <= 512; }

template <class T>
int launch_experts(GroupArgs& a, bool vec, hipStream_t s);
template <class T>
int launch_lora(GroupArgs& a, bool vec, bool by_segment, hipStream_t s);

}  // namespace pmg
