// Dense products with a fused epilogue: out[m][n] = act((a_scale * sum_k x[m][k] w[n][k]) * w_scale[n] + bias[n]) + residual[m][n]
// for fp32, fp16, bf16 (fp32 sums, no scales) and int8 (exact int32 sums).
//
// Two kernels, both with w's rows as the matrix instruction's row operand, so that a lane holds four neighbouring n of
// one m. `linear_tile_k`: a block's BM x BN outputs from tiles of 128 bytes of k in LDS, filled by direct loads to LDS
// one tile ahead; the sums go through LDS once so that residual and output move as whole rows. `linear_rows_k`: few
// outputs; the block's waves share out k, operands straight into registers.
#include "pmg_dense.h"

namespace pmg {

struct LinearArgs {
    const void* x;
    const void* w;
    const float* bias;     // [N] or NULL
    const float* w_scale;  // int8: [N] or NULL (ones)
    const void* res;       // [M][N] or NULL
    void* out;
    int64_t M, ldx, ldr, ldo;
    int K, N, ldw;
    int act, res_type, out_type;
    float a_scale;
    int vec_res, vec_out;  // rows of res / out take 16-byte accesses
    uint32_t tiles_n, tiles;
};

// --------------------------------------------------------------------------------------------------------- epilogue
// erf within 1.5e-7 (Abramowitz and Stegun 7.1.26), an eighth of erff's instructions: for outputs of 16 bits, whose
// half step is 2^-12 of the value at the least; fp32 outputs take erff.
__device__ inline float erf_as(float x) {
    const float a = __builtin_fabsf(x);
    const float t = __builtin_amdgcn_rcpf(__builtin_fmaf(0.3275911f, a, 1.0f));
    float p = __builtin_fmaf(1.061405429f, t, -1.453152027f);
    p = __builtin_fmaf(p, t, 1.421413741f);
    p = __builtin_fmaf(p, t, -0.284496736f);
    p = __builtin_fmaf(p, t, 0.254829592f);
    const float e = __builtin_amdgcn_exp2f(-(a * a) * PMG_LOG2E);
    return __builtin_copysignf(__builtin_fmaf(-(p * t), e, 1.0f), x);
}

__device__ inline float activate(float y, int act, bool wide) {
    switch (act) {
        case PMG_ACT_RELU: return y < 0.0f ? 0.0f : y;  // (NaN stays)
        case PMG_ACT_SILU: return silu_fast(y);
        case PMG_ACT_GELU: return 0.5f * y * (1.0f + (wide ? erff(y * 0.70710678f) : erf_as(y * 0.70710678f)));
        case PMG_ACT_GELU_TANH: {
            const float u = 0.7978845608f * __builtin_fmaf(0.044715f * y * y, y, y);
            // (1 + tanh(u)) / 2 = 1 / (1 + exp(-2 u))
            return y * __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(u * (-2.0f * PMG_LOG2E)));
        }
        default: return y;
    }
}

template <class E>
__device__ inline void load8(const E* p, int n, bool vec, float (&v)[8]) {
    if (vec && n == 8) {
        constexpr int C = 16 / sizeof(E);
        typedef E vec_t __attribute__((ext_vector_type(C)));
#pragma unroll
        for (int c = 0; c < 8 / C; ++c) {
            const vec_t t = *(const vec_t*)(p + c * C);
#pragma unroll
            for (int i = 0; i < C; ++i) v[c * C + i] = (float)t[i];
        }
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = i < n ? (float)p[i] : 0.0f;
    }
}
template <class E>
__device__ inline void store8(E* p, int n, bool vec, const float (&v)[8]) {
    if (vec && n == 8) {
        constexpr int C = 16 / sizeof(E);
        typedef E vec_t __attribute__((ext_vector_type(C)));
#pragma unroll
        for (int c = 0; c < 8 / C; ++c) {
            vec_t t;
#pragma unroll
            for (int i = 0; i < C; ++i) t[i] = (E)v[c * C + i];
            *(vec_t*)(p + c * C) = t;
        }
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (i < n) p[i] = (E)v[i];
    }
}

// n <= 8 outputs of row m from column n0 on: v holds scaled sums plus bias.
__device__ inline void finish8(const LinearArgs& a, int64_t m, int n0, int n, float (&v)[8]) {
    const bool wide = a.out_type == PMG_TYPE_F32;
    if (a.act != PMG_ACT_NONE)
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = activate(v[i], a.act, wide);
    if (a.res) {
        float r[8];
        const int64_t o = m * a.ldr + n0;
        if (a.res_type == PMG_TYPE_F32) load8((const float*)a.res + o, n, a.vec_res, r);
        else if (a.res_type == PMG_TYPE_F16) load8((const _Float16*)a.res + o, n, a.vec_res, r);
        else load8((const __bf16*)a.res + o, n, a.vec_res, r);
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = v[i] + r[i];
    }
    const int64_t o = m * a.ldo + n0;
    if (a.out_type == PMG_TYPE_F32) store8((float*)a.out + o, n, a.vec_out, v);
    else if (a.out_type == PMG_TYPE_F16) store8((_Float16*)a.out + o, n, a.vec_out, v);
    else store8((__bf16*)a.out + o, n, a.vec_out, v);
}

// Scale and bias of columns n0 .. n0 + 7 (0 behind N).
template <class T>
__device__ inline void columns8(const LinearArgs& a, int n0, float (&sc)[8], float (&bs)[8]) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const bool in = n0 + i < a.N;
        sc[i] = sizeof(T) == 1 && a.w_scale && in ? a.w_scale[n0 + i] : 1.0f;
        bs[i] = a.bias && in ? a.bias[n0 + i] : 0.0f;
    }
}

// 16 bytes of a row from element k on, element by element: zeros behind K (rows of any alignment).
template <class T>
__device__ inline typename Mat<T>::chunk load_chunk_any(const T* row, int k, int K) {
    typedef T vec_t __attribute__((ext_vector_type(Mat<T>::kPer)));
    vec_t v;
#pragma unroll
    for (int i = 0; i < Mat<T>::kPer; ++i) v[i] = k + i < K ? row[k + i] : (T)0;
    return __builtin_bit_cast(typename Mat<T>::chunk, v);
}

// ------------------------------------------------------------------------------------------------------ tile kernel
// VEC: rows of x and w start on 16 bytes and K is a whole number of 16-byte chunks; the loads go straight to LDS, and
// a chunk behind K or a row behind M or N is given an offset beyond the buffer's record count, which reads zeros.
template <class T, int BM, int BN, int WM, int WN, bool VEC>
__global__ __launch_bounds__(64 * WM * WN) void linear_tile_k(LinearArgs a) {
    constexpr int NT = 64 * WM * WN, KB = 128, KE = KB / (int)sizeof(T);
    constexpr int TM = BM / WM, TN = BN / WN, MT = TM / 32, NTL = TN / 32;
    constexpr int kStage = (BM + BN) * KB;
    typedef typename Mat<T>::chunk chunk;
    typedef typename Mat<T>::acc32 acc32;
    extern __shared__ __attribute__((aligned(16))) char lds[];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int wm = wave / WN, wn = wave % WN;
    const uint32_t tile = xcd_tile(blockIdx.x, a.tiles);
    const int64_t m0 = (int64_t)(tile / a.tiles_n) * BM;
    const int n0 = (int)(tile % a.tiles_n) * BN;
    const T* xb = (const T*)a.x + m0 * a.ldx;
    const T* wb = (const T*)a.w + (int64_t)n0 * a.ldw;
    const int rows_m = a.M - m0 < BM ? (int)(a.M - m0) : BM, rows_n = a.N - n0 < BN ? a.N - n0 : BN;
    const int nk = (a.K + KE - 1) / KE;

    auto fill = [&](int t, int buf) {
        char* base = lds + buf * kStage;
        if constexpr (VEC) {
            const auto rx = __builtin_amdgcn_make_buffer_rsrc((void*)xb, 0, (int)(((int64_t)(rows_m - 1) * a.ldx + a.K) * (int)sizeof(T)), 0x00027000);
            const auto rw = __builtin_amdgcn_make_buffer_rsrc((void*)wb, 0, (int)(((int64_t)(rows_n - 1) * a.ldw + a.K) * (int)sizeof(T)), 0x00027000);
#pragma unroll
            for (int i = 0; i < (BM + BN) / 8 / (WM * WN); ++i) {
                const int g = i * WM * WN + wave;  // 8 rows of x's or w's tile (uniform over the wave)
                const int r = (g < BM / 8 ? g : g - BM / 8) * 8 + (lane >> 3);
                const int c = swz8(r, lane & 7) * Mat<T>::kPer + t * KE;
                const bool isx = g < BM / 8;
                const bool in = c < a.K && r < (isx ? rows_m : rows_n);
                const uint32_t off = in ? (uint32_t)(((int64_t)r * (isx ? a.ldx : (int64_t)a.ldw) + c) * (int)sizeof(T)) : 0x7ffffff0u;
                __builtin_amdgcn_raw_ptr_buffer_load_lds(isx ? rx : rw, (__attribute__((address_space(3))) void*)(base + g * 1024), 16, off, 0, 0, 0);
            }
        } else {
            for (int e = tid; e < (BM + BN) * 8; e += NT) {
                const int r = e >> 3, c = e & 7, k = t * KE + c * Mat<T>::kPer;
                chunk v{};
                if (r < BM) {
                    if (r < rows_m) v = load_chunk_any<T>(xb + r * a.ldx, k, a.K);
                } else if (r - BM < rows_n) {
                    v = load_chunk_any<T>(wb + (int64_t)(r - BM) * a.ldw, k, a.K);
                }
                const int lr = r < BM ? r : r - BM;
                *(chunk*)(base + r * KB + 16 * swz8(lr, c)) = v;
            }
        }
    };

    acc32 acc[MT][NTL];
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int j = 0; j < NTL; ++j) acc[i][j] = acc32{};

    fill(0, 0);
    __syncthreads();
    for (int t = 0; t < nk; ++t) {
        const char* cur = lds + (t & 1) * kStage;
        if (t + 1 < nk) fill(t + 1, (t + 1) & 1);
#pragma unroll
        for (int s = 0; s < 4; ++s) {
            const int r = lane & 31, c = 2 * s + (lane >> 5);
            chunk fx[MT], fw[NTL];
#pragma unroll
            for (int i = 0; i < MT; ++i) {
                const int row = wm * TM + 32 * i + r;
                fx[i] = *(const chunk*)(cur + row * KB + 16 * swz8(row, c));
            }
#pragma unroll
            for (int j = 0; j < NTL; ++j) {
                const int row = wn * TN + 32 * j + r;
                fw[j] = *(const chunk*)(cur + (BM + row) * KB + 16 * swz8(row, c));
            }
#pragma unroll
            for (int i = 0; i < MT; ++i)
#pragma unroll
                for (int j = 0; j < NTL; ++j) acc[i][j] = Mat<T>::mma32(fw[j], fx[i], acc[i][j]);
        }
        __syncthreads();
    }

    // Sums through LDS: 32 rows of the wave's TN columns at a time, in fp32.
    constexpr int LD = TN + 4;
    float* st = (float*)lds + wave * 32 * LD;
    constexpr int LPR = TN / 8, RPP = 64 / LPR;  // lanes a row, rows a pass
    const int nc = n0 + wn * TN + 8 * (lane % LPR);
    const int left = a.N - nc < 8 ? a.N - nc : 8;
    float sc[8], bs[8];
    columns8<T>(a, nc, sc, bs);
#pragma unroll
    for (int i = 0; i < MT; ++i) {
#pragma unroll
        for (int j = 0; j < NTL; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                v4f v;
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    if constexpr (sizeof(T) == 1) v[q] = (float)acc[i][j][4 * e + q];
                    else v[q] = acc[i][j][4 * e + q];
                }
                *(v4f*)(st + (lane & 31) * LD + 32 * j + 8 * e + 4 * (lane >> 5)) = v;
            }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
#pragma unroll
        for (int p = 0; p < 32 / RPP; ++p) {
            const int r = p * RPP + lane / LPR;
            const int64_t m = m0 + wm * TM + 32 * i + r;
            const v4f u0 = *(const v4f*)(st + r * LD + 8 * (lane % LPR)), u1 = *(const v4f*)(st + r * LD + 8 * (lane % LPR) + 4);
            float v[8];
#pragma unroll
            for (int q = 0; q < 8; ++q) {
                const float s = q < 4 ? u0[q & 3] : u1[q & 3];
                v[q] = sizeof(T) == 1 ? (s * a.a_scale) * sc[q] + bs[q] : s + bs[q];
            }
            if (m < a.M && left > 0) finish8(a, m, nc, left, v);
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
    }
}

// ------------------------------------------------------------------------------------------------------- few outputs
// 16 MT rows of x by 16 rows of w a block, k shared out over the block's NW waves in steps of 64 bytes; each wave holds
// its sums, which are added in wave order through LDS.
template <class T, int MT, int NW, bool VEC>
__global__ __launch_bounds__(64 * NW) void linear_rows_k(LinearArgs a) {
    typedef typename Mat<T>::chunk chunk;
    typedef typename Mat<T>::acc16 acc16;
    constexpr int PER = Mat<T>::kPer, U = 4;
    typedef decltype(acc16{}[0] + 0) sum_t;
    __shared__ sum_t red[NW][16 * MT][17];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, r = lane & 15, g = lane >> 4;
    const uint32_t tile = blockIdx.x;
    const int64_t m0 = (int64_t)(tile / a.tiles_n) * 16 * MT;
    const int n0 = (int)(tile % a.tiles_n) * 16;
    const T* wr = (const T*)a.w + (int64_t)(n0 + r < a.N ? n0 + r : a.N - 1) * a.ldw;
    const T* xr[MT];
#pragma unroll
    for (int i = 0; i < MT; ++i) {
        const int64_t m = m0 + 16 * i + r;
        xr[i] = (const T*)a.x + (m < a.M ? m : a.M - 1) * a.ldx;
    }
    const int nsteps = (a.K + 4 * PER - 1) / (4 * PER);
    acc16 acc[MT];
#pragma unroll
    for (int i = 0; i < MT; ++i) acc[i] = acc16{};
    auto get = [&](const T* row, int k) -> chunk {
        if constexpr (VEC) {
            // (a chunk behind K reads the row's first one instead and counts as zeros)
            const chunk v = *(const chunk*)(row + (k < a.K ? k : 0));
            return k < a.K ? v : chunk{};
        } else {
            return load_chunk_any<T>(row, k, a.K);
        }
    };
    for (int s0 = wave; s0 < nsteps; s0 += NW * U) {
        chunk fw[U], fx[U][MT];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int k = (4 * (s0 + u * NW) + g) * PER;
            fw[u] = get(wr, k);
#pragma unroll
            for (int i = 0; i < MT; ++i) fx[u][i] = get(xr[i], k);
        }
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int i = 0; i < MT; ++i) acc[i] = Mat<T>::mma16(fw[u], fx[u][i], acc[i]);
    }
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) red[wave][16 * i + r][4 * g + e] = acc[i][e];
    __syncthreads();
    // 8 outputs a thread
    const int t = threadIdx.x;
    if (t < 16 * MT * 2) {
        const int row = t >> 1, c = 8 * (t & 1);
        const int64_t m = m0 + row;
        const int left = a.N - (n0 + c) < 8 ? a.N - (n0 + c) : 8;
        if (m < a.M && left > 0) {
            float sc[8], bs[8], v[8];
            columns8<T>(a, n0 + c, sc, bs);
#pragma unroll
            for (int q = 0; q < 8; ++q) {
                sum_t s = 0;
#pragma unroll
                for (int w = 0; w < NW; ++w) s = s + red[w][row][c + q];
                v[q] = sizeof(T) == 1 ? ((float)s * a.a_scale) * sc[q] + bs[q] : (float)s + bs[q];
            }
            finish8(a, m, n0 + c, left, v);
        }
    }
}

// ------------------------------------------------------------------------------------------------------------- launch
template <class T, int BM, int BN, int WM, int WN, bool VEC>
static int launch_tile(LinearArgs& a, hipStream_t s) {
    constexpr int kStage = (BM + BN) * 128, kOut = WM * WN * 32 * (BN / WN + 4) * 4;
    const int nk = (a.K * (int)sizeof(T) + 127) / 128;
    int bytes = kStage * (nk > 1 ? 2 : 1);
    if (bytes < kOut) bytes = kOut;
    const int64_t tm = (a.M + BM - 1) / BM;
    a.tiles_n = (uint32_t)((a.N + BN - 1) / BN);
    PMG_REQUIRE(tm * a.tiles_n < (int64_t)1 << 31, "too many outputs");
    a.tiles = (uint32_t)(tm * a.tiles_n);
    hipLaunchKernelGGL((linear_tile_k<T, BM, BN, WM, WN, VEC>), dim3(a.tiles), dim3(64 * WM * WN), bytes, s, a);
    return check_launch("linear_tile_k");
}

template <class T, int MT, int NW, bool VEC>
static int launch_rows(LinearArgs& a, hipStream_t s) {
    const int64_t tm = (a.M + 16 * MT - 1) / (16 * MT);
    a.tiles_n = (uint32_t)((a.N + 15) / 16);
    PMG_REQUIRE(tm * a.tiles_n < (int64_t)1 << 31, "too many outputs");
    a.tiles = (uint32_t)(tm * a.tiles_n);
    hipLaunchKernelGGL((linear_rows_k<T, MT, NW, VEC>), dim3(a.tiles), dim3(64 * NW), 0, s, a);
    return check_launch("linear_rows_k");
}

template <class T, bool VEC>
static int launch_linear(LinearArgs& a, hipStream_t s) {
    const int64_t t64 = ((a.M + 63) / 64) * ((a.N + 63) / 64), t128 = ((a.M + 127) / 128) * ((a.N + 127) / 128);
    if (a.M <= 16) return launch_rows<T, 1, 8, VEC>(a, s);
    if (t64 < 128) return launch_rows<T, 2, 4, VEC>(a, s);
    if (t128 < 512 || a.N <= 64) return launch_tile<T, 64, 64, 2, 2, VEC>(a, s);
    return launch_tile<T, 128, 128, 2, 2, VEC>(a, s);
}

}  // namespace pmg

using namespace pmg;

extern "C" int pmg_linear(const pmg_linear_args* p, void* stream) {
    PMG_REQUIRE(p, "null args");
    const pmg_linear_args& q = *p;
    auto bytes = [](int t) { return t == PMG_TYPE_F32 ? 4 : t == PMG_TYPE_I8 ? 1 : 2; };
    PMG_REQUIRE(q.type >= PMG_TYPE_F32 && q.type <= PMG_TYPE_I8, "type must be f32, f16, bf16 or i8");
    PMG_REQUIRE(q.out_type >= PMG_TYPE_F32 && q.out_type <= PMG_TYPE_BF16, "out_type must be f32, f16 or bf16");
    PMG_REQUIRE(q.act >= PMG_ACT_NONE && q.act <= PMG_ACT_GELU_TANH, "unknown activation");
    PMG_REQUIRE(q.M >= 0 && q.M < (int64_t)1 << 31, "M out of range");
    PMG_REQUIRE(q.K >= 1 && q.K <= 131072 && q.N >= 1 && q.N <= (1 << 24), "K must be 1 .. 131072 and N 1 .. 2^24");
    const int es = bytes(q.type);
    PMG_REQUIRE(q.ldx >= q.K && q.ldx <= (1 << 22) / es && q.ldo >= q.N && (!q.residual || q.ldr >= q.N), "row strides must cover the row (x: at most 4 MiB)");
    if (q.M == 0) return PMG_OK;
    PMG_REQUIRE(q.x && q.w && q.out, "null buffer");
    const auto at = [](const void* v, int n) { return (reinterpret_cast<uintptr_t>(v) & (uintptr_t)(n - 1)) == 0; };
    PMG_REQUIRE(at(q.x, es) && at(q.w, es) && at(q.out, bytes(q.out_type)) && at(q.bias, 4) && at(q.w_scale, 4), "buffers must be aligned to their elements");
    LinearArgs a{};
    a.x = q.x;
    a.w = q.w;
    a.bias = q.bias;
    a.w_scale = q.w_scale;
    a.res = q.residual;
    a.out = q.out;
    a.M = q.M;
    a.K = q.K;
    a.N = q.N;
    a.ldw = q.K;
    a.ldx = q.ldx;
    a.ldr = q.ldr;
    a.ldo = q.ldo;
    a.act = q.act;
    a.out_type = q.out_type;
    a.res_type = q.residual_type;
    a.a_scale = q.a_scale;
    if (q.residual) {
        PMG_REQUIRE(q.residual_type >= PMG_TYPE_F32 && q.residual_type <= PMG_TYPE_BF16, "residual_type must be f32, f16 or bf16");
        PMG_REQUIRE(at(q.residual, bytes(q.residual_type)), "buffers must be aligned to their elements");
        a.vec_res = at(q.residual, 16) && q.ldr * bytes(q.residual_type) % 16 == 0;
    }
    a.vec_out = at(q.out, 16) && q.ldo * bytes(q.out_type) % 16 == 0;
    const bool vec = at(q.x, 16) && at(q.w, 16) && q.ldx * es % 16 == 0 && (int64_t)q.K * es % 16 == 0;
    hipStream_t s = (hipStream_t)stream;
    switch (q.type) {
        case PMG_TYPE_F32: return vec ? launch_linear<float, true>(a, s) : launch_linear<float, false>(a, s);
        case PMG_TYPE_F16: return vec ? launch_linear<_Float16, true>(a, s) : launch_linear<_Float16, false>(a, s);
        case PMG_TYPE_BF16: return vec ? launch_linear<__bf16, true>(a, s) : launch_linear<__bf16, false>(a, s);
        default: return vec ? launch_linear<int8_t, true>(a, s) : launch_linear<int8_t, false>(a, s);
    }
}
