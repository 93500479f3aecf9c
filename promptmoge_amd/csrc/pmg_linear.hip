// Dense products with a fused epilogue: out[m][n] = act((a_scale * sum_k x[m][k] w[n][k]) * w_scale[n] + bias[n]) + residual[m][n]
// for fp32, fp16, bf16 (fp32 sums, no scales) and int8 (exact int32 sums).
//
// Two kernels, both with w's rows as the matrix instruction's row operand, so that a lane holds four neighbouring n of
// one m. `linear_tile_k`: a block's BM x BN outputs from tiles of KB bytes of k (64 or 128) in NS LDS buffers, filled by
// direct loads to LDS several tiles ahead; the sums go through LDS once so that residual and output move as whole rows.
// `linear_rows_k`: few outputs; the block's waves share out k, operands straight into registers.
//
// Measured (MI355X), and what bounds it: 4800 x 1024 bf16 to 4096 columns, gelu: 54 us, 745 TFLOP/s (the 16-bit tiles take
// what the chip's power leaves of the matrix units' rate, and the epilogue after them; a library's product without an
// epilogue takes 50); one row of 1024 fp16 to 1024: 4.2 us, a load's latency four times over; 76,800 rows of 64 fp32 to
// 128, silu: 22.3 us (59 MB; matrix units 8 us, loads and epilogue of blocks of two tiles of k lie one behind the other).
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
// gelu(y) = max(y, 0) - |y| q(|y|), q(a) = erfc(a / sqrt 2) / 2 = exp(-a^2 / 2) t P(t), t = 1 / (1 + 0.3 a), for outputs of 16
// bits. P, of degree 5, is a least-squares fit reweighted towards the least largest error, against the relative error of q: within
// 2.6e-5 of gelu(y) for y down to -13.2 (1.0e-5 above -3, 1.5e-6 above -1), evaluated in fp32; a 16-bit result's half step is
// 2.4e-4 at the least. (A form whose absolute error is small instead is off by two half steps of fp16 at y = -4.) fp32 outputs take
// erff, several times as long.
__device__ inline float gelu_16(float y) {
    const float x = __builtin_fminf(y, 3.0e38f);  // (+inf: 0 times it would be NaN; -inf and NaN give NaN, as -inf times 0 does)
    const float t = __builtin_amdgcn_rcpf(__builtin_fmaf(0.3f, __builtin_fabsf(x), 1.0f));
    float p = __builtin_fmaf(-0.07936996565f, t, 0.2220676572f);
    p = __builtin_fmaf(p, t, -0.02275388003f);
    p = __builtin_fmaf(p, t, 0.1466454889f);
    p = __builtin_fmaf(p, t, 0.1133136998f);
    p = __builtin_fmaf(p, t, 0.1200967116f);
    const float q = (p * t) * __builtin_amdgcn_exp2f((x * x) * (-0.5f * PMG_LOG2E));
    return __builtin_fmaf(-__builtin_fabsf(x), q, y < 0.0f ? 0.0f : y);
}

// 1 / (1 + exp(-z)) for fp32 outputs, within 2^-21 of its value: the exponential of -|z|, which cannot overflow, its argument in two
// parts (in one, as silu_fast has it, |z| 2^-24 of the result is lost: 20 times the rest at -80), then 1 ulp each for exp2 and
// reciprocal. Values below 2^-126 may be 0.
__device__ inline float sigmoid_wide(float z) {
    const float a = __builtin_fminf(__builtin_fabsf(z), 200.0f), hi = a * -PMG_LOG2E;  // (infinity times the second part would be NaN)
    const float lo = __builtin_fmaf(a, -1.92596299e-8f, __builtin_fmaf(a, -PMG_LOG2E, -hi));
    const float e2 = __builtin_amdgcn_exp2f(hi), e = __builtin_fmaf(e2, lo * 0.69314718f, e2), r = __builtin_amdgcn_rcpf(1.0f + e);
    return z < 0.0f ? e * r : r;
}

// act of 8 values in place; wide: for fp32 outputs.
__device__ inline void activate8(float (&v)[8], int act, bool wide) {
    switch (act) {
        case PMG_ACT_RELU:
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = v[i] < 0.0f ? 0.0f : v[i];  // (NaN stays)
            break;
        case PMG_ACT_SILU:
            if (wide) {
#pragma unroll
                for (int i = 0; i < 8; ++i) v[i] = v[i] * sigmoid_wide(v[i]);
            } else {
#pragma unroll
                for (int i = 0; i < 8; ++i) v[i] = silu_fast(v[i]);
            }
            break;
        case PMG_ACT_GELU:
            if (wide) {
#pragma unroll
                for (int i = 0; i < 8; ++i) v[i] = 0.5f * v[i] * (1.0f + erff(v[i] * 0.70710678f));
            } else {
#pragma unroll
                for (int i = 0; i < 8; ++i) v[i] = gelu_16(v[i]);
            }
            break;
        case PMG_ACT_GELU_TANH: {  // (1 + tanh(c u)) / 2 = 1 / (1 + exp(-2 c u)), c = sqrt(2 / pi)
            constexpr float c2 = 2.0f * 0.7978845608f;
            const auto u = [](float y) { return __builtin_fmaf(0.044715f * y * y, y, y); };
            if (wide) {
#pragma unroll
                for (int i = 0; i < 8; ++i) v[i] = v[i] * sigmoid_wide(u(v[i]) * c2);
            } else {
#pragma unroll
                for (int i = 0; i < 8; ++i) v[i] = v[i] * __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(u(v[i]) * (-c2 * PMG_LOG2E)));
            }
            break;
        }
        default: break;
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

// 8 values of the residual as they lie in memory (16-bit types: the first half), and as numbers.
struct Raw8 {
    uint4 a, b;
};
__device__ inline Raw8 raw8(const LinearArgs& a, int64_t m, int n0) {
    Raw8 r{};
    const int64_t o = m * a.ldr + n0;
    if (a.res_type == PMG_TYPE_F32) {
        r.a = *(const uint4*)((const float*)a.res + o);
        r.b = *(const uint4*)((const float*)a.res + o + 4);
    } else {
        r.a = *(const uint4*)((const _Float16*)a.res + o);
    }
    return r;
}
__device__ inline void numbers8(const LinearArgs& a, const Raw8& r, float (&v)[8]) {
    if (a.res_type == PMG_TYPE_F32) {
        const v4f x = __builtin_bit_cast(v4f, r.a), y = __builtin_bit_cast(v4f, r.b);
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = i < 4 ? x[i & 3] : y[i & 3];
    } else if (a.res_type == PMG_TYPE_F16) {
        const v8h x = __builtin_bit_cast(v8h, r.a);
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = (float)x[i];
    } else {
        const v8bf x = __builtin_bit_cast(v8bf, r.a);
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = (float)x[i];
    }
}

// n <= 8 outputs of row m from column n0 on: v holds scaled sums plus bias. `early`: the residual, if it is there already.
__device__ inline void finish8(const LinearArgs& a, int64_t m, int n0, int n, float (&v)[8], const Raw8* early = nullptr) {
    const bool wide = a.out_type == PMG_TYPE_F32;
    activate8(v, a.act, wide);
    if (a.res) {
        float r[8];
        const int64_t o = m * a.ldr + n0;
        if (early) numbers8(a, *early, r);
        else if (a.res_type == PMG_TYPE_F32) load8((const float*)a.res + o, n, a.vec_res, r);
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
// a chunk behind K or a row behind M or N is given an offset behind the buffer's end, which reads zeros. One barrier a
// tile.
constexpr uint32_t kNowhere = 0x7ffffff0u;

template <class T, int BM, int BN, int WM, int WN, int KB, int NS, bool VEC>
__global__ __launch_bounds__(64 * WM * WN, (BM / WM) * (BN / WN) >= 128 * 128 ? 1 : 2) void linear_tile_k(LinearArgs a) {
    constexpr int NW = WM * WN, NT = 64 * NW, KE = KB / (int)sizeof(T), PER = Mat<T>::kPer;
    constexpr int CPR = KB / 16, RPL = 64 / CPR, STEPS = CPR / 2;  // chunks a row, rows a load, steps a tile
    constexpr int TM = BM / WM, TN = BN / WN, MT = TM / 32, NTL = TN / 32;
    constexpr int NL = ((BM + BN) / RPL + NW - 1) / NW, kStage = VEC ? NL * NW * 1024 : (BM + BN) * KB;  // a wave's loads a tile
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

    acc32 acc[MT][NTL];
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int j = 0; j < NTL; ++j) acc[i][j] = acc32{};
    // the lane's chunks of a tile's steps (row r of a 32-row operand)
    const int r = lane & 31;
    int at[STEPS];
#pragma unroll
    for (int s = 0; s < STEPS; ++s) at[s] = r * KB + 16 * swizzle<CPR>(r, 2 * s + (lane >> 5));
    // what the epilogue needs is asked for first: scale, bias, and in the small tile the residual
    constexpr int LPR = TN / 8, RPP = 64 / LPR, NP = 32 / RPP;  // lanes a row, rows a pass, passes
    const int nc = n0 + wn * TN + 8 * (lane % LPR);
    const int left = a.N - nc < 8 ? a.N - nc : 8;
    float sc[8], bs[8];
    columns8<T>(a, nc, sc, bs);
    Raw8 early[MT == 1 ? NP : 1];
    const bool ahead = MT == 1 && a.res && a.vec_res && a.N % 8 == 0;
    if constexpr (MT == 1) {
        if (ahead) {
#pragma unroll
            for (int p = 0; p < NP; ++p) {
                const int64_t m = m0 + wm * TM + p * RPP + lane / LPR;
                if (m < a.M && left > 0) early[p] = raw8(a, m, nc);
            }
        }
    }

    chunk fx[2][MT], fw[2][NTL];
    const auto operands = [&](const char* st, int s) {  // step s of the tile at st
        const char* sx = st + wm * TM * KB + at[s];
        const char* sw = st + (BM + wn * TN) * KB + at[s];
#pragma unroll
        for (int j = 0; j < NTL; ++j) fw[s & 1][j] = *(const chunk*)(sw + j * 32 * KB);
#pragma unroll
        for (int i = 0; i < MT; ++i) fx[s & 1][i] = *(const chunk*)(sx + i * 32 * KB);
        __builtin_amdgcn_sched_barrier(0);
    };
    const auto multiply = [&](int s) {
#pragma unroll
        for (int i = 0; i < MT; ++i)
#pragma unroll
            for (int j = 0; j < NTL; ++j) acc[i][j] = Mat<T>::mma32(fw[s & 1][j], fx[s & 1][i], acc[i][j]);
        __builtin_amdgcn_sched_barrier(0);
    };

    if constexpr (VEC) {
        const v4i rx = buffer_of(xb, (uint32_t)(((int64_t)(rows_m - 1) * a.ldx + a.K) * (int)sizeof(T)));
        const v4i rw = buffer_of(wb, (uint32_t)(((int64_t)(rows_n - 1) * a.ldw + a.K) * (int)sizeof(T)));
        uint32_t off[NL];
        const int kbytes = a.K * (int)sizeof(T);
        int kc[NL];  // byte of k of the lane's chunk in tile 0
#pragma unroll
        for (int i = 0; i < NL; ++i) {
            const int row = (i * NW + wave) * RPL + lane / CPR;
            const bool isx = (i * NW + wave) * RPL < BM;  // (uniform over the wave)
            const int rr = isx ? row : row - BM;
            kc[i] = 16 * swizzle<CPR>(rr, lane % CPR);
            off[i] = rr < (isx ? rows_m : rows_n) ? (uint32_t)((int64_t)rr * (isx ? a.ldx : (int64_t)a.ldw) * (int)sizeof(T)) + kc[i] : kNowhere;
        }
        const uint32_t base = lds_address(lds);
        const auto fill = [&](int t, uint32_t place) {
            const bool whole = (t + 1) * KB <= kbytes;
#pragma unroll
            for (int i = 0; i < NL; ++i) {
                const uint32_t o = whole || t * KB + kc[i] < kbytes ? off[i] : kNowhere;
                buffer_to_lds((i * NW + wave) * RPL < BM ? rx : rw, o, (uint32_t)(t * KB), base + place * kStage + (i * NW + wave) * 1024);
            }
        };
        // While one step's products are formed the next step's operands are read; before the last step of tile t all
        // waves have its operands in registers, so its place takes tile t + NS.
#pragma unroll
        for (int t = 0; t < NS; ++t)
            if (t < nk) fill(t, t);
        if (NS - 1 < nk) landed_barrier<(NS - 1) * NL>();
        else landed_barrier<0>();
        operands(lds, 0);
        uint32_t place = 0;
        for (int t = 0; t < nk; ++t) {
#pragma unroll
            for (int s = 0; s + 1 < STEPS; ++s) {
                operands(lds + place * kStage, s + 1);
                multiply(s);
            }
            if (t + 1 < nk) {
                if (t + NS - 1 < nk) landed_barrier<(NS - 2) * NL>();
                else landed_barrier<0>();
                if (t + NS < nk) fill(t + NS, place);
                place = place + 1 == NS ? 0 : place + 1;
                operands(lds + place * kStage, 0);
            }
            multiply(STEPS - 1);
        }
    } else {
        for (int t = 0; t < nk; ++t) {
            for (int e = tid; e < (BM + BN) * CPR; e += NT) {
                const int row = e / CPR, c = e % CPR, k = t * KE + c * PER;
                chunk v{};
                if (row < BM) {
                    if (row < rows_m) v = load_chunk_any<T>(xb + row * a.ldx, k, a.K);
                } else if (row - BM < rows_n) {
                    v = load_chunk_any<T>(wb + (int64_t)(row - BM) * a.ldw, k, a.K);
                }
                *(chunk*)(lds + row * KB + 16 * swizzle<CPR>(row < BM ? row : row - BM, c)) = v;
            }
            __syncthreads();
#pragma unroll
            for (int s = 0; s < STEPS; ++s) {
                operands(lds, s);
                multiply(s);
            }
            __syncthreads();
        }
    }
    __syncthreads();

    // Sums through LDS: 32 rows of the wave's TN columns at a time, in fp32.
    constexpr int LD = TN + 4;
    float* st = (float*)lds + wave * 32 * LD;
#pragma unroll
    for (int i = 0; i < MT; ++i) {
#pragma unroll
        for (int j = 0; j < NTL; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                v4f v;
#pragma unroll
                for (int q = 0; q < 4; ++q) v[q] = (float)acc[i][j][4 * e + q];
                *(v4f*)(st + r * LD + 32 * j + 8 * e + 4 * (lane >> 5)) = v;
            }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
        const auto pass = [&](int p, const Raw8* res) {
            const int row = p * RPP + lane / LPR;
            const int64_t m = m0 + wm * TM + 32 * i + row;
            const v4f u0 = *(const v4f*)(st + row * LD + 8 * (lane % LPR)), u1 = *(const v4f*)(st + row * LD + 8 * (lane % LPR) + 4);
            float v[8];
#pragma unroll
            for (int q = 0; q < 8; ++q) {
                const float s = q < 4 ? u0[q & 3] : u1[q & 3];
                v[q] = sizeof(T) == 1 ? (s * a.a_scale) * sc[q] + bs[q] : s + bs[q];
            }
            if (m < a.M && left > 0) finish8(a, m, nc, left, v, res);
        };
        if (MT == 1 && ahead) {
#pragma unroll
            for (int p = 0; p < NP; ++p) pass(p, &early[MT == 1 ? p : 0]);
        } else {
#pragma unroll 1
            for (int p = 0; p < NP; ++p) pass(p, nullptr);
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
template <class T, int BM, int BN, int WM, int WN, int KB, int NS, bool VEC>
static int launch_tile(LinearArgs& a, hipStream_t s) {
    constexpr int NW = WM * WN, RPL = 1024 / KB;
    constexpr int kStage = VEC ? ((BM + BN) / RPL + NW - 1) / NW * NW * 1024 : (BM + BN) * KB, kOut = NW * 32 * (BN / WN + 4) * 4;
    const int nk = (a.K * (int)sizeof(T) + KB - 1) / KB;
    int bytes = kStage * (!VEC ? 1 : nk < NS ? nk : NS);
    if (bytes < kOut) bytes = kOut;
    a.tiles_n = (uint32_t)((a.N + BN - 1) / BN);
    const int64_t most = grid_blocks(64 * NW) / a.tiles_n * BM;  // rows a launch
    for (int64_t m0 = 0; m0 < a.M; m0 += most) {
        LinearArgs b = a;
        b.M = a.M - m0 < most ? a.M - m0 : most;
        b.x = (const T*)a.x + m0 * a.ldx;
        if (a.res) b.res = (const char*)a.res + m0 * a.ldr * (a.res_type == PMG_TYPE_F32 ? 4 : 2);
        b.out = (char*)a.out + m0 * a.ldo * (a.out_type == PMG_TYPE_F32 ? 4 : 2);
        b.tiles = (uint32_t)((b.M + BM - 1) / BM) * a.tiles_n;
        hipLaunchKernelGGL((linear_tile_k<T, BM, BN, WM, WN, KB, NS, VEC>), dim3(b.tiles), dim3(64 * NW), bytes, s, b);
        if (int e = check_launch("linear_tile_k")) return e;
    }
    return PMG_OK;
}

template <class T, int MT, int NW, bool VEC>
static int launch_rows(LinearArgs& a, hipStream_t s) {
    a.tiles_n = (uint32_t)((a.N + 15) / 16);
    a.tiles = (uint32_t)((a.M + 16 * MT - 1) / (16 * MT)) * a.tiles_n;  // (512 at most)
    hipLaunchKernelGGL((linear_rows_k<T, MT, NW, VEC>), dim3(a.tiles), dim3(64 * NW), 0, s, a);
    return check_launch("linear_rows_k");
}

// Few outputs (at most a block a CU): the kernel whose waves share out k and whose operands go straight to registers; for
// fp32, whose products take 16 times as long on the matrix units, up to two. Eight waves where k is long enough to give
// each two rounds of loads, else four. Measured, K = 1024, fp16: 64 rows to 1024 columns 4.5 us (64 x 64 tiles: 7.3),
// 1000 rows to 256 columns 8.7 (7.6); fp32: 8.4 (23) and 14 (24).
//
// Tiles, by what a CU's share of them costs, fitted to the times of 20 products: k in units of 128 bytes, then the epilogue,
// in microseconds. Measured, us:
//                                          64 x 64   128 x 64   128 x 128   256 x 256   320 x 256
//   11213 x 512 to 256, fp16                  10        11.4        11.3
//   76800 x 256 to 256, fp16                  32        30          32          49          33
//   4800 x 1024 to 1024, bf16                 23        20          21          41          50
//   4800 x 4096 to 1024, bf16                 76        62          53          109         137
//   19200 x 1024 to 1024, int8                45        47          41          65          43
//   4800 x 1024 to 4096, bf16, gelu           77        67          62          82          56
//   8192 x 4096 to 4096, bf16                                       310         281
// A CU holds five blocks of 64 x 64, three of 128 x 64, two of 128 x 128 (where it has two at most the chip clocks higher) and
// one of the largest, whose LDS reads are a quarter fewer a product. fp32 takes 64 x 64: its products are 16 times as long.
template <class T, bool VEC>
static int launch_linear(LinearArgs& a, hipStream_t s) {
    const int64_t tn = (a.N + 15) / 16, n1 = (a.M + 15) / 16 * tn, n2 = (a.M + 31) / 32 * tn;
    const bool lengthy = (int64_t)a.K * (int)sizeof(T) >= 48 * 64;
    if (n1 <= 256) return lengthy ? launch_rows<T, 1, 8, VEC>(a, s) : launch_rows<T, 1, 4, VEC>(a, s);
    if (n2 <= (sizeof(T) == 4 ? 512 : 256)) return lengthy ? launch_rows<T, 2, 8, VEC>(a, s) : launch_rows<T, 2, 4, VEC>(a, s);
    if constexpr (VEC && sizeof(T) < 4) {
        const double k = (double)(((int64_t)a.K * (int)sizeof(T) + 127) / 128);
        const auto rounds = [&](int bm, int bn) { return (double)(((a.M + bm - 1) / bm * ((a.N + bn - 1) / bn) + 255) / 256); };
        const double r = rounds(128, 128);
        const double c[5] = {rounds(64, 64) * (0.24 * k + 0.6), rounds(128, 64) * (0.31 * k + 1.5),
                             r > 2.0 ? r * (0.55 * k + 3.5) : (r < 2.0 ? 1.5 : r) * (0.36 * k + 4.7),
                             rounds(256, 256) * (2.0 * k + 15.0), rounds(320, 256) * (2.4 * k + 20.0)};
        int best = 0;
        for (int i = 1; i < 5; ++i)
            if (c[i] < c[best]) best = i;
        if (best == 1) return launch_tile<T, 128, 64, 4, 2, 128, 2, VEC>(a, s);
        if (best == 2) return launch_tile<T, 128, 128, 4, 2, 128, 2, VEC>(a, s);
        if (best == 3) return launch_tile<T, 256, 256, 2, 4, 64, 4, VEC>(a, s);
        if (best == 4) return launch_tile<T, 320, 256, 2, 4, 64, 3, VEC>(a, s);
    }
    return launch_tile<T, 64, 64, 2, 2, 128, 2, VEC>(a, s);
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
    // (int8: 131072 products of -128 by -128 are 2^31)
    PMG_REQUIRE(q.K >= 1 && q.K <= (q.type == PMG_TYPE_I8 ? 131071 : 131072) && q.N >= 1 && q.N <= (1 << 24), "K must be 1 .. 131072 (int8: 131071) and N 1 .. 2^24");
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
