// What the products' and norms' kernels do with finished sums: activation, residual, one rounding, and the rows' stores.
#pragma once
#include "pmg_dense.h"

namespace pmg {

// What the functions below take from a kernel's arguments, which derive from it or have members of these names.
struct Epilogue {
    const void* res;  // rows of ldr or NULL
    void* out;        // rows of ldo
    int64_t ldr, ldo;
    int act, res_type, out_type;
    int vec_res, vec_out;  // rows of res / out take 16-byte accesses
};

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

// act(y), WIDE: for fp32 outputs.
template <int ACT, bool WIDE>
__device__ inline float activated(float y) {
    if constexpr (ACT == PMG_ACT_RELU) {
        return y < 0.0f ? 0.0f : y;  // (NaN stays)
    } else if constexpr (ACT == PMG_ACT_SILU) {
        return WIDE ? y * sigmoid_wide(y) : silu_fast(y);
    } else if constexpr (ACT == PMG_ACT_GELU) {
        return WIDE ? 0.5f * y * (1.0f + erff(y * 0.70710678f)) : gelu_16(y);
    } else if constexpr (ACT == PMG_ACT_GELU_TANH) {  // (1 + tanh(c u)) / 2 = 1 / (1 + exp(-2 c u)), c = sqrt(2 / pi)
        constexpr float c2 = 2.0f * 0.7978845608f;
        const float u = __builtin_fmaf(0.044715f * y * y, y, y);
        return WIDE ? y * sigmoid_wide(u * c2) : y * __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(u * (-c2 * PMG_LOG2E)));
    } else {
        return y;
    }
}

// f(constant of act): code for each activation of its own, chosen once.
template <int ACT>
struct ActOf {
    static constexpr int value = ACT;
};
template <class F>
__device__ inline void with_act(int act, const F& f) {
    switch (act) {
        case PMG_ACT_RELU: f(ActOf<PMG_ACT_RELU>{}); break;
        case PMG_ACT_SILU: f(ActOf<PMG_ACT_SILU>{}); break;
        case PMG_ACT_GELU: f(ActOf<PMG_ACT_GELU>{}); break;
        case PMG_ACT_GELU_TANH: f(ActOf<PMG_ACT_GELU_TANH>{}); break;
        default: f(ActOf<PMG_ACT_NONE>{}); break;
    }
}

// act of 8 values in place; wide: for fp32 outputs.
__device__ inline void activate8(float (&v)[8], int act, bool wide) {
    switch (act) {
        case PMG_ACT_RELU:
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = activated<PMG_ACT_RELU, false>(v[i]);
            break;
        case PMG_ACT_SILU:
            if (wide) {
#pragma unroll
                for (int i = 0; i < 8; ++i) v[i] = activated<PMG_ACT_SILU, true>(v[i]);
            } else {
#pragma unroll
                for (int i = 0; i < 8; ++i) v[i] = activated<PMG_ACT_SILU, false>(v[i]);
            }
            break;
        case PMG_ACT_GELU:
            if (wide) {
#pragma unroll
                for (int i = 0; i < 8; ++i) v[i] = activated<PMG_ACT_GELU, true>(v[i]);
            } else {
#pragma unroll
                for (int i = 0; i < 8; ++i) v[i] = activated<PMG_ACT_GELU, false>(v[i]);
            }
            break;
        case PMG_ACT_GELU_TANH:
            if (wide) {
#pragma unroll
                for (int i = 0; i < 8; ++i) v[i] = activated<PMG_ACT_GELU_TANH, true>(v[i]);
            } else {
#pragma unroll
                for (int i = 0; i < 8; ++i) v[i] = activated<PMG_ACT_GELU_TANH, false>(v[i]);
            }
            break;
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
// PAST: past the caches, as the grouped products' tiles and combine store, whatever the result's size. By itself that is a large call's
// gain (us, without and with: 76,800 x 256 fp32 of two fp16 slots each 44.3 and 38.5, 131k scattered rows of 128 fp16 29.3 and 27.1; small
// ones the same either way). Where the next call reads the result at once it costs: up, down and combine one behind the other, rows x
// width (inner width), 2 of 8 or 16 experts: 76,800 x 256 (256) 122 and 131, 19,200 x 256 (512) 64.6 and 70.1, 4800 x 1024 (4096) 244 and
// 251; 9600 x 128 (256) and 4 x 1024 (4096) gain 3 and 5 %, others are the same to 4 % worse.
template <bool PAST = false, class E>
__device__ inline void store8(E* p, int n, bool vec, const float (&v)[8]) {
    if (vec && n == 8) {
        constexpr int C = 16 / sizeof(E);
        typedef E vec_t __attribute__((ext_vector_type(C)));
#pragma unroll
        for (int c = 0; c < 8 / C; ++c) {
            vec_t t;
#pragma unroll
            for (int i = 0; i < C; ++i) t[i] = (E)v[c * C + i];
            if constexpr (PAST) __builtin_nontemporal_store(t, (vec_t*)(p + c * C));
            else *(vec_t*)(p + c * C) = t;
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
template <class A>
__device__ inline Raw8 raw8(const A& a, int64_t m, int n0) {
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
template <class A>
__device__ inline void numbers8(const A& a, const Raw8& r, float (&v)[8]) {
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

// n <= 8 values of the residual's row m from column n0 on, as numbers.
template <class A>
__device__ inline void residual8(const A& a, int64_t m, int n0, int n, float (&r)[8]) {
    const int64_t o = m * a.ldr + n0;
    if (a.res_type == PMG_TYPE_F32) load8((const float*)a.res + o, n, a.vec_res, r);
    else if (a.res_type == PMG_TYPE_F16) load8((const _Float16*)a.res + o, n, a.vec_res, r);
    else load8((const __bf16*)a.res + o, n, a.vec_res, r);
}
// n <= 8 finished values of row m from column n0 on, rounded and stored.
template <bool PAST = false, class A>
__device__ inline void put8(const A& a, int64_t m, int n0, int n, const float (&v)[8]) {
    const int64_t o = m * a.ldo + n0;
    if (a.out_type == PMG_TYPE_F32) store8<PAST>((float*)a.out + o, n, a.vec_out, v);
    else if (a.out_type == PMG_TYPE_F16) store8<PAST>((_Float16*)a.out + o, n, a.vec_out, v);
    else store8<PAST>((__bf16*)a.out + o, n, a.vec_out, v);
}
// n <= 8 outputs of row m from column n0 on: v holds scaled sums plus bias. `early`: the residual, if it is there already.
template <bool PAST = false, class A>
__device__ inline void finish8(const A& a, int64_t m, int n0, int n, float (&v)[8], const Raw8* early = nullptr) {
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
    if (a.out_type == PMG_TYPE_F32) store8<PAST>((float*)a.out + o, n, a.vec_out, v);
    else if (a.out_type == PMG_TYPE_F16) store8<PAST>((_Float16*)a.out + o, n, a.vec_out, v);
    else store8<PAST>((__bf16*)a.out + o, n, a.vec_out, v);
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

}  // namespace pmg
