// Norms of queries and keys per head with the rotation by voxel coordinates, in one pass over both.
//
// u = x - mean (LayerNorm only), u * rsqrt(mean(u^2) + eps) * weight (+ bias), then each pair (a, b) turned by its angle
// t = sum over axes of coords[m][axis] * freqs[p][axis]: (a cos t - b sin t, a sin t + b cos t).
//
// A lane holds four pairs of a head, so that a pair never leaves its lane; a head is D / 8 lanes (made up to a power of
// two). The angles are the same for every head: a block forms those of its rows once, in 64 bits (the product of a
// 32-bit coordinate and an fp32 frequency is exact there, and the reduction to one turn loses nothing an fp32 sine
// could show), and keeps their sines and cosines in LDS.
#include "pmg_dense.h"

namespace pmg {

struct RopeArgs {
    const void* q;
    const void* k;
    void* q_out;
    void* k_out;
    int64_t M, q_row, q_head, k_row, k_head, qo_row, qo_head, ko_row, ko_head;  // strides in elements
    int Hq, Hk, D, P;  // P rotated pairs (<= D / 2)
    const int32_t* coords;
    const float* freqs;
    const float* q_weight;
    const float* k_weight;
    const float* q_bias;
    const float* k_bias;
    int layer, interleaved;
    float eps;
    int rows;  // rows a block
};

template <class T>
__device__ inline void load4(const T* p, float* v) {
    typedef T v4t __attribute__((ext_vector_type(4)));
    const v4t t = *(const v4t*)p;
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = (float)t[i];
}
template <class T>
__device__ inline void store4(T* p, const float* v) {
    typedef T v4t __attribute__((ext_vector_type(4)));
    v4t t;
#pragma unroll
    for (int i = 0; i < 4; ++i) t[i] = (T)v[i];
    *(v4t*)p = t;
}

// G lanes a head (a power of two >= D / 8).
template <class T, int G>
__global__ __launch_bounds__(256) void qk_norm_rope_k(RopeArgs a) {
    extern __shared__ float2 turn[];  // [rows][P] (cos, sin)
    const int tid = threadIdx.x, g = tid & (G - 1), D = a.D, h2 = D / 2;
    const int64_t m0 = (int64_t)blockIdx.x * a.rows;
    const int rows = a.M - m0 < a.rows ? (int)(a.M - m0) : a.rows;
    for (int e = tid; e < rows * a.P; e += 256) {
        const int r = e / a.P, p = e - r * a.P;
        const int32_t* c = a.coords + (m0 + r) * 4;
        double t = (double)c[1] * (double)a.freqs[3 * p];
        t = __builtin_fma((double)c[2], (double)a.freqs[3 * p + 1], t);
        t = __builtin_fma((double)c[3], (double)a.freqs[3 * p + 2], t);
        t = t * 0.15915494309189535;  // turns
        float s, co;
        sincospif((float)(2.0 * (t - __builtin_rint(t))), &s, &co);
        turn[e] = make_float2(co, s);
    }
    __syncthreads();
    // the lane's four pairs: elements pa .. pa + 3 and pb .. pb + 3, or 8 neighbouring ones
    const bool lane_in = 8 * g < D;
    const int p0 = lane_in ? 4 * g : 0, pa = a.interleaved ? 2 * p0 : p0, pb = a.interleaved ? pa + 4 : h2 + p0;
    float wq[8], wk[8], bq[8], bk[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const int d = i < 4 ? pa + i : pb + i - 4;
        wq[i] = a.q_weight ? a.q_weight[d] : 1.0f;
        wk[i] = a.k_weight ? a.k_weight[d] : 1.0f;
        bq[i] = a.q_bias ? a.q_bias[d] : 0.0f;
        bk[i] = a.k_bias ? a.k_bias[d] : 0.0f;
    }
    const float inv = 1.0f / (float)D;
    const int heads = a.Hq + a.Hk;
    const int items = rows * heads, rounds = (items + 256 / G - 1) / (256 / G);
    for (int it = 0; it < rounds; ++it) {  // (every lane of a wave takes part in the sums)
        const int item = it * (256 / G) + tid / G;
        const bool on = item < items && lane_in;
        const int r = item < items ? item / heads : 0, h = item < items ? item - r * heads : 0;
        const bool isq = h < a.Hq;
        const int64_t m = m0 + r;
        float v[8] = {0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f};
        if (on) {
            const T* x = isq ? (const T*)a.q + m * a.q_row + h * a.q_head : (const T*)a.k + m * a.k_row + (h - a.Hq) * a.k_head;
            load4(x + pa, v);
            load4(x + pb, v + 4);
        }
        float s = 0.0f, mean = 0.0f;
        if (a.layer) {
#pragma unroll
            for (int i = 0; i < 8; ++i) s = s + v[i];
#pragma unroll
            for (int o = 1; o < G; o <<= 1) s = s + __shfl_xor(s, o, 64);
            mean = s * inv;
        }
        float ss = 0.0f;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            v[i] = on ? v[i] - mean : 0.0f;
            ss = __builtin_fmaf(v[i], v[i], ss);
        }
#pragma unroll
        for (int o = 1; o < G; o <<= 1) ss = ss + __shfl_xor(ss, o, 64);
        const float rstd = 1.0f / __builtin_sqrtf(__builtin_fmaf(ss, inv, a.eps));
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = __builtin_fmaf(v[i] * rstd, isq ? wq[i] : wk[i], isq ? bq[i] : bk[i]);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            if (p0 + j < a.P && on) {
                const float2 t = turn[r * a.P + p0 + j];
                const int ia = a.interleaved ? 2 * j : j, ib = a.interleaved ? 2 * j + 1 : 4 + j;
                float& x = v[ia];
                float& y = v[ib];
                const float u = x, w = y;
                x = __builtin_fmaf(u, t.x, -(w * t.y));
                y = __builtin_fmaf(u, t.y, w * t.x);
            }
        }
        if (on) {
            T* o = isq ? (T*)a.q_out + m * a.qo_row + h * a.qo_head : (T*)a.k_out + m * a.ko_row + (h - a.Hq) * a.ko_head;
            store4(o + pa, v);
            store4(o + pb, v + 4);
        }
    }
}

template <class T>
static int launch_rope(RopeArgs& a, hipStream_t s) {
    // about 256 angles a block, and work for its lanes
    const int G = a.D <= 8 ? 1 : a.D <= 16 ? 2 : a.D <= 32 ? 4 : a.D <= 64 ? 8 : 16;
    int rows = a.P > 0 ? 256 / a.P : 32;
    rows = rows < 1 ? 1 : rows > 32 ? 32 : rows;
    a.rows = rows;
    const int64_t blocks = (a.M + rows - 1) / rows;
    const size_t lds = sizeof(float2) * (size_t)rows * (size_t)(a.P > 0 ? a.P : 1);
    const dim3 grid((unsigned)blocks), block(256);
    switch (G) {
        case 1: hipLaunchKernelGGL((qk_norm_rope_k<T, 1>), grid, block, lds, s, a); break;
        case 2: hipLaunchKernelGGL((qk_norm_rope_k<T, 2>), grid, block, lds, s, a); break;
        case 4: hipLaunchKernelGGL((qk_norm_rope_k<T, 4>), grid, block, lds, s, a); break;
        case 8: hipLaunchKernelGGL((qk_norm_rope_k<T, 8>), grid, block, lds, s, a); break;
        default: hipLaunchKernelGGL((qk_norm_rope_k<T, 16>), grid, block, lds, s, a); break;
    }
    return check_launch("qk_norm_rope_k");
}

}  // namespace pmg

using namespace pmg;

extern "C" int pmg_qk_norm_rope(const pmg_rope_args* p, void* stream) {
    PMG_REQUIRE(p, "null args");
    const pmg_rope_args& r = *p;
    PMG_REQUIRE(r.type >= PMG_TYPE_F32 && r.type <= PMG_TYPE_BF16, "type must be f32, f16 or bf16");
    PMG_REQUIRE(r.M >= 0 && r.M < (int64_t)1 << 31, "M out of range");
    PMG_REQUIRE(r.Hq >= 1 && r.Hk >= 0 && r.Hq <= 4096 && r.Hk <= 4096, "1 .. 4096 query heads, 0 .. 4096 key heads");
    PMG_REQUIRE(r.D >= 8 && r.D <= 128 && r.D % 8 == 0, "head width must be a multiple of 8 up to 128");
    PMG_REQUIRE(r.pairs >= 0 && r.pairs <= r.D / 2, "at most D / 2 rotated pairs");
    PMG_REQUIRE(r.eps >= 0.0f, "eps must not be negative");
    if (r.M == 0) return PMG_OK;
    PMG_REQUIRE(r.q && r.q_out && (r.Hk == 0 || (r.k && r.k_out)), "null buffer");
    PMG_REQUIRE(r.pairs == 0 || (r.coords && r.freqs), "rotation needs coords and freqs");
    const int es = r.type == PMG_TYPE_F32 ? 4 : 2;
    auto ok = [&](const void* b, int64_t row, int64_t head) {
        return (reinterpret_cast<uintptr_t>(b) & (uintptr_t)(4 * es - 1)) == 0 && row % 4 == 0 && head % 4 == 0;
    };
    PMG_REQUIRE(ok(r.q, r.q_row, r.q_head) && ok(r.q_out, r.q_out_row, r.q_out_head), "q, q_out: buffers and strides in whole groups of 4 elements");
    PMG_REQUIRE(r.Hk == 0 || (ok(r.k, r.k_row, r.k_head) && ok(r.k_out, r.k_out_row, r.k_out_head)), "k, k_out: buffers and strides in whole groups of 4 elements");
    RopeArgs a{};
    a.q = r.q;
    a.k = r.k;
    a.q_out = r.q_out;
    a.k_out = r.k_out;
    a.M = r.M;
    a.q_row = r.q_row;
    a.q_head = r.q_head;
    a.k_row = r.k_row;
    a.k_head = r.k_head;
    a.qo_row = r.q_out_row;
    a.qo_head = r.q_out_head;
    a.ko_row = r.k_out_row;
    a.ko_head = r.k_out_head;
    a.Hq = r.Hq;
    a.Hk = r.Hk;
    a.D = r.D;
    a.P = r.pairs;
    a.coords = r.coords;
    a.freqs = r.freqs;
    a.q_weight = r.q_weight;
    a.k_weight = r.k_weight;
    a.q_bias = r.q_bias;
    a.k_bias = r.k_bias;
    a.layer = r.layer;
    a.interleaved = r.interleaved;
    a.eps = r.eps;
    hipStream_t s = (hipStream_t)stream;
    if (r.type == PMG_TYPE_F32) return launch_rope<float>(a, s);
    if (r.type == PMG_TYPE_F16) return launch_rope<_Float16>(a, s);
    return launch_rope<__bf16>(a, s);
}
