// Norms of queries and keys per head with the rotation by voxel coordinates, in one pass over both.
//
// u = x - mean (LayerNorm only), u * rsqrt(mean(u^2) + eps) * weight (+ bias), then each pair (a, b) turned by its angle
// t = sum over axes of coords[m][axis] * freqs[p][axis]: (a cos t - b sin t, a sin t + b cos t).
//
// A lane holds four pairs of a head, so that a pair never leaves its lane; a head is D / 8 lanes (made up to a power of
// two). The angles are the same for every head: a block forms those of its rows once, in 64 bits (the product of a
// coordinate below 2^29 and an fp32 frequency is exact there, and the reduction of angles below 2^27 to one turn loses nothing
// that an fp32 sine could show), and keeps their sines and cosines in LDS.
//
// Bound by memory: 76,800 rows, 8 and 8 heads of 32, fp16: 157 MB in 32.6 us, 4.8 TB/s (a copy reaches 5.0).
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
    uint32_t q_magic, k_magic;
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

// Sum over groups of G neighbouring lanes (a power of two up to 16), the same in each of them: neighbours, pairs, then
// mirrored halves and rows.
template <int G>
__device__ inline float group_sum(float v) {
    if constexpr (G >= 2) v = v + u2f(dpp_u32<0xB1, 0xf>(f2u(v)));
    if constexpr (G >= 4) v = v + u2f(dpp_u32<0x4E, 0xf>(f2u(v)));
    if constexpr (G >= 8) v = v + u2f(dpp_u32<0x141, 0xf>(f2u(v)));
    if constexpr (G >= 16) v = v + u2f(dpp_u32<0x140, 0xf>(f2u(v)));
    return v;
}

// The heads of one of the two tensors, rows m0 .. m0 + rows - 1.
struct RopeSide {
    const void* x;
    void* out;
    int64_t row, head, orow, ohead;
    int H;
    uint32_t magic;  // ceil(2^32 / H): item / H for items below 2^16
    const float* weight;
    const float* bias;
};

template <class T, int G, bool INTER, bool LAYER>
__device__ inline void rope_side(const RopeArgs& a, const RopeSide& s, const float2* turn, int64_t m0, int rows) {
    const int tid = threadIdx.x, g = tid & (G - 1), D = a.D;
    // the lane's four pairs: elements pa .. pa + 3 and pb .. pb + 3, or 8 neighbouring ones
    const bool lane_in = 8 * g < D;
    const int p0 = lane_in ? 4 * g : 0, pa = INTER ? 2 * p0 : p0, pb = INTER ? pa + 4 : D / 2 + p0;
    float w[8] = {1.0f, 1.0f, 1.0f, 1.0f, 1.0f, 1.0f, 1.0f, 1.0f}, b[8] = {};
    if (s.weight) {
#pragma unroll
        for (int i = 0; i < 8; ++i) w[i] = s.weight[i < 4 ? pa + i : pb + i - 4];
    }
    if (s.bias) {
#pragma unroll
        for (int i = 0; i < 8; ++i) b[i] = s.bias[i < 4 ? pa + i : pb + i - 4];
    }
    const float inv = 1.0f / (float)D;
    const T* x0 = (const T*)s.x + m0 * s.row;
    T* o0 = (T*)s.out + m0 * s.orow;
    const int items = rows * s.H;
    for (int at = 0; at < items; at += 256 / G) {  // (every lane of a wave takes part in the sums)
        const int item = at + tid / G;
        const bool on = item < items && lane_in;
        const int r = s.H > 1 ? (int)__umulhi((uint32_t)item, s.magic) : item, h = item - r * s.H;
        float v[8] = {};
        if (on) {
            const T* x = x0 + r * s.row + h * s.head;
            load4(x + pa, v);
            load4(x + pb, v + 4);
        }
        if constexpr (LAYER) {
            float t = 0.0f;
#pragma unroll
            for (int i = 0; i < 8; ++i) t = t + v[i];
            const float mean = group_sum<G>(t) * inv;
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = on ? v[i] - mean : 0.0f;
        }
        float ss = 0.0f;
#pragma unroll
        for (int i = 0; i < 8; ++i) ss = __builtin_fmaf(v[i], v[i], ss);
        const float rstd = __builtin_amdgcn_rsqf(__builtin_fmaf(group_sum<G>(ss), inv, a.eps));
        if (!on) continue;
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = __builtin_fmaf(v[i] * rstd, w[i], b[i]);
        if (p0 + 4 <= a.P && a.P % 4 == 0) {
            const v4f t01 = *(const v4f*)(turn + r * a.P + p0), t23 = *(const v4f*)(turn + r * a.P + p0 + 2);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const float c = j < 2 ? t01[2 * (j & 1)] : t23[2 * (j & 1)], sn = j < 2 ? t01[2 * (j & 1) + 1] : t23[2 * (j & 1) + 1];
                float& x = v[INTER ? 2 * j : j];
                float& y = v[INTER ? 2 * j + 1 : 4 + j];
                const float u = x, z = y;
                x = __builtin_fmaf(u, c, -(z * sn));
                y = __builtin_fmaf(u, sn, z * c);
            }
        } else {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                if (p0 + j >= a.P) continue;
                const float2 t = turn[r * a.P + p0 + j];
                float& x = v[INTER ? 2 * j : j];
                float& y = v[INTER ? 2 * j + 1 : 4 + j];
                const float u = x, z = y;
                x = __builtin_fmaf(u, t.x, -(z * t.y));
                y = __builtin_fmaf(u, t.y, z * t.x);
            }
        }
        T* o = o0 + r * s.orow + h * s.ohead;
        store4(o + pa, v);
        store4(o + pb, v + 4);
    }
}

// G lanes a head (a power of two >= D / 8).
template <class T, int G, bool INTER, bool LAYER>
__global__ __launch_bounds__(256) void qk_norm_rope_k(RopeArgs a) {
    extern __shared__ __attribute__((aligned(16))) float2 turn[];  // [rows][P] (cos, sin)
    const int64_t m0 = (int64_t)blockIdx.x * a.rows;
    const int rows = a.M - m0 < a.rows ? (int)(a.M - m0) : a.rows;
    for (int e = threadIdx.x; e < rows * a.P; e += 256) {
        const int r = e / a.P, p = e - r * a.P;
        const int4 c = *(const int4*)(a.coords + (m0 + r) * 4);
        double t = (double)c.y * (double)a.freqs[3 * p];
        t = __builtin_fma((double)c.z, (double)a.freqs[3 * p + 1], t);
        t = __builtin_fma((double)c.w, (double)a.freqs[3 * p + 2], t);
        t = t * 0.15915494309189535;  // turns
        float s, co;
        sincospif((float)(2.0 * (t - __builtin_rint(t))), &s, &co);
        turn[e] = make_float2(co, s);
    }
    __syncthreads();
    rope_side<T, G, INTER, LAYER>(a, RopeSide{a.q, a.q_out, a.q_row, a.q_head, a.qo_row, a.qo_head, a.Hq, a.q_magic, a.q_weight, a.q_bias}, turn, m0, rows);
    if (a.Hk) rope_side<T, G, INTER, LAYER>(a, RopeSide{a.k, a.k_out, a.k_row, a.k_head, a.ko_row, a.ko_head, a.Hk, a.k_magic, a.k_weight, a.k_bias}, turn, m0, rows);
}

template <class T, int G>
static void launch_rope_g(const RopeArgs& a, dim3 grid, size_t lds, hipStream_t s) {
    const dim3 block(256);
    if (a.interleaved) {
        if (a.layer) hipLaunchKernelGGL((qk_norm_rope_k<T, G, true, true>), grid, block, lds, s, a);
        else hipLaunchKernelGGL((qk_norm_rope_k<T, G, true, false>), grid, block, lds, s, a);
    } else {
        if (a.layer) hipLaunchKernelGGL((qk_norm_rope_k<T, G, false, true>), grid, block, lds, s, a);
        else hipLaunchKernelGGL((qk_norm_rope_k<T, G, false, false>), grid, block, lds, s, a);
    }
}

template <class T>
static int launch_rope(RopeArgs& a, hipStream_t s) {
    // about 256 angles a block, and work for its lanes
    const int G = a.D <= 8 ? 1 : a.D <= 16 ? 2 : a.D <= 32 ? 4 : a.D <= 64 ? 8 : 16;
    int rows = a.P > 0 ? 256 / a.P : 32;
    rows = rows < 1 ? 1 : rows > 32 ? 32 : rows;
    a.rows = rows;
    const size_t lds = sizeof(float2) * (size_t)rows * (size_t)(a.P > 0 ? a.P : 1);
    a.q_magic = (uint32_t)((((uint64_t)1 << 32) + a.Hq - 1) / (uint64_t)a.Hq);
    a.k_magic = a.Hk ? (uint32_t)((((uint64_t)1 << 32) + a.Hk - 1) / (uint64_t)a.Hk) : 0;
    const int64_t most = grid_blocks(256) * rows;  // rows a launch
    for (int64_t m0 = 0; m0 < a.M; m0 += most) {
        RopeArgs b = a;
        b.M = a.M - m0 < most ? a.M - m0 : most;
        b.q = (const T*)a.q + m0 * a.q_row;
        b.q_out = (T*)a.q_out + m0 * a.qo_row;
        if (a.Hk) {
            b.k = (const T*)a.k + m0 * a.k_row;
            b.k_out = (T*)a.k_out + m0 * a.ko_row;
        }
        if (a.P > 0) b.coords = a.coords + m0 * 4;
        const dim3 grid((unsigned)((b.M + rows - 1) / rows));
        switch (G) {
            case 1: launch_rope_g<T, 1>(b, grid, lds, s); break;
            case 2: launch_rope_g<T, 2>(b, grid, lds, s); break;
            case 4: launch_rope_g<T, 4>(b, grid, lds, s); break;
            case 8: launch_rope_g<T, 8>(b, grid, lds, s); break;
            default: launch_rope_g<T, 16>(b, grid, lds, s); break;
        }
        if (int e = check_launch("qk_norm_rope_k")) return e;
    }
    return PMG_OK;
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
    PMG_REQUIRE(aligned16(r.coords), "coords must be 16-byte aligned");
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
