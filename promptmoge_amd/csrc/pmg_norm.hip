// Group norm of rows with channels last, with an activation: for each segment of rows (a frame) and group of C / G channels,
// y = act((x - mean) rsqrt(var + eps) weight[c] + bias[c]), mean and var over the segment's rows and the group's channels.
//
// Sums of x and x^2 are held in 64 bits: their products are exact and nothing overflows, and mean and var come out to fp32's
// accuracy where the mean is 10^4 times the spread (for fp32 inputs E[x^2] - mean^2 in 64 bits loses 2^-53 (mean / spread)^2).
// The mean is subtracted in two fp32 parts; spreads near the ends of fp32's range are brought inside by a power of two.
//
// Measured (MI355X), and what bounds it: 307,200 rows of 64 fp16 with silu 31 us (11 the sums, 19 the results; two reads and a write
// are 23 at a copy's rate, the rest is a block's start: its segment, the segment's sums, a barrier); 4 x 2745 rows of 512 fp32 to bf16
// with gelu 21 us (8 and 13); 8 segments of one row of 256: 4.4 us, three latencies.
#include "pmg_epilogue.h"
#include "pmg_pieces.h"

namespace pmg {

struct NormArgs : Epilogue, Pieces {
    const void* x;
    const float* weight;  // [C] or NULL
    const float* bias;
    double2* parts;       // [G][ids]: sums of x and x^2 of each tile
    int64_t ldx, ids;
    int C, G, gw;         // gw: channels a group
    int slab, slabs;      // groups a block takes; blocks over the groups
    int rows;             // a tile's rows
    int vec_x, fresh;
    float eps;
    uint32_t id0;
};

constexpr int kRest = 2048;  // blocks that rows of no segment are shared out over

struct Stat {
    float hi, lo, r;  // mean in two parts, 1 / spread; r < 0: -1 / spread, all of the values times a power of two (times())
};
// What a group's values are taken times before its mean is subtracted: 1, but where the spread is at an end of fp32's range.
__device__ inline float times(const Stat& st) { return st.r < 0.0f ? st.r > -1.0f ? 0x1p-64f : 0x1p64f : 1.0f; }

// Types whose values have fp32's range.
template <class T>
constexpr bool kWide = !__is_same(T, _Float16);

// 8 values of a row as they lie in memory (16-bit types: the first half), and as numbers.
template <class T, bool VEC>
__device__ inline Raw8 norm_get(const NormArgs& a, int64_t m, int c, int n) {
    const T* p = (const T*)a.x + m * a.ldx + c;
    Raw8 r{};
    if (VEC || (a.vec_x && n == 8)) {
        r.a = *(const uint4*)p;
        if constexpr (sizeof(T) == 4) r.b = *(const uint4*)(p + 4);
    } else {
        T v[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = i < n ? p[i] : (T)0.0f;
        __builtin_memcpy(&r, v, sizeof(v));
    }
    return r;
}
template <class T>
__device__ inline void norm_numbers(const Raw8& r, float (&v)[8]) {
    typedef T vec_t __attribute__((ext_vector_type(16 / sizeof(T))));
    constexpr int C = 16 / sizeof(T);
    const vec_t x = __builtin_bit_cast(vec_t, r.a), y = __builtin_bit_cast(vec_t, r.b);
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = (float)(i < C ? x[i % C] : y[i % C]);
}

// A block's slab of whole groups (8 channels a thread, `wide` threads a row) of a tile's rows. WHOLE: a tile is a segment, sums
// and results in one launch; else SUMS writes the tile's sums, and without it the segment's are added up (in an order that only
// their number sets) and applied, behind the loads of the block's first rows.
template <class T, class O, int NT, bool WHOLE, bool SUMS>
__global__ __launch_bounds__(NT) void norm_k(NormArgs a) {
    __shared__ double red[SUMS ? NT * 8 : 1];
    __shared__ Stat stats[64];  // (a slab has at most 64 groups)
    // Rows a thread has under way twice. The loops over whole rounds of rows have neither conditional loads nor conditional stores:
    // loads and stores share one counter, and where the compiler cannot count them it waits for all of them.
    constexpr int U = SUMS && NT > 512 ? 4 : 2;
    const int tid = threadIdx.x;
    const int slab = (int)(blockIdx.x % (uint32_t)a.slabs);
    const uint32_t id = a.id0 + blockIdx.x / (uint32_t)a.slabs;
    Piece p;
    int front = 0, back = a.P;  // WHOLE: where the segments start and end
    if constexpr (WHOLE) {
        p.p0 = 0;
        p.p1 = id == 1 ? a.P : 0;
        if (a.offsets) {  // (the four bounds are asked for at once)
            const int64_t i = id, o0 = a.offsets[i < 1 ? 0 : i - 1], o1 = a.offsets[i < a.S ? i : a.S], of = a.offsets[0], ob = a.offsets[a.S];
            const auto held = [&](int64_t o) { return o < 0 ? 0 : o > a.P ? a.P : (int)o; };
            p.p0 = i < 1 ? 0 : held(o0);
            p.p1 = i > a.S ? a.P : held(o1);
            if (a.fresh && id < kRest) front = held(of), back = held(ob);
        }
        p.first = p.p0;
        p.n = p.p1 - p.p0;
        p.s = id >= 1 && (int64_t)id <= a.S ? (int)(id - 1) : -1;
    } else {
        p = piece_of(a, id, a.rows);
    }
    if (!WHOLE && (p.n < 1 || (p.s < 0 && (SUMS || !a.fresh)))) return;
    const int g0 = slab * a.slab, ng = a.G - g0 < a.slab ? a.G - g0 : a.slab;
    const int c0 = g0 * a.gw, width = ng * a.gw, wide = (width + 7) / 8;
    const int tx = tid % wide, ty = tid / wide, deep = NT / wide;  // (threads behind the last whole row: ty == deep, idle)
    const int c = c0 + 8 * tx, n = c0 + width - c < 8 ? c0 + width - c : 8;
    const bool busy = ty < deep;
    const float z[8] = {};
    if constexpr (WHOLE) {
        // Rows in front of the segments and behind them are shared out over the slab's (first kRest) blocks, for they may be most of all
        // (1000 segments of 20 rows of 256 fp16 and 20,000 rows behind: 194 us where the two blocks in front and behind set them to 0).
        const int64_t rest = (int64_t)front + (a.P - back);
        const int step = (a.ids < kRest ? (int)a.ids : kRest) * deep;
        for (int64_t r = (int64_t)id * deep + ty; busy && r < rest; r += step)
            store8((O*)a.out + (r < front ? r : back + (r - front)) * a.ldo + c, n, a.vec_out, z);
        if (p.n < 1 || p.s < 0) return;
    } else if (p.s < 0) {
        for (int r = ty; busy && r < p.n; r += deep) {
            const int64_t o = (int64_t)(p.first + r) * a.ldo + c;
            store8((O*)a.out + o, n, a.vec_out, z);
        }
        return;
    }
    const int full = p.n / deep, rounds = full / U;  // rows that every thread has; rounds of U of them
    const auto row = [&](int j) { return (int64_t)p.first + ty + (j < full ? j : full - 1) * deep; };
    Raw8 now[U], next[U];
    float weight[8], shift[8];
    if constexpr (!SUMS || WHOLE) {
        const float* w = a.weight && busy ? a.weight + c : nullptr;
        const float* b = a.bias && busy ? a.bias + c : nullptr;
#pragma unroll
        for (int i = 0; i < 8; ++i) weight[i] = 1.0f, shift[i] = 0.0f;
        if (w)
#pragma unroll
            for (int i = 0; i < 8; ++i) weight[i] = w[i < n ? i : n - 1];
        if (b)
#pragma unroll
            for (int i = 0; i < 8; ++i) shift[i] = b[i < n ? i : n - 1];
    }
    const bool quick = busy && rounds && a.vec_x && a.vec_out && n == 8;
    const auto start = [&] {
#pragma unroll
        for (int u = 0; u < U; ++u) now[u] = norm_get<T, true>(a, row(u), c, 8);
    };
    if (!SUMS && quick) start();
    // `per` lanes of a wave share a group's sums
    int per = 64;
    while (per * ng > NT) per >>= 1;
    const int g = tid / per, l = tid % per;
    double2 t{0.0, 0.0};
    if constexpr (SUMS) {
        double s[8] = {}, q[8] = {};
        const auto add = [&](const Raw8& raw) {
            float v[8];
            norm_numbers<T>(raw, v);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const double d = (double)v[i];
                s[i] += d;
                q[i] = __builtin_fma(d, d, q[i]);
            }
        };
        int r = ty;
        if (quick) {
            start();
#pragma unroll 1
            for (int j = 0; j < rounds; ++j) {
#pragma unroll
                for (int u = 0; u < U; ++u) next[u] = norm_get<T, true>(a, row((j + 1) * U + u), c, 8);
#pragma unroll
                for (int u = 0; u < U; ++u) add(now[u]);
#pragma unroll
                for (int u = 0; u < U; ++u) now[u] = next[u];
            }
            r += rounds * U * deep;
        }
        if (busy)
#pragma unroll 1
            for (; r < p.n; r += deep) add(norm_get<T, false>(a, p.first + r, c, n));
        // The threads' sums of each group: where 8 channels lie in one group (or two), a value a thread and group, else one a channel.
        const int fold = a.gw % 8 == 0 ? 1 : a.gw == 4 ? 2 : 0;
        if (fold) {
            double2* f = (double2*)red;
            const double s0 = (s[0] + s[1]) + (s[2] + s[3]), s1 = (s[4] + s[5]) + (s[6] + s[7]);
            const double q0 = (q[0] + q[1]) + (q[2] + q[3]), q1 = (q[4] + q[5]) + (q[6] + q[7]);
            if (fold == 1) {
                f[tid] = double2{s0 + s1, q0 + q1};
            } else {
                f[2 * tid] = double2{s0, q0};
                f[2 * tid + 1] = double2{s1, q1};
            }
            __syncthreads();
            const int cw = fold == 1 ? a.gw / 8 : 1, all = deep * cw;  // values a row and group; a group's
            if (g < ng)
                for (int e = l; e < all; e += per) {
                    const int y = e / cw, x = e - y * cw;
                    const double2 v = fold == 1 ? f[y * wide + g * cw + x] : f[y * 2 * wide + g];
                    t.x += v.x;
                    t.y += v.y;
                }
        } else {
#pragma unroll 1
            for (int k = 0; k < 2; ++k) {
                if (busy)
#pragma unroll
                    for (int i = 0; i < 8; ++i) red[(ty * wide + tx) * 8 + i] = k ? q[i] : s[i];
                __syncthreads();
                double sum = 0.0;
                if (g < ng)
                    for (int e = l; e < deep * a.gw; e += per) {
                        const int y = e / a.gw;
                        sum += red[y * wide * 8 + g * a.gw + (e - y * a.gw)];
                    }
                if (k) t.y = sum;
                else t.x = sum;
                __syncthreads();
            }
        }
    } else {
        const int tiles = (int)((uint32_t)(p.p1 - p.p0 + a.rows - 1) / (uint32_t)a.rows);
        if (g < ng) {
            const double2* v = a.parts + (int64_t)(g0 + g) * a.ids + p.id0;
            for (int i = l; i < tiles; i += 8 * per) {  // (eight on their way at a time)
                double2 u[8];
#pragma unroll
                for (int k = 0; k < 8; ++k) u[k] = v[i + k * per < tiles ? i + k * per : tiles - 1];
#pragma unroll
                for (int k = 0; k < 8; ++k) {
                    const bool in = i + k * per < tiles;
                    t.x += in ? u[k].x : 0.0;
                    t.y += in ? u[k].y : 0.0;
                }
            }
        }
    }
    for (int o = 1; o < per; o <<= 1) {
        t.x += __shfl_xor(t.x, o, 64);
        t.y += __shfl_xor(t.y, o, 64);
    }
    if constexpr (SUMS && !WHOLE) {
        if (g < ng && l == 0) a.parts[(int64_t)(g0 + g) * a.ids + id] = t;
        return;
    } else {
        if (g < ng && l == 0) {
            // (the quotient by two steps of Newton, the root by one, on the unit's values, to 2^-40 and better: a few instructions,
            // where the library's take a kilobyte of code)
            const double count = (double)(p.p1 - p.p0) * (double)a.gw;
            double one = __builtin_amdgcn_rcp(count);
            one = __builtin_fma(__builtin_fma(-count, one, 1.0), one, one);
            one = __builtin_fma(__builtin_fma(-count, one, 1.0), one, one);
            const double mean = t.x * one;
            double var = t.y * one - mean * mean;
            var = (var < 0.0 ? 0.0 : var) + (double)a.eps;  // (NaN stays)
            double r = __builtin_amdgcn_rsq(var);
            r = r * __builtin_fma(-0.5 * var * r, r, 1.5);
            Stat st;
            st.hi = (float)mean;
            st.lo = (float)(mean - (double)st.hi);
            st.r = (float)r;
            if (kWide<T> && !(st.r > 0x1p-100f && st.r < 0x1p100f)) {
                // Differences from the mean could overflow, or 1 / spread could (eps 0). (A mean above 1 has no differences that small.)
                const bool large = st.r < 1.0f, small = st.r > 1.0f && mean < 1.0 && mean > -1.0;
                if (large || small) {
                    const double by = large ? 0x1p-64 : 0x1p64;
                    st.hi = (float)(mean * by);
                    st.lo = (float)(mean * by - (double)st.hi);
                    st.r = -(float)(r * (large ? 0x1p64 : 0x1p-64));
                }
            }
            stats[g] = st;
        }
        __syncthreads();
        if (!busy) return;
        // per channel: x less the mean (two parts), times scale, plus shift
        float hi[8], lo[8], scale[8];
        bool far = false;  // some are taken times a power of two first
        const auto stat = [&](int i) { return stats[(c - c0 + (i < n ? i : n - 1)) / a.gw]; };
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const Stat st = stat(i);
            hi[i] = st.hi;
            lo[i] = st.lo;
            scale[i] = (kWide<T> ? __builtin_fabsf(st.r) : st.r) * weight[i];
            if (kWide<T>) far = far || st.r < 0.0f;
        }
        // (a loop for each activation, short: what a block has to fetch of its code for the first time costs it a microsecond a
        // few KB)
        with_act(a.act, [&](auto one) {
            const auto result = [&](const Raw8& raw, float (&v)[8], bool scaled) {
                norm_numbers<T>(raw, v);
                if (scaled)
#pragma unroll 1
                    for (int i = 0; i < 8; ++i) {
                        const float by = times(stat(i));
#pragma unroll
                        for (int q = 0; q < 8; ++q) v[q] = q == i ? v[q] * by : v[q];
                    }
#pragma unroll
                for (int i = 0; i < 8; ++i) v[i] = activated<decltype(one)::value, sizeof(O) == 4>(__builtin_fmaf((v[i] - hi[i]) - lo[i], scale[i], shift[i]));
            };
            int r = ty;
            if (quick && !(kWide<T> && far)) {
                if constexpr (SUMS) start();
#pragma unroll 1
                for (int j = 0; j < rounds; ++j) {
#pragma unroll
                    for (int u = 0; u < U; ++u) next[u] = norm_get<T, true>(a, row((j + 1) * U + u), c, 8);
#pragma unroll
                    for (int u = 0; u < U; ++u) {
                        float v[8];
                        result(now[u], v, false);
                        store8((O*)a.out + row(j * U + u) * a.ldo + c, 8, true, v);
                    }
#pragma unroll
                    for (int u = 0; u < U; ++u) now[u] = next[u];
                }
                r += rounds * U * deep;
            }
#pragma unroll 1
            for (; r < p.n; r += deep) {
                float v[8];
                result(norm_get<T, false>(a, p.first + r, c, n), v, kWide<T> && far);
                store8((O*)a.out + (int64_t)(p.first + r) * a.ldo + c, n, a.vec_out, v);
            }
        });
    }
}

struct NormPlan {
    int slab, slabs, rows, threads;  // rows 0: a tile is a segment
    int64_t ids;
};
// A block a segment and slab where segments have up to 512 rows by the mean (a wave where up to 32, or up to 256 and 1024 such blocks
// and more: 76,800 segments of one row of 256 fp16 303 to 358 us, 1000 of 40 13, 422 of 182 22; with 512 threads 2347, 43, 29), or where
// that is the shorter of two estimates, in microseconds: a CU goes over 1000 rows of a slab in 11 (fp32 16), against two launches, 14
// and the bytes of two reads and a write. Measured, us, in one launch and in two: 33 segments of 700 rows of 256 fp16: 17 and 37; 33
// of 2500: 33 and 67; 8 of 1200 of 1024: 22 and 26; 16 of 4800 of 128: 50 and 25; 4 of 2745 of 512 fp32: 47 and 23. What this costs
// where lengths differ: one segment of 300,000 rows of 64 fp16 among 600 of one row takes 2.7 ms (alone 31 us), one of 100,000 among
// 20,000, which a wave goes over, 5.0 ms.
static NormPlan norm_plan(const pmg_group_norm_args& q) {
    NormPlan p;
    const int gw = q.C / q.groups;
    // whole groups, whole 16 bytes (where the groups allow it), 64 channels or more
    int unit = 1;
    while (unit < 8 && unit * gw % 8) unit *= 2;
    p.slab = unit;
    while (p.slab * gw < 64) p.slab += unit;
    if (p.slab > q.groups) p.slab = q.groups;
    p.slabs = (q.groups + p.slab - 1) / p.slab;
    p.rows = 0;
    p.threads = 512;
    p.ids = q.segments + 2;
    const int64_t S = q.segments > 0 ? q.segments : 1;
    const double mean = (double)q.M / (double)S;
    if ((mean <= 32.0 || (mean <= 256.0 && S * p.slabs >= 1024)) && p.slab * gw <= 512) p.threads = 64;
    if (mean <= 512.0) return p;
    const int es = q.type == PMG_TYPE_F32 ? 4 : 2, os = q.out_type == PMG_TYPE_F32 ? 4 : 2;
    const double one = 6.0 + (double)((S * p.slabs + 255) / 256) * mean * (es == 4 ? 0.016 : 0.011);
    // (one or two rounds of a block a CU, which take 13 each whatever they do, by how much of them the segments' tiles fill; one a
    // segment may end inside a tile)
    const double bytes = (double)q.M * q.C * (2 * es + os) / 7.5e6;
    double two = 1e30;
    int64_t each = 1;
    for (int rounds = 1; rounds <= 2; ++rounds) {
        const int64_t want = 256 * rounds / p.slabs, e = (want - (S + 1) / 2) / S;
        if (e < 1) continue;
        const double t = 1.0 + 13.0 * rounds + bytes * want / (double)(S * e);
        if (t < two) {
            two = t;
            each = e;
        }
    }
    p.threads = 1024;
    if (one < two) return p;
    p.rows = (int)__builtin_ceil(mean / (double)each);
    p.ids = piece_tiles(q.M, q.segments, p.rows);
    return p;
}

template <class T, class O, int NT, bool WHOLE, bool SUMS>
static int launch_norm_k(NormArgs& a, const NormPlan& pl, hipStream_t s) {
    const int64_t most = grid_blocks(NT) / pl.slabs;
    for (int64_t i = 0; i < pl.ids; i += most) {
        a.id0 = (uint32_t)i;
        const dim3 grid((uint32_t)((pl.ids - i < most ? pl.ids - i : most) * pl.slabs));
        hipLaunchKernelGGL((norm_k<T, O, NT, WHOLE, SUMS>), grid, dim3(NT), 0, s, a);
        if (int e = check_launch("norm_k")) return e;
    }
    return PMG_OK;
}
template <class T, class O>
static int launch_norm_to(NormArgs& a, const NormPlan& pl, hipStream_t s) {
    if (pl.rows) return launch_norm_k<T, O, 1024, false, false>(a, pl, s);
    if (pl.threads == 64) return launch_norm_k<T, O, 64, true, true>(a, pl, s);
    return pl.threads == 512 ? launch_norm_k<T, O, 512, true, true>(a, pl, s) : launch_norm_k<T, O, 1024, true, true>(a, pl, s);
}
template <class T>
static int launch_norm(NormArgs& a, const NormPlan& pl, hipStream_t s) {
    if (pl.rows)
        if (int e = launch_norm_k<T, T, 1024, false, true>(a, pl, s)) return e;
    if (a.out_type == PMG_TYPE_F32) return launch_norm_to<T, float>(a, pl, s);
    if (a.out_type == PMG_TYPE_F16) return launch_norm_to<T, _Float16>(a, pl, s);
    return launch_norm_to<T, __bf16>(a, pl, s);
}

}  // namespace pmg

using namespace pmg;

static int norm_args(const pmg_group_norm_args& q) {
    PMG_REQUIRE(q.type >= PMG_TYPE_F32 && q.type <= PMG_TYPE_BF16, "type must be f32, f16 or bf16");
    PMG_REQUIRE(q.out_type >= PMG_TYPE_F32 && q.out_type <= PMG_TYPE_BF16, "out_type must be f32, f16 or bf16");
    PMG_REQUIRE(q.act >= PMG_ACT_NONE && q.act <= PMG_ACT_GELU_TANH, "unknown activation");
    PMG_REQUIRE(q.M >= 0 && q.M < ((int64_t)1 << 31) - 2048, "M out of range");  // (a block counts a round of up to 1024 rows past the last)
    PMG_REQUIRE(q.C >= 1 && q.C <= 4096 && q.groups >= 1 && q.C % q.groups == 0, "C must be 1 .. 4096 and a multiple of groups");
    PMG_REQUIRE(q.ldx >= q.C && q.ldo >= q.C, "row strides must cover the row");
    PMG_REQUIRE(q.segments >= 0 && q.segments < (int64_t)1 << 31, "segments out of range");
    PMG_REQUIRE(q.offsets || q.segments == 1, "without offsets there is one segment");
    PMG_REQUIRE(q.eps >= 0.0f && q.eps <= 1.0e30f, "eps must be 0 .. 1e30");
    return PMG_OK;
}

extern "C" size_t pmg_group_norm_workspace_bytes(const pmg_group_norm_args* p) {
    if (!p || norm_args(*p) != PMG_OK || p->M == 0) return 0;
    const NormPlan pl = norm_plan(*p);
    return pl.rows ? (size_t)pl.ids * (size_t)p->groups * sizeof(double2) : 0;
}

extern "C" int pmg_group_norm(const pmg_group_norm_args* p, void* workspace, size_t workspace_bytes, void* stream) {
    PMG_REQUIRE(p, "null args");
    const pmg_group_norm_args& q = *p;
    if (int e = norm_args(q)) return e;
    if (q.M == 0) return PMG_OK;
    PMG_REQUIRE(q.x && q.out, "null buffer");
    const auto at = [](const void* v, int n) { return (reinterpret_cast<uintptr_t>(v) & (uintptr_t)(n - 1)) == 0; };
    const int es = q.type == PMG_TYPE_F32 ? 4 : 2, os = q.out_type == PMG_TYPE_F32 ? 4 : 2;
    PMG_REQUIRE(at(q.x, es) && at(q.out, os) && at(q.weight, 4) && at(q.bias, 4) && at(q.offsets, 8), "buffers must be aligned to their elements");
    const NormPlan pl = norm_plan(q);
    PMG_REQUIRE(!pl.rows || (workspace && aligned16(workspace) && workspace_bytes >= pmg_group_norm_workspace_bytes(p)), "workspace too small, null or not 16-byte aligned");
    NormArgs a{};
    a.x = q.x;
    a.ldx = q.ldx;
    a.P = (int)q.M;
    a.ids = pl.ids;
    a.C = q.C;
    a.G = q.groups;
    a.gw = q.C / q.groups;
    a.weight = q.weight;
    a.bias = q.bias;
    a.offsets = q.offsets;
    a.S = q.segments;
    a.eps = q.eps;
    a.act = q.act;
    a.out = q.out;
    a.out_type = q.out_type;
    a.ldo = q.ldo;
    a.fresh = q.zero_rest;
    a.slab = pl.slab;
    a.slabs = pl.slabs;
    a.rows = pl.rows;
    a.parts = (double2*)workspace;
    const bool even = pl.slabs == 1 || pl.slab * a.gw % 8 == 0;  // (blocks start on whole chunks)
    a.vec_x = even && at(q.x, 16) && q.ldx * es % 16 == 0;
    a.vec_out = even && at(q.out, 16) && q.ldo * os % 16 == 0;
    hipStream_t s = (hipStream_t)stream;
    if (q.type == PMG_TYPE_F32) return launch_norm<float>(a, pl, s);
    if (q.type == PMG_TYPE_F16) return launch_norm<_Float16>(a, pl, s);
    return launch_norm<__bf16>(a, pl, s);
}
