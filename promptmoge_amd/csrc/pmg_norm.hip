// Group norm of rows with channels last, with an activation: for each segment of rows (a frame) and group of C / G channels,
// y = act((x - mean) rsqrt(var + eps) weight[c] + bias[c]), mean and var over the segment's rows and the group's channels.
//
// Sums of x and x^2 are held in 64 bits: their products are exact and nothing overflows, and mean and var come out to fp32's
// accuracy where the mean is 10^4 times the spread (for fp32 inputs E[x^2] - mean^2 in 64 bits loses 2^-53 (mean / spread)^2).
// The mean is subtracted in two fp32 parts.
#include "pmg_epilogue.h"

namespace pmg {

struct NormArgs : Epilogue {
    const void* x;
    const float* weight;  // [C] or NULL
    const float* bias;
    const int64_t* offsets;  // [S + 1], or NULL: one segment of all rows
    double2* parts;          // [tile][G]: sums of x and x^2
    int64_t ldx, S;
    int M, C, G, gw, type;  // gw: channels a group
    int slab, slabs;        // groups a block takes; blocks over the groups
    int rows;               // a tile's rows
    int vec_x, fresh;
    float eps;
    uint32_t tiles, id0;
};

// Pieces and the numbers of their tiles: as in the grouped products, those in front of segment 0, the segments, those behind the last.
__device__ inline int norm_bound(const NormArgs& a, int64_t j) {
    if (j <= 0) return 0;
    if (j > a.S + 1) return a.M;
    if (!a.offsets) return j == 1 ? 0 : a.M;
    const int64_t o = a.offsets[j - 1];
    return o < 0 ? 0 : o > a.M ? a.M : (int)o;
}
struct NormPiece {
    int first, n, p0, p1, s;  // a tile's rows first .. first + n - 1 of the piece p0 .. p1; segment s (-1: of none)
    uint32_t id0;             // number of the piece's first tile
};
__device__ inline NormPiece norm_piece(const NormArgs& a, uint32_t id, bool whole) {
    const int lane = threadIdx.x & 63;
    int64_t lo = 0;
    if (whole) {
        lo = id;
    } else {
        int64_t n = a.S + 2;
        while (n > 1) {
            const int64_t step = (n + 63) >> 6, c = lo + lane * step;
            const bool in = lane * step < n && (int64_t)((uint32_t)norm_bound(a, c) / (uint32_t)a.rows) + c <= (int64_t)id;
            const uint64_t not_in = ~__ballot(in);
            int64_t cnt = not_in ? __builtin_ctzll(not_in) : 64;
            cnt = cnt < 1 ? 0 : cnt - 1;
            lo += cnt * step;
            n = n - cnt * step < step ? n - cnt * step : step;
        }
    }
    NormPiece p;
    p.p0 = __builtin_amdgcn_readfirstlane(norm_bound(a, lo));
    p.p1 = __builtin_amdgcn_readfirstlane(norm_bound(a, lo + 1));
    p.s = __builtin_amdgcn_readfirstlane(lo >= 1 && lo <= a.S ? (int)(lo - 1) : -1);
    p.id0 = whole ? id : __builtin_amdgcn_readfirstlane((uint32_t)p.p0 / (uint32_t)a.rows + (uint32_t)lo);
    const int64_t first = whole ? p.p0 : p.p0 + (int64_t)(id - p.id0) * a.rows;
    const int64_t end = whole || p.p1 - first < a.rows ? p.p1 : first + a.rows;
    p.n = first < p.p0 || first >= p.p1 ? 0 : (int)(end - first);
    p.first = p.n > 0 ? (int)first : 0;
    return p;
}

template <class T>
__device__ inline void get8(const NormArgs& a, int64_t m, int c, int n, float (&v)[8]) {
    load8((const T*)a.x + m * a.ldx + c, n, a.vec_x, v);
}

constexpr int kNormThreads = 512;

struct Stat {
    float hi, lo, r;  // mean in two parts, 1 / spread
};

// A block's slab of whole groups (8 channels a thread, `wide` threads a row) of a tile's rows. WHOLE: a tile is a segment, sums
// and results in one launch; else SUMS writes the tile's sums, and without it the segment's are added up (in the order of its
// tiles) and applied.
template <class T, bool WHOLE, bool SUMS>
__global__ __launch_bounds__(kNormThreads) void norm_k(NormArgs a) {
    __shared__ double red[kNormThreads * 8];
    __shared__ Stat stats[64];  // (a slab has at most 64 groups)
    double2 total{0.0, 0.0};
    const int tid = threadIdx.x;
    const int slab = (int)(blockIdx.x % (uint32_t)a.slabs);
    const uint32_t id = a.id0 + blockIdx.x / (uint32_t)a.slabs;
    const NormPiece p = norm_piece(a, id, WHOLE);
    if (p.n < 1) return;
    if (p.s < 0 && (SUMS ? !WHOLE || !a.fresh : !a.fresh)) return;
    const int g0 = slab * a.slab, ng = a.G - g0 < a.slab ? a.G - g0 : a.slab;
    const int c0 = g0 * a.gw, width = ng * a.gw, wide = (width + 7) / 8;
    const int tx = tid % wide, ty = tid / wide, deep = kNormThreads / wide;  // (threads behind the last whole row: ty == deep, idle)
    const int c = c0 + 8 * tx, n = c0 + width - c < 8 ? c0 + width - c : 8;
    const bool busy = ty < deep;
    if (p.s < 0) {
        const float z[8] = {};
        for (int r = ty; busy && r < p.n; r += deep) {
            const int64_t o = (int64_t)(p.first + r) * a.ldo + c;
            if (a.out_type == PMG_TYPE_F32) store8((float*)a.out + o, n, a.vec_out, z);
            else store8((_Float16*)a.out + o, n, a.vec_out, z);
        }
        return;
    }
    if constexpr (SUMS) {
        double s[8] = {}, q[8] = {};
        const auto add = [&](const float (&v)[8]) {
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const double d = (double)v[i];
                s[i] += d;
                q[i] = __builtin_fma(d, d, q[i]);
            }
        };
        if (busy) {
            int r = ty;
            for (; r + 3 * deep < p.n; r += 4 * deep) {
                float v[4][8];
#pragma unroll
                for (int u = 0; u < 4; ++u) get8<T>(a, p.first + r + u * deep, c, n, v[u]);
#pragma unroll
                for (int u = 0; u < 4; ++u) add(v[u]);
            }
            for (; r < p.n; r += deep) {
                float v[8];
                get8<T>(a, p.first + r, c, n, v);
                add(v);
            }
        }
        // over the block's rows, then over a group's channels
        double2 t{0.0, 0.0};
#pragma unroll 1
        for (int k = 0; k < 2; ++k) {
            if (busy)
#pragma unroll
                for (int i = 0; i < 8; ++i) red[(ty * wide + tx) * 8 + i] = k ? q[i] : s[i];
            __syncthreads();
            double col[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const int e = tid + i * kNormThreads;
                col[i] = 0.0;
                if (e < 8 * wide)
                    for (int y = 0; y < deep; ++y) col[i] += red[y * wide * 8 + e];
            }
            __syncthreads();
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (tid + i * kNormThreads < 8 * wide) red[tid + i * kNormThreads] = col[i];
            __syncthreads();
            if (tid < ng) {
                double sum = 0.0;
                for (int e = tid * a.gw; e < (tid + 1) * a.gw; ++e) sum += red[e];
                if (k) t.y = sum;
                else t.x = sum;
            }
            __syncthreads();
        }
        if constexpr (!WHOLE) {
            if (tid < ng) a.parts[(int64_t)id * a.G + g0 + tid] = t;
            return;
        }
        total = t;
    } else {
        // the sums of the segment's tiles, shared out over the threads and added in order
        const uint32_t tiles = (uint32_t)(p.p1 - p.p0 + a.rows - 1) / (uint32_t)a.rows;
        const int of = kNormThreads / ng, part = tid / ng, g = tid % ng;
        double2 t{0.0, 0.0};
        if (part < of) {
            for (uint32_t i = part; i < tiles; i += of) {
                const double2 v = a.parts[(int64_t)(p.id0 + i) * a.G + g0 + g];
                t.x += v.x;
                t.y += v.y;
            }
            red[part * ng + g] = t.x;
            red[kNormThreads + part * ng + g] = t.y;
        }
        __syncthreads();
        if (tid < ng)
            for (int i = 0; i < of; ++i) {
                total.x += red[i * ng + tid];
                total.y += red[kNormThreads + i * ng + tid];
            }
    }
    if (tid < ng) {
        const double count = (double)(p.p1 - p.p0) * (double)a.gw, mean = total.x / count;
        double var = total.y / count - mean * mean;
        var = var < 0.0 ? 0.0 : var;  // (NaN stays)
        Stat t;
        t.hi = (float)mean;
        t.lo = (float)(mean - (double)t.hi);
        t.r = (float)(1.0 / __builtin_sqrt(var + (double)a.eps));
        stats[tid] = t;
    }
    __syncthreads();
    if (!busy) return;
    // per channel: x less the mean (two parts), times scale, plus shift
    float hi[8], lo[8], scale[8], shift[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const int ch = c + (i < n ? i : n - 1);
        const Stat t = stats[(ch - c0) / a.gw];
        hi[i] = t.hi;
        lo[i] = t.lo;
        scale[i] = a.weight ? t.r * a.weight[ch] : t.r;
        shift[i] = a.bias ? a.bias[ch] : 0.0f;
    }
    const auto apply = [&](int64_t m, float (&v)[8]) {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = __builtin_fmaf((v[i] - hi[i]) - lo[i], scale[i], shift[i]);
        activate8(v, a.act, a.out_type == PMG_TYPE_F32);
        const int64_t o = m * a.ldo + c;
        if (a.out_type == PMG_TYPE_F32) store8((float*)a.out + o, n, a.vec_out, v);
        else if (a.out_type == PMG_TYPE_F16) store8((_Float16*)a.out + o, n, a.vec_out, v);
        else store8((__bf16*)a.out + o, n, a.vec_out, v);
    };
    int r = ty;
    for (; r + 3 * deep < p.n; r += 4 * deep) {
        float v[4][8];
#pragma unroll
        for (int u = 0; u < 4; ++u) get8<T>(a, p.first + r + u * deep, c, n, v[u]);
#pragma unroll
        for (int u = 0; u < 4; ++u) apply(p.first + r + u * deep, v[u]);
    }
    for (; r < p.n; r += deep) {
        float v[8];
        get8<T>(a, p.first + r, c, n, v);
        apply(p.first + r, v);
    }
}

struct NormPlan {
    int slab, slabs, rows;  // rows 0: a tile is a segment
    int64_t ids;
};
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
    p.ids = q.segments + 2;
    const double mean = (double)q.M / (double)(q.segments > 0 ? q.segments : 1);
    if (mean > 512.0) {
        const int64_t want = (512 + p.slabs - 1) / p.slabs;  // tiles, for about two blocks a CU
        p.rows = (int)((q.M + want - 1) / want);
        if (p.rows < 64) p.rows = 64;
        p.ids = q.M / p.rows + q.segments + 2;
    }
    return p;
}

template <class T>
static int launch_norm(NormArgs& a, const NormPlan& pl, hipStream_t s) {
    const int64_t most = grid_blocks(kNormThreads) / pl.slabs;
    for (int sums = pl.rows ? 1 : 0; sums >= 0; --sums) {
        for (int64_t i = 0; i < pl.ids; i += most) {
            a.id0 = (uint32_t)i;
            const dim3 grid((uint32_t)((pl.ids - i < most ? pl.ids - i : most) * pl.slabs));
            if (!pl.rows) hipLaunchKernelGGL((norm_k<T, true, true>), grid, dim3(kNormThreads), 0, s, a);
            else if (sums) hipLaunchKernelGGL((norm_k<T, false, true>), grid, dim3(kNormThreads), 0, s, a);
            else hipLaunchKernelGGL((norm_k<T, false, false>), grid, dim3(kNormThreads), 0, s, a);
            if (int e = check_launch("norm_k")) return e;
        }
    }
    return PMG_OK;
}

}  // namespace pmg

using namespace pmg;

static int norm_args(const pmg_group_norm_args& q) {
    PMG_REQUIRE(q.type >= PMG_TYPE_F32 && q.type <= PMG_TYPE_BF16, "type must be f32, f16 or bf16");
    PMG_REQUIRE(q.out_type >= PMG_TYPE_F32 && q.out_type <= PMG_TYPE_BF16, "out_type must be f32, f16 or bf16");
    PMG_REQUIRE(q.act >= PMG_ACT_NONE && q.act <= PMG_ACT_GELU_TANH, "unknown activation");
    PMG_REQUIRE(q.M >= 0 && q.M < ((int64_t)1 << 31) - 512, "M out of range");
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
    a.M = (int)q.M;
    a.C = q.C;
    a.G = q.groups;
    a.gw = q.C / q.groups;
    a.type = q.type;
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
