// Routing of rows to experts: each row's k best experts with their weights, and the pairs (row, slot) in the order of the
// experts, as the grouped products take them; and the rows' experts put together again.
//
// Measured (MI355X), and what bounds it: 76,800 rows to 2 of 16, fp32: 12.2 us (choices 6.5, order 5.7: chains of loads, barriers and
// counts); 4800 rows to 8 of 256: 21 us; one row to 4 of 64: 6.8. combine of 76,800 x 2 x 256 fp16 onto fp32: 37.7 us, 5.9 TB/s.
#include "pmg_epilogue.h"

namespace pmg {

struct RouteArgs {
    const void* logits;
    const uint8_t* mask;
    float* weights;    // [M][k]
    int32_t* experts;  // [M][k]
    int64_t* offsets;  // [E + 1]
    int32_t* pairs;    // [M k]
    int32_t* rows;     // [M k]
    int32_t* counts;   // [blocks][E + 1]: a block's pairs of each expert (E: of none)
    int64_t ld;
    int M, E, k, sigmoid, normalize;
    int per, blocks;   // rows a block
};

constexpr int kRouteThreads = 1024, kRouteWaves = kRouteThreads / 64;

// A key that rises with x, 0 for what is not chosen (-infinity, NaN); and x of a key. -0 is 0, as in a comparison.
__device__ inline uint32_t key_of(float x) {
    const uint32_t u = f2u(x + 0.0f);
    return x > -__builtin_inff() ? (u >> 31 ? ~u : u | 0x80000000u) : 0u;
}
__device__ inline float of_key(uint32_t k) { return u2f(k >> 31 ? k & 0x7fffffffu : ~k); }

// exp(d) for d <= 0, within 2^-21 of its value, its argument in two parts; below 2^-126 it may be 0. NaN stays.
__device__ inline float exp_below(float d) {
    const float b = __builtin_fminf(-d, 200.0f), hi = b * -PMG_LOG2E;
    const float lo = __builtin_fmaf(b, -1.92596299e-8f, __builtin_fmaf(b, -PMG_LOG2E, -hi));
    const float e = __builtin_amdgcn_exp2f(hi);
    return d != d ? d : __builtin_fmaf(e, lo * 0.69314718f, e);
}

// f(value of another lane) over groups of L lanes, until all of a group have met: within 16 lanes by moves between
// neighbours (quads, then mirrored, which after a step is as good as swapped), beyond by the exchange through LDS. A register move
// takes a tenth of that exchange, and a row's k rounds are one behind the other.
template <int CTRL>
__device__ inline uint32_t from_lane(uint32_t v) {
    return (uint32_t)__builtin_amdgcn_update_dpp((int)v, (int)v, CTRL, 0xf, 0xf, false);
}
template <int L, class F>
__device__ inline void over_lanes(const F& f) {
    if constexpr (L > 1) f([](uint32_t v) { return from_lane<0xb1>(v); });   // lane ^ 1
    if constexpr (L > 2) f([](uint32_t v) { return from_lane<0x4e>(v); });   // lane ^ 2
    if constexpr (L > 4) f([](uint32_t v) { return from_lane<0x141>(v); });  // 7 - lane of eight
    if constexpr (L > 8) f([](uint32_t v) { return from_lane<0x140>(v); });  // 15 - lane of 16
    if constexpr (L > 16) f([](uint32_t v) { return (uint32_t)__shfl_xor((int)v, 16, 64); });
    if constexpr (L > 32) f([](uint32_t v) { return (uint32_t)__shfl_xor((int)v, 32, 64); });
}

// The k best of a row on L lanes of a wave, I experts a lane, in k rounds of a largest (key, lowest index first). Gives the
// lane's slot's expert (-1: none).
template <class T, int I, int L>
__device__ inline int choose(const RouteArgs& a, int64_t m, bool there, int l) {
    const bool on = there && (!a.mask || a.mask[m]);
    const T* row = (const T*)a.logits + m * a.ld;
    uint32_t key[I];
    float top = -__builtin_inff(), sum = 0.0f, x[I];
#pragma unroll
    for (int i = 0; i < I; ++i) {
        const int e = l + i * L;
        x[i] = there && e < a.E ? (float)row[e] : -__builtin_inff();
    }
#pragma unroll
    for (int i = 0; i < I; ++i) {
        key[i] = key_of(x[i]);
        top = x[i] > top ? x[i] : top;
    }
    if (!a.sigmoid) {
        over_lanes<L>([&](auto other) {
            const float t = u2f(other(f2u(top)));
            top = t > top ? t : top;
        });
        top = top > -__builtin_inff() ? top : 0.0f;
#pragma unroll
        for (int i = 0; i < I; ++i) sum += exp_below(x[i] - top);  // (NaN, and infinity less itself: the row's weights are NaN)
        over_lanes<L>([&](auto other) { sum += u2f(other(f2u(sum))); });
    }
    float mine = 0.0f, chosen = 0.0f;  // lane j keeps the j-th
    float base = 0.0f;                 // sigmoids that are only looked at relative to each other: times exp(-base), none is lost
    int expert = -1;
    for (int j = 0; j < a.k; ++j) {
        uint32_t k = key[0];
        int e = l;
#pragma unroll
        for (int i = 1; i < I; ++i)
            if (key[i] > k) {
                k = key[i];
                e = l + i * L;
            }
        over_lanes<L>([&](auto other) {
            const uint32_t k2 = other(k);
            const int e2 = (int)other((uint32_t)e);
            const bool better = k2 > k || (k2 == k && e2 < e);
            k = better ? k2 : k;
            e = better ? e2 : e;
        });
        const float v = of_key(k);
        if (j == 0 && a.normalize && k != 0 && v < 0.0f) base = v;
        const float s = base == 0.0f ? sigmoid_wide(v) : exp_below(v - base) * sigmoid_wide(-v);
        const float w = k == 0 ? 0.0f : a.sigmoid ? s : exp_below(v - top) * __builtin_amdgcn_rcpf(sum);
        chosen += w;
        if (l == j) {
            mine = w;
            expert = k == 0 ? -1 : e;
        }
#pragma unroll
        for (int i = 0; i < I; ++i)
            if (l + i * L == e) key[i] = 0;
    }
    if (a.normalize) mine = chosen == 0.0f ? 0.0f : mine * __builtin_amdgcn_rcpf(chosen);
    expert = on ? expert : -1;
    if (there && l < a.k) {
        a.weights[m * a.k + l] = expert >= 0 ? mine : 0.0f;
        a.experts[m * a.k + l] = expert;
    }
    return expert;
}

// Choices of a block's rows, counted in `table` [E + 1] (E: no expert), or kept in `kept` as they are written.
template <class T, int I, int L>
__device__ inline void choose_rows(const RouteArgs& a, int first, int end, int32_t* table, int16_t* kept) {
    constexpr int per = kRouteThreads / L;
    const int l = (int)threadIdx.x % L;
    for (int64_t m0 = first; m0 < end; m0 += per) {  // (every lane takes part: those behind the last row bring nothing)
        const int64_t m = m0 + threadIdx.x / L;
        const int e = choose<T, I, L>(a, m, m < end, l);
        if (m < end && l < a.k) {
            if (table) atomicAdd(table + (e < 0 ? a.E : e), 1);
            else kept[(int)(m - first) * a.k + l] = (int16_t)e;
        }
    }
}

template <class T, int I, int L>
__global__ __launch_bounds__(kRouteThreads) void route_choose_k(RouteArgs a) {
    extern __shared__ int32_t table[];
    const int first = (int)blockIdx.x * a.per, end = a.M - first < a.per ? a.M : first + a.per;
    for (int e = threadIdx.x; e <= a.E; e += kRouteThreads) table[e] = 0;
    __syncthreads();
    choose_rows<T, I, L>(a, first, end, table, nullptr);
    __syncthreads();
    for (int e = threadIdx.x; e <= a.E; e += kRouteThreads) a.counts[(int64_t)blockIdx.x * (a.E + 1) + e] = table[e];
}

// The place of each pair: pairs of lower experts, of this expert in earlier blocks, in this block's earlier waves (a wave has a
// range of its pairs), and in the wave itself, which goes over them 64 at a time. ONE: the choices too, in one block.
template <class T, int I, int L, bool ONE>
__global__ __launch_bounds__(kRouteThreads) void route_order_k(RouteArgs a) {
    constexpr int NW = kRouteWaves;
    extern __shared__ int32_t table[];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, E1 = a.E + 1;
    int32_t* base = table;                    // [E1] each expert's first place, then this block's
    int32_t* all = table + E1;                // [E1] pairs of each expert in all
    int32_t* next = table + (2 + wave) * E1;  // [E1] a wave's: its pairs of each expert, then their next place
    int16_t* kept = (int16_t*)(table + (2 + NW) * E1);  // ONE: the pairs' experts
    const auto of_wave = [&](int w, int e) -> int32_t& { return table[(2 + w) * E1 + e]; };
    const int first = (int)blockIdx.x * a.per, end = a.M - first < a.per ? a.M : first + a.per;
    for (int e = tid; e < (2 + NW) * E1; e += kRouteThreads) table[e] = 0;
    if constexpr (ONE) choose_rows<T, I, L>(a, first, end, nullptr, kept);
    __syncthreads();
    // this block's pairs, a range a wave
    const int64_t p0 = (int64_t)first * a.k, np = (int64_t)(end - first) * a.k;
    const int64_t share = (np + 64 * NW - 1) / (64 * NW) * 64;
    const int64_t w0 = p0 + (wave * share < np ? wave * share : np), w1 = p0 + ((wave + 1) * share < np ? (wave + 1) * share : np);
    const auto expert = [&](int64_t i) -> int {
        const int e = ONE ? (int)kept[i - p0] : a.experts[i];
        return e < 0 ? a.E : e;
    };
    for (int64_t i = w0 + lane; i < w1; i += 64) atomicAdd(next + expert(i), 1);
    if constexpr (!ONE) {
        const uint32_t all_counts = (uint32_t)(a.blocks * E1);
        for (uint32_t i0 = tid; i0 < all_counts; i0 += 8 * kRouteThreads) {  // (eight on their way at a time)
            int32_t n[8];
#pragma unroll
            for (int u = 0; u < 8; ++u) n[u] = a.counts[i0 + u * kRouteThreads < all_counts ? i0 + u * kRouteThreads : i0];
#pragma unroll
            for (int u = 0; u < 8; ++u) {
                const uint32_t i = i0 + u * kRouteThreads;
                const int b = (int)(i / (uint32_t)E1), e = (int)(i - (uint32_t)(b * E1));
                if (n[u] && i < all_counts) {
                    atomicAdd(all + e, n[u]);
                    if (b < (int)blockIdx.x) atomicAdd(base + e, n[u]);
                }
            }
        }
    }
    __syncthreads();
    if constexpr (ONE) {
        for (int e = tid; e < E1; e += kRouteThreads)
            for (int w = 0; w < NW; ++w) all[e] += of_wave(w, e);
        __syncthreads();
    }
    // where each expert starts (one wave), then where each wave does
    if (wave == 0) {
        int32_t before = 0;
        for (int e0 = 0; e0 < E1; e0 += 64) {
            const int e = e0 + lane, n = e < E1 ? all[e] : 0;
            const int32_t incl = (int32_t)wave_incl_scan_u32((uint32_t)n);
            if (e < E1) {
                base[e] += before + incl - n;
                if (blockIdx.x == 0) a.offsets[e] = before + incl - n;
            }
            before += __shfl(incl, 63, 64);
        }
    }
    __syncthreads();
    for (int e = tid; e < E1; e += kRouteThreads) {
        int32_t at = base[e];
        for (int w = 0; w < NW; ++w) {
            const int32_t n = of_wave(w, e);
            of_wave(w, e) = at;
            at += n;
        }
    }
    __syncthreads();
    int bits = 0;
    while ((1 << bits) < E1) ++bits;
    for (int64_t i0 = w0; i0 < w1; i0 += 64) {
        const int64_t i = i0 + lane;
        const bool there = i < w1;
        const int e = there ? expert(i) : a.E;
        const bool none = e == a.E;
        uint64_t same = __ballot(there);
        for (int b = 0; b < bits; ++b) {
            const uint64_t set = __ballot((e >> b) & 1);
            same &= (e >> b) & 1 ? set : ~set;
        }
        const int ahead = __popcll(same & ((1ull << lane) - 1)), n = __popcll(same);
        const int32_t at = there ? next[e] : 0;
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
        if (there) {
            if (ahead == 0) next[e] = at + n;
            a.pairs[at + ahead] = none ? -1 : (int32_t)i;
            a.rows[at + ahead] = none ? -1 : (int32_t)(i / a.k);
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
    }
}

// ------------------------------------------------------------------------------------------------------------ combine
// out[m] = sum_j weights[m][j] y[m][j] + residual[m] in fp32, slots in order; a slot of weight 0 is not read. 8 columns a thread.
struct CombineArgs : Epilogue {
    const void* y;
    const float* weights;
    int64_t M, y_row, y_slot;
    int k, N, vec_y, groups;  // groups of 8 columns a row
};

template <class T>
__global__ __launch_bounds__(256) void combine_k(CombineArgs a) {
    const int64_t all = a.M * a.groups, step = (int64_t)gridDim.x * 256;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < all; i += step) {
        const int64_t m = i / a.groups;
        const int c = 8 * (int)(i - m * a.groups), n = a.N - c < 8 ? a.N - c : 8;
        const T* y = (const T*)a.y + m * a.y_row + c;
        float v[8] = {};
        for (int j = 0; j < a.k; ++j) {
            const float w = a.weights[m * a.k + j];
            if (w != 0.0f) {
                float u[8];
                load8(y + j * a.y_slot, n, a.vec_y, u);
#pragma unroll
                for (int q = 0; q < 8; ++q) v[q] = __builtin_fmaf(w, u[q], v[q]);
            }
        }
        finish8<true>(a, m, c, n, v);
    }
}

}  // namespace pmg

using namespace pmg;

namespace {

struct RoutePlan {
    int lanes, per, blocks;  // lanes a row, rows a block
};
// Four experts a lane of up to 64, 16 of more (a lane's own are looked through faster than other lanes': 4800 rows to 8 of 256 36
// us with four), and at least k lanes. One block where it goes over its rows at most four times; else 512 blocks or fewer, of as
// many rows as they take at once or more, whose table of counts, which each block reads whole, stays within 32,768 (307,200 rows to
// 2 of 8: 17 us; 256 rows a block: 31).
RoutePlan route_plan(const pmg_route_args& q) {
    RoutePlan p;
    p.lanes = q.E > 64 ? 8 : 1;
    while (p.lanes < q.k || (q.E > 64 ? 16 : 4) * p.lanes < q.E) p.lanes *= 2;
    int64_t most = 32768 / (q.E + 1);
    most = most > 512 ? 512 : most;
    int64_t per = (q.M + most - 1) / most;
    if (per < kRouteThreads / p.lanes) per = kRouteThreads / p.lanes;
    if (q.M * p.lanes <= 4 * kRouteThreads && q.M * q.k <= 4096) per = q.M > 0 ? q.M : 1;
    p.per = (int)per;
    p.blocks = (int)((q.M + per - 1) / per);
    return p;
}

int route_args(const pmg_route_args& q) {
    PMG_REQUIRE(q.type >= PMG_TYPE_F32 && q.type <= PMG_TYPE_BF16, "type must be f32, f16 or bf16");
    PMG_REQUIRE(q.M >= 0 && q.E >= 1 && q.E <= 1024 && q.k >= 1 && q.k <= 32 && q.k <= q.E, "E must be 1 .. 1024, k 1 .. 32 and at most E");
    PMG_REQUIRE(q.M < (((int64_t)1 << 31) - 512) / q.k, "M k out of range");
    PMG_REQUIRE(q.ld >= q.E, "row strides must cover the row");
    PMG_REQUIRE(q.score == PMG_SCORE_SOFTMAX || q.score == PMG_SCORE_SIGMOID, "unknown score");
    return PMG_OK;
}

template <class T, int I, int L>
int launch_route(const RouteArgs& a, int bytes, hipStream_t s) {
    if (a.blocks <= 1) {
        hipLaunchKernelGGL((route_order_k<T, I, L, true>), dim3(1), dim3(kRouteThreads), bytes + 2 * a.M * a.k, s, a);
        return check_launch("route_order_k");
    }
    hipLaunchKernelGGL((route_choose_k<T, I, L>), dim3(a.blocks), dim3(kRouteThreads), (a.E + 1) * 4, s, a);
    if (int e = check_launch("route_choose_k")) return e;
    hipLaunchKernelGGL((route_order_k<float, 1, 1, false>), dim3(a.blocks), dim3(kRouteThreads), bytes, s, a);
    return check_launch("route_order_k");
}
template <class T>
int launch_route_of(const RouteArgs& a, int lanes, int bytes, hipStream_t s) {
    if (a.E <= 64) {
        switch (lanes) {
            case 1: return launch_route<T, 4, 1>(a, bytes, s);
            case 2: return launch_route<T, 4, 2>(a, bytes, s);
            case 4: return launch_route<T, 4, 4>(a, bytes, s);
            case 8: return launch_route<T, 4, 8>(a, bytes, s);
            case 16: return launch_route<T, 4, 16>(a, bytes, s);
            default: return launch_route<T, 4, 32>(a, bytes, s);
        }
    }
    switch (lanes) {
        case 8: return launch_route<T, 16, 8>(a, bytes, s);
        case 16: return launch_route<T, 16, 16>(a, bytes, s);
        case 32: return launch_route<T, 16, 32>(a, bytes, s);
        default: return launch_route<T, 16, 64>(a, bytes, s);
    }
}

}  // namespace

extern "C" size_t pmg_route_workspace_bytes(const pmg_route_args* p) {
    if (!p || route_args(*p) != PMG_OK) return 0;
    const RoutePlan pl = route_plan(*p);
    return pl.blocks > 1 ? (size_t)pl.blocks * (size_t)(p->E + 1) * 4 : 0;
}

extern "C" int pmg_route(const pmg_route_args* p, void* workspace, size_t workspace_bytes, void* stream) {
    PMG_REQUIRE(p, "null args");
    const pmg_route_args& q = *p;
    if (int e = route_args(q)) return e;
    PMG_REQUIRE(q.offsets && (q.M == 0 || (q.logits && q.weights && q.experts && q.pairs && q.rows)), "null buffer");
    const auto at = [](const void* v, int n) { return (reinterpret_cast<uintptr_t>(v) & (uintptr_t)(n - 1)) == 0; };
    PMG_REQUIRE(at(q.logits, q.type == PMG_TYPE_F32 ? 4 : 2) && at(q.weights, 4) && at(q.experts, 4) && at(q.offsets, 8) && at(q.pairs, 4) && at(q.rows, 4), "buffers must be aligned to their elements");
    const RoutePlan pl = route_plan(q);
    PMG_REQUIRE(pl.blocks <= 1 || (workspace && at(workspace, 4) && workspace_bytes >= pmg_route_workspace_bytes(p)), "workspace too small, null or not aligned");
    RouteArgs a{};
    a.logits = q.logits;
    a.mask = q.mask;
    a.weights = q.weights;
    a.experts = q.experts;
    a.offsets = q.offsets;
    a.pairs = q.pairs;
    a.rows = q.rows;
    a.counts = (int32_t*)workspace;
    a.ld = q.ld;
    a.M = (int)q.M;
    a.E = q.E;
    a.k = q.k;
    a.sigmoid = q.score == PMG_SCORE_SIGMOID;
    a.normalize = q.normalize;
    a.per = pl.per;
    a.blocks = pl.blocks;
    const int bytes = (2 + kRouteWaves) * (q.E + 1) * 4;
    hipStream_t s = (hipStream_t)stream;
    if (q.type == PMG_TYPE_F32) return launch_route_of<float>(a, pl.lanes, bytes, s);
    if (q.type == PMG_TYPE_F16) return launch_route_of<_Float16>(a, pl.lanes, bytes, s);
    return launch_route_of<__bf16>(a, pl.lanes, bytes, s);
}

extern "C" int pmg_combine(const pmg_combine_args* p, void* stream) {
    PMG_REQUIRE(p, "null args");
    const pmg_combine_args& q = *p;
    PMG_REQUIRE(q.type >= PMG_TYPE_F32 && q.type <= PMG_TYPE_BF16, "type must be f32, f16 or bf16");
    PMG_REQUIRE(q.out_type >= PMG_TYPE_F32 && q.out_type <= PMG_TYPE_BF16, "out_type must be f32, f16 or bf16");
    PMG_REQUIRE(q.M >= 0 && q.M < (int64_t)1 << 31 && q.k >= 1 && q.k <= 32 && q.N >= 1 && q.N <= (1 << 24), "M, k (1 .. 32) or N (1 .. 2^24) out of range");
    PMG_REQUIRE(q.y_slot >= 0 && q.y_row >= 0 && q.ldo >= q.N && (!q.residual || q.ldr >= q.N), "row strides must cover the row");
    if (q.M == 0) return PMG_OK;
    PMG_REQUIRE(q.y && q.weights && q.out, "null buffer");
    const auto at = [](const void* v, int n) { return (reinterpret_cast<uintptr_t>(v) & (uintptr_t)(n - 1)) == 0; };
    const auto bytes = [](int t) { return t == PMG_TYPE_F32 ? 4 : 2; };
    const int es = bytes(q.type), os = bytes(q.out_type);
    PMG_REQUIRE(at(q.y, es) && at(q.out, os) && at(q.weights, 4), "buffers must be aligned to their elements");
    CombineArgs a{};
    a.y = q.y;
    a.weights = q.weights;
    a.M = q.M;
    a.y_row = q.y_row;
    a.y_slot = q.y_slot;
    a.k = q.k;
    a.N = q.N;
    a.groups = (q.N + 7) / 8;
    a.vec_y = at(q.y, 16) && q.y_row * es % 16 == 0 && q.y_slot * es % 16 == 0;
    a.out = q.out;
    a.out_type = q.out_type;
    a.ldo = q.ldo;
    a.vec_out = at(q.out, 16) && q.ldo * os % 16 == 0;
    if (q.residual) {
        PMG_REQUIRE(q.residual_type >= PMG_TYPE_F32 && q.residual_type <= PMG_TYPE_BF16, "residual_type must be f32, f16 or bf16");
        PMG_REQUIRE(at(q.residual, bytes(q.residual_type)), "buffers must be aligned to their elements");
        a.res = q.residual;
        a.res_type = q.residual_type;
        a.ldr = q.ldr;
        a.vec_res = at(q.residual, 16) && q.ldr * bytes(q.residual_type) % 16 == 0;
    }
    const int64_t blocks = (q.M * a.groups + 255) / 256;
    const dim3 grid((uint32_t)(blocks < 16384 ? blocks : 16384));
    hipStream_t s = (hipStream_t)stream;
    if (q.type == PMG_TYPE_F32) hipLaunchKernelGGL(combine_k<float>, grid, dim3(256), 0, s, a);
    else if (q.type == PMG_TYPE_F16) hipLaunchKernelGGL(combine_k<_Float16>, grid, dim3(256), 0, s, a);
    else hipLaunchKernelGGL(combine_k<__bf16>, grid, dim3(256), 0, s, a);
    return check_launch("combine_k");
}
