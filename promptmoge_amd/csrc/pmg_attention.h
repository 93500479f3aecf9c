// Attention inside segments of rows (frames, pool cells): the kernel, instantiated per element type.
//
//   o[i] = sum_j p_ij v[j],  p_i = softmax over the keys j of i's segment that k_mask leaves of
//          cap(scale q_i . k_j) - sum over axes of slope[head][axis] |c_i - c_j|[axis],   cap(x) = cap tanh(x / cap)
//
// One pass over the keys with the running maximum m and sum l of the softmax (fp32, in powers of two). A wave owns 32
// slots: a slot is a query position and one of the G query heads that share a key head. The products are
// formed transposed, S^T = K Q^T and O^T = V^T P^T, so that a lane holds 16 scores of ONE slot: maximum and sum are
// taken in the lane and once across the two halves of the wave, and the scores, rounded to the inputs' type (the
// weights of the second product; l sums the unrounded ones), are that product's operand as they lie. V^T comes from
// row-major V by the transposing LDS read (fp32: by plain reads). K and V tiles go from memory straight to LDS, one tile
// ahead into the other of two buffers: each lane names the 16 bytes it fetches, so rows are gathered by index, the
// banks' swizzle is made by the choice of chunk, and an absent row (masked, behind its segment, a bad index) is fetched
// from a line of zeros. The rows' numbers, mask and coordinates are looked up a key a thread, a group of tiles ahead.
//
// Queries are taken in order of position, 32 NW / G positions a block, whatever segments they fall in: the block
// walks over the keys of all its segments, and each lane counts the keys of its own. No work list is needed, and small
// cells share a wave. A weight of 0 times a value that is infinite or NaN is NaN: where outputs of a block over
// several segments are not finite, the block goes over its segments one by one. (SEG: a block per segment, for few
// queries on many keys.) The keys of a block can be split over gridDim blocks, whose (m, l, O) a second kernel joins.
#pragma once
#include <type_traits>

#include "pmg_dense.h"

namespace pmg {

struct AttnArgs {
    const void* q;
    const void* k;
    const void* v;
    void* out;
    int64_t q_row, q_head, k_row, k_head, v_row, v_head, o_row, o_head;  // strides in elements
    int64_t Mq, Mk;  // rows
    int64_t Pq, Pk;  // positions: the index's length, or the rows
    int64_t S;
    const int64_t* q_off;
    const int64_t* k_off;
    const int32_t* q_index;
    const int32_t* k_index;
    const int32_t* q_coords;
    const int32_t* k_coords;
    const float* slopes;
    const uint8_t* k_mask;
    int Hq, Hk, G, D;
    float scale2;         // scale log2(e)
    float cap2, cap_arg;  // cap log2(e) (0: none); what its argument is multiplied by: 1 / cap for tanh, 2 log2(e) / cap for the exponential
    int seg, splits, zero_rest, fine;
    int whole;  // blocks of one segment each
    int near;   // K and V each below 4 GiB, heads of full width: rows are fetched by 32-bit byte offsets
    uint32_t blocks;
    uint32_t sweep;  // blocks in front of them, which look after what the tables miss
    float* part_o;  // [splits][Hq][Pq][D]; (m, l) [splits][Hq][Pq], l < 0: a position of no segment
    float2* part_ml;
};

// 16-bit types: caps (times log2 e) up to which cap tanh(x / cap) is formed as cap - 2 cap / (1 + e^(2 x / cap)), whose error is
// that of the cap itself: 3e-7 of it, so weights within 8e-5, a sixth of a half step of fp16. Above, as in fp32.
constexpr float kFineCap = 256.0f * 1.44269504f;

__device__ inline int64_t clamp64(int64_t v, int64_t lo, int64_t hi) { return v < lo ? lo : v > hi ? hi : v; }

// The segment of position p: the last s with off[s] <= p, if p < off[s + 1]; -1 otherwise.
__device__ inline int32_t segment_of(const int64_t* off, int64_t S, int64_t p) {
    int64_t lo = 0, hi = S;  // off[lo] <= p is unknown until checked; invariant: answer in [lo - 1, hi - 1]
    while (lo < hi) {
        const int64_t mid = (lo + hi) >> 1;
        if (off[mid] <= p) lo = mid + 1;
        else hi = mid;
    }
    if (lo == 0) return -1;
    return p < off[lo] ? (int32_t)(lo - 1) : -1;
}

// Whether segment s (or -1), found by a search, holds position p, which it may not where offsets fall.
__device__ inline bool in_segment(const int64_t* off, int32_t s, int64_t p) { return s >= 0 && off[s] <= p && p < off[s + 1]; }

// The segment (as above) of position p of each lane, all lanes of a wave taking part; first: a lower bound of the p. A
// search with 64 probes a round for `first`, then among the 64 offsets that follow.
__device__ inline int32_t wave_segment(const int64_t* off, int64_t S, int32_t first, int32_t p) {
    const int lane = threadIdx.x & 63;
    int64_t lo = 0, n = S < 64 ? 0 : S + 1;  // entries before lo are <= first, those from lo + n on are not; (few: all are read)
    while (n > 0) {
        const int64_t step = (n + 63) >> 6, j = (lane + 1) * step - 1;
        const bool le = j < n && off[lo + j] <= first;
        const int t = __popcll(__ballot(le));
        lo += t * step;
        n -= t * step;
        n = n < step - 1 ? n : step - 1;
    }
    const int32_t e = lo + lane <= S ? (int32_t)clamp64(off[lo + lane], -1, 0x7fffffff) : 0x7fffffff;
    int c = 0;
#pragma unroll
    for (int b = 32; b > 0; b >>= 1) c += __shfl(e, c + b - 1, 64) <= p ? b : 0;
    c += __shfl(e, 63, 64) <= p ? 1 : 0;  // (only where all before are)
    if (c == 64) return segment_of(off, S, p);
    const int64_t s = lo + c - 1;
    return s < S ? (int32_t)s : -1;
}

// Whether up to kLook offsets rise, as blocks of one segment each need it.
constexpr int kLook = 64;
__device__ inline bool offsets_rise(const int64_t* off, int64_t S) {
    const int j = threadIdx.x & 63;
    return __all(j >= S || off[j] <= off[j + 1]);
}

// Blocks that hold one segment each: interval j of S + 2 (the rows before the segments, the segments, the rows behind) from
// starts(j) on has the blocks from floor(G starts(j) / per) + j on, which are enough for its slots, one too many at most;
// so block `unit` finds its interval, and its slots [slot0, slot1), by a search in the offsets alone. Returns the segment, or -1.
__device__ inline int32_t unit_segment(const int64_t* off, int64_t S, int64_t P, int G, int per, uint32_t unit, int64_t& slot0, int64_t& slot1) {
    const int lane = threadIdx.x & 63;
    const auto starts = [&](int64_t j) { return j == 0 ? 0 : clamp64(off[j - 1], 0, P); };
    const auto first = [&](int64_t j) { return starts(j) * G / per + j; };
    int64_t lo = 0, n = S + 2;  // intervals before lo start at or before the block, those from lo + n on do not
    while (n > 0) {
        const int64_t step = (n + 63) >> 6, j = (lane + 1) * step - 1;
        const bool le = j < n && first(lo + j) <= (int64_t)unit;
        const int t = __popcll(__ballot(le));
        lo += t * step;
        n -= t * step;
        n = n < step - 1 ? n : step - 1;
    }
    const int64_t j = lo > 0 ? lo - 1 : 0, nth = (int64_t)unit - first(j);
    slot1 = j <= S ? starts(j + 1) * G : P * G;
    slot0 = nth >= 0 ? starts(j) * G + nth * per : slot1;  // (negative: offsets that decrease)
    slot1 = slot0 + per < slot1 ? slot0 + per : slot1;
    return j >= 1 && j <= S ? (int32_t)(j - 1) : -1;
}

// slot / G (a 64-bit division is some hundred instructions).
__device__ inline int32_t position_of(int64_t slot, int G) {
    return (int32_t)(G == 1 ? slot : slot >> 32 ? slot / G : (int64_t)((uint32_t)slot / (uint32_t)G));
}

// What absent keys and values are fetched from.
__device__ const uint4 g_zeros = {0u, 0u, 0u, 0u};

// Maximum / sum over lanes l and l ^ 32.
__device__ inline float halves_max(float v) {
    const auto r = __builtin_amdgcn_permlane32_swap(f2u(v), f2u(v), false, false);
    return __builtin_fmaxf(u2f(r[0]), u2f(r[1]));
}
__device__ inline float halves_sum(float v) {
    const auto r = __builtin_amdgcn_permlane32_swap(f2u(v), f2u(v), false, false);
    return u2f(r[0]) + u2f(r[1]);
}
// Minimum / maximum over the wave, the same in every lane: rotations within rows of 16 lanes, then across the rows.
template <bool MAX>
__device__ inline int32_t wave_extreme(int32_t v) {
    const auto f = [](int32_t x, int32_t y) { return (MAX ? x > y : x < y) ? x : y; };
    v = f(v, (int32_t)dpp_u32<0x128, 0xf>((uint32_t)v));
    v = f(v, (int32_t)dpp_u32<0x124, 0xf>((uint32_t)v));
    v = f(v, (int32_t)dpp_u32<0x122, 0xf>((uint32_t)v));
    v = f(v, (int32_t)dpp_u32<0x121, 0xf>((uint32_t)v));
    const auto a = __builtin_amdgcn_permlane16_swap((uint32_t)v, (uint32_t)v, false, false);
    v = f((int32_t)a[0], (int32_t)a[1]);
    const auto b = __builtin_amdgcn_permlane32_swap((uint32_t)v, (uint32_t)v, false, false);
    v = f((int32_t)b[0], (int32_t)b[1]);
    return __builtin_amdgcn_readfirstlane(v);
}

// tanh without branches, within 2 ulp: below 0.55 y + y^3 P(y^2), P of degree 4 through (tanh(y) / y - 1) / y^2 at the
// Chebyshev nodes of that range (2^-24 of the value, coefficients and evaluation in fp32); above 1 - 2 / (e^2y + 1).
__device__ inline float tanh_f32(float y) {
    const float z = y * y;
    float p = __builtin_fmaf(-0.00661022774875164f, z, 0.021309388801455498f);
    p = __builtin_fmaf(p, z, -0.05390942841768265f);
    p = __builtin_fmaf(p, z, 0.13333113491535187f);
    p = __builtin_fmaf(p, z, -0.3333333134651184f);
    const float r = __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(2.0f * PMG_LOG2E * __builtin_fabsf(y)));
    return __builtin_fabsf(y) < 0.55f ? __builtin_fmaf(y * z, p, y) : __builtin_copysignf(__builtin_fmaf(-2.0f, r, 1.0f), y);
}

// The thread's number, hidden from the compiler: what is derived from it is formed where it is used, not kept in registers
// through the loop over the keys.
__device__ inline int thread_again() {
    int t = threadIdx.x;
    asm volatile("" : "+v"(t));
    return t;
}

// The kernel's arguments, read anew from here on (kept in scalar registers through the loop over the keys they would be
// spilled to vector registers, lane by lane).
typedef const __attribute__((address_space(4))) AttnArgs ConstArgs;
__device__ inline ConstArgs& args_again() {
    auto p = (uint64_t)__builtin_amdgcn_kernarg_segment_ptr();
    asm volatile("" : "+s"(p));
    return *(ConstArgs*)p;
}

// Zeros in the rows of a wave's lanes that want it.
template <class T>
__device__ inline void zero_rows(ConstArgs& a, bool want, int64_t row) {
    typedef T v4t __attribute__((ext_vector_type(4)));
    const int quads = a.D / 4;
    for (uint64_t todo = __ballot(want); todo; todo &= todo - 1) {
        const int64_t r = __shfl(row, __ffsll((unsigned long long)todo) - 1, 64);
        for (int d = threadIdx.x & 63; d < a.Hq * quads; d += 64) *(v4t*)((T*)a.out + r * a.o_row + d / quads * a.o_head + d % quads * 4) = v4t{};
    }
}

// What a block of the sweep does, beside the blocks that compute: its share of the rows and positions is looked through for rows
// that no position names (they are set to 0: nobody else writes them), and where the offsets of blocks of one segment each fall,
// for slots that no block has (set to 0, or marked as of no segment for the join). Each of the 8 to 32 blocks reads the whole index
// for it, mostly from L2. 76,800 rows in 433 cells: 107.8 us without, 110.6 with it; with a kernel of zeros in front 115.0, and
// small calls 3 us longer for its launch.
constexpr int kSweepBits = 32768;  // the share: a bit each, in LDS
template <class T, int NT>
__device__ inline void attention_sweep(uint32_t* bits, int per_block) {
    ConstArgs& a = args_again();  // (read here: kept from the kernel's start, they cost the other blocks registers)
    const int tid = thread_again();
    const int64_t n = a.Mq > a.Pq ? a.Mq : a.Pq, share = (n + a.sweep - 1) / a.sweep, lo = blockIdx.x * share;
    const auto clear = [&]() {
        __syncthreads();
        for (int i = tid; i < kSweepBits / 32; i += NT) bits[i] = 0;
        __syncthreads();
    };
    const auto set = [&](int64_t i) { atomicOr(&bits[i >> 5], 1u << (i & 31)); };
    const auto is = [&](int64_t i) { return (bits[i >> 5] >> (i & 31) & 1u) != 0; };
    if (a.q_index && a.zero_rest) {
        const int64_t hi = lo + share < a.Mq ? lo + share : a.Mq;
        clear();
#pragma unroll 16
        for (int64_t p = tid; p < a.Pq; p += NT) {
            const int64_t r = a.q_index[p];
            if (r >= lo && r < hi) set(r - lo);
        }
        __syncthreads();
        for (int64_t r0 = lo; r0 < hi; r0 += NT) zero_rows<T>(a, r0 + tid < hi && !is(r0 + tid - lo), r0 + tid);
    }
    if (!a.whole || a.S <= kLook) return;
    bool fall = false;
#pragma unroll 8
    for (int64_t j = tid; j < a.S; j += NT) fall = fall || a.q_off[j] > a.q_off[j + 1];
    if (!__syncthreads_or(fall)) return;
    const int64_t end = (lo + share < a.Pq ? lo + share : a.Pq) * a.G;
    const uint32_t units = a.blocks / (uint32_t)(a.Hk * a.splits);
    for (int64_t s0 = lo * a.G; s0 < end; s0 += kSweepBits) {
        const int64_t s1 = s0 + kSweepBits < end ? s0 + kSweepBits : end;
        clear();
        for (uint32_t u = tid >> 6; u < units; u += NT / 64) {
            int64_t from, to;
            unit_segment(a.q_off, a.S, a.Pq, a.G, per_block, u, from, to);
            for (int64_t i = from + (tid & 63); i < to; i += 64)
                if (i >= s0 && i < s1) set(i - s0);
        }
        __syncthreads();
        for (int64_t i = s0 + tid; i < s1; i += NT) {
            if (is(i - s0)) continue;
            const int64_t pos = i / a.G;
            const int64_t row = a.q_index ? a.q_index[pos] : pos;
            for (int hk = 0; hk < a.Hk; ++hk) {
                const int head = hk * a.G + (int)(i - pos * a.G);
                if (a.splits > 1) a.part_ml[(int64_t)head * a.Pq + pos] = make_float2(-__builtin_inff(), -1.0f);
                else if (a.zero_rest && row >= 0 && row < a.Mq)
                    for (int d = 0; d < a.D; ++d) ((T*)a.out)[row * a.o_row + head * a.o_head + d] = (T)0.0f;
            }
        }
    }
}

// Waves a SIMD the registers are kept to (what the LDS of a block allows, too).
constexpr int waves_of(int DP, int NW, int ES, bool BIAS) {
    if (NW == 1) return DP == 128 ? 1 : 2;
    if (ES == 4) return (DP == 32 ? 4 : DP == 64 ? 3 : 2) - BIAS;
    return DP == 32 ? 4 : DP == 64 ? 4 - BIAS : 2;
}

// Bound by the ordinary instructions: 32 x 32 scores of heads of 64 take 9 matrix and some 100 ordinary ones, with a bias 11
// and 142 (three axes' distances are 48 of them, exponentials 16 that count double), which share a SIMD's issue slots; the
// matrix units are at work a third of the time. Measured (MI355X): 19200 rows, 4 heads of 64, bf16: 500 us (755 TFLOP/s),
// biased 635; 4 frames of 2745 rows, 8 heads, masked: 101 us, where a CU has two or three blocks and so only two
// waves a SIMD; 8 x 1 query on 153,600 rows, 4 key heads of 64, fp16: 28 us, 5.6 TB/s.
//
// Registers: with at most 256 the matrix instructions' results stay in ordinary vector registers, where the softmax
// works on them; only the widest fp32 form of one wave needs more.
// MASK: absent keys are taken out by a product (not with BIAS, whose registers are all in use). FINE: caps by tanh_f32 (a branch
// inside the loop spills 2 to 8 registers), and 16-bit weights in two parts. Rounded to 8 or 11 bits as one, they add as much error
// as the result's own rounding (2.3e-3 of the result's size for 1.7e-3 in bf16, 2.8e-4 for 2.1e-4 in fp16); in two parts they add
// nothing that shows, for 16 % more time (cells, 8 heads of 32 fp16, biased: 115 -> 133 us), 41 % (4 frames of 2745 rows, 8 heads of
// 64 bf16, masked: 108 -> 152), 29 % (19200 rows, 4 heads of 64 bf16, biased: 643 -> 833), 7 % (pooled queries: 34 -> 37): the
// caller's choice, or with a large cap. (Times without the host, calls in one graph.)
template <class T, int DP, int NW, bool BIAS, bool MASK, bool FINE>
__global__ __launch_bounds__(64 * NW, waves_of(DP, NW, sizeof(T), BIAS)) void attention_k(AttnArgs a0) {
    const AttnArgs& a = a0;
    constexpr int ES = sizeof(T), PER = 16 / ES, CPR = DP / PER, NT = 64 * NW;
    constexpr int BK = (NW == 1 || ES == 4 || DP == 128) ? 32 : 64, KB = BK / 32;
    constexpr int NCH = BK * CPR / NT;         // 16-byte chunks of K (and of V) a thread stages
    constexpr int NB = DP / 32;                // 32-column blocks of O
    constexpr bool SEG = NW == 1;               // a block per segment
    constexpr int QC = CPR / 2;                // operand chunks of a query a lane holds
    // (the maximum looked for every time, where the test's registers would be spilled: 300 cells of 256 rows, 8 heads, 91 us
    // for 95; with three waves a SIMD, nothing spilled, 94)
    constexpr bool LOOK = BIAS && DP == 32;
    typedef typename Mat<T>::chunk chunk;
    static_assert(NCH * NT == BK * CPR, "whole chunks");
    __shared__ __attribute__((aligned(16))) char s_k[2][BK * DP * ES];
    __shared__ __attribute__((aligned(16))) char s_v[2][BK * DP * ES];
    constexpr int SB = NT, TPS = SB / BK;  // keys (and tiles) whose numbers are looked up at a time, one a thread
    __shared__ uint32_t s_ok[2][SB / 32];  // which keys there are
    __shared__ uint2 s_row[2][SB];         // their rows of K and V: byte offsets (near), or the row's number
    __shared__ __attribute__((aligned(16))) uint4 s_xy[2 * (BIAS ? SB : 1) + 1];  // coordinates; their parts' weights
    __shared__ __attribute__((aligned(16))) uint2 s_z[2 * (BIAS ? SB : 1) + 1];
    static_assert(TPS >= 2, "a group's numbers are written while its predecessor's first tile is worked on");
    __shared__ int32_t s_r[3][NW];
    __shared__ int s_flag[NW];

    if (blockIdx.x < a.sweep) {
        static_assert(sizeof(s_k) >= kSweepBits / 8, "the share's bits");
        attention_sweep<T, NT>((uint32_t*)s_k, 32 * NW);
        return;
    }
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    // block -> (split, key head, tile or segment): an XCD's blocks are neighbours, on one head's keys
    const uint32_t id = xcd_tile(blockIdx.x - a.sweep, a.blocks);  // (a.sweep is a multiple of 8)
    const uint32_t per_head = a.blocks / (uint32_t)(a.Hk * a.splits);
    const uint32_t unit = id % per_head;
    const int hk = (int)(id / per_head) % a.Hk, split = (int)(id / per_head) / a.Hk;

    const auto kswz = [](int row, int c) { return swizzle<CPR>(row, c); };
    // V: 32-byte units of a row, so that the four rows of a transposing read lie in different banks
    const auto vswz = [](int row, int c) {
        if constexpr (ES == 4) return c;
        return c ^ (DP == 64 ? 4 * ((row >> 1) & 1) : DP == 128 ? 4 * (row & 3) : 0);
    };

    // slots of the block: [slot0, slot1) of all positions' G slots (SEG: of the segment's)
    int64_t slot0, slot1;
    int32_t own = -1;  // the block's segment, with blocks of one segment each
    bool whole = false;
    int32_t seg_lo = 0, seg_hi = 0;  // (positions and rows fit 32 bits)
    if constexpr (SEG) {
        const int64_t p0 = clamp64(a.q_off[unit], 0, a.Pq), p1 = clamp64(a.q_off[unit + 1], 0, a.Pq);
        slot0 = p0 * a.G;
        slot1 = p1 * a.G;
        seg_lo = (int32_t)clamp64(a.k_off[unit], 0, a.Pk);
        seg_hi = (int32_t)clamp64(a.k_off[unit + 1], seg_lo, a.Pk);
    } else if (a.whole && (whole = a.S > kLook || offsets_rise(a.q_off, a.S))) {
        own = unit_segment(a.q_off, a.S, a.Pq, a.G, 32 * NW, unit, slot0, slot1);
    } else {  // (where offsets fall, blocks of one segment each would miss rows; there are enough of them for these tiles. Of more
              // segments than a wave looks through at once the sweep or attention_fill_k sees to what is missed)
        slot0 = (int64_t)unit * (32 * NW);
        slot1 = slot0 + 32 * NW;
        if (slot1 > a.Pq * a.G) slot1 = a.Pq * a.G;
    }

    if (slot0 >= slot1) return;
    for (int64_t base = slot0;;) {
        // ---- the lane's slots
        const int tid = thread_again(), lane = tid & 63, half = lane >> 5;
        int32_t blo = (int32_t)a.Pk, bhi = 0;
        const int64_t wfirst = base + wave * 32;
        const int64_t slot = base + wave * 32 + (lane & 31);
        const bool in = slot < slot1;
        const int32_t pos = in ? position_of(slot, a.G) : -1;
        const int head = hk * a.G + (in ? (int)(slot - (int64_t)pos * a.G) : 0);
        int32_t row = in ? pos : -1, seg = -1, lo = 0, hi = 0;
        if (in && a.q_index) row = a.q_index[pos];  // (looked at below: nothing waits for it here)
        int32_t wlo, whi;  // the wave's keys
        if (SEG || whole) {
            if constexpr (!SEG) {
                seg_lo = own >= 0 ? (int32_t)clamp64(a.k_off[own], 0, a.Pk) : 0;
                seg_hi = own >= 0 ? (int32_t)clamp64(a.k_off[own + 1], seg_lo, a.Pk) : 0;
            }
            if (in) {
                seg = SEG ? (int32_t)unit : own;
                lo = seg_lo;
                hi = seg_hi;
            }
            blo = wlo = seg_lo;
            bhi = seg_hi;
            whi = wfirst < slot1 ? seg_hi : seg_lo;  // (a wave without slots does nothing)
        } else {
            if (wfirst < slot1) seg = wave_segment(a.q_off, a.S, position_of(wfirst, a.G), in ? pos : 0x7ffffffe);
            if (!in) seg = -1;
            if (seg >= 0) {
                lo = (int32_t)clamp64(a.k_off[seg], 0, a.Pk);
                hi = (int32_t)clamp64(a.k_off[seg + 1], lo, a.Pk);
                if (hi > lo) {
                    blo = lo;
                    bhi = hi;
                }
            }
            // the block's keys, and whether some lane sees only a part of them
            blo = wlo = wave_extreme<false>(blo);
            bhi = whi = wave_extreme<true>(bhi);
            if constexpr (NW > 1) {
                __syncthreads();
                if (lane == 0) {
                    s_r[0][wave] = blo;
                    s_r[1][wave] = bhi;
                }
                __syncthreads();
#pragma unroll
                for (int w = 0; w < NW; ++w) {
                    blo = s_r[0][w] < blo ? s_r[0][w] : blo;
                    bhi = s_r[1][w] > bhi ? s_r[1][w] : bhi;
                }
            }
            blo = __builtin_amdgcn_readfirstlane(blo);
            bhi = __builtin_amdgcn_readfirstlane(bhi);
        }
        // keys that every slot of the wave sees (slots of no segment take whatever comes)
        int32_t ilo = 0, ihi = 0x7fffffff;
        if (seg >= 0) {
            ilo = lo;
            ihi = hi;
        }
        ilo = wave_extreme<true>(ilo);
        ihi = wave_extreme<false>(ihi);
        const bool part_seen = seg >= 0 && hi > lo && (lo != blo || hi != bhi);
        if (a.splits > 1 && bhi > blo) {
            const int64_t each = (((int64_t)bhi - blo + a.splits - 1) / a.splits + BK - 1) / BK * BK;
            blo = (int32_t)(blo + split * each < bhi ? blo + split * each : bhi);
            bhi = (int32_t)(blo + each < bhi ? blo + each : bhi);
        }

        // the first keys' numbers, on their way with the queries' own
        const auto number = [](const int32_t* k_index, int tid, int32_t g, int32_t from, int32_t to) -> int32_t {
            if (g * (int64_t)SB >= to - from || tid >= to - from - g * SB) return -1;
            const int32_t p = from + g * SB + tid;
            return k_index ? k_index[p] : p;  // (looked at in about(): nothing waits for it here)
        };
        const int32_t first0 = number(a.k_index, tid, 0, blo, bhi), first1 = number(a.k_index, tid, 1, blo, bhi);

        // ---- the queries, and their coordinates' operands
        row = row >= 0 && row < a.Mq ? row : -1;
        chunk qf[QC];
        v8bf qc[3];
        float sl[3];
        const T* qp = (const T*)a.q + (int64_t)(row >= 0 ? row : 0) * a.q_row + head * a.q_head;
#pragma unroll
        for (int c = 0; c < QC; ++c) {
            const int cc = 2 * c + half;
            qf[c] = chunk{};
            if (row >= 0 && cc * PER < a.D) qf[c] = *(const chunk*)(qp + cc * PER);
        }
        if constexpr (BIAS) {
            // The difference of two coordinates as a product of 16 terms: the key's parts (8 bits each, exact in
            // bf16) times their weights 1, 2^8, 2^16, 2^24 in the lower half's lanes, the weights times the query's
            // negated parts in the upper half's; exact up to 2^23. The key's operand holds two axes at a time, the
            // query's is 0 for the other one.
#pragma unroll
            for (int x = 0; x < 3; ++x) {
                const int32_t c = row >= 0 ? a.q_coords[(int64_t)row * 4 + 1 + x] : 0;
                sl[x] = -a.slopes[head * 3 + x] * PMG_LOG2E;
                const float p[4] = {(float)(c & 255), (float)((c >> 8) & 255), (float)((c >> 16) & 255), (float)(c >> 24)};
                const float w[4] = {1.0f, 256.0f, 65536.0f, 16777216.0f};
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    qc[x][i] = (__bf16)(x == 1 ? 0.0f : half ? -p[i] : w[i]);
                    qc[x][4 + i] = (__bf16)(x != 1 ? 0.0f : half ? -p[i] : w[i]);
                }
            }
        }
        if constexpr (BIAS) {
            if (tid == 0) {
                s_xy[2 * SB] = make_uint4(0x43803f80u, 0x4b804780u, 0x43803f80u, 0x4b804780u);
                s_z[2 * SB] = make_uint2(0x43803f80u, 0x4b804780u);
            }
        }

        int32_t only = -1;  // >= 0: the one segment this turn is for
        for (;;) {
            const int tid = thread_again(), lane = tid & 63, half = lane >> 5;
            ConstArgs& a = args_again();
            int32_t klo = blo, khi = bhi;
            if (only >= 0) {
                const int32_t l0 = (int32_t)clamp64(a.k_off[only], 0, a.Pk), h0 = (int32_t)clamp64(a.k_off[only + 1], l0, a.Pk);
                klo = l0 > blo ? l0 : blo;
                khi = h0 < bhi ? h0 : bhi;
            }
            const int32_t nt = khi > klo ? (khi - klo + (BK - 1)) / BK : 0;

            v16f O[NB];
            float m, l, grow;
            bool look;  // the maximum is looked for: some slot of the wave has none yet, or a weight grew too large
            const float k2 = a.cap2 != 0.0f ? 1.0f : a.scale2;
            m = 0.0f;
            grow = -__builtin_inff();
            l = 0.0f;
            look = true;
#pragma unroll
            for (int b = 0; b < NB; ++b) O[b] = v16f{};

            // ---- the keys' numbers, mask and coordinates, by groups of SB
            int32_t mi = -1;  // the thread's row in the group whose mask and coordinates come next
            int4 mc = make_int4(0, 0, 0, 0);
            uint8_t mm = 1;
            const auto about = [&]() {  // of row mi
                mi = mi < (int32_t)a.Mk ? mi : -1;
                const int64_t r = mi >= 0 ? mi : 0;
                if (a.k_mask) mm = a.k_mask[r];
                if constexpr (BIAS) mc = *(const int4*)(a.k_coords + r * 4);
            };
            const auto note = [&](int b) {
                const bool on = mi >= 0 && mm != 0;
                const uint64_t w = __ballot(on);
                if (lane < 2) s_ok[b][2 * wave + lane] = (uint32_t)(w >> (32 * lane));
                // (absent: behind the buffer's end, whichever chunk is added; or -1)
                s_row[b][tid] = !on ? make_uint2(0xffff0000u, 0xffff0000u)
                                    : make_uint2((uint32_t)mi * (a.near ? (uint32_t)a.k_row * ES : 1u), (uint32_t)mi * (a.near ? (uint32_t)a.v_row * ES : 1u));
            };
            const auto note_where = [&](int b) {
                if constexpr (BIAS) {
                    const auto b16 = [](int v) { return f2u((float)v) >> 16; };  // (exact: 8 bits)
                    const auto p01 = [&](int v) { return b16(v & 255) | (b16((v >> 8) & 255) << 16); };
                    const auto p23 = [&](int v) { return b16((v >> 16) & 255) | (b16(v >> 24) << 16); };
                    s_xy[b * SB + tid] = make_uint4(p01(mc.y), p23(mc.y), p01(mc.z), p23(mc.z));
                    s_z[b * SB + tid] = make_uint2(p01(mc.w), p23(mc.w));
                }
            };
            // Tile t into buffer b. Near: a load behind the buffer's end is a row of zeros. Otherwise 64-bit addresses (rows
            // are less than 2^31 bytes apart); absent rows and chunks behind the head's width come from a line of zeros.
            const bool near = a.near;
            const v4i kr = buffer_of((const T*)a.k + hk * a.k_head, (uint32_t)((a.Mk - 1) * a.k_row + DP) * ES);
            const v4i vr = buffer_of((const T*)a.v + hk * a.v_head, (uint32_t)((a.Mk - 1) * a.v_row + DP) * ES);
            const uint32_t lk = lds_address(s_k[0]) + wave * 1024, lv = lds_address(s_v[0]) + wave * 1024;
            const auto fetch = [&](int b, uint32_t t) {
                const uint2* rows = &s_row[(t / TPS) & 1][(t % TPS) * BK];
                if (near) {
#pragma unroll
                    for (int i = 0; i < NCH; ++i) {
                        const int e = (i * NW + wave) * 64 + lane, r = e / CPR, p = e % CPR;
                        const uint2 row = rows[r];
                        const uint32_t to = b * (BK * DP * ES) + i * NW * 1024;
                        buffer_to_lds(kr, row.x + kswz(r, p) * 16, 0, lk + to);
                        buffer_to_lds(vr, row.y + vswz(r, p) * 16, 0, lv + to);
                    }
                } else {
                    const int lane = thread_again() & 63;  // (its addresses are not kept in registers)
#pragma unroll
                    for (int i = 0; i < NCH; ++i) {
                        const int e = (i * NW + wave) * 64 + lane, r = e / CPR, p = e % CPR;
                        const int ck = kswz(r, p) * 16, cv = vswz(r, p) * 16;
                        const uint2 row = rows[r];
                        const uint32_t to = b * (BK * DP * ES) + i * NW * 1024;
                        const bool on = (int32_t)row.x >= 0;
                        const char* kp = (const char*)((const T*)a.k + hk * a.k_head) + (uint64_t)row.x * ((uint32_t)a.k_row * ES) + ck;
                        const char* vp = (const char*)((const T*)a.v + hk * a.v_head) + (uint64_t)row.y * ((uint32_t)a.v_row * ES) + cv;
                        load_to_lds(on && ck < a.D * ES ? kp : (const char*)&g_zeros, lk + to);
                        load_to_lds(on && cv < a.D * ES ? vp : (const char*)&g_zeros, lv + to);
                    }
                }
            };
            if (nt > 0) {
                mi = only < 0 ? first0 : number(a.k_index, tid, 0, klo, khi);
                about();
                note(0);
                __syncthreads();
                fetch(0, 0);
                note_where(0);
                mi = only < 0 ? first1 : number(a.k_index, tid, 1, klo, khi);
                loads_landed<0>();
            }
            // Keys can be taken out by a product with -inf where no query is infinite or NaN (an absent key's zeros times
            // that) and no cap makes it finite.
            uint32_t minus = 0xffffffffu;
            if constexpr (MASK) {
                bool odd = a.cap2 != 0.0f;
                v16f z = {};
#pragma unroll
                for (int c = 0; c < QC; ++c) z = Mat<T>::mma32(chunk{}, qf[c], z);
                odd = odd || z[0] != 0.0f;
                if (__any(odd)) minus = 0u;
            }
            // (vmcnt(0) as the compiler counts: else it waits for the queries, and with them for the next tile, at their
            // every use in the loop)
            __builtin_amdgcn_s_waitcnt(0x0f70);
            __syncthreads();

            for (int32_t it = 0; it < nt; ++it) {
                const int cur = it & 1;
                const bool more = it + 1 < nt;
                const int slot = ((uint32_t)it / TPS) & 1, k0 = (int)((uint32_t)it % TPS) * BK;  // where its keys' numbers are
                const bool ahead = k0 == 0 && it + TPS < nt;  // look up the next group
                int32_t mn = -1;
                if (more) fetch(cur ^ 1, it + 1);
                if (ahead) {
                    about();
                    mn = number(a.k_index, tid, (uint32_t)it / TPS + 2, klo, khi);
                }
                // 32 keys at a time: more waves on a SIMD are worth more than longer runs of one (a single wave issues
                // an ordinary instruction every 5 cycles, two or more together one every 2.5, measured)
#pragma unroll 1
                for (int b = 0; b < KB; ++b) {
                    const int32_t p0 = klo + it * BK + 32 * b;
                    if (p0 >= whi || wlo - p0 >= 32) continue;
                    const char* sk = s_k[cur] + 32 * b * DP * ES;
                    const char* sv = s_v[cur] + 32 * b * DP * ES;
                    const int kn = slot * SB + k0 + 32 * b;  // its keys' numbers
                    const uint32_t ok = __builtin_amdgcn_readfirstlane((&s_ok[0][0])[kn / 32]);
                    const bool inside = p0 >= ilo && ihi - p0 >= 32;  // every slot's keys
                    // ---- scores
                    v16f s;
                    const auto scores = [&]() {
                        s = v16f{};
                        // keys that are absent for every slot: -inf from one more product, of (0 or -inf) x 1. The select
                        // below costs two instructions a score
                        if constexpr (MASK) {
                            const uint32_t off = ((half ? 0u : ~ok & minus) >> (lane & 31)) & 1u;
                            typedef short v4s __attribute__((ext_vector_type(4)));
                            const v4s kx = {(short)(off * 0xff80u), 0, 0, 0}, qx = {(short)(half ? 0 : 0x3f80), 0, 0, 0};
                            s = __builtin_amdgcn_mfma_f32_32x32x8bf16_1k(kx, qx, s, 0, 0, 0);
                        }
                        constexpr int QG = QC < 4 ? QC : 4;  // operand chunks at a time
#pragma unroll
                        for (int c0 = 0; c0 < QC; c0 += QG) {
                            chunk kf[QG];
                            const int r = lane & 31;
#pragma unroll
                            for (int c = 0; c < QG; ++c) kf[c] = *(const chunk*)(sk + r * DP * ES + 16 * kswz(r, 2 * (c0 + c) + half));
#pragma unroll
                            for (int c = 0; c < QG; ++c)  // (fp32: 256 cycles a chunk, not spent behind the head's width)
                                if (ES == 2 || 2 * (c0 + c) * PER < a.D) s = Mat<T>::mma32(kf[c], qf[c0 + c], s);
                        }
                        // less the maximum so far, in powers of two
                        if (a.cap2 != 0.0f) {
#pragma unroll
                            for (int e = 0; e < 16; ++e) {
                                if constexpr (FINE) s[e] = a.cap2 * tanh_f32(s[e] * a.cap_arg);
                                else s[e] = __builtin_fmaf(-2.0f * a.cap2, __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(s[e] * a.cap_arg)), a.cap2);
                            }
                        }
                        if constexpr (BIAS) {
                            const int kc = half ? 2 * SB : kn + (lane & 31);
                            const uint2 z = s_z[kc];
                            const v8bf kxy = __builtin_bit_cast(v8bf, s_xy[kc]), kz = __builtin_bit_cast(v8bf, make_uint4(z.x, z.y, 0u, 0u));
                            v16f u;
#pragma unroll
                            for (int x = 0; x < 3; ++x) {
                                const v16f d = Mat<__bf16>::mma32(x < 2 ? kxy : kz, qc[x], v16f{});
#pragma unroll
                                for (int e = 0; e < 16; ++e) u[e] = __builtin_fmaf(__builtin_fabsf(d[e]), sl[x], x == 0 ? -m : u[e]);
                                __builtin_amdgcn_sched_barrier(0);  // (one difference's registers at a time)
                            }
#pragma unroll
                            for (int e = 0; e < 16; ++e) s[e] = __builtin_fmaf(s[e], k2, u[e]);
                        } else {
#pragma unroll
                            for (int e = 0; e < 16; ++e) s[e] = __builtin_fmaf(s[e], k2, -m);
                        }
                        // ---- the keys that count for the lane's slot
                        if (!inside || (ok | (MASK ? minus : 0u)) != 0xffffffffu) {
                            const int x = lo - p0, y = hi - p0;
                            uint32_t w = y >= 32 ? 0xffffffffu : y <= 0 ? 0u : (1u << y) - 1u;
                            w &= x <= 0 ? 0xffffffffu : x >= 32 ? 0u : ~((1u << x) - 1u);
                            w = (w & ok) >> (4 * half);
#pragma unroll
                            for (int e = 0; e < 16; ++e) {
                                const uint32_t on = (uint32_t)((int32_t)(w << (31 - ((e & 3) + 8 * (e >> 2)))) >> 31);
                                s[e] = u2f((on & f2u(s[e])) | (~on & 0xff800000u));
                            }
                        }
                    };
                    // ---- weights, in units that put the running maximum at 2^kTop. It is set by the first keys, then moved only when
                    // a weight grows beyond 2^kMost (up to 2^(kMost + 4) nothing is lost). That shows in the sum of a lane's 16
                    // weights: only then the scores are formed again and their maximum looked for. fp16, whose numbers end
                    // at 2^-24, has the maximum at 2^7: a weight is off by at most 2^-32 of it, a million small ones by 2^-12 (at 1
                    // they would lose 2^-25 each: 150,000 keys 0.4 % of the result).
                    constexpr bool HALF = std::is_same<T, _Float16>::value;
                    constexpr float kTop = HALF ? 7.0f : 0.0f, kMost = HALF ? 11.0f : 8.0f, kSum = HALF ? 32768.0f : 4096.0f;
                    float sum;
                    const auto weights = [&]() {
                        float part[4];
#pragma unroll
                        for (int e = 0; e < 16; ++e) {
                            s[e] = __builtin_amdgcn_exp2f(s[e]);
                            part[e & 3] = e < 4 ? s[e] : part[e & 3] + s[e];
                        }
                        sum = (part[0] + part[1]) + (part[2] + part[3]);
                    };
                    if (!LOOK && !look) {
                        scores();
                        weights();
                        look = __any(sum > kSum);
                    }
                    if (LOOK || look) {
                        scores();
                        float mx = s[0];
#pragma unroll
                        for (int e = 1; e < 16; ++e) mx = __builtin_fmaxf(mx, s[e]);
                        mx = halves_max(mx);
                        if (__any(mx > grow)) {
                            const bool any = mx > -__builtin_inff();  // (a slot without a key so far keeps m = 0)
                            const float up = any && (mx > kTop || grow < 0.0f) ? mx - kTop : 0.0f;
                            // (nothing to scale before the first key, whose score may be far below -2^7)
                            const float al = grow < 0.0f ? 1.0f : __builtin_amdgcn_exp2f(-up);
                            grow = any ? kMost : grow;
                            m = m + up;
                            l = l * al;
#pragma unroll
                            for (int e = 0; e < 16; ++e) s[e] = s[e] - up;
#pragma unroll
                            for (int n = 0; n < NB; ++n)
#pragma unroll
                                for (int e = 0; e < 16; ++e) O[n][e] = O[n][e] * al;
                        }
                        weights();
                        look = __any(grow < 0.0f);
                    }
                    l = l + sum;
                    typedef short v4s __attribute__((ext_vector_type(4)));
                    typedef short v8s __attribute__((ext_vector_type(8)));
                    typedef __attribute__((address_space(3))) v4s* lds4;
                    const auto values = [&](int f, int n) {  // V^T: columns 32 n on, keys 16 f on
                        const int i = lane & 15, c = 4 * n + 2 * ((lane >> 4) & 1) + ((i & 3) >> 1);
                        const int r = 16 * f + 4 * half + (i >> 2);
                        const v4s v0 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4)(sv + r * DP * 2 + 16 * vswz(r, c) + (i & 1) * 8));
                        const v4s v1 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4)(sv + (r + 8) * DP * 2 + 16 * vswz(r + 8, c) + (i & 1) * 8));
                        return __builtin_bit_cast(chunk, __builtin_shufflevector(v0, v1, 0, 1, 2, 3, 4, 5, 6, 7));
                    };
                    // ---- O^T += V^T P^T
                    // (two parts: the first one less than the weight by more than its rounding, so that the second one is
                    // positive and an infinite value stays infinite)
                    constexpr float kLess = 1.0f - (HALF ? 1.0f / 1024 : 1.0f / 128);
                    if constexpr (ES == 4) {
#pragma unroll
                        for (int e = 0; e < 16; ++e) {
                            const int r = (e & 3) + 8 * (e >> 2) + 4 * half;
#pragma unroll
                            for (int n = 0; n < NB; ++n) {
                                const float vf = *(const float*)(sv + r * DP * 4 + (32 * n + (lane & 31)) * 4);
                                O[n] = __builtin_amdgcn_mfma_f32_32x32x2f32(vf, s[e], O[n], 0, 0, 0);
                            }
                        }
                    } else {
#pragma unroll
                        for (int f = 0; f < 2; ++f) {
                            chunk pf;
#pragma unroll
                            for (int i = 0; i < 8; ++i) pf[i] = (T)(FINE ? s[8 * f + i] * kLess : s[8 * f + i]);
                            if constexpr (FINE) {  // what that left, in a product of its own
                                chunk pr;
#pragma unroll
                                for (int i = 0; i < 8; ++i) pr[i] = (T)(s[8 * f + i] - (float)pf[i]);
#pragma unroll
                                for (int n = 0; n < NB; ++n) O[n] = Mat<T>::mma32(values(f, n), pr, O[n]);
                            }
#pragma unroll
                            for (int n = 0; n < NB; ++n) O[n] = Mat<T>::mma32(values(f, n), pf, O[n]);
                        }
                    }
                }
                if (ahead) {
                    note(slot ^ 1);
                    note_where(slot ^ 1);
                    mi = mn;
                }
                loads_landed<0>();
                __syncthreads();
            }

            {
            const int tid = thread_again(), lane = tid & 63, half = lane >> 5;
            ConstArgs& a = args_again();
            // ---- values of other segments that are not finite: once more, segment by segment
            if (only < 0) {
                float bad = 0.0f;
#pragma unroll
                for (int b = 0; b < NB; ++b)
#pragma unroll
                    for (int e = 0; e < 16; ++e) bad = __builtin_fmaf(O[b][e], 0.0f, bad);
                // (a wave that sees part of the keys: its own lanes; each wave's keys are the block's)
                bool again = __any(part_seen) && __any(bad != 0.0f);
                if constexpr (NW > 1) {
                    if (lane == 0) s_flag[wave] = again;
                    __syncthreads();
                    again = false;
#pragma unroll
                    for (int w = 0; w < NW; ++w) again = again || s_flag[w];
                }
                if (again) {
                    only = -2;  // the first segment is looked for below
                }
            }
            // ---- results (before a second turn: those of no segment only)
            const float lt = halves_sum(l);
            const bool mine = only == -2 ? seg < 0 : only < 0 || seg == only;
            if (a.splits > 1) {
                const int64_t o = ((int64_t)split * a.Hq + head) * a.Pq + pos;
                if (mine && pos >= 0 && half == 0)
                    a.part_ml[o] = make_float2(grow > 0.0f ? m : -__builtin_inff(), seg >= 0 ? lt : -1.0f);
                if (mine && seg >= 0) {
#pragma unroll
                    for (int b = 0; b < NB; ++b)
#pragma unroll
                        for (int g = 0; g < 4; ++g) {
                            const int d = 32 * b + 8 * g + 4 * half;
                            if (d < a.D) *(float4*)(a.part_o + o * a.D + d) = make_float4(O[b][4 * g], O[b][4 * g + 1], O[b][4 * g + 2], O[b][4 * g + 3]);
                        }
                }
            } else if (mine && row >= 0 && (seg >= 0 || a.zero_rest)) {
                const bool none = lt == 0.0f || seg < 0;  // no key left
                const float inv = 1.0f / lt;
                T* op = (T*)a.out + (int64_t)row * a.o_row + head * a.o_head;
#pragma unroll
                for (int b = 0; b < NB; ++b)
#pragma unroll
                    for (int g = 0; g < 4; ++g) {
                        const int d = 32 * b + 8 * g + 4 * half;
                        typedef T v4t __attribute__((ext_vector_type(4)));
                        v4t v;
#pragma unroll
                        for (int i = 0; i < 4; ++i) v[i] = (T)(none ? 0.0f : O[b][4 * g + i] * inv);
                        if (d < a.D) *(v4t*)(op + d) = v;
                    }
            }
            if (only == -1) break;
            // the next segment of the block
            int32_t next = 0x7fffffff;
            if (seg >= 0 && seg > only && seg < next) next = seg;
            next = wave_extreme<false>(next);
            if constexpr (NW > 1) {
                __syncthreads();
                if (lane == 0) s_r[2][wave] = next;
                __syncthreads();
#pragma unroll
                for (int w = 0; w < NW; ++w) next = s_r[2][w] < next ? s_r[2][w] : next;
            }
            if (next == 0x7fffffff) break;
            only = __builtin_amdgcn_readfirstlane(next);
            }
        }
        if constexpr (!SEG) break;
        base += 32 * NW;
        if (base >= slot1) break;
    }
}

// Joins the splits of each (position, head): groups of CL lanes, 4 columns a lane. WIDE (many splits): a wave a position, each
// group on every (64 / CL)-th split, the groups' sums added in order at the end. Otherwise a group a position, its splits
// in order. One pass with the running maximum, the loads of U splits under way at once with the row's number: such a small
// kernel is a chain of loads (8 positions of 16 heads of 64, 64 splits: 5 us; 19200 rows of 4 heads of 64, 5 splits: 18 us, 6 TB/s).
template <class T, int CL, bool WIDE>
__global__ __launch_bounds__(256) void attention_join_k(AttnArgs a) {
    constexpr int G = 64 / CL, PER = WIDE ? 4 : 4 * G;  // positions a block
    constexpr int U = WIDE ? 8 : 4, EACH = WIDE ? G : 1;
    const int lane = threadIdx.x & 63, g = lane / CL, d = 4 * (lane % CL), head = blockIdx.y;
    const int64_t first = (int64_t)blockIdx.x * PER + (WIDE ? threadIdx.x >> 6 : (threadIdx.x >> 6) * G);  // the wave's
    const int64_t pos = WIDE ? first : first + g;
    if (first >= a.Pq) return;
    const bool there = pos < a.Pq;
    const int64_t step = (int64_t)a.Hq * a.Pq, at = (int64_t)head * a.Pq + (there ? pos : first);
    int32_t r = there ? a.q_index ? a.q_index[pos] : (int32_t)pos : -1;
    const float y0 = a.part_ml[at].y;
    float m = -__builtin_inff(), l = 0.0f;
    v4f acc = {0.0f, 0.0f, 0.0f, 0.0f};
    for (int s0 = WIDE ? g : 0; s0 < a.splits; s0 += U * EACH) {
        float2 ml[U];
        v4f po[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int64_t s = at + (s0 + u * EACH < a.splits ? s0 + u * EACH : s0) * step;
            ml[u] = a.part_ml[s];
            po[u] = *(const v4f*)(a.part_o + s * a.D + (d < a.D ? d : 0));
            if (s0 + u * EACH >= a.splits) ml[u] = make_float2(-__builtin_inff(), 0.0f);
        }
        float mx = m;
#pragma unroll
        for (int u = 0; u < U; ++u) mx = __builtin_fmaxf(mx, ml[u].x);
        const float ms = mx == -__builtin_inff() ? 0.0f : mx, was = __builtin_amdgcn_exp2f(m - ms);
        m = mx;
        l = l * was;
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[i] = acc[i] * was;
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const float w = __builtin_amdgcn_exp2f(ml[u].x - ms);
            if (ml[u].y != 0.0f) {  // (a part without keys counts for nothing)
                l = __builtin_fmaf(ml[u].y, w, l);
#pragma unroll
                for (int i = 0; i < 4; ++i) acc[i] = __builtin_fmaf(po[u][i], w, acc[i]);
            }
        }
    }
    if constexpr (WIDE) {
        float mx = m;
#pragma unroll
        for (int o = CL; o < 64; o <<= 1) mx = __builtin_fmaxf(mx, __shfl_xor(mx, o, 64));
        const float w = m == -__builtin_inff() ? 0.0f : __builtin_amdgcn_exp2f(m - mx);
        l = l * w;
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[i] = acc[i] * w;
#pragma unroll
        for (int o = CL; o < 64; o <<= 1) {
            l = l + __shfl_xor(l, o, 64);
#pragma unroll
            for (int i = 0; i < 4; ++i) acc[i] = acc[i] + __shfl_xor(acc[i], o, 64);
        }
    }
    // (blocks by segment write nothing for positions of no segment)
    bool in = y0 >= 0.0f || y0 != y0;
    if (a.seg) in = in_segment(a.q_off, wave_segment(a.q_off, a.S, (int32_t)first, there ? (int32_t)pos : (int32_t)first), pos);
    if (r < 0 || r >= a.Mq || (!in && !a.zero_rest) || (WIDE && g != 0) || d >= a.D) return;
    typedef T v4t __attribute__((ext_vector_type(4)));
    const float inv = 1.0f / l;
    v4t v;
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = (T)(!in || l == 0.0f ? 0.0f : acc[i] * inv);
    *(v4t*)((T*)a.out + (int64_t)r * a.o_row + head * a.o_head + d) = v;
}

template <class T, int CL>
static int launch_join(const AttnArgs& a, hipStream_t s) {
    const bool wide = a.splits >= 16;
    const int per = wide ? 4 : 4 * (64 / CL);
    const dim3 grid((unsigned)((a.Pq + per - 1) / per), (unsigned)a.Hq);
    if (wide) hipLaunchKernelGGL((attention_join_k<T, CL, true>), grid, dim3(256), 0, s, a);
    else hipLaunchKernelGGL((attention_join_k<T, CL, false>), grid, dim3(256), 0, s, a);
    return check_launch("attention_join_k");
}

// In front of the others, where a sweep would take too long or there is none: zeros in a result that the tables may not name whole,
// and no segment in the parts' (m, l) where blocks of one segment each may miss some.
template <class T>
__global__ __launch_bounds__(256) void attention_fill_k(AttnArgs a, int64_t rows, int64_t chunks, int64_t parts) {
    const int64_t first = (int64_t)blockIdx.x * 256 + threadIdx.x, step = (int64_t)gridDim.x * 256;
    for (int64_t i = first; i < chunks; i += step) ((uint4*)a.out)[i] = make_uint4(0u, 0u, 0u, 0u);  // (a contiguous result)
    typedef T v4t __attribute__((ext_vector_type(4)));
    const int per = a.Hq * (a.D / 4);
    for (int64_t r = first >> 6; r < rows; r += step >> 6)
        for (int d = threadIdx.x & 63; d < per; d += 64) *(v4t*)((T*)a.out + r * a.o_row + d / (a.D / 4) * a.o_head + d % (a.D / 4) * 4) = v4t{};
    for (int64_t i = first; i < parts; i += step) a.part_ml[i] = make_float2(-__builtin_inff(), -1.0f);
}

template <class T>
static int launch_fill(AttnArgs& a, hipStream_t s) {
    const int64_t chunks = a.Mq * a.Hq * a.D * (int64_t)sizeof(T) / 16;  // (D is a multiple of 8)
    const bool split = a.splits > 1, unnamed = a.zero_rest && a.q_index, missed = a.whole && a.S > kLook && (a.zero_rest || split);
    // The sweep's blocks read the index as often as there are shares: up to a million rows that is 134 MB.
    const int64_t n = a.Mq > a.Pq ? a.Mq : a.Pq, shares = (n + 2047) / 2048;
    const bool sweep = (unnamed || missed) && a.Pq > 0 && n <= 32 * (int64_t)kSweepBits;
    if (sweep) a.sweep = (uint32_t)(shares < 32 ? (shares + 7) / 8 * 8 : 32);
    const bool fill = a.zero_rest && (a.Pq < a.Mq && !a.q_index || a.seg && !split || !sweep && (unnamed || missed));
    const bool straight = a.o_head == a.D && a.o_row == (int64_t)a.Hq * a.D && aligned16(a.out);
    const int64_t wide = fill && straight ? chunks : 0, rows = fill && !straight ? a.Mq : 0, parts = split && missed && !sweep ? a.splits * a.Pq * a.Hq : 0;
    const int64_t most = wide > rows * 64 ? wide : rows * 64, blocks = ((most > parts ? most : parts) + 1023) / 1024;
    if (blocks == 0) return PMG_OK;
    hipLaunchKernelGGL((attention_fill_k<T>), dim3((unsigned)(blocks < 8192 ? blocks : 8192)), dim3(256), 0, s, a, rows, wide, parts);
    return check_launch("attention_fill_k");
}

template <class T, int DP, int NW>
static int launch_attention_w(AttnArgs& a, hipStream_t s) {
    const int64_t units = NW == 1 ? a.S : a.whole ? a.Pq * a.G / (32 * NW) + a.S + 2 : (a.Pq * a.G + 32 * NW - 1) / (32 * NW);
    const int64_t blocks = units * a.Hk * a.splits;
    PMG_REQUIRE(blocks + a.sweep <= grid_blocks(64 * NW), "too many slots or segments for one launch");
    a.blocks = (uint32_t)blocks;
    const auto launch = [&](auto kernel) { hipLaunchKernelGGL(kernel, dim3(a.blocks + a.sweep), dim3(64 * NW), 0, s, a); };
    constexpr bool F32 = sizeof(T) == 4;
    if (!F32 && a.fine) {
        if (a.slopes) launch(attention_k<T, DP, NW, true, false, true>);
        else launch(attention_k<T, DP, NW, false, false, true>);
    } else if (a.slopes) launch(attention_k<T, DP, NW, true, false, F32>);
    else if (a.k_mask) launch(attention_k<T, DP, NW, false, true, F32>);
    else launch(attention_k<T, DP, NW, false, false, F32>);
    return check_launch("attention_k");
}

template <class T, int DP>
static int launch_attention_d(AttnArgs& a, hipStream_t s) {
    return a.seg ? launch_attention_w<T, DP, 1>(a, s) : launch_attention_w<T, DP, 4>(a, s);
}

template <class T>
int launch_attention_t(AttnArgs& a, hipStream_t s) {
    if (int e = launch_fill<T>(a, s)) return e;
    if (a.Pq == 0) return PMG_OK;
    if (int e = a.D <= 32 ? launch_attention_d<T, 32>(a, s) : a.D <= 64 ? launch_attention_d<T, 64>(a, s) : launch_attention_d<T, 128>(a, s)) return e;
    if (a.splits > 1) return a.D <= 64 ? launch_join<T, 16>(a, s) : launch_join<T, 32>(a, s);
    return PMG_OK;
}

int launch_attention_f16(AttnArgs& a, hipStream_t s);
int launch_attention_bf16(AttnArgs& a, hipStream_t s);
int launch_attention_f32(AttnArgs& a, hipStream_t s);

}  // namespace pmg
