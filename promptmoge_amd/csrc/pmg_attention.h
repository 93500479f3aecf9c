// Attention inside segments of rows (frames, pool cells): the kernel, instantiated per element type.
//
//   o[i] = sum_j p_ij v[j],  p_i = softmax over the keys j of i's segment that k_mask leaves of
//          cap(scale q_i . k_j) - sum over axes of slope[head][axis] |c_i - c_j|[axis],   cap(x) = cap tanh(x / cap)
//
// One pass over the keys with the running maximum m and sum l of the softmax (fp32, in powers of two). A wave owns 32
// slots (QT times): a slot is a query position and one of the G query heads that share a key head. The products are
// formed transposed, S^T = K Q^T and O^T = V^T P^T, so that a lane holds 16 scores of ONE slot: maximum and sum are
// taken in the lane and once across the two halves of the wave, and the scores, rounded to the inputs' type (the
// weights of the second product; l sums the unrounded ones), are that product's operand as they lie. V^T comes from
// row-major V by the transposing LDS read (fp32: by plain reads). K and V tiles go from memory straight to LDS, one tile
// ahead into the other of two buffers: each lane names the 16 bytes it fetches, so rows are gathered by index, the
// banks' swizzle is made by the choice of chunk, and an absent row (masked, behind its segment, a bad index) is fetched
// from a line of zeros. The rows' numbers, mask and coordinates run two and three tiles ahead.
//
// Queries are taken in order of position, 32 NW QT / G positions a block, whatever segments they fall in: the block
// walks over the keys of all its segments, and each lane counts the keys of its own. No work list is needed, and small
// cells share a wave. A weight of 0 times a value that is infinite or NaN is NaN: where outputs of a block over
// several segments are not finite, the block goes over its segments one by one. (SEG: a block per segment, for few
// queries on many keys.) The keys of a block can be split over gridDim blocks, whose (m, l, O) a second kernel joins.
#pragma once
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
    float cap2, cap_arg;  // cap log2(e); the factor of tanh's argument (0 cap: none)
    int seg, splits, zero_rest;
    uint32_t blocks;
    float* part_o;  // [splits][Pq][Hq][D]
    float2* part_ml;
};

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

// The segment (as above) of position p of each lane, all lanes of a wave taking part; first: a lower bound of the p. A
// search with 64 probes a round for `first`, then among the 64 offsets that follow.
__device__ inline int32_t wave_segment(const int64_t* off, int64_t S, int32_t first, int32_t p) {
    const int lane = threadIdx.x & 63;
    int64_t lo = 0, n = S + 1;  // entries before lo are <= first, those from lo + n on are not
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

// What absent keys and values are fetched from.
__device__ const uint4 g_zeros = {0u, 0u, 0u, 0u};

// The other half's value (lane l <-> l ^ 32).
__device__ inline float other_half(float v) {
    const uint32_t u = f2u(v);
    const auto r = __builtin_amdgcn_permlane32_swap(u, u, false, false);
    return u2f((threadIdx.x & 32) ? r[0] : r[1]);
}

// The kernel's arguments, read anew from here on (kept in scalar registers through the loop over the keys they would be
// spilled to vector registers, lane by lane).
__device__ inline const AttnArgs& args_again() {
    auto p = (uint64_t)__builtin_amdgcn_kernarg_segment_ptr();
    asm volatile("" : "+s"(p));
    return *(const AttnArgs*)p;
}

// Registers: with at most 256 the matrix instructions' results stay in ordinary vector registers, where the softmax
// works on them; only the widest fp32 form of one wave needs more.
template <class T, int DP, int NW, int QT, bool BIAS>
__global__ __launch_bounds__(64 * NW, sizeof(T) == 4 && DP == 128 && NW == 1 ? 1 : 2) void attention_k(AttnArgs a0) {
    const AttnArgs& a = a0;
    constexpr int ES = sizeof(T), PER = 16 / ES, CPR = DP / PER, NT = 64 * NW;
    constexpr int BK = (NW == 1 || ES == 4) ? 32 : 64, KB = BK / 32;
    constexpr int NCH = BK * CPR / NT;         // 16-byte chunks of K (and of V) a thread stages
    constexpr int NB = DP / 32;                // 32-column blocks of O
    constexpr int QC = CPR / 2;                // operand chunks of a query a lane holds
    typedef typename Mat<T>::chunk chunk;
    static_assert(NCH * NT == BK * CPR, "whole chunks");
    __shared__ __attribute__((aligned(16))) char s_k[2][BK * DP * ES];
    __shared__ __attribute__((aligned(16))) char s_v[2][BK * DP * ES];
    __shared__ uint32_t s_ok[3][KB];  // which keys there are
    __shared__ int32_t s_row[3][BK];
    __shared__ __attribute__((aligned(16))) uint2 s_c[3][BIAS ? 3 : 1][BIAS ? BK : 1];
    __shared__ int32_t s_r[3][NW];
    __shared__ int s_flag[NW];

    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), half = lane >> 5;
    // block -> (split, key head, tile or segment): an XCD's blocks are neighbours, on one head's keys
    const uint32_t id = xcd_tile(blockIdx.x, a.blocks);
    const uint32_t per_head = a.blocks / (uint32_t)(a.Hk * a.splits);
    const uint32_t unit = id % per_head;
    const int hk = (int)(id / per_head) % a.Hk, split = (int)(id / per_head) / a.Hk;

    const auto kswz = [](int row, int c) {
        if constexpr (CPR >= 8) return c ^ ((row ^ (row >> 3)) & 7);
        else return c ^ (((row >> 1) ^ (row >> 3)) & 3);
    };
    // V: 32-byte units of a row, so that the four rows of a transposing read lie in different banks
    const auto vswz = [](int row, int c) {
        if constexpr (ES == 4) return c;
        return c ^ (DP == 64 ? 4 * ((row >> 1) & 1) : DP == 128 ? 4 * (row & 3) : 0);
    };

    // slots of the block: [slot0, slot1) of all positions' G slots (SEG: of the segment's)
    int64_t slot0, slot1;
    int32_t seg_lo = 0, seg_hi = 0;  // (positions and rows fit 32 bits)
    if (a.seg) {
        const int64_t p0 = clamp64(a.q_off[unit], 0, a.Pq), p1 = clamp64(a.q_off[unit + 1], 0, a.Pq);
        slot0 = p0 * a.G;
        slot1 = p1 * a.G;
        seg_lo = (int32_t)clamp64(a.k_off[unit], 0, a.Pk);
        seg_hi = (int32_t)clamp64(a.k_off[unit + 1], seg_lo, a.Pk);
    } else {
        slot0 = (int64_t)unit * (32 * NW * QT);
        slot1 = slot0 + 32 * NW * QT;
        if (slot1 > a.Pq * a.G) slot1 = a.Pq * a.G;
    }

    for (int64_t base = slot0; base < slot1; base += 32 * NW * QT) {
        // ---- the lane's slots
        int32_t pos[QT], lo[QT], hi[QT], row[QT], seg[QT], head[QT];
        int32_t blo = (int32_t)a.Pk, bhi = 0;
        const int64_t wfirst = base + wave * QT * 32;
#pragma unroll
        for (int t = 0; t < QT; ++t) {
            const int64_t slot = base + (wave * QT + t) * 32 + (lane & 31);
            const bool in = slot < slot1;
            pos[t] = in ? (int32_t)(slot / a.G) : -1;
            head[t] = hk * a.G + (in ? (int)(slot - (int64_t)pos[t] * a.G) : 0);
            row[t] = -1;
            seg[t] = -1;
            lo[t] = hi[t] = 0;
            int32_t sg = (int32_t)unit;
            if (!a.seg && wfirst < slot1) sg = wave_segment(a.q_off, a.S, (int32_t)(wfirst / a.G), in ? pos[t] : 0x7ffffffe);
            if (in) {
                const int32_t r = a.q_index ? a.q_index[pos[t]] : pos[t];
                row[t] = r >= 0 && r < a.Mq ? r : -1;
                seg[t] = sg;
                if (seg[t] >= 0) {
                    lo[t] = a.seg ? seg_lo : (int32_t)clamp64(a.k_off[seg[t]], 0, a.Pk);
                    hi[t] = a.seg ? seg_hi : (int32_t)clamp64(a.k_off[seg[t] + 1], lo[t], a.Pk);
                    if (hi[t] > lo[t]) {
                        blo = lo[t] < blo ? lo[t] : blo;
                        bhi = hi[t] > bhi ? hi[t] : bhi;
                    }
                }
            }
        }
        // the block's keys, and whether some lane sees only a part of them
        for (int o = 32; o > 0; o >>= 1) {
            const int32_t x = __shfl_xor(blo, o, 64), y = __shfl_xor(bhi, o, 64);
            blo = x < blo ? x : blo;
            bhi = y > bhi ? y : bhi;
        }
        blo = __builtin_amdgcn_readfirstlane(blo);
        bhi = __builtin_amdgcn_readfirstlane(bhi);
        const int32_t wlo = blo, whi = bhi;  // the wave's
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
            blo = __builtin_amdgcn_readfirstlane(blo);
            bhi = __builtin_amdgcn_readfirstlane(bhi);
        }
        // keys that every slot of the wave sees (slots of no segment take whatever comes)
        int32_t ilo = 0, ihi = 0x7fffffff;
#pragma unroll
        for (int t = 0; t < QT; ++t)
            if (seg[t] >= 0) {
                ilo = lo[t] > ilo ? lo[t] : ilo;
                ihi = hi[t] < ihi ? hi[t] : ihi;
            }
        for (int o = 32; o > 0; o >>= 1) {
            const int32_t x = __shfl_xor(ilo, o, 64), y = __shfl_xor(ihi, o, 64);
            ilo = x > ilo ? x : ilo;
            ihi = y < ihi ? y : ihi;
        }
        ilo = __builtin_amdgcn_readfirstlane(ilo);
        ihi = __builtin_amdgcn_readfirstlane(ihi);
        bool part_seen = false;
#pragma unroll
        for (int t = 0; t < QT; ++t) part_seen = part_seen || (seg[t] >= 0 && hi[t] > lo[t] && (lo[t] != blo || hi[t] != bhi));
        if (a.splits > 1 && bhi > blo) {
            const int64_t each = (((int64_t)bhi - blo + a.splits - 1) / a.splits + BK - 1) / BK * BK;
            blo = (int32_t)(blo + split * each < bhi ? blo + split * each : bhi);
            bhi = (int32_t)(blo + each < bhi ? blo + each : bhi);
        }

        // ---- the queries, and their coordinates' operands
        chunk qf[QT][QC];
        v8bf qc[QT][3];
        float sl[QT][3];
#pragma unroll
        for (int t = 0; t < QT; ++t) {
            const T* qp = (const T*)a.q + (int64_t)(row[t] >= 0 ? row[t] : 0) * a.q_row + head[t] * a.q_head;
#pragma unroll
            for (int c = 0; c < QC; ++c) {
                const int cc = 2 * c + half;
                qf[t][c] = chunk{};
                if (row[t] >= 0 && cc * PER < a.D) qf[t][c] = *(const chunk*)(qp + cc * PER);
            }
            if constexpr (BIAS) {
                // the difference of two coordinates as a product: key parts (8 bits each, exact in bf16) times
                // their weights, minus the weights times the query's parts; exact up to 2^24
#pragma unroll
                for (int x = 0; x < 3; ++x) {
                    const int32_t c = row[t] >= 0 ? a.q_coords[(int64_t)row[t] * 4 + 1 + x] : 0;
                    sl[t][x] = -a.slopes[head[t] * 3 + x] * PMG_LOG2E;
                    const float p[4] = {(float)(c & 255), (float)((c >> 8) & 255), (float)((c >> 16) & 255), (float)(c >> 24)};
                    const float w[4] = {1.0f, 256.0f, 65536.0f, 16777216.0f};
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        qc[t][x][i] = (__bf16)(half ? 0.0f : w[i]);
                        qc[t][x][4 + i] = (__bf16)(half ? 0.0f : -p[i]);
                    }
                }
            }
        }

        int32_t only = -1;  // >= 0: the one segment this turn is for
        for (;;) {
            int32_t klo = blo, khi = bhi;
            if (only >= 0) {
                const int32_t l0 = (int32_t)clamp64(a.k_off[only], 0, a.Pk), h0 = (int32_t)clamp64(a.k_off[only + 1], l0, a.Pk);
                klo = l0 > blo ? l0 : blo;
                khi = h0 < bhi ? h0 : bhi;
            }
            const int32_t nt = khi > klo ? (khi - klo + (BK - 1)) / BK : 0;

            v16f O[QT][NB];
            float m[QT], l[QT], grow[QT];
            const float k2 = a.cap2 != 0.0f ? 1.0f : a.scale2;
#pragma unroll
            for (int t = 0; t < QT; ++t) {
                m[t] = 0.0f;
                grow[t] = -__builtin_inff();
                l[t] = 0.0f;
#pragma unroll
                for (int b = 0; b < NB; ++b) O[t][b] = v16f{};
            }

            // ---- the keys: row numbers three tiles ahead, mask and coordinates two, data one
            const bool mt = tid < BK;  // a thread that looks after a key of each tile
            int32_t mi = -1;           // its row in the tile whose mask and coordinates come next
            const auto number = [&](int32_t t) -> int32_t {
                if (!mt || t >= nt || tid >= khi - klo - t * BK) return -1;
                const int32_t p = klo + t * BK + tid, r = a.k_index ? a.k_index[p] : p;
                return r >= 0 && r < (int32_t)a.Mk ? r : -1;
            };
            int4 mc = make_int4(0, 0, 0, 0);
            uint8_t mm = 1;
            const auto about = [&]() {  // of row mi
                const int64_t r = mi >= 0 ? mi : 0;
                if (a.k_mask) mm = a.k_mask[r];
                if constexpr (BIAS) mc = *(const int4*)(a.k_coords + r * 4);
            };
            const auto note = [&](int b, int32_t r) {
                if (wave == 0) {
                    const bool on = r >= 0 && mm != 0;
                    const uint64_t w = __ballot(mt && on);
                    if (tid < KB) s_ok[b][tid] = (uint32_t)(w >> (32 * tid));
                    if (mt) s_row[b][tid] = on ? r : -1;
                    if constexpr (BIAS) {
                        if (mt) {
                            const int32_t c[3] = {mc.y, mc.z, mc.w};
#pragma unroll
                            for (int x = 0; x < 3; ++x) {
                                const auto b16 = [](int v) { return f2u((float)v) >> 16; };  // (exact: 8 bits)
                                s_c[b][x][tid] = make_uint2(b16(c[x] & 255) | (b16((c[x] >> 8) & 255) << 16),
                                                            b16((c[x] >> 16) & 255) | (b16(c[x] >> 24) << 16));
                            }
                        }
                    }
                }
            };
            // (rows are less than 2^31 bytes apart; a chunk behind the head's width is the line of zeros of every row)
            const char *kb[NCH], *vb[NCH];
            uint32_t ks[NCH], vs[NCH];
#pragma unroll
            for (int i = 0; i < NCH; ++i) {
                const int e = (i * NW + wave) * 64 + lane, r = e / CPR, p = e % CPR;
                const int ck = kswz(r, p) * PER, cv = vswz(r, p) * PER;
                kb[i] = ck < a.D ? (const char*)((const T*)a.k + hk * a.k_head + ck) : (const char*)&g_zeros;
                vb[i] = cv < a.D ? (const char*)((const T*)a.v + hk * a.v_head + cv) : (const char*)&g_zeros;
                ks[i] = ck < a.D ? (uint32_t)a.k_row * ES : 0u;
                vs[i] = cv < a.D ? (uint32_t)a.v_row * ES : 0u;
            }
            const auto fetch = [&](int b, int nb) {  // the tile noted in slot nb, into buffer b
#pragma unroll
                for (int i = 0; i < NCH; ++i) {
                    const int32_t row = s_row[nb][((i * NW + wave) * 64 + lane) / CPR];
                    const char* kp = row >= 0 ? kb[i] + (uint64_t)(uint32_t)row * ks[i] : (const char*)&g_zeros;
                    const char* vp = row >= 0 ? vb[i] + (uint64_t)(uint32_t)row * vs[i] : (const char*)&g_zeros;
                    typedef __attribute__((address_space(1))) const void* gp;
                    typedef __attribute__((address_space(3))) void* lp;
                    __builtin_amdgcn_global_load_lds((gp)kp, (lp)(s_k[b] + (i * NW + wave) * 1024), 16, 0, 0);
                    __builtin_amdgcn_global_load_lds((gp)vp, (lp)(s_v[b] + (i * NW + wave) * 1024), 16, 0, 0);
                }
            };
            if (nt > 0) {
                mi = number(0);
                about();
                const int32_t m1 = number(1);
                note(0, mi);
                mi = m1;
                about();
                const int32_t m2 = number(2);
                note(1, mi);
                mi = m2;
                __syncthreads();
                fetch(0, 0);
            }
            __syncthreads();

            for (int32_t it = 0; it < nt; ++it) {
                const int cur = it & 1;
                const bool more = it + 1 < nt;
                const int slot = it % 3, next_slot = (it + 1) % 3;
                int32_t mn = -1;
                if (more) {
                    fetch(cur ^ 1, next_slot);
                    about();
                    mn = number(it + 3);
                }
                const int32_t p0 = klo + it * BK;
                if (p0 < whi && wlo - p0 < BK) {
#pragma unroll
                    for (int t = 0; t < QT; ++t) {
                        v16f s[KB];
                        // ---- scores
#pragma unroll
                        for (int b = 0; b < KB; ++b) s[b] = v16f{};
                        constexpr int QG = QC < 4 ? QC : 4;  // operand chunks at a time
#pragma unroll
                        for (int c0 = 0; c0 < QC; c0 += QG) {
                            chunk kf[KB][QG];
#pragma unroll
                            for (int c = 0; c < QG; ++c)
#pragma unroll
                                for (int b = 0; b < KB; ++b) {
                                    const int kr_ = 32 * b + (lane & 31);
                                    kf[b][c] = *(const chunk*)(s_k[cur] + kr_ * DP * ES + 16 * kswz(kr_, 2 * (c0 + c) + half));
                                }
                            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                            for (int c = 0; c < QG; ++c)
#pragma unroll
                                for (int b = 0; b < KB; ++b) s[b] = Mat<T>::mma32(kf[b][c], qf[t][c0 + c], s[b]);
                        }
                        // less the maximum so far, in powers of two
                        if (a.cap2 != 0.0f) {
#pragma unroll
                            for (int b = 0; b < KB; ++b)
#pragma unroll
                                for (int e = 0; e < 16; ++e) {
                                    if constexpr (ES == 4) s[b][e] = a.cap2 * tanhf(s[b][e] * a.cap_arg);
                                    else s[b][e] = __builtin_fmaf(-2.0f * a.cap2, __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(s[b][e] * a.cap_arg)), a.cap2);
                                }
                        }
                        if constexpr (BIAS) {
#pragma unroll
                            for (int b = 0; b < KB; ++b) {
                                v16f u;
#pragma unroll
                                for (int x = 0; x < 3; ++x) {
                                    const uint2 kp = s_c[slot][x][32 * b + (lane & 31)];
                                    // parts, then the weights 1, 2^8, 2^16, 2^24 in bf16
                                    // (both halves of the wave hold them: the query's are 0 in the upper one)
                                    const v4i kc = v4i{(int)kp.x, (int)kp.y, (int)0x43803f80u, (int)0x4b804780u};
                                    const v16f d = Mat<__bf16>::mma32(__builtin_bit_cast(v8bf, kc), qc[t][x], v16f{});
#pragma unroll
                                    for (int e = 0; e < 16; ++e) u[e] = __builtin_fmaf(__builtin_fabsf(d[e]), sl[t][x], x == 0 ? -m[t] : u[e]);
                                }
#pragma unroll
                                for (int e = 0; e < 16; ++e) s[b][e] = __builtin_fmaf(s[b][e], k2, u[e]);
                            }
                        } else {
#pragma unroll
                            for (int b = 0; b < KB; ++b)
#pragma unroll
                                for (int e = 0; e < 16; ++e) s[b][e] = __builtin_fmaf(s[b][e], k2, -m[t]);
                        }
                        // ---- the keys that count for the lane's slot
                        const int jl = lo[t] - p0, jh = hi[t] - p0;
                        const bool inside = p0 >= ilo && ihi - p0 >= BK;
#pragma unroll
                        for (int b = 0; b < KB; ++b) {
                            const uint32_t ok = __builtin_amdgcn_readfirstlane(s_ok[slot][b]);
                            if (!inside || ok != 0xffffffffu) {
                                const int x = jl - 32 * b, y = jh - 32 * b;
                                uint32_t w = y >= 32 ? 0xffffffffu : y <= 0 ? 0u : (1u << y) - 1u;
                                w &= x <= 0 ? 0xffffffffu : x >= 32 ? 0u : ~((1u << x) - 1u);
                                w = (w & ok) >> (4 * half);
#pragma unroll
                                for (int e = 0; e < 16; ++e) {
                                    const uint32_t on = (uint32_t)((int32_t)(w << (31 - ((e & 3) + 8 * (e >> 2)))) >> 31);
                                    s[b][e] = u2f((on & f2u(s[b][e])) | (~on & 0xff800000u));
                                }
                            }
                        }
                        // ---- running maximum: set by the first keys, then moved only when it grows by more than
                        // 2^8 for some slot of the wave (weights of up to 2^8 lose nothing)
                        float mx = s[0][0];
#pragma unroll
                        for (int b = 0; b < KB; ++b)
#pragma unroll
                            for (int e = 0; e < 16; ++e) mx = __builtin_fmaxf(mx, s[b][e]);
                        mx = __builtin_fmaxf(mx, other_half(mx));
                        if (__any(mx > grow[t])) {
                            const bool any = mx > -__builtin_inff();  // (a slot without a key so far keeps m = 0)
                            const float up = any && (mx > 0.0f || grow[t] < 0.0f) ? mx : 0.0f;
                            const float al = __builtin_amdgcn_exp2f(-up);
                            grow[t] = any ? 8.0f : grow[t];
                            m[t] = m[t] + up;
                            l[t] = l[t] * al;
#pragma unroll
                            for (int b = 0; b < KB; ++b)
#pragma unroll
                                for (int e = 0; e < 16; ++e) s[b][e] = s[b][e] - up;
#pragma unroll
                            for (int b = 0; b < NB; ++b)
#pragma unroll
                                for (int e = 0; e < 16; ++e) O[t][b][e] = O[t][b][e] * al;
                        }
                        // (the first operands of V are on their way while the exponentials are formed)
                        chunk vf[2][NB];
                        const auto values = [&](int b, int f) {
                            typedef short v4s __attribute__((ext_vector_type(4)));
                            typedef short v8s __attribute__((ext_vector_type(8)));
                            typedef __attribute__((address_space(3))) v4s* lds4;
#pragma unroll
                            for (int n = 0; n < NB; ++n) {
                                const int i = lane & 15, c = 4 * n + 2 * ((lane >> 4) & 1) + ((i & 3) >> 1);
                                const int r0 = 32 * b + 16 * f + 4 * half + (i >> 2);
                                const v4s v0 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4)(s_v[cur] + r0 * DP * 2 + 16 * vswz(r0, c) + (i & 1) * 8));
                                const v4s v1 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4)(s_v[cur] + (r0 + 8) * DP * 2 + 16 * vswz(r0 + 8, c) + (i & 1) * 8));
                                const v8s vv = __builtin_shufflevector(v0, v1, 0, 1, 2, 3, 4, 5, 6, 7);
                                vf[f][n] = __builtin_bit_cast(chunk, vv);
                            }
                        };
                        if constexpr (ES == 2) {
                            values(0, 0);
                            values(0, 1);
                            __builtin_amdgcn_sched_barrier(0);
                        }
                        float sum = 0.0f;
#pragma unroll
                        for (int b = 0; b < KB; ++b)
#pragma unroll
                            for (int e = 0; e < 16; ++e) {
                                s[b][e] = __builtin_amdgcn_exp2f(s[b][e]);
                                sum = sum + s[b][e];
                            }
                        l[t] = l[t] + sum;
                        // ---- O^T += V^T P^T
#pragma unroll
                        for (int b = 0; b < KB; ++b) {
                            if constexpr (ES == 4) {
#pragma unroll
                                for (int e = 0; e < 16; ++e) {
                                    const int kr_ = 32 * b + (e & 3) + 8 * (e >> 2) + 4 * half;
#pragma unroll
                                    for (int n = 0; n < NB; ++n) {
                                        const float vf = *(const float*)(s_v[cur] + kr_ * DP * 4 + (32 * n + (lane & 31)) * 4);
                                        O[t][n] = __builtin_amdgcn_mfma_f32_32x32x2f32(vf, s[b][e], O[t][n], 0, 0, 0);
                                    }
                                }
                            } else {
#pragma unroll
                                for (int f = 0; f < 2; ++f) {
                                    chunk pf;
#pragma unroll
                                    for (int i = 0; i < 8; ++i) pf[i] = (T)s[b][8 * f + i];
#pragma unroll
                                    for (int n = 0; n < NB; ++n) O[t][n] = Mat<T>::mma32(vf[f][n], pf, O[t][n]);
                                    if (b + 1 < KB) values(b + 1, f);
                                }
                            }
                        }
                    }
                }
                if (more) {
                    note((it + 2) % 3, mi);
                    mi = mn;
                }
                __syncthreads();
            }

            const AttnArgs& a = args_again();
            // ---- values of other segments that are not finite: once more, segment by segment
            if (only < 0) {
                float bad = 0.0f;
#pragma unroll
                for (int t = 0; t < QT; ++t)
#pragma unroll
                    for (int b = 0; b < NB; ++b)
#pragma unroll
                        for (int e = 0; e < 16; ++e) bad = __builtin_fmaf(O[t][b][e], 0.0f, bad);
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
#pragma unroll
            for (int t = 0; t < QT; ++t) {
                const float lt = l[t] + other_half(l[t]);
                const bool mine = only == -2 ? seg[t] < 0 : only < 0 || seg[t] == only;
                if (a.splits > 1) {
                    if (mine && seg[t] >= 0) {
                        const int64_t o = ((int64_t)split * a.Pq + pos[t]) * a.Hq + head[t];
                        if (half == 0) a.part_ml[o] = make_float2(grow[t] > 0.0f ? m[t] : -__builtin_inff(), lt);
#pragma unroll
                        for (int b = 0; b < NB; ++b)
#pragma unroll
                            for (int g = 0; g < 4; ++g) {
                                const int d = 32 * b + 8 * g + 4 * half;
                                if (d < a.D) *(float4*)(a.part_o + o * a.D + d) = make_float4(O[t][b][4 * g], O[t][b][4 * g + 1], O[t][b][4 * g + 2], O[t][b][4 * g + 3]);
                            }
                    }
                } else if (mine && row[t] >= 0 && (seg[t] >= 0 || a.zero_rest)) {
                    const bool none = lt == 0.0f || seg[t] < 0;  // no key left
                    const float inv = 1.0f / lt;
                    T* op = (T*)a.out + (int64_t)row[t] * a.o_row + head[t] * a.o_head;
#pragma unroll
                    for (int b = 0; b < NB; ++b)
#pragma unroll
                        for (int g = 0; g < 4; ++g) {
                            const int d = 32 * b + 8 * g + 4 * half;
                            typedef T v4t __attribute__((ext_vector_type(4)));
                            v4t v;
#pragma unroll
                            for (int i = 0; i < 4; ++i) v[i] = (T)(none ? 0.0f : O[t][b][4 * g + i] * inv);
                            if (d < a.D) *(v4t*)(op + d) = v;
                        }
                }
            }
            if (only == -1) break;
            // the next segment of the block
            int32_t next = 0x7fffffff;
#pragma unroll
            for (int t = 0; t < QT; ++t)
                if (seg[t] >= 0 && seg[t] > only && seg[t] < next) next = seg[t];
            for (int o = 32; o > 0; o >>= 1) {
                const int32_t x = __shfl_xor(next, o, 64);
                next = x < next ? x : next;
            }
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
}

// Joins the splits: a wave a (position, head). Its lanes are G groups of 16 or 32, each on every G-th split and 4 columns a
// lane; the groups' sums are added in order at the end.
template <class T, int CL>
__global__ __launch_bounds__(256) void attention_join_k(AttnArgs a) {
    constexpr int G = 64 / CL;
    const int lane = threadIdx.x & 63, g = lane / CL, d = 4 * (lane % CL);
    const int64_t item = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    if (item >= a.Pq * a.Hq) return;
    const int64_t pos = item / a.Hq;
    const int head = (int)(item - pos * a.Hq);
    const int32_t r = a.q_index ? a.q_index[pos] : (int32_t)pos;
    const bool in = segment_of(a.q_off, a.S, pos) >= 0;
    if (r < 0 || r >= a.Mq || (!in && !a.zero_rest)) return;
    typedef T v4t __attribute__((ext_vector_type(4)));
    v4t* op = (v4t*)((T*)a.out + (int64_t)r * a.o_row + head * a.o_head + d);
    const bool mine = g == 0 && d < a.D;
    if (!in) {
        if (mine) *op = v4t{(T)0.0f, (T)0.0f, (T)0.0f, (T)0.0f};
        return;
    }
    const int64_t step = a.Pq * a.Hq;
    float m = -__builtin_inff();
    for (int s = lane; s < a.splits; s += 64) m = __builtin_fmaxf(m, a.part_ml[item + s * step].x);
    for (int o = 32; o > 0; o >>= 1) m = __builtin_fmaxf(m, __shfl_xor(m, o, 64));
    const float ms = m == -__builtin_inff() ? 0.0f : m;
    float l = 0.0f;
    v4f acc = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll 4
    for (int s = g; s < a.splits; s += G) {
        const float2 ml = a.part_ml[item + s * step];
        const v4f po = d < a.D ? *(const v4f*)(a.part_o + (item + s * step) * a.D + d) : v4f{0.0f, 0.0f, 0.0f, 0.0f};
        const float w = __builtin_amdgcn_exp2f(ml.x - ms);
        if (ml.y != 0.0f) {  // (a part without keys counts for nothing)
            l = __builtin_fmaf(ml.y, w, l);
#pragma unroll
            for (int i = 0; i < 4; ++i) acc[i] = __builtin_fmaf(po[i], w, acc[i]);
        }
    }
#pragma unroll
    for (int o = CL; o < 64; o <<= 1) {
        l = l + __shfl_xor(l, o, 64);
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[i] = acc[i] + __shfl_xor(acc[i], o, 64);
    }
    if (!mine) return;
    const float inv = 1.0f / l;
    v4t v;
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = (T)(l == 0.0f ? 0.0f : acc[i] * inv);
    *op = v;
}

// The rows outside every segment, where blocks go by segment.
template <class T>
__global__ __launch_bounds__(256) void attention_rest_k(AttnArgs a) {
    const int64_t item = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    if (item >= a.Pq) return;
    if (segment_of(a.q_off, a.S, item) >= 0) return;
    const int64_t r = a.q_index ? a.q_index[item] : item;
    if (r < 0 || r >= a.Mq) return;
    for (int h = 0; h < a.Hq; ++h)
        for (int d = threadIdx.x & 63; d < a.D; d += 64) ((T*)a.out)[r * a.o_row + h * a.o_head + d] = (T)0.0f;
}

template <class T, int DP, int NW, int QT>
static int launch_attention_w(AttnArgs& a, hipStream_t s) {
    const int64_t units = a.seg ? a.S : (a.Pq * a.G + 32 * NW * QT - 1) / (32 * NW * QT);
    const int64_t blocks = units * a.Hk * a.splits;
    PMG_REQUIRE(blocks < (int64_t)1 << 31, "too many blocks");
    a.blocks = (uint32_t)blocks;
    if (a.slopes) hipLaunchKernelGGL((attention_k<T, DP, NW, QT, true>), dim3(a.blocks), dim3(64 * NW), 0, s, a);
    else hipLaunchKernelGGL((attention_k<T, DP, NW, QT, false>), dim3(a.blocks), dim3(64 * NW), 0, s, a);
    return check_launch("attention_k");
}

template <class T, int DP>
static int launch_attention_d(AttnArgs& a, int waves, hipStream_t s) {
    return waves == 1 ? launch_attention_w<T, DP, 1, 1>(a, s) : launch_attention_w<T, DP, 4, 1>(a, s);
}

template <class T>
int launch_attention_t(AttnArgs& a, int waves, hipStream_t s) {
    int e = a.D <= 32 ? launch_attention_d<T, 32>(a, waves, s) : a.D <= 64 ? launch_attention_d<T, 64>(a, waves, s) : launch_attention_d<T, 128>(a, waves, s);
    if (e) return e;
    if (a.splits > 1) {
        const dim3 grid((unsigned)((a.Pq * a.Hq + 3) / 4));
        if (a.D <= 64) hipLaunchKernelGGL((attention_join_k<T, 16>), grid, dim3(256), 0, s, a);
        else hipLaunchKernelGGL((attention_join_k<T, 32>), grid, dim3(256), 0, s, a);
        return check_launch("attention_join_k");
    }
    if (a.seg && a.zero_rest) {
        hipLaunchKernelGGL((attention_rest_k<T>), dim3((unsigned)((a.Pq + 3) / 4)), dim3(256), 0, s, a);
        return check_launch("attention_rest_k");
    }
    return PMG_OK;
}

int launch_attention_f16(AttnArgs& a, int waves, hipStream_t s);
int launch_attention_bf16(AttnArgs& a, int waves, hipStream_t s);
int launch_attention_f32(AttnArgs& a, int waves, hipStream_t s);

}  // namespace pmg
