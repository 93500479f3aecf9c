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
// row-major V by the transposing LDS read (fp32: by plain reads). K and V tiles are staged through registers (rows are
// gathered by index, absent ones become zeros) one tile ahead into the other of two LDS buffers.
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

__device__ inline int64_t clamp64(int64_t v, int64_t lo, int64_t hi) { return v < lo ? lo : v > hi ? hi : v; }

// The other half's value (lane l <-> l ^ 32).
__device__ inline float other_half(float v) {
    const uint32_t u = f2u(v);
    const auto r = __builtin_amdgcn_permlane32_swap(u, u, false, false);
    return u2f((threadIdx.x & 32) ? r[0] : r[1]);
}

template <class T, int DP, int NW, int QT, bool BIAS>
__global__ __launch_bounds__(64 * NW) void attention_k(AttnArgs a) {
    constexpr int ES = sizeof(T), PER = 16 / ES, CPR = DP / PER, NT = 64 * NW;
    constexpr int BK = (NW == 1 || ES == 4) ? 32 : 64, KB = BK / 32;
    constexpr int NCH = BK * CPR / NT;         // 16-byte chunks of K (and of V) a thread stages
    constexpr int NB = DP / 32;                // 32-column blocks of O
    constexpr int QC = CPR / 2;                // operand chunks of a query a lane holds
    typedef typename Mat<T>::chunk chunk;
    static_assert(NCH * NT == BK * CPR, "whole chunks");
    __shared__ __attribute__((aligned(16))) char s_k[2][BK * DP * ES];
    __shared__ __attribute__((aligned(16))) char s_v[2][BK * DP * ES];
    __shared__ uint32_t s_ok[2][KB];
    __shared__ __attribute__((aligned(16))) uint2 s_c[2][BIAS ? 3 : 1][BIAS ? BK : 1];
    __shared__ int64_t s_r[4][NW];
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
    const auto vadr = [](int row, int c) {
        if constexpr (ES == 4) return row * DP * 4 + c * 16;
        const int f = DP == 64 ? 2 * ((row >> 1) & 1) : DP == 128 ? 2 * (row & 3) : 0;
        return row * DP * 2 + (((c >> 1) ^ f) * 32) + (c & 1) * 16;
    };

    // slots of the block: [slot0, slot1) of all positions' G slots (SEG: of the segment's)
    int64_t slot0, slot1, seg_lo = 0, seg_hi = 0;
    if (a.seg) {
        const int64_t p0 = clamp64(a.q_off[unit], 0, a.Pq), p1 = clamp64(a.q_off[unit + 1], 0, a.Pq);
        slot0 = p0 * a.G;
        slot1 = p1 * a.G;
        seg_lo = clamp64(a.k_off[unit], 0, a.Pk);
        seg_hi = clamp64(a.k_off[unit + 1], seg_lo, a.Pk);
    } else {
        slot0 = (int64_t)unit * (32 * NW * QT);
        slot1 = slot0 + 32 * NW * QT;
        if (slot1 > a.Pq * a.G) slot1 = a.Pq * a.G;
    }

    for (int64_t base = slot0; base < slot1; base += 32 * NW * QT) {
        // ---- the lane's slots
        int64_t pos[QT], lo[QT], hi[QT], row[QT];
        int32_t seg[QT];
        int head[QT];
        int64_t blo = a.Pk, bhi = 0;
#pragma unroll
        for (int t = 0; t < QT; ++t) {
            const int64_t slot = base + (wave * QT + t) * 32 + (lane & 31);
            const bool in = slot < slot1;
            pos[t] = in ? slot / a.G : -1;
            head[t] = hk * a.G + (in ? (int)(slot - pos[t] * a.G) : 0);
            row[t] = -1;
            seg[t] = -1;
            lo[t] = hi[t] = 0;
            if (in) {
                int64_t r = a.q_index ? a.q_index[pos[t]] : pos[t];
                row[t] = r >= 0 && r < a.Mq ? r : -1;
                seg[t] = a.seg ? (int32_t)unit : segment_of(a.q_off, a.S, pos[t]);
                if (seg[t] >= 0) {
                    lo[t] = a.seg ? seg_lo : clamp64(a.k_off[seg[t]], 0, a.Pk);
                    hi[t] = a.seg ? seg_hi : clamp64(a.k_off[seg[t] + 1], lo[t], a.Pk);
                    if (hi[t] > lo[t]) {
                        blo = lo[t] < blo ? lo[t] : blo;
                        bhi = hi[t] > bhi ? hi[t] : bhi;
                    }
                }
            }
        }
        // the block's keys, and whether some lane sees only a part of them
        for (int o = 32; o > 0; o >>= 1) {
            const int64_t x = __shfl_xor(blo, o, 64), y = __shfl_xor(bhi, o, 64);
            blo = x < blo ? x : blo;
            bhi = y > bhi ? y : bhi;
        }
        int64_t wlo = blo, whi = bhi;  // the wave's
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
        bool part_seen = false;
#pragma unroll
        for (int t = 0; t < QT; ++t) part_seen = part_seen || (seg[t] >= 0 && hi[t] > lo[t] && (lo[t] != blo || hi[t] != bhi));
        if (a.splits > 1 && bhi > blo) {
            const int64_t each = ((bhi - blo + a.splits - 1) / a.splits + BK - 1) / BK * BK;
            blo = blo + split * each < bhi ? blo + split * each : bhi;
            bhi = blo + each < bhi ? blo + each : bhi;
        }

        // ---- the queries, and their coordinates' operands
        chunk qf[QT][QC];
        v8bf qc[QT][3];
        float sl[QT][3];
#pragma unroll
        for (int t = 0; t < QT; ++t) {
            const T* qp = (const T*)a.q + (row[t] >= 0 ? row[t] : 0) * a.q_row + head[t] * a.q_head;
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
                    const int32_t c = row[t] >= 0 ? a.q_coords[row[t] * 4 + 1 + x] : 0;
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
            int64_t klo = blo, khi = bhi;
            if (only >= 0) {
                const int64_t l0 = clamp64(a.k_off[only], 0, a.Pk), h0 = clamp64(a.k_off[only + 1], l0, a.Pk);
                klo = l0 > blo ? l0 : blo;
                khi = h0 < bhi ? h0 : bhi;
            }
            const int64_t nt = khi > klo ? (khi - klo + BK - 1) / BK : 0;

            v16f O[QT][NB];
            float m[QT], l[QT];
#pragma unroll
            for (int t = 0; t < QT; ++t) {
                m[t] = -__builtin_inff();
                l[t] = 0.0f;
#pragma unroll
                for (int b = 0; b < NB; ++b) O[t][b] = v16f{};
            }

            // ---- staging: row numbers two tiles ahead, data one tile ahead
            int32_t idx[NCH], midx = -1;
            chunk kr[NCH], vr[NCH];
            bool okr[NCH];
            int4 mc = make_int4(0, 0, 0, 0);
            bool mok = false;
            const auto row_at = [&](int64_t p) -> int32_t {
                if (p >= khi) return -1;
                const int64_t r = a.k_index ? (int64_t)a.k_index[p] : p;
                return r >= 0 && r < a.Mk ? (int32_t)r : -1;
            };
            const auto rows = [&](int64_t t) {
#pragma unroll
                for (int i = 0; i < NCH; ++i) idx[i] = row_at(klo + t * BK + (i * NT + tid) / CPR);
                if (tid < BK) midx = row_at(klo + t * BK + tid);
            };
            const auto load = [&]() {
#pragma unroll
                for (int i = 0; i < NCH; ++i) {
                    const int c = (i * NT + tid) % CPR;
                    const int64_t r = idx[i] >= 0 ? idx[i] : 0;
                    const int cc = c * PER < a.D ? c * PER : 0;
                    okr[i] = idx[i] >= 0 && c * PER < a.D;
                    kr[i] = *(const chunk*)((const T*)a.k + r * a.k_row + hk * a.k_head + cc);
                    vr[i] = *(const chunk*)((const T*)a.v + r * a.v_row + hk * a.v_head + cc);
                    if (a.k_mask) okr[i] = okr[i] && a.k_mask[r] != 0;
                }
                if (tid < BK) {
                    const int64_t r = midx >= 0 ? midx : 0;
                    mok = midx >= 0 && (!a.k_mask || a.k_mask[r] != 0);
                    if constexpr (BIAS) mc = *(const int4*)(a.k_coords + r * 4);
                }
            };
            const auto put = [&](int b) {
#pragma unroll
                for (int i = 0; i < NCH; ++i) {
                    const int e = i * NT + tid, r = e / CPR, c = e % CPR;
                    *(chunk*)(s_k[b] + r * DP * ES + 16 * kswz(r, c)) = okr[i] ? kr[i] : chunk{};
                    *(chunk*)(s_v[b] + vadr(r, c)) = okr[i] ? vr[i] : chunk{};
                }
                if (wave == 0) {
                    const uint64_t w = __ballot(tid < BK && mok);
                    if (tid < KB) s_ok[b][tid] = (uint32_t)(w >> (32 * tid));
                    if constexpr (BIAS) {
                        if (tid < BK) {
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
            if (nt > 0) {
                rows(0);
                load();
                rows(1);
                put(0);
            }
            __syncthreads();

            for (int64_t it = 0; it < nt; ++it) {
                const int cur = (int)(it & 1);
                const bool more = it + 1 < nt;
                if (more) {
                    load();
                    rows(it + 2);
                }
                const int64_t p0 = klo + it * BK;
                if (p0 < whi && p0 + BK > wlo) {
#pragma unroll
                    for (int t = 0; t < QT; ++t) {
                        v16f s[KB];
                        // ---- scores, in powers of two
#pragma unroll
                        for (int b = 0; b < KB; ++b) {
                            s[b] = v16f{};
                            const int kr_ = 32 * b + (lane & 31);
#pragma unroll
                            for (int c = 0; c < QC; ++c) {
                                const chunk kf = *(const chunk*)(s_k[cur] + kr_ * DP * ES + 16 * kswz(kr_, 2 * c + half));
                                s[b] = Mat<T>::mma32(kf, qf[t][c], s[b]);
                            }
                        }
                        float k2 = a.scale2;  // what s is still to be multiplied by
                        if (a.cap2 != 0.0f) {
#pragma unroll
                            for (int b = 0; b < KB; ++b)
#pragma unroll
                                for (int e = 0; e < 16; ++e) {
                                    if constexpr (ES == 4) s[b][e] = a.cap2 * tanhf(s[b][e] * a.cap_arg);
                                    else s[b][e] = __builtin_fmaf(-2.0f * a.cap2, __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(s[b][e] * a.cap_arg)), a.cap2);
                                }
                            k2 = 1.0f;
                        }
                        if constexpr (BIAS) {
#pragma unroll
                            for (int b = 0; b < KB; ++b) {
#pragma unroll
                                for (int e = 0; e < 16; ++e) s[b][e] = s[b][e] * k2;
#pragma unroll
                                for (int x = 0; x < 3; ++x) {
                                    const uint2 kp = s_c[cur][x][32 * b + (lane & 31)];
                                    // parts, then the weights 1, 2^8, 2^16, 2^24 in bf16
                                    const v4i kc = half ? v4i{0, 0, 0, 0} : v4i{(int)kp.x, (int)kp.y, (int)0x43803f80u, (int)0x4b804780u};
                                    const v16f d = Mat<__bf16>::mma32(__builtin_bit_cast(v8bf, kc), qc[t][x], v16f{});
#pragma unroll
                                    for (int e = 0; e < 16; ++e) s[b][e] = __builtin_fmaf(__builtin_fabsf(d[e]), sl[t][x], s[b][e]);
                                }
                            }
                            k2 = 1.0f;
                        }
                        // ---- the keys that count for the lane's slot
                        const int64_t rl = lo[t] - p0, rh = hi[t] - p0;
                        const int jl = (int)(rl < 0 ? 0 : rl > BK ? BK : rl), jh = (int)(rh < 0 ? 0 : rh > BK ? BK : rh);
#pragma unroll
                        for (int b = 0; b < KB; ++b) {
                            const int x = jl - 32 * b, y = jh - 32 * b;
                            uint32_t w = y >= 32 ? 0xffffffffu : y <= 0 ? 0u : (1u << y) - 1u;
                            w &= x <= 0 ? 0xffffffffu : x >= 32 ? 0u : ~((1u << x) - 1u);
                            w &= s_ok[cur][b];
                            if (!__all(w == 0xffffffffu)) {
                                w >>= 4 * half;
#pragma unroll
                                for (int e = 0; e < 16; ++e) {
                                    const uint32_t on = (uint32_t)((int32_t)(w << (31 - ((e & 3) + 8 * (e >> 2)))) >> 31);
                                    s[b][e] = u2f((on & f2u(s[b][e])) | (~on & 0xff800000u));
                                }
                            }
                        }
                        // ---- running maximum: moved only when it grows by more than 2^8 somewhere in the wave
                        float mx = s[0][0];
#pragma unroll
                        for (int b = 0; b < KB; ++b)
#pragma unroll
                            for (int e = 0; e < 16; ++e) mx = __builtin_fmaxf(mx, s[b][e]);
                        mx = __builtin_fmaxf(mx, other_half(mx)) * k2;
                        if (__any(mx > m[t] + 8.0f)) {
                            const float mn = __builtin_fmaxf(m[t], mx);
                            const float al = m[t] == mn ? 1.0f : __builtin_amdgcn_exp2f(m[t] - mn);
                            m[t] = mn;
                            l[t] = l[t] * al;
#pragma unroll
                            for (int b = 0; b < NB; ++b)
#pragma unroll
                                for (int e = 0; e < 16; ++e) O[t][b][e] = O[t][b][e] * al;
                        }
                        const float ms = m[t] == -__builtin_inff() ? 0.0f : m[t];
                        float sum = 0.0f;
#pragma unroll
                        for (int b = 0; b < KB; ++b)
#pragma unroll
                            for (int e = 0; e < 16; ++e) {
                                s[b][e] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[b][e], k2, -ms));
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
                                    for (int n = 0; n < NB; ++n) {
                                        typedef short v4s __attribute__((ext_vector_type(4)));
                                        typedef __attribute__((address_space(3))) v4s* lds4;
                                        const int i = lane & 15, c = 4 * n + 2 * ((lane >> 4) & 1) + ((i & 3) >> 1);
                                        const int r0 = 32 * b + 16 * f + 4 * half + (i >> 2);
                                        const v4s v0 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4)(s_v[cur] + vadr(r0, c) + (i & 1) * 8));
                                        const v4s v1 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4)(s_v[cur] + vadr(r0 + 8, c) + (i & 1) * 8));
                                        typedef short v8s __attribute__((ext_vector_type(8)));
                                        const v8s vv = __builtin_shufflevector(v0, v1, 0, 1, 2, 3, 4, 5, 6, 7);
                                        O[t][n] = Mat<T>::mma32(__builtin_bit_cast(chunk, vv), pf, O[t][n]);
                                    }
                                }
                            }
                        }
                    }
                }
                if (more) put(cur ^ 1);
                __syncthreads();
            }

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
                        if (half == 0) a.part_ml[o] = make_float2(m[t], lt);
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
                    T* op = (T*)a.out + row[t] * a.o_row + head[t] * a.o_head;
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
            int64_t next = (int64_t)1 << 40;
#pragma unroll
            for (int t = 0; t < QT; ++t)
                if (seg[t] >= 0 && seg[t] > only && seg[t] < next) next = seg[t];
            for (int o = 32; o > 0; o >>= 1) {
                const int64_t x = __shfl_xor(next, o, 64);
                next = x < next ? x : next;
            }
            if constexpr (NW > 1) {
                __syncthreads();
                if (lane == 0) s_r[2][wave] = next;
                __syncthreads();
#pragma unroll
                for (int w = 0; w < NW; ++w) next = s_r[2][w] < next ? s_r[2][w] : next;
            }
            if (next == (int64_t)1 << 40) break;
            only = (int32_t)next;
        }
    }
}

// Joins the splits: a wave a (position, head).
template <class T>
__global__ __launch_bounds__(256) void attention_join_k(AttnArgs a) {
    const int lane = threadIdx.x & 63;
    const int64_t item = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    if (item >= a.Pq * a.Hq) return;
    const int64_t pos = item / a.Hq;
    const int head = (int)(item - pos * a.Hq);
    const int64_t r = a.q_index ? a.q_index[pos] : pos;
    if (r < 0 || r >= a.Mq) return;
    T* op = (T*)a.out + r * a.o_row + head * a.o_head;
    if (segment_of(a.q_off, a.S, pos) < 0) {
        if (a.zero_rest)
            for (int d = lane; d < a.D; d += 64) op[d] = (T)0.0f;
        return;
    }
    const int64_t step = a.Pq * a.Hq;
    float m = -__builtin_inff();
    for (int s = lane; s < a.splits; s += 64) {
        const float2 ml = a.part_ml[item + s * step];
        m = __builtin_fmaxf(m, ml.x);
    }
    for (int o = 32; o > 0; o >>= 1) m = __builtin_fmaxf(m, __shfl_xor(m, o, 64));
    const float ms = m == -__builtin_inff() ? 0.0f : m;
    float l = 0.0f, o0 = 0.0f, o1 = 0.0f;
    for (int s = 0; s < a.splits; ++s) {  // in the splits' order
        const float2 ml = a.part_ml[item + s * step];
        const float w = __builtin_amdgcn_exp2f(ml.x - ms);
        if (ml.y == 0.0f) continue;  // a part without keys
        l = __builtin_fmaf(ml.y, w, l);
        const float* po = a.part_o + (item + s * step) * a.D;
        if (lane < a.D) o0 = __builtin_fmaf(po[lane], w, o0);
        if (lane + 64 < a.D) o1 = __builtin_fmaf(po[lane + 64], w, o1);
    }
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
    if (lane < a.D) op[lane] = (T)(l == 0.0f ? 0.0f : o0 * inv);
    if (lane + 64 < a.D) op[lane + 64] = (T)(l == 0.0f ? 0.0f : o1 * inv);
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
        hipLaunchKernelGGL((attention_join_k<T>), dim3((unsigned)((a.Pq * a.Hq + 3) / 4)), dim3(256), 0, s, a);
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
