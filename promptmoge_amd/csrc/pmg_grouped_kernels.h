// Kernels of the grouped products; both have w's rows as the matrix instruction's row operand, so that a lane holds four
// neighbouring columns of one row of the result.
//
// Measured (MI355X), and what bounds it: 9600 gathered rows of 1024 bf16, 8 experts, to 4096, gelu: 110 to 120 us, 670 to 730
// TFLOP/s (the matrix units at what the chip's power leaves of their rate, a third round of tiles half full, the epilogue under them);
// 131k rows of 256 fp16, 16 experts, to 128, scattered: 25 to 27 us, 4 TB/s; 8 rows, 8 experts, 1024 to 4096 bf16: 12 us, 44 MB of
// weights; 4800 rows of 1024 fp16 to 1024 with adapters of rank 16 and a residual: 30 us, 6 of them the first half.
#pragma once
#include "pmg_grouped.h"

namespace pmg {

constexpr uint32_t kBehind = 0x7ffffff0u;  // an offset behind every buffer's end: reads zeros

// ------------------------------------------------------------------------------------------------------------ tiles
// A block's BM positions by BN columns from tiles of KB bytes of k in NS LDS buffers, filled by direct loads to LDS several
// tiles ahead (VEC: rows of x and w on 16 bytes, K whole 16-byte chunks, gathered rows below 2 GiB; else element by element).
// Tiles start where a segment starts (kRowAdapters: every BM rows), so that a tile has one w (one adapter).
// kAdapters: the low products come in front, as more k: rows of x's parts against `up` as often, their sums multiplied
// by the row's factor before the k of x and w.
template <class T, int BM, int BN, int WM, int WN, int KB, int NS, bool VEC, int KIND>
__global__ __launch_bounds__(64 * WM * WN, 2) void grouped_tile_k(GroupArgs a) {
    static_assert(KIND != kAdapters || VEC, "parts are read 16 bytes at a time");
    constexpr int NW = WM * WN, NT = 64 * NW, KE = KB / (int)sizeof(T), PER = Mat<T>::kPer, ES = (int)sizeof(T);
    constexpr int CPR = KB / 16, RPL = 64 / CPR, STEPS = CPR / 2;  // chunks a row, rows a load, steps a tile
    constexpr int TM = BM / WM, TN = BN / WN, MT = TM / 32, NTL = TN / 32;
    constexpr int NL = ((BM + BN) / RPL + NW - 1) / NW, kStage = VEC ? NL * NW * 1024 : (BM + BN) * KB;  // a wave's loads a tile
    typedef typename Mat<T>::chunk chunk;
    typedef typename Mat<T>::acc32 acc32;
    extern __shared__ __attribute__((aligned(16))) char lds[];
    __shared__ int to[BM];                   // each row's place in the result
    __shared__ int from[VEC ? 1 : BM];       // and in x
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int wm = wave / WN, wn = wave % WN;
    uint32_t tile;
    Piece pc;
    if constexpr (KIND == kRowAdapters) {
        tile = xcd_tile(blockIdx.x, a.tiles);
        pc.first = (int)((a.id0 + tile / a.tiles_n) * BM);
        pc.n = a.P - pc.first < BM ? a.P - pc.first : BM;
        pc.s = 0;
    } else if (a.S <= 254) {
        const auto counted = [&](const auto& c) {
            const uint32_t rest = c.total > a.id0 ? c.total - a.id0 : 0u, most = a.tiles / a.tiles_n;
            const uint32_t tiles = (rest < most ? rest : most) * a.tiles_n;
            if (blockIdx.x >= tiles) return false;
            tile = xcd_tile(blockIdx.x, tiles);
            pc = c.at(a, a.id0 + tile / a.tiles_n, BM);
            return true;
        };
        const bool ends = KIND == kAdapters || a.fresh;
        if (!(a.S <= 62 ? counted(PieceCount<1>(a, BM, ends)) : counted(PieceCount<4>(a, BM, ends)))) return;
    } else {
        tile = xcd_tile(blockIdx.x, a.tiles);
        pc = piece_of(a, a.id0 + tile / a.tiles_n, BM);
    }
    const int n0 = (int)(tile % a.tiles_n) * BN;
    if (pc.n < 1) return;
    const int rows_n = a.N - n0 < BN ? a.N - n0 : BN;
    if (KIND == kExperts && pc.s < 0) {  // positions of no segment
        if (a.fresh) {
            constexpr int G = BN / 8;
            for (int e = tid; e < pc.n * G; e += NT) {
                const int c = 8 * (e % G);
                if (c < rows_n) zero8(a, pc.first + e / G, n0 + c, rows_n - c < 8 ? rows_n - c : 8);
            }
        }
        return;
    }
    const int seg = KIND == kExperts ? pc.s : 0;
    const int ad = KIND == kAdapters ? adapter_of(a, pc.tag) : -1;
    const bool gather = KIND == kExperts && a.index;
    const T* xb = (const T*)a.x + (gather ? 0 : (int64_t)pc.first * a.ldx);
    const T* wb = (const T*)a.w + (int64_t)seg * a.w_next + (int64_t)n0 * a.K;
    const int nk = (a.K + KE - 1) / KE;
    constexpr int LPR = TN / 8, RPP = 64 / LPR, NP = 32 / RPP;  // lanes a row, rows a pass, passes
    const int nc = n0 + wn * TN + 8 * (lane % LPR);
    const int left = a.N - nc < 8 ? a.N - nc : 8;
    // All that the tile looks up in tables is asked for at once: the rows of the lane's loads, a row's place, the bias.
    static_assert(BM <= NT, "a row's place a thread");
    int rows[VEC ? NL : 1];
    float bs[8];
    if constexpr (VEC) {
        const int last = pc.first + pc.n - 1;
#pragma unroll
        for (int i = 0; i < NL; ++i) {
            const int p = pc.first + (i * NW + wave) * RPL + lane / CPR;
            rows[i] = gather ? a.index[p < last ? p : last] : p - pc.first;
        }
    }
    {
        const int p = pc.first + (tid < pc.n ? tid : 0), from_p = gather ? a.index[p] : p;
        const int to_p = KIND == kExperts ? row_out(a, p, from_p) : p;
        bias8(a, seg, nc, bs);
        if (tid < BM) {
            to[tid] = tid < pc.n ? to_p : -1;
            if constexpr (!VEC) from[tid] = tid >= pc.n || !in_x(a, from_p) ? -1 : gather ? from_p : tid;
        }
    }
    if constexpr (!VEC) __syncthreads();

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
        const int kbytes = a.K * ES, lowbytes = kParts<T> * a.r * ES;
        const int ne = ad >= 0 ? (lowbytes + KB - 1) / KB : 0, nt = ne + nk;  // tiles of parts, tiles in all
        const int64_t xspan = ((gather ? a.x_rows : (int64_t)pc.n) - 1) * a.ldx + a.K;
        const v4i rx = buffer_of(xb, (uint32_t)(xspan * ES));
        const v4i rw = buffer_of(wb, (uint32_t)(((int64_t)(rows_n - 1) * a.K + a.K) * ES));
        v4i rl = rx, ru = rw;
        if (KIND == kAdapters && ad >= 0) {
            rl = buffer_of((const char*)a.low + (int64_t)pc.first * lowbytes, (uint32_t)(pc.n * lowbytes));
            ru = buffer_of((const T*)a.up + ((int64_t)ad * a.N + n0) * a.r, (uint32_t)(rows_n * a.r * ES));
        }
        uint32_t off[NL];
        int kc[NL];  // byte of k of the lane's chunk in tile 0
#pragma unroll
        for (int i = 0; i < NL; ++i) {
            const int row = (i * NW + wave) * RPL + lane / CPR;
            const bool isx = (i * NW + wave) * RPL < BM;  // (uniform over the wave)
            const int rr = isx ? row : row - BM;
            kc[i] = 16 * swizzle<CPR>(rr, lane % CPR);
            if (isx) {
                // (gathered: below 2 GiB; else a tile's rows are, of 4 MiB each)
                off[i] = rr < pc.n && (!gather || in_x(a, rows[i])) ? (uint32_t)rows[i] * ((uint32_t)a.ldx * ES) + kc[i] : kBehind;
            } else {
                off[i] = rr < rows_n ? (uint32_t)rr * ((uint32_t)a.K * ES) + kc[i] : kBehind;
            }
        }
        const uint32_t base = lds_address(lds);
        const auto fill = [&](int t, uint32_t place) {
            if (KIND == kAdapters && t < ne) {
#pragma unroll
                for (int i = 0; i < NL; ++i) {
                    const int row = (i * NW + wave) * RPL + lane / CPR;
                    const bool isx = (i * NW + wave) * RPL < BM;
                    const int rr = isx ? row : row - BM, b = t * KB + kc[i], rb = a.r * ES;
                    const int ub = b >= 2 * rb ? b - 2 * rb : b >= rb ? b - rb : b;
                    const bool there = b < lowbytes && rr < (isx ? pc.n : rows_n);
                    const uint32_t o = !there ? kBehind : isx ? (uint32_t)(rr * lowbytes + b) : (uint32_t)(rr * rb + ub);
                    buffer_to_lds(isx ? rl : ru, o, 0, base + place * kStage + (i * NW + wave) * 1024);
                }
                return;
            }
            const int tk = t - ne;
            const bool whole = (tk + 1) * KB <= kbytes;
#pragma unroll
            for (int i = 0; i < NL; ++i) {
                const uint32_t o = whole || tk * KB + kc[i] < kbytes ? off[i] : kBehind;
                buffer_to_lds((i * NW + wave) * RPL < BM ? rx : rw, o, (uint32_t)(tk * KB), base + place * kStage + (i * NW + wave) * 1024);
            }
        };
        // While one step's products are formed the next step's operands are read; before the last step of tile t all
        // waves have its operands in registers, so its place takes tile t + NS.
#pragma unroll
        for (int t = 0; t < NS; ++t)
            if (t < nt) fill(t, t);
        if (NS - 1 < nt) landed_barrier<(NS - 1) * NL>();
        else landed_barrier<0>();
        operands(lds, 0);
        uint32_t place = 0;
        for (int t = 0; t < nt; ++t) {
#pragma unroll
            for (int s = 0; s + 1 < STEPS; ++s) {
                operands(lds + place * kStage, s + 1);
                multiply(s);
            }
            if (t + 1 < nt) {
                if (t + NS - 1 < nt) landed_barrier<(NS - 2) * NL>();
                else landed_barrier<0>();
                if (t + NS < nt) fill(t + NS, place);
                place = place + 1 == NS ? 0 : place + 1;
                operands(lds + place * kStage, 0);
            }
            multiply(STEPS - 1);
            if constexpr (KIND == kAdapters && __is_same(T, _Float16)) {
                if (t + 1 == ne) {
#pragma unroll
                    for (int i = 0; i < MT; ++i) {
                        const int row = wm * TM + 32 * i + r;
                        const float f = row < pc.n ? a.low_factor[pc.first + row] : 1.0f;
#pragma unroll
                        for (int j = 0; j < NTL; ++j)
#pragma unroll
                            for (int e = 0; e < 16; ++e) acc[i][j][e] = acc[i][j][e] * f;
                    }
                }
            }
        }
    } else {
        for (int t = 0; t < nk; ++t) {
            for (int e = tid; e < (BM + BN) * CPR; e += NT) {
                const int row = e / CPR, c = e % CPR, k = t * KE + c * PER;
                chunk v{};
                if (row < BM) {
                    if (from[row] >= 0) v = load_chunk_any<T>(xb + from[row] * a.ldx, k, a.K);
                } else if (row - BM < rows_n) {
                    v = load_chunk_any<T>(wb + (int64_t)(row - BM) * a.K, k, a.K);
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

    // Sums through LDS: 32 rows of the wave's TN columns at a time, in fp32. The passes over them are a loop that loads nothing from
    // memory, for a load would have the wave wait for the stores in front of it too (loads and stores share one counter);
    // where a wave has 32 rows, their residuals are numbers in registers before the first store.
    constexpr int LD = TN + 4;
    float* st = (float*)lds + wave * 32 * LD;
    const auto place = [&](int i, int p) { return left > 0 ? to[wm * TM + 32 * i + p * RPP + lane / LPR] : -1; };
    const auto sums = [&](int p, float (&v)[8]) {
        const float* from = st + (p * RPP + lane / LPR) * LD + 8 * (lane % LPR);
        const v4f u0 = *(const v4f*)from, u1 = *(const v4f*)(from + 4);
#pragma unroll
        for (int q = 0; q < 8; ++q) v[q] = (q < 4 ? u0[q & 3] : u1[q & 3]) + bs[q];
    };
#pragma unroll
    for (int i = 0; i < MT; ++i) {
#pragma unroll
        for (int j = 0; j < NTL; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                v4f v;
#pragma unroll
                for (int q = 0; q < 4; ++q) v[q] = acc[i][j][4 * e + q];
                *(v4f*)(st + r * LD + 32 * j + 8 * e + 4 * (lane >> 5)) = v;
            }
        float res[MT == 1 ? NP : 1][8];
        if (MT == 1 && a.res) {
#pragma unroll
            for (int p = 0; p < NP; ++p) {
                const int m = place(i, p);
                if (m >= 0) residual8(a, m, nc, left, res[MT == 1 ? p : 0]);
            }
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
        const auto pass = [&](int p, const float* add) {
            const int m = place(i, p);
            float v[8];
            sums(p, v);
            if (m >= 0) {
                if constexpr (KIND == kRowAdapters) add_low<T>(a, m, nc, left, v);
                if (add) {
                    activate8(v, a.act, a.out_type == PMG_TYPE_F32);
#pragma unroll
                    for (int q = 0; q < 8; ++q) v[q] = v[q] + add[q];
                    put8<true>(a, m, nc, left, v);
                } else {
                    finish8<true>(a, m, nc, left, v);
                }
            } else if (KIND == kExperts && m < -1) {
                zero8(a, -2 - m, nc, left);
            }
        };
        if (MT == 1 && a.res) {
#pragma unroll
            for (int p = 0; p < NP; ++p) pass(p, res[MT == 1 ? p : 0]);
        } else {
#pragma unroll 1
            for (int p = 0; p < NP; ++p) pass(p, nullptr);
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
    }
}

// --------------------------------------------------------------------------------------------------------- few rows
// 16 positions of a segment (kRowAdapters: 16 rows) by 16 NC columns a block, k shared out over the block's NW waves in steps
// of 64 bytes, operands straight to registers; the waves' sums are added in wave order through LDS.
template <class T, int NC, int U, int NW, bool VEC, int KIND>
__global__ __launch_bounds__(64 * NW) void grouped_rows_k(GroupArgs a) {
    typedef typename Mat<T>::chunk chunk;
    typedef typename Mat<T>::acc16 acc16;
    constexpr int PER = Mat<T>::kPer;
    __shared__ float red[NW][16][16 * NC + 1];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, r = lane & 15, g = lane >> 4;
    const uint32_t id = a.id0 + blockIdx.x / a.tiles_n;
    const int n0 = (int)(blockIdx.x % a.tiles_n) * 16 * NC;
    Piece pc;
    if constexpr (KIND == kRowAdapters) {
        pc.first = (int)(id * 16);
        pc.n = a.P - pc.first < 16 ? a.P - pc.first : 16;
        pc.s = 0;
    } else {
        pc = piece_of(a, id, 16);
    }
    if (pc.n < 1) return;
    const int t = threadIdx.x, row = t / (2 * NC), c = n0 + 8 * (t % (2 * NC));  // 8 outputs a thread
    const int left = a.N - c < 8 ? a.N - c : 8;
    const bool out = t < 32 * NC && row < pc.n && left > 0;
    if (KIND == kExperts && pc.s < 0) {
        if (a.fresh && out) zero8(a, pc.first + row, c, left);
        return;
    }
    const int seg = KIND == kExperts ? pc.s : 0;
    const T* wr[NC];
#pragma unroll
    for (int j = 0; j < NC; ++j) {
        const int n = n0 + 16 * j + r;
        wr[j] = (const T*)a.w + (int64_t)seg * a.w_next + (int64_t)(n < a.N ? n : a.N - 1) * a.K;
    }
    const int p_in = pc.first + (r < pc.n ? r : pc.n - 1), p_out = pc.first + (out ? row : 0);
    const int m = KIND == kExperts ? row_in(a, p_in) : p_in, m_out = KIND == kExperts ? row_in(a, p_out) : p_out;
    const T* xr = (const T*)a.x + (int64_t)(KIND != kExperts || in_x(a, m) ? m : 0) * a.ldx;  // (an absent position's sums are not used)
    const int place = !out ? -1 : KIND == kExperts ? row_out(a, p_out, m_out) : p_out;
    float v[8];
    bias8(a, seg, c < a.N ? c : 0, v);
    const int nsteps = (a.K + 4 * PER - 1) / (4 * PER);
    acc16 acc[NC];
#pragma unroll
    for (int j = 0; j < NC; ++j) acc[j] = acc16{};
    auto get = [&](const T* p, int k) -> chunk {
        if constexpr (VEC) {
            // (a chunk behind K reads the row's first one instead and counts as zeros)
            const chunk v = *(const chunk*)(p + (k < a.K ? k : 0));
            return k < a.K ? v : chunk{};
        } else {
            return load_chunk_any<T>(p, k, a.K);
        }
    };
    for (int s0 = wave; s0 < nsteps; s0 += NW * U) {
        chunk fw[U][NC], fx[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int k = (4 * (s0 + u * NW) + g) * PER;
#pragma unroll
            for (int j = 0; j < NC; ++j) fw[u][j] = get(wr[j], k);
        }
#pragma unroll
        for (int u = 0; u < U; ++u) fx[u] = get(xr, (4 * (s0 + u * NW) + g) * PER);  // (w's rows are known before x's)
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int j = 0; j < NC; ++j) acc[j] = Mat<T>::mma16(fw[u][j], fx[u], acc[j]);
    }
#pragma unroll
    for (int j = 0; j < NC; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) red[wave][r][16 * j + 4 * g + e] = acc[j][e];
    __syncthreads();
    if (place == -1) return;
    if (KIND == kExperts && place < 0) {
        zero8(a, -2 - place, c, left);
        return;
    }
#pragma unroll
    for (int q = 0; q < 8; ++q) {
        float s = 0.0f;
#pragma unroll
        for (int w = 0; w < NW; ++w) s = s + red[w][row][8 * (t % (2 * NC)) + q];
        v[q] = s + v[q];
    }
    if constexpr (KIND == kRowAdapters) add_low<T>(a, place, c, left, v);
    finish8(a, place, c, left, v);
}

// ------------------------------------------------------------------------------------------------- the adapters' first half
// low[m][j] = scale[i] sum_k x[m][k] down[i][j][k], i the adapter of row m's segment, for 16 rows of a segment and all r <= 16 NR of
// its values: x is read once. Where each row is a segment: for `rows` (1 or 16) rows, once for each adapter among them.
// For grouped_tile_k's kAdapters (PARTS) as [m][part][r] in T, fp16's multiplied by a power of two that brings the row's largest
// finite value to 2^14 .. 2^15 (low_factor: its inverse), which neither overflows nor is lost below 2^-24; else as [m][r] in fp32, with
// each row's adapter.
template <class T, int NR, int NW, bool VEC, bool PARTS>
__global__ __launch_bounds__(64 * NW) void lora_low_k(GroupArgs a, int rows) {
    typedef typename Mat<T>::chunk chunk;
    typedef typename Mat<T>::acc16 acc16;
    constexpr int PER = Mat<T>::kPer, U = 4 / NR < 1 ? 1 : 4 / NR;
    __shared__ float red[NW][16][16 * NR + 1];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, r = lane & 15, g = lane >> 4;
    const uint32_t id = a.id0 + blockIdx.x;
    int first, n, tag = -1;
    if (a.offsets) {
        const Piece pc = piece_of(a, id, 16);
        first = pc.first;
        n = pc.n;
        tag = pc.tag;
    } else {
        first = (int)id * rows;
        n = a.P - first < rows ? a.P - first : rows;
    }
    if (n < 1) return;
    const int mine = r < n ? r : n - 1;
    const T* xr = (const T*)a.x + (int64_t)(first + mine) * a.ldx;
    const int nsteps = (a.K + 4 * PER - 1) / (4 * PER);
    auto get = [&](const T* p, int k) -> chunk {
        if constexpr (VEC) {
            const chunk v = *(const chunk*)(p + (k < a.K ? k : 0));
            return k < a.K ? v : chunk{};
        } else {
            return load_chunk_any<T>(p, k, a.K);
        }
    };
    chunk fx[U];  // (the first round's rows of x are on their way while the adapter is looked up)
    const auto rows_of = [&](int s0) {
#pragma unroll
        for (int u = 0; u < U; ++u) fx[u] = get(xr, (4 * (s0 + u * NW) + g) * PER);
    };
    if (wave < nsteps) rows_of(wave);
    const int own = adapter_of(a, a.offsets ? tag : a.tag[first + mine]);  // of the lane's row r
    const int t = threadIdx.x, row = t >> 4, c = t & 15;
    if (!PARTS && t < n) a.row_adapter[first + t] = own;  // (t is r there)
    uint32_t todo = (uint32_t)(__ballot(own >= 0) & (n < 16 ? (1u << n) - 1u : 0xffffu));  // rows of an adapter (nothing reads the others' low products)
    bool again = false;
    while (todo) {
        const int ad = __builtin_amdgcn_readlane(own, __builtin_ctz(todo));
        const uint32_t these = (uint32_t)__ballot(own == ad) & todo;
        todo &= ~these;
        const float sc = a.scale ? a.scale[ad] : 1.0f;
        const T* wr[NR];
#pragma unroll
        for (int j = 0; j < NR; ++j) {
            const int q = 16 * j + r;
            wr[j] = (const T*)a.down + ((int64_t)ad * a.r + (q < a.r ? q : a.r - 1)) * a.K;
        }
        acc16 acc[NR];
#pragma unroll
        for (int j = 0; j < NR; ++j) acc[j] = acc16{};
        for (int s0 = wave; s0 < nsteps; s0 += NW * U) {
            chunk fw[U][NR];
            if (s0 != wave || again) rows_of(s0);
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int k = (4 * (s0 + u * NW) + g) * PER;
#pragma unroll
                for (int j = 0; j < NR; ++j) fw[u][j] = get(wr[j], k);
            }
#pragma unroll
            for (int u = 0; u < U; ++u)
#pragma unroll
                for (int j = 0; j < NR; ++j) acc[j] = Mat<T>::mma16(fw[u][j], fx[u], acc[j]);
        }
        if (again) __syncthreads();
        again = true;
#pragma unroll
        for (int j = 0; j < NR; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e) red[wave][r][16 * j + 4 * g + e] = acc[j][e];
        __syncthreads();
        if (t >= 256) continue;
        const int m = first + row;
        const bool writes = (these >> row) & 1;
        float v[NR], top = 0.0f;
#pragma unroll
        for (int j = 0; j < NR; ++j) {
            float s = 0.0f;
#pragma unroll
            for (int w = 0; w < NW; ++w) s = s + red[w][row][16 * j + c];
            v[j] = 16 * j + c < a.r ? s * sc : 0.0f;
            top = __builtin_fabsf(v[j]) < __builtin_inff() ? __builtin_fmaxf(top, __builtin_fabsf(v[j])) : top;
        }
        if constexpr (!PARTS) {
            float* h = (float*)a.low + (int64_t)m * a.r;
#pragma unroll
            for (int j = 0; j < NR; ++j)
                if (writes && 16 * j + c < a.r) h[16 * j + c] = v[j];
        } else {
            float f = 1.0f;
            if constexpr (__is_same(T, _Float16)) {
#pragma unroll
                for (int o = 1; o < 16; o <<= 1) top = __builtin_fmaxf(top, __shfl_xor(top, o, 16));
                const int e = (int)(f2u(top) >> 23);  // (0: zero or subnormal)
                const int up = 127 + 14 + 127 - e;    // exponent field of 2^14 / 2^(e - 127)
                f = top == 0.0f ? 1.0f : u2f((uint32_t)(up > 247 ? 247 : up) << 23);
                if (writes && c == 0) a.low_factor[m] = 1.0f / f;
            }
            T* h = (T*)a.low + (int64_t)m * kParts<T> * a.r;
#pragma unroll
            for (int j = 0; j < NR; ++j) {
                float x = v[j] * f;
                const bool ends = !(__builtin_fabsf(x) < __builtin_inff());  // (infinity less itself would be NaN)
#pragma unroll
                for (int p = 0; p < kParts<T>; ++p) {
                    T y = (T)x;
                    if constexpr (__is_same(T, __bf16)) {  // (the largest that is finite: what is above it rounds to infinity)
                        constexpr float most = 0x1.fep127f;
                        y = ends ? y : (T)__builtin_fminf(__builtin_fmaxf(x, -most), most);
                    }
                    if (writes && 16 * j + c < a.r) h[p * a.r + 16 * j + c] = y;
                    x = ends ? 0.0f : x - (float)y;
                }
            }
        }
    }
}

// -------------------------------------------------------------------------------------- few rows of an adapter each, in one launch
// All rows, kFew at the most, by 16 NC columns a block, where every row is a segment and r <= 16: each wave forms its share of k of
// the low products too, once for each adapter among the rows (a lane keeps what its own row's adapter gave), and the epilogue adds
// them from LDS. What the matrix instruction has of rows behind the last is not kept.
template <class T, int NC, int NW, bool VEC>
__global__ __launch_bounds__(64 * NW) void lora_few_k(GroupArgs a) {
    typedef typename Mat<T>::chunk chunk;
    typedef typename Mat<T>::acc16 acc16;
    constexpr int PER = Mat<T>::kPer, U = 4, A = 4, R = kFew;
    __shared__ float red[NW][R][16 * NC + 1], red_low[NW][R][17], low[R][16];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, r = lane & 15, g = lane >> 4;
    const int n0 = (int)blockIdx.x * 16 * NC, n = a.P, mine = r < n ? r : n - 1;
    const T* xr = (const T*)a.x + (int64_t)mine * a.ldx;
    const T* wr[NC];
#pragma unroll
    for (int j = 0; j < NC; ++j) {
        const int c = n0 + 16 * j + r;
        wr[j] = (const T*)a.w + (int64_t)(c < a.N ? c : a.N - 1) * a.K;
    }
    const int own = adapter_of(a, a.tag[mine]);  // of the lane's row r
    const float own_scale = own >= 0 ? (a.scale ? a.scale[own] : 1.0f) : 0.0f;
    const int t = threadIdx.x, row = t / (2 * NC), c = n0 + 8 * (t % (2 * NC));  // 8 outputs a thread
    const int left = a.N - c < 8 ? a.N - c : 8;
    const bool out = row < n && left > 0;
    float v[8];
    bias8(a, 0, c < a.N ? c : 0, v);
    const uint32_t rows = (uint32_t)(__ballot(own >= 0) & ((1u << n) - 1u));  // rows of an adapter
    const int nsteps = (a.K + 4 * PER - 1) / (4 * PER);
    acc16 acc[NC], acc_low = acc16{};
#pragma unroll
    for (int j = 0; j < NC; ++j) acc[j] = acc16{};
    auto get = [&](const T* p, int k) -> chunk {
        if constexpr (VEC) {
            // (a chunk behind K reads the row's first one instead and counts as zeros)
            const chunk x = *(const chunk*)(p + (k < a.K ? k : 0));
            return k < a.K ? x : chunk{};
        } else {
            return load_chunk_any<T>(p, k, a.K);
        }
    };
    for (int s0 = wave; s0 < nsteps; s0 += NW * U) {
        chunk fw[U][NC], fx[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int k = (4 * (s0 + u * NW) + g) * PER;
            fx[u] = get(xr, k);
#pragma unroll
            for (int j = 0; j < NC; ++j) fw[u][j] = get(wr[j], k);
        }
        for (uint32_t todo = rows; todo;) {  // four adapters' loads on their way at a time
            chunk fd[A][U];
            int ad[A];
#pragma unroll
            for (int i = 0; i < A; ++i) {
                ad[i] = todo ? __builtin_amdgcn_readlane(own, __builtin_ctz(todo)) : -1;
                if (ad[i] < 0) continue;
                todo &= ~(uint32_t)__ballot(own == ad[i]);
                const T* dr = (const T*)a.down + ((int64_t)ad[i] * a.r + (r < a.r ? r : a.r - 1)) * a.K;
#pragma unroll
                for (int u = 0; u < U; ++u) fd[i][u] = get(dr, (4 * (s0 + u * NW) + g) * PER);
            }
#pragma unroll
            for (int i = 0; i < A; ++i) {
                if (ad[i] < 0) continue;
                acc16 got = acc_low;
#pragma unroll
                for (int u = 0; u < U; ++u) got = Mat<T>::mma16(fd[i][u], fx[u], got);
#pragma unroll
                for (int e = 0; e < 4; ++e) acc_low[e] = own == ad[i] ? got[e] : acc_low[e];
            }
        }
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int j = 0; j < NC; ++j) acc[j] = Mat<T>::mma16(fw[u][j], fx[u], acc[j]);
    }
    if (r < R) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
#pragma unroll
            for (int j = 0; j < NC; ++j) red[wave][r][16 * j + 4 * g + e] = acc[j][e];
            red_low[wave][r][4 * g + e] = acc_low[e];
        }
    }
    __syncthreads();
    if (t < 16 * R) {
        float s = 0.0f;
#pragma unroll
        for (int w = 0; w < NW; ++w) s = s + red_low[w][t >> 4][t & 15];
        const float sc = __shfl(own_scale, t >> 4, 64);  // (lanes 0 .. R - 1 of every wave hold the rows' scales)
        low[t >> 4][t & 15] = s * sc;
    }
    __syncthreads();
    if (!out) return;
#pragma unroll
    for (int q = 0; q < 8; ++q) {
        float s = 0.0f;
#pragma unroll
        for (int w = 0; w < NW; ++w) s = s + red[w][row][8 * (t % (2 * NC)) + q];
        v[q] = s + v[q];
    }
    const int ad = adapter_of(a, a.tag[row]);
    if (ad >= 0) add_low8<T>(a, ad, low[row], c, left, v);
    finish8(a, row, c, left, v);
}

// ------------------------------------------------------------------------------------------------------------- launch
template <class T, int BM, int BN, int WM, int WN, int KB, int NS, bool VEC, int KIND>
static int launch_grouped_tile(GroupArgs& a, hipStream_t s) {
    constexpr int NW = WM * WN, RPL = 1024 / KB;
    constexpr int kStage = VEC ? ((BM + BN) / RPL + NW - 1) / NW * NW * 1024 : (BM + BN) * KB, kOut = NW * 32 * (BN / WN + 4) * 4;
    const int nk = (a.K * (int)sizeof(T) + KB - 1) / KB + (KIND == kAdapters ? (kParts<T> * a.r * (int)sizeof(T) + KB - 1) / KB : 0);
    int bytes = kStage * (!VEC ? 1 : nk < NS ? nk : NS);
    if (bytes < kOut) bytes = kOut;
    a.tiles_n = (uint32_t)((a.N + BN - 1) / BN);
    const uint32_t ids = KIND == kRowAdapters ? (uint32_t)(((int64_t)a.P + BM - 1) / BM) : piece_tiles(a.P, a.S, BM);
    const uint32_t most = (uint32_t)(grid_blocks(64 * NW) / a.tiles_n);  // (N is at most 2^16 tiles of 64)
    for (uint32_t i = 0; i < ids; i += most) {
        a.id0 = i;
        a.tiles = (ids - i < most ? ids - i : most) * a.tiles_n;
        hipLaunchKernelGGL((grouped_tile_k<T, BM, BN, WM, WN, KB, NS, VEC, KIND>), dim3(a.tiles), dim3(64 * NW), bytes, s, a);
        if (int e = check_launch("grouped_tile_k")) return e;
        if (ids - i <= most) break;
    }
    return PMG_OK;
}

template <class T, int NC, int U, int NW, bool VEC, int KIND>
static int launch_grouped_rows(GroupArgs& a, hipStream_t s) {
    a.tiles_n = (uint32_t)((a.N + 16 * NC - 1) / (16 * NC));
    const uint32_t ids = KIND == kRowAdapters ? (uint32_t)(((int64_t)a.P + 15) / 16) : piece_tiles(a.P, a.S, 16);
    const uint32_t most = (uint32_t)(grid_blocks(64 * NW) / a.tiles_n);
    for (uint32_t i = 0; i < ids; i += most) {
        a.id0 = i;
        a.tiles = (ids - i < most ? ids - i : most) * a.tiles_n;
        hipLaunchKernelGGL((grouped_rows_k<T, NC, U, NW, VEC, KIND>), dim3(a.tiles), dim3(64 * NW), 0, s, a);
        if (int e = check_launch("grouped_rows_k")) return e;
        if (ids - i <= most) break;
    }
    return PMG_OK;
}

// Without offsets a block takes a row, or 16 of many rows (which may have one adapter).
template <class T, bool VEC, bool PARTS>
static int launch_low(GroupArgs& a, hipStream_t s) {
    const int rows = a.P <= 4096 ? 1 : 16;
    const uint32_t ids = a.offsets ? piece_tiles(a.P, a.S, 16) : (uint32_t)(((int64_t)a.P + rows - 1) / rows);
    const uint32_t most = (uint32_t)grid_blocks(512);
    for (uint32_t i = 0; i < ids; i += most) {
        a.id0 = i;
        const dim3 grid(ids - i < most ? ids - i : most);
        if (a.r <= 16) hipLaunchKernelGGL((lora_low_k<T, 1, 8, VEC, PARTS>), grid, dim3(512), 0, s, a, rows);
        else if (a.r <= 32) hipLaunchKernelGGL((lora_low_k<T, 2, 8, VEC, PARTS>), grid, dim3(512), 0, s, a, rows);
        else if (a.r <= 64) hipLaunchKernelGGL((lora_low_k<T, 4, 4, VEC, PARTS>), grid, dim3(256), 0, s, a, rows);
        else hipLaunchKernelGGL((lora_low_k<T, 8, 4, VEC, PARTS>), grid, dim3(256), 0, s, a, rows);
        if (int e = check_launch("lora_low_k")) return e;
        if (ids - i <= most) break;
    }
    return PMG_OK;
}

// Shape I of tile_shape's, by WM x WN waves, tiles of KB bytes of k.
template <class T, int I, int WM, int WN, int KB, bool VEC, int KIND>
static int launch_shape(GroupArgs& a, hipStream_t s) {
    constexpr const int* p = sizeof(T) == 4 ? kShapes32[I] : kShapes16[I];
    return launch_grouped_tile<T, p[0], p[1], WM, WN, KB, p[2], VEC, KIND>(a, s);
}
template <class T, bool VEC, int KIND>
static int launch_tiles(GroupArgs& a, hipStream_t s) {
    if constexpr (VEC) {
        const int shape = tile_shape(sizeof(T) == 4, true, KIND, a.P, a.S, a.K, a.N);
        if constexpr (sizeof(T) == 4) {
            if (shape == 1) return launch_shape<T, 1, 2, 2, 64, VEC, KIND>(a, s);
            if (shape == 2) return launch_shape<T, 2, 2, 4, 128, VEC, KIND>(a, s);
        } else {
            if (shape == 1) return launch_shape<T, 1, 2, 2, 128, VEC, KIND>(a, s);
            if (shape == 2) return launch_shape<T, 2, 2, 4, 128, VEC, KIND>(a, s);
            if (shape == 3) return launch_shape<T, 3, 4, 2, 128, VEC, KIND>(a, s);
            if (shape == 4) return launch_shape<T, 4, 2, 4, 64, VEC, KIND>(a, s);
            if (shape == 5) return launch_shape<T, 5, 6, 2, 128, VEC, KIND>(a, s);
        }
    }
    return launch_shape<T, 0, 2, 2, 128, VEC, KIND>(a, s);
}

template <class T>
int launch_experts(GroupArgs& a, bool vec, hipStream_t s) {
    if (few_a_segment(a.P, a.S)) return vec ? launch_grouped_rows<T, 2, 4, 4, true, kExperts>(a, s) : launch_grouped_rows<T, 1, 4, 4, false, kExperts>(a, s);
    return vec ? launch_tiles<T, true, kExperts>(a, s) : launch_tiles<T, false, kExperts>(a, s);
}

template <class T>
int launch_lora(GroupArgs& a, bool vec, bool by_segment, hipStream_t s) {
    if (!a.low) {
        constexpr int NC = 2;
        const dim3 grid((uint32_t)((a.N + 16 * NC - 1) / (16 * NC)));  // (2^17 at the most)
        if (vec) hipLaunchKernelGGL((lora_few_k<T, NC, 8, true>), grid, dim3(512), 0, s, a);
        else hipLaunchKernelGGL((lora_few_k<T, NC, 8, false>), grid, dim3(512), 0, s, a);
        return check_launch("lora_few_k");
    }
    if (by_segment) {
        if (int e = launch_low<T, true, true>(a, s)) return e;
        return launch_tiles<T, true, kAdapters>(a, s);
    }
    if (int e = vec ? launch_low<T, true, false>(a, s) : launch_low<T, false, false>(a, s)) return e;
    if (few_outputs(a.P, a.N))
        return vec ? launch_grouped_rows<T, 1, 4, 8, true, kRowAdapters>(a, s) : launch_grouped_rows<T, 1, 4, 4, false, kRowAdapters>(a, s);
    return vec ? launch_tiles<T, true, kRowAdapters>(a, s) : launch_tiles<T, false, kRowAdapters>(a, s);
}

}  // namespace pmg
