// Segments of positions, found by the blocks themselves (the offsets are on the device).
#pragma once
#include "pmg_common.h"

namespace pmg {

// Positions [0, P) fall into S + 2 pieces: those in front of segment 0, the segments, those behind the last. Tiles of `rows`
// positions start where a piece starts; piece j's have the numbers bound(j) / rows + j and up, so that a tile's piece is found
// without a sum over the pieces (a piece may have a number more than it has tiles): P / rows + S + 2 in all.
struct Pieces {
    const int64_t* offsets;  // [S + 1], or NULL: one segment of all positions (S = 1)
    int64_t S;
    int P;
    const int32_t* tag;      // [S], or NULL: a number of each segment, looked up with its bounds
    __device__ inline int bound(int64_t j) const {
        if (j <= 0) return 0;
        if (j > S + 1) return P;
        if (!offsets) return j == 1 ? 0 : P;
        const int64_t o = offsets[j - 1];
        return o < 0 ? 0 : o > P ? P : (int)o;
    }
};
inline uint32_t piece_tiles(int64_t P, int64_t S, int rows) { return (uint32_t)(P / rows + S + 2); }

struct Piece {
    int first, n;  // positions first .. first + n - 1 (n < 1: none)
    int s;         // of segment s (-1: of none)
    int p0, p1;    // which holds p0 .. p1 - 1
    uint32_t id0;  // and whose tiles have the numbers from id0 on
    int tag;       // the segment's (-1: none)
};
// The positions of tile `id`; all lanes of a wave return the same. A wave looks at 64 pieces at a time. Where offsets fall, some tile
// within [0, P).
__device__ inline Piece piece_of(const Pieces& a, uint32_t id, int rows) {
    const int lane = threadIdx.x & 63;
    int64_t lo = 0, n = a.S + 2;
    int here = 0, tag = -1;  // the lane's piece's bound and tag, in the last round
    int64_t cnt = 0;
    for (;;) {
        const int64_t step = (n + 63) >> 6, c = lo + lane * step;
        here = a.bound(c);
        if (a.tag && c >= 1 && c <= a.S) tag = a.tag[c - 1];
        const bool in = lane * step < n && (int64_t)((uint32_t)here / (uint32_t)rows) + c <= (int64_t)id;
        const uint64_t not_in = ~__ballot(in);
        cnt = not_in ? __builtin_ctzll(not_in) : 64;
        cnt = cnt < 1 ? 0 : cnt - 1;
        lo += cnt * step;
        if (step == 1) break;
        n = n - cnt * step < step ? n - cnt * step : step;
    }
    const int at = __builtin_amdgcn_readfirstlane((int)cnt);
    Piece p;
    p.p0 = __builtin_amdgcn_readlane(here, at);
    p.p1 = __builtin_amdgcn_readfirstlane(at < 63 ? __builtin_amdgcn_readlane(here, (at + 1) & 63) : a.bound(lo + 1));
    p.s = __builtin_amdgcn_readfirstlane(lo >= 1 && lo <= a.S ? (int)(lo - 1) : -1);
    p.tag = p.s < 0 ? -1 : __builtin_amdgcn_readlane(tag, at);
    p.id0 = __builtin_amdgcn_readfirstlane((uint32_t)p.p0 / (uint32_t)rows + (uint32_t)lo);
    const int64_t first = p.p0 + (int64_t)(id - p.id0) * rows;
    const bool there = first >= p.p0 && first < p.p1;
    p.n = __builtin_amdgcn_readfirstlane(!there ? 0 : p.p1 - first < rows ? (int)(p.p1 - first) : rows);
    p.first = __builtin_amdgcn_readfirstlane(there ? (int)first : 0);
    return p;
}

// Pieces counted, L a lane (S + 2 <= 64 L): their tiles numbered without gaps, so that the blocks that have one come first and lie
// evenly on the chip. ends: the pieces in front of the segments and behind them have tiles too. Where offsets fall, a tile within
// [0, P) or none. (The blocks of short tiles feel four a lane: 153,600 positions of 256 fp16 to 128 take 25.6 us with one, 27.7
// with four, 26.4 numbered with gaps.)
template <int L>
struct PieceCount {
    int here[L + 1], tag[L];  // the lane's pieces' bounds and tags
    uint32_t tiles[L];        // and tiles
    uint32_t upto;            // all tiles up to the lane's last
    uint32_t total;
    __device__ inline PieceCount(const Pieces& a, int rows, bool ends) {
        const int j = L * (threadIdx.x & 63);
#pragma unroll
        for (int i = 0; i <= L; ++i) here[i] = a.bound(j + i);
#pragma unroll
        for (int i = 0; i < L; ++i) tag[i] = a.tag && j + i >= 1 && j + i <= a.S ? a.tag[j + i - 1] : -1;
        uint32_t sum = 0;
#pragma unroll
        for (int i = 0; i < L; ++i) {
            const int n = here[i + 1] - here[i];
            const bool none = n < 1 || (!ends && (j + i == 0 || j + i == a.S + 1));
            tiles[i] = none ? 0u : ((uint32_t)n + (uint32_t)rows - 1u) / (uint32_t)rows;
            sum += tiles[i];
        }
        upto = wave_incl_scan_u32(sum);
        total = __builtin_amdgcn_readlane(upto, 63);
    }
    __device__ inline Piece at(const Pieces& a, uint32_t id, int rows) const {
        const uint64_t from = __ballot(upto > id);
        const int lane = from ? __builtin_ctzll(from) : 63;
        uint32_t behind = __builtin_amdgcn_readlane(upto, lane);
        Piece p{};
#pragma unroll
        for (int i = L - 1; i >= 0; --i) {  // the lane's first piece that ends behind id
            const bool takes = L == 1 || behind > id;
            behind -= __builtin_amdgcn_readlane(tiles[i], lane);
            if (takes) {
                p.p0 = __builtin_amdgcn_readlane(here[i], lane);
                p.p1 = __builtin_amdgcn_readlane(here[i + 1], lane);
                p.tag = __builtin_amdgcn_readlane(tag[i], lane);
                p.s = L * lane + i - 1;
                p.id0 = behind;
            }
        }
        if (p.s >= a.S) p.s = -1;
        const int64_t first = p.p0 + (int64_t)(id - p.id0) * rows;
        const bool there = first < p.p1;
        p.n = !there ? 0 : p.p1 - first < rows ? (int)(p.p1 - first) : rows;
        p.first = there ? (int)first : 0;
        return p;
    }
};

}  // namespace pmg
