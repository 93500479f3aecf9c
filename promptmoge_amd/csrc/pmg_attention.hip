// Entry points of the attention inside segments: argument checks, and the choice of the kernel's form.
#include "pmg_attention.h"

using namespace pmg;

namespace {

struct Plan {
    int seg, whole, splits;
};

size_t parts_bytes(const pmg_attention_args& r, const Plan& p) {
    return p.splits <= 1 ? 0 : (size_t)p.splits * (size_t)r.q_positions * (size_t)r.Hq * ((size_t)r.D * 4 + 8);
}

// The forms, by the mean lengths (the offsets are on the device).
//
// A block per segment (seg) where the queries of a segment fill no half wave and its keys are many, the keys split so that
// about 2048 waves (8 a CU) read them.
//
// Else tiles of 128 slots, from each segment's start on (whole) where segments have more than 160 slots, else through all
// segments: a tile of two segments goes over the keys of both. Measured (MI355X, 40,000 rows, 8 heads of 64, bf16, segments of
// about L rows; through all against whole): L = 32: 46 and 78 us, 64: 48 and 54, 100: 53 and 48, 128: 54 and 57, 192: 60 and
// 53, 512: 97 and 76, 2048: 262 and 222; 4 frames of 2745 rows: 168 and 102.
//
// Tiles' keys are split where the tiles would lie unevenly on the CUs, or too few on each to hide what they wait for. 19200
// rows in one segment, 4 heads of 64 (600 tiles), 1 .. 6 parts: 617, 558, 534, 521, 502, 519 us; 4 frames of 2745 rows, 8
// heads (688 tiles): 102, 119, 122, 120, 131, 140.
Plan plan_of(const pmg_attention_args& r) {
    Plan p{0, 0, 1};
    if (r.segments < 1) return p;
    const double G = (double)(r.Hq / r.Hk);
    const double nq = (double)r.q_positions / (double)r.segments, nk = (double)r.k_positions / (double)r.segments;
    p.seg = nq * G <= 16.0 && nk >= 128.0;
    if (p.seg) {
        const int64_t s = 2048 / (r.segments * r.Hk), most = (int64_t)(nk / 256.0);
        p.splits = (int)(s < most ? s : most);
        p.splits = p.splits < 1 ? 1 : p.splits > 256 ? 256 : p.splits;
        return p;
    }
    p.whole = nq * G > 160.0;
    const int64_t slots = r.q_positions * (r.Hq / r.Hk);
    const int64_t blocks = (p.whole ? slots / 128 + r.segments + 2 : (slots + 127) / 128) * r.Hk;
    // Microseconds, as measured: 64 keys of a tile at a CU's full throughput; a block's start; the share of that
    // throughput that 1 .. 4 blocks on a CU reach; a part's O written and read.
    // (a tile's keys: segments with an index are taken for pool cells, which are ragged. Cells of 16, 24 and 32 voxels of depth maps
    // of 61 x 83 to 480 x 640: their rows lie in cells of 1.1 to 1.6 times the mean length, the longest has 1.2 to 2.7 times,
    // whose tiles are at work last and alone. Rows in order are taken for frames of about one length: 12 of 800 rows, 4 heads
    // of 128, in one part 39 us, in two 54, as ragged ones would be; 8 of 300, 4 heads of 64, biased: 1 .. 4 parts 17.7, 17.5,
    // 17.6, 18.1. A block alone on its CU reaches half of the throughput; fp32 without bias or cap, bound by the matrix
    // units, 0.9 of it: 8 frames of 600, 4 heads of 64: 1 .. 5 parts 56, 60, 62, 51, 60)
    const bool ragged = r.q_index != nullptr;
    const double keys = (ragged ? 1.5 : 1.0) * nk * (p.whole || nq <= 0.0 ? 1.0 : 1.0 + 128.0 / G / nq);
    const bool f32 = r.type == PMG_TYPE_F32;
    const double tile = (f32 ? 0.07 * (r.D <= 32 ? 32 : r.D <= 64 ? 64 : 128) : r.D <= 32 ? 0.52 : r.D <= 64 ? 0.66 : 1.37) + (r.slopes ? 0.3 : 0.0);
    const double reach[5] = {1.0, 0.5, 0.81, 0.91, 1.0};
    const int resident = f32 || r.D > 64 ? 2 : r.slopes && r.D > 32 ? 3 : 4;
    const double part = (double)r.q_positions * (double)r.Hq * (double)r.D * 8.0 / 8.0e6;
    double best = 0.0;
    for (int s = 1; s <= 64 && s <= (int)(keys / 128.0) + 1; ++s) {
        const int64_t each = (blocks * s + 255) / 256, rem = each % resident;  // a CU's blocks; those that do not fill it
        const double slow = rem == 0 || f32 ? 1.0 : reach[resident] / reach[rem];
        const double rounds = (double)(each - rem) + (double)rem * (each < resident ? slow : 0.5 + 0.5 * slow);
        const double alone = (ragged ? 2.5 : 1.0) * nk / 64.0 * tile / s / (f32 && !r.slopes && r.cap == 0.0f ? 0.9 : 0.5) + 1.5;
        const double all = rounds * (keys / 64.0 * tile / s + 1.5);
        const double t = (all > alone ? all : alone) + (s > 1 ? 6.0 + s * part : 0.0);
        if (s > 1 && parts_bytes(r, Plan{0, 0, s}) > (size_t)1 << 28) break;  // (256 MB of parts at most)
        if (s == 1 || t < 0.98 * best) {
            best = t;
            p.splits = s;
        }
    }
    return p;
}

int attention_args(const pmg_attention_args& r) {
    PMG_REQUIRE(r.type >= PMG_TYPE_F32 && r.type <= PMG_TYPE_BF16, "type must be f32, f16 or bf16");
    PMG_REQUIRE(r.Hq >= 1 && r.Hk >= 1 && r.Hq <= 4096 && r.Hq % r.Hk == 0, "query heads must be a multiple of key heads (up to 4096)");
    PMG_REQUIRE(r.D >= 8 && r.D <= 128 && r.D % 8 == 0, "head width must be a multiple of 8 up to 128");
    PMG_REQUIRE(r.q_rows >= 0 && r.k_rows >= 0 && r.q_positions >= 0 && r.k_positions >= 0 && r.segments >= 0, "negative size");
    const int64_t big = ((int64_t)1 << 31) - 64;  // (a tile behind the last key still counts in 32 bits)
    PMG_REQUIRE(r.q_rows < big && r.k_rows < big && r.q_positions < big && r.k_positions < big && r.segments < big, "2^31 - 64 rows, positions or segments");
    PMG_REQUIRE(r.q_index || r.q_positions <= r.q_rows, "more query positions than rows");
    PMG_REQUIRE(r.k_index || r.k_positions <= r.k_rows, "more key positions than rows");
    PMG_REQUIRE(r.scale > 0.0f && r.scale <= 1.0e30f, "scale must be positive, up to 1e30");
    PMG_REQUIRE(r.cap >= 0.0f && r.cap <= 1.0e30f, "cap must not be negative, nor above 1e30");
    PMG_REQUIRE(r.cap == 0.0f || (double)r.scale / (double)r.cap <= 1.0e37, "cap is too small for the scale");
    return PMG_OK;
}

}  // namespace

extern "C" size_t pmg_attention_workspace_bytes(const pmg_attention_args* p) {
    if (!p || attention_args(*p) != PMG_OK) return 0;
    return parts_bytes(*p, plan_of(*p));
}

extern "C" int pmg_attention(const pmg_attention_args* p, void* workspace, size_t workspace_bytes, void* stream) {
    PMG_REQUIRE(p, "null args");
    const pmg_attention_args& r = *p;
    if (int e = attention_args(r)) return e;
    if (r.q_rows == 0 || (r.q_positions == 0 && !r.zero_rest)) return PMG_OK;
    PMG_REQUIRE(r.out && (r.q_positions == 0 || (r.q && r.q_offsets && r.k_offsets)), "null buffer");
    PMG_REQUIRE(r.k_rows == 0 || r.k_positions == 0 || (r.k && r.v), "null buffer");
    PMG_REQUIRE(!r.slopes || (r.q_coords && (r.k_coords || r.k_rows == 0)), "slopes need coordinates");
    const int es = r.type == PMG_TYPE_F32 ? 4 : 2;
    auto ok = [&](const void* b, int64_t row, int64_t head, int n) {
        return (reinterpret_cast<uintptr_t>(b) & (uintptr_t)(n * es - 1)) == 0 && row % n == 0 && head % n == 0;
    };
    const int per = 16 / es;
    PMG_REQUIRE(ok(r.q, r.q_row, r.q_head, per) && ok(r.k, r.k_row, r.k_head, per) && ok(r.v, r.v_row, r.v_head, per), "q, k, v: buffers and strides in whole 16 bytes");
    PMG_REQUIRE(r.k_row >= 0 && r.v_row >= 0 && r.k_row < ((int64_t)1 << 31) / es && r.v_row < ((int64_t)1 << 31) / es, "k, v: rows further than 2 GiB apart");
    PMG_REQUIRE(ok(r.out, r.out_row, r.out_head, 4), "out: buffer and strides in whole groups of 4 elements");
    PMG_REQUIRE(!r.slopes || (aligned16(r.q_coords) && aligned16(r.k_coords)), "coordinates must be 16-byte aligned");
    const Plan pl = plan_of(r);
    const size_t need = parts_bytes(r, pl);
    PMG_REQUIRE(need == 0 || (workspace && workspace_bytes >= need && aligned16(workspace)), "workspace too small, null or not 16-byte aligned");
    AttnArgs a{};
    a.q = r.q;
    a.k = r.k;
    a.v = r.v;
    a.out = r.out;
    a.q_row = r.q_row;
    a.q_head = r.q_head;
    a.k_row = r.k_row;
    a.k_head = r.k_head;
    a.v_row = r.v_row;
    a.v_head = r.v_head;
    a.o_row = r.out_row;
    a.o_head = r.out_head;
    a.Mq = r.q_rows;
    a.Mk = r.k_rows;
    a.Pq = r.q_positions;
    a.Pk = r.k_rows > 0 ? r.k_positions : 0;
    a.S = r.segments;
    a.q_off = r.q_offsets;
    a.k_off = r.k_offsets;
    a.q_index = r.q_index;
    a.k_index = r.k_index;
    a.q_coords = r.q_coords;
    a.k_coords = r.k_coords;
    a.slopes = r.slopes;
    a.k_mask = r.k_mask;
    a.Hq = r.Hq;
    a.Hk = r.Hk;
    a.G = r.Hq / r.Hk;
    a.D = r.D;
    const double log2e = 1.4426950408889634;
    a.scale2 = (float)((double)r.scale * log2e);
    a.fine = r.type == PMG_TYPE_F32 || r.precise;
    if (r.cap > 0.0f) {
        a.cap2 = (float)((double)r.cap * log2e);
        if (a.cap2 > kFineCap) a.fine = 1;
        a.cap_arg = (float)((double)r.scale / (double)r.cap * (a.fine ? 1.0 : 2.0 * log2e));
    }
    a.seg = pl.seg;
    a.whole = pl.whole;
    a.splits = pl.splits;
    a.zero_rest = r.zero_rest;
    const int64_t end = (a.Mk - 1) * (r.k_row > r.v_row ? r.k_row : r.v_row) * es + (int64_t)r.D * es;
    a.near = (r.D == 32 || r.D == 64 || r.D == 128) && end <= 0xffff0000;
    if (need) {
        a.part_o = (float*)workspace;
        a.part_ml = (float2*)((char*)workspace + (size_t)pl.splits * (size_t)r.q_positions * (size_t)r.Hq * (size_t)r.D * 4);
    }
    hipStream_t s = (hipStream_t)stream;
    if (r.type == PMG_TYPE_F32) return launch_attention_f32(a, s);
    if (r.type == PMG_TYPE_F16) return launch_attention_f16(a, s);
    return launch_attention_bf16(a, s);
}
