// Entry points of the grouped products: argument checks, and the choice of the adapters' form.
#include "pmg_grouped.h"

using namespace pmg;

namespace {

int type_bytes(int t) { return t == PMG_TYPE_F32 ? 4 : 2; }
bool at(const void* v, int n) { return (reinterpret_cast<uintptr_t>(v) & (uintptr_t)(n - 1)) == 0; }
size_t up256(size_t n) { return (n + 255) / 256 * 256; }

// What both entries ask of x, w, residual and result; fills in the rest of `a`.
int products(GroupArgs& a, int type, const void* x, int64_t ldx, int K, int N, int act, const void* residual, int residual_type,
             int64_t ldr, void* out, int out_type, int64_t ldo) {
    PMG_REQUIRE(type >= PMG_TYPE_F32 && type <= PMG_TYPE_BF16, "type must be f32, f16 or bf16");
    PMG_REQUIRE(out_type >= PMG_TYPE_F32 && out_type <= PMG_TYPE_BF16, "out_type must be f32, f16 or bf16");
    PMG_REQUIRE(act >= PMG_ACT_NONE && act <= PMG_ACT_GELU_TANH, "unknown activation");
    PMG_REQUIRE(K >= 1 && K <= 131072 && N >= 1 && N <= (1 << 22), "K must be 1 .. 131072 and N 1 .. 2^22");
    const int es = type_bytes(type);
    PMG_REQUIRE(ldx >= K && ldx <= (1 << 22) / es && ldo >= N && (!residual || ldr >= N), "row strides must cover the row (x: at most 4 MiB)");
    PMG_REQUIRE(at(x, es) && at(out, type_bytes(out_type)), "buffers must be aligned to their elements");
    a.x = x;
    a.ldx = ldx;
    a.K = K;
    a.N = N;
    a.act = act;
    a.res = residual;
    a.res_type = residual_type;
    a.ldr = ldr;
    a.out = out;
    a.out_type = out_type;
    a.ldo = ldo;
    if (residual) {
        PMG_REQUIRE(residual_type >= PMG_TYPE_F32 && residual_type <= PMG_TYPE_BF16, "residual_type must be f32, f16 or bf16");
        PMG_REQUIRE(at(residual, type_bytes(residual_type)), "buffers must be aligned to their elements");
        a.vec_res = at(residual, 16) && ldr * type_bytes(residual_type) % 16 == 0;
    }
    a.vec_out = at(out, 16) && ldo * type_bytes(out_type) % 16 == 0;
    return PMG_OK;
}

// The low products' form: more k of 16-byte parts, in tiles that start where a segment starts, where parts and whole tiles allow it and
// the rows that tiles of 64 hold (segments fill them by mean / 64) cost less than 80 products a rank and row in the epilogue,
// which the row form takes as long as. Measured, bf16, row form and segment form, us: 33 segments of 8 rows, K = 1024 to 4096,
// rank 16: 24 and 38; of 40 rows: 46 and 42; K = 512 to 1024, rank 64: 42 and 17; 130 of 4 rows, 1024 to 1024, rank 16: 17 and 33; 130
// of 40: 47 and 39.
bool by_segment(const pmg_lora_linear_args& q) {
    const int es = type_bytes(q.type);
    if (!q.offsets || q.segments < 1 || !(at(q.x, 16) && at(q.w, 16) && at(q.down, 16) && at(q.up, 16))) return false;
    if (q.ldx * es % 16 != 0 || (int64_t)q.K * es % 16 != 0 || q.rank * es % 16 != 0) return false;
    const double held = (double)q.segments * 64.0 * __builtin_ceil((double)q.M / 64.0 / (double)q.segments);
    return held * q.K <= (double)q.M * (q.K + 80.0 * q.rank);
}
// Up to eight rows of an adapter each are done in one launch, without a workspace, where their ranks add up to 64 at most: one row of
// 1024 bf16 to 1024, rank 8, 7.2 us for 8.6 in two, 8 rows 10.9 for 9.1, but 8.2 and 12 for 12.8 a call from Python; 33 rows 13.5 for 9.6.
bool few_rows(const pmg_lora_linear_args& q) { return !q.offsets && q.M <= kFew && q.rank <= 16 && q.M * q.rank <= 64; }
int parts_of(int type) { return type == PMG_TYPE_F32 ? kParts<float> : type == PMG_TYPE_F16 ? kParts<_Float16> : kParts<__bf16>; }
size_t low_bytes(const pmg_lora_linear_args& q) {
    return up256((size_t)q.M * (size_t)q.rank * (by_segment(q) ? (size_t)(parts_of(q.type) * type_bytes(q.type)) : sizeof(float)));
}

int lora_args(const pmg_lora_linear_args& q, GroupArgs& a) {
    if (int e = products(a, q.type, q.x, q.ldx, q.K, q.N, q.act, q.residual, q.residual_type, q.ldr, q.out, q.out_type, q.ldo)) return e;
    PMG_REQUIRE(q.M >= 0 && q.M < ((int64_t)1 << 31) - 512, "M out of range");
    PMG_REQUIRE(q.rank >= 1 && q.rank <= 128, "rank must be 1 .. 128");
    PMG_REQUIRE(q.adapters >= 0 && q.segments >= 0 && q.segments < (int64_t)1 << 31, "adapters or segments out of range");
    PMG_REQUIRE(q.offsets || q.segments == q.M, "without offsets every row is a segment");
    return PMG_OK;
}

// Checks the call and fills in `a` (P stays 0 where there is nothing to do); vec: rows are read 16 bytes at a time.
int grouped_args(const pmg_grouped_linear_args& q, GroupArgs& a, bool& vec) {
    if (int e = products(a, q.type, q.x, q.ldx, q.K, q.N, q.act, q.residual, q.residual_type, q.ldr, q.out, q.out_type, q.ldo)) return e;
    const int64_t big = ((int64_t)1 << 31) - 512;
    PMG_REQUIRE(q.positions >= 0 && q.positions < big && q.x_rows >= 0 && q.x_rows < big && q.out_rows >= 0 && q.out_rows < big, "positions or rows out of range");
    PMG_REQUIRE(q.segments >= 0 && q.segments < (int64_t)1 << 24, "segments out of range");
    PMG_REQUIRE(q.index || q.positions <= q.x_rows, "more positions than rows of x");
    PMG_REQUIRE(q.out_index || q.positions <= q.out_rows, "more positions than rows of the result");
    PMG_REQUIRE(!q.zero_rest || !q.out_index, "zero_rest goes without out_index");
    if (q.positions == 0) return PMG_OK;
    PMG_REQUIRE(q.out && q.offsets && (q.x || q.x_rows == 0) && (q.w || q.segments == 0), "null buffer");
    const int es = type_bytes(q.type);
    PMG_REQUIRE(at(q.w, es) && at(q.bias, 4) && at(q.offsets, 8) && at(q.index, 4) && at(q.out_index, 4), "buffers must be aligned to their elements");
    a.w = q.w;
    a.bias = q.bias;
    a.offsets = q.offsets;
    a.index = q.index;
    a.out_index = q.out_index;
    a.x_rows = q.x_rows;
    a.out_rows = q.out_rows;
    a.S = q.x_rows > 0 ? q.segments : 0;  // (no row of x: no position is in a segment, nothing is read)
    a.w_next = (int64_t)q.N * q.K;
    a.b_next = q.N;
    a.P = (int)q.positions;
    a.fresh = q.zero_rest;
    vec = at(q.x, 16) && at(q.w, 16) && q.ldx * es % 16 == 0 && (int64_t)q.K * es % 16 == 0 &&
          (!q.index || ((q.x_rows - 1) * q.ldx + q.K) * es < 0x7ffffff0);
    return PMG_OK;
}
bool lora_vec(const pmg_lora_linear_args& q) {
    const int es = type_bytes(q.type);
    return at(q.x, 16) && at(q.w, 16) && at(q.down, 16) && q.ldx * es % 16 == 0 && (int64_t)q.K * es % 16 == 0;
}

int set_form(int* form, int kind, int rows, int cols, int places, bool vec) {
    const int f[5] = {kind, rows, cols, places, vec};
    for (int i = 0; i < 5; ++i) form[i] = f[i];
    return PMG_OK;
}
int set_tile(int* form, int type, int kind, bool vec, int64_t P, int64_t S, int K, int N) {
    const bool fp32 = type == PMG_TYPE_F32;
    const int i = tile_shape(fp32, vec, kind, P, S, K, N);
    const int* p = fp32 ? kShapes32[i] : kShapes16[i];
    return set_form(form, kind, p[0], p[1], vec ? p[2] : 1, vec);
}

}  // namespace

extern "C" int pmg_debug_grouped_form(const pmg_grouped_linear_args* p, int* form) {
    PMG_REQUIRE(p && form, "null args");
    GroupArgs a{};
    bool vec = false;
    if (int e = grouped_args(*p, a, vec)) return e;
    if (few_a_segment(a.P, a.S)) return set_form(form, kExperts, 16, vec ? 32 : 16, 0, vec);
    return set_tile(form, p->type, kExperts, vec, a.P, a.S, a.K, a.N);
}

extern "C" int pmg_debug_lora_form(const pmg_lora_linear_args* p, int* form) {
    PMG_REQUIRE(p && form, "null args");
    const pmg_lora_linear_args& q = *p;
    GroupArgs a{};
    if (int e = lora_args(q, a)) return e;
    const bool vec = lora_vec(q);
    if (few_rows(q)) return set_form(form, kFewRows, kFew, 32, 0, vec);
    if (by_segment(q)) return set_tile(form, q.type, kAdapters, true, q.M, q.segments, q.K, q.N);
    if (few_outputs(q.M, q.N)) return set_form(form, kRowAdapters, 16, 16, 0, vec);
    return set_tile(form, q.type, kRowAdapters, vec, q.M, q.segments, q.K, q.N);
}

extern "C" int pmg_grouped_linear(const pmg_grouped_linear_args* p, void* stream) {
    PMG_REQUIRE(p, "null args");
    const pmg_grouped_linear_args& q = *p;
    GroupArgs a{};
    bool vec = false;
    if (int e = grouped_args(q, a, vec)) return e;
    if (a.P == 0) return PMG_OK;
    hipStream_t s = (hipStream_t)stream;
    if (q.type == PMG_TYPE_F32) return launch_experts<float>(a, vec, s);
    if (q.type == PMG_TYPE_F16) return launch_experts<_Float16>(a, vec, s);
    return launch_experts<__bf16>(a, vec, s);
}

extern "C" size_t pmg_lora_linear_workspace_bytes(const pmg_lora_linear_args* p) {
    GroupArgs a{};
    if (!p || lora_args(*p, a) != PMG_OK || p->M == 0 || few_rows(*p)) return 0;
    return low_bytes(*p) + up256((size_t)p->M * 4);
}

extern "C" int pmg_lora_linear(const pmg_lora_linear_args* p, void* workspace, size_t workspace_bytes, void* stream) {
    PMG_REQUIRE(p, "null args");
    const pmg_lora_linear_args& q = *p;
    GroupArgs a{};
    if (int e = lora_args(q, a)) return e;
    if (q.M == 0) return PMG_OK;
    PMG_REQUIRE(q.x && q.w && q.out, "null buffer");
    PMG_REQUIRE(q.segments == 0 || q.adapter, "null buffer");
    PMG_REQUIRE(q.adapters == 0 || (q.down && q.up), "null buffer");
    const int es = type_bytes(q.type);
    PMG_REQUIRE(at(q.w, es) && at(q.down, es) && at(q.up, es) && at(q.bias, 4) && at(q.scale, 4) && at(q.adapter, 4) && at(q.offsets, 8), "buffers must be aligned to their elements");
    const bool few = few_rows(q);
    PMG_REQUIRE(few || (workspace && aligned16(workspace) && workspace_bytes >= pmg_lora_linear_workspace_bytes(p)), "workspace too small, null or not 16-byte aligned");
    const size_t low = few ? 0 : low_bytes(q);
    a.w = q.w;
    a.bias = q.bias;
    a.offsets = q.offsets;
    a.x_rows = a.out_rows = q.M;
    a.S = q.segments;
    a.P = (int)q.M;
    if (!few) {
        a.low = workspace;
        a.low_factor = (float*)((char*)workspace + low);
        a.row_adapter = (int32_t*)((char*)workspace + low);
    }
    a.down = q.down;
    a.up = q.up;
    a.scale = q.scale;
    a.tag = q.adapter;
    a.r = q.rank;
    a.adapters = q.adapters;
    a.vec_up = at(q.up, 16) && q.rank * es % 16 == 0;
    const bool vec = lora_vec(q);
    const bool seg = by_segment(q);
    hipStream_t s = (hipStream_t)stream;
    if (q.type == PMG_TYPE_F32) return launch_lora<float>(a, vec, seg, s);
    if (q.type == PMG_TYPE_F16) return launch_lora<_Float16>(a, vec, seg, s);
    return launch_lora<__bf16>(a, vec, seg, s);
}
