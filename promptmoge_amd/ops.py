"""Torch-facing wrappers of the libpmg entry points.

Tensors are device tensors (HIP); every call enqueues on torch's current stream and returns without synchronising.
Inputs are validated here (device, dtype, shape, contiguity) before the C ABI validates them again.
"""
from __future__ import annotations

import ctypes as C
from typing import NamedTuple, Optional, Sequence, Tuple

import torch
from torch.autograd import forward_ad

from . import _lib
from ._lib import EPI_ACC, EPI_BIAS, EPI_Q, EPI_QLIN, EPI_R, EPI_RLN, EPI_ROUT, EPI_SILU, ConvEpilogue, call, check, lib

__all__ = [
    "voxelize", "nmap_column", "nmap_hash", "row_order", "nmap_from_rows", "kmap_compact", "spconv_i8",
    "spconv_i8_ordered", "spconv_f16", "spconv_bf16",
    "spconv_f32", "spconv_col", "ln_silu_quant", "ln_silu_f16", "fit_scale_shift", "fit_prompt", "fit_final",
    "post_depth",
    "math_device", "gauge_poly",
    "nearest_fill",
    "linear", "linear_i8", "qk_norm_rope", "sparse_attention",
    "group_norm", "route", "Routes", "grouped_linear", "combine", "lora_linear",
    "EPI_ACC", "EPI_Q", "EPI_R", "EPI_BIAS", "EPI_SILU", "EPI_RLN", "EPI_ROUT", "EPI_QLIN",
]


def _stream() -> C.c_void_p:
    return C.c_void_p(torch.cuda.current_stream().cuda_stream)


def _p(t: Optional[torch.Tensor]) -> Optional[int]:
    return None if t is None else t.data_ptr()


def _dev(t: torch.Tensor, name: str, dtype: Optional[torch.dtype] = None) -> torch.Tensor:
    if not isinstance(t, torch.Tensor) or not t.is_cuda:
        raise ValueError(f"{name} must be a GPU tensor")
    if dtype is not None and t.dtype != dtype:
        raise ValueError(f"{name} must be {dtype}, got {t.dtype}")
    if not t.is_contiguous():
        raise ValueError(f"{name} must be contiguous")
    return t


def math_device(op: int, x: torch.Tensor) -> torch.Tensor:
    """Test hook: op 0/1/2 = exp/log/silu of x; op 3 = the epilogues' int8 SiLU code of x[:, 0] at mult x[:, 1]."""
    x = _dev(x, "x", torch.float32)
    if op == 3:
        if x.ndim != 2 or x.shape[1] != 2:
            raise ValueError("op 3 takes (n, 2) pairs (y, mult)")
        out = torch.empty((x.shape[0],), dtype=torch.float32, device=x.device)
        n = x.shape[0]
    else:
        out = torch.empty_like(x)
        n = x.numel()
    call("pmg_math_device", op, _p(x), _p(out), n, _stream())
    return out


# ------------------------------------------------------------------------------------------------------------- (1)
def voxelize(logz: torch.Tensor, resolution: float = 256.0, stride: int = 1,
             shape: Optional[Tuple[int, int, int]] = None):
    """zq = rint(logz * resolution) and per-batch (min, max). logz: [B, H, W] (stride 1) or the point map
    [B, H, W, 3] viewed from its third channel (pass points[..., 2:] with stride 3 and shape=(B, H, W))."""
    if shape is None:
        B, H, W = logz.shape
    else:
        B, H, W = shape
    dev = logz.device
    zq = torch.empty((B, H, W), dtype=torch.int32, device=dev)
    zmin = torch.empty((B,), dtype=torch.int32, device=dev)
    zmax = torch.empty((B,), dtype=torch.int32, device=dev)
    call("pmg_voxelize", _p(logz), stride, B, H, W, float(resolution), _p(zq), _p(zmin), _p(zmax), _stream())
    return zq, zmin, zmax


# ------------------------------------------------------------------------------------------------------------- (2)
def nmap_column(zq: torch.Tensor, zmin: Optional[torch.Tensor] = None, *, taps: bool = True, rows: bool = False,
                coords: bool = False):
    """Level-0 column-stencil map. Returns (nmap_t [27, M] | None, tile_mask [ceil(M/16)], nmap_rows [M, 27] | None,
    coords [M, 4] | None)."""
    zq = _dev(zq, "zq", torch.int32)
    B, H, W = zq.shape
    M = B * H * W
    dev = zq.device
    nt = torch.empty((27, M), dtype=torch.int32, device=dev) if taps else None
    nr = torch.empty((M, 27), dtype=torch.int32, device=dev) if rows else None
    tm = torch.empty(((M + 15) // 16,), dtype=torch.int32, device=dev)
    cd = torch.empty((M, 4), dtype=torch.int32, device=dev) if coords else None
    if coords and zmin is None:
        raise ValueError("coords need zmin")
    call("pmg_nmap_column", _p(zq), _p(zmin), B, H, W, _p(nt), _p(nr), _p(tm), _p(cd), _stream())
    return nt, tm, nr, cd


def nmap_hash(coords: torch.Tensor, sparse_shape: Sequence[int], *, taps: bool = True, rows: bool = False,
              row_mask: bool = False):
    """Generic map over unique (b, x, y, z) coords. Returns (nmap_t [27, M] | None, tile_mask, nmap_rows | None), and
    with row_mask=True a fourth item, each row's 27-bit tap mask [M] (int32)."""
    coords = _dev(coords, "coords", torch.int32)
    if coords.ndim != 2 or coords.shape[1] != 4:
        raise ValueError("coords must be (M, 4)")
    M = coords.shape[0]
    dev = coords.device
    nt = torch.empty((27, M), dtype=torch.int32, device=dev) if taps else None
    nr = torch.empty((M, 27), dtype=torch.int32, device=dev) if rows else None
    tm = torch.empty(((M + 15) // 16,), dtype=torch.int32, device=dev)
    ws_bytes = lib().pmg_hash_workspace_bytes(M)
    ws = torch.empty((ws_bytes,), dtype=torch.uint8, device=dev)
    rm = torch.empty((M,), dtype=torch.int32, device=dev) if row_mask else None
    shape = (C.c_int64 * 4)(*[int(s) for s in sparse_shape[:4]])
    call("pmg_nmap_hash", _p(coords), M, shape, _p(nt), _p(nr), _p(tm), _p(rm), _p(ws), ws_bytes, _stream())
    return (nt, tm, nr, rm) if row_mask else (nt, tm, nr)


def sorted_workspace(sparse_shape: Sequence[int], device) -> torch.Tensor:
    """A workspace for nmap_sorted: its status word zeroed, the rest uninitialised (reusable by later calls)."""
    shape = (C.c_int64 * 4)(*[int(s) for s in sparse_shape[:4]])
    nbytes = lib().pmg_sorted_workspace_bytes(shape)
    if nbytes == 0:
        raise ValueError("nmap_sorted: more than 2^31 (b, x, y) columns")
    ws = torch.empty((nbytes,), dtype=torch.uint8, device=device)
    ws[:256].zero_()
    return ws


def sorted_workspace_fits(sparse_shape: Sequence[int]) -> bool:
    """Whether nmap_sorted takes this sparse shape (at most 2^31 (b, x, y) columns)."""
    shape = (C.c_int64 * 4)(*[int(s) for s in sparse_shape[:4]])
    return lib().pmg_sorted_workspace_bytes(shape) > 0


def sorted_status(ws: torch.Tensor) -> int:
    """The status word of an nmap_sorted workspace (reads it back): 0 while every call saw sorted coordinates."""
    return int(ws[:4].view(torch.int32).item())


def nmap_sorted(coords: torch.Tensor, sparse_shape: Sequence[int], *, taps: bool = True, rows: bool = False,
                row_mask: bool = False, workspace: Optional[torch.Tensor] = None):
    """nmap_hash for coords in strictly increasing _linearise order (the order _SortedIndex sorts into): the same
    outputs, from the (b, x, y) columns' row runs. The order is checked on the device; `workspace` (sorted_workspace)
    carries the sticky status word, read with sorted_status -- without one, a fresh workspace is checked here (one
    synchronisation) and a violation raises."""
    coords = _dev(coords, "coords", torch.int32)
    if coords.ndim != 2 or coords.shape[1] != 4:
        raise ValueError("coords must be (M, 4)")
    M = coords.shape[0]
    dev = coords.device
    own = workspace is None
    ws = sorted_workspace(sparse_shape, dev) if own else workspace
    nt = torch.empty((27, M), dtype=torch.int32, device=dev) if taps else None
    nr = torch.empty((M, 27), dtype=torch.int32, device=dev) if rows else None
    tm = torch.empty(((M + 15) // 16,), dtype=torch.int32, device=dev)
    rm = torch.empty((M,), dtype=torch.int32, device=dev) if row_mask else None
    shape = (C.c_int64 * 4)(*[int(s) for s in sparse_shape[:4]])
    call("pmg_nmap_sorted", _p(coords), M, shape, _p(nt), _p(nr), _p(tm), _p(rm), _p(ws), ws.numel(), _stream())
    if own and sorted_status(ws) != 0:
        raise ValueError("nmap_sorted: coords are not in increasing _linearise order (or lie outside sparse_shape)")
    return (nt, tm, nr, rm) if row_mask else (nt, tm, nr)


ROW_ORDER_WINDOW = 1 << 18


def row_order(row_mask: torch.Tensor, nmap_rows: Optional[torch.Tensor] = None, window: int = ROW_ORDER_WINDOW):
    """Processing order for spconv_i8_ordered: within windows of `window` consecutive rows (0: one window), rows
    stably sorted by their 27-bit tap mask; the tile masks [ceil(M/16)] of that order and, given the row-major map
    (nmap_hash(rows=True)), the tap-major map in that order (the map spconv_i8_ordered reads).
    Returns (order [M] int32, order_tile_mask, nmap_o [27, M] | None)."""
    row_mask = _dev(row_mask, "row_mask", torch.int32)
    M = row_mask.shape[0]
    dev = row_mask.device
    order = torch.empty((M,), dtype=torch.int32, device=dev)
    otm = torch.empty(((M + 15) // 16,), dtype=torch.int32, device=dev)
    nmo = None
    if nmap_rows is not None:
        nmap_rows = _dev(nmap_rows, "nmap_rows", torch.int32)
        if tuple(nmap_rows.shape) != (M, 27) or not nmap_rows.is_contiguous():
            raise ValueError("nmap_rows must be a contiguous (M, 27) map")
        nmo = torch.empty((27, M), dtype=torch.int32, device=dev)
    ws_bytes = lib().pmg_row_order_workspace_bytes(M)
    ws = torch.empty((max(ws_bytes, 1),), dtype=torch.uint8, device=dev)
    call("pmg_row_order", _p(row_mask), _p(nmap_rows), M, int(window), _p(order), _p(otm), _p(nmo), _p(ws), ws_bytes, _stream())
    return order, otm, nmo


def pool_cache(coords: torch.Tensor, sparse_shape: Sequence[int], stride: Sequence[int],
               out_sparse_shape: Sequence[int]):
    """build_pool_cache (_core.py:339-395), perfect partition, output coordinates not given. Returns
    (out_coords [N, 4] int32, parent [M] int32, seg_indices [M] int32, seg_offsets [N + 1] int64). Reads the
    output count back to the host once (the reference's int(...) sync)."""
    coords = _dev(coords, "coords", torch.int32)
    if coords.ndim != 2 or coords.shape[1] != 4:
        raise ValueError("coords must be (M, 4)")
    M = coords.shape[0]
    dev = coords.device
    oc = torch.empty((max(M, 1), 4), dtype=torch.int32, device=dev)
    parent = torch.empty((M,), dtype=torch.int32, device=dev)
    seg = torch.empty((M,), dtype=torch.int32, device=dev)
    offs = torch.empty((M + 1,), dtype=torch.int64, device=dev)
    counts = torch.empty((2,), dtype=torch.int64, device=dev)
    ws_bytes = lib().pmg_pool_cache_workspace_bytes(M)
    ws = torch.empty((max(ws_bytes, 1),), dtype=torch.uint8, device=dev)
    shp = (C.c_int64 * 4)(*[int(v) for v in sparse_shape[:4]])
    st = (C.c_int32 * 3)(*[int(v) for v in stride[:3]])
    osh = (C.c_int64 * 4)(*[int(v) for v in out_sparse_shape[:4]])
    call("pmg_pool_cache", _p(coords), M, shp, st, osh, _p(oc), _p(parent), _p(seg), _p(offs), _p(counts), _p(ws),
         ws_bytes, _stream())
    n, bad = (int(v) for v in counts.cpu())
    if bad:
        raise ValueError(f"pool_cache: {bad} voxels lie outside the sparse shape {tuple(sparse_shape[:4])}")
    return oc[:n], parent, seg, offs[:n + 1]


def sparse_pool(feats: torch.Tensor, seg_indices: torch.Tensor, seg_offsets: torch.Tensor, num_out: int,
                reduce: str = "mean") -> torch.Tensor:
    """sparse_pool's reduction (_core.py:464-476) over a pool cache: fp32 sums in input order, / group size."""
    if reduce not in ("mean", "sum"):
        raise NotImplementedError(f"reduce={reduce!r} not needed by MoGe")
    feats = _dev(feats, "feats", torch.float32)
    M, Cc = feats.shape
    out = torch.empty((num_out, Cc), dtype=torch.float32, device=feats.device)
    call("pmg_sparse_pool", _p(feats), M, Cc, _p(seg_indices), _p(seg_offsets), num_out, 1 if reduce == "mean" else 0,
         _p(out), _stream())
    return out


def sparse_upsample(feats: torch.Tensor, parent: torch.Tensor) -> torch.Tensor:
    """Nearest upsampling (_core.py:484-505): out[i] = feats[parent[i]]."""
    feats = _dev(feats, "feats")
    parent = _dev(parent, "parent", torch.int32)
    out = torch.empty((parent.shape[0],) + tuple(feats.shape[1:]), dtype=feats.dtype, device=feats.device)
    row_bytes = feats[0].numel() * feats.element_size() if feats.shape[0] else 16
    call("pmg_sparse_upsample", _p(feats), row_bytes, _p(parent), parent.shape[0], _p(out), _stream())
    return out


def nmap_from_rows(nmap_rows: torch.Tensor):
    """(M, 27) map -> (nmap_t [27, M], tile_mask)."""
    nmap_rows = _dev(nmap_rows, "nmap_rows", torch.int32)
    M = nmap_rows.shape[0]
    nt = torch.empty((27, M), dtype=torch.int32, device=nmap_rows.device)
    tm = torch.empty(((M + 15) // 16,), dtype=torch.int32, device=nmap_rows.device)
    call("pmg_nmap_from_rows", _p(nmap_rows), M, _p(nt), _p(tm), _stream())
    return nt, tm


def kmap_compact(nmap_t: torch.Tensor, capacity: Optional[int] = None):
    """Per-tap compacted kernel maps: (offsets [28] int64, out_rows, in_rows). Synchronises the stream."""
    nmap_t = _dev(nmap_t, "nmap_t", torch.int32)
    M = nmap_t.shape[1]
    cap = 27 * M if capacity is None else int(capacity)
    dev = nmap_t.device
    off = torch.empty((28,), dtype=torch.int64, device=dev)
    out_rows = torch.empty((max(cap, 1),), dtype=torch.int32, device=dev)
    in_rows = torch.empty((max(cap, 1),), dtype=torch.int32, device=dev)
    ws_bytes = lib().pmg_kmap_workspace_bytes(M)
    ws = torch.empty((ws_bytes,), dtype=torch.uint8, device=dev)
    call("pmg_kmap_compact", _p(nmap_t), M, _p(off), _p(out_rows), _p(in_rows), cap, _p(ws), ws_bytes, _stream())
    total = int(off[27].item())
    return off, out_rows[:total], in_rows[:total]


# ------------------------------------------------------------------------------------------------------------- (3)
def _conv_out(M: int, Co: int, epilogue: int, elt: str, dev) -> torch.Tensor:
    if elt == "i8":
        dt = {EPI_ACC: torch.int32, EPI_Q: torch.int8, EPI_QLIN: torch.int8}.get(epilogue, torch.float32)
    elif elt == "f16":
        dt = torch.float16 if epilogue == EPI_SILU else torch.float32
    else:
        dt = torch.float32
    return torch.empty((M, Co), dtype=dt, device=dev)


def spconv_i8(x: torch.Tensor, nmap_t: torch.Tensor, tile_mask: torch.Tensor, w: torch.Tensor, epilogue: int = EPI_ACC,
              *, a_scale: float = 1.0, w_scale: Optional[torch.Tensor] = None, bias: Optional[torch.Tensor] = None,
              out_mult: float = 1.0, skip: Optional[torch.Tensor] = None,
              out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """int8 submanifold conv. x: (M, Ci) int8; w: (Co, 3, 3, 3, Ci) or (Co, 27, Ci) int8."""
    x = _dev(x, "x", torch.int8)
    w = _dev(w, "w", torch.int8)
    M, Ci = x.shape
    Co = w.shape[0]
    if w.numel() != Co * 27 * Ci:
        raise ValueError("weight must be (Co, 3, 3, 3, Ci)")
    if out is None:
        out = _conv_out(M, Co, epilogue, "i8", x.device)
    call("pmg_spconv_i8", _p(x), _p(nmap_t), _p(tile_mask), M, Ci, Co, _p(w), epilogue, float(a_scale), _p(w_scale),
         _p(bias), float(out_mult), _p(skip), _p(out), _stream())
    return out


def spconv_i8_ordered(x: torch.Tensor, nmap_o: torch.Tensor, order: torch.Tensor, order_tile_mask: torch.Tensor,
                      w: torch.Tensor, epilogue: int = EPI_ACC, *, a_scale: float = 1.0,
                      w_scale: Optional[torch.Tensor] = None, bias: Optional[torch.Tensor] = None,
                      out_mult: float = 1.0, skip: Optional[torch.Tensor] = None,
                      out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """spconv_i8 with rows processed in `order`, reading the map permuted into that order (row_order's nmap_o):
    identical results, fewer taps per chunk of rows. Ci = Co = 64, 128."""
    x = _dev(x, "x", torch.int8)
    w = _dev(w, "w", torch.int8)
    order = _dev(order, "order", torch.int32)
    M, Ci = x.shape
    Co = w.shape[0]
    if w.numel() != Co * 27 * Ci:
        raise ValueError("weight must be (Co, 3, 3, 3, Ci)")
    if out is None:
        out = _conv_out(M, Co, epilogue, "i8", x.device)
    call("pmg_spconv_i8_ordered", _p(x), _p(nmap_o), _p(order), _p(order_tile_mask), M, Ci, Co, _p(w), epilogue,
         float(a_scale), _p(w_scale), _p(bias), float(out_mult), _p(skip), _p(out), _stream())
    return out


def spconv_f16(x: torch.Tensor, nmap_t: torch.Tensor, tile_mask: torch.Tensor, w: torch.Tensor,
               epilogue: int = EPI_ACC, *, bias: Optional[torch.Tensor] = None, skip: Optional[torch.Tensor] = None,
               out: Optional[torch.Tensor] = None) -> torch.Tensor:
    x = _dev(x, "x", torch.float16)
    w = _dev(w, "w", torch.float16)
    M, Ci = x.shape
    Co = w.shape[0]
    if w.numel() != Co * 27 * Ci:
        raise ValueError("weight must be (Co, 3, 3, 3, Ci)")
    if out is None:
        out = _conv_out(M, Co, epilogue, "f16", x.device)
    call("pmg_spconv_f16", _p(x), _p(nmap_t), _p(tile_mask), M, Ci, Co, _p(w), epilogue, _p(bias), _p(skip), _p(out),
         _stream())
    return out


def spconv_bf16(x: torch.Tensor, nmap_t: torch.Tensor, tile_mask: torch.Tensor, w: torch.Tensor,
                epilogue: int = EPI_ACC, *, bias: Optional[torch.Tensor] = None, skip: Optional[torch.Tensor] = None,
                out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """bf16 features (M, Ci) and weights (Co, 3, 3, 3, Ci): bf16 MFMA, fp32 accumulation, fp32 output (M, Co);
    epilogues ACC, BIAS (+ bias) and R (+ bias + skip)."""
    x = _dev(x, "x", torch.bfloat16)
    w = _dev(w, "w", torch.bfloat16)
    M, Ci = x.shape
    Co = w.shape[0]
    if w.numel() != Co * 27 * Ci:
        raise ValueError("weight must be (Co, 3, 3, 3, Ci)")
    if out is None:
        out = torch.empty((M, Co), dtype=torch.float32, device=x.device)
    call("pmg_spconv_bf16", _p(x), _p(nmap_t), _p(tile_mask), M, Ci, Co, _p(w), epilogue, _p(bias), _p(skip), _p(out),
         _stream())
    return out


def spconv_f32(x: torch.Tensor, nmap_t: torch.Tensor, tile_mask: torch.Tensor, w: torch.Tensor,
               bias: Optional[torch.Tensor] = None) -> torch.Tensor:
    x = _dev(x, "x", torch.float32)
    w = _dev(w, "w", torch.float32)
    M, Ci = x.shape
    Co = w.shape[0]
    if w.numel() != Co * 27 * Ci:
        raise ValueError("weight must be (Co, 3, 3, 3, Ci)")
    out = torch.empty((M, Co), dtype=torch.float32, device=x.device)
    call("pmg_spconv_f32", _p(x), _p(nmap_t), _p(tile_mask), M, Ci, Co, _p(w),
         EPI_BIAS if bias is not None else EPI_ACC, _p(bias), _p(out), _stream())
    return out


def spconv_col(x: torch.Tensor, zq: torch.Tensor, w: torch.Tensor, epilogue: int = EPI_ACC, *, a_scale: float = 1.0,
               w_scale: Optional[torch.Tensor] = None, bias: Optional[torch.Tensor] = None, out_mult: float = 1.0,
               skip: Optional[torch.Tensor] = None, out: Optional[torch.Tensor] = None,
               ln_gamma: Optional[torch.Tensor] = None, ln_beta: Optional[torch.Tensor] = None, ln_eps: float = 1e-6,
               next_mult: float = 1.0, next_q: Optional[torch.Tensor] = None, out_w: Optional[torch.Tensor] = None,
               out_b: Optional[torch.Tensor] = None, points: Optional[torch.Tensor] = None,
               points_out: Optional[torch.Tensor] = None):
    """Level-0 conv from the voxel keys zq [B, H, W] (no neighbour map). x: (M, C) int8 or fp16; w: (C, 3, 3, 3, C).
    Returns the main output (or points_out for EPI_ROUT)."""
    prec = {torch.int8: _lib.PREC_INT8, torch.float16: _lib.PREC_FP16}[x.dtype]
    x = _dev(x, "x")
    zq = _dev(zq, "zq", torch.int32)
    w = _dev(w, "w", x.dtype)
    B, H, W = zq.shape
    M, Cc = x.shape
    if M != B * H * W or w.numel() != Cc * 27 * Cc:
        raise ValueError("shape mismatch")
    if out is None and epilogue != EPI_ROUT:
        if epilogue == EPI_ACC:
            dt = torch.int32 if prec == _lib.PREC_INT8 else torch.float32
        elif epilogue == EPI_Q:
            dt = x.dtype
        else:
            dt = torch.float32
        out = torch.empty((M, Cc), dtype=dt, device=x.device)
    e = ConvEpilogue(float(a_scale), _p(w_scale), _p(bias), float(out_mult), _p(skip), _p(out), _p(ln_gamma),
                     _p(ln_beta), float(ln_eps), float(next_mult), _p(next_q), _p(out_w), _p(out_b), _p(points),
                     _p(points_out))
    call("pmg_spconv_col", prec, _p(x), _p(zq), B, H, W, Cc, _p(w), epilogue, C.byref(e), _stream())
    return points_out if epilogue == EPI_ROUT else out


def ln_silu_quant(x: torch.Tensor, gamma: torch.Tensor, beta: torch.Tensor, out_mult: float,
                  eps: float = 1e-6) -> torch.Tensor:
    x = _dev(x, "x", torch.float32)
    M, Cc = x.shape
    q = torch.empty((M, Cc), dtype=torch.int8, device=x.device)
    call("pmg_ln_silu_quant", _p(x), M, Cc, _p(gamma), _p(beta), float(eps), float(out_mult), _p(q), _stream())
    return q


def ln_silu_f16(x: torch.Tensor, gamma: torch.Tensor, beta: torch.Tensor, eps: float = 1e-6) -> torch.Tensor:
    x = _dev(x, "x", torch.float32)
    M, Cc = x.shape
    h = torch.empty((M, Cc), dtype=torch.float16, device=x.device)
    call("pmg_ln_silu_f16", _p(x), M, Cc, _p(gamma), _p(beta), float(eps), _p(h), _stream())
    return h


# ------------------------------------------------------------------------------------------------------------- (4)
_FIT_WS: dict = {}


def _fit_workspace(nbytes: int, device: torch.device) -> torch.Tensor:
    """The metric fit's workspace: zero-filled once, then reused by every call on the same (device, stream), since the
    fit kernel leaves it ready for the next launch. Calls on one stream are ordered, so they never share it at once."""
    key = (device.index, torch.cuda.current_stream(device).cuda_stream)
    ws = _FIT_WS.get(key)
    if ws is None or ws.numel() < nbytes:
        ws = torch.zeros((nbytes,), dtype=torch.uint8, device=device)
        _FIT_WS[key] = ws
    return ws


def fit_scale_shift(z: torch.Tensor, target: torch.Tensor, mask: torch.Tensor, iters: int = 4, trim: float = 0.2,
                    min_points: int = 32, differentiable: bool = False, *, return_info: bool = False):
    """fit_scale_shift (prompt_stem.py:211-240) on the GPU, same arguments: z, target, mask [B, ...] (flattened
    from dim 1). Returns s, t: [B] fp32 (and, with return_info, info [B, 5] int32 = count, k, ok, threshold bits,
    error flag). A batch item whose device-wide wait expired (the grid could not run co-resident) gets s = t = NaN
    and error flag 1; the workspace is ready for the next call either way. The result carries no gradient;
    `differentiable=True` under grad mode is refused."""
    if differentiable and torch.is_grad_enabled() and z.requires_grad:
        raise NotImplementedError("the GPU metric fit is inference-only (differentiable=True needs autograd)")
    z = _dev(z.float().reshape(z.shape[0], -1).contiguous(), "z")
    target = _dev(target.float().reshape(target.shape[0], -1).contiguous(), "target")
    m8 = _dev(mask.reshape(mask.shape[0], -1).to(torch.uint8).contiguous(), "mask")
    B, N = z.shape
    st = torch.empty((B, 2), dtype=torch.float32, device=z.device)
    info = torch.empty((B, 5), dtype=torch.int32, device=z.device)
    ws_bytes = lib().pmg_fit_workspace_bytes(N, iters)
    ws = _fit_workspace(ws_bytes, z.device)
    call("pmg_fit_scale_shift", _p(z), _p(target), _p(m8), B, N, int(iters), float(trim), int(min_points), _p(st),
         _p(info), _p(ws), ws_bytes, _stream())
    if return_info:
        return st[:, 0], st[:, 1], info
    return st[:, 0], st[:, 1]


def fit_prompt(points: torch.Tensor, lidar: torch.Tensor, conf: torch.Tensor, iters: int = 4, trim: float = 0.2,
               min_points: int = 32, return_info: bool = False):
    """Prompt fit of _lidar_in_affine_frame (v3.py:362-378) on the point map [B, H, W, 3] and LiDAR [B, dh, dw]."""
    points = _dev(points, "points", torch.float32)
    lidar = _dev(lidar.float().contiguous(), "lidar")
    conf = _dev(conf.float().contiguous(), "conf")
    B, H, W, _ = points.shape
    dh, dw = lidar.shape[-2:]
    st = torch.empty((B, 2), dtype=torch.float32, device=points.device)
    info = torch.empty((B, 5), dtype=torch.int32, device=points.device)
    ws_bytes = lib().pmg_fit_workspace_bytes(H * W, iters)
    ws = _fit_workspace(ws_bytes, points.device)
    call("pmg_fit_prompt", points.data_ptr() + 8, 3, _p(lidar), _p(conf), B, H, W, dh, dw, int(iters), float(trim),
         int(min_points), _p(st), _p(info), _p(ws), ws_bytes, _stream())
    if return_info:
        return st[:, 0], st[:, 1], info
    return st[:, 0], st[:, 1]


def fit_final(points: torch.Tensor, lidar: torch.Tensor, conf: torch.Tensor, mask_binary: Optional[torch.Tensor] = None,
              iters: int = 4, trim: float = 0.2, min_points: int = 32, return_info: bool = False):
    """Final metric fit (v3.py:768-778) of the depth exp(logz) of the point map [B, H, W, 3] against LiDAR
    [B, dh, dw] at LiDAR resolution (area-pooled depth). Returns (s, t) [B] (and the per-item info [B, 5])."""
    points = _dev(points, "points", torch.float32)
    lidar = _dev(lidar.float().contiguous(), "lidar")
    conf = _dev(conf.float().contiguous(), "conf")
    B, H, W, _ = points.shape
    dh, dw = lidar.shape[-2:]
    mb = None
    if mask_binary is not None:
        mb = _dev(mask_binary.to(torch.uint8).contiguous(), "mask_binary")
        if mb.numel() != B * H * W:
            raise ValueError("mask_binary must be [B, H, W]")
    st = torch.empty((B, 2), dtype=torch.float32, device=points.device)
    info = torch.empty((B, 5), dtype=torch.int32, device=points.device)
    ws_bytes = lib().pmg_fit_final_workspace_bytes(B, dh, dw, iters)
    ws = _fit_workspace(ws_bytes, points.device)
    call("pmg_fit_final", points.data_ptr() + 8, 3, _p(lidar), _p(conf), _p(mb), B, H, W, dh, dw, int(iters),
         float(trim), int(min_points), _p(st), _p(info), _p(ws), ws_bytes, _stream())
    if return_info:
        return st[:, 0], st[:, 1], info
    return st[:, 0], st[:, 1]

def post_depth(points: torch.Tensor, st: torch.Tensor, mask: Optional[torch.Tensor] = None,
               out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """post_depth (MetricFit.metal:200-211; v3.py:776): metric depth s * exp(logz) + t of the point map
    [B, H, W, 3] with the per-frame final fit st [B, 2] (read on the device, no synchronisation); +inf where mask
    [B, H, W] (bool / uint8, optional) is false or the depth is not positive. Returns [B, H, W] fp32."""
    points = _dev(points, "points", torch.float32)
    st = _dev(st.float().contiguous(), "st")
    B, H, W, _ = points.shape
    if st.shape != (B, 2):
        raise ValueError("st must be [B, 2]")
    m8 = None
    if mask is not None:
        m8 = _dev(mask.to(torch.uint8).contiguous(), "mask")
        if m8.numel() != B * H * W:
            raise ValueError("mask must be [B, H, W]")
    if out is None:
        out = torch.empty((B, H, W), dtype=torch.float32, device=points.device)
    call("pmg_post_depth", points.data_ptr() + 8, 3, _p(m8), B, H, W, _p(st), _p(out), _stream())
    return out


def nearest_fill(depth: torch.Tensor, conf: Optional[torch.Tensor] = None, *, return_index: bool = False,
                 out: Optional[Tuple[torch.Tensor, Optional[torch.Tensor]]] = None):
    """nearest_fill (promptmoge/model.py:61-72) on the GPU for depth (and conf) maps [..., h, w] fp32.

    Pixels with depth <= 0 (or NaN) take the depth of the nearest valid pixel -- the pixel scipy's exact EDT
    feature transform names: least distance, ties to the smaller column, then the smaller row -- and conf 1; an
    image without a valid pixel is returned as it is. Returns (depth, conf | None[, src_index]); `out` may be the
    inputs themselves (in-place fill). src_index holds i*w + j of each pixel's source (-1: no valid pixel).
    """
    depth = _dev(depth, "depth", torch.float32)
    if depth.ndim < 2:
        raise ValueError("depth must be [..., h, w]")
    h, w = depth.shape[-2:]
    B = depth.numel() // max(h * w, 1)
    if conf is not None:
        conf = _dev(conf, "conf", torch.float32)
        if conf.shape != depth.shape:
            raise ValueError("conf must have the shape of depth")
    if out is None:
        d_out = torch.empty_like(depth)
        c_out = torch.empty_like(conf) if conf is not None else None
    else:
        d_out, c_out = out
        d_out = _dev(d_out, "depth_out", torch.float32)
        if d_out.shape != depth.shape or (conf is not None and (c_out is None or c_out.shape != conf.shape)):
            raise ValueError("out must match the inputs")
    idx = torch.empty(depth.shape, dtype=torch.int32, device=depth.device) if return_index else None
    if depth.numel() > 0:
        ws_bytes = lib().pmg_nearest_fill_workspace_bytes(B, h, w)
        ws = torch.empty((ws_bytes,), dtype=torch.uint8, device=depth.device)
        call("pmg_nearest_fill", _p(depth), _p(conf), B, h, w, _p(d_out), _p(c_out) if conf is not None else None,
             _p(idx), _p(ws), ws_bytes, _stream())
    if return_index:
        return d_out, c_out, idx
    return d_out, c_out


def gauge_poly(depth: torch.Tensor, lidar: torch.Tensor, conf: Optional[torch.Tensor] = None, degree: int = 2,
               iters: int = 3, *, return_coef: bool = False):
    """MoGeModel.prompt_gauge_poly (moge/model/v3.py:151-183) on the GPU: the [B, H, W] correction exp(poly(u, v))
    fitted by IRLS to log(prompt / area-pooled prediction) on confident prompt pixels (fewer than 200: 1).

    depth [B, H, W] fp32; lidar (and conf, or None) [B, h, w] or [B, 1, h, w] fp32. With return_coef also the
    per-frame coefficients [B, 8] (basis order (1, u, v, u^2, uv, v^2); [:, 7] is 1 where the frame was fitted).
    """
    depth = _dev(depth, "depth", torch.float32)
    if depth.ndim != 3:
        raise ValueError("depth must be [B, H, W]")
    B, H, W = depth.shape
    lidar = _dev(lidar, "lidar", torch.float32)
    h, w = lidar.shape[-2:]
    if lidar.numel() != B * h * w:
        raise ValueError("lidar must be [B, h, w] or [B, 1, h, w]")
    if conf is not None:
        conf = _dev(conf, "conf", torch.float32)
        if conf.numel() != B * h * w:
            raise ValueError("conf must match lidar")
    corr = torch.empty_like(depth)
    coef = torch.empty((B, 8), dtype=torch.float32, device=depth.device)
    ws_bytes = lib().pmg_gauge_poly_workspace_bytes(B, h, w)
    ws = torch.empty((ws_bytes,), dtype=torch.uint8, device=depth.device)
    call("pmg_gauge_poly", _p(depth), B, H, W, _p(lidar), _p(conf), h, w, int(degree), int(iters), _p(corr),
         _p(coef), _p(ws), ws_bytes, _stream())
    return (corr, coef) if return_coef else corr


# ---------------------------------------------------------------------------------- (5) dense operators around the maps
# (These calls last a few microseconds: the checks below are written so that a valid call passes each in one step.)
_TYPES = {torch.float32: _lib.TYPE_F32, torch.float16: _lib.TYPE_F16, torch.bfloat16: _lib.TYPE_BF16,
          torch.int8: _lib.TYPE_I8}


def _in_forward_ad() -> bool:
    return getattr(forward_ad, "_current_level", 0) >= 0


def _refuse(needed: str, **named: Optional[torch.Tensor]) -> int:
    """Says which of the tensors (None: absent, but those needed) is not on the first one's GPU or needs a gradient; that
    GPU's index if none."""
    dev = None
    for name, t in named.items():
        if t is None and name not in needed.split():
            continue
        if not isinstance(t, torch.Tensor) or not t.is_cuda:
            raise ValueError(f"{name} must be a GPU tensor")
        dev = t.device if dev is None else dev
        if t.device != dev:
            raise ValueError(f"{name} is on {t.device}, the other tensors on {dev}")
        if (t.requires_grad and torch.is_grad_enabled()) or (
                _in_forward_ad() and forward_ad.unpack_dual(t).tangent is not None):
            raise RuntimeError("the libpmg operators are inference-only; run under torch.no_grad(), without tangents")
    return dev.index


def _one_gpu(*tensors: Optional[torch.Tensor]) -> int:
    """The index of the one GPU that all the tensors (None: absent) are on; negative if that takes a closer look (_refuse):
    one may not be on a GPU, on another one, or need a gradient."""
    grad = torch.is_grad_enabled()
    tensor = torch.Tensor
    d = -2  # (none seen; a host tensor's is -1)
    for t in tensors:
        if t is None:
            continue
        if not isinstance(t, tensor) or (grad and t.requires_grad):
            return -1
        i = t.get_device()
        if i != d:
            if i < 0 or d >= 0:
                return -1
            d = i
    return -1 if _in_forward_ad() else d


# The current stream's handle without building a torch.cuda.Stream (1 us); what the compiled torch code itself calls.
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (
    lambda d: torch.cuda.current_stream(d).cuda_stream)
_current_device = getattr(torch._C, "_cuda_getDevice", None) or torch.cuda.current_device
_ENTRIES: dict = {}


def _entry(name: str):
    entry = _ENTRIES.get(name)
    if entry is None:
        entry = _ENTRIES[name] = getattr(lib(), name)
    return entry


def _on(d: int, name: str, *args) -> None:
    """call() on GPU d (the current one or not; there are tensors on it), on its current stream."""
    entry = _ENTRIES.get(name) or _entry(name)
    if d == _current_device():
        code = entry(*args, _raw_stream(d))
    else:
        with torch.cuda.device(d):
            code = entry(*args, _raw_stream(d))
    if code:
        check(code)


def _floating(t: torch.Tensor, name: str) -> int:
    ty = _TYPES.get(t.dtype, _lib.TYPE_I8)
    if ty == _lib.TYPE_I8:
        raise ValueError(f"{name} must be float32, float16 or bfloat16, got {t.dtype}")
    return ty


def _ptr(t: Optional[torch.Tensor]) -> int:
    return 0 if t is None else t.data_ptr()


def _rows(t: torch.Tensor, name: str) -> int:
    """The row stride of an (M, C) tensor whose rows are contiguous and do not overlap."""
    if t.ndim != 2:
        raise ValueError(f"{name} must be 2-D, got {tuple(t.shape)}")
    (M, width), (row, one) = t.shape, t.stride()
    if (one == 1 or width <= 1) and row >= width:
        return max(row, 1)
    if M <= 1 and (one == 1 or width <= 1):
        return max(width, 1)
    raise ValueError(f"{name} must have contiguous rows that do not overlap, got strides {t.stride()}")


def _layout(t: torch.Tensor) -> Tuple[int, int, int, int]:
    """(address, end, period, width) in bytes: `width` bytes from the address on, and again every `period` bytes (the
    widest stride; 0: once), hold all of a tensor that is not empty."""
    axes = [(st, n - 1) for st, n in zip(t.stride(), t.shape) if n > 1]
    span, (period, more) = sum(st * n for st, n in axes) + 1, max(axes, default=(0, 0))
    es = t.element_size()
    return t.data_ptr(), t.data_ptr() + span * es, period * es, (span - period * more) * es


def _overlap(a: torch.Tensor, b: torch.Tensor) -> bool:
    """Whether two tensors share memory. Columns of one buffer (equal widest strides) are told apart; of other tensors
    laced into each other it is taken that they do."""
    if a.is_contiguous() and b.is_contiguous():  # (most are)
        a0, b0, na, nb = a.data_ptr(), b.data_ptr(), a.nbytes, b.nbytes
        return na > 0 and nb > 0 and a0 < b0 + nb and b0 < a0 + na
    if not a.numel() or not b.numel():
        return False
    (a0, a1, pa, wa), (b0, b1, pb, wb) = _layout(a), _layout(b)
    if a1 <= b0 or b1 <= a0:
        return False
    if pa != pb and a1 - a0 <= pb:  # (all of a in one of b's periods, as one row)
        pa, wa = pb, a1 - a0
    elif pa != pb and b1 - b0 <= pa:
        pb, wb = pa, b1 - b0
    if pa != pb or wa > pa or wb > pb:
        return True
    ahead = (b0 - a0) % pa
    return ahead < wa or ahead + wb > pa


def _apart(out: torch.Tensor, name: str, **others: Optional[torch.Tensor]) -> None:
    """Refuses a result on an argument that other blocks still read when it is written."""
    for other, t in others.items():
        if t is not None and _overlap(out, t):
            raise ValueError(f"{name} must not overlap {other}")


def _linear(x, w, bias, a_scale, w_scale, act, residual, out_dtype, out) -> torch.Tensor:
    d = _one_gpu(x, w, bias, w_scale, residual, out) if x is not None and w is not None else -1
    if d < 0:
        d = _refuse("x w", x=x, w=w, bias=bias, w_scale=w_scale, residual=residual, out=out)
    ldx = _rows(x, "x")
    M, K = x.shape
    if w.dtype != x.dtype:
        raise ValueError(f"w must be {x.dtype}, got {w.dtype}")
    if w.ndim != 2 or not w.is_contiguous():
        raise ValueError("w must be a contiguous (N, K) matrix")
    N, kw = w.shape
    if kw != K:
        raise ValueError(f"w expects {kw} input channels, x has {K}")
    if bias is not None:
        _vector(bias, "bias", N)
    if w_scale is not None:
        _vector(w_scale, "w_scale", N)
    code = _lib.ACTS.get(act)
    if code is None:
        raise ValueError(f"act must be one of {sorted(_lib.ACTS)}, got {act!r}")
    rt = ldr = 0
    if residual is not None:
        rt, ldr = _floating(residual, "residual"), _rows(residual, "residual")
        if residual.shape != (M, N):
            raise ValueError(f"residual must be ({M}, {N}), got {tuple(residual.shape)}")
    if out is None:
        if out_dtype is None:
            out_dtype = x.dtype if x.dtype != torch.int8 else torch.float32
        out = x.new_empty((M, N), dtype=out_dtype) if out_dtype != x.dtype else x.new_empty((M, N))
        ldo = N
    else:
        if out.shape != (M, N):
            raise ValueError(f"out must be ({M}, {N}), got {tuple(out.shape)}")
        if out_dtype is not None and out_dtype != out.dtype:
            raise ValueError(f"out_dtype is {out_dtype}, out has {out.dtype}")
        _apart(out, "out", x=x, w=w, bias=bias, w_scale=w_scale)
        if residual is not None and _overlap(out, residual) and not (
                out.data_ptr() == residual.data_ptr() and out.dtype == residual.dtype
                and out.stride() == residual.stride()):
            raise ValueError("out may be residual itself, but not overlap it otherwise")
        ldo = _rows(out, "out")
    args = _lib.LINEAR_PACK.pack(_TYPES[x.dtype], x.data_ptr(), ldx, w.data_ptr(), M, K, N, a_scale, _ptr(w_scale),
                                 _ptr(bias), code, _ptr(residual), rt, ldr, out.data_ptr(), _floating(out, "out"), ldo)
    _on(d, "pmg_linear", args)
    return out


def linear(x: torch.Tensor, w: torch.Tensor, bias: Optional[torch.Tensor] = None, *, act: str = "none",
           residual: Optional[torch.Tensor] = None, out_dtype: Optional[torch.dtype] = None,
           out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """act(x w^T + bias) + residual in one kernel: nn.Linear of the U-Net's PoolDown, NearestUp and projections with what
    follows it. x: (M, K) fp32 / fp16 / bf16 (rows may be strided); w: (N, K) of x's type; bias: (N,) fp32; act: "none",
    "relu", "silu", "gelu" (erf) or "gelu_tanh"; residual: (M, N) of any of the three types. Sums in fp32, rounded
    once to out_dtype (default: out's, or x's). `out` may be the residual itself. Forward only."""
    if isinstance(x, torch.Tensor):
        _floating(x, "x")
    return _linear(x, w, bias, 1.0, None, act, residual, out_dtype, out)


def linear_i8(x: torch.Tensor, w: torch.Tensor, bias: Optional[torch.Tensor] = None, *, a_scale: float = 1.0,
              w_scale: Optional[torch.Tensor] = None, act: str = "none", residual: Optional[torch.Tensor] = None,
              out_dtype: Optional[torch.dtype] = None, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """linear on int8 codes: act((acc * a_scale) * w_scale[n] + bias) + residual with the exact int32 sums acc, the
    arithmetic of spconv_i8. x: (M, K) int8; w: (N, K) int8; w_scale, bias: (N,) fp32; result fp32 (default), fp16 or
    bf16."""
    if isinstance(x, torch.Tensor) and x.dtype != torch.int8:
        raise ValueError(f"x must be torch.int8, got {x.dtype}")
    return _linear(x, w, bias, float(a_scale), w_scale, act, residual, out_dtype, out)


def _off_units(t: torch.Tensor, unit: int) -> bool:
    """Whether an (M, H, D) tensor's heads are not contiguous, or some not on `unit` bytes."""
    row, head, one = t.stride()
    return one != 1 or (t.data_ptr() | row * t.element_size() | head * t.element_size()) & (unit - 1) != 0


def _heads(t: torch.Tensor, name: str, unit: int) -> torch.Tensor:
    """An (M, H, D) tensor whose heads are contiguous, on `unit` bytes; copied where its strides or address are not."""
    if t.ndim != 3:
        raise ValueError(f"{name} must be (rows, heads, width), got {tuple(t.shape)}")
    return t.clone(memory_format=torch.contiguous_format) if _off_units(t, unit) else t  # (contiguous() keeps an odd address)


def _laced(t: torch.Tensor) -> bool:
    """Whether an (M, H, D) tensor's heads may overlap one another: neither its rows lie apart within a head's stride nor its
    heads within a row's."""
    (M, H, D), (row, head, _) = t.shape, t.stride()
    apart = lambda n, near, m, far: (n <= 1 or near >= D) and (m <= 1 or far >= (n - 1) * near * (n > 1) + D)  # noqa: E731
    return t.numel() > 0 and not (apart(H, head, M, row) or apart(M, row, H, head))


def _coords(t: torch.Tensor, name: str, rows: int) -> torch.Tensor:
    if t.dtype != torch.int32 or t.shape != (rows, 4):
        raise ValueError(f"{name} must be ({rows}, 4) int32, got {tuple(t.shape)} {t.dtype}")
    return t if t.is_contiguous() and t.data_ptr() % 16 == 0 else t.clone(memory_format=torch.contiguous_format)


def _vector(t: torch.Tensor, name: str, n: int) -> None:
    if t.dtype != torch.float32 or t.shape != (n,) or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous float32 ({n},) vector")


def qk_norm_rope(q: torch.Tensor, k: Optional[torch.Tensor], coords: torch.Tensor, freqs: torch.Tensor, *,
                 q_weight: Optional[torch.Tensor] = None, k_weight: Optional[torch.Tensor] = None,
                 q_bias: Optional[torch.Tensor] = None, k_bias: Optional[torch.Tensor] = None, norm: str = "rms",
                 eps: float = 1e-6, interleaved: bool = False,
                 out: Optional[Tuple[torch.Tensor, Optional[torch.Tensor]]] = None):
    """The norms of queries and keys per head, then the rotation by voxel coordinates, in one pass over both.

    q: (M, Hq, D), k: (M, Hk, D) or None, fp32 / fp16 / bf16, slices of one product allowed; D a multiple of 8 up to 128.
    norm: "rms" (x * rsqrt(mean(x^2) + eps) * weight + bias) or "layer" (of x - mean). coords: (M, 4) int32
    (b, x, y, z); freqs: (P, 3) fp32, P <= D / 2: pair p is turned by the angle x f[p, 0] + y f[p, 1] + z f[p, 2], formed in 64
    bits. Pair p is (p, p + D/2), or with interleaved (2p, 2p + 1). Returns (q, k) in new tensors, or in `out` (which
    may be the inputs). Forward only."""
    qo, ko = out if out is not None else (None, None)
    d = _one_gpu(q, k, coords, freqs, q_weight, k_weight, q_bias, k_bias, qo, ko) if q is not None else -1
    if d < 0:
        d = _refuse("q coords freqs", q=q, k=k, coords=coords, freqs=freqs, q_weight=q_weight, k_weight=k_weight,
                    q_bias=q_bias, k_bias=k_bias, out_q=qo, out_k=ko)
    ty = _floating(q, "q")
    unit = 4 * q.element_size()
    if norm not in ("rms", "layer"):
        raise ValueError(f"norm must be 'rms' or 'layer', got {norm!r}")
    if q.ndim != 3:
        raise ValueError(f"q must be (rows, heads, width), got {tuple(q.shape)}")
    M, Hq, D = q.shape
    if k is not None and (k.ndim != 3 or k.shape[0] != M or k.shape[2] != D or k.dtype != q.dtype):
        raise ValueError(f"k must be ({M}, heads, {D}) of q's type")
    coords = _coords(coords, "coords", M)
    if freqs.dtype != torch.float32 or freqs.ndim != 2 or freqs.shape[1] != 3 or not freqs.is_contiguous():
        raise ValueError("freqs must be a contiguous (pairs, 3) float32 tensor")
    if q_weight is not None:
        _vector(q_weight, "q_weight", D)
    if k_weight is not None:
        _vector(k_weight, "k_weight", D)
    if q_bias is not None:
        _vector(q_bias, "q_bias", D)
    if k_bias is not None:
        _vector(k_bias, "k_bias", D)
    if out is None:
        qo = q.new_empty((M, Hq, D))
        if k is not None:
            ko = q.new_empty((M, k.shape[1], D))
    else:
        for i, (name, t, o) in enumerate((("out[0]", q, qo), ("out[1]", k, ko))):
            if (t is None) != (o is None) or (t is not None and (o.shape != t.shape or o.dtype != q.dtype)):
                raise ValueError(f"{name} must match its input")
            if o is not None and _off_units(o, unit):
                raise ValueError(f"{name}: strides and address must be whole groups of 4 elements")
            if o is not None and _laced(o):
                raise ValueError(f"{name}: its own rows and heads must not overlap")
            for j, other in enumerate((q, k)):  # (its input itself is fine: each head is read whole before it is written)
                if o is not None and other is not None and _overlap(o, other) and not (
                        i == j and o.data_ptr() == t.data_ptr() and o.stride() == t.stride()):
                    raise ValueError(f"{name} may be its input itself, but not overlap the inputs otherwise")
            if o is not None:
                _apart(o, name, coords=coords, freqs=freqs, q_weight=q_weight, k_weight=k_weight, q_bias=q_bias, k_bias=k_bias)
        if ko is not None and _overlap(qo, ko):
            raise ValueError("out[0] and out[1] must not overlap")
    q = _heads(q, "q", unit)
    k = _heads(k, "k", unit) if k is not None else None
    Hk, (ks, kh), (kos, koh) = 0, (0, 0), (0, 0)
    if k is not None:
        Hk, (ks, kh, _), (kos, koh, _) = k.shape[1], k.stride(), ko.stride()
    (qs, qh, _), (qos, qoh, _) = q.stride(), qo.stride()
    args = _lib.ROPE_PACK.pack(ty, M, Hq, Hk, D, freqs.shape[0], q.data_ptr(), qs, qh, _ptr(k), ks, kh, qo.data_ptr(),
                               qos, qoh, _ptr(ko), kos, koh, coords.data_ptr(), freqs.data_ptr(), _ptr(q_weight),
                               _ptr(k_weight), _ptr(q_bias), _ptr(k_bias), norm == "layer", bool(interleaved), eps)
    _on(d, "pmg_qk_norm_rope", args)
    return qo, ko


def _index(t: torch.Tensor, name: str) -> None:
    if t.dtype != torch.int32 or t.ndim != 1 or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous 1-D int32 tensor")


def _offsets(t: torch.Tensor, name: str) -> None:
    if t.dtype != torch.int64 or t.ndim != 1 or t.numel() < 1 or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous (segments + 1,) int64 tensor")


def sparse_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, offsets: torch.Tensor,
                     kv_offsets: Optional[torch.Tensor] = None, *, index: Optional[torch.Tensor] = None,
                     kv_index: Optional[torch.Tensor] = None, coords: Optional[torch.Tensor] = None,
                     kv_coords: Optional[torch.Tensor] = None, slopes: Optional[torch.Tensor] = None,
                     kv_mask: Optional[torch.Tensor] = None, cap: float = 0.0, scale: Optional[float] = None,
                     precise: bool = False, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Attention inside segments of rows: the frames of a batch, or the cells of a pool cache (its seg_offsets as
    `offsets` and seg_indices as `index`).

    q: (Mq, Hq, D); k, v: (Mk, Hk, D), Hq a multiple of Hk; fp32 / fp16 / bf16, D a multiple of 8 up to 128. offsets: (S + 1,)
    int64, rising: segment s holds the positions offsets[s] .. offsets[s + 1] - 1; position p is row index[p] (int32), or
    row p. Without kv_offsets the keys' segments (and index, and coordinates) are the queries'; with them, segment s of
    the queries attends to segment s of the keys. Scores: scale q.k (scale: default D^-1/2); cap > 0: cap tanh(x / cap);
    slopes (Hq, 3) fp32: minus sum over the axes of slopes[h, axis] |difference of coords (M, 4) int32 (b, x, y, z)|;
    kv_mask (Mk,) bool / uint8: rows with 0 are not attended to. A query with no key left gets 0.

    Sums, maxima and scores are fp32. In fp16 and bf16 the softmax's weights are rounded to that type for the second product, which
    adds about the error of the result's own rounding; precise keeps them to fp32's accuracy, for 7 to 41 % more time.

    Rows that no position of a segment names are 0 in a new result and left as they were in a given `out`. A row named by
    two query positions gets either's result. Where offsets fall, what the rows get is not said. Forward only."""
    d = -1
    if q is not None:
        d = _one_gpu(q, k, v, offsets, kv_offsets, index, kv_index, coords, kv_coords, slopes, kv_mask, out)
    if d < 0:
        d = _refuse("q k v offsets", q=q, k=k, v=v, offsets=offsets, kv_offsets=kv_offsets, index=index,
                    kv_index=kv_index, coords=coords, kv_coords=kv_coords, slopes=slopes, kv_mask=kv_mask, out=out)
    ty = _floating(q, "q")
    if q.ndim != 3 or k.ndim != 3 or v.shape != k.shape or k.shape[2] != q.shape[2]:
        raise ValueError(f"q must be (Mq, Hq, D), k and v (Mk, Hk, D); got {tuple(q.shape)}, {tuple(k.shape)}, {tuple(v.shape)}")
    if k.dtype != q.dtype or v.dtype != q.dtype:
        raise ValueError("k and v must have q's type")
    Mq, Hq, D = q.shape
    Mk, Hk = k.shape[:2]
    if Hk < 1 or Hq % Hk:
        raise ValueError(f"{Hq} query heads are not a multiple of {Hk} key heads")
    own = kv_offsets is None
    if own:
        if kv_index is not None or kv_coords is not None:
            raise ValueError("kv_index and kv_coords go with kv_offsets")
        if Mk != Mq:
            raise ValueError(f"without kv_offsets the keys are the queries' rows: {Mq} and {Mk}")
        kv_offsets, kv_index, kv_coords = offsets, index, coords
    _offsets(offsets, "offsets")
    if index is not None:
        _index(index, "index")
    if not own:
        _offsets(kv_offsets, "kv_offsets")
        if kv_offsets.numel() != offsets.numel():
            raise ValueError("offsets and kv_offsets must have the same length")
        if kv_index is not None:
            _index(kv_index, "kv_index")
    if slopes is not None:
        if slopes.dtype != torch.float32 or slopes.shape != (Hq, 3) or not slopes.is_contiguous():
            raise ValueError(f"slopes must be a contiguous ({Hq}, 3) float32 tensor")
        if coords is None or kv_coords is None:
            raise ValueError("slopes need coords (and kv_coords with kv_offsets)")
        same = kv_coords is coords
        coords = _coords(coords, "coords", Mq)
        kv_coords = coords if same and Mk == Mq else _coords(kv_coords, "kv_coords", Mk)
    if kv_mask is not None:
        if kv_mask.dtype not in (torch.bool, torch.uint8) or kv_mask.shape != (Mk,) or not kv_mask.is_contiguous():
            raise ValueError(f"kv_mask must be a contiguous ({Mk},) bool or uint8 tensor")
    fresh = out is None
    if fresh:
        out = q.new_empty((Mq, Hq, D))
    else:
        if out.shape != q.shape or out.dtype != q.dtype:
            raise ValueError(f"out must be {tuple(q.shape)} {q.dtype}")
        if _off_units(out, 4 * q.element_size()):
            raise ValueError("out: strides and address must be whole groups of 4 elements")
        if _laced(out):
            raise ValueError("out: its own rows and heads must not overlap")
        _apart(out, "out", q=q, k=k, v=v, offsets=offsets, kv_offsets=kv_offsets, index=index, kv_index=kv_index,
               coords=coords, kv_coords=kv_coords, slopes=slopes, kv_mask=kv_mask)
    q, k, v = _heads(q, "q", 16), _heads(k, "k", 16), _heads(v, "v", 16)
    (qs, qh, _), (ks, kh, _), (vs, vh, _), (os, oh, _) = q.stride(), k.stride(), v.stride(), out.stride()
    args = _lib.ATTENTION_PACK.pack(
        ty, Hq, Hk, D, q.data_ptr(), qs, qh, k.data_ptr(), ks, kh, v.data_ptr(), vs, vh, out.data_ptr(), os, oh, Mq, Mk,
        Mq if index is None else index.shape[0], Mk if kv_index is None else kv_index.shape[0], offsets.shape[0] - 1,
        offsets.data_ptr(), kv_offsets.data_ptr(), _ptr(index), _ptr(kv_index), _ptr(coords) if slopes is not None else 0,
        _ptr(kv_coords) if slopes is not None else 0, _ptr(slopes), _ptr(kv_mask), (D or 1) ** -0.5 if scale is None else scale,
        cap, fresh, bool(precise))
    ws_bytes = _entry("pmg_attention_workspace_bytes")(args)
    ws = q.new_empty((ws_bytes,), dtype=torch.uint8) if ws_bytes else None
    _on(d, "pmg_attention", args, _ptr(ws), ws_bytes)
    return out


# ------------------------------------------------------------------------------------- (6) a conditional layer on rows
def _act(act: str) -> int:
    code = _lib.ACTS.get(act)
    if code is None:
        raise ValueError(f"act must be one of {sorted(_lib.ACTS)}, got {act!r}")
    return code


def _residual(residual: Optional[torch.Tensor], rows: int, N: int) -> Tuple[int, int]:
    """The type and row stride of a (rows, N) residual (None: 0, 0)."""
    if residual is None:
        return 0, 0
    rt, ldr = _floating(residual, "residual"), _rows(residual, "residual")
    if residual.shape != (rows, N):
        raise ValueError(f"residual must be ({rows}, {N}), got {tuple(residual.shape)}")
    return rt, ldr


def _new(like: torch.Tensor, ty: int, rows: int, N: int, out_dtype: Optional[torch.dtype]) -> Tuple[torch.Tensor, int, int]:
    """A new (rows, N) result of out_dtype (None: of `like`'s type, whose code is ty), its type and its row stride."""
    if out_dtype is None or out_dtype == like.dtype:
        return like.new_empty((rows, N)), ty, N
    out = like.new_empty((rows, N), dtype=out_dtype)
    return out, _floating(out, "out"), N


def _given(out: torch.Tensor, out_dtype: Optional[torch.dtype], rows: int, N: int, same: str, same_as: Optional[torch.Tensor],
           **others: Optional[torch.Tensor]) -> Tuple[torch.Tensor, int, int]:
    """A given (rows, N) result, its type and its row stride. It may be `same_as` (named `same`) itself but lie on nothing else
    of the call."""
    if out.shape != (rows, N):
        raise ValueError(f"out must be ({rows}, {N}), got {tuple(out.shape)}")
    if out_dtype is not None and out_dtype != out.dtype:
        raise ValueError(f"out_dtype is {out_dtype}, out has {out.dtype}")
    if same_as is not None and _overlap(out, same_as) and not (
            out.data_ptr() == same_as.data_ptr() and out.dtype == same_as.dtype and out.stride() == same_as.stride()):
        raise ValueError(f"out may be {same} itself, but not overlap it otherwise")
    _apart(out, "out", **others)
    return out, _floating(out, "out"), _rows(out, "out")


def _workspace(entry: str, like: torch.Tensor, args: bytes) -> Tuple[Optional[torch.Tensor], int]:
    n = _entry(entry)(args)
    return (like.new_empty((n,), dtype=torch.uint8) if n else None), n


def group_norm(x: torch.Tensor, groups: int, weight: Optional[torch.Tensor] = None, bias: Optional[torch.Tensor] = None, *,
               offsets: Optional[torch.Tensor] = None, eps: float = 1e-5, act: str = "none",
               out_dtype: Optional[torch.dtype] = None, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Group norm with channels last, then the activation: act((x - mean) / sqrt(var + eps) * weight + bias), mean and var over
    a segment's rows and a group's C / groups channels (torch's GroupNorm on a frame's (C, rows)).

    x: (M, C) fp32 / fp16 / bf16, C up to 4096 (rows may be strided); weight, bias: (C,) fp32; offsets: (S + 1,) int64, rising:
    segment s holds the rows offsets[s] .. offsets[s + 1] - 1 (a batch's frames); without, all rows are one segment. act:
    as for linear. Sums in 64 bits, one rounding, to out_dtype (default: out's, or x's). Rows of no segment are 0 in a new
    result and left as they were in a given `out`, which may be x itself. Where offsets fall, what the rows get is
    not said. The form goes by M / S: a segment far longer than the others, where M / S is at most 512, is right but slow (one
    block goes over it, 9 to 50 us for 1000 rows). Forward only."""
    d = _one_gpu(x, weight, bias, offsets, out) if x is not None else -1
    if d < 0:
        d = _refuse("x", x=x, weight=weight, bias=bias, offsets=offsets, out=out)
    ty, ldx = _floating(x, "x"), _rows(x, "x")
    M, C_ = x.shape
    if groups < 1 or C_ % groups or C_ < 1:
        raise ValueError(f"{C_} channels are not a multiple of {groups} groups")
    if weight is not None:
        _vector(weight, "weight", C_)
    if bias is not None:
        _vector(bias, "bias", C_)
    if offsets is not None:
        _offsets(offsets, "offsets")
    code = _act(act)
    fresh = out is None
    if fresh:
        out, ot, ldo = _new(x, ty, M, C_, out_dtype)
    else:
        out, ot, ldo = _given(out, out_dtype, M, C_, "x", x, weight=weight, bias=bias, offsets=offsets)
    S = 1 if offsets is None else offsets.shape[0] - 1
    args = _lib.GROUP_NORM_PACK.pack(ty, x.data_ptr(), ldx, M, C_, groups, _ptr(weight), _ptr(bias), _ptr(offsets), S, eps, code,
                                     out.data_ptr(), ot, ldo, fresh)
    ws, n = (None, 0) if M <= 512 * S else _workspace("pmg_group_norm_workspace_bytes", x, args)  # (short segments need none)
    _on(d, "pmg_group_norm", args, _ptr(ws), n)
    return out


class Routes(NamedTuple):
    """Which experts the rows go to, and the tables that group the pairs m k + slot of a row and its slot by expert."""

    weights: torch.Tensor  # (M, k) fp32: 0 for a slot without an expert
    experts: torch.Tensor  # (M, k) int32: -1 for a slot without an expert
    offsets: torch.Tensor  # (E + 1,) int64: expert e's pairs are pairs[offsets[e]:offsets[e + 1]]
    pairs: torch.Tensor    # (M k,) int32: in the order of the experts, then their own; -1 from offsets[E] on
    rows: torch.Tensor     # (M k,) int32: pairs // k


def route(logits: torch.Tensor, k: int, *, score: str = "softmax", normalize: bool = False,
          mask: Optional[torch.Tensor] = None) -> Routes:
    """The k experts of largest logit of each row (equal ones: the lowest index first), their weights, and the pairs in the
    order of the experts, for grouped_linear and combine:

        r = route(logits, k)
        h = grouped_linear(x, w_up, r.offsets, index=r.rows, act="gelu")
        y = grouped_linear(h, w_down, r.offsets, out_index=r.pairs, out=h.new_empty((M * k, N)))
        z = combine(y.view(M, k, N), r.weights, residual=x)

    logits: (M, E) fp32 / fp16 / bf16 (rows may be strided), E up to 1024, k up to 32; score: "softmax" over the row's
    logits, or "sigmoid"; normalize: the weights over the sum of the row's. An expert whose logit is -inf or NaN is not
    chosen: the slot holds -1 and weight 0 (the others' softmax over a row with a NaN or +inf is NaN, as its sum is). So do
    the rows with 0 in mask, (M,) bool / uint8, whose pairs come in no segment. Forward only."""
    d = _one_gpu(logits, mask) if logits is not None else -1
    if d < 0:
        d = _refuse("logits", logits=logits, mask=mask)
    ty, ld = _floating(logits, "logits"), _rows(logits, "logits")
    M, E = logits.shape
    if not 1 <= E <= 1024 or not 1 <= k <= min(E, 32):
        raise ValueError(f"{k} of {E} experts: there may be 1 to 1024, and 1 to 32 a row")
    code = _lib.SCORES.get(score)
    if code is None:
        raise ValueError(f"score must be one of {sorted(_lib.SCORES)}, got {score!r}")
    if mask is not None and (mask.dtype not in (torch.bool, torch.uint8) or mask.shape != (M,) or not mask.is_contiguous()):
        raise ValueError(f"mask must be a contiguous ({M},) bool or uint8 tensor")
    weights = logits.new_empty((M, k), dtype=torch.float32)
    # W: the entry's workspace at the most, E + 1 counts for each 16 rows and 32,768 in all; one block, of up to 64 rows, needs none. (It
    # lies behind the tables and lives as long as they do: an allocation of its own costs 1.4 us of a call's 14.)
    P, W = M * k, 0 if M <= 64 else min((M + 15) // 16 * (E + 1), 32_768)
    tables = logits.new_empty((3 * P + W,), dtype=torch.int32)
    offsets = logits.new_empty((E + 1,), dtype=torch.int64)
    experts = tables.as_strided((M, k), (k, 1))
    pairs, rows = tables.as_strided((P,), (1,), P), tables.as_strided((P,), (1,), 2 * P)
    at = tables.data_ptr()
    args = _lib.ROUTE_PACK.pack(ty, logits.data_ptr(), ld, M, E, k, code, bool(normalize), _ptr(mask), weights.data_ptr(),
                                at, offsets.data_ptr(), at + 4 * P, at + 8 * P)
    _on(d, "pmg_route", args, at + 12 * P if W else 0, 4 * W)
    return Routes(weights, experts, offsets, pairs, rows)


def grouped_linear(x: torch.Tensor, w: torch.Tensor, offsets: torch.Tensor, bias: Optional[torch.Tensor] = None, *,
                   index: Optional[torch.Tensor] = None, out_index: Optional[torch.Tensor] = None, act: str = "none",
                   residual: Optional[torch.Tensor] = None, out_dtype: Optional[torch.dtype] = None,
                   out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """linear with a matrix per segment: act(x w[s]^T + bias[s]) + residual for the rows of segment s (an expert's rows, or a
    frame's).

    x: (Mx, K) fp32 / fp16 / bf16 (rows may be strided); w: (S, N, K) of x's type; bias: (S, N) fp32; offsets: (S + 1,) int64,
    rising: segment s holds the positions offsets[s] .. offsets[s + 1] - 1. Position p reads row index[p] of x (int32), or row p,
    and gives row out_index[p] of the result (int32; needs `out`), or row p; residual is added row by row of the result. Sums in
    fp32, one rounding, to out_dtype (default: out's, or x's).

    Positions of no segment and those whose index lies outside the rows give nothing: their rows are 0 in a new result and
    left as they were in a given `out`, which may be the residual itself. Where two positions of out_index name a row, each of
    its values is either's. Where offsets fall, what the rows get is not said. Forward only."""
    d = -1
    if x is not None and w is not None and offsets is not None:
        d = _one_gpu(x, w, offsets, bias, index, out_index, residual, out)
    if d < 0:
        d = _refuse("x w offsets", x=x, w=w, offsets=offsets, bias=bias, index=index, out_index=out_index,
                    residual=residual, out=out)
    ty, ldx = _floating(x, "x"), _rows(x, "x")
    Mx, K = x.shape
    if w.dtype != x.dtype:
        raise ValueError(f"w must be {x.dtype}, got {w.dtype}")
    if w.ndim != 3 or not w.is_contiguous():
        raise ValueError("w must be a contiguous (S, N, K) tensor")
    S, N, kw = w.shape
    if kw != K:
        raise ValueError(f"w expects {kw} input channels, x has {K}")
    _offsets(offsets, "offsets")
    if offsets.shape[0] != S + 1:
        raise ValueError(f"offsets of {offsets.shape[0] - 1} segments, w of {S}")
    if bias is not None and (bias.dtype != torch.float32 or bias.shape != (S, N) or not bias.is_contiguous()):
        raise ValueError(f"bias must be a contiguous float32 ({S}, {N}) tensor")
    P = Mx
    if index is not None:
        _index(index, "index")
        P = index.shape[0]
    rows = P
    if out_index is not None:
        _index(out_index, "out_index")
        if out is None:
            raise ValueError("out_index needs out")
        if out_index.shape[0] != P:
            raise ValueError(f"out_index must have {P} positions, got {out_index.shape[0]}")
        if out.ndim == 2:
            rows = out.shape[0]
    code = _act(act)
    rt, ldr = _residual(residual, rows, N)
    fresh = out is None
    if fresh:
        out, ot, ldo = _new(x, ty, rows, N, out_dtype)
    else:
        out, ot, ldo = _given(out, out_dtype, rows, N, "residual", residual, x=x, w=w, offsets=offsets, bias=bias, index=index,
                              out_index=out_index)
    args = _lib.GROUPED_PACK.pack(ty, x.data_ptr(), ldx, Mx, w.data_ptr(), P, S, K, N, offsets.data_ptr(), _ptr(index),
                                  _ptr(out_index), _ptr(bias), code, _ptr(residual), rt, ldr, out.data_ptr(), ot, ldo, rows, fresh)
    _on(d, "pmg_grouped_linear", args)
    return out


def combine(y: torch.Tensor, weights: torch.Tensor, *, residual: Optional[torch.Tensor] = None,
            out_dtype: Optional[torch.dtype] = None, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """A row's experts put together: sum over the slots j of weights[m, j] y[m, j], plus residual[m], in fp32 and rounded once.

    y: (M, k, N) fp32 / fp16 / bf16, N contiguous, k up to 32; weights: (M, k) fp32; residual: (M, N) of any of the three types. A
    slot of weight 0 is not read: it may hold anything, as pairs without an expert do. `out` may be the residual itself.
    Forward only."""
    d = _one_gpu(y, weights, residual, out) if y is not None and weights is not None else -1
    if d < 0:
        d = _refuse("y weights", y=y, weights=weights, residual=residual, out=out)
    ty = _floating(y, "y")
    if y.ndim != 3 or (y.stride(2) != 1 and y.shape[2] > 1):
        raise ValueError(f"y must be (rows, slots, N) with contiguous N, got {tuple(y.shape)}, strides {y.stride()}")
    M, k, N = y.shape
    if not 1 <= k <= 32:
        raise ValueError(f"y must have 1 to 32 slots, got {k}")
    if weights.dtype != torch.float32 or weights.shape != (M, k) or not weights.is_contiguous():
        raise ValueError(f"weights must be a contiguous float32 ({M}, {k}) tensor")
    rt, ldr = _residual(residual, M, N)
    if out is None:
        out, ot, ldo = _new(y, ty, M, N, out_dtype)
    else:
        out, ot, ldo = _given(out, out_dtype, M, N, "residual", residual, y=y, weights=weights)
    args = _lib.COMBINE_PACK.pack(ty, y.data_ptr(), y.stride(0), y.stride(1), M, k, N, weights.data_ptr(), _ptr(residual), rt, ldr,
                                  out.data_ptr(), ot, ldo)
    _on(d, "pmg_combine", args)
    return out


def lora_linear(x: torch.Tensor, w: torch.Tensor, down: torch.Tensor, up: torch.Tensor, adapter: torch.Tensor,
                bias: Optional[torch.Tensor] = None, *, offsets: Optional[torch.Tensor] = None,
                scale: Optional[torch.Tensor] = None, act: str = "none", residual: Optional[torch.Tensor] = None,
                out_dtype: Optional[torch.dtype] = None, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """linear with a low-rank adapter per segment: act(x w^T + bias + scale[i] (x down[i]^T) up[i]^T) + residual, i = adapter[s] for
    the rows of segment s. A batch's frames, each with the adapter of its sensor, share one projection.

    x: (M, K) fp32 / fp16 / bf16 (rows may be strided); w: (N, K), down: (A, r, K), up: (A, N, r) of x's type, r up to 128;
    adapter: (S,) int32, one outside 0 .. A - 1: none; scale: (A,) fp32; offsets: (S + 1,) int64, rising: segment s holds the rows
    offsets[s] .. offsets[s + 1] - 1; without, S is M and every row is a segment. Rows of no segment have the projection alone.
    x down^T is held to fp32's accuracy for the second product; sums in fp32, one rounding, to out_dtype (default: out's,
    or x's). `out` may be the residual itself. Where offsets fall, what the rows get is not said. Forward only."""
    d = -1
    if x is not None and w is not None and down is not None and up is not None and adapter is not None:
        d = _one_gpu(x, w, down, up, adapter, bias, offsets, scale, residual, out)
    if d < 0:
        d = _refuse("x w down up adapter", x=x, w=w, down=down, up=up, adapter=adapter, bias=bias, offsets=offsets,
                    scale=scale, residual=residual, out=out)
    ty, ldx, t = _floating(x, "x"), _rows(x, "x"), x.dtype
    M, K = x.shape
    if w.dtype != t or down.dtype != t or up.dtype != t:
        raise ValueError(f"w, down and up must be {t}")
    ws_, ds, us = w.shape, down.shape, up.shape
    if len(ws_) != 2 or ws_[1] != K or not w.is_contiguous():
        raise ValueError(f"w must be a contiguous (N, {K}) matrix, got {tuple(ws_)}")
    N = ws_[0]
    if len(ds) != 3 or ds[2] != K or not down.is_contiguous():
        raise ValueError(f"down must be a contiguous (A, r, {K}) tensor, got {tuple(ds)}")
    A, r, _ = ds
    if us != (A, N, r) or not up.is_contiguous():
        raise ValueError(f"up must be a contiguous ({A}, {N}, {r}) tensor, got {tuple(us)}")
    if not 1 <= r <= 128:
        raise ValueError(f"adapters of rank 1 to 128, got {r}")
    S = M
    if offsets is not None:
        _offsets(offsets, "offsets")
        S = offsets.shape[0] - 1
    if adapter.dtype != torch.int32 or adapter.shape != (S,) or not adapter.is_contiguous():
        raise ValueError(f"adapter must be a contiguous int32 ({S},) tensor")
    if bias is not None:
        _vector(bias, "bias", N)
    if scale is not None:
        _vector(scale, "scale", A)
    code = _act(act)
    rt, ldr = _residual(residual, M, N)
    if out is None:
        out, ot, ldo = _new(x, ty, M, N, out_dtype)
    else:
        out, ot, ldo = _given(out, out_dtype, M, N, "residual", residual, x=x, w=w, down=down, up=up, adapter=adapter, bias=bias,
                              offsets=offsets, scale=scale)
    args = _lib.LORA_PACK.pack(ty, x.data_ptr(), ldx, M, K, N, w.data_ptr(), down.data_ptr(), up.data_ptr(), r, A, _ptr(scale),
                               adapter.data_ptr(), _ptr(offsets), S, _ptr(bias), code, _ptr(residual), rt, ldr, out.data_ptr(), ot, ldo)
    if offsets is None and M <= 8 and r <= 16 and M * r <= 64:  # (one launch, no workspace)
        _on(d, "pmg_lora_linear", args, 0, 0)
        return out
    # (what the entry asks for at the most: r values of 6 bytes and one of 4 a row, on 256 bytes)
    n = (6 * r + 4) * M + 512
    ws = x.new_empty((n,), dtype=torch.uint8)
    _on(d, "pmg_lora_linear", args, ws.data_ptr(), n)
    return out
