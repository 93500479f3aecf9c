"""Sizes of grouped_linear and lora_linear calls that take each of their kernels, by type and kind: what a call's sizes choose is
asked of the library itself (pmg_debug_grouped_form, pmg_debug_lora_form), so that no change of its costs drops a kernel unseen."""
import ctypes as C

from promptmoge_amd import _lib

EXPERTS, SEGMENTS, ROWS, FEW = range(4)  # a matrix a segment; tiles of one adapter; an adapter a row; up to eight rows
AT = 1 << 12  # an address on 16 bytes that is not looked at

# (rows, K, N, rank, segments or None: every row one), (kind, a block's rows, columns, LDS places, 16 bytes at a time)
OF_16_BITS = [
    ((40, 72, 40, 0, 5), (EXPERTS, 16, 32, 0, 1)), ((50, 71, 40, 0, 5), (EXPERTS, 16, 16, 0, 0)), ((700, 65, 130, 0, 3), (EXPERTS, 64, 64, 1, 0)),
    ((300, 64, 72, 0, 3), (EXPERTS, 64, 64, 2, 1)), ((300, 1040, 72, 0, 3), (EXPERTS, 64, 64, 3, 1)), ((900, 72, 2350, 0, 20), (EXPERTS, 64, 128, 2, 1)),
    ((12_340, 72, 385, 0, 4), (EXPERTS, 128, 128, 2, 1)), ((14_200, 200, 774, 0, 3), (EXPERTS, 128, 256, 3, 1)), ((12_300, 408, 263, 0, 20), (EXPERTS, 192, 128, 3, 1)),
    ((300, 64, 72, 8, 3), (SEGMENTS, 64, 64, 2, 1)), ((300, 1040, 72, 32, 3), (SEGMENTS, 64, 64, 3, 1)), ((900, 72, 2350, 24, 3), (SEGMENTS, 64, 128, 2, 1)),
    ((12_340, 72, 385, 128, 4), (SEGMENTS, 128, 128, 2, 1)), ((19_200, 256, 1024, 16, 4), (SEGMENTS, 128, 128, 2, 1)), ((14_200, 200, 774, 40, 3), (SEGMENTS, 128, 256, 3, 1)),
    ((4800, 1024, 4096, 16, 4), (SEGMENTS, 128, 256, 3, 1)), ((12_300, 408, 263, 16, 20), (SEGMENTS, 192, 128, 3, 1)),
    ((7, 72, 40, 9, None), (FEW, 8, 32, 0, 1)), ((8, 71, 40, 8, None), (FEW, 8, 32, 0, 0)),
    ((90, 72, 40, 5, None), (ROWS, 16, 16, 0, 1)), ((90, 71, 40, 8, None), (ROWS, 16, 16, 0, 0)), ((4300, 72, 40, 8, None), (ROWS, 64, 64, 2, 1)), ((700, 65, 264, 5, None), (ROWS, 64, 64, 1, 0)),
    ((700, 33, 264, 16, 3), (ROWS, 64, 64, 1, 0)), ((9600, 920, 16, 33, None), (ROWS, 64, 64, 3, 1)), ((17_440, 72, 70, 16, None), (ROWS, 64, 128, 2, 1)), ((12_340, 72, 385, 7, None), (ROWS, 128, 128, 2, 1)),
    ((14_200, 200, 774, 8, None), (ROWS, 128, 256, 3, 1)), ((11_110, 392, 327, 64, None), (ROWS, 192, 128, 3, 1)), ((4500, 1024, 1024, 16, None), (ROWS, 192, 128, 3, 1)),
    ((1291, 704, 2315, 8, 20), (ROWS, 64, 128, 2, 1)),
]
OF_32_BITS = [
    ((40, 72, 40, 0, 5), (EXPERTS, 16, 32, 0, 1)), ((50, 71, 40, 0, 5), (EXPERTS, 16, 16, 0, 0)), ((700, 65, 130, 0, 3), (EXPERTS, 64, 64, 1, 0)),
    ((300, 520, 72, 0, 3), (EXPERTS, 64, 64, 2, 1)), ((300, 64, 72, 0, 3), (EXPERTS, 64, 64, 3, 1)), ((8300, 100, 100, 0, 20), (EXPERTS, 64, 128, 2, 1)),
    ((300, 520, 72, 8, 3), (SEGMENTS, 64, 64, 2, 1)), ((300, 64, 72, 36, 3), (SEGMENTS, 64, 64, 3, 1)), ((8300, 100, 100, 12, 20), (SEGMENTS, 64, 128, 2, 1)),
    ((7, 72, 40, 9, None), (FEW, 8, 32, 0, 1)), ((8, 71, 40, 8, None), (FEW, 8, 32, 0, 0)),
    ((90, 72, 40, 5, None), (ROWS, 16, 16, 0, 1)), ((90, 71, 40, 8, None), (ROWS, 16, 16, 0, 0)), ((8300, 520, 40, 8, None), (ROWS, 64, 64, 2, 1)), ((700, 65, 264, 5, None), (ROWS, 64, 64, 1, 0)),
    ((8420, 64, 40, 33, None), (ROWS, 64, 64, 3, 1)), ((8300, 100, 100, 16, None), (ROWS, 64, 128, 2, 1)), ((260, 328, 3767, 8, 20), (ROWS, 64, 128, 2, 1)),
]


def cases(bits):
    return OF_16_BITS if bits == 16 else OF_32_BITS


def form_of(libpmg, bits, M, K, N, rank, S):
    type_, form = _lib.TYPE_F16 if bits == 16 else _lib.TYPE_F32, (C.c_int * 5)()
    if not rank:
        a = _lib.GroupedLinearArgs(type_, AT, K, M, AT, M, S, K, N, AT, None, None, None, 0, None, 0, 0, AT, type_, N, M, 1)
        code = libpmg.pmg_debug_grouped_form(C.byref(a), form)
    else:
        a = _lib.LoraLinearArgs(type_, AT, K, M, K, N, AT, AT, AT, rank, 4, None, AT, None if S is None else AT, M if S is None else S, None, 0, None, 0, 0, AT, type_, N)
        code = libpmg.pmg_debug_lora_form(C.byref(a), form)
    assert code == _lib.PMG_OK, libpmg.pmg_last_error()
    return tuple(form)
