"""The C entry points of attention with modified scores and of the caches around it reject bad arguments before
they touch the GPU: every call here is refused (or has nothing to do), so its pointers are never followed."""
import ctypes
import os
import re

import pytest

REPO = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
LIB = os.path.join(REPO, "flash_attn_v100_amd", "libflash_attn_mi355x.so")
OK, INVALID, WORKSPACE, UNSUPPORTED = 0, 1, 2, 3
P, I, F, Z = ctypes.c_void_p, ctypes.c_int, ctypes.c_float, ctypes.c_size_t
PTR = 1 << 20  # an aligned address that nothing reads


@pytest.fixture(scope="module")
def lib():
    import torch  # noqa: F401  (shares torch's HIP runtime)

    L = ctypes.CDLL(LIB)
    L.fa_last_error.restype = ctypes.c_char_p
    L.fa_scored_fp16.argtypes = L.fa_scored_fp32.argtypes = [P] * 5 + [I] * 6 + [F] + [P] * 4
    L.fa_scored_backward_fp16.argtypes = L.fa_scored_backward_fp32.argtypes = [P] * 9 + [I] * 6 + [F] + [P] * 4 + [Z, P]
    L.fa_decode_scored_fp16.argtypes = [P] * 5 + [I] * 5 + [F] + [P] * 2 + [Z, P]
    L.fa_decode_weighted_fp16.argtypes = [P] * 7 + [I] * 5 + [F] + [P] * 2 + [Z, P, Z, P]
    L.fa_paged_append_kv8.argtypes = [P] * 9 + [I] * 9 + [P]
    L.fa_paged_decode_kv8.argtypes = [P] * 8 + [I] * 8 + [F] + [P] * 2 + [Z, P]
    L.fa_evict_by_weight.argtypes = [P] * 9 + [I] * 7 + [P]
    for name, n in (("fa_scored_backward_workspace_size", 3), ("fa_decode_weighted_scratch_size", 3),
                    ("fa_decode_workspace_size", 5)):
        getattr(L, name).restype, getattr(L, name).argtypes = Z, [I] * n
    return L


def refused(lib, rc, code, name):
    assert rc == code, (rc, lib.fa_last_error())
    if code != OK:
        assert lib.fa_last_error().decode().startswith(name + ":")


SIZES = dict(B=1, HQ=4, HKV=2, N=64, D=64, causal=1, cap=0.0, prefix=None)
BAD_SCORED = [(dict(B=-1), INVALID), (dict(N=-1), INVALID), (dict(HQ=0), INVALID), (dict(HKV=0), INVALID), (dict(D=0), INVALID),
              (dict(HQ=3), INVALID), (dict(HQ=1), INVALID), (dict(D=257), UNSUPPORTED), (dict(cap=-1.0), INVALID),
              (dict(cap=1e-3), INVALID), (dict(cap=1e4), INVALID), (dict(cap=float("nan")), INVALID),
              (dict(cap=float("inf")), INVALID), (dict(causal=0, prefix=PTR), INVALID),
              (dict(B=1 << 20, HQ=1 << 10, HKV=1 << 10), UNSUPPORTED), (dict(N=0x7fffffff), UNSUPPORTED),
              (dict(B=0), OK), (dict(N=0), OK)]


@pytest.mark.parametrize("change,code", BAD_SCORED)
@pytest.mark.parametrize("half", [True, False])
def test_scored(lib, half, change, code):
    a = {**SIZES, **change}
    sizes = (a["B"], a["HQ"], a["HKV"], a["N"], a["D"], a["causal"], a["cap"], None, None, a["prefix"])
    kind = "fp16" if half else "fp32"
    refused(lib, getattr(lib, "fa_scored_" + kind)(PTR, PTR, PTR, PTR, None, *sizes, None), code, "fa_scored_" + kind)
    refused(lib, getattr(lib, "fa_scored_backward_" + kind)(*[PTR] * 9, *sizes, PTR, 1 << 40, None), code,
            "fa_scored_backward_" + kind)


@pytest.mark.parametrize("half", [True, False])
def test_scored_pointers_widths_and_workspace(lib, half):
    kind = "fp16" if half else "fp32"
    fwd, bwd = getattr(lib, "fa_scored_" + kind), getattr(lib, "fa_scored_backward_" + kind)
    sizes = (1, 4, 2, 64, 64, 1, 0.0, None, None, None)
    for i in range(4):
        args = [PTR] * 4
        args[i] = None
        refused(lib, fwd(*args, None, *sizes, None), INVALID, "fa_scored_" + kind)
    need = lib.fa_scored_backward_workspace_size(1, 4, 64)
    assert need == 2 * 4 * 64 * 4
    for i in range(9):
        args = [PTR] * 9
        args[i] = None
        refused(lib, bwd(*args, *sizes, PTR, need, None), INVALID, "fa_scored_backward_" + kind)
    refused(lib, bwd(*[PTR] * 9, *sizes, PTR, need - 1, None), WORKSPACE, "fa_scored_backward_" + kind)
    refused(lib, bwd(*[PTR] * 9, *sizes, None, need, None), WORKSPACE, "fa_scored_backward_" + kind)
    wide = (1, 4, 2, 64, 136, 1, 0.0, None, None, None)
    refused(lib, bwd(*[PTR] * 9, *wide, PTR, 1 << 40, None), UNSUPPORTED, "fa_scored_backward_" + kind)
    if not half:
        refused(lib, fwd(*[PTR] * 4, None, *wide, None), UNSUPPORTED, "fa_scored_fp32")
    assert [lib.fa_scored_backward_workspace_size(*s) for s in ((0, 4, 64), (1, 0, 64), (1, 4, 0), (-1, 4, 64))] == [0] * 4


DECODE = dict(B=2, HQ=4, HKV=2, N=64, D=64, cap=0.0)
BAD_DECODE = [(dict(B=-1), INVALID), (dict(HQ=0), INVALID), (dict(HKV=0), INVALID), (dict(D=0), INVALID), (dict(HQ=3), INVALID),
              (dict(HQ=1), INVALID), (dict(D=257), UNSUPPORTED), (dict(cap=-1.0), INVALID), (dict(cap=float("nan")), INVALID),
              (dict(cap=5e3), INVALID), (dict(N=0), INVALID), (dict(N=-5), INVALID), (dict(N=1 << 21), UNSUPPORTED),
              (dict(B=1 << 20, HQ=1 << 11, HKV=1 << 11), UNSUPPORTED), (dict(B=0), OK)]


@pytest.mark.parametrize("change,code", BAD_DECODE)
def test_decode(lib, change, code):
    a = {**DECODE, **change}
    sizes = (a["B"], a["HQ"], a["HKV"], a["N"], a["D"], a["cap"], None)
    refused(lib, lib.fa_decode_scored_fp16(*[PTR] * 5, *sizes, PTR, 1 << 40, None), code, "fa_decode_scored_fp16")
    far = PTR + (1 << 50)
    refused(lib, lib.fa_decode_weighted_fp16(*[PTR] * 6, far, *sizes, PTR, 1 << 60, PTR, 1 << 40, None), code,
            "fa_decode_weighted_fp16")


def test_decode_pointers_and_workspace(lib):
    sizes = (2, 4, 2, 64, 64, 0.0, None)
    scratch = lib.fa_decode_weighted_scratch_size(2, 4, 64)
    assert scratch == 2 * 4 * 65 * 4
    for i in range(5):
        args = [PTR] * 5
        args[i] = None
        refused(lib, lib.fa_decode_scored_fp16(*args, *sizes, PTR, 1 << 40, None), INVALID, "fa_decode_scored_fp16")
    for i in range(7):
        args = [PTR] * 7
        args[i] = None
        refused(lib, lib.fa_decode_weighted_fp16(*args, *sizes, PTR, scratch, PTR, 1 << 40, None), INVALID, "fa_decode_weighted_fp16")
    for s, n, code in ((None, scratch, WORKSPACE), (PTR, scratch - 1, WORKSPACE), (PTR + 4, scratch, INVALID)):
        refused(lib, lib.fa_decode_weighted_fp16(*[PTR] * 7, *sizes, s, n, PTR, 1 << 40, None), code, "fa_decode_weighted_fp16")
    many = (1, 1, 1, 65536, 64, 0.0, None)
    need = lib.fa_decode_workspace_size(1, 1, 1, 65536, 64)
    for ws, n in ((None, need), (PTR, 0)):
        refused(lib, lib.fa_decode_scored_fp16(*[PTR] * 5, *many, ws, n, None), WORKSPACE, "fa_decode_scored_fp16")
    assert lib.fa_decode_weighted_scratch_size(0, 4, 64) == lib.fa_decode_weighted_scratch_size(2, 4, -1) == 0
    pairs = (65536, 1, 1, 8, 64, 0.0, None)
    refused(lib, lib.fa_decode_weighted_fp16(*[PTR] * 7, *pairs, PTR, 1 << 40, PTR, 1 << 40, None), UNSUPPORTED, "fa_decode_weighted_fp16")


@pytest.mark.parametrize("shift", [4, 128, 2 * 2 * 64 * 4 - 4])
def test_weights_that_overlap_in_part(lib, shift):
    sizes = (2, 4, 2, 64, 64, 0.0, None)
    for w, out in ((PTR, PTR + shift), (PTR + shift, PTR)):
        refused(lib, lib.fa_decode_weighted_fp16(*[PTR] * 5, w, out, *sizes, PTR, 1 << 40, PTR, 1 << 40, None), INVALID,
                "fa_decode_weighted_fp16")


# keys at which one unit, or a few, are split for certain
@pytest.mark.parametrize("b,hq,hkv,n,d", [(1, 1, 1, 8192, 64), (1, 32, 8, 4097, 128), (3, 48, 2, 20000, 80), (2, 33, 1, 65536, 256),
                                          (128, 32, 8, 32768, 128), (512, 8, 8, 32768, 64), (600, 4, 4, 100000, 40)])
def test_decode_workspace_covers_the_plan(lib, b, hq, hkv, n, d):
    rc = lib.fa_decode_scored_fp16(*[PTR] * 5, b, hq, hkv, n, d, 0.0, None, None, 0, None)
    assert rc == WORKSPACE
    need = int(re.search(rb"workspace of (\d+) bytes", lib.fa_last_error()).group(1))
    assert need <= lib.fa_decode_workspace_size(b, hq, hkv, n, d)


APPEND = dict(fp8=0, B=2, total=4, max_new=2, HKV=2, D=64, pages=6, page=16, blocks=3)
PAGED = dict(fp8=0, B=2, HQ=4, HKV=2, D=64, pages=6, page=16, blocks=3, cap=0.0)


@pytest.mark.parametrize("change,code", [
    (dict(B=-1), INVALID), (dict(total=-1), INVALID), (dict(max_new=-1), INVALID), (dict(HKV=0), INVALID), (dict(D=0), INVALID),
    (dict(pages=-1), INVALID), (dict(blocks=-1), INVALID), (dict(D=272), UNSUPPORTED), (dict(page=8), UNSUPPORTED),
    (dict(page=24), UNSUPPORTED), (dict(page=512), UNSUPPORTED), (dict(page=0), UNSUPPORTED), (dict(page=-16), UNSUPPORTED),
    (dict(B=1 << 20, total=1 << 30, max_new=1 << 30), UNSUPPORTED),
    (dict(B=0), OK), (dict(total=0), OK), (dict(max_new=0), OK), (dict(pages=0), OK), (dict(blocks=0), OK)])
def test_append(lib, change, code):
    refused(lib, lib.fa_paged_append_kv8(*[PTR] * 9, *{**APPEND, **change}.values(), None), code, "fa_paged_append_kv8")


def test_append_pointers(lib):
    for i in range(9):
        args = [PTR] * 9
        args[i] = None
        refused(lib, lib.fa_paged_append_kv8(*args, *APPEND.values(), None), INVALID, "fa_paged_append_kv8")


@pytest.mark.parametrize("change,code", [
    (dict(B=-1), INVALID), (dict(HQ=3), INVALID), (dict(HQ=1), INVALID), (dict(HKV=0), INVALID), (dict(D=0), INVALID),
    (dict(D=272), UNSUPPORTED), (dict(page=8), UNSUPPORTED), (dict(page=24), UNSUPPORTED), (dict(page=512), UNSUPPORTED),
    (dict(pages=-1), INVALID), (dict(blocks=-1), INVALID), (dict(blocks=0x7fffffff), UNSUPPORTED), (dict(cap=-1.0), INVALID),
    (dict(cap=float("nan")), INVALID), (dict(blocks=1 << 20), UNSUPPORTED), (dict(B=0), OK)])
def test_paged_decode(lib, change, code):
    refused(lib, lib.fa_paged_decode_kv8(*[PTR] * 8, *{**PAGED, **change}.values(), None, PTR, 1 << 40, None), code,
            "fa_paged_decode_kv8")


def test_paged_decode_pointers_and_workspace(lib):
    for i in range(8):
        args = [PTR] * 8
        args[i] = None
        refused(lib, lib.fa_paged_decode_kv8(*args, *PAGED.values(), None, PTR, 1 << 40, None), INVALID, "fa_paged_decode_kv8")
    long = {**PAGED, "blocks": 4096}
    refused(lib, lib.fa_paged_decode_kv8(*[PTR] * 8, *long.values(), None, None, 0, None), WORKSPACE, "fa_paged_decode_kv8")


EVICT = dict(B=2, HKV=2, N=64, D=64, budget=8, recent=2, capacity=16)


@pytest.mark.parametrize("change,code", [
    (dict(B=-1), INVALID), (dict(HKV=0), INVALID), (dict(N=-1), INVALID), (dict(D=0), INVALID), (dict(budget=-1), INVALID),
    (dict(recent=-1), INVALID), (dict(capacity=-1), INVALID), (dict(recent=9), INVALID), (dict(budget=17), INVALID),
    (dict(B=65536, HKV=1), UNSUPPORTED), (dict(N=0x7fffffff), UNSUPPORTED), (dict(capacity=0x7fffffff), UNSUPPORTED), (dict(B=0), OK)])
def test_evict(lib, change, code):
    refused(lib, lib.fa_evict_by_weight(*[PTR] * 9, *{**EVICT, **change}.values(), None), code, "fa_evict_by_weight")


def test_evict_pointers(lib):
    for i in range(9):
        args = [PTR] * 9
        args[i] = None
        refused(lib, lib.fa_evict_by_weight(*args, *EVICT.values(), None), INVALID, "fa_evict_by_weight")
