"""MXFP4 entry points without a GPU: sizes at the end of the int range and operands that overlap come back as FW_E_BADARG before anything is
launched, and one row may have any stride."""
import ctypes

import pytest
import torch

from fantasy_world_amd import hip_ops
from test_mxfp4_cpu import lib, p, refused  # noqa: F401

TOP = 0x7fffffff


@pytest.mark.parametrize("K", [TOP, TOP - 254, TOP - 255])
def test_rows_too_long_for_32_bit_columns(lib, p, K):
    """Up to 2^31 - 257 values a row: past that the padded row's columns do not fit an int."""
    refused(lib, lib.fw_mxfp4_quant_rows(p(), K, 1, p(), 1 << 31, p(), 1, K, None), "fw_mxfp4_quant_rows: bf16")
    refused(lib, lib.fw_mxfp4_dequant_rows(p(), 1 << 31, p(), p(), K, 1, 1, K, None), "fw_mxfp4_dequant_rows: bf16")
    refused(lib, lib.fw_gemm_mxfp4(p(), 128, p(), p(), 128, p(), p(), 64, 1, None, 4, 64, K, None, 0, None, None, None, 0, 0, None), "fw_gemm_mxfp4")
    refused(lib, lib.fw_linear_mxfp4(p(), K, p(), 128, p(), p(), 64, 1, None, 4, 64, K, None, 0, None, None, None, 0, 0, p(), 1 << 40, None), "fw_gemm_mxfp4")
    assert lib.fw_linear_mxfp4_workspace_bytes(1, K) == (K + 255) // 256 * (128 + 256)


def test_more_rows_or_columns_than_tiles_can_count(lib, p):
    for M, N in ((TOP, 64), (TOP - 200, 64), (4, TOP), (4, TOP - 200)):
        refused(lib, lib.fw_gemm_mxfp4(p(), 128, p(), p(), 128, p(), p(), 1 << 31, 1, None, M, N, 64, None, 0, None, None, None, 0, 0, None), "2^31 - 256")
    assert lib.fw_linear_mxfp4_workspace_bytes(TOP, 64) == TOP * 128 + (1 << 26) * 256


# ---- overlaps: addresses that nothing reads, since a call that is not refused ends at the launch where there is no GPU -------------------

no_gpu = pytest.mark.skipif(torch.cuda.is_available(), reason="an accepted call stops at the launch only where there is no GPU")
far = lambda i, off=0: ctypes.c_void_p((i << 44) + off)


def shares_a_byte(a, a_pitch, a_width, b, b_pitch, b_width, rows):
    mine = {a + i * a_pitch + j for i in range(rows) for j in range(a_width)}
    return any(b + i * b_pitch + j in mine for i in range(rows) for j in range(b_width))


@no_gpu
def test_an_output_that_meets_its_residual_is_refused(lib):
    """Against a byte-by-byte comparison: equal strides, interleaved columns, unequal strides, single rows; the residual itself is accepted."""
    import random
    rng = random.Random(0)
    seen = [0, 0, 0]
    for _ in range(1500):
        M, N = rng.choice([1, 2, 3, 7]), rng.choice([1, 2, 5])
        odt, rdt = rng.choice([(2, 2), (1, 1), (1, 2), (2, 1)])
        ce, re = 2 * odt, 2 * rdt
        ldc = N + rng.choice([0, 0, 1, 3, 8])
        ldr = rng.choice([ldc, N, N + 2, 2 * ldc, 3 * ldc + 1])
        base = 1 << 44
        at = base + rng.choice([0, 0, 4, -4, 8, 4 * N, ldc * ce, -ldc * ce, 2 * ldc * ce, 4 * rng.randrange(-40, 40)]) // max(ce, re) * max(ce, re)
        rc = lib.fw_gemm_mxfp4(far(2), 128, far(3), far(4), 128, far(5), ctypes.c_void_p(base), ldc, odt, None, M, N, 64, None, 0, None, None, ctypes.c_void_p(at), ldr, rdt, None)
        itself = at == base and odt == rdt and (ldc == ldr or M == 1)
        bad = shares_a_byte(base, ldc * ce, N * ce, at, ldr * re, N * re, M) and not itself
        assert (rc == -1) == bad, (M, N, odt, rdt, ldc, ldr, at - base, rc, lib.fw_last_error())
        seen[0 if itself else 1 if bad else 2] += 1
    assert min(seen) > 50, seen


@no_gpu
def test_an_output_that_meets_an_operand_is_refused(lib):
    base = dict(A=far(1), lda=128, sa=far(2), W=far(3), ldw=128, sw=far(4), C=far(5), ldc=64, odt=1, cs=None, M=40, N=64, K=64, bias=far(6), act=0, g1=far(7), g0=far(8),
                res=None, ldr=0, rdt=0, st=None)
    call = lambda **k: lib.fw_gemm_mxfp4(*[k.get(n, v) for n, v in base.items()])
    assert call() not in (0, -1)
    for i, size in ((1, 40 * 128), (2, 2 * 256), (3, 64 * 128), (4, 2 * 256), (6, 256), (7, 256), (8, 256)):
        for at in (0, size - 16, -40 * 128 + 16):
            refused(lib, call(C=far(i, at)), "overlaps")
            refused(lib, call(C=far(i, at), odt=3, ldc=128, cs=far(9)), "overlaps")
            refused(lib, call(odt=3, ldc=128, cs=far(i, max(at, -512 + 16))), "overlaps")
        assert call(C=far(i, size)) != -1 and call(C=far(i, -40 * 128)) != -1
    refused(lib, call(odt=3, ldc=128, cs=far(5, 40 * 128 - 16)), "overlaps")
    refused(lib, call(odt=3, ldc=128, cs=far(9), res=far(5), ldr=64, rdt=1), "overlaps")
    # the whole linear: bf16 rows quantised inside the product or in the workspace; columns of one buffer interleave without meeting
    base = dict(x=far(1), ldx=128, W=far(3), ldw=128, sw=far(4), C=far(5), ldc=64, odt=1, cs=None, M=40, N=64, K=64, bias=None, act=0, g1=None, g0=None, res=None, ldr=0, rdt=0,
                ws=far(6), n=1 << 20, st=None)
    whole = lambda **k: lib.fw_linear_mxfp4(*[k.get(n, v) for n, v in base.items()])
    for M in (8, 40):
        refused(lib, whole(M=M, C=far(1, 256), ldc=128), "overlaps")
        refused(lib, whole(M=M, C=far(1, 126), ldc=128), "overlaps")
        assert whole(M=M, C=far(1, 128), ldc=128) != -1
    refused(lib, whole(C=far(6, 40 * 128)), "overlaps")
    refused(lib, whole(x=far(6, 0)), "overlap")


@no_gpu
def test_rows_that_meet_their_codes_are_refused(lib):
    quant = lambda x, q, s: lib.fw_mxfp4_quant_rows(x, 512, 1, q, 1024, s, 40, 256, None)
    assert quant(far(1), far(2), far(3)) != -1 and quant(far(1), far(1, 512), far(3)) != -1          # behind the 512 bytes of a row of 1024
    for q, s in ((far(1), far(3)), (far(1, 496), far(3)), (far(2), far(1, 4)), (far(2), far(2, 16))):
        refused(lib, quant(far(1), q, s), "overlap")
    back = lambda q, s, y: lib.fw_mxfp4_dequant_rows(q, 512, s, y, 256, 1, 40, 256, None)
    assert back(far(1), far(2), far(3)) != -1
    for y in (far(1), far(1, 128 - 512 * 40), far(2, 500)):
        refused(lib, back(far(1), far(2), y), "overlap")


@no_gpu
def test_a_norm_whose_outputs_meet_an_operand_is_refused(lib):
    base = dict(x=far(1), ldx=64, xo=far(2), ldxo=64, xdt=1, y=far(3), ldy=64, ydt=1, bias=None, g1=None, g0=None, post=0, post_w=None, norm=1, w=None, b=None, scale=None,
                shift=None, eps=ctypes.c_float(1e-6), h=far(4), ldh=64, hdt=1, hs=None, rows=40, C=64, rpm=10, st=None)
    f = lambda **k: lib.fw_residual_norm(*[k.get(n, v) for n, v in base.items()])
    # an output may be x or y, the same rows in the same type
    for ok in (dict(), dict(xo=far(1)), dict(xo=far(3)), dict(h=far(1)), dict(h=far(3)), dict(xo=far(1), h=far(3)), dict(y=far(1), xo=far(1)), dict(y=None, h=far(1)),
               dict(h=far(2, 128), ldxo=128, ldh=128)):
        assert f(**ok) not in (0, -1), (ok, lib.fw_last_error())
    for bad in (dict(xo=far(1, 2)), dict(xo=far(1, 128)), dict(xo=far(1), ldxo=65), dict(xo=far(3, 2)), dict(h=far(2)), dict(h=far(2, 128)), dict(h=far(1, 128)),
                dict(h=far(3, 128)), dict(xo=far(1), h=far(1)), dict(y=None, h=far(1, 2)), dict(xdt=2, h=far(1)), dict(xdt=2, xo=far(3)), dict(ydt=2, h=far(3)),
                dict(hdt=3, ldh=128, hs=far(5), h=far(1)), dict(hdt=3, ldh=128, hs=far(1)), dict(hdt=3, ldh=128, hs=far(4, 128)), dict(hdt=3, ldh=128, hs=far(2))):
        refused(lib, f(**bad), "overlaps")
    for v, runs in (("bias", 1), ("w", 1), ("g1", 4), ("g0", 4), ("scale", 4), ("shift", 4)):
        for out in (2, 4):
            refused(lib, f(**{v: far(out, 128)}), "overlaps")
            refused(lib, f(**{v: far(out, -256 * runs + 16)}), "overlaps")
            assert f(**{v: far(out, -256 * runs)}) != -1
    refused(lib, f(post=1, post_w=far(4)), "overlaps")
    refused(lib, f(w=far(6), b=far(4)), "overlaps")


def test_one_row_of_codes_has_any_stride():
    """A tensor of one row may carry any stride for it; the rows' distance is then their width."""
    s = torch.zeros(1, 2, 32, 8, dtype=torch.uint8)
    for q in (torch.zeros(256, 1, dtype=torch.uint8).t(), torch.zeros(1, 256, dtype=torch.uint8).as_strided((1, 256), (7, 1)), torch.zeros(4, 256, dtype=torch.uint8)[1:2]):
        assert q.shape == (1, 256) and hip_ops.MXFP4Rows(q, s, 300).ldq == 256
    assert hip_ops.MXFP4Rows(torch.zeros(4, 400, dtype=torch.uint8)[:, :256], s, 300).ldq == 400
