"""MXFP4 entry points without a GPU: every bad call comes back as FW_E_BADARG with a message before anything is launched, empty problems
are accepted, and the Python containers refuse rows that are not MXFP4 rows."""
import ctypes

import pytest
import torch

from fantasy_world_amd import hip_ops

F32 = ctypes.c_float


@pytest.fixture(scope="module")
def lib():
    return hip_ops.load_library()


@pytest.fixture(scope="module")
def p():
    buf = (ctypes.c_uint8 * 8192)()
    base = ctypes.addressof(buf)
    yield lambda off=0: ctypes.c_void_p(base + (-base) % 16 + off)
    del buf


def refused(lib, rc, needle):
    assert rc == -1 and needle in lib.fw_last_error().decode(), (rc, lib.fw_last_error())


def test_quantiser_refusals(lib, p):
    q = lambda **k: lib.fw_mxfp4_quant_rows(*[k.get(n, d) for n, d in dict(x=p(), ldx=64, dt=1, q=p(), ldq=128, s=p(), M=4, K=64, st=None).items()])
    for bad in (dict(x=None), dict(q=None), dict(s=None), dict(ldx=63), dict(dt=0), dict(dt=3), dict(ldq=112), dict(ldq=136), dict(K=0), dict(K=-5), dict(K=257, ldx=257),
                dict(q=p(8)), dict(s=p(2)), dict(x=p(1)), dict(x=p(2), dt=2)):
        refused(lib, q(**bad), "fw_mxfp4_quant_rows")
    refused(lib, q(M=0x7fffffff, K=8192, ldx=8192, ldq=4096), "grid too large")
    assert q(M=0) == 0
    d = lambda **k: lib.fw_mxfp4_dequant_rows(*[k.get(n, v) for n, v in dict(q=p(), ldq=128, s=p(), y=p(), ldy=64, dt=1, M=4, K=64, st=None).items()])
    for bad in (dict(q=None), dict(s=None), dict(y=None), dict(ldy=63), dict(dt=3), dict(ldq=64), dict(K=0), dict(q=p(4)), dict(y=p(1))):
        refused(lib, d(**bad), "fw_mxfp4_dequant_rows")
    assert d(M=0) == 0


def test_product_refusals(lib, p):
    base = dict(A=p(), lda=128, sa=p(), W=p(), ldw=128, sw=p(), C=p(), ldc=64, odt=1, cs=None, M=4, N=64, K=64, bias=None, act=0, g1=None, g0=None, res=None, ldr=0, rdt=0, st=None)
    g = lambda **k: lib.fw_gemm_mxfp4(*[k.get(n, v) for n, v in base.items()])
    for bad in (dict(A=None), dict(W=None), dict(sa=None), dict(sw=None), dict(C=None), dict(lda=112), dict(ldw=136), dict(lda=1 << 23), dict(K=0), dict(K=257), dict(A=p(8)),
                dict(W=p(4)), dict(sa=p(1)), dict(act=5), dict(act=-1), dict(odt=0), dict(odt=4), dict(ldc=63), dict(C=p(1)), dict(C=p(2), odt=2), dict(odt=3, ldc=128),
                dict(odt=3, cs=p(), ldc=64), dict(odt=3, cs=p(), ldc=136), dict(odt=3, cs=p(2), ldc=128), dict(odt=3, cs=p(), ldc=128, C=p(8)), dict(rdt=1), dict(rdt=3, res=p(), ldr=64),
                dict(rdt=2, res=p(), ldr=63), dict(rdt=2, res=p(2), ldr=64), dict(bias=p(2)), dict(g1=p(1)), dict(g0=p(3))):
        refused(lib, g(**bad), "fw_gemm_mxfp4")
    assert g(M=0) == 0 and g(N=0) == 0


def test_whole_linear_refusals(lib, p):
    base = dict(x=p(), ldx=64, W=p(), ldw=128, sw=p(), C=p(), ldc=64, odt=1, cs=None, M=40, N=64, K=64, bias=None, act=0, g1=None, g0=None, res=None, ldr=0, rdt=0, ws=p(), n=1 << 20, st=None)
    f = lambda **k: lib.fw_linear_mxfp4(*[k.get(n, v) for n, v in base.items()])
    assert lib.fw_linear_mxfp4_workspace_bytes(20, 64) == 20 * 128 + 256 and lib.fw_linear_mxfp4_workspace_bytes(33, 257) == 33 * 256 + 2 * 512
    assert lib.fw_linear_mxfp4_workspace_bytes(0, 64) == 0 and lib.fw_linear_mxfp4_workspace_bytes(4, 0) == 0
    assert lib.fw_linear_mxfp4_workspace_bytes(1 << 20, 13824) == (1 << 20) * 54 * 128 + (1 << 15) * 54 * 256
    for bad in (dict(x=None), dict(ldx=63), dict(x=p(1)), dict(ws=None, n=0), dict(n=40 * 128 + 511), dict(ws=p(8)),
                dict(M=20, K=63, ws=None, n=0), dict(M=4, K=63, ws=None, n=0), dict(M=4, ldx=65, ws=None, n=0), dict(M=4, x=p(2), ws=None, n=0)):
        refused(lib, f(**bad), "fw_linear_mxfp4")
    for m in (4, 20, 40):                    # one launch or two: the product's own refusals come first
        for bad in (dict(W=None), dict(ldw=112), dict(C=None), dict(act=9), dict(odt=0), dict(ldc=63), dict(odt=3), dict(rdt=1), dict(g1=p(2)), dict(K=0), dict(sw=p(1))):
            refused(lib, f(M=m, **bad), "fw_gemm_mxfp4" if "K" not in bad or m == 4 else "")
    assert f(M=0) == 0 and f(N=0) == 0


def test_residual_norm_refusals(lib, p):
    base = dict(x=p(), ldx=64, xo=p(), ldxo=64, xdt=2, y=p(), ldy=64, ydt=1, bias=None, g1=None, g0=None, post=0, post_w=None, norm=1, w=None, b=None, scale=None, shift=None,
                eps=F32(1e-6), h=p(), ldh=64, hdt=1, hs=None, rows=4, C=64, rpm=4, st=None)
    f = lambda **k: lib.fw_residual_norm(*[k.get(n, v) for n, v in base.items()])
    for bad in (dict(x=None), dict(h=None), dict(C=0), dict(C=8193, ldx=9000), dict(ldx=63), dict(xdt=0), dict(xdt=3), dict(x=p(2)), dict(rpm=0), dict(ydt=0), dict(ldy=63), dict(y=p(1)),
                dict(xo=None), dict(ldxo=63), dict(xo=p(2)), dict(norm=0), dict(norm=3), dict(post=3), dict(post=-1), dict(post_w=p()), dict(b=p()), dict(hdt=2), dict(ldh=63), dict(h=p(1)),
                dict(hdt=3, ldh=128), dict(hdt=3, hs=p(), ldh=64), dict(hdt=3, hs=p(2), ldh=128), dict(bias=p(2)), dict(scale=p(1)),
                dict(y=None, bias=p()), dict(y=None, g1=p()), dict(y=None, g0=p()), dict(y=None, post=1)):
        refused(lib, f(**bad), "fw_residual_norm")
    assert f(rows=0) == 0


def test_containers_refuse_what_is_not_mxfp4_rows():
    q, s = torch.zeros(40, 256, dtype=torch.uint8), torch.zeros(2, 2, 32, 8, dtype=torch.uint8)
    assert hip_ops.MXFP4Rows(q, s, 300).shape == (40, 300) and hip_ops.LinearMXFP4(q, s, torch.zeros(40), 512).N == 40
    for a, b, K in ((q, s, 256), (q, s, 513), (q, s, 0), (q[:, ::2], s, 256), (q.to(torch.int8), s, 300), (q, s[:1], 300), (q, s.int(), 300), (q[0], s, 300), (q, s.transpose(0, 1), 300)):
        with pytest.raises(ValueError):
            hip_ops.MXFP4Rows(a, b, K)
    for bias in (torch.zeros(39), torch.zeros(40, dtype=torch.bfloat16), torch.zeros(80)[::2], torch.zeros(1, 40)):
        with pytest.raises(ValueError):
            hip_ops.LinearMXFP4(q, s, bias, 300)
