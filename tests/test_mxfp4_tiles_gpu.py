"""-m gpu: the 256 x 256 kernel of the MXFP4 linear, which carries the large products, against the definition in 64 bits: plain, every
epilogue, MXFP4 output, views, and the bits of its rows against the smaller tiles.

The launcher's rule is restated here (choice), and its table is read out of the source: a retuned rule that sends these shapes to another
kernel fails the first test instead of leaving the kernel untested."""
import os
import re

import pytest
import torch

from conftest import ROOT
from test_mxfp4_gpu import bytes_of, close, product64, rnd

pytestmark = pytest.mark.gpu

SHAPE = [(64, 128, 300, 2500), (64, 256, 560, 5000), (128, 256, 950, 7500), (256, 256, 1550, 11000)]
LARGE = 3

# rows % 256: none, a tail that is split off (1, 100, 128), one that is not (129, 200); N % 256: none, whole 8s, odd; K: whole slabs and not, 4 slabs and more
SHAPES = [(4352, 4096, 1024), (4196, 4096, 1024), (4196, 3590, 2048), (4196, 3600, 1283), (4224, 3591, 1000), (4097, 4096, 1536), (4225, 4090, 1024), (4296, 3848, 1280)]


def choice(M, N, K, mx=False):
    n, slabs = (N + 255) // 256 * 256 if mx else N, (K + 255) // 256
    best, least = 0, None
    for i, (bm, bn, slab, rest) in enumerate(SHAPE[:4 if slabs >= 4 else 3]):
        tiles = -(-M // bm) * -(-n // bn)
        rounds = -(-tiles // 256)
        per = slab * (rounds * 256 + tiles) // (rounds * 512) if i else (300 if tiles > 256 else 370)
        t = rounds * (slabs * per + rest)
        if least is None or t < least:
            best, least = i, t
    return best


def test_the_shapes_take_the_large_tile():
    src = open(os.path.join(ROOT, "fantasy_world_amd", "csrc", "gemm_mxfp4.hip")).read()
    table = re.search(r"shape\[4\]\[4\] = \{(.*?)\};", src).group(1)
    assert [tuple(int(v) for v in row.split(",")) for row in re.findall(r"\{(.*?)\}", table)] == SHAPE
    for M, N, K in SHAPES:
        assert choice(M, N, K) == choice(M, N, K, mx=True) == LARGE, (M, N, K)


@pytest.fixture(scope="module")
def ops():
    from fantasy_world_amd.hip_ops import HipOps
    return HipOps("cuda:0")


@pytest.mark.parametrize("M,N,K", SHAPES)
def test_plain_and_rows_of_the_smaller_tiles(ops, M, N, K):
    x, w, b = rnd(M, K, seed=1), rnd(N, K, seed=2, scale=K ** -0.5), rnd(N, seed=3, scale=0.1, dtype=torch.float32)
    lin, xd = ops.pack_linear_mxfp4(w, b), x.cuda()
    want, err = product64(x, w, b)
    got = ops.linear(xd, lin, out_f32=True)
    close(got, want, err)
    assert torch.equal(ops.linear(xd, lin), got.bfloat16())
    # rows of the first and the last tiles, from ring tiles of every kind: the same bits
    seen = set()
    for a, n in ((0, 40), (200, 300), (M - 333, 333), (M - 1000, 1000), (0, 2000), (M - 140, 140)):
        kind = choice(n, N, K)
        if kind != LARGE:
            seen.add(kind)
            assert torch.equal(ops.linear(xd[a:a + n], lin, out_f32=True), got[a:a + n]), (a, n)
    assert seen


@pytest.mark.parametrize("M,N,K", [(4196, 4096, 1024), (4196, 3590, 2048), (4097, 4096, 1536), (4225, 4090, 1024)])
@pytest.mark.parametrize("act,gate,res", [("gelu_tanh", False, None), ("gelu_erf", True, "bf16"), ("silu", True, "f32"), ("none", False, "bf16"), ("none", True, "f32")])
def test_epilogues(ops, M, N, K, act, gate, res):
    x, w, b = rnd(M, K, seed=4), rnd(N, K, seed=5, scale=K ** -0.5), rnd(N, seed=6, dtype=torch.float32)
    g1, g0 = (rnd(N, seed=7, dtype=torch.float32).cuda(), rnd(N, seed=8, dtype=torch.float32).cuda()) if gate else (None, None)
    r = None if res is None else rnd(M, N, seed=9, dtype=torch.float32 if res == "f32" else torch.bfloat16).cuda()
    lin, xd = ops.pack_linear_mxfp4(w, b), x.cuda()
    want, err = product64(x, w, b, act, g1, g0, r)
    for f32 in (True, False):
        close(ops.linear(xd, lin, act=act, g1=g1, g0=g0, res=r, out_f32=f32), want, err)
    if r is not None:
        buf = r.clone()
        assert ops.linear(xd, lin, act=act, g1=g1, g0=g0, res=buf, out=buf) is buf
        close(buf, want, err)


@pytest.mark.parametrize("M,N,K", SHAPES)
def test_mxfp4_output(ops, M, N, K):
    x, lin = rnd(M, K, seed=1).cuda(), ops.pack_linear_mxfp4(rnd(N, K, seed=2, scale=K ** -0.5), rnd(N, seed=3, scale=0.1))
    for act in ("none", "gelu_tanh"):
        got, want = ops.linear(x, lin, act=act, out_mxfp4=True), ops.quantize_mxfp4_rows(ops.linear(x, lin, act=act))
        assert torch.equal(bytes_of(got), bytes_of(want)) and torch.equal(got.q, want.q)


@pytest.mark.parametrize("M", [4196, 4225])
def test_views_and_odd_alignments(ops, M):
    N, K = 4000, 1100
    assert choice(M, N, K) == LARGE
    w, b = rnd(N, K, seed=2, scale=K ** -0.5), rnd(N, seed=3, scale=0.1, dtype=torch.float32)
    lin = ops.pack_linear_mxfp4(w, b)
    wide, big, rbig = rnd(M, K + 40, seed=1).cuda(), torch.full((M, N + 30), 7.0, device="cuda"), rnd(M, N + 24, seed=5, dtype=torch.float32).cuda()
    for ox, oo, orr in ((0, 0, 0), (8, 16, 8), (3, 5, 7)):
        x, out, res = wide[:, ox:ox + K], big[:, oo:oo + N], rbig[:, orr:orr + N]
        want, err = product64(x, w, b, res=res)
        before = big.clone()
        ops.linear(x, lin, res=res, out=out)
        close(out, want, err)
        mask = torch.ones_like(big, dtype=torch.bool)
        mask[:, oo:oo + N] = False
        assert torch.equal(big[mask], before[mask])
