"""-m gpu: the MXFP4 linear where its values, tiles, tails and overlaps have an edge, against the definition in 64 bits."""
import pytest
import torch

from test_mxfp4_gpu import act64, bytes_of, close, mx64, product64, rnd

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops():
    from fantasy_world_amd.hip_ops import HipOps
    return HipOps("cuda:0")


SPECIAL = [float("inf"), float("-inf"), float("nan"), 3e38, -3e38, 9.0, -9.0, 0.0, -0.0]


def same_special(got, want):
    """Infinities and NaN where the definition has them."""
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    assert torch.equal(torch.isinf(got) * torch.sign(got.double()).nan_to_num(), torch.isinf(want) * torch.sign(want).nan_to_num())


# one kernel each: up to 16 and 32 rows (bf16 rows), ring tiles, the 256 x 256 tile
@pytest.mark.parametrize("M,N,K", [(3, 264, 256), (20, 264, 256), (40, 264, 300), (300, 1032, 512), (4352, 4096, 1024)])
@pytest.mark.parametrize("act", ["gelu_erf", "gelu_tanh", "silu"])
def test_activations_at_infinity(ops, M, N, K, act):
    """Infinite, undefined and very large arguments by way of the bias, whose addition they survive unchanged."""
    x, w, b = rnd(M, K, seed=1), rnd(N, K, seed=2, scale=K ** -0.5), rnd(N, seed=3, dtype=torch.float32)
    at = torch.arange(len(SPECIAL)) * 29
    b[at] = torch.tensor(SPECIAL)
    lin = ops.pack_linear_mxfp4(w, b)
    got = ops.linear(x.cuda(), lin, act=act, out_f32=True)
    v = (mx64(x.cuda())[0] @ mx64(w.cuda())[0].t() + b.double().cuda())
    same_special(got, act64(v, act))
    assert torch.isinf(got[:, 0]).all() and (got[:, 0] > 0).all() and torch.isnan(got[:, 58]).all()
    keep = ~torch.isnan(got)
    assert torch.equal(ops.linear(x.cuda(), lin, act=act)[keep], got.bfloat16()[keep])


@pytest.mark.parametrize("M,N,K", [(3, 264, 256), (20, 264, 256), (40, 264, 300), (300, 1032, 512), (4352, 4096, 1024)])
@pytest.mark.parametrize("act", ["none", "relu", "gelu_erf", "gelu_tanh", "silu"])
def test_nan_products_stay_nan_through_the_activation(ops, M, N, K, act):
    """A row of x and a row of w with an infinity in one block: their whole row and column of the product is NaN, and nothing else is."""
    x, w = rnd(M, K, seed=1), rnd(N, K, seed=2, scale=K ** -0.5)
    x[M // 2, 40], w[7, 200] = float("inf"), float("nan")
    lin = ops.pack_linear_mxfp4(w, rnd(N, seed=3, dtype=torch.float32))
    want = torch.zeros(M, N, dtype=torch.bool, device="cuda")
    want[M // 2], want[:, 7] = True, True
    for kw in (dict(out_f32=True), dict()):
        assert torch.equal(torch.isnan(ops.linear(x.cuda(), lin, act=act, **kw)), want)
    # MXFP4 output: the blocks that hold a NaN, and they alone
    back = ops.dequantize_mxfp4_rows(ops.linear(x.cuda(), lin, act=act, out_mxfp4=True))
    block = want.clone()
    block[:, :32] = True
    assert torch.equal(torch.isnan(back), block)


@pytest.mark.parametrize("M", [3, 40, 1000])
def test_strides_up_to_the_limit(ops, M):
    """Weight rows almost 2^23 bytes apart, the last row ending with its buffer; activation rows the same way.  The result is that of
    close rows."""
    N, K, ld = 256, 300, (1 << 23) - 16
    x, wm = rnd(M, K, seed=1).cuda(), ops.quantize_mxfp4_rows(rnd(N, K, seed=2, scale=K ** -0.5).cuda())
    mx = ops.quantize_mxfp4_rows(x)
    want = ops.linear(mx, ops.linear_from_mxfp4(wm.q, wm.s, None, K))
    from fantasy_world_amd.hip_ops import MXFP4Rows

    def spread(rows):
        n, width = rows.shape
        far = torch.empty((n - 1) * ld + width, dtype=torch.uint8, device="cuda").as_strided((n, width), (ld, 1))
        far.copy_(rows)
        return far
    assert torch.equal(want, ops.linear(mx, ops.linear_from_mxfp4(spread(wm.q), wm.s, None, K)))
    assert torch.equal(want, ops.linear(MXFP4Rows(spread(mx.q), mx.s, K), ops.linear_from_mxfp4(wm.q, wm.s, None, K)))


@pytest.mark.parametrize("M", [5, 40, 300])
def test_outputs_beside_and_across_operands(ops, M):
    """Columns of one buffer share nothing; the residual itself is a place for the output; a shifted view of x or of the residual is refused."""
    N = K = 256
    wide, lin = rnd(M, 3 * K + 16, seed=1).cuda(), ops.pack_linear_mxfp4(rnd(N, K, seed=2, scale=K ** -0.5), rnd(N, seed=3))
    x, res, out = wide[:, :K], wide[:, K:2 * K], wide[:, 2 * K:3 * K]
    want = ops.linear(x, lin, res=res)
    assert torch.equal(ops.linear(x, lin, res=res, out=out), want)
    for bad in (dict(out=wide[:, 8:8 + N]), dict(res=res, out=wide[:, K + 8:K + 8 + N]), dict(out=wide[:, K - 1:K - 1 + N])):
        with pytest.raises(RuntimeError, match="overlaps"):
            ops.linear(x, lin, **bad)
    with pytest.raises(RuntimeError, match="overlaps"):
        ops.linear(x[:-1], lin, res=res[:-1], out=res[1:])
    f32 = torch.zeros(M, N, device="cuda")
    with pytest.raises(RuntimeError, match="overlaps"):              # the residual's memory in another type
        ops.linear(x, lin, res=f32, out=f32.view(torch.bfloat16)[:, :N])
    with pytest.raises(RuntimeError, match="overlaps"):              # the output in the linear's own codes
        ops.linear(x[:5], lin, out=lin.q[:20].reshape(-1).view(torch.bfloat16).view(5, N))
    assert torch.equal(ops.linear(x, lin, res=res, out=res), want) and torch.equal(res, want)


@pytest.mark.parametrize("M,N", [(3, 4096), (20, 4096), (300, 4096), (4352, 4096)])
@pytest.mark.parametrize("spread", [0.3, 1.0, 3.0])
def test_gelu_keeps_the_digits_of_fp32(ops, M, N, spread):
    """fp32 output of the erf GELU on arguments that carry no error of their own (a zero product, the bias is the argument).
    Each of |x| / 2, the tail's exponent, its power of two and the result rounds once or is good to a unit in the last place: 2^-24 of values that
    are no larger than |x| / 2 each, 1e-5 of the tail where it is below 1e-3.  In the 2-norm over random arguments the result is within 5e-8,
    which 0.5 x (1 + erf) in fp32 just reaches (4e-8)."""
    b = rnd(N, seed=3, scale=spread, dtype=torch.float32)
    lin = ops.pack_linear_mxfp4(rnd(N, 1024, seed=2), b)
    got = ops.linear(torch.zeros(M, 1024, dtype=torch.bfloat16, device="cuda"), lin, act="gelu_erf", out_f32=True)
    want = act64(b.double(), "gelu_erf").cuda()
    assert torch.equal(got, got[:1].expand_as(got))
    off = (got[0].double() - want).abs()
    assert (off <= 4 * 2.0 ** -24 * want.abs().clamp(min=0) + 4 * 2.0 ** -24 * 0.5 * b.double().abs().cuda()).all()
    assert (got[0].double() - want).norm() / want.norm() < 5e-8
