"""-m gpu: MXFP4 rows and the MXFP4 linear (include/fw_mi355x.h) against their definition in 64 bits.

Tolerances.  Codes and scale bytes are integer work: exact.  A product: products of e2m1 values and their sums inside one MFMA are exact in
fp32, every further addition rounds by at most 2^-24 of the running sum; n = K / 64 instructions in a row, so an output is off by at most
n * 2^-24 * sum |terms| (+ 4 * 2^-24 of the largest intermediate for the epilogue's own operations and 2^-19 where an activation's
exponential is involved: v_exp_f32 and v_rcp_f32 are good to a few units of 2^-23 and act on arguments up to ~16).  A bf16 output adds half
a step, 2^-8 of the value (relative to the next power of two below: 2^-9 to 2^-8); an MXFP4 output is compared code by code with the
quantised bf16 output of the same call."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

LEVELS = torch.tensor([0, .5, 1, 1.5, 2, 3, 4, 6], dtype=torch.float64)


@pytest.fixture(scope="module")
def ops():
    from fantasy_world_amd.hip_ops import HipOps
    return HipOps("cuda:0")


def mx64(x):
    """(values, scale bytes) of the definition, by search over the levels, where x lies."""
    rows, K = x.shape
    kp = (K + 255) // 256 * 256
    v = torch.zeros(rows, kp, dtype=torch.float64, device=x.device)
    v[:, :K] = x.double()
    v = v.view(rows, -1, 32)
    top = v.abs().amax(2)
    nan = ~torch.isfinite(v).all(2)
    m, e = torch.frexp(torch.where(nan, torch.ones_like(top), top))
    byte = torch.where(top == 0, torch.zeros_like(e), (e - 1 - 2 + (m >= 0.875).int() + 127).clamp(0, 252))
    # magnitudes below the smallest normal fp32 count as exponent field 0: the clamp above covers them
    scale = torch.exp2(byte.double() - 127).unsqueeze(2)       # exact for whole numbers; torch.pow(2, n) is not, on a GPU
    a = torch.where(nan.unsqueeze(2), torch.zeros_like(v), v / scale)
    level = LEVELS.to(x.device)
    dist = (a.abs().clamp(max=6).unsqueeze(-1) - level).abs()
    best = dist.amin(-1, keepdim=True)
    tie = dist == best
    even = torch.tensor([True, False] * 4, device=x.device)
    pick = torch.where((tie & even).any(-1), (tie & even).int().argmax(-1), tie.int().argmax(-1))
    out = level[pick] * torch.sign(a) * scale
    out = torch.where(nan.unsqueeze(2), torch.full_like(out, math.nan), out)
    byte = torch.where(nan, torch.full_like(byte, 255), byte)
    return out.view(rows, -1)[:, :K], byte


def bytes_of(mx):
    """Scale bytes [M, Kp / 32] of MXFP4Rows."""
    return mx.s.cpu().permute(0, 2, 1, 3).reshape(mx.s.shape[0] * 32, -1)[:mx.M].int()


def check_rows(mx, x, ops):
    want, byte = mx64(x.cpu())
    assert torch.equal(bytes_of(mx), byte)
    for dt in (torch.bfloat16, torch.float32):
        got = ops.dequantize_mxfp4_rows(mx, dt)
        assert got.dtype == dt and got.shape == x.shape
        assert torch.equal(torch.nan_to_num(got.cpu().double(), nan=-77.0), torch.nan_to_num(want, nan=-77.0))
    pad = mx.q[:, (mx.K + 1) // 2:]
    assert not pad.any() and (mx.K % 2 == 0 or not (mx.q[:, mx.K // 2] >> 4).any())


def rnd(*shape, seed=0, scale=1.0, dtype=torch.bfloat16):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(*shape, generator=g) * scale).to(dtype)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("M,K", [(1, 1), (1, 5120), (3, 31), (33, 257), (31, 64), (64, 1000), (257, 1283), (130, 1024)])
def test_rows_are_exact(ops, M, K, dtype):
    x = (rnd(M, K, seed=M + K, dtype=torch.float32) * torch.exp(2 * rnd(M, K, seed=K, dtype=torch.float32))).to(dtype)
    check_rows(ops.quantize_mxfp4_rows(x.cuda()), x, ops)


def test_rows_of_views_and_of_nothing(ops):
    wide = rnd(70, 900, seed=1).cuda()
    for x in (wide[:, 8:520], wide[:, 3:516], wide[::3, 64:320], wide.float()[:, 5:600], wide[:1, :7]):
        check_rows(ops.quantize_mxfp4_rows(x), x, ops)
    mx = ops.quantize_mxfp4_rows(wide[:0])
    assert mx.shape == (0, 900) and ops.dequantize_mxfp4_rows(mx).shape == (0, 900)


def test_rows_every_bf16_value_and_every_border(ops):
    """All finite bf16 magnitudes, each alone with a top that fixes the scale; zeros, subnormals, the largest finite values, ties."""
    every = torch.arange(0x7f80, dtype=torch.int32).to(torch.int16).view(torch.bfloat16)
    alone = torch.zeros(every.numel(), 32, dtype=torch.bfloat16)
    alone[:, 5], alone[:, 17] = every, -every
    check_rows(ops.quantize_mxfp4_rows(alone.cuda()), alone, ops)
    tops = torch.tensor([2.0 ** e * m for e in (-133, -126, -125, -20, 0, 3, 100, 127) for m in (1.0, 1.25, 1.5, 1.7421875, 1.75, 1.9921875)])
    ratios = torch.tensor([0.0, 0.03, 0.0625, 0.125, 0.1875, 0.25, 0.3125, 0.4375, 0.5, 0.625, 0.75, 0.875, 0.99, 1.0])
    grid = torch.zeros(tops.numel(), 32)
    grid[:, 0], grid[:, 1:1 + ratios.numel()] = tops, -tops[:, None] * ratios
    for dt in (torch.bfloat16, torch.float32):
        x = grid.to(dt)
        check_rows(ops.quantize_mxfp4_rows(x.cuda()), x, ops)


def test_infinities_and_nan_stay_in_their_block(ops):
    x = rnd(4, 128, seed=3)
    x[1, 40], x[2, 100], x[3, 0] = float("inf"), float("nan"), float("-inf")
    mx = ops.quantize_mxfp4_rows(x.cuda())
    check_rows(mx, x, ops)
    lin = ops.pack_linear_mxfp4(rnd(64, 128, seed=4).cuda(), None)
    y = ops.linear(mx, lin)
    assert torch.isfinite(y[0]).all() and torch.isnan(y[1:]).all()
    w = rnd(64, 128, seed=4)
    w[7, 3] = float("inf")
    y = ops.linear(x[:1].cuda(), ops.pack_linear_mxfp4(w.cuda(), None))
    assert torch.isnan(y[:, 7]).all() and torch.isfinite(y[:, :7]).all() and torch.isfinite(y[:, 8:]).all()


# ---- the product ----------------------------------------------------------------------------------------------------------------------


def act64(v, act):
    return {"none": lambda: v, "relu": lambda: v.clamp(min=0), "silu": lambda: v * torch.sigmoid(v),
            "gelu_tanh": lambda: 0.5 * v * (1 + torch.tanh((2 / math.pi) ** 0.5 * (v + 0.044715 * v ** 3))),
            "gelu_erf": lambda: 0.5 * v * torch.special.erfc(-v / 2 ** 0.5)}[act]()


def product64(x, w, b=None, act="none", g1=None, g0=None, res=None):
    """(value, bound of the kernel's fp32 error) in 64 bits on the device."""
    xv, wv = mx64(x.cuda())[0], mx64(w.cuda())[0]
    v, mag = xv @ wv.t(), xv.abs() @ wv.abs().t()
    err = mag * (x.shape[1] / 64 + 1) * 2.0 ** -24
    if b is not None:
        v, mag = v + b.double().cuda(), mag + b.double().abs().cuda()
    v = act64(v, act)
    err = 1.2 * err + 4 * 2.0 ** -24 * mag + (0 if act in ("none", "relu") else 2.0 ** -19) * (mag + 1e-3)
    if g1 is not None:
        v, err, mag = v * g1.double().cuda(), err * g1.double().abs().cuda(), mag * g1.double().abs().cuda()
    if g0 is not None:
        v, mag = v + g0.double().cuda(), mag + g0.double().abs().cuda()
    if res is not None:
        v, mag = v + res.double(), mag + res.double().abs()
    return v, err + 4 * 2.0 ** -24 * mag


def close(got, want, err):
    if got.dtype == torch.bfloat16:
        err = err + want.abs() * 2.0 ** -8
    off = (got.double() - want).abs()
    assert torch.isfinite(got).all() and (off <= err).all(), f"off by {(off / err).max().item():.2f} of the bound at {divmod((off / err).argmax().item(), got.shape[1])}"


SHAPES = [(1, 1, 1), (1, 64, 32), (1, 5120, 5120), (2, 33, 300), (7, 130, 257), (15, 257, 1000), (16, 4096, 1024), (17, 512, 512), (21, 4096, 1024), (33, 1000, 768),
          (64, 640, 2048), (100, 72, 5120), (128, 128, 256), (129, 250, 1283), (257, 1536, 640), (512, 1280, 1280), (1000, 264, 13824), (1565, 1030, 1024),
          (2048, 1024, 1024), (2300, 1288, 1280), (4133, 1096, 768)]


@pytest.mark.parametrize("M,N,K", SHAPES)
def test_linear_plain(ops, M, N, K):
    x, w, b = rnd(M, K, seed=1), rnd(N, K, seed=2, scale=K ** -0.5, dtype=torch.float32), rnd(N, seed=3, scale=0.1, dtype=torch.float32)
    lin = ops.pack_linear_mxfp4(w, b)
    want, err = product64(x, w, b)
    for f32 in (True, False):
        got = ops.linear(x.cuda(), lin, out_f32=f32)
        assert got.dtype == (torch.float32 if f32 else torch.bfloat16) and got.shape == (M, N)
        close(got, want, err)
    # rows quantised ahead: the same bits
    assert torch.equal(ops.linear(ops.quantize_mxfp4_rows(x.cuda()), lin), got)


@pytest.mark.parametrize("M,N,K", [(1, 200, 320), (13, 250, 512), (19, 256, 256), (70, 1000, 300), (300, 328, 512), (2500, 1096, 512)])
@pytest.mark.parametrize("act,gate,res", [("gelu_tanh", False, None), ("gelu_erf", True, "bf16"), ("silu", True, None), ("relu", False, "f32"), ("none", True, "f32")])
def test_linear_epilogue(ops, M, N, K, act, gate, res):
    x, w, b = rnd(M, K, seed=4), rnd(N, K, seed=5, scale=K ** -0.5), rnd(N, seed=6, dtype=torch.float32)
    g1, g0 = (rnd(N, seed=7, dtype=torch.float32).cuda(), rnd(N, seed=8, dtype=torch.float32).cuda()) if gate else (None, None)
    r = None if res is None else rnd(M, N, seed=9, dtype=torch.float32 if res == "f32" else torch.bfloat16).cuda()
    lin = ops.pack_linear(w, b, mxfp4=True)
    want, err = product64(x, w, b, act, g1, g0, r)
    got = ops.linear(x.cuda(), lin, act=act, g1=g1, g0=g0, res=r, out_f32=True)
    close(got, want, err)
    if r is not None:                       # in place on the residual
        buf = r.clone()
        assert ops.linear(x.cuda(), lin, act=act, g1=g1, g0=g0, res=buf, out=buf) is buf
        close(buf, want, err)


@pytest.mark.parametrize("M,N,K", [(1, 320, 256), (5, 77, 512), (40, 256, 300), (300, 1000, 512), (2304, 1280, 512), (2400, 1100, 768)])
def test_mxfp4_output_is_the_quantised_bf16_output(ops, M, N, K):
    x, lin = rnd(M, K, seed=1).cuda(), ops.pack_linear_mxfp4(rnd(N, K, seed=2, scale=K ** -0.5), rnd(N, seed=3, scale=0.1))
    for act in ("none", "gelu_tanh"):
        got, want = ops.linear(x, lin, act=act, out_mxfp4=True), ops.quantize_mxfp4_rows(ops.linear(x, lin, act=act))
        assert torch.equal(bytes_of(got), bytes_of(want)) and torch.equal(got.q, want.q)
        nxt = ops.pack_linear_mxfp4(rnd(96, N, seed=5, scale=N ** -0.5), None)
        assert torch.equal(ops.linear(got, nxt), ops.linear(want, nxt))


@pytest.mark.parametrize("M", [1, 9, 40, 300, 2304])
def test_views_and_odd_alignments(ops, M):
    """Column slices as input, residual and output, at element offsets that are not multiples of the access width."""
    N, K = 1040, 576
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
        assert torch.equal(big[mask], before[mask])          # nothing written beside the slice


def test_rows_do_not_depend_on_the_rows_beside_them(ops):
    """A row's result is the same bits whatever other rows the same kernel computes with it."""
    x, lin = rnd(2600, 768, seed=1).cuda(), ops.pack_linear_mxfp4(rnd(1288, 768, seed=2, scale=0.03), rnd(1288, seed=3))
    full = ops.linear(x, lin, out_f32=True)
    assert torch.equal(ops.linear(x[:2400], lin, out_f32=True), full[:2400])
    assert torch.equal(full, ops.linear(x, lin, out_f32=True))


def test_large_offsets(ops):
    """More than 2^31 bytes of output and of residual behind one call."""
    M, N, K = 70000, 8200, 256
    g = torch.Generator(device="cuda").manual_seed(0)
    x, w = torch.randn(M, K, generator=g, device="cuda").bfloat16(), rnd(N, K, seed=2, scale=K ** -0.5)
    lin = ops.pack_linear_mxfp4(w, None)
    res = torch.ones(M, N, device="cuda")
    got = ops.linear(x, lin, res=res, out_f32=True)
    for a in (0, 33000, 69990):
        want, err = product64(x[a:a + 10], w, res=res[a:a + 10])
        close(got[a:a + 10], want, err)


def test_other_streams_and_graphs(ops):
    """On a stream of the caller's own; captured, replayed several times with other work between, two graphs at once: the eager bits."""
    lins = [ops.pack_linear_mxfp4(rnd(1024, 768, seed=2, scale=0.03), rnd(1024, seed=3)), ops.pack_linear_mxfp4(rnd(512, 1024, seed=4, scale=0.03), None)]

    def chain(x):
        h = ops.residual_norm(x, None, out="mxfp4")
        return ops.linear(ops.linear(h, lins[0], act="gelu_tanh", out_mxfp4=True), lins[1])

    ins = [rnd(M, 768, seed=M, dtype=torch.float32).cuda() for M in (1, 300, 2300)]
    want = [chain(x) for x in ins]
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        other = [chain(x) for x in ins]
    torch.cuda.current_stream().wait_stream(st)
    assert all(torch.equal(a, b) for a, b in zip(want, other))
    graphs, outs = [], []
    for x in ins:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(chain(x))
        graphs.append(g)
    for _ in range(3):
        for o in outs:
            o.fill_(-3)
        for g in graphs:
            g.replay()
        again = [chain(x) for x in ins]
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) and torch.equal(a, c) for a, b, c in zip(want, outs, again))


def test_the_half_block_against_64_bits(ops):
    """Norm -> first linear + GELU -> second linear, MXFP4 between all of them, as the FFN half of a block runs them.
    Two chains of the same definition can put an fp32 value on either side of a rounding border: that moves one code of a row by a step and
    the row's output by that step times a weight.  Counted on the codes: at most 1e-4 of them may differ; the outputs then agree to
    sqrt(1e-4) times the step-to-value ratio (0.5) plus half a bf16 step: 1e-2 in the 2-norm."""
    M, C, F = 300, 1024, 2048
    x, y = rnd(M, C, seed=1, dtype=torch.float32).cuda(), rnd(M, C, seed=2).cuda()
    g1, sc, sh, bias = (rnd(C, seed=s, scale=0.5, dtype=torch.float32).cuda() for s in (3, 4, 5, 6))
    w0, w2 = rnd(F, C, seed=7, scale=C ** -0.5), rnd(C, F, seed=8, scale=F ** -0.5)
    l0, l2 = ops.pack_linear_mxfp4(w0, None), ops.pack_linear_mxfp4(w2, None)
    xs = x.clone()
    h = ops.residual_norm(xs, y, bias=bias, g1=g1, scale=sc, shift=sh, out="mxfp4")
    f = ops.linear(h, l0, act="gelu_tanh", out_mxfp4=True)
    out = ops.linear(f, l2)
    x64 = x.double() + (y.double() + bias.double()) * g1.double()
    n = (x64 - x64.mean(1, keepdim=True)) / (x64.var(1, unbiased=False, keepdim=True) + 1e-6).sqrt()
    h64 = (n * (1 + sc.double()) + sh.double()).bfloat16()
    f64 = act64(mx64(h64)[0] @ mx64(w0.cuda())[0].t(), "gelu_tanh").bfloat16()
    o64 = mx64(f64)[0] @ mx64(w2.cuda())[0].t()
    assert (ops.dequantize_mxfp4_rows(h, torch.float32).double() != mx64(h64)[0]).double().mean() < 1e-4
    assert (ops.dequantize_mxfp4_rows(f, torch.float32).double() != mx64(f64)[0]).double().mean() < 1e-3
    assert (out.double() - o64).norm() / o64.norm() < 1e-2


def test_refusals(ops):
    lin, plain = ops.pack_linear_mxfp4(rnd(64, 96, seed=1), None), ops.pack_linear(rnd(64, 128, seed=1), None)
    x = rnd(4, 96, seed=2).cuda()
    for bad in (lambda: ops.linear(x[:, :64], lin), lambda: ops.linear(x.float(), lin), lambda: ops.linear(ops.quantize_mxfp4_rows(x), plain),
                lambda: ops.linear(rnd(4, 128).cuda(), plain, out_mxfp4=True), lambda: ops.linear(x, lin, out_mxfp4=True, out_f32=True),
                lambda: ops.linear(x, lin, res=torch.zeros(4, 63, device="cuda")), lambda: ops.linear(x, lin, g1=torch.ones(63, device="cuda")),
                lambda: ops.linear(x, lin, g1=torch.ones(64, device="cuda", dtype=torch.bfloat16)), lambda: ops.linear(x, lin, out=torch.zeros(4, 65, device="cuda")),
                lambda: ops.linear_mxfp4(x, plain), lambda: ops.quantize_mxfp4_rows(x.half()), lambda: ops.quantize_mxfp4_rows(x.t()),
                lambda: ops.linear_from_mxfp4(lin.q, lin.s[:, :, :16], None, 96), lambda: ops.linear_from_mxfp4(lin.q, lin.s, None, 300),
                lambda: ops.linear_from_mxfp4(lin.q, lin.s, torch.zeros(63, device="cuda"), 96)):
        with pytest.raises((ValueError, TypeError)):
            bad()
    with pytest.raises(RuntimeError):
        ops.quantize_mxfp4_rows(x.cpu())
    with pytest.raises(KeyError):
        ops.linear(x, lin, act="tanh")


@pytest.mark.parametrize("M", [1, 2, 15, 16, 17, 31, 32, 33])
@pytest.mark.parametrize("N,K", [(40, 96), (1030, 2816), (4100, 288), (5000, 1440), (9000, 512)])
def test_few_rows(ops, M, N, K):
    """Every width of a work-group's columns (it follows N), one launch and two (rows behind an odd row stride), bf16 and MXFP4 output: one result."""
    x, w, b = rnd(M, K, seed=1).cuda(), rnd(N, K, seed=2, scale=K ** -0.5), rnd(N, seed=3, scale=0.1, dtype=torch.float32)
    wide = torch.zeros(M, K + 3, dtype=torch.bfloat16, device="cuda")
    wide[:, :K] = x
    lin, res = ops.pack_linear_mxfp4(w, b), rnd(M, N, seed=4).cuda()
    want, err = product64(x, w, b, "gelu_erf", res=res)
    got = ops.linear(x, lin, act="gelu_erf", res=res, out_f32=True)
    close(got, want, err)
    assert torch.equal(got, ops.linear(wide[:, :K], lin, act="gelu_erf", res=res, out_f32=True))
    assert torch.equal(got, ops.linear(ops.quantize_mxfp4_rows(x), lin, act="gelu_erf", res=res, out_f32=True))
    h, f = ops.linear(x, lin, act="gelu_erf"), ops.linear(x, lin, act="gelu_erf", out_mxfp4=True)
    q = ops.quantize_mxfp4_rows(h)
    assert torch.equal(q.q, f.q) and torch.equal(bytes_of(q), bytes_of(f))


def test_rows_of_the_callers_own(ops):
    """Codes that are a column slice of a wider buffer, as activations and as weights; a transposed weight view; what the kernels cannot read."""
    M, N, K = 70, 96, 512
    x, w, b = rnd(M, K, seed=1).cuda(), rnd(N, K, seed=2, scale=K ** -0.5).cuda(), rnd(N, seed=3, dtype=torch.float32).cuda()
    mx, wm = ops.quantize_mxfp4_rows(x), ops.quantize_mxfp4_rows(w)
    want = ops.linear(x, ops.pack_linear_mxfp4(w, b))
    assert torch.equal(want, ops.linear(x, ops.pack_linear_mxfp4(w.t().contiguous().t(), b)))
    from fantasy_world_amd.hip_ops import MXFP4Rows
    wide = torch.full((N, 512), 0x77, dtype=torch.uint8, device="cuda")
    for at in (0, 16, 256):
        wq, xq = wide.clone(), torch.full((M, 544), 0x77, dtype=torch.uint8, device="cuda")
        xq[:, at:at + 256], wq[:, at:at + 256] = mx.q, wm.q
        lin = ops.linear_from_mxfp4(wq[:, at:at + 256], wm.s, b, K)
        assert torch.equal(want, ops.linear(MXFP4Rows(xq[:, at:at + 256], mx.s, K), lin))
        assert torch.equal(ops.dequantize_mxfp4_rows(MXFP4Rows(xq[:, at:at + 256], mx.s, K)), ops.dequantize_mxfp4_rows(mx))
    odd = torch.zeros(M, 544, dtype=torch.uint8, device="cuda")
    with pytest.raises(RuntimeError):
        ops.linear(MXFP4Rows(odd[:, 8:264], mx.s, K), ops.pack_linear_mxfp4(w, b))
    with pytest.raises(ValueError):
        MXFP4Rows(odd[:, :250], mx.s, K)


def test_the_output_is_not_the_input(ops):
    lin, x = ops.pack_linear_mxfp4(rnd(256, 256, seed=1, scale=0.06), None), rnd(9, 256, seed=2).cuda()
    with pytest.raises(ValueError):
        ops.linear(x, lin, out=x)
    want = ops.linear(x, lin, res=x)
    buf = torch.empty_like(x)
    assert torch.equal(ops.linear(x, lin, res=x, out=buf), want)


def test_arrays_larger_than_the_caches(ops):
    """Outputs, residuals and rows of more than 256 MB are accessed past the caches: the bits of the same rows in smaller calls."""
    g = torch.Generator(device="cuda").manual_seed(0)
    M, N, K = 13200, 10304, 1024
    x = torch.randn(M, K, generator=g, device="cuda").bfloat16()
    lin, gate = ops.pack_linear_mxfp4(rnd(N, K, seed=2, scale=K ** -0.5), rnd(N, seed=3)), rnd(N, seed=4, dtype=torch.float32).cuda()
    part = 2048                                           # enough rows for the same tiles, 84 MB of fp32 output
    for rdt, kw in ((None, dict()), (None, dict(act="gelu_tanh")), (None, dict(out_f32=True)), (torch.bfloat16, dict(g1=gate)), (torch.bfloat16, dict(out_f32=True)),
                    (torch.float32, dict(g1=gate, out_f32=True)), (torch.float32, dict()), (torch.float32, dict(act="silu", out_f32=True))):
        res = None if rdt is None else torch.randn(M, N, generator=g, device="cuda").to(rdt)
        got = ops.linear(x, lin, res=res, **kw)
        for a in (0, 5 * part, M - part):
            assert torch.equal(got[a:a + part], ops.linear(x[a:a + part], lin, res=None if res is None else res[a:a + part], **kw)), (rdt, kw)
        if rdt is not None and got.dtype == rdt:          # in place
            assert ops.linear(x, lin, res=res, out=res, **kw) is res and torch.equal(res, got)
        del res, got
    for dt in (torch.bfloat16, torch.float32):
        rows = torch.randn(M, N, generator=g, device="cuda").to(dt)
        mx = ops.quantize_mxfp4_rows(rows)
        for a in (0, 4096, 12800):
            assert torch.equal(mx.q[a:a + 400], ops.quantize_mxfp4_rows(rows[a:a + 400]).q)
        back = ops.dequantize_mxfp4_rows(mx, dt)
        check_rows(ops.quantize_mxfp4_rows(rows[12800:12864]), rows[12800:12864].cpu(), ops)
        assert torch.equal(back[12800:12864], ops.dequantize_mxfp4_rows(ops.quantize_mxfp4_rows(rows[12800:12864]), dt))
        assert torch.equal(back, ops.dequantize_mxfp4_rows(ops.quantize_mxfp4_rows(back), dt))       # values of the format are kept
