"""-m gpu: fw_residual_norm against its definition in 64 bits.

Tolerances.  x' in fp32: y + bias, the affine and the sum round at most four times: 4 * 2^-24 of the magnitudes involved; with a post norm
the statistics (C terms in fp32, summed in lanes of at most 32 chunks and six shuffle steps) add at most 64 * 2^-24 relative.  x' in bf16:
half a step, 2^-8 of the value, more.  h: the norm of the STORED x' (taken from the kernel's own output, so its rounding does not count
twice), 64 * 2^-24 for the statistics relative to the row's largest magnitude over its deviation, and half a bf16 step."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops():
    from fantasy_world_amd.hip_ops import HipOps
    return HipOps("cuda:0")


def rnd(*shape, seed=0, scale=1.0, dtype=torch.float32):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(*shape, generator=g) * scale).to(dtype).cuda()


def norm64(v, kind, eps):
    if kind == "layer":
        v = v - v.mean(1, keepdim=True)
    return v / (v.square().mean(1, keepdim=True) + eps).sqrt()


def rows_of(v, rows):
    return v.double().view(-1, v.shape[-1]).repeat_interleave(rows // (v.numel() // v.shape[-1]), 0)


def check(ops, x, y, norm="layer", post=None, out="bf16", eps=1e-6, x_out=None, **vec):
    rows, C = x.shape
    src, buf = x.clone(), x_out
    h = ops.residual_norm(x, y, norm=norm, post=post, eps=eps, out=out, x_out=buf, **vec)
    stored = x if buf is None else buf
    stat = 64 * 2.0 ** -24
    if y is not None:
        t = y.double()
        mag = t.abs()
        if vec.get("bias") is not None:
            t, mag = t + vec["bias"].double(), mag + vec["bias"].double().abs()
        rel = 4 * 2.0 ** -24
        if post:
            t = norm64(t, post, eps)
            # the mean cancels: the error of (t - mean) is relative to the row's largest magnitude, scaled by 1 / std
            mag = t.abs() + t.abs().amax(1, keepdim=True)
            rel = stat
            if vec.get("post_w") is not None:
                t, mag = t * vec["post_w"].double(), mag * vec["post_w"].double().abs()
        if vec.get("g1") is not None:
            t, mag = t * rows_of(vec["g1"], rows), mag * rows_of(vec["g1"], rows).abs()
        if vec.get("g0") is not None:
            t, mag = t + rows_of(vec["g0"], rows), mag + rows_of(vec["g0"], rows).abs()
        want = src.double() + t
        err = rel * mag + 2 * 2.0 ** -24 * (src.double().abs() + mag)
        if x.dtype == torch.bfloat16:
            err = err + want.abs() * 2.0 ** -8
        assert ((stored.double() - want).abs() <= err).all(), ((stored.double() - want).abs() / err).max()
    else:
        assert torch.equal(x, src)
    n = norm64(stored.double(), norm, eps)
    # the mean is a sum of C values in fp32: at most 32 additions in a lane, 2 inside a chunk, 6 shuffle steps and the product with 1 / C, each
    # off by 2^-24 of a partial result that is at most C * max|v| (before the 1 / C): 41 * 2^-24 * max|v|, which h sees divided by the
    # deviation -- a row whose mean is 1000 deviations carries 1000 times that
    v = stored.double()
    dev = ((v - (v.mean(1, keepdim=True) if norm == "layer" else 0)).square().mean(1, keepdim=True) + eps).sqrt()
    mag = n.abs() + v.abs().amax(1, keepdim=True) / dev
    if vec.get("w") is not None:
        n, mag = n * vec["w"].double(), mag * vec["w"].double().abs()
        if vec.get("b") is not None:
            n, mag = n + vec["b"].double(), mag + vec["b"].double().abs()
    if vec.get("scale") is not None:
        n, mag = n * (1 + rows_of(vec["scale"], rows)), mag * (1 + rows_of(vec["scale"], rows)).abs()
    if vec.get("shift") is not None:
        n, mag = n + rows_of(vec["shift"], rows), mag + rows_of(vec["shift"], rows).abs()
    if out == "mxfp4":
        # the rows are those of the bf16 result, code by code
        again = ops.residual_norm(stored, None, norm=norm, eps=eps, **{k: v for k, v in vec.items() if k in ("w", "b", "scale", "shift")})
        want = ops.quantize_mxfp4_rows(again)
        assert torch.equal(h.q, want.q)
        assert torch.equal(h.s.permute(0, 2, 1, 3).reshape(-1, h.s.shape[1] * 8)[:rows], want.s.permute(0, 2, 1, 3).reshape(-1, h.s.shape[1] * 8)[:rows])
        h = again
    err = stat * mag + n.abs() * 2.0 ** -8 + 1e-30
    assert h.dtype == torch.bfloat16 and h.shape == x.shape and ((h.double() - n).abs() <= err).all(), ((h.double() - n).abs() / err).max()
    return h


def vectors(C, groups=1, seed=10, post=None, affine=True, mod=True, gate=True):
    v = lambda s, n=1: rnd(n, C, seed=seed + s, scale=0.5) if n > 1 else rnd(C, seed=seed + s, scale=0.5)
    out = dict(bias=v(0))
    if gate:
        out.update(g1=v(1, groups), g0=v(2, groups))
    if post:
        out.update(post_w=1 + v(3))
    if affine:
        out.update(w=1 + v(4), b=v(5))
    if mod:
        out.update(scale=v(6, groups), shift=v(7, groups))
    return out


WIDTHS = [(1, 1), (1, 5120), (3, 7), (5, 64), (4, 255), (33, 256), (2, 257), (9, 1000), (130, 1024), (7, 1283), (6, 2048), (3, 4100), (257, 5120), (2, 5121), (5, 8192), (4100, 1024), (4099, 5120)]


@pytest.mark.parametrize("out", ["bf16", "mxfp4"])
@pytest.mark.parametrize("rows,C", WIDTHS)
def test_update_and_norm(ops, rows, C, out):
    x, y = rnd(rows, C, seed=1, scale=2.0), rnd(rows, C, seed=2, dtype=torch.bfloat16)
    check(ops, x, y, out=out, **vectors(C))


@pytest.mark.parametrize("xdt,ydt", [(torch.float32, torch.float32), (torch.bfloat16, torch.bfloat16), (torch.bfloat16, torch.float32), (torch.bfloat16, None), (torch.float32, None)])
@pytest.mark.parametrize("norm,post", [("layer", None), ("rms", "rms"), ("layer", "layer"), ("rms", "layer")])
@pytest.mark.parametrize("rows,C", [(12, 513), (66, 1024), (10, 5120)])
def test_types_and_norms(ops, rows, C, xdt, ydt, norm, post):
    x = rnd(rows, C, seed=3, scale=3.0, dtype=xdt) + 0.5
    y = None if ydt is None else rnd(rows, C, seed=4, dtype=ydt)
    v = vectors(C, 2, post=post if y is not None else None)
    if y is None:
        v = {k: t for k, t in v.items() if k in ("w", "b", "scale", "shift")}
        post = None
    check(ops, x, y, norm=norm, post=post, **v)
    check(ops, x, y, norm=norm, post=post, out="mxfp4", x_out=None if y is None else torch.empty_like(x), **v)


def test_absent_vectors_views_and_nothing(ops):
    x, y = rnd(37, 700, seed=1), rnd(37, 700, seed=2, dtype=torch.bfloat16)
    check(ops, x.clone(), y)
    check(ops, x.clone(), None, norm="rms")
    check(ops, x.clone(), y, w=rnd(700, seed=3))
    check(ops, x.clone(), y, shift=rnd(700, seed=3), post="rms")
    for a, b in ((4, 260), (3, 300)):          # column slices, aligned and not; what lies beside them stays
        wide, ywide = x.clone(), y.clone()
        xs = wide[:, a:b]
        before = wide.clone()
        check(ops, xs, ywide[:, a:b], **vectors(b - a))
        keep = torch.ones_like(wide, dtype=torch.bool)
        keep[:, a:b] = False
        assert torch.equal(wide[keep], before[keep])
    assert ops.residual_norm(x[:0], y[:0]).shape == (0, 700)
    assert ops.residual_norm(x[:0], y[:0], out="mxfp4").shape == (0, 700)


def test_constant_rows_and_large_means(ops):
    """A row without variance gives zeros (eps in the root), a mean 1000 times the deviation keeps its digits (no E[x^2] - mean^2)."""
    x = torch.full((5, 1024), 3.0, device="cuda")
    assert not ops.residual_norm(x, None).any()
    x = torch.zeros(5, 700, device="cuda")
    assert not ops.residual_norm(x, None, norm="rms", out="bf16").any()
    check(ops, rnd(9, 1024, seed=1) + 1000.0, None, eps=1e-5)


def test_infinite_and_nan_rows_stay_alone(ops):
    x, y = rnd(6, 1024, seed=1), rnd(6, 1024, seed=2)
    want = ops.residual_norm(x.clone(), y)
    x[2, 5], y[4, 900] = float("nan"), float("inf")
    h = ops.residual_norm(x, y)
    rows = [0, 1, 3, 5]
    assert torch.equal(h[rows], want[rows]) and torch.isnan(h[2]).all() and torch.isnan(h[4]).any()


@pytest.mark.parametrize("rows", [3, 40, 4103])
@pytest.mark.parametrize("C", [1024, 5120])
@pytest.mark.parametrize("form", ["mod", "affine", "both"])
def test_same_bits_as_the_separate_passes(ops, rows, C, form):
    """residual_add, then layernorm."""
    v = vectors(C, affine=form != "mod", mod=form != "affine")
    up = {k: v.pop(k) for k in ("bias", "g1", "g0")}
    for ydt in (torch.bfloat16, torch.float32):
        x, y = rnd(rows, C, seed=1, scale=2.0), rnd(rows, C, seed=2, dtype=ydt)
        x2 = x.clone()
        h = ops.residual_norm(x, y, eps=1e-6, **up, **v)
        ops.residual_add(x2, y, **up)
        assert torch.equal(x, x2) and torch.equal(h, ops.layernorm(x2, eps=1e-6, **v))


def test_refusals(ops):
    x, y, c = rnd(6, 64, seed=1), rnd(6, 64, seed=2), rnd(64, seed=3)
    for kw in (dict(y=y[:5]), dict(y=y, g1=c[:63]), dict(y=y, g1=c.bfloat16()), dict(y=y, g1=rnd(4, 64)), dict(y=y, g1=rnd(2, 64), scale=rnd(3, 64)), dict(y=y, bias=rnd(2, 64)),
               dict(norm="batch"), dict(y=y, post="batch"), dict(out="fp8"), dict(y=y, x_out=torch.empty(6, 64, dtype=torch.bfloat16, device="cuda")), dict(y=y, x_out=torch.empty(6, 65, device="cuda")),
               dict(w=c.view(32, 2).t().reshape(64)[::1][:32])):
        with pytest.raises(ValueError):
            ops.residual_norm(x, **kw)
    with pytest.raises(ValueError):
        ops.residual_norm(x.half())
    with pytest.raises(ValueError):
        ops.residual_norm(x.t())
    with pytest.raises(RuntimeError):
        ops.residual_norm(x, b=c)                 # an offset without its weight
    with pytest.raises(RuntimeError):
        ops.residual_norm(x.cpu())
    with pytest.raises(RuntimeError):
        ops.residual_norm(x, y.cpu())
    with pytest.raises(RuntimeError):
        ops.residual_norm(rnd(2, 8193))


@pytest.mark.parametrize("post", [None, "rms"])
@pytest.mark.parametrize("rows,C,groups", [(4098, 1024, 3), (8194, 5120, 2), (4160, 256, 64), (4160, 512, 65)])
def test_many_rows_in_groups(ops, rows, C, groups, post):
    """Runs of rows with vectors of their own, from a run per work-group up to more runs than the kernel with staged vectors takes."""
    x, y, v = rnd(rows, C, seed=1, scale=2.0), rnd(rows, C, seed=2, dtype=torch.bfloat16), vectors(C, groups, post=post)
    check(ops, x.clone(), y, post=post, **v)
    check(ops, x, y, post=post, out="mxfp4", x_out=torch.empty_like(x), **v)


@pytest.mark.parametrize("rows,C", [(7, 5120), (4100, 5120), (4100, 640), (50, 333)])
def test_captured_and_into_the_callers_rows(ops, rows, C):
    """h in a column slice of the caller's, the rest of it untouched; a captured call replayed with eager work between: the eager bits."""
    x, y, v = rnd(rows, C, seed=1), rnd(rows, C, seed=2, dtype=torch.bfloat16), vectors(C, post="layer")
    xo = torch.empty_like(x)
    want = ops.residual_norm(x, y, post="layer", x_out=xo, **v)
    keep_x = xo.clone()
    wide = torch.full((rows, C + 24), 5.0, dtype=torch.bfloat16, device="cuda")
    for at in (0, 8, 3):
        part = wide[:, at:at + C]
        assert ops.residual_norm(x, y, post="layer", x_out=xo, h_out=part, **v) is part and torch.equal(part, want)
        assert (wide[:, :at] == 5).all() and (wide[:, at + C:] == 5).all()
        wide.fill_(5.0)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        h = ops.residual_norm(x, y, post="layer", x_out=xo, **v)
        q = ops.residual_norm(xo, None, out="mxfp4", w=v["w"], b=v["b"], scale=v["scale"], shift=v["shift"])
    for _ in range(3):
        xo.zero_()
        h.zero_()
        graph.replay()
        again = ops.residual_norm(x, y, post="layer", x_out=torch.empty_like(x), **v)
        torch.cuda.synchronize()
        assert torch.equal(h, want) and torch.equal(xo, keep_x) and torch.equal(again, want)
        assert torch.equal(q.q, ops.quantize_mxfp4_rows(want).q)
    for bad in (wide[:, :C - 1], wide.float()[:, :C], wide[:rows - 1, :C]):
        with pytest.raises(ValueError):
            ops.residual_norm(x, y, h_out=bad, x_out=xo)
    with pytest.raises(ValueError):
        ops.residual_norm(x, y, h_out=wide[:, :C], x_out=xo, out="mxfp4")


@pytest.mark.parametrize("post", [None, "layer"])
@pytest.mark.parametrize("xdt", [torch.float32, torch.bfloat16])
def test_streams_larger_than_the_caches(ops, xdt, post):
    """A stream of more than 256 MB is accessed past the caches: the bits of the same rows in smaller calls."""
    rows, C = (13200, 5120) if xdt == torch.float32 else (26400, 5120)
    g = torch.Generator(device="cuda").manual_seed(0)
    x, y = torch.randn(rows, C, generator=g, device="cuda").to(xdt), torch.randn(rows, C, generator=g, device="cuda").bfloat16()
    v = vectors(C, post=post)
    xo = torch.empty_like(x)
    h = ops.residual_norm(x, y, post=post, x_out=xo, **v)
    q = ops.residual_norm(x, y, post=post, x_out=torch.empty_like(x), out="mxfp4", **v)
    for a in (0, 6000, rows - 5000):
        part = x[a:a + 5000].clone()
        want = ops.residual_norm(part, y[a:a + 5000], post=post, **v)
        assert torch.equal(h[a:a + 5000], want) and torch.equal(xo[a:a + 5000], part)
        assert torch.equal(q.q[a:a + 5000], ops.quantize_mxfp4_rows(want).q)
    src = x.clone()
    assert torch.equal(ops.residual_norm(x, y, post=post, **v), h) and torch.equal(x, xo) and not torch.equal(x, src)


@pytest.mark.parametrize("out", ["bf16", "mxfp4"])
@pytest.mark.parametrize("rows,C,groups", [(4103, 2087, 1), (4104, 5119, 3), (4100, 1282, 2), (300, 4097, 1)])
def test_rows_of_odd_length(ops, rows, C, groups, out):
    """Rows and vectors that start at any element, with 1, 2 or 3 values behind the last four, from 2049 columns on with staged vectors; in
    slices of wider rows, what lies beside them stays."""
    wide, ywide = rnd(rows, C + 6, seed=1, scale=2.0), rnd(rows, C + 7, seed=2, dtype=torch.bfloat16)
    before = wide.clone()
    check(ops, wide[:, 3:C + 3], ywide[:, 5:C + 5], out=out, **vectors(C, groups))
    assert torch.equal(wide[:, :3], before[:, :3]) and torch.equal(wide[:, C + 3:], before[:, C + 3:])
    xb = before[:, :C].bfloat16()
    check(ops, xb, ywide[:, :C], out=out, post="layer", norm="rms", **vectors(C, groups, post="layer"))
