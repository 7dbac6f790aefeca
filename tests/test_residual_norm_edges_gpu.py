"""-m gpu: fw_residual_norm at argument values and overlaps that its header allows or refuses."""
import ctypes

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


def ptr(t):
    return ctypes.c_void_p(0 if t is None else t.data_ptr())


@pytest.mark.parametrize("rows,C", [(7, 256), (4096, 256), (5000, 1024), (4100, 2050)])
@pytest.mark.parametrize("short", [0, 1, 3000, 4094, 1 << 30])
def test_one_vector_for_all_rows(ops, rows, C, short):
    """rows_per_mod from rows up to the largest int is one run: the bits of rows_per_mod = rows, every row written."""
    x, y, bias, g1 = rnd(rows, C, seed=1), rnd(rows, C, seed=2, dtype=torch.bfloat16), rnd(C, seed=3), rnd(C, seed=4)
    xo, h = torch.full_like(x, 7.0), torch.full((rows, C), 7.0, dtype=torch.bfloat16, device="cuda")
    want_x = torch.empty_like(x)
    want = ops.residual_norm(x, y, bias=bias, g1=g1, x_out=want_x)
    rc = ops.lib.fw_residual_norm(ptr(x), C, ptr(xo), C, 2, ptr(y), C, 1, ptr(bias), ptr(g1), None, 0, None, 1, None, None, None, None, ctypes.c_float(1e-6),
                                  ptr(h), C, 1, None, rows, C, 0x7fffffff - short, ctypes.c_void_p(torch.cuda.current_stream().cuda_stream))
    assert rc == 0 and torch.equal(xo, want_x) and torch.equal(h, want)


@pytest.mark.parametrize("post", [None, "layer"])
@pytest.mark.parametrize("rows,C", [(5, 1024), (4100, 1024), (4100, 5120), (70, 333), (4100, 2051)])
def test_outputs_in_place_of_inputs(ops, rows, C, post):
    """x_out and h_out as x or y themselves: the bits of outputs of their own."""
    x, y, g1 = rnd(rows, C, seed=1, dtype=torch.bfloat16), rnd(rows, C, seed=2, dtype=torch.bfloat16), rnd(C, seed=3)
    want_x = torch.empty_like(x)
    want = ops.residual_norm(x, y, g1=g1, post=post, x_out=want_x)
    for xo, ho in (("x", None), ("y", None), ("new", "x"), ("new", "y"), ("x", "y"), ("y", "x")):
        t = dict(x=x.clone(), y=y.clone(), new=torch.empty_like(x))
        h = ops.residual_norm(t["x"], t["y"], g1=g1, post=post, x_out=t[xo], h_out=None if ho is None else t[ho])
        assert torch.equal(h, want) and torch.equal(t[xo], want_x), (xo, ho)
    alone = ops.residual_norm(x, None)
    assert torch.equal(ops.residual_norm(x, None, h_out=x), alone)


def test_outputs_beside_and_across_inputs(ops):
    """Columns of one buffer share nothing; a shifted view does, and is refused."""
    wide = rnd(300, 3 * 264, seed=1, dtype=torch.bfloat16)
    x, y, h = wide[:, :260], wide[:, 264:524], wide[:, 528:788]
    src, want_x = x.clone(), torch.empty(300, 260, dtype=torch.bfloat16, device="cuda")
    want = ops.residual_norm(src, y, x_out=want_x)
    assert torch.equal(ops.residual_norm(x, y, h_out=h), want) and torch.equal(x, want_x)
    for kw in (dict(x_out=wide[:, 1:261]), dict(h_out=wide[:, 520:780]), dict(h_out=x), dict(x_out=wide[:, 262:522])):
        with pytest.raises(RuntimeError, match="overlaps"):
            ops.residual_norm(x, y, **kw)
    with pytest.raises(RuntimeError, match="overlaps"):
        ops.residual_norm(x[:-1], y[1:], x_out=x[1:])


@pytest.mark.parametrize("C", [512, 640, 1024, 1280, 1536, 2048, 4096, 5120])
def test_a_reduced_update_and_its_norm_at_any_width(ops, C):
    """The tensor-parallel engine's update with a norm behind it returns the bits of residual_add, then layernorm, at every width."""
    from fantasy_world_amd.tensor_parallel import TensorShard, TPFusionEngine, _drain
    rows = 8192
    eng = TPFusionEngine.__new__(TPFusionEngine)
    eng.ops, eng.tp = ops, TensorShard(0, 1, chunks=2, chunk_rows=64)
    a, y = rnd(rows, C, seed=1, scale=2.0) + 0.3, rnd(rows, 64, seed=2, dtype=torch.bfloat16)
    lin, bias, g1, w, b = ops.pack_linear(rnd(C, 64, seed=3).cpu(), None), rnd(C, seed=4), rnd(C, seed=5), rnd(C, seed=6), rnd(C, seed=7)
    norm = dict(w=w, b=b, eps=1e-6)
    x, box = a.clone(), {}

    def fused():
        box["rows"] = yield from eng._reduce_into(x, y, lin, bias, g1=g1, norm=norm)
    _drain(fused())
    _drain(eng._reduce_into(a, y, lin, bias, g1=g1))
    assert torch.equal(x, a) and torch.equal(box["rows"], ops.layernorm(a, **norm))
    if C in ops.RESIDUAL_NORM_SAME_BITS:
        part = ops.linear(y, lin, out_f32=eng.tp.reduce_dtype == torch.float32)
        again = rnd(rows, C, seed=1, scale=2.0) + 0.3
        assert torch.equal(ops.residual_norm(again, part, bias=bias, g1=g1, **norm), box["rows"]) and torch.equal(again, a)
