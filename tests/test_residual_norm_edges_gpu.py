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
