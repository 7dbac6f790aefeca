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
