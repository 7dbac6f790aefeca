"""precision="mxfp4" without a GPU: the host logic of the mode on the CPU op set, unsharded and under tensor parallelism (gloo).

The mode has no reference semantics.  Its price against exact linears: e2m1 rounds with a relative error of 0.11 to 0.14 (normal to
GELU-shaped values), both operands of a linear together 0.16 to 0.2, which the residual streams and the linears that stay exact dilute: the
forward must lie between a tenth of that and twice that from the exact one.  Two runs of the mode that differ in summation order differ
where a value sits on a rounding border, far less often than every value: less than half the price apart."""
import os

import pytest
import torch
import torch.multiprocessing as mp

from conftest import ROOT, rel_l2
from oracle.ref_ops import TorchRefOps
from test_tensor_parallel_cpu import _cfg, _free_port, _hc, _worker


def _kw(ins):
    return dict(clip_feature=ins["clip_feature"], y=ins["y"], plucker_fea=ins["plucker_fea"], plucker_context_lens=ins["plucker_context_lens"])


def test_engine_mxfp4_linears(case_l2):
    from fantasy_world_amd.engine import FusionEngine
    case, ins = case_l2, case_l2.inputs
    eng = FusionEngine(case.cfg, case.weights.__getitem__, TorchRefOps(), precision="mxfp4")
    for blk in eng.dit:
        assert all(lin.mxfp4 for lin in (blk.qkv, blk.o, blk.cq, blk.ckv, blk.co, blk.ffn0, blk.ffn2))
    assert not any(lin.mxfp4 for lin in (eng.patch, eng.head, eng.proj, eng.frame[0].qkv, eng.bicross[0].out1))
    got, _ = eng.joint_forward(ins["x"], ins["timestep"], ins["context"], **_kw(ins))
    price = rel_l2(got, case.golden["noise_pred"])
    print(f"mxfp4 linears against the exact reference: {price:.3f}")
    assert 1.6e-2 < price < 0.4, price


def test_mxfp4_needs_an_op_set_that_has_it(case_l2):
    from fantasy_world_amd.engine import FusionEngine

    class Without(TorchRefOps):
        pack_linear_mxfp4 = property()
    for bad in (dict(ops=Without(), precision="mxfp4"), dict(ops=TorchRefOps(), precision="fp4")):
        with pytest.raises(ValueError, match="precision"):
            FusionEngine(case_l2.cfg, case_l2.weights.__getitem__, bad["ops"], precision=bad["precision"])


def test_mxfp4_linears_under_tensor_parallelism(tmp_path):
    """Heads and FFN units are cut on block borders, so every rank's codes are slices of the unsharded ones and nothing is exchanged for them;
    the residual updates run fused with the norms behind them."""
    from fantasy_world_amd import synth
    from fantasy_world_amd.engine import FusionEngine
    grid, cfg, opts = (3, 8, 8), _cfg(), dict(precision="mxfp4")
    W = synth.make_weights(cfg)
    W.update(synth.make_heads_weights(_hc()))
    path = str(tmp_path / "weights.pt")
    torch.save(dict(W), path)
    ins = synth.make_inputs(cfg, *grid, seed=3)
    run = lambda **kw: FusionEngine(cfg, W.__getitem__, TorchRefOps(exact=True), **kw).joint_forward(ins["x"], ins["timestep"], ins["context"], **_kw(ins))[0]
    want, full = run(**opts), run()
    price = rel_l2(want, full)
    mp.spawn(_worker, args=(2, _free_port(), grid, str(tmp_path), path, False, opts), nprocs=2, join=True)
    for r in range(2):
        (got, _), kinds = torch.load(os.path.join(str(tmp_path), f"tp_{r}.pt"))
        assert rel_l2(got, want) < 0.5 * price, (r, rel_l2(got, want), price)
        assert "all_reduce_amax" not in kinds and "all_reduce" in kinds, kinds


def test_fused_update_and_norm_return_the_rows_of_the_separate_passes():
    """TensorParallel's _reduce_into with a norm behind it: same stream, same rows, block by block."""
    from fantasy_world_amd.tensor_parallel import TensorShard, TPFusionEngine, _drain
    eng = TPFusionEngine.__new__(TPFusionEngine)
    eng.ops, eng.tp = TorchRefOps(), TensorShard(0, 1, chunks=2, chunk_rows=8)
    g = torch.Generator().manual_seed(0)
    x, h = torch.randn(40, 64, generator=g), torch.randn(40, 128, generator=g)
    lin, v = eng.ops.pack_linear(torch.randn(64, 128, generator=g), None), torch.randn(4, 64, generator=g)
    a, b = x.clone(), x.clone()
    norm = dict(w=v[2], b=v[3], eps=1e-5)
    box = {}

    def fused():
        box["rows"] = yield from eng._reduce_into(a, h, lin, v[0], g1=v[1], norm=norm)
    _drain(fused())
    _drain(eng._reduce_into(b, h, lin, v[0], g1=v[1]))
    assert torch.equal(a, b) and torch.equal(box["rows"], eng.ops.layernorm(b, **norm))
