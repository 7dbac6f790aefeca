"""precision="mxfp4" over two gloo ranks with the torch op set: the first-run check of a multi-rank run holds the mode to its own distance from
the golden, and a sequence shard returns the unsharded forward."""
import os

import torch
import torch.distributed as dist
import torch.multiprocessing as mp

from test_multi_gpu_first_run_cpu import _free_port, _init
from test_sequence_shard_cpu import _cfg, _hc, _worker, shared_weights  # noqa: F401


def _golden_worker(rank, world, port, outdir, bad_rank):
    parallel, topo = _init(rank, world, port)
    from oracle.ref_ops import TorchRefOps

    class Ops(TorchRefOps):
        """On the bad rank an eighth of every MXFP4 weight's rows carries scales one binade too high."""

        def pack_linear_mxfp4(self, w, b):
            lin = super().pack_linear_mxfp4(w, b)
            if rank == bad_rank:
                lin.w = lin.w.clone()
                lin.w[:lin.N // 8] *= 2
            return lin
    res = parallel.golden_self_check(topo, Ops(), case="wan21_l3_f2_12x8", precision="mxfp4")
    torch.save(res, os.path.join(outdir, f"golden_{rank}.pt"))
    dist.barrier()
    dist.destroy_process_group()


def test_the_first_run_check_refuses_a_rank_with_wrong_scales(tmp_path):
    """The mode lies 0.134 to 0.146 from the golden, over two ranks as over one; a rank with wrong scales in an eighth of its weights adds an
    error of its own that must not pass."""
    mp.spawn(_golden_worker, args=(2, _free_port(), str(tmp_path), 1), nprocs=2, join=True)
    res = [torch.load(tmp_path / f"golden_{r}.pt", weights_only=False) for r in range(2)]
    print(res[0])
    assert res[0] == res[1] and not res[0]["ok"] and res[0]["rel_l2_max_over_ranks"] > 0.2, res[0]


def test_a_sequence_shard_returns_the_unsharded_forward(tmp_path, shared_weights):  # noqa: F811
    """Block scales belong to a row, so a shard of rows exchanges nothing for them.  Products are accumulated in fp64 on both sides; what is
    left are last-bit differences that may put a value on the other side of an e2m1 border: far less than a tenth of the mode's own price, which
    a wrong row, slice or scale exceeds."""
    from fantasy_world_amd import synth
    from fantasy_world_amd.engine import FusionEngine
    from oracle.ref_ops import TorchRefOps
    W, wpath = shared_weights
    grid, opts = (3, 4, 12), dict(precision="mxfp4")
    ins = synth.make_inputs(_cfg(), *grid, seed=3)
    kw = dict(clip_feature=ins["clip_feature"], y=ins["y"], plucker_fea=ins["plucker_fea"], plucker_context_lens=ins["plucker_context_lens"])
    run = lambda **o: FusionEngine(_cfg(), W.__getitem__, TorchRefOps(exact=True), heads_cfg=_hc(), **o).joint_forward(
        ins["x"], ins["timestep"], ins["context"], return_prediction=True, **kw)
    (want, wpred), (exact, _) = run(**opts), run()
    mp.spawn(_worker, args=(2, _free_port(), grid, str(tmp_path), wpath, False, opts, True), nprocs=2, join=True)
    rel = lambda a, b: ((a.double() - b.double()).norm() / b.double().norm()).item()
    price = rel(want, exact)
    assert price > 1.6e-2
    for r in range(2):
        got, pred, _ = torch.load(os.path.join(str(tmp_path), f"out_{r}.pt"))
        print(r, rel(got, want), price)
        assert rel(got, want) < 0.1 * price, (r, rel(got, want), price)
        assert all(pred[k].shape == v.shape for k, v in wpred.items())
