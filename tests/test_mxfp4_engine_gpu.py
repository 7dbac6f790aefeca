"""-m gpu: precision="mxfp4" through the whole forward, and the tensor-parallel engine's fused residual updates.

The mode has no reference semantics: the HIP engine is held to the CPU statement of it (TorchRefOps), within half of what the mode itself
costs against exact linears -- two runs of it that differ by a bf16 rounding put some values on the other side of an e2m1 border."""
import pytest
import torch

from conftest import rel_l2
from oracle.ref_ops import TorchRefOps

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops():
    from fantasy_world_amd.hip_ops import HipOps
    return HipOps("cuda:0")


def _cond(d):
    return dict(clip_feature=d["clip_feature"], y=d["y"], plucker_fea=d["plucker_fea"], plucker_context_lens=d["plucker_context_lens"])


def _device(ins):
    return {k: (v.cuda() if torch.is_tensor(v) else v) for k, v in ins.items()}


def test_forward_matches_the_cpu_statement(ops, case_l2):
    from fantasy_world_amd.engine import FusionEngine
    case, ins, d = case_l2, case_l2.inputs, _device(case_l2.inputs)
    want, _ = FusionEngine(case.cfg, case.weights.__getitem__, TorchRefOps(emulate_bf16=True), precision="mxfp4").joint_forward(
        ins["x"], ins["timestep"], ins["context"], **_cond(ins))
    got, _ = FusionEngine(case.cfg, case.weights.__getitem__, ops, precision="mxfp4").joint_forward(d["x"], d["timestep"], d["context"], **_cond(d))
    price = rel_l2(want, case.golden["noise_pred"])
    print(f"mxfp4: HIP vs CPU statement {rel_l2(got.float(), want):.3e}, statement vs exact {price:.3e}")
    assert 1.6e-2 < price < 0.4 and rel_l2(got.float(), want) < 0.5 * price


def test_full_width_forward_and_merged_pair(ops, case_cfg1):
    """L = 9216: the large tiles.  Against the golden within the mode's price, merged pair = two forwards bit for bit, again the same bits."""
    from fantasy_world_amd.engine import FusionEngine
    case, d = case_cfg1, _device(case_cfg1.inputs)
    eng = FusionEngine(case.cfg, case.weights.__getitem__, ops, precision="mxfp4")
    pos, _ = eng.joint_forward(d["x"], d["timestep"], d["context"], **_cond(d))
    neg, _ = eng.joint_forward(d["x"], d["timestep"], d["context_neg"], **_cond(d))
    e = rel_l2(pos.float(), case.golden["noise_pred"])
    print(f"mxfp4 linears, {case.name}: {e:.3f} from the reference")
    assert 1.6e-2 < e < 0.4
    p2, n2, _ = eng.joint_forward_pair(d["x"], d["timestep"], d["context"], d["context_neg"], **_cond(d))
    assert torch.equal(p2, pos) and torch.equal(n2, neg)


@pytest.mark.parametrize("precision", ["bf16", "mxfp4"])
def test_tensor_parallel_fused_updates_return_the_same_bits(ops, case_l2, precision):
    """One rank: every residual update that a norm follows runs as one pass; with the two passes in its place the forward's bits are the same."""
    from fantasy_world_amd.hip_ops import HipOps
    from fantasy_world_amd.tensor_parallel import TensorShard, TPFusionEngine

    class Separate(HipOps):
        fused = 0

        def residual_norm(self, x, y=None, bias=None, g1=None, g0=None, h_out=None, **norm):
            if y is None:
                return super().residual_norm(x, None, **norm)
            Separate.fused += 1
            self.residual_add(x, y, bias=bias, g1=g1, g0=g0)
            return self.layernorm(x, out=h_out, **norm)
    case, d = case_l2, _device(case_l2.inputs)
    outs = []
    for o in (ops, Separate("cuda:0")):
        eng = TPFusionEngine(case.cfg, case.weights.__getitem__, o, TensorShard(0, 1, chunks=2, chunk_rows=16), precision=precision)
        outs.append(eng.joint_forward(d["x"], d["timestep"], d["context"], **_cond(d))[0])
    assert Separate.fused >= 4 and torch.equal(outs[0], outs[1])


def test_stand_alone_block_takes_the_mode(ops, case_l2):
    """install_dit_block's runner packs a block's linears for the mode as well."""
    from fantasy_world_amd.blocks import _BlockRunner
    r = _BlockRunner(case_l2.cfg, ops, "mxfp4")
    g, lin, lin_cat = r._packers(case_l2.weights.__getitem__)
    blk = r._pack_dit(0, g, lin, lin_cat)
    assert blk.ffn0.mxfp4 and blk.ffn0.q.is_cuda and not blk.a_g1.mxfp4
