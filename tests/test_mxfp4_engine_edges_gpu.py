"""-m gpu: precision="mxfp4" through the whole forward, at bounds taken from what the mode measures (0.134 to 0.146 from the reference; the HIP
engine 0.04 from the CPU statement)."""
import pytest

from conftest import rel_l2
from oracle.ref_ops import TorchRefOps
from test_mxfp4_engine_gpu import _cond, _device

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops():
    from fantasy_world_amd.hip_ops import HipOps
    return HipOps("cuda:0")


def test_the_first_run_check_passes_on_one_gpu(ops):
    from fantasy_world_amd import parallel
    res = parallel.golden_self_check(None, ops, precision="mxfp4")
    print(res)
    assert res["ok"] and res["tol"] <= 0.18 and res["rel_l2_max_over_ranks"] > 0.1, res


def test_forward_within_the_measured_distances(ops, case_l2):
    from fantasy_world_amd.engine import FusionEngine
    case, ins, d = case_l2, case_l2.inputs, _device(case_l2.inputs)
    want, _ = FusionEngine(case.cfg, case.weights.__getitem__, TorchRefOps(emulate_bf16=True), precision="mxfp4").joint_forward(
        ins["x"], ins["timestep"], ins["context"], **_cond(ins))
    got, _ = FusionEngine(case.cfg, case.weights.__getitem__, ops, precision="mxfp4").joint_forward(d["x"], d["timestep"], d["context"], **_cond(d))
    price, off = rel_l2(got.float(), case.golden["noise_pred"]), rel_l2(got.float(), want)
    print(f"HIP from the reference {price:.3f}, from the CPU statement {off:.3f}")
    # two runs of the mode that differ by bf16 roundings are 0.04 apart where a value sits on a border; half of the mode's price is no longer that
    assert 0.1 < price < 0.18 and off < 0.06, (price, off)
