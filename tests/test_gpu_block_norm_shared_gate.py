"""dlmi_block_norm_fwd / _bwd with a gate shared by rows that are wider than a wavefront, against the formula in 64 bits and its
gradient; tolerances and checks of test_gpu_block_norm.py.  A workgroup takes at least four rows: runs of 3 are whole in one
workgroup, runs of 17 and of all rows are cut into slices; rows wider than 8192 read the gate again for every row."""
import pytest

from test_gpu_block_norm import BF16, F32, run


@pytest.mark.gpu
@pytest.mark.parametrize("kind", [F32, BF16])
@pytest.mark.parametrize("act", ["SIGMOID", "TANH"])
@pytest.mark.parametrize("gate_rows", [3, 17, 45])
@pytest.mark.parametrize("H", [130, 777, 1030, 4096, 5000, 9001, 16384])
def test_wide_rows_share_a_gate(dl, pkg, H, gate_rows, act, kind):
    run(dl, pkg, 45, H, kind, "RMS", "LAYER", gate_rows=gate_rows, act=act, bs=0.5)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", [F32, BF16])
def test_runs_of_a_training_batch(dl, pkg, kind):
    run(dl, pkg, 1550, 777, kind, "LAYER", "LAYER", gate_rows=50, act="TANH", bs=0.5)
    run(dl, pkg, 2500, 1024, kind, "RMS", "RMS", gate_rows=2500, act="TANH", biases=False, bs=0.25)
