"""The vocabulary cross entropy, the orthogonalization and the block norms at the largest counts of rows, features, classes and
columns that their headers name, the other sizes small; tolerances of their own test files."""
import pytest
import torch

import test_gpu_block_norm
import test_gpu_vocab_ce_tiles
from test_gpu_muon import COEFFS, iterate

KINDS = [torch.float32, torch.bfloat16]


@pytest.mark.gpu
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("B,K,V", [(262144, 9, 300), (3, 65536, 40), (70, 65536, 200), (66, 5, 2 ** 20 + 77), (5, 3, 2 ** 21 + 1)])
def test_vocab_ce(dl, B, K, V, kind):
    test_gpu_vocab_ce_tiles.check(dl, B, K, V, kind, left_out=0.1 if B > 10 else 0.0)


@pytest.mark.gpu
def test_vocab_ce_beyond(dl, pkg):
    for B, K in ((262145, 1), (1, 65537)):
        X, W = torch.ones(B, K, device="cuda"), torch.ones(2, K, device="cuda")
        with pytest.raises(pkg.DlmiError, match="too many"):
            dl.vocab_ce_fwd(X, W, torch.zeros(B, device="cuda", dtype=torch.int32))


@pytest.mark.gpu
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("shape", [(1, 65536), (65536, 1), (65536, 33), (70, 65536)])
def test_orthogonalize(dl, shape, kind):
    gen = torch.Generator(device="cuda").manual_seed(3)
    G = torch.randn(shape, generator=gen, device="cuda").to(kind)
    out, exp = dl.orthogonalize(G), iterate(G)
    tol = 5 * 12 * 2.0 ** -22 * COEFFS[0] ** 5 + (2.0 ** -8 * exp.norm().item() if kind == torch.bfloat16 else 0.0)
    assert (out.double() - exp).norm().item() <= tol


@pytest.mark.gpu
@pytest.mark.parametrize("kind", KINDS)
def test_block_norm(dl, pkg, kind):
    test_gpu_block_norm.run(dl, pkg, 300000, 3, kind, "RMS", "LAYER", gate_rows=7, act="TANH", bs=0.5)
    test_gpu_block_norm.run(dl, pkg, 70000, 64, kind, "LAYER", "RMS", gate_rows=70000, act="SIGMOID", bs=0.5)
    test_gpu_block_norm.run(dl, pkg, 1, 16384, kind, "LAYER", "LAYER", gate_rows=1, act="TANH", bs=0.5)
