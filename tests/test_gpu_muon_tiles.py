"""dlmi_orthogonalize and dlmi_opt_muon at sizes that reach the wide tiles and the sharing of tiles between workgroups, as the
planner chooses on 256 CUs, against the iteration in 64 bits.  Tolerances as derived in test_gpu_muon.py."""
import pytest
import torch

from test_gpu_muon import COEFFS, iterate, muon_exact

TOL = 5 * 12 * 2.0 ** -22 * COEFFS[0] ** 5


@pytest.mark.gpu
@pytest.mark.parametrize("kind", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("shape", [(4096, 4096),    # 256 wide; the 136 symmetric tiles shared by all CUs
                                   (4000, 3900),    # the same with padding, transposed
                                   (300, 40000),    # 256 wide; the last 58 of the update's 314 tiles shared too
                                   (2048, 1800),    # 128 wide, the symmetric products shared
                                   (1100, 9000),    # 128 wide, long loops shared
                                   (100, 20000)])   # 64 wide, three tiles with long loops shared
def test_orthogonalize_wide_tiles(dl, shape, kind):
    gen = torch.Generator(device="cuda").manual_seed(7)
    G = torch.randn(shape, generator=gen, device="cuda").to(kind)
    out = dl.orthogonalize(G)
    exp = iterate(G)
    assert out.dtype == kind and torch.isfinite(out).all()
    err = (out.double() - exp).norm().item()
    tol = TOL + (2.0 ** -8 * exp.norm().item() if kind == torch.bfloat16 else 0.0)
    assert err <= tol, "off by %.3g, allowed %.3g" % (err, tol)
    assert torch.equal(out, dl.orthogonalize(G))


@pytest.mark.gpu
@pytest.mark.parametrize("count,shape", [(16, (2000, 2040)),   # 256 wide: whole rounds, and the last 64 of 576 tiles shared
                                         (20, (1030, 1100)),   # the same with much padding
                                         (3, (300, 8000)),     # 256 wide: the tiles of all three products shared
                                         (11, (112, 3141))])   # 128 wide, eleven tiles with long loops shared
def test_grouped_steps_in_wide_tiles(dl, count, shape):
    gen = torch.Generator(device="cuda").manual_seed(11)
    data = [[torch.randn(shape, generator=gen, device="cuda") for _ in range(3)] for _ in range(count)]
    old = [[t.clone() for t in d] for d in data]
    dl.opt_muon([tuple(d) for d in data], lr=0.02, momentum=0.9, wd=0.01)
    for (p, g, m), (op, og, om) in zip(data, old):
        ep, em = muon_exact(op, og, om, 0.02, 0.9, 0.01, True)
        assert torch.count_nonzero(g) == 0
        # two roundings of values below 8; the step's error times lr, and three roundings of values below 8
        assert (m.double() - em).abs().max() <= 2 * 2.0 ** -24 * 8
        assert (p.double() - ep).norm() <= 0.02 * TOL + 3 * 2.0 ** -24 * ep.norm()
