"""dlmi_orthogonalize and dlmi_opt_muon against the iteration in 64 bits.

Tolerances.  With |X|_F = 1 at the start, one step stores X, A = X X^T and b A + c A A in two f16 planes: each element off
by at most 2^-23 of itself (hi and lo of 11 bits, rounded to nearest; below 2^-18 of a matrix's largest element an absolute
2^-37 instead), and multiplies with sums in fp32.  Let r = 2^-22 stand for one storing plus the dropped lo lo terms and the
sums.  The error a step adds to X, in the Frobenius norm, is at most r |X| (|a| from storing X, |b| + |c| from storing the
products, which are bounded by 2 on the way: at most 12 r |X|, |X|_F growing by at most a factor a a step until it is the
result's), and a later step multiplies an error by at most a.  Summed: |error|_F <= steps * 12 * 2^-22 * a^steps.  Against
the result's norm that is the relative tolerance `tol` below; a bf16 result is off by half a step, 2^-8 of each element at
most, more (0.43 of that in the norm, roundings being spread evenly: what is left of 2^-8, 2.2e-3, is above the 2^-12 of its
last step's operands times the 3.4 that step multiplies by at most, 8.4e-4)."""
import ctypes

import numpy as np
import pytest
import torch

COEFFS = (3.4445, -4.7750, 2.0315)


def iterate(G, steps=5, coefs=COEFFS, eps=1e-7):
    a, b, c = coefs
    X = G.double()
    X = X / (X.norm() + eps)
    flip = X.shape[0] > X.shape[1]
    X = X.t() if flip else X
    for _ in range(steps):
        A = X @ X.t()
        X = a * X + (b * A + c * A @ A) @ X
    return X.t() if flip else X


def close(got, exp, steps=5, coefs=COEFFS):
    got, exp = got.double().cpu(), exp.cpu()
    assert torch.isfinite(got).all()
    tol = steps * 12 * 2.0 ** -22 * coefs[0] ** steps
    if got.dtype == torch.bfloat16:
        tol += 2.0 ** -8 * exp.norm().item()
    err = (got - exp).norm().item()
    assert err <= tol, "off by %.3g, allowed %.3g" % (err, tol)
    return err


SHAPES = [(1, 1), (1, 7), (5, 1), (3, 3), (16, 16), (31, 33), (64, 64), (65, 64), (64, 127), (128, 784), (500, 130), (257, 255),
          (10, 1000), (1000, 10)]


@pytest.mark.gpu
@pytest.mark.parametrize("kind", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("shape", SHAPES)
def test_orthogonalize(dl, shape, kind):
    gen = torch.Generator().manual_seed(shape[0] * 1000 + shape[1])
    G = torch.randn(shape, generator=gen).to(kind)
    out = dl.orthogonalize(G.cuda())
    assert out.dtype == kind
    exp = iterate(G)
    tol = 5 * 12 * 2.0 ** -22 * COEFFS[0] ** 5 + (2.0 ** -8 * exp.norm().item() if kind == torch.bfloat16 else 0.0)
    err = (out.double().cpu() - exp).norm().item()
    assert err <= tol, (shape, err, tol)


@pytest.mark.gpu
@pytest.mark.parametrize("shape", [(512, 512), (1024, 1100), (2048, 1800), (3000, 520)])
def test_orthogonalize_large(dl, shape):
    """Sizes that take the larger tiles; the 64-bit iteration runs on the GPU."""
    gen = torch.Generator(device="cuda").manual_seed(7)
    G = torch.randn(shape, generator=gen, device="cuda")
    close(dl.orthogonalize(G), iterate(G))


@pytest.mark.gpu
def test_orthogonalize_low_rank_and_scales(dl):
    """Rank 4 plus noise: the weak directions are the ones the iteration multiplies; gradients of 1e-20 and 1e15."""
    gen = torch.Generator().manual_seed(3)
    G = torch.randn(96, 4, generator=gen) @ torch.randn(4, 200, generator=gen) + 0.01 * torch.randn(96, 200, generator=gen)
    for scale in (1.0, 1e-20, 1e15):
        g = (G * scale).float()
        close(dl.orthogonalize(g.cuda(), eps=0.0), iterate(g, eps=0.0))


@pytest.mark.gpu
@pytest.mark.parametrize("steps", [1, 2, 7])
def test_orthogonalize_steps_and_alias(dl, steps):
    gen = torch.Generator().manual_seed(5)
    G = torch.randn(70, 150, generator=gen)
    exp = iterate(G, steps, (2.0, -1.5, 0.5))
    d = G.cuda()
    out = dl.orthogonalize(d, steps=steps, coefficients=(2.0, -1.5, 0.5), out=d)
    assert out.data_ptr() == d.data_ptr()
    close(out, exp, steps, (2.0, -1.5, 0.5))


@pytest.mark.gpu
def test_orthogonalize_zero_and_nonfinite(dl):
    assert torch.equal(dl.orthogonalize(torch.zeros(40, 70, device="cuda")), torch.zeros(40, 70, device="cuda"))
    for bad in (float("nan"), float("inf")):
        G = torch.ones(40, 70, device="cuda")
        G[3, 5] = bad
        assert not torch.isfinite(dl.orthogonalize(G)).any()
    assert dl.orthogonalize(torch.empty(0, 5, device="cuda")).shape == (0, 5)


def muon_exact(p, g, m, lr, mom, wd, nesterov, eps=1e-7):
    p, g, m = p.double(), g.double(), m.double()
    m = mom * m + g
    u = g + mom * m if nesterov else m
    return p - lr * iterate(u, eps=eps) - wd * p, m


@pytest.mark.gpu
@pytest.mark.parametrize("nesterov", [True, False])
def test_muon_step_of_several_shapes(dl, nesterov):
    gen = torch.Generator().manual_seed(11)
    shapes = [(64, 96), (130, 40), (64, 96), (1, 9), (64, 96), (96, 64)]
    data = [[torch.randn(s, generator=gen) for _ in range(3)] for s in shapes]
    dev = [[t.cuda() for t in d] for d in data]
    lrs = [0.01 * (i + 1) for i in range(len(shapes))]
    dl.opt_muon([(p, g, m, lr) for (p, g, m), lr in zip(dev, lrs)], lr=0.0, momentum=0.9, wd=0.01, nesterov=nesterov)
    for (p, g, m), (dp, dg, dm), lr in zip(data, dev, lrs):
        ep, em = muon_exact(p, g, m, lr, 0.9, 0.01, nesterov)
        assert torch.count_nonzero(dg) == 0
        # the momentum: two roundings; the parameter: the step's error times lr, and three roundings of values below 8
        assert (dm.cpu().double() - em).abs().max() <= 2 * 2.0 ** -24 * 8
        tol = lr * 5 * 12 * 2.0 ** -22 * COEFFS[0] ** 5 + 3 * 2.0 ** -24 * ep.norm().item()
        assert (dp.cpu().double() - ep).norm() <= tol


@pytest.mark.gpu
def test_muon_grouped_is_one_by_one(dl):
    """Many matrices of one shape share launches, more than one launch's worth of them: same bits as one at a time where
    the tile is the same."""
    gen = torch.Generator().manual_seed(2)
    data = [[torch.randn(20, 30, generator=gen) for _ in range(3)] for _ in range(37)]
    one, all_ = [[t.cuda() for t in d] for d in data], [[t.cuda() for t in d] for d in data]
    for d in one:
        dl.opt_muon([d], lr=0.02)
    dl.opt_muon(all_, lr=0.02)
    for a, b in zip(one, all_):
        assert all(torch.equal(x, y) for x, y in zip(a, b))


@pytest.mark.gpu
def test_muon_unaligned_views_leave_the_rest_alone(dl):
    """Matrices inside one packed array at odd offsets, as a model's parameters lie."""
    gen = torch.Generator().manual_seed(4)
    R, C = 33, 47
    bufs = [torch.randn(R * C + 11, generator=gen) for _ in range(3)]
    dev = [b.cuda() for b in bufs]
    v = [d[3:3 + R * C].view(R, C) for d in dev]
    dl.opt_muon([v], lr=0.02, momentum=0.95, wd=0.0)
    ep, _ = muon_exact(*[b[3:3 + R * C].view(R, C) for b in bufs], 0.02, 0.95, 0.0, True)
    assert (v[0].cpu().double() - ep).norm() <= 0.02 * 5 * 12 * 2.0 ** -22 * COEFFS[0] ** 5 + 3 * 2.0 ** -24 * ep.norm()
    for b, d in zip(bufs, dev):
        assert torch.equal(b[:3], d[:3].cpu()) and torch.equal(b[3 + R * C:], d[3 + R * C:].cpu())


@pytest.mark.gpu
def test_muon_captured_and_replayed(pkg):
    """A step recorded into a HIP graph, replayed with eager work between: every replay is the eager step's bits."""
    d = pkg.Dlmi(0)
    try:
        stream = torch.cuda.Stream()
        d.set_stream(stream)
        gen = torch.Generator().manual_seed(9)
        p0, m0 = torch.randn(100, 60, generator=gen), torch.randn(100, 60, generator=gen)
        gs = [torch.randn(100, 60, generator=gen) for _ in range(4)]
        pe, me, ge = p0.cuda(), m0.cuda(), gs[0].cuda()
        p, m, g = p0.cuda(), m0.cuda(), gs[0].cuda()
        torch.cuda.synchronize()
        with torch.cuda.stream(stream):
            d.opt_muon([(pe.clone(), ge.clone(), me.clone())], lr=0.02)     # grows the scratch outside the capture
            stream.synchronize()
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=stream):
                d.opt_muon([(p, g, m)], lr=0.02)
            for k in range(4):
                ge.copy_(gs[k])
                g.copy_(gs[k])
                d.opt_muon([(pe, ge, me)], lr=0.02)
                graph.replay()
                stream.synchronize()
                assert torch.equal(p, pe) and torch.equal(m, me) and torch.count_nonzero(g) == 0
    finally:
        torch.cuda.synchronize()
        d.close()


@pytest.mark.gpu
def test_muon_refusals(dl, pkg):
    a, b, c = (torch.ones(8, 8, device="cuda") for _ in range(3))
    with pytest.raises(pkg.DlmiError, match="overlap"):
        dl.opt_muon([(a, b, a)], lr=0.1)
    with pytest.raises(pkg.DlmiError, match="overlap"):
        dl.opt_muon([(a, b, c), (a, b.clone(), c.clone())], lr=0.1)
    with pytest.raises(pkg.DlmiError, match="steps"):
        dl.orthogonalize(a, steps=0)
    with pytest.raises(pkg.DlmiError, match="steps"):
        dl.orthogonalize(a, steps=65)
    with pytest.raises(pkg.DlmiError, match="coefficients"):
        dl.orthogonalize(a, coefficients=(30.0, 1.0, 1.0))
    with pytest.raises(pkg.DlmiError, match="coefficients"):
        dl.orthogonalize(a, coefficients=(float("nan"), 1.0, 1.0))
    with pytest.raises(pkg.DlmiError, match="eps"):
        dl.orthogonalize(a, eps=-1.0)
    with pytest.raises(AssertionError):
        dl.orthogonalize(a.half())
    with pytest.raises(AssertionError):
        dl.orthogonalize(torch.ones(8, 4, device="cuda").t())
    with pytest.raises(AssertionError):
        dl.opt_muon([(a, b.bfloat16(), c)], lr=0.1)
    with pytest.raises(AssertionError):
        dl.orthogonalize(torch.ones(8, 8))
    assert torch.equal(a, torch.ones_like(a)) and torch.equal(b, torch.ones_like(b))
    lib = dl.lib
    ns = pkg.NewtonSchulz(*COEFFS, 5, 1e-7)
    sz = ctypes.c_size_t
    assert lib.dlmi_orthogonalize(None, 0, sz(8), sz(8), None, None, ctypes.byref(ns)) == -1
    assert lib.dlmi_orthogonalize(dl.ctx, 0, sz(8), sz(8), None, None, ctypes.byref(ns)) == -1
    assert lib.dlmi_orthogonalize(dl.ctx, 5, sz(8), sz(8), None, None, ctypes.byref(ns)) == -1
    assert lib.dlmi_orthogonalize(dl.ctx, 0, sz(1 << 20), sz(8), None, None, ctypes.byref(ns)) == -1
    assert lib.dlmi_orthogonalize(dl.ctx, 0, sz(8), sz(8), None, None, None) == -1
    assert lib.dlmi_opt_muon(dl.ctx, sz(1), None, ctypes.c_float(0), 0, ctypes.c_float(0), ctypes.byref(ns)) == -1
