"""A bf16 result of dlmi_orthogonalize is the iteration's result rounded once.

An element that is not the 64-bit result rounded to bf16 must have been off, before its rounding, by its distance to the nearest
tie between two bf16 values.  With |error|_F <= tol, m such elements need the m smallest distances squared to add up to at most
tol^2, which bounds how many there may be.  tol, with r = 2^-22 for storing a matrix in two planes and a product's dropped terms
and sums, |X| <= 1 and |A| <= 1 in a first step: A is off by 3 r, a I + b A + c A A by (|b| + 2 |c|) 3 r + reach r, and their product
by that and 2 reach r more, reach the largest of |a + b q + c q^2|, q in [0, 1].  (Of more steps the bound is too wide to say
anything about single elements; they repeat the same products.)"""
import pytest
import torch

from test_gpu_muon import COEFFS, iterate

WILD = (2.8, -22.4, 22.4)  # 2.8 times a Chebyshev polynomial: as steep as coefficients that are accepted may be


def allowed(exp, tol):
    b = exp.to(torch.bfloat16)
    i = b.view(torch.int16)
    away = torch.where(b.double().abs() > exp.abs(), i - 1, i + 1).view(torch.bfloat16)  # the value on the other side of exp
    d = ((b.double() + away.double()) / 2 - exp).abs().flatten()
    return int((torch.cumsum(d.sort().values ** 2, 0) <= tol ** 2).sum())


@pytest.mark.gpu
@pytest.mark.parametrize("coefs", [COEFFS, WILD])
@pytest.mark.parametrize("shape", [(300, 401), (401, 300), (2048, 1800), (4000, 3900)])
def test_bf16_result_is_rounded_once(dl, shape, coefs):
    gen = torch.Generator(device="cuda").manual_seed(17)
    r = lambda *s: torch.randn(*s, generator=gen, device="cuda")
    # one direction near the largest singular value, where steep coefficients are steepest, and the rest
    G = (r(shape[0], 1) @ r(1, shape[1]) + 0.05 * r(*shape)).bfloat16()
    reach = max(abs(coefs[0] + coefs[1] * q + coefs[2] * q * q) for q in (i / 1000 for i in range(1001)))
    tol = 2.0 ** -22 * ((abs(coefs[1]) + 2 * abs(coefs[2])) * 3 + 3 * reach)
    exp = iterate(G, 1, coefs).contiguous()
    got = dl.orthogonalize(G, steps=1, coefficients=coefs)
    off = int((got != exp.to(torch.bfloat16)).sum())
    most = allowed(exp, tol)
    assert most < 0.2 * exp.numel() and off <= most, "%d of %d elements are not the result rounded, at most %d may be" % (off, exp.numel(), most)
