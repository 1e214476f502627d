"""dlmi_vocab_ce_fwd / _bwd at sizes that reach every tile the planner chooses among, as it chooses on 256 CUs, against the
definition in 64 bits.

Tolerances as derived in test_gpu_vocab_ce.py and test_gpu_vocab_ce_far.py, but for the rounding of a plane of 11 bits: values of
[1, 2) are 2^-10 apart, half of that is 2^-11 of the value.  It counts once for an element of dL of bf16 tensors and once more,
in dW, for X times dloss (`plane`); where one term carries a whole sum, it is all there is."""
import pytest
import torch

from test_gpu_vocab_ce import BF16, F32, dz_of, exact, make, within
from test_gpu_vocab_ce_far import held

KINDS = [F32, BF16]


def check(dl, B, K, V, kind, bias=True, left_out=0.0, dloss=False, seed=0):
    X, W, b, labels = make(B, K, V, kind, bias, left_out, seed + B * 7 + K * 3 + V)
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dl_rows = torch.randn(B, generator=gen, device="cuda") if dloss else None
    g = torch.full((B,), 0.37, device="cuda") * (dl_rows if dloss else 1.0)
    loss, lse = dl.vocab_ce_fwd(X, W, labels, bias=b)
    eloss, else_, edX, edW, edb, mags, mX, mW, mb, floor = exact(X, W, b, labels, g)
    dz = dz_of(kind, K, mags)
    top = else_.abs().max().item()
    within(lse, else_, dz + 2.0 ** -22 + 2.0 ** -24 * top, "lse")
    within(loss, eloss, 2 * dz + 2.0 ** -22 + 2.0 ** -23 * (top + mags[0]), "loss")
    dX, dW, db = dl.vocab_ce_bwd(X, W, labels, lse, bias=b, dloss=dl_rows, scale=0.37)
    plane, half = (2.0 ** -11, 2.0 ** -8) if kind == BF16 else (0.0, 0.0)
    rel = 2 * dz + 2.0 ** -20
    within(dX, edX, (rel + plane + V * 2.0 ** -24) * mX + half * edX.abs() + floor[0], "dX")
    within(dW, edW, (rel + (2 * plane if dloss else plane) + B * 2.0 ** -24) * mW + half * edW.abs() + floor[1], "dW")
    assert (dX[labels < 0] == 0).all()
    if bias:
        within(db, edb, (rel + B * 2.0 ** -24) * mb + floor[2], "db")


@pytest.mark.gpu
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("B,K,V", [(8192, 1030, 30000),   # 256 wide in four pieces, the last shorter; dW 256 (BF16), 128 (FP32)
                                   (777, 1000, 30011),    # one piece in many slices of dX; 256 (BF16), 128 (FP32)
                                   (900, 500, 30000),     # 256 and dW 256 in both
                                   (3000, 1100, 9000),    # 256 and dW 128 (BF16), 128 and 128 (FP32)
                                   (5789, 415, 17032),    # 256 and dW 64
                                   (2000, 600, 20011)])   # 128 and dW 128, two pieces
def test_large_tiles(dl, B, K, V, kind):
    check(dl, B, K, V, kind, left_out=0.1, dloss=True)
    check(dl, B, K, V, kind, bias=False, seed=1)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("B", [40, 300])
@pytest.mark.parametrize("K", [1500, 2100])
def test_wide_rows(dl, B, K, kind):
    """Rows of more than 1024 features are packed from more registers, of more than 2048 read twice."""
    check(dl, B, K, 1003, kind, left_out=0.1)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("bias", [False, True])
@pytest.mark.parametrize("B,K", [(1, 1020), (7, 1020), (16, 77), (24, 1020), (32, 2048), (50, 1020), (64, 130)])
def test_few_rows_against_many_classes(dl, B, K, bias, kind):
    """So many classes that every workgroup of the few-row forward takes several blocks of 64 of them."""
    V = 70001
    X, W, b, labels = make(B, K, V, kind, bias, 0.0, 3 + B)
    labels[0] = V - 1
    loss, lse = dl.vocab_ce_fwd(X, W, labels, bias=b)
    eloss, else_, _, _, _, mags, _, _, _, _ = exact(X, W, b, labels, torch.ones(B, device="cuda"))
    dz = dz_of(kind, K, mags)
    top = else_.abs().max().item()
    within(lse, else_, dz + 2.0 ** -22 + 2.0 ** -24 * top, "lse")
    within(loss, eloss, 2 * dz + 2.0 ** -22 + 2.0 ** -23 * (top + mags[0]), "loss")


@pytest.mark.gpu
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("B,K,V", [(900, 500, 30000), (2000, 600, 20011), (3000, 1100, 9000)])
def test_far_classes_in_large_tiles(dl, B, K, V, kind):
    """A class 2^40 larger than the rest, masked, in the last piece alone; rows of far smaller weight among the others."""
    X, W, b, labels = make(B, K, V, kind, True, 0.1, 53)
    W[V - 2] = (W[V - 2].float() * 2.0 ** 40).to(kind)
    b[V - 2] = float("-inf")
    labels[labels == V - 2] = 0
    held(dl, X, W, b, labels, torch.full((B,), 0.5, device="cuda"), kind)
    g = torch.where(torch.arange(B, device="cuda") % 3 == 0, 2.0 ** -30, 1.0)
    held(dl, X, W, b, labels, g, kind)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", KINDS)
def test_the_same_bits_again(dl, kind):
    X, W, b, labels = make(3000, 1100, 9000, kind, True, 0.1, 59)
    one = dl.vocab_ce_fwd(X, W, labels, bias=b)
    two = dl.vocab_ce_fwd(X, W, labels, bias=b)
    assert all(torch.equal(x, y) for x, y in zip(one, two))
    one = dl.vocab_ce_bwd(X, W, labels, two[1], bias=b, scale=0.1)
    again = dl.vocab_ce_bwd(X, W, labels, two[1], bias=b, scale=0.1)
    assert all(torch.equal(x, y) for x, y in zip(one, again))
