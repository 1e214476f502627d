"""dlmi_vocab_ce_bwd where rows and classes are of very different magnitudes, against the definition in 64 bits.

Tolerances as derived in test_gpu_vocab_ce.py, taken row by row: a row of X multiplied by a large factor has logits that no
32-bit sum knows to better than that factor's share, and only its own gradient may show it."""
import pytest
import torch

from test_gpu_vocab_ce import BF16, F32, make

KINDS = [F32, BF16]


def definition(X, W, b, labels, g):
    """Rows' dz, and (dX, dW, db) with the sums of magnitudes behind them, in 64 bits; g [B]."""
    X, W = X.double(), W.double()
    z = X @ W.t() + (0.0 if b is None else b.double())
    mag = (X.abs() @ W.t().abs()).amax(1)
    live = (labels >= 0) & (labels < W.shape[0])
    d = torch.softmax(z, 1)
    d.scatter_add_(1, labels.long().clamp(0, W.shape[0] - 1)[:, None], torch.full_like(z[:, :1], -1.0))
    d = torch.where(live[:, None], d * g.double()[:, None], 0.0)
    return mag, d, d @ W, d.t() @ X, d.sum(0)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("B", [1, 16, 50, 64, 90])
@pytest.mark.parametrize("far", [1e6, 1e7, 1e12])
def test_far_logits_keep_their_gradients_finite(dl, B, far, kind):
    """Logits of 10^6 and more, formed once by the forward and once by the backward, differ by more than 1: no probability
    passes 1 for that, so nothing overflows and |dL| stays at most |g|."""
    K, V = 1024, 2000
    X, W, b, labels = make(B, K, V, kind, True, 0.0, 31 + B)
    X = (X.float() * far).to(kind)
    loss, lse = dl.vocab_ce_fwd(X, W, labels, bias=b)
    dX, dW, db = dl.vocab_ce_bwd(X, W, labels, lse, bias=b, scale=0.5)
    for t in (loss, lse, dX, dW, db):
        assert torch.isfinite(t).all()
    # |dL| <= 1 for each class, so a sum over classes or rows is at most that of the magnitudes (and its roundings: 1 %)
    assert (db.abs() <= 0.505 * B).all()
    assert (dX.double().abs() <= 0.505 * W.double().abs().sum(0)).all()
    assert (dW.double().abs() <= 0.505 * X.double().abs().sum(0)).all()


@pytest.mark.gpu
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("B", [50, 90])
def test_a_far_row_leaves_the_others_alone(dl, B, kind):
    """dX of the other rows is as exact as without it."""
    K, V = 96, 700
    X, W, b, labels = make(B, K, V, kind, True, 0.1, 5)
    X[4] = (X[4].float() * 1e12).to(kind)
    X[9] = (X[9].float() * 1e6).to(kind)
    labels[4] = labels[9] = 3
    g = torch.full((B,), 0.25, device="cuda")
    mag, d, eX, eW, eb = definition(X, W, b, labels, g)
    loss, lse = dl.vocab_ce_fwd(X, W, labels, bias=b)
    dX, dW, db = dl.vocab_ce_bwd(X, W, labels, lse, bias=b, scale=0.25)
    assert all(torch.isfinite(t).all() for t in (dX, dW, db))
    rest = torch.tensor([i for i in range(B) if i not in (4, 9)], device="cuda")
    dz = ((3 * 2.0 ** -22 if kind == F32 else 0.0) + K * 2.0 ** -24) * mag + 2.0 ** -24 * b.abs().max().item()
    rel = 2 * dz + 2.0 ** -20 + (2.0 ** -12 if kind == BF16 else 0.0) + V * 2.0 ** -24
    tol = rel[:, None] * (d.abs() @ W.double().abs()) + (2.0 ** -8 if kind == BF16 else 0.0) * eX.abs() + 2.0 ** -39 * 0.25 * W.double().abs().max() * V
    assert ((dX.double() - eX).abs() <= tol)[rest].all()
