"""vocab_ce_bwd of the binding: gradients that are not needed are not formed, the others are the same bits."""
import pytest
import torch

from test_gpu_vocab_ce import BF16, F32, make


@pytest.mark.gpu
@pytest.mark.parametrize("kind", [F32, BF16])
@pytest.mark.parametrize("bias", [False, True])
def test_only_what_is_needed(dl, kind, bias):
    X, W, b, labels = make(90, 70, 900, kind, bias, 0.2, 6)
    loss, lse = dl.vocab_ce_fwd(X, W, labels, bias=b)
    full = dict(zip(("dX", "dW", "db"), dl.vocab_ce_bwd(X, W, labels, lse, bias=b, scale=0.5)))
    assert (full["db"] is None) == (not bias)
    for needs in (("dX",), ("dW",), ("dX", "dW"), ("dW", "db"), ("dX", "db")):
        got = dict(zip(("dX", "dW", "db"), dl.vocab_ce_bwd(X, W, labels, lse, bias=b, scale=0.5, needs=needs)))
        for k, v in got.items():
            if k in needs and full[k] is not None:
                assert torch.equal(v, full[k]), (needs, k)
            else:
                assert v is None, (needs, k)


@pytest.mark.gpu
def test_needs_and_accumulate(dl, pkg):
    X, W, b, labels = make(40, 30, 300, F32, True, 0.0, 7)
    loss, lse = dl.vocab_ce_fwd(X, W, labels, bias=b)
    dX, dW, db = dl.vocab_ce_bwd(X, W, labels, lse, bias=b)
    ones = torch.ones_like(db)
    got = dl.vocab_ce_bwd(X, W, labels, lse, bias=b, db=ones, accumulate=True, needs=("db",))
    assert got[0] is None and got[1] is None and torch.equal(got[2], 1.0 + db)
    with pytest.raises(AssertionError, match="so far"):
        dl.vocab_ce_bwd(X, W, labels, lse, bias=b, accumulate=True, needs=("dW",))
    with pytest.raises(AssertionError, match="needs"):
        dl.vocab_ce_bwd(X, W, labels, lse, bias=b, needs=("dx",))
    with pytest.raises(AssertionError, match="not needed"):
        dl.vocab_ce_bwd(X, W, labels, lse, bias=b, dX=dX, needs=("dW",))
    with pytest.raises(pkg.DlmiError, match="no gradient"):
        dl.vocab_ce_bwd(X, W, labels, lse, bias=b, needs=())
    with pytest.raises(pkg.DlmiError, match="no gradient"):
        dl.vocab_ce_bwd(X, W, labels, lse, needs=("db",))
