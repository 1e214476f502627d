"""dlmi_vocab_ce_bwd where rows and classes are of very different magnitudes, against the definition in 64 bits.

Tolerances as derived in test_gpu_vocab_ce.py, taken row by row: a row of X multiplied by a large factor has logits that no
32-bit sum knows to better than that factor's share, and only its own gradient may show it.  One plane holds 11 bits: values of
[1, 2) are 2^-10 apart, so a rounding is off by up to 2^-11 of the value (and two planes by 2^-11 of what the first lost, 2^-22)."""
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
    rel = 2 * dz + 2.0 ** -20 + (2.0 ** -11 if kind == BF16 else 0.0) + V * 2.0 ** -24
    tol = rel[:, None] * (d.abs() @ W.double().abs()) + (2.0 ** -8 if kind == BF16 else 0.0) * eX.abs() + 2.0 ** -39 * 0.25 * W.double().abs().max() * V
    assert ((dX.double() - eX).abs() <= tol)[rest].all()


def elements(X, W, b, labels, g, kind):
    """(dL g, how far an element of it may be off) in 64 bits, element by element.  z is off by dz = (3 2^-22 [fp32] + K 2^-24)
    sum |x w| + 2^-24 |bias|, lse by the mean of dz over the row's probabilities, p by p times twice both plus 2^-21; the
    element is rounded to its planes (2^-22, bf16 2^-11).  fp32 ends at 2^-126: what is smaller may be 0, an element
    (before g) and a result."""
    K = X.shape[1]
    X, W = X.double(), W.double()
    bias = torch.zeros(W.shape[0], device="cuda", dtype=torch.float64) if b is None else b.double()
    dz = ((3 * 2.0 ** -22 if kind == F32 else 0.0) + K * 2.0 ** -24) * (X.abs() @ W.t().abs()) + 2.0 ** -24 * bias.abs()
    dz = torch.where(torch.isfinite(dz), dz, 0.0)  # (a masked class: p is 0)
    p = torch.softmax(X @ W.t() + bias, 1)
    live = (labels >= 0) & (labels < W.shape[0])
    d = p.scatter_add(1, labels.long().clamp(0, W.shape[0] - 1)[:, None], torch.full_like(p[:, :1], -1.0))
    gg = torch.where(live, g.double(), 0.0)[:, None]
    off = p * (2 * dz + 2 * (p * dz).sum(1, keepdim=True) + 2.0 ** -21)
    off = torch.minimum(off, torch.ones_like(off)) + d.abs() * (2.0 ** -22 if kind == F32 else 2.0 ** -11) + 2.0 ** -126
    return d * gg, off * gg.abs()


def bounds(X, W, d, off, kind):
    """Of dX and of dW where magnitudes lie far apart, and no share of the largest is left out of a bound: elements' errors times
    the other operand, whose own rounding is 2^-22 (X times dloss in bf16: 2^-11) of itself, sums in fp32.  Half a step for bf16."""
    X, W = X.double().abs(), W.double().abs()
    again = 2.0 ** -22 if kind == F32 else 2.0 ** -11
    half = 2.0 ** -8 if kind == BF16 else 0.0
    tX = (off + (again + W.shape[0] * 2.0 ** -24) * d.abs()) @ W
    tW = (off + (again + X.shape[0] * 2.0 ** -24) * d.abs()).t() @ X
    return lambda eX: tX + half * eX.abs() + 2.0 ** -126, lambda eW: tW + half * eW.abs() + 2.0 ** -126


def held(dl, X, W, b, labels, g, kind):
    loss, lse = dl.vocab_ce_fwd(X, W, labels, bias=b)
    dX, dW, db = dl.vocab_ce_bwd(X, W, labels, lse, bias=b, dloss=g)
    d, off = elements(X, W, b, labels, g, kind)
    eX, eW = d @ W.double(), d.t() @ X.double()
    tX, tW = bounds(X, W, d, off, kind)
    for got, exp, tol, what in ((dX, eX, tX(eX), "dX"), (dW, eW, tW(eW), "dW")):
        assert torch.isfinite(got).all(), what
        err = (got.double() - exp).abs()
        at = int((err - tol).argmax())
        assert (err <= tol).all(), "%s: off by %.3g where %.3g is allowed, of %.3g" % (what, err.flatten()[at], tol.flatten()[at], exp.flatten()[at])


SIZES = [(90, 96, 700), (700, 70, 1500), (20, 130, 9000)]


@pytest.mark.gpu
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("B,K,V", SIZES)
@pytest.mark.parametrize("far", [30, 60])
def test_a_far_class_that_nobody_chooses(dl, B, K, V, far, kind):
    """Rows of W that are 2^30 and 2^60 larger than the rest (padding left as it was), their classes masked by the bias: the
    others' gradients are those of a vocabulary without them."""
    X, W, b, labels = make(B, K, V, kind, True, 0.1, 41)
    masked = [3, V // 2, V - 1]
    for i, v in enumerate(masked):
        W[v] = (W[v].float() * 2.0 ** (far - i)).to(kind)
        b[v] = float("-inf")
        labels[labels == v] = 0
    g = torch.full((B,), 0.5, device="cuda")
    held(dl, X, W, b, labels, g, kind)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("B,K,V", SIZES)
@pytest.mark.parametrize("low", [-20, -45])
def test_rows_of_far_smaller_weight(dl, B, K, V, low, kind):
    """Half of the rows count 2^-20 or 2^-45 of the others and choose among classes that the others give no probability: dW of
    those classes is theirs alone, as exact as anybody's."""
    X, W, b, labels = make(B, K, V, kind, False, 0.0, 43)
    small = torch.arange(B, device="cuda") % 2 == 1
    theirs = torch.arange(V, device="cuda") % 2 == 1
    # the two kinds of rows and classes share no feature but the first, which keeps them apart by 120
    X[small, K // 2:] = 0
    X[~small, 1:K // 2] = 0
    W[theirs, K // 2:] = 0
    W[~theirs, 1:K // 2] = 0
    X[:, 0] = torch.where(small, 8.0, -8.0).to(kind)
    W[:, 0] = torch.where(theirs, 7.5, -7.5).to(kind)
    labels = torch.where(small, labels // 2 * 2 + 1, labels // 2 * 2).clamp(0, V - 1).int()
    labels[(labels % 2 == 1) != small] -= 1
    labels = torch.where(small, torch.where(labels % 2 == 1, labels, 1), torch.where(labels % 2 == 0, labels, 0)).int()
    g = torch.where(small, 2.0 ** low, 1.0)
    held(dl, X, W, b, labels, g, kind)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", KINDS)
def test_magnitudes_spread_over_many_powers(dl, kind):
    """Rows of W, rows of X and dloss each over 2^40, zero rows and rows left out among them."""
    B, K, V = 130, 64, 900
    X, W, b, labels = make(B, K, V, kind, True, 0.2, 47)
    gen = torch.Generator(device="cuda").manual_seed(5)
    power = lambda n, lo, hi: 2.0 ** torch.randint(lo, hi, (n,), generator=gen, device="cuda").float()
    X = (X.float() * power(B, -40, 1)[:, None]).to(kind)
    W = (W.float() * power(V, -40, 1)[:, None]).to(kind)
    X[7] = 0
    W[11] = 0
    g = power(B, -40, 1)
    g[13] = 0
    held(dl, X, W, b, labels, g, kind)


@pytest.mark.gpu
def test_far_classes_recorded_and_replayed(pkg):
    """One recorded step, replayed on ordinary and on far rows in turn: every replay is the eager step's bits."""
    d = pkg.Dlmi(0)
    try:
        stream = torch.cuda.Stream()
        d.set_stream(stream)
        X, W, b, labels = make(90, 64, 800, F32, True, 0.2, 12)
        far = W.clone()
        far[5] *= 2.0 ** 40
        b[5] = float("-inf")
        labels[labels == 5] = 6
        now = W.clone()
        out = dict(loss=torch.empty(90, device="cuda"), lse=torch.empty(90, device="cuda"))
        grads = dict(dX=torch.empty_like(X), dW=torch.empty_like(W), db=torch.empty_like(b))
        torch.cuda.synchronize()
        def step(o, g):
            d.vocab_ce_fwd(X, now, labels, bias=b, **o)
            d.vocab_ce_bwd(X, now, labels, o["lse"], bias=b, scale=0.1, **g)
        with torch.cuda.stream(stream):
            eo, eg = {k: v.clone() for k, v in out.items()}, {k: v.clone() for k, v in grads.items()}
            step(eo, eg)
            stream.synchronize()
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=stream):
                step(out, grads)
            for w in (W, far, W, far):
                now.copy_(w)
                step(eo, eg)
                graph.replay()
                stream.synchronize()
                assert all(torch.equal(out[k], eo[k]) for k in out) and all(torch.equal(grads[k], eg[k]) for k in grads)
    finally:
        torch.cuda.synchronize()
        d.close()
