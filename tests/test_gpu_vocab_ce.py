"""dlmi_vocab_ce_fwd / _bwd against the definition in 64 bits.

Tolerances.  A logit of fp32 tensors is a sum of K products of two-plane operands: each operand off by at most 2^-22 of itself
(hi and lo of 11 bits; elements below 2^-18 of their row's or piece's largest by 2^-40 of that), the dropped lo lo another
2^-22, and sums in fp32 of at most K 2^-24: with A = max_bv sum_k |x w| it is off by (3 * 2^-22 + K 2^-24) A + 2^-24 |bias|.
bf16 tensors: products exact, the sums only.  `dz` below.  lse is off by dz plus 2^-22 (exp to 2 ulp, the joins) plus
2^-24 |lse|; loss by twice that.  An element of dL = p - [v = label] is then off by p (2 dz + 2^-21) + 2^-22 (fp32) or 2^-12
(bf16: one plane) of itself, or, where it is small, by half of f16's smallest step.  Held times 2^15 and times a share f <= 1
of the largest factor M that undoes a row's scale (W's rows for dX, dloss times X's for dW), that is 2^-24 / 2 / 2^15 = 2^-40 of
M, and it multiplies a scaled value of at most 2^15, where M 2^15 is at most twice the largest |W| (dX) or |dloss x| (dW): a
term is off by 2^-39 of that largest value, times |g| for dX.  db is summed in fp32 from unrounded elements.  (`floor`.)
dX and dW are sums of such elements times W or X (two planes, or exact; X times dloss is rounded to its planes again,
another 2^-12 for bf16), so they are off by at most (2 dz + 2^-20 [+ 2^-12 or 2 2^-12] + n 2^-24) of the sum of magnitudes, n the number of terms; bf16 results by half a step, 2^-8,
more."""
import ctypes

import pytest
import torch

F32, BF16 = torch.float32, torch.bfloat16


def make(B, K, V, kind, bias, left_out, seed, scale=2.0):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=gen, device="cuda")
    X, W = r(B, K).to(kind), (r(V, K) * scale / K ** 0.5).to(kind)
    b = r(V) * 0.5 if bias else None
    labels = torch.randint(0, V, (B,), generator=gen, device="cuda", dtype=torch.int32)
    if left_out:
        labels[torch.rand(B, generator=gen, device="cuda") < left_out] = -1
    return X, W, b, labels


def exact(X, W, b, labels, g):
    """(loss, lse, dX, dW, db, dz, |g dL| |W|, |g dL|^T |X|, sum |g dL|) in 64 bits; g [B] with rows left out zero."""
    X, W = X.double(), W.double()
    V = W.shape[0]
    z = X @ W.t()
    mag = (X.abs() @ W.t().abs()).max().item()
    if b is not None:
        z = z + b.double()
    live = (labels >= 0) & (labels < V)
    at = labels.long().clamp(0, V - 1)[:, None]
    lse = torch.logsumexp(z, 1)
    loss = torch.where(live, lse - z.gather(1, at)[:, 0], 0.0)
    d = (z - lse[:, None]).exp()
    d.scatter_add_(1, at, torch.full_like(lse[:, None], -1.0))
    d = torch.where(live[:, None], d * g.double()[:, None], 0.0)
    a = d.abs()
    bias_mag = 0.0 if b is None else b.abs().max().item()
    ga = torch.where(live, g.double().abs(), 0.0)
    xg = torch.where(live, ga * X.abs().amax(1), 0.0).max()
    floor = [2.0 ** -39 * t for t in (ga[:, None] * W.abs().max() * W.shape[0], X.shape[0] * xg, ga.sum())]
    return loss, lse, d @ W, d.t() @ X, d.sum(0), (mag, bias_mag), a @ W.abs(), a.t() @ X.abs(), a.sum(0), floor


def dz_of(kind, K, mags):
    return ((3 * 2.0 ** -22 if kind == F32 else 0.0) + K * 2.0 ** -24) * mags[0] + 2.0 ** -24 * mags[1]


def within(got, exp, tol, what):
    got = got.double()
    assert torch.isfinite(got).all(), what
    err = (got - exp).abs()
    assert (err <= tol).all(), "%s: off by %.3g where %.3g is allowed" % (what, err.max(), (tol if torch.is_tensor(tol) else torch.tensor(tol)).max())


def check(dl, B, K, V, kind, bias=True, left_out=0.0, dloss=False, seed=0, parts=("dX", "dW", "db")):
    X, W, b, labels = make(B, K, V, kind, bias, left_out, seed + B * 7 + K * 3 + V)
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dl_rows = torch.randn(B, generator=gen, device="cuda") if dloss else None
    scale = 0.37
    g = torch.full((B,), scale, device="cuda") * (dl_rows if dloss else 1.0)
    loss, lse = dl.vocab_ce_fwd(X, W, labels, bias=b)
    eloss, else_, edX, edW, edb, mags, mX, mW, mb, floor = exact(X, W, b, labels, g)
    dz = dz_of(kind, K, mags)
    top = else_.abs().max().item()
    within(lse, else_, dz + 2.0 ** -22 + 2.0 ** -24 * top, "lse")
    within(loss, eloss, 2 * dz + 2.0 ** -22 + 2.0 ** -23 * (top + mags[0]), "loss")
    assert (loss[labels < 0] == 0).all()
    dX, dW, db = dl.vocab_ce_bwd(X, W, labels, lse, bias=b, dloss=dl_rows, scale=scale)
    rel = 2 * dz + 2.0 ** -20 + (2.0 ** -12 if kind == BF16 else 0.0)
    half = 2.0 ** -8 if kind == BF16 else 0.0
    within(dX, edX, (rel + V * 2.0 ** -24) * mX + half * edX.abs() + floor[0], "dX")
    again = 2.0 ** -12 if kind == BF16 and dloss else 0.0
    within(dW, edW, (rel + again + B * 2.0 ** -24) * mW + half * edW.abs() + floor[1], "dW")
    assert (dX[labels < 0] == 0).all()
    if bias:
        within(db, edb, (2 * dz + 2.0 ** -20 + B * 2.0 ** -24) * mb + floor[2], "db")
    else:
        assert db is None


@pytest.mark.gpu
@pytest.mark.parametrize("kind", [F32, BF16])
@pytest.mark.parametrize("B,K,V", [(1, 1, 1), (1, 1, 2), (2, 3, 5), (1, 64, 1000), (4, 65, 63), (7, 100, 1031), (33, 17, 129), (64, 128, 4096),
                                   (65, 96, 300), (100, 1000, 2000), (129, 31, 127), (513, 70, 515), (600, 257, 1030), (1025, 64, 2049)])
def test_sizes(dl, B, K, V, kind):
    check(dl, B, K, V, kind)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", [F32, BF16])
@pytest.mark.parametrize("bias", [False, True])
@pytest.mark.parametrize("dloss", [False, True])
def test_rows_left_out_and_weights(dl, kind, bias, dloss):
    check(dl, 90, 50, 700, kind, bias=bias, left_out=0.4, dloss=dloss)
    check(dl, 700, 130, 1500, kind, bias=bias, left_out=0.4, dloss=dloss)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", [F32, BF16])
def test_several_pieces(dl, kind):
    """More classes than one piece holds (about 1024 tiles): the last piece is shorter."""
    check(dl, 40, 64, 70001, kind)
    check(dl, 2000, 40, 33333, kind, left_out=0.1)


@pytest.mark.gpu
def test_all_rows_left_out(dl):
    X, W, b, labels = make(20, 30, 400, F32, True, 0.0, 1)
    for bad in (-1, -(2 ** 31), 400, 2 ** 31 - 1):
        labels.fill_(bad)
        loss, lse = dl.vocab_ce_fwd(X, W, labels, bias=b)
        assert (loss == 0).all() and torch.isfinite(lse).all()
        dX, dW, db = dl.vocab_ce_bwd(X, W, labels, lse, bias=b)
        assert (dX == 0).all() and (dW == 0).all() and (db == 0).all()


@pytest.mark.gpu
@pytest.mark.parametrize("kind", [F32, BF16])
def test_garbage_in_rows_left_out(dl, kind):
    """A padding row full of NaN, infinities or huge values changes nothing but its own lse."""
    X, W, b, labels = make(90, 50, 700, kind, True, 0.0, 3)
    labels[10] = labels[70] = -1
    loss, lse = dl.vocab_ce_fwd(X, W, labels, bias=b)
    dX, dW, db = dl.vocab_ce_bwd(X, W, labels, lse, bias=b)
    keep = [i for i in range(90) if i not in (10, 70)]
    for bad in (float("nan"), float("inf"), 1e30):
        X2 = X.clone()
        X2[10] = bad
        X2[70, ::2] = -bad
        loss2, lse2 = dl.vocab_ce_fwd(X2, W, labels, bias=b)
        assert torch.equal(loss, loss2) and torch.equal(lse[keep], lse2[keep])
        dX2, dW2, db2 = dl.vocab_ce_bwd(X2, W, labels, lse2, bias=b)
        assert torch.equal(dX, dX2) and torch.equal(dW, dW2) and torch.equal(db, db2)


@pytest.mark.gpu
def test_masked_classes_and_far_rows(dl):
    """Classes switched off by a bias of -infinity or the lowest float; rows and classes of very different magnitudes."""
    X, W, b, labels = make(50, 40, 300, F32, True, 0.0, 4)
    labels %= 100
    for off in (float("-inf"), torch.finfo(F32).min):
        b2 = b.clone()
        b2[100:] = off
        loss, lse = dl.vocab_ce_fwd(X, W, labels, bias=b2)
        l1, s1 = dl.vocab_ce_fwd(X, W[:100].contiguous(), labels, bias=b[:100].contiguous())
        assert (lse - s1).abs().max() < 1e-4 and (loss - l1).abs().max() < 1e-4
        dX, dW, db = dl.vocab_ce_bwd(X, W, labels, lse, bias=b2)
        assert (dW[100:] == 0).all() and (db[100:] == 0).all() and torch.isfinite(dX).all() and torch.isfinite(dW).all()
    X[3] *= 1e-12
    X[4] *= 1e12
    W[7] *= 1e-9
    loss, lse = dl.vocab_ce_fwd(X, W, labels)
    e = exact(X, W, None, labels, torch.ones(50, device="cuda"))
    rest = [i for i in range(50) if i != 4]
    mag = (X.double().abs() @ W.double().t().abs()).max(1).values
    tol = 2 * ((3 * 2.0 ** -22 + 40 * 2.0 ** -24) * mag) + 2.0 ** -22 + 2.0 ** -23 * (mag + e[1].abs())
    assert ((loss.double() - e[0]).abs() <= tol).all() and ((lse.double() - e[1]).abs() <= tol).all() and rest


@pytest.mark.gpu
def test_weights_that_underflow(dl):
    """A row whose dloss X is below every fp32 value counts nothing, and costs the others nothing."""
    X, W, b, labels = make(70, 48, 300, F32, True, 0.0, 23)
    X[9] *= 1e-30
    g = torch.ones(70, device="cuda")
    g[9] = 1e-25
    eloss, else_, edX, edW, edb, mags, mX, mW, mb, floor = exact(X, W, b, labels, g)
    loss, lse = dl.vocab_ce_fwd(X, W, labels, bias=b)
    dX, dW, db = dl.vocab_ce_bwd(X, W, labels, lse, bias=b, dloss=g)
    rel = 2 * dz_of(F32, 48, mags) + 2.0 ** -20
    within(dW, edW, (rel + 70 * 2.0 ** -24) * mW + floor[1], "dW")
    within(dX, edX, (rel + 300 * 2.0 ** -24) * mX + floor[0], "dX")


@pytest.mark.gpu
@pytest.mark.parametrize("kind", [F32, BF16])
def test_rows_of_zeros(dl, kind):
    """Rows of X and of W that are zero, or all of X or W: they scale nobody's planes."""
    for what in ("some", "X", "W"):
        X, W, b, labels = make(90, 70, 600, kind, True, 0.1, 21)
        if what == "some":
            X[5] = X[6] = W[3] = W[500] = 0
        else:
            {"X": X, "W": W}[what].zero_()
        loss, lse = dl.vocab_ce_fwd(X, W, labels, bias=b)
        g = torch.full((90,), 0.25, device="cuda")
        eloss, else_, edX, edW, edb, mags, mX, mW, mb, floor = exact(X, W, b, labels, g)
        dz = dz_of(kind, 70, mags)
        within(lse, else_, dz + 2.0 ** -22 + 2.0 ** -24 * else_.abs().max().item(), "lse")
        dX, dW, db = dl.vocab_ce_bwd(X, W, labels, lse, bias=b, scale=0.25)
        rel = 2 * dz + 2.0 ** -20 + (2.0 ** -12 if kind == BF16 else 0.0)
        half = 2.0 ** -8 if kind == BF16 else 0.0
        within(dX, edX, (rel + 600 * 2.0 ** -24) * mX + half * edX.abs() + floor[0], "dX")
        within(dW, edW, (rel + 90 * 2.0 ** -24) * mW + half * edW.abs() + floor[1], "dW")
        within(db, edb, (2 * dz + 2.0 ** -20 + 90 * 2.0 ** -24) * mb + floor[2], "db")


@pytest.mark.gpu
def test_nonfinite_rows_stay_alone_forward(dl):
    X, W, b, labels = make(80, 33, 500, F32, False, 0.0, 5)
    loss, lse = dl.vocab_ce_fwd(X, W, labels)
    X2 = X.clone()
    X2[5, 1] = float("nan")
    loss2, lse2 = dl.vocab_ce_fwd(X2, W, labels)
    keep = [i for i in range(80) if i != 5]
    assert torch.equal(loss[keep], loss2[keep]) and torch.equal(lse[keep], lse2[keep]) and torch.isnan(loss2[5]) and torch.isnan(lse2[5])


@pytest.mark.gpu
@pytest.mark.parametrize("kind", [F32, BF16])
def test_accumulate_parts_and_repeat(dl, pkg, kind):
    X, W, b, labels = make(130, 70, 900, kind, True, 0.2, 6)
    loss, lse = dl.vocab_ce_fwd(X, W, labels, bias=b)
    dX, dW, db = dl.vocab_ce_bwd(X, W, labels, lse, bias=b, scale=0.5)
    again = dl.vocab_ce_bwd(X, W, labels, lse, bias=b, scale=0.5)
    assert all(torch.equal(x, y) for x, y in zip((dX, dW, db), again))
    w0, b0 = torch.randn_like(W), torch.randn_like(b)
    acc = dl.vocab_ce_bwd(X, W, labels, lse, bias=b, scale=0.5, dW=w0.clone(), db=b0.clone(), accumulate=True)
    assert torch.equal(acc[0], dX) and torch.equal(acc[2], b0 + db)
    one = 2.0 ** -8 if kind == BF16 else 2.0 ** -24     # the sum is rounded once more; dW itself once less
    assert ((acc[1].double() - w0.double() - dW.double()).abs() <= one * (acc[1].double().abs() + 2 * dW.double().abs())).all()
    # one gradient at a time, through the C entry point
    sz, p = ctypes.c_size_t, lambda t: ctypes.c_void_p(t.data_ptr())
    for only in range(3):
        out = [torch.full_like(t, 9.0) for t in (dX, dW, db)]
        ptr = [p(t) if i == only else None for i, t in enumerate(out)]
        code = {F32: 0, BF16: 1}[kind]
        assert dl.lib.dlmi_vocab_ce_bwd(dl.ctx, code, sz(130), sz(70), sz(900), p(X), p(W), p(b), p(labels), p(lse), None,
                                        ctypes.c_float(0.5), *ptr, 0) == 0
        for i, (t, e) in enumerate(zip(out, (dX, dW, db))):
            assert torch.equal(t, e) if i == only else (t == 9.0).all()


@pytest.mark.gpu
def test_unaligned_operands(dl):
    """X, W and the gradients at odd element offsets of packed arrays: nothing beside them is touched."""
    for kind in (F32, BF16):
        B, K, V = 37, 45, 333
        X, W, b, labels = make(B, K, V, kind, True, 0.1, 8)
        loss, lse = dl.vocab_ce_fwd(X, W, labels, bias=b)
        dX, dW, db = dl.vocab_ce_bwd(X, W, labels, lse, bias=b)
        def at_odd(t):
            buf = torch.full((t.numel() + 8,), 3.0, dtype=t.dtype, device="cuda")
            v = buf[1:1 + t.numel()].view(t.shape)
            v.copy_(t)
            return buf, v
        (_, X1), (_, W1), (_, b1) = at_odd(X), at_odd(W), at_odd(b)
        outs = [at_odd(t) for t in (dX, dW, db)]
        l1, s1 = dl.vocab_ce_fwd(X1, W1, labels, bias=b1)
        dl.vocab_ce_bwd(X1, W1, labels, s1, bias=b1, dX=outs[0][1], dW=outs[1][1], db=outs[2][1])
        assert torch.equal(l1, loss) and torch.equal(s1, lse)
        for (buf, v), e in zip(outs, (dX, dW, db)):
            assert torch.equal(v, e) and buf[0] == 3.0 and (buf[1 + e.numel():] == 3.0).all()


@pytest.mark.gpu
def test_against_differences(dl):
    """dX and dW along a random direction against central differences of the forward in fp32.  Step 2^-6: a third of its
    square times a third derivative of the order of the direction's cubed logits, below 1e-2 of the derivative's scale, and
    loss roundings of 2^-21 over 2^-6 = 3e-5 per row."""
    B, K, V = 40, 24, 90
    X, W, b, labels = make(B, K, V, F32, True, 0.1, 9)
    gen = torch.Generator(device="cuda").manual_seed(2)
    dx, dw = torch.randn(B, K, generator=gen, device="cuda"), torch.randn(V, K, generator=gen, device="cuda") / K ** 0.5
    s = 2.0 ** -6
    f = lambda t: dl.vocab_ce_fwd(X + t * dx, W + t * dw, labels, bias=b)[0].double().sum()
    # the fourth-order combination of two steps: truncation of the order of the step to the fourth
    diff = (8 * (f(s) - f(-s)) - (f(2 * s) - f(-2 * s))) / (12 * s)
    loss, lse = dl.vocab_ce_fwd(X, W, labels, bias=b)
    dX, dW, _ = dl.vocab_ce_bwd(X, W, labels, lse, bias=b)
    along = (dX.double() * dx.double()).sum() + (dW.double() * dw.double()).sum()
    assert abs(diff - along) <= B * 3 * 3e-5 + 1e-3 * abs(along)


@pytest.mark.gpu
def test_captured_and_replayed(pkg):
    d = pkg.Dlmi(0)
    try:
        stream = torch.cuda.Stream()
        d.set_stream(stream)
        X, W, b, labels = make(70, 64, 800, BF16, True, 0.2, 12)
        Xs = [torch.randn_like(X) for _ in range(4)]
        out = dict(loss=torch.empty(70, device="cuda"), lse=torch.empty(70, device="cuda"))
        grads = dict(dX=torch.empty_like(X), dW=torch.empty_like(W), db=torch.empty_like(b))
        torch.cuda.synchronize()
        def step(x, o, g):
            d.vocab_ce_fwd(x, W, labels, bias=b, **o)
            d.vocab_ce_bwd(x, W, labels, o["lse"], bias=b, scale=0.1, **g)
        with torch.cuda.stream(stream):
            eo, eg = {k: v.clone() for k, v in out.items()}, {k: v.clone() for k, v in grads.items()}
            step(X, eo, eg)
            stream.synchronize()
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=stream):
                step(X, out, grads)
            for x in Xs:
                X.copy_(x)
                step(x, eo, eg)
                graph.replay()
                stream.synchronize()
                assert all(torch.equal(out[k], eo[k]) for k in out) and all(torch.equal(grads[k], eg[k]) for k in grads)
    finally:
        torch.cuda.synchronize()
        d.close()


@pytest.mark.gpu
def test_refusals(dl, pkg):
    X, W, b, labels = make(8, 16, 40, F32, True, 0.0, 1)
    loss, lse = dl.vocab_ce_fwd(X, W, labels, bias=b)
    with pytest.raises(AssertionError):
        dl.vocab_ce_fwd(X, W, labels.long())
    with pytest.raises(AssertionError):
        dl.vocab_ce_fwd(X, W.bfloat16(), labels)
    with pytest.raises(AssertionError):
        dl.vocab_ce_fwd(X, W[:, :8], labels)
    with pytest.raises(AssertionError):
        dl.vocab_ce_fwd(X.half(), W.half(), labels)
    with pytest.raises(AssertionError):
        dl.vocab_ce_fwd(X, W, labels[:4])
    with pytest.raises(AssertionError):
        dl.vocab_ce_bwd(X, W, labels, lse, bias=b, accumulate=True)
    with pytest.raises(pkg.DlmiError, match="written over"):
        dl.vocab_ce_bwd(X, W, labels, lse, dX=X)
    both = torch.zeros(8 * 16 + 40 * 16, device="cuda")
    for over in (dict(dX=both[:128].view(8, 16), dW=both[120:760].view(40, 16)), dict(dW=W), dict(dX=lse.new_zeros(8, 16), dW=W),
                 dict(db=b), dict(db=W.flatten()[:40])):
        with pytest.raises(pkg.DlmiError, match="written over"):
            dl.vocab_ce_bwd(X, W, labels, lse, bias=b, **over)
    with pytest.raises(pkg.DlmiError, match="written over"):
        dl.vocab_ce_fwd(X, W, labels, bias=b, loss=loss, lse=loss)
    with pytest.raises(pkg.DlmiError, match="written over"):
        dl.vocab_ce_fwd(X, W, labels, bias=b, loss=loss, lse=X.flatten()[4:12])
    sz, p = ctypes.c_size_t, lambda t: ctypes.c_void_p(t.data_ptr())
    lib = dl.lib
    f = lib.dlmi_vocab_ce_fwd
    assert f(None, 0, sz(8), sz(16), sz(40), p(X), p(W), None, p(labels), p(loss), p(lse)) == -1
    assert f(dl.ctx, 9, sz(8), sz(16), sz(40), p(X), p(W), None, p(labels), p(loss), p(lse)) == -1
    assert f(dl.ctx, 0, sz(8), sz(0), sz(40), p(X), p(W), None, p(labels), p(loss), p(lse)) == -1
    assert f(dl.ctx, 0, sz(8), sz(16), sz(0), p(X), p(W), None, p(labels), p(loss), p(lse)) == -1
    assert f(dl.ctx, 0, sz(8), sz(16), sz(40), p(X), p(W), None, None, p(loss), p(lse)) == -1
    assert f(dl.ctx, 0, sz(1 << 20), sz(16), sz(40), p(X), p(W), None, p(labels), p(loss), p(lse)) == -1
    assert f(dl.ctx, 0, sz(0), sz(16), sz(40), None, None, None, None, None, None) == 0
    g = lib.dlmi_vocab_ce_bwd
    assert g(dl.ctx, 0, sz(8), sz(16), sz(40), p(X), p(W), None, p(labels), p(lse), None, ctypes.c_float(1), None, None, None, 0) == -1
    assert g(dl.ctx, 0, sz(0), sz(16), sz(40), p(X), p(W), None, p(labels), p(lse), None, ctypes.c_float(1), p(X.clone()), None, None, 0) == -1
    assert g(dl.ctx, 0, sz(8), sz(16), sz(40), p(X), p(W), None, p(labels), None, None, ctypes.c_float(1), p(X.clone()), None, None, 0) == -1
