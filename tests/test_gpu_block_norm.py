"""dlmi_block_norm_fwd / _bwd against the formula in 64 bits and its gradient by automatic differentiation.

Tolerances (fp32).  A sum over a row runs through at most 16 additions in a thread, 6 in a wavefront and 16 over
wavefronts: 38 roundings of at most the sum of magnitudes; a mean, the centring, the squares, the root and the quotient add
less than 16, the weights, gate and sums to the result another 10: 64 roundings, 64 * 2^-24, of the largest magnitude that
enters an element.  `LOOSE` = 8 stands for how much larger than the result those magnitudes can be here (a mean as large as
twice the deviation enters the centring; the gradient subtracts two projections from a term of the size of all of them).
The gradients' sums over B rows add B roundings of the sum of magnitudes.  bf16 results are off by half a step more: 2^-8."""
import pytest
import torch

U = 2.0 ** -24
LOOSE = 8
F32, BF16 = torch.float32, torch.bfloat16


def reference(c, t, post, pre, act, gate_rows, rs, bs):
    """(y, h) in 64 bits; t: dict of leaves."""
    def norm(v, how, w, b):
        if how == "NONE":
            return v
        if how == "LAYER":
            v = v - v.mean(1, keepdim=True)
        v = v / torch.sqrt((v * v).mean(1, keepdim=True) + 1e-5)
        v = v if w is None else v * w
        return v if b is None else v + b
    n = norm(t["u"], post, t["w_post"], t["b_post"])
    if gate_rows:
        g = t["gate"].repeat_interleave(gate_rows, 0)[:n.shape[0]]
        n = n * {"LINEAR": lambda v: v, "SIGMOID": torch.sigmoid, "TANH": torch.tanh}[act](g)
    y = rs * t["x"] + bs * n
    return y, (lambda v: norm(v, pre, t["w_pre"], t["b_pre"]))


def make(B, H, kind, post, pre, gate_rows, weights, biases, seed):
    gen = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=gen)
    t = dict(x=r(B, H) * 1.5, u=r(B, H) * 0.7 + 0.5, gate=r(-(-B // gate_rows), H) if gate_rows else None)
    t = {k: v if v is None else v.to(kind) for k, v in t.items()}
    for k, on in (("w_post", post), ("b_post", post), ("w_pre", pre), ("b_pre", pre)):
        want = on != "NONE" and (weights if k[0] == "w" else biases)
        t[k] = (1 + 0.3 * r(H) if k[0] == "w" else 0.2 * r(H)) if want else None
    t["dy"], t["dh"] = r(B, H).to(kind), r(B, H).to(kind)
    return t


def dev(t):
    return {k: None if v is None else v.cuda() for k, v in t.items()}


def check(got, exp, what, roundings=64, scale=None):
    got, exp = got.cpu(), exp.detach()
    assert got.shape == exp.shape, what
    m = max(scale or 0.0, exp.abs().max().item())
    tol = LOOSE * roundings * U * m + (2.0 ** -8 * exp.abs() if got.dtype == BF16 else 0.0)
    err = (got.double() - exp).abs()
    assert (err <= tol).all(), "%s: off by %.3g where %.3g is allowed" % (what, err.max(), torch.as_tensor(tol).max())


def run(dl, pkg, B, H, kind, post, pre, gate_rows=0, act="LINEAR", weights=True, biases=True, rs=1.0, bs=1.0, no_dy=False,
        no_dh=False):
    t = make(B, H, kind, post, pre, gate_rows, weights, biases, B * 131 + H)
    d = dev(t)
    desc = pkg.Dlmi.block_norm_desc(post=pkg.ROW_NORM[post], pre=pkg.ROW_NORM[pre], gate_act=pkg.GATE_ACT[act],
                                    gate_rows=gate_rows, residual_scale=rs, branch_scale=bs)
    params = {k: d[k] for k in ("w_post", "b_post", "w_pre", "b_pre")}
    y, h = dl.block_norm_fwd(desc, d["x"], d["u"], gate=d["gate"], **params)
    leaf = {k: None if v is None else v.double().requires_grad_(True) for k, v in t.items()}
    ey, pre_of = reference(None, leaf, post, pre, act, gate_rows, rs, bs)
    check(y, ey, "y")
    check(h, pre_of(ey), "h")
    # the gradient at the y that is stored
    g = dl.block_norm_bwd(desc, d["u"], y, None if no_dy else d["dy"], None if no_dh else d["dh"], gate=d["gate"], **params)
    at = y.cpu().double().requires_grad_(True)
    back = torch.zeros_like(ey)
    if not no_dh:
        pre_of(at).backward(t["dh"].double())
        back = back + at.grad
    if not no_dy:
        back = back + t["dy"].double()
    ey.backward(back)
    # y enters through its own rounding only: in bf16 the reference is taken at the same stored y
    big = max(1.0, back.abs().max().item())
    check(g["dx"], leaf["x"].grad, "dx", scale=big)
    check(g["du"], leaf["u"].grad, "du", scale=big * (1 + abs(bs)))
    if gate_rows:
        shared = min(gate_rows, B)
        check(g["dgate"], leaf["gate"].grad, "dgate", roundings=64 + shared, scale=shared ** 0.5 * big * 4)
    else:
        assert g["dgate"] is None
    for k in ("w_post", "b_post", "w_pre", "b_pre"):
        if t[k] is None:
            assert g["d" + k] is None
            continue
        exp = leaf[k].grad if leaf[k].grad is not None else torch.zeros(H, dtype=torch.float64)
        check(g["d" + k], exp, "d" + k, roundings=64 + B, scale=B ** 0.5 * big * 4)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", [F32, BF16])
@pytest.mark.parametrize("B,H", [(1, 1), (1, 2), (3, 7), (2, 64), (5, 65), (130, 200), (17, 511), (9, 513), (33, 777), (6, 1024),
                                 (7, 2047), (3, 4096), (3, 5000), (2, 8192), (2, 9001), (2, 16384)])
def test_sizes(dl, pkg, B, H, kind):
    run(dl, pkg, B, H, kind, "LAYER", "RMS", gate_rows=1, act="SIGMOID", bs=0.5)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", [F32, BF16])
@pytest.mark.parametrize("post", ["NONE", "RMS", "LAYER"])
@pytest.mark.parametrize("pre", ["NONE", "RMS", "LAYER"])
def test_norms(dl, pkg, post, pre, kind):
    run(dl, pkg, 37, 300, kind, post, pre, gate_rows=1, act="TANH", rs=0.75)
    run(dl, pkg, 37, 300, kind, post, pre, weights=False)
    run(dl, pkg, 12, 96, kind, post, pre, biases=False, no_dy=True)
    run(dl, pkg, 12, 96, kind, post, pre, biases=False, no_dh=True)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", [F32, BF16])
@pytest.mark.parametrize("B,gate_rows", [(40, 2), (41, 3), (41, 50), (41, 41), (1000, 1000), (1000, 70), (1, 5), (3000, 7), (9000, 9)])
def test_gate_shared_by_rows(dl, pkg, B, gate_rows, kind):
    run(dl, pkg, B, 72, kind, "RMS", "LAYER", gate_rows=gate_rows, act="LINEAR", bs=0.5)


@pytest.mark.gpu
def test_many_rows_take_several_each(dl, pkg):
    run(dl, pkg, 20000, 66, F32, "RMS", "RMS", gate_rows=20000, act="SIGMOID")
    run(dl, pkg, 2100, 1030, F32, "LAYER", "LAYER", gate_rows=0)


@pytest.mark.gpu
def test_accumulate_alias_and_repeat(dl, pkg):
    """accumulate adds to what is there; dx may be dy, du dh, y x, h u; the same call gives the same bits."""
    t = dev(make(50, 130, F32, "RMS", "LAYER", 4, True, True, 1))
    desc = pkg.Dlmi.block_norm_desc(post=1, pre=2, gate_rows=4)
    params = {k: t[k] for k in ("w_post", "b_post", "w_pre", "b_pre")}
    y, h = dl.block_norm_fwd(desc, t["x"], t["u"], gate=t["gate"], **params)
    x2, u2 = t["x"].clone(), t["u"].clone()
    y2, h2 = dl.block_norm_fwd(desc, x2, u2, gate=t["gate"], y=x2, h=u2, **params)
    assert torch.equal(y, y2) and torch.equal(h, h2) and y2.data_ptr() == x2.data_ptr()
    a = dl.block_norm_bwd(desc, t["u"], y, t["dy"], t["dh"], gate=t["gate"], **params)
    dy2, dh2 = t["dy"].clone(), t["dh"].clone()
    start = {k: torch.randn(130, device="cuda") for k in ("dw_post", "db_post", "dw_pre", "db_pre")}
    b = dl.block_norm_bwd(desc, t["u"], y, dy2, dh2, gate=t["gate"], dx=dy2, du=dh2, grads={k: v.clone() for k, v in start.items()},
                          accumulate=True, **params)
    assert torch.equal(a["dx"], b["dx"]) and torch.equal(a["du"], b["du"]) and torch.equal(a["dgate"], b["dgate"])
    for k, v in start.items():
        assert torch.equal(v + a[k], b[k]), k


@pytest.mark.gpu
def test_unaligned_rows(dl, pkg):
    """Tensors at odd element offsets of a larger buffer, rows of an odd length: nothing outside is touched."""
    for kind in (F32, BF16):
        B, H = 6, 77
        t = make(B, H, kind, "RMS", "RMS", 0, False, False, 3)
        buf = {k: torch.full((B * H + 9,), 7.0, dtype=kind, device="cuda") for k in ("x", "u", "y", "h")}
        v = {k: b[1:1 + B * H].view(B, H) for k, b in buf.items()}
        v["x"].copy_(t["x"])
        v["u"].copy_(t["u"])
        desc = pkg.Dlmi.block_norm_desc(post=1, pre=1)
        dl.block_norm_fwd(desc, v["x"], v["u"], y=v["y"], h=v["h"])
        y, h = dl.block_norm_fwd(desc, t["x"].cuda(), t["u"].cuda())
        assert torch.equal(v["y"], y) and torch.equal(v["h"], h)
        for k, b in buf.items():
            assert (b[:1] == 7).all() and (b[1 + B * H:] == 7).all(), k


@pytest.mark.gpu
def test_against_differences(dl, pkg):
    """The gradient along a random direction against central differences of the forward.  With step s the differences are
    off by s^2 times a third derivative (of the order of the loss's own size, 1 per row here) and by the roundings of y and
    h, 64 * 2^-24 * |y| each, over s: for s = 2^-7 1e-4 and 64 * 6e-8 * 4 * 128 = 2e-3 of a term, and the terms of a random
    direction add like sqrt(n)."""
    B, H = 16, 64
    t = make(B, H, F32, "LAYER", "RMS", 4, True, True, 8)
    desc = pkg.Dlmi.block_norm_desc(post=2, pre=1, gate_act=pkg.GATE_ACT["SIGMOID"], gate_rows=4, branch_scale=0.5)
    names = ("x", "u", "gate", "w_post", "b_post", "w_pre", "b_pre")
    gen = torch.Generator().manual_seed(1)
    v = {k: torch.randn(t[k].shape, generator=gen) for k in names}
    def loss(s):
        d = {k: (t[k].double() + s * v[k].double()).float().cuda() for k in names}
        y, h = dl.block_norm_fwd(desc, **d)
        return (y.double().cpu() * t["dy"].double()).sum() + (h.double().cpu() * t["dh"].double()).sum()
    s = 2.0 ** -7
    diff = (loss(s) - loss(-s)) / (2 * s)
    d = dev(t)
    y, _ = dl.block_norm_fwd(desc, **{k: d[k] for k in names})
    g = dl.block_norm_bwd(desc, d["u"], y, d["dy"], d["dh"], **{k: d[k] for k in names[2:]})
    grads = dict(x="dx", u="du", gate="dgate", w_post="dw_post", b_post="db_post", w_pre="dw_pre", b_pre="db_pre")
    along = sum((g[o].cpu().double() * v[k].double()).sum() for k, o in grads.items())
    assert abs(diff - along) <= 3e-3 * (B * H) ** 0.5


@pytest.mark.gpu
def test_nonfinite_rows_stay_alone(dl, pkg):
    t = dev(make(8, 100, F32, "RMS", "LAYER", 1, True, True, 5))
    desc = pkg.Dlmi.block_norm_desc(post=1, pre=2, gate_rows=1)
    params = {k: t[k] for k in ("w_post", "b_post", "w_pre", "b_pre")}
    y, h = dl.block_norm_fwd(desc, t["x"], t["u"], gate=t["gate"], **params)
    t["u"][3, 50] = float("nan")
    t["x"][5, 0] = float("inf")
    y2, h2 = dl.block_norm_fwd(desc, t["x"], t["u"], gate=t["gate"], **params)
    keep = [0, 1, 2, 4, 6, 7]
    assert torch.equal(y[keep], y2[keep]) and torch.equal(h[keep], h2[keep])
    assert torch.isnan(y2[3]).all() and torch.isinf(y2[5, 0]) and not torch.isfinite(h2[5]).any()


@pytest.mark.gpu
def test_captured_and_replayed(pkg):
    """Forward and backward recorded into a HIP graph and replayed with eager work between: the eager bits every time."""
    d = pkg.Dlmi(0)
    try:
        stream = torch.cuda.Stream()
        d.set_stream(stream)
        t = dev(make(60, 300, BF16, "RMS", "LAYER", 7, True, True, 2))
        desc = pkg.Dlmi.block_norm_desc(post=1, pre=2, gate_rows=7, gate_act=pkg.GATE_ACT["TANH"])
        params = {k: t[k] for k in ("w_post", "b_post", "w_pre", "b_pre")}
        new = lambda: (dict(y=torch.empty_like(t["x"]), h=torch.empty_like(t["x"])),
                       dict(dx=torch.empty_like(t["x"]), du=torch.empty_like(t["x"]), dgate=torch.empty_like(t["gate"]),
                            grads={k: torch.empty(300, device="cuda") for k in ("dw_post", "db_post", "dw_pre", "db_pre")}))
        xs = [torch.randn_like(t["x"]) for _ in range(4)]
        def step(x, o, g):
            d.block_norm_fwd(desc, x, t["u"], gate=t["gate"], **params, **o)
            d.block_norm_bwd(desc, t["u"], o["y"], t["dy"], t["dh"], gate=t["gate"], **params, **g)
        flat = lambda o, g: list(o.values()) + [g["dx"], g["du"], g["dgate"]] + list(g["grads"].values())
        (eo, eg), (go, gg), x = new(), new(), t["x"].clone()
        torch.cuda.synchronize()
        with torch.cuda.stream(stream):
            step(x, eo, eg)
            stream.synchronize()
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=stream):
                step(x, go, gg)
            for v in xs:
                x.copy_(v)
                step(v, eo, eg)
                graph.replay()
                stream.synchronize()
                assert all(torch.equal(p, q) for p, q in zip(flat(eo, eg), flat(go, gg)))
    finally:
        torch.cuda.synchronize()
        d.close()


@pytest.mark.gpu
@pytest.mark.parametrize("kind", [F32, BF16])
@pytest.mark.parametrize("H", [5, 130])
def test_outputs_over_inputs(dl, pkg, kind, H):
    """What the documentation lets an output be: the bits are those of separate outputs."""
    t = dev(make(37, H, kind, "RMS", "LAYER", 5, True, True, 3))
    desc = pkg.Dlmi.block_norm_desc(post=1, pre=2, gate_rows=5, gate_act=pkg.GATE_ACT["SIGMOID"])
    params = {k: t[k] for k in ("w_post", "b_post", "w_pre", "b_pre")}
    y, h = dl.block_norm_fwd(desc, t["x"], t["u"], gate=t["gate"], **params)
    for names in (("x", "u"), ("u", "x")):
        x, u = t["x"].clone(), t["u"].clone()
        o = dict(x=x, u=u)
        dl.block_norm_fwd(desc, x, u, gate=t["gate"], y=o[names[0]], h=o[names[1]], **params)
        assert torch.equal(o[names[0]], y) and torch.equal(o[names[1]], h)
    g = dl.block_norm_bwd(desc, t["u"], y, t["dy"], t["dh"], gate=t["gate"], **params)
    for names in (("dy", "dh"), ("dh", "dy"), ("u", "y")):
        o = dict(u=t["u"].clone(), y=y.clone(), dy=t["dy"].clone(), dh=t["dh"].clone())
        r = dl.block_norm_bwd(desc, o["u"], o["y"], o["dy"], o["dh"], gate=t["gate"], dx=o[names[0]], du=o[names[1]], **params)
        assert all(torch.equal(r[k], g[k]) for k in g)


@pytest.mark.gpu
def test_a_gate_for_all_and_no_rows(dl, pkg):
    """gate_rows beyond B: one row of the gate for all.  B = 0: the parameters' gradients are 0, or stay."""
    t = dev(make(9, 64, F32, "RMS", "RMS", 9, True, False, 2))
    w = dict(w_post=t["w_post"], w_pre=t["w_pre"])
    both = []
    for rows in (9, 2 ** 64 - 1):
        desc = pkg.Dlmi.block_norm_desc(gate_rows=rows)
        y, h = dl.block_norm_fwd(desc, t["x"], t["u"], gate=t["gate"], **w)
        g = dl.block_norm_bwd(desc, t["u"], y, t["dy"], t["dh"], gate=t["gate"], **w)
        both.append([y, h, g["dx"], g["du"], g["dgate"], g["dw_post"], g["dw_pre"]])
    assert all(torch.equal(p, q) for p, q in zip(*both))
    e = torch.empty(0, 64, device="cuda")
    for accumulate, left in ((False, 0.0), (True, 3.0)):
        grads = dict(dw_post=torch.full((64,), 3.0, device="cuda"), dw_pre=torch.full((64,), 3.0, device="cuda"))
        dl.block_norm_bwd(pkg.Dlmi.block_norm_desc(), e, e, e, e, grads=grads, accumulate=accumulate, **w)
        assert bool((grads["dw_post"] == left).all()) and bool((grads["dw_pre"] == left).all())


@pytest.mark.gpu
def test_outputs_belong_to_the_contexts_stream(pkg):
    """A context on a stream that is not the current one: results are right once that stream is waited for."""
    d = pkg.Dlmi(0)
    try:
        stream = torch.cuda.Stream()
        d.set_stream(stream)
        t = dev(make(40, 200, F32, "RMS", "RMS", 0, True, False, 2))
        torch.cuda.synchronize()
        desc = pkg.Dlmi.block_norm_desc()
        y, h = d.block_norm_fwd(desc, t["x"], t["u"], w_post=t["w_post"], w_pre=t["w_pre"])
        g = d.block_norm_bwd(desc, t["u"], y, t["dy"], t["dh"], w_post=t["w_post"], w_pre=t["w_pre"])
        stream.synchronize()
        d.set_stream(torch.cuda.current_stream())
        y2, h2 = d.block_norm_fwd(desc, t["x"], t["u"], w_post=t["w_post"], w_pre=t["w_pre"])
        g2 = d.block_norm_bwd(desc, t["u"], y2, t["dy"], t["dh"], w_post=t["w_post"], w_pre=t["w_pre"])
        torch.cuda.synchronize()
        assert torch.equal(y, y2) and torch.equal(h, h2) and torch.equal(g["dx"], g2["dx"]) and torch.equal(g["dw_pre"], g2["dw_pre"])
    finally:
        torch.cuda.synchronize()
        d.close()


@pytest.mark.gpu
def test_refusals(dl, pkg):
    x = torch.ones(4, 8, device="cuda")
    w = torch.ones(8, device="cuda")
    D = pkg.Dlmi.block_norm_desc
    with pytest.raises(pkg.DlmiError, match="unknown norm"):
        dl.block_norm_fwd(D(post=7), x, x.clone())
    with pytest.raises(pkg.DlmiError, match="gate_rows without"):
        dl.block_norm_fwd(D(gate_rows=1), x, x.clone())
    with pytest.raises(pkg.DlmiError, match="without gate_rows"):
        dl.block_norm_fwd(D(), x, x.clone(), gate=x)
    with pytest.raises(pkg.DlmiError, match="activation"):
        dl.block_norm_fwd(D(gate_act=pkg.ACT["RELU"]), x, x.clone())
    with pytest.raises(pkg.DlmiError, match="without a norm"):
        dl.block_norm_fwd(D(post=0), x, x.clone(), w_post=w)
    with pytest.raises(pkg.DlmiError, match="eps"):
        dl.block_norm_fwd(D(eps_pre=float("nan")), x, x.clone())
    with pytest.raises(pkg.DlmiError, match="no gradient"):
        dl.block_norm_bwd(D(), x, x, None, None)
    with pytest.raises(pkg.DlmiError, match="wider"):
        z = torch.ones(1, 16385, device="cuda")
        dl.block_norm_fwd(D(), z, z.clone())
    with pytest.raises(AssertionError):
        dl.block_norm_fwd(D(), x, x.bfloat16())
    with pytest.raises(AssertionError):
        dl.block_norm_fwd(D(gate_rows=2), x, x.clone(), gate=x)
    with pytest.raises(AssertionError):
        dl.block_norm_fwd(D(), x, x.clone(), w_pre=w.double())
    with pytest.raises(AssertionError):
        dl.block_norm_fwd(D(), x, torch.ones(8, 4, device="cuda").t())
    flat = torch.ones(40, device="cuda")
    a, c = flat[:32].view(4, 8), flat[8:].view(4, 8)
    u = x.clone()
    for over in (dict(y=a, h=a), dict(y=a, h=c)):
        with pytest.raises(pkg.DlmiError, match="overlaps"):
            dl.block_norm_fwd(D(), x, u, **over)
    with pytest.raises(pkg.DlmiError, match="overlaps"):
        dl.block_norm_fwd(D(), a, u, y=c)
    with pytest.raises(pkg.DlmiError, match="overlaps"):
        dl.block_norm_fwd(D(gate_rows=1), x, u, gate=a, h=a)
    with pytest.raises(pkg.DlmiError, match="overlaps"):
        dl.block_norm_fwd(D(), x, u, w_pre=flat[:8], h=a)
    for over in (dict(dx=a, du=a), dict(dx=a, du=c), dict(dx=a, grads=dict(dw_post=flat[:8])), dict(grads=dict(dw_post=w))):
        with pytest.raises(pkg.DlmiError, match="overlaps"):
            dl.block_norm_bwd(D(), u, x, x.clone(), None, w_post=w, **over)
    with pytest.raises(pkg.DlmiError, match="overlaps"):
        dl.block_norm_bwd(D(gate_rows=1), u, x, x.clone(), None, gate=a, dgate=a)
    e = torch.empty(0, 8, device="cuda")
    y, h = dl.block_norm_fwd(D(), e, e.clone())
    assert y.shape == (0, 8)
