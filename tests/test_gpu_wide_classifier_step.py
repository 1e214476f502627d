"""A training step of a wide residual classifier, the operators run together as a program would: a layer, the block's tail
with its norms, the cross entropy over a large vocabulary, all gradients, and the Muon step of both weight matrices.

Against the same step in 64 bits.  Every operator is held to its own tolerance elsewhere; here each adds at most a few
2^-20 of the magnitudes it works on (two-plane and fp32 products of up to 1000 terms, row sums), seven of them in a row, and
the orthogonalization multiplies a relative error of the gradient by at most 3.4445^5 = 485 in its weakest directions: the
loss is held to 1e-5, gradients to 1e-4 of their norm, and the updated weights to lr * (485 * 1e-4) of the update's norm."""
import pytest
import torch

COEFFS = (3.4445, -4.7750, 2.0315)


def orthogonal(G):
    X = G / (G.norm() + 1e-7)
    flip = X.shape[0] > X.shape[1]
    X = X.t() if flip else X
    for _ in range(5):
        A = X @ X.t()
        X = COEFFS[0] * X + (COEFFS[1] * A + COEFFS[2] * A @ A) @ X
    return X.t() if flip else X


def data(B, H, V, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=gen, device="cuda")
    labels = torch.randint(0, V, (B,), generator=gen, device="cuda", dtype=torch.int32)
    labels[::7] = -1
    return dict(x=r(B, H), W=r(H, H) / H ** 0.5, Wo=r(V, H) * 2 / H ** 0.5, bo=r(V) * 0.1, gate=r(1, H), w_post=1 + 0.1 * r(H),
                w_pre=1 + 0.1 * r(H)), labels


def step(dl, pkg, t, labels, mom, lr):
    """One step in place; returns (loss rows, gradients)."""
    B = t["x"].shape[0]
    desc = pkg.Dlmi.block_norm_desc(post=pkg.ROW_NORM["RMS"], pre=pkg.ROW_NORM["LAYER"], gate_rows=B, branch_scale=0.5)
    u = dl.fc_fwd(t["x"], t["W"])
    y, h = dl.block_norm_fwd(desc, t["x"], u, gate=t["gate"], w_post=t["w_post"], w_pre=t["w_pre"])
    loss, lse = dl.vocab_ce_fwd(h, t["Wo"], labels, bias=t["bo"])
    dh, dWo, dbo = dl.vocab_ce_bwd(h, t["Wo"], labels, lse, bias=t["bo"], scale=1.0 / B)
    g = dl.block_norm_bwd(desc, u, y, None, dh, gate=t["gate"], w_post=t["w_post"], w_pre=t["w_pre"])
    dW, _ = dl.fc_bwd_dw(t["x"], g["du"])
    grads = dict(W=dW.clone(), Wo=dWo.clone(), bo=dbo, gate=g["dgate"], w_post=g["dw_post"], w_pre=g["dw_pre"])
    dl.opt_muon([(t["W"], dW, mom["W"]), (t["Wo"], dWo, mom["Wo"])], lr=lr, momentum=0.9)
    return loss, grads


def exact(t, labels, mom, lr):
    t = {k: v.double().requires_grad_(True) for k, v in t.items()}
    B = t["x"].shape[0]
    u = t["x"] @ t["W"].t()
    n = u / torch.sqrt((u * u).mean(1, keepdim=True) + 1e-5) * t["w_post"]
    y = t["x"] + 0.5 * t["gate"] * n
    c = y - y.mean(1, keepdim=True)
    h = c / torch.sqrt((c * c).mean(1, keepdim=True) + 1e-5) * t["w_pre"]
    z = h @ t["Wo"].t() + t["bo"]
    live = labels >= 0
    loss = torch.where(live, torch.logsumexp(z, 1) - z.gather(1, labels.long().clamp_min(0)[:, None])[:, 0], 0.0)
    (loss.sum() / B).backward()
    new = {}
    for k in ("W", "Wo"):
        m = 0.9 * mom[k].double() + t[k].grad
        new[k] = t[k].detach() - lr * orthogonal(t[k].grad + 0.9 * m)
    return loss.detach(), {k: v.grad for k, v in t.items()}, new


@pytest.mark.gpu
@pytest.mark.parametrize("B,H,V", [(64, 96, 1500), (300, 130, 2111)])
def test_step(dl, pkg, B, H, V):
    t, labels = data(B, H, V, 5)
    mom = {k: torch.zeros_like(t[k]) for k in ("W", "Wo")}
    lr = 0.02
    eloss, egrads, enew = exact(t, labels, mom, lr)
    loss, grads = step(dl, pkg, t, labels, mom, lr)
    assert (loss.double() - eloss).abs().max() <= 1e-5 * max(1.0, eloss.abs().max().item())
    for k, g in grads.items():
        e = egrads[k].reshape(g.shape)
        assert (g.double() - e).norm() <= 1e-4 * e.norm(), k
    for k, e in enew.items():
        assert (t[k].double() - e).norm() <= lr * 485 * 1e-4 * min(t[k].shape) ** 0.5, k


@pytest.mark.gpu
def test_steps_recorded_and_replayed(pkg):
    """The whole step recorded into a HIP graph: three replays leave the weights that three eager steps leave, bit for bit."""
    d = pkg.Dlmi(0)
    try:
        stream = torch.cuda.Stream()
        d.set_stream(stream)
        t, labels = data(128, 96, 1000, 6)
        copy = lambda: {k: v.clone() for k, v in t.items()}
        eager, rec = copy(), copy()
        em, rm = ({k: torch.zeros_like(t[k]) for k in ("W", "Wo")} for _ in range(2))
        torch.cuda.synchronize()
        with torch.cuda.stream(stream):
            step(d, pkg, copy(), labels, {k: torch.zeros_like(t[k]) for k in ("W", "Wo")}, 0.02)  # grows the scratch
            stream.synchronize()
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=stream):
                step(d, pkg, rec, labels, rm, 0.02)
            losses = []
            for _ in range(3):
                loss, _ = step(d, pkg, eager, labels, em, 0.02)
                graph.replay()
                stream.synchronize()
                losses.append(loss.sum().item())
                for k in ("W", "Wo"):
                    assert torch.equal(eager[k], rec[k]) and torch.equal(em[k], rm[k])
            assert all(v == v for v in losses)
    finally:
        torch.cuda.synchronize()
        d.close()
