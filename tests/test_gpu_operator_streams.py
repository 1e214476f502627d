"""The vocabulary cross entropy, the orthogonalization and the block norms called from two contexts on two streams at once, eager
and as recorded graphs: each context has its own scratch and tickets, so every result is the one it gives alone."""
import pytest
import torch

from test_gpu_vocab_ce import make

ROWS = [(24, 300, 70001), (130, 200, 9000)]  # the one-launch forward with its ticket, and the packed one


class Side:
    def __init__(self, pkg, kind, seed):
        self.dl, self.pkg = pkg.Dlmi(0), pkg
        self.stream = torch.cuda.Stream()
        self.dl.set_stream(self.stream)
        self.ce = [make(B, K, V, kind, True, 0.1, seed + i) for i, (B, K, V) in enumerate(ROWS)]
        gen = torch.Generator(device="cuda").manual_seed(seed)
        r = lambda *s: torch.randn(*s, generator=gen, device="cuda").to(kind)
        self.G, self.x, self.u, self.gate = r(500, 700), r(600, 777), r(600, 777), r(1, 777)
        self.w = torch.rand(777, generator=gen, device="cuda") + 0.5
        self.desc = pkg.Dlmi.block_norm_desc(gate_act=pkg.GATE_ACT["TANH"], gate_rows=600)
        torch.cuda.synchronize()

    def step(self):
        out = []
        with torch.cuda.stream(self.stream):
            for X, W, b, labels in self.ce:
                loss, lse = self.dl.vocab_ce_fwd(X, W, labels, bias=b)
                out += [loss, lse, *self.dl.vocab_ce_bwd(X, W, labels, lse, bias=b, scale=0.1)]
            out.append(self.dl.orthogonalize(self.G))
            y, h = self.dl.block_norm_fwd(self.desc, self.x, self.u, gate=self.gate, w_post=self.w, w_pre=self.w)
            g = self.dl.block_norm_bwd(self.desc, self.u, y, self.x, self.x, gate=self.gate, w_post=self.w, w_pre=self.w)
            out += [y, h] + [g[k] for k in ("dx", "du", "dgate", "dw_post", "dw_pre")]
        return out


@pytest.mark.gpu
@pytest.mark.parametrize("kind", [torch.float32, torch.bfloat16])
def test_two_contexts_at_once(pkg, kind):
    sides = [Side(pkg, kind, 5), Side(pkg, kind, 6)]
    try:
        alone = []
        for s in sides:
            alone.append(s.step())
            torch.cuda.synchronize()
        for _ in range(5):
            both = [s.step() for s in sides]
            torch.cuda.synchronize()
            for a, b in zip(alone, both):
                assert all(torch.equal(x, y) for x, y in zip(a, b))
        graphs, outs = [], []
        for s in sides:
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=s.stream):
                outs.append(s.step())
            graphs.append(graph)
        for _ in range(5):
            for t in outs[0] + outs[1]:
                t.zero_()
            torch.cuda.synchronize()
            for s, graph in zip(sides, graphs):
                with torch.cuda.stream(s.stream):
                    graph.replay()
            torch.cuda.synchronize()
            for a, b in zip(alone, outs):
                assert all(torch.equal(x, y) for x, y in zip(a, b))
    finally:
        torch.cuda.synchronize()
        for s in sides:
            s.dl.close()
