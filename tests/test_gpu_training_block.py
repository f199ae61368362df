"""The operators of a block together, as a model uses them: projections that keep their inputs in 8 bits, attention over sampled
neighbours, residual and norm.

Tolerances.  In float32 each stage's sums are of some hundred products, so values and gradients are within a few hundred roundings of
2^-24 of the size that they have here (500 * 2^-24 of the largest, doubled for the chain of five stages).  A weight's gradient is taken
from rows of which each value is within a / 254 of its own, a the largest magnitude in its row's 128 columns: entry (o, c) is off by at
most sum over rows n of |g[n, o]| a[n, c] / 254 besides."""
import importlib

import pytest
import torch

pytestmark = pytest.mark.gpu
CHAIN = 2 * 500 * 2.0 ** -24


@pytest.mark.parametrize("dim,hidden,fanouts,bits", [(36, 64, "5,5", 32), (33, 96, "3,4,2", 8)])
def test_the_example_runs(dim, hidden, fanouts, bits, capsys):
    example = importlib.import_module("dist-gpu-sampling_b200.train_nodes")
    losses = example.main(["--nodes", "20000", "--steps", "12", "--batch", "300", "--classes", "12", "--hidden", str(hidden), "--dim", str(dim),
                           "--fanouts", fanouts, "--bits", str(bits), "--model", "attention"])
    assert len(losses) == 12 and all(torch.isfinite(torch.tensor(losses)))
    assert "step   11" in capsys.readouterr().out


def block(n_src=150, n_dst=60, edges=500, D=40, heads=4, seed=0):
    """Parameters in float32, and a block whose last three destinations have no neighbour."""
    g = torch.Generator().manual_seed(seed)
    row = torch.randint(0, n_dst - 3, (edges,), generator=g).sort().values.cuda()
    col = torch.randint(0, n_src, (edges,), generator=g).cuda()
    p = {"x": torch.randn(n_src, D, generator=g), "query": torch.randn(D, D, generator=g) * 0.2, "kv": torch.randn(D, D, generator=g) * 0.2,
         "out": torch.randn(D, D, generator=g) * 0.2, "gate": torch.rand(D, generator=g) + 0.5, "norm": torch.rand(D, generator=g) + 0.5}
    return {k: v.cuda().requires_grad_() for k, v in p.items()}, row, col, n_dst, heads


def own(pkg, p, row, col, n_dst, heads):
    D = p["x"].shape[1]
    indptr, indices = pkg.block_csc(row, col, n_dst)
    q = pkg.linear_8bit(p["x"][:n_dst], p["query"]).view(n_dst, heads, -1)
    kv = pkg.linear_8bit(p["x"], p["kv"])[indices].view(-1, heads, D // heads)
    seen = pkg.attention(q, kv[:, :heads // 2], kv[:, heads // 2:], torch.arange(n_dst + 1, device="cuda"), indptr)
    return pkg.residual_norm(p["x"][:n_dst], pkg.linear_8bit(seen.reshape(n_dst, D), p["out"]), p["gate"], weight=p["norm"])


def plain(p, row, col, n_dst, heads):
    """The formulas in 64 bits; the projections' (input, result) too."""
    D = p["x"].shape[1]
    pairs = {}

    def linear(name, x):
        y = x @ p[name].t()
        y.retain_grad()
        pairs[name] = (x, y)
        return y

    q = linear("query", p["x"][:n_dst]).view(n_dst, heads, -1)
    kv = linear("kv", p["x"])[col].view(-1, heads, D // heads)
    k, v = (t.repeat_interleave(2, 1) for t in (kv[:, :heads // 2], kv[:, heads // 2:]))
    score = (q[row] * k).sum(-1) * (D // heads) ** -0.5
    e = (score - score.detach().amax() if score.numel() else score).exp()
    total = torch.zeros(n_dst, heads, dtype=e.dtype, device=e.device).index_add(0, row, e)
    seen = torch.zeros(n_dst, heads, D // heads, dtype=e.dtype, device=e.device).index_add(0, row, e[..., None] * v)
    seen = seen / torch.where(total > 0, total, torch.ones_like(total))[..., None]
    rows = p["x"][:n_dst] + p["gate"] * linear("out", seen.reshape(n_dst, D))
    return rows, rows * (rows.square().mean(-1, keepdim=True) + 1e-6).rsqrt() * p["norm"], pairs


@pytest.mark.parametrize("sizes", [{}, {"n_src": 4, "n_dst": 4, "edges": 1, "D": 8}, {"n_src": 700, "n_dst": 5, "edges": 3000, "D": 136},
                                   {"n_src": 300, "n_dst": 299, "edges": 0, "D": 20}])
def test_a_block_and_its_gradients(pkg, sizes):
    p, *graph = block(**sizes)
    wide = {k: v.detach().double().requires_grad_() for k, v in p.items()}
    g = torch.Generator(device="cuda").manual_seed(1)
    rows, out = own(pkg, p, *graph)
    want_rows, want, pairs = plain(wide, *graph)
    ds, do = (torch.randn(rows.shape, device="cuda", generator=g) for _ in range(2))
    torch.autograd.backward((rows, out), (ds, do))
    torch.autograd.backward((want_rows, want), (ds.double(), do.double()))
    for a, b in ((rows, want_rows), (out, want)):
        assert (a.double() - b).abs().max() <= CHAIN * b.abs().max()
    for name in p:
        a, b = p[name].grad.double(), wide[name].grad
        room = CHAIN * max(1.0, b.abs().max().item())
        if name in pairs:
            x, y = pairs[name]
            D = x.shape[1]
            largest = torch.cat([x[:, c:c + 128].abs().amax(1, keepdim=True).expand(-1, min(128, D - c)) for c in range(0, D, 128)], 1)
            room = room + (y.grad.abs().t() @ largest).detach() / 254
        assert ((a - b).abs() <= room).all(), name


def test_recorded_with_its_gradients(pkg):
    """Forward and backward as one graph: replays on new values give what the eager calls give."""
    p, *graph = block()
    names = sorted(p)
    indptr, indices = pkg.block_csc(graph[0], graph[1], graph[2])
    queries = torch.arange(graph[2] + 1, device="cuda")

    def step():
        n_dst, heads, D = graph[2], graph[3], p["x"].shape[1]
        q = pkg.linear_8bit(p["x"][:n_dst], p["query"]).view(n_dst, heads, -1)
        kv = pkg.linear_8bit(p["x"], p["kv"])[indices].view(-1, heads, D // heads)
        seen = pkg.attention(q, kv[:, :heads // 2], kv[:, heads // 2:], queries, indptr)
        rows, out = pkg.residual_norm(p["x"][:n_dst], pkg.linear_8bit(seen.reshape(n_dst, D), p["out"]), p["gate"], weight=p["norm"])
        return (rows.detach(), out.detach(), *torch.autograd.grad((rows + out * 0.5).square().sum(), [p[k] for k in names]))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    recorded = torch.cuda.CUDAGraph()
    with torch.cuda.graph(recorded):
        got = step()
    for seed in (5, 6):
        fresh = block(seed=seed)[0]
        with torch.no_grad():
            for k in names:
                p[k].copy_(fresh[k])
        recorded.replay()
        torch.cuda.synchronize()
        for i, (a, b) in enumerate(zip(got, step())):
            # (torch adds the rows that are indexed twice with atomics, in any order: kv's share of the gradients)
            assert (a - b).abs().max() <= CHAIN * max(1.0, b.abs().max().item()), i


def test_under_autocast(pkg):
    """linear_8bit computes in its operands' type, whatever autocast would choose, in both passes."""
    x, w = torch.randn(30, 20, device="cuda", requires_grad=True), torch.randn(10, 20, device="cuda", requires_grad=True)
    plain_y = pkg.linear_8bit(x, w)
    plain_grads = torch.autograd.grad(plain_y.sum(), (x, w))
    with torch.autocast("cuda", dtype=torch.bfloat16):
        y = pkg.linear_8bit(x, w)
        assert y.dtype == torch.float32 and torch.equal(y, plain_y)
        for a, b in zip(torch.autograd.grad(y.sum(), (x, w)), plain_grads):
            assert a.dtype == torch.float32 and torch.equal(a, b)
