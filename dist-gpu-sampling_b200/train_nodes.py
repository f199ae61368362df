"""A small node classifier trained on sampled mini-batches, from the sampler to the optimizer:

    python dist-gpu-sampling_b200/train_nodes.py [--nodes 200000] [--steps 100] [--bits 8] [--model attention]

PipelinedSampler delivers blocks and feature rows with several batches in flight; the rows go through layer_norm, two
mean-aggregation layers (plain torch), and linear_cross_entropy against the classes; AdamW steps 32-bit masters and writes the
16-bit parameters that the model reads.  --model attention: the layers are attention over the sampled neighbours, between linear_8bit
projections and residual_norm.  The role of the reference's training loop (oppo_bench/single_node/chunktensor.py:120-172)
without DGL.  The graph is synthetic: nodes of one class are linked more often, and their features lean one way.
"""
import argparse
import importlib
import os
import sys
import time

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
if ROOT not in sys.path:
    sys.path.insert(0, ROOT)


def make_graph(nodes, degree, classes, dim, seed):
    """CSC graph, features and labels: half of a node's neighbours share its class."""
    import numpy as np
    rng = np.random.default_rng(seed)
    labels = rng.integers(0, classes, size=nodes)
    order = np.argsort(labels, kind="stable")
    first = np.searchsorted(labels[order], np.arange(classes + 1))
    deg = rng.integers(1, 2 * degree, size=nodes)
    indptr = np.concatenate([[0], np.cumsum(deg)]).astype(np.int64)
    of = np.repeat(labels, deg)
    same = order[first[of] + (rng.random(of.size) * (first[of + 1] - first[of])).astype(np.int64)]
    indices = np.where(rng.random(of.size) < 0.5, same, rng.integers(0, nodes, size=of.size)).astype(np.int64)
    centres = rng.standard_normal((classes, dim)).astype(np.float32)
    feats = centres[labels] * 0.3 + rng.standard_normal((nodes, dim)).astype(np.float32)
    return indptr, indices, feats, labels.astype(np.int64)


class Sage:
    """Two layers h' = relu(norm(h_dst W_self + mean of the sampled neighbours' h W_neigh)) and a row per class."""

    def __init__(self, dim, hidden, classes, hops, seed=0):
        import torch
        g = torch.Generator().manual_seed(seed)

        def weight(a, b):
            return (torch.randn(a, b, generator=g) / a ** 0.5)

        sizes = [dim] + [hidden] * hops
        masters = {"norm_in": torch.ones(dim), "bias_in": torch.zeros(dim), "head": weight(hidden, classes).t().contiguous()}
        for i in range(hops):
            masters.update({"self%d" % i: weight(sizes[i], hidden), "neigh%d" % i: weight(sizes[i], hidden),
                            "norm%d" % i: torch.ones(hidden), "bias%d" % i: torch.zeros(hidden)})
        self.masters = {k: v.cuda() for k, v in masters.items()}
        self.p = {k: v.bfloat16().requires_grad_() for k, v in self.masters.items()}
        self.hops = hops

    def hidden(self, pkg, x, blocks):
        import torch
        p = self.p
        h = pkg.layer_norm(x, p["norm_in"], p["bias_in"]).bfloat16()
        for i, (row, col, n_src, n_dst) in enumerate(blocks):
            count = torch.zeros(n_dst, device="cuda").index_add_(0, row, torch.ones_like(row, dtype=torch.float32))
            total = torch.zeros(n_dst, h.shape[1], device="cuda").index_add(0, row, h[col].float())
            mean = (total / count.clamp_min(1.0)[:, None]).bfloat16()
            h = h[:n_dst] @ p["self%d" % i] + mean @ p["neigh%d" % i]
            h = torch.relu(pkg.layer_norm(h, p["norm%d" % i], p["bias%d" % i]))
        return h


class Attend:
    """Blocks h' = norm(h_dst + gate * W_out attention(W_query h_dst, the sampled neighbours' W_key_value h)) and a row per class.  Query
    heads share key heads in pairs, and the projections keep their inputs for the backward pass in 8 bits."""

    def __init__(self, dim, hidden, classes, hops, heads=4, seed=0):
        import torch
        if heads % 2 or hidden % heads or hidden // heads > 128:
            raise ValueError("Attend: hidden %d does not make an even number of %d heads of up to 128" % (hidden, heads))
        g = torch.Generator().manual_seed(seed)

        def weight(rows, cols):
            return torch.randn(rows, cols, generator=g) / cols ** 0.5

        masters = {"norm_in": torch.ones(dim), "bias_in": torch.zeros(dim), "into": weight(hidden, dim), "norm": torch.ones(hidden),
                   "bias": torch.zeros(hidden), "head": weight(classes, hidden)}
        for i in range(hops):
            masters.update({"query%d" % i: weight(hidden, hidden), "key_value%d" % i: weight(hidden, hidden), "out%d" % i: weight(hidden, hidden),
                            "gate%d" % i: torch.full((hidden,), 0.5), "norm%d" % i: torch.ones(hidden)})
        self.masters = {k: v.cuda() for k, v in masters.items()}
        self.p = {k: v.bfloat16().requires_grad_() for k, v in self.masters.items()}
        self.hops, self.heads, self.width = hops, heads, hidden // heads

    def hidden(self, pkg, x, blocks):
        import torch
        p, heads, width = self.p, self.heads, self.width
        x = pkg.layer_norm(x, p["norm_in"], p["bias_in"]).bfloat16()
        rows = pkg.linear_8bit(x, p["into"])  # the residual rows; h: their norm, which a block reads
        h = pkg.layer_norm(rows, p["norm"], p["bias"])
        for i, (row, col, n_src, n_dst) in enumerate(blocks):
            indptr, indices = pkg.block_csc(row, col, n_dst)
            query = pkg.linear_8bit(h[:n_dst], p["query%d" % i]).view(n_dst, heads, width)
            key_value = pkg.linear_8bit(h, p["key_value%d" % i])[indices].view(-1, heads, width)
            key, value = key_value[:, :heads // 2], key_value[:, heads // 2:]
            seen = pkg.attention(query, key, value, torch.arange(n_dst + 1, device=x.device), indptr)
            rows, h = pkg.residual_norm(rows[:n_dst], pkg.linear_8bit(seen.reshape(n_dst, heads * width), p["out%d" % i]), p["gate%d" % i],
                                        weight=p["norm%d" % i])
        return h


def main(argv=None):
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--nodes", type=int, default=200_000)
    ap.add_argument("--degree", type=int, default=15)
    ap.add_argument("--classes", type=int, default=47)
    ap.add_argument("--dim", type=int, default=100)
    ap.add_argument("--hidden", type=int, default=256)
    ap.add_argument("--batch", type=int, default=1024)
    ap.add_argument("--fanouts", default="10,10")
    ap.add_argument("--steps", type=int, default=100)
    ap.add_argument("--lr", type=float, default=3e-3)
    ap.add_argument("--bits", type=int, default=32, choices=(8, 32))
    ap.add_argument("--model", default="sage", choices=("sage", "attention"), help="mean aggregation, or attention over the neighbours")
    ap.add_argument("--unlabelled", type=float, default=0.1, help="share of the training nodes without a label")
    a = ap.parse_args(argv)

    import torch
    pkg = importlib.import_module("dist-gpu-sampling_b200")
    pkg.load_ops()
    indptr, indices, feats, labels = (torch.from_numpy(t) for t in make_graph(a.nodes, a.degree, a.classes, a.dim, seed=1))
    g = torch.Generator().manual_seed(2)
    labels[torch.rand(a.nodes, generator=g) < a.unlabelled] = -100
    labels = labels.cuda()

    def chunk(t):
        ct = torch.classes.dgs_classes.ChunkTensor(list(t.shape), t.dtype, t.numel() * t.element_size())
        ct._CAPI_load_from_tensor(t)
        return ct

    c_indptr, c_indices, c_feats = chunk(indptr), chunk(indices), chunk(feats)
    fanouts = [int(k) for k in a.fanouts.split(",")]
    sampler = pkg.PipelinedSampler(c_indptr, c_indices, fanouts, features=c_feats, max_seeds=a.batch, depth=3)
    model = (Attend if a.model == "attention" else Sage)(a.dim, a.hidden, a.classes, len(fanouts))
    names = sorted(model.masters)
    optimizer = pkg.AdamW([model.masters[k] for k in names], lr=a.lr, bits=a.bits, copies=[model.p[k] for k in names])
    torch.manual_seed(3)
    batches = [torch.randperm(a.nodes, generator=g)[:a.batch] for _ in range(a.steps)]
    losses, seeds = [], iter(batches)
    began = None
    train = torch.cuda.Stream(priority=-1)  # not behind the sampling kernels of the batches in flight
    with torch.cuda.stream(train):
        for _, blocks, _, x in sampler(b.cuda() for b in batches):
            target = labels[next(seeds).cuda()]
            h = model.hidden(pkg, x, blocks)
            loss = pkg.linear_cross_entropy(h, model.p["head"], target)
            loss.backward()
            optimizer.step()
            optimizer.zero_grad()
            losses.append(loss.detach())
            if len(losses) == 10:
                torch.cuda.synchronize()
                began = time.perf_counter()
    torch.cuda.synchronize()
    losses = [v.item() for v in losses]
    if began is not None and a.steps > 10:
        print("%.2f ms a step" % ((time.perf_counter() - began) / (a.steps - 10) * 1e3))
    for i in range(0, a.steps, max(1, a.steps // 10)):
        print("step %4d  loss %.4f" % (i, losses[i]))
    print("step %4d  loss %.4f" % (a.steps - 1, losses[-1]))
    del sampler
    return losses


if __name__ == "__main__":
    main()
