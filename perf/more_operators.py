"""Further operators of a training step on sampled batches, as measurable cases.

Three kinds, each in a plain form (elementary torch operations in 32 bits) and through torch.ops.dgs_ops:

  attention  softmax attention of packed sequences of different lengths, with grouped heads: every seed over its sampled
             neighbours, the nodes of a neighbourhood or a walk among themselves, a read-out over a whole graph; forward alone
             or with the gradients of queries, keys and values
  norm       the end of a block: its output normalised, gated, scaled and added to the residual rows, and the norm before
             the next block; forward alone or with its backward pass
  kept       rows kept for the backward pass in 8 bits ("keep": codes and scales, and the values they stand for), and the
             gradient of a linear layer's weight from rows kept so ("grad")

Sequences are rows [offset[i], offset[i + 1]) of q and of k and v; rows behind the last one are padding.
"""
import importlib
import math
import random

import torch

own = False

DTYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}
ESZ = {"float32": 4, "bfloat16": 2, "float16": 2}
EPS = 1e-6
GROUP = 128  # elements of a row that share a scale


def listed():
    return [
        # the seeds of a small batch over their sampled neighbours, at inference: the smallest call, all latency
        dict(name="attention_small", kind="attention", mode="one", seqs=64, q_hi=1, k_lo=0, k_hi=10, spread=1, heads=4, kv_heads=4, dim=32,
             dtype="float32", causal=False, layout="apart", pad=0, train=False),
        # 60 000 nodes of a hop over up to 15 sampled neighbours each, some without any; buffers longer than the batch
        dict(name="attention_neighbours", kind="attention", mode="one", seqs=60_000, q_hi=1, k_lo=0, k_hi=15, spread=2, heads=4, kv_heads=4,
             dim=64, dtype="bfloat16", causal=False, layout="apart", pad=128, train=True),
        # walks or neighbourhoods of very different lengths, every node over those before it, q, k and v from one product
        dict(name="attention_walks", kind="attention", mode="same", seqs=700, q_hi=0, k_lo=1, k_hi=1000, spread=3, heads=8, kv_heads=2,
             dim=64, dtype="bfloat16", causal=True, layout="fused", pad=0, train=True),
        # long sequences, shared key heads: the largest one
        dict(name="attention_long", kind="attention", mode="same", seqs=4, q_hi=0, k_lo=8192, k_hi=8192, spread=4, heads=16, kv_heads=4,
             dim=128, dtype="bfloat16", causal=True, layout="apart", pad=0, train=True),
        # one read-out query for each of a few large graphs
        dict(name="attention_readout", kind="attention", mode="one", seqs=8, q_hi=1, k_lo=50_000, k_hi=200_000, spread=5, heads=8,
             kv_heads=8, dim=128, dtype="float16", causal=False, layout="apart", pad=0, train=False),
        # queries and keys of different odd lengths, the last query at the last key: rows that see no key at all
        dict(name="attention_odd", kind="attention", mode="cross", seqs=333, q_hi=300, k_lo=0, k_hi=500, spread=6, heads=6, kv_heads=3,
             dim=40, dtype="float16", causal=True, layout="apart", pad=7, train=True),
        # one batch's seeds at inference: the smallest call, all latency
        dict(name="norm_batch", kind="norm", rows=1024, dim=256, dtype="float32", params="float32", post="rms", pre="rms", gate="none",
             pad=0, train=False),
        # wide rows in mixed precision, a learned gate for each column
        dict(name="norm_wide", kind="norm", rows=16_384, dim=4096, dtype="bfloat16", params="bfloat16", post="layer", pre="layer",
             gate="column", pad=0, train=True),
        # a hop's rows, an odd width, rows of a wider table, a gate for each element
        dict(name="norm_odd", kind="norm", rows=33_333, dim=75, dtype="float16", params="float16", post="rms", pre="layer", gate="element",
             pad=6, train=True),
        # the gathered features of one batch's input nodes, Products-shaped
        dict(name="keep_features", kind="kept", step="keep", rows=430_000, dim=100, out=0, dtype="bfloat16", pad=0, bias=False),
        # a layer from hidden rows to the classes of a data set
        dict(name="kept_grad_classes", kind="kept", step="grad", rows=430_000, dim=256, out=47, dtype="bfloat16", pad=0, bias=True),
        # a wide layer
        dict(name="kept_grad_wide", kind="kept", step="grad", rows=16_384, dim=4096, out=1024, dtype="bfloat16", pad=0, bias=True),
    ]


def _log(rng, lo, hi):
    """A whole number from lo to hi, spread over its logarithm."""
    return min(hi, max(lo, int(round(lo * (hi / lo) ** rng.random()))))


def draw(rng):
    kind = rng.choice(["attention", "attention", "norm", "kept"])
    if kind == "attention":
        mode = rng.choice(["one", "same", "cross"])
        heads = rng.choice([1, 2, 4, 6, 8, 12, 16])
        kv = rng.choice([k for k in (1, 2, 3, 4, 6, 8, 16) if heads % k == 0])
        dim = rng.choice([16, 32, 40, 64, 64, 75, 96, 128, 128])
        dtype = rng.choice(["bfloat16", "bfloat16", "float16"])
        spread = rng.randrange(1 << 20)
        if mode == "one":
            hi = _log(rng, 1, 200_000)
            seqs = _log(rng, 1, max(1, min(60_000, 600_000_000 // (hi * kv * dim))))
            return dict(kind=kind, mode=mode, seqs=seqs, q_hi=1, k_lo=rng.choice([0, 1]), k_hi=hi, spread=spread, heads=heads, kv_heads=kv,
                        dim=dim, dtype=rng.choice([dtype, "float32"]), causal=False, layout="apart", pad=rng.choice([0, 33]),
                        train=rng.random() < 0.5)
        hi = _log(rng, 1, 8192)
        seqs = _log(rng, 1, max(1, min(2000, 2_000_000_000 // (hi * hi * heads), 100_000_000 // (hi * heads * dim))))
        return dict(kind=kind, mode=mode, seqs=seqs, q_hi=_log(rng, 1, hi) if mode == "cross" else 0, k_lo=rng.choice([0, 1]), k_hi=hi,
                    spread=spread, heads=heads, kv_heads=kv, dim=dim, dtype=dtype, causal=rng.random() < 0.6,
                    layout="fused" if mode == "same" and rng.random() < 0.5 else "apart", pad=rng.choice([0, 5]), train=rng.random() < 0.6)
    if kind == "norm":
        dtype = rng.choice(["float32", "bfloat16", "float16"])
        dim = _log(rng, 2, 8192)
        rows = _log(rng, 1, max(1, min(430_000, 67_000_000 // dim)))
        post, pre = rng.choice([("rms", "rms"), ("layer", "layer"), ("none", "rms"), ("none", "layer"), ("rms", "none"), ("rms", "layer")])
        return dict(kind=kind, rows=rows, dim=dim, dtype=dtype, params=dtype, post=post, pre=pre,
                    gate=rng.choice(["none", "column", "row", "element"]), pad=rng.choice([0, 0, 0, 1, 8]), train=rng.random() < 0.7)
    if rng.random() < 0.4:
        dim = _log(rng, 2, 4096)
        return dict(kind=kind, step="keep", rows=_log(rng, 1, max(1, min(430_000, 100_000_000 // dim))), dim=dim, out=0,
                    dtype=rng.choice(["float32", "bfloat16", "float16"]), pad=rng.choice([0, 0, 1, 8]), bias=False)
    dim, out = _log(rng, 8, 4096), _log(rng, 2, 1024)
    return dict(kind=kind, step="grad", rows=_log(rng, 1, max(1, min(430_000, 110_000_000 // max(dim, out)))), dim=dim, out=out,
                dtype=rng.choice(["bfloat16", "bfloat16", "float16"]), pad=rng.choice([0, 0, 3]), bias=rng.random() < 0.5)


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------
_lengths_of = {}


def _lengths(case):
    """Lengths of every sequence, (queries, keys): of the case, whatever the seed."""
    key = tuple(case[k] for k in ("mode", "seqs", "q_hi", "k_lo", "k_hi", "spread"))
    if key not in _lengths_of:
        rng = random.Random(case["spread"])
        lo, hi = case["k_lo"], case["k_hi"]
        if hi <= 16:
            k = [rng.randint(lo, hi) for _ in range(case["seqs"])]
        else:
            # (every twentieth has none where there may be none)
            k = [0 if lo == 0 and rng.random() < 0.05 else _log(rng, max(1, lo), hi) for _ in range(case["seqs"])]
        if case["mode"] == "one":
            q = [1] * len(k)
        elif case["mode"] == "same":
            q = k
        else:
            q = [rng.randint(0, case["q_hi"]) if rng.random() < 0.5 else _log(rng, 1, case["q_hi"]) for _ in k]
        _lengths_of.clear()
        _lengths_of[key] = q, k
    return _lengths_of[key]


def _pairs(case):
    """How many (query, key) pairs count, a head."""
    total = 0
    for q, k in zip(*_lengths(case)):
        if not case["causal"]:
            total += q * k
        else:  # query i sees the first i + 1 + k - q keys
            n = min(q, k)
            total += n * k - n * (n - 1) // 2
    return total


def _offsets(lengths):
    at, out = 0, [0]
    for n in lengths:
        at += n
        out.append(at)
    return out


def _strided(rows, dim, pad, dtype, g, scale, shift):
    """[rows, dim], the first columns of a table that is `pad` wider."""
    t = torch.randn((rows, dim + pad), device="cuda", generator=g)
    return t.mul_(scale).add_(shift).to(dtype)[:, :dim]


def _kept_plain(x):
    """Codes (as 32-bit floats) and scales: the nearest of 255 even steps, a scale for every 128 elements of a row."""
    n, d = x.shape
    groups = -(-d // GROUP)
    r = torch.nn.functional.pad(x.float(), (0, groups * GROUP - d)).view(n, groups, GROUP)
    top = r.abs().amax(2, keepdim=True)
    # (torch.div: `number / tensor` is a reciprocal and a product, which rounds twice)
    per = torch.where(top > 0, torch.div(torch.full_like(top, 127.0), top), 0.0)
    codes = torch.round(r * per).clamp_(-127.0, 127.0)
    return codes, torch.div(top, torch.full_like(top, 127.0))


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    s = dict(case)
    dt = DTYPES[case["dtype"]]

    def rand(*shape, scale=1.0, shift=0.0, dtype=dt):
        return torch.randn(shape, device="cuda", generator=g).mul_(scale).add_(shift).to(dtype)

    if case["kind"] == "attention":
        q_lens, k_lens = _lengths(case)
        nq, nk = sum(q_lens) + case["pad"], sum(k_lens) + case["pad"]
        h, hk, d = case["heads"], case["kv_heads"], case["dim"]
        if case["layout"] == "fused":
            both = rand(nq, h + 2 * hk, d)
            s["q"], s["k"], s["v"] = both[:, :h], both[:, h:h + hk], both[:, h + hk:]
        else:
            s["q"], s["k"], s["v"] = rand(nq, h, d), rand(nk, hk, d), rand(nk, hk, d)
        s["q_offsets"] = torch.tensor(_offsets(q_lens), device="cuda")
        s["k_offsets"] = torch.tensor(_offsets(k_lens), device="cuda")
        s["scale"] = 1.0 / math.sqrt(d)
        if case["train"]:
            s["dout"] = rand(nq, h, d)
    elif case["kind"] == "norm":
        n, d, pt = case["rows"], case["dim"], DTYPES[case["params"]]
        s["x"] = _strided(n, d, case["pad"], dt, g, 1.0, 0.1)
        s["y"] = _strided(n, d, case["pad"], dt, g, 1.5, 0.5)
        shape = {"column": (d,), "row": (n, 1), "element": (n, d)}.get(case["gate"])
        s["gate"] = rand(*shape, scale=0.3, shift=0.5, dtype=pt if case["gate"] == "column" else dt) if shape else None
        for which in ("post", "pre"):
            s[which + "_weight"] = rand(d, scale=0.1, shift=1.0, dtype=pt) if case[which] != "none" else None
            s[which + "_bias"] = rand(d, scale=0.1, dtype=pt) if case[which] == "layer" else None
        s["x_scale"], s["y_scale"] = 0.9, 0.7
        if case["train"]:
            s["dsum"], s["dout"] = rand(n, d), rand(n, d) if case["pre"] != "none" else None
    else:
        n, d = case["rows"], case["dim"]
        x = _strided(n, d, case["pad"] if case["step"] == "keep" else 0, dt, g, 1.0, 0.2)
        if case["step"] == "keep":
            s["x"] = x
        else:
            # hidden rows behind an activation: many of them are zeros
            codes, scales = _kept_plain(x.clamp_min_(0.0))
            s["codes"] = codes.view(n, -1)[:, :d].to(torch.int8).contiguous()
            s["scales"] = scales[:, :, 0].contiguous()
            s["grad"] = _strided(n, case["out"], case["pad"], dt, g, 1.0 / n ** 0.5, 0.0)
    return s


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------
_loaded = []


def _ops():
    if not _loaded:
        importlib.import_module("dist-gpu-sampling_b200").load_ops()
        _loaded.append(torch.ops.dgs_ops)
    return _loaded[0]


def _batches(s, budget=1 << 28):
    """Sequences of similar lengths, side by side: lists of their numbers with the longest lengths among them."""
    q_lens, k_lens = _lengths(s)
    by = {}
    for i, (q, k) in enumerate(zip(q_lens, k_lens)):
        if q and k:
            by.setdefault((q.bit_length(), k.bit_length()), []).append(i)
    for some in by.values():
        lq, lk = max(q_lens[i] for i in some), max(k_lens[i] for i in some)
        most = max(1, budget // max(lq * lk * s["heads"], (lq + lk) * s["heads"] * s["dim"]))
        for a in range(0, len(some), most):
            part = some[a:a + most]
            # one key head at a time where all of them would be too much at once
            step = s["kv_heads"] if len(part) * lq * lk * s["heads"] <= 2 * budget else 1
            for head in range(0, s["kv_heads"], step):
                yield torch.tensor(part, device="cuda"), lq, lk, head, step


def _attention_plain(s):
    q, k, v = s["q"], s["k"], s["v"]
    (nq, h, d), (nk, hk, _) = q.shape, k.shape
    g, train = h // hk, s["train"]
    out = torch.zeros((nq, h, d), device="cuda")
    lse = torch.full((h, nq), -math.inf, device="cuda")
    if train:
        dq, dk, dv = torch.zeros((nq, h, d), device="cuda"), torch.zeros((nk, hk, d), device="cuda"), torch.zeros((nk, hk, d), device="cuda")
    qo, ko = s["q_offsets"], s["k_offsets"]
    for seqs, lq, lk, head, count in _batches(s):
        b = seqs.numel()
        ql, kl = (qo[seqs + 1] - qo[seqs])[:, None], (ko[seqs + 1] - ko[seqs])[:, None]
        iq, ik = torch.arange(lq, device="cuda"), torch.arange(lk, device="cuda")
        there_q, there_k = iq < ql, ik < kl
        rq, rk = torch.where(there_q, qo[seqs][:, None] + iq, 0), torch.where(there_k, ko[seqs][:, None] + ik, 0)
        hs, ks = slice(head * g, (head + count) * g), slice(head, head + count)
        # [b, key head, queries of its group, d] and [b, key head, keys, d]
        rows = lambda t: t[:, hs][rq].float().view(b, lq, count, g, d).permute(0, 2, 3, 1, 4).reshape(b, count, g * lq, d)
        keys = lambda t: t[:, ks][rk].float().permute(0, 2, 1, 3)
        Q, K, V = rows(q), keys(k), keys(v)
        seen = there_q[:, :, None] & there_k[:, None, :]
        if s["causal"]:
            seen = seen & (ik[None, None, :] <= iq[None, :, None] + (kl - ql)[:, :, None])
        seen = seen[:, None, None]
        x = (Q @ K.transpose(2, 3)).mul_(s["scale"]).view(b, count, g, lq, lk)
        x = torch.where(seen, x, -math.inf)
        top = x.amax(4, keepdim=True)
        top = torch.where(top == -math.inf, 0.0, top)
        p = x.sub_(top).exp_()
        total = p.sum(4, keepdim=True)
        p.div_(torch.where(total > 0, total, 1.0))
        p = p.view(b, count, g * lq, lk)
        o = p @ V
        L = (top + total.log())[..., 0]
        back = lambda t: t.view(b, count, g, lq, d).permute(0, 3, 1, 2, 4).reshape(b, lq, count * g, d)[there_q]
        at = rq[there_q]
        out[at, hs] = back(o)
        lse[hs, at] = L.permute(1, 2, 0, 3).reshape(count * g, b, lq)[:, there_q]
        if train:
            dO = rows(s["dout"]) * there_q[:, None, None, :, None].expand(b, 1, g, lq, 1).reshape(b, 1, g * lq, 1)
            dV = p.transpose(2, 3) @ dO
            ds = dO @ V.transpose(2, 3)
            ds.sub_((dO * o).sum(3, keepdim=True)).mul_(p).mul_(s["scale"])
            dq[at, hs] = back(ds @ K)
            ak = rk[there_k]
            dk[ak, ks] = (ds.transpose(2, 3) @ Q).permute(0, 2, 1, 3)[there_k]
            dv[ak, ks] = dV.permute(0, 2, 1, 3)[there_k]
    dt = q.dtype
    if not train:
        return out.to(dt), lse
    return out.to(dt), lse, dq.to(dt), dk.to(dt), dv.to(dt)


def _attention_own(s):
    ops = _ops()
    a = s["q"], s["k"], s["v"]
    out, lse = ops._CAPI_attention(*a, s["q_offsets"], s["k_offsets"], s["causal"], s["scale"])
    if not s["train"]:
        return out, lse
    return (out, lse, *ops._CAPI_attention_backward(s["dout"], *a, out, lse, s["q_offsets"], s["k_offsets"], s["causal"], s["scale"],
                                                    True, True))


def _normed(kind, x):
    """(x - mean) / sqrt(var + eps), or x / sqrt(mean square + eps); the second is 1 / the root."""
    c = x - x.mean(1, keepdim=True) if kind == "layer" else x
    r = 1.0 / (c.square().mean(1, keepdim=True) + EPS).sqrt()
    return c * r, r


def _norm_back(kind, dxh, xh, r):
    dx = dxh - xh * (dxh * xh).mean(1, keepdim=True)
    if kind == "layer":
        dx = dx - dxh.mean(1, keepdim=True)
    return dx * r


def _norm_plain(s):
    dt, pt = s["x"].dtype, DTYPES[s["params"]]
    x, y = s["x"].float(), s["y"].float()
    z = y
    if s["post"] != "none":
        yh, yr = _normed(s["post"], y)
        z = yh * s["post_weight"].float()
        if s["post_bias"] is not None:
            z = z + s["post_bias"].float()
    gate = s["gate"].float() if s["gate"] is not None else None
    u = z * gate if gate is not None else z
    total = (x * s["x_scale"] + u * s["y_scale"]).to(dt)
    out = None
    if s["pre"] != "none":
        t = total.float()  # the norm is of the rows as they are stored
        th, tr = _normed(s["pre"], t)
        out = th * s["pre_weight"].float()
        if s["pre_bias"] is not None:
            out = out + s["pre_bias"].float()
        out = out.to(dt)
    if not s["train"]:
        return total, out
    res = {"sum": total, "out": out}
    d = s["dsum"].float()
    if s["pre"] != "none":
        do = s["dout"].float()
        res["pre_weight"] = (do * th).sum(0).to(pt)
        if s["pre_bias"] is not None:
            res["pre_bias"] = do.sum(0).to(pt)
        d = d + _norm_back(s["pre"], do * s["pre_weight"].float(), th, tr)
    res["x"] = (d * s["x_scale"]).to(dt)
    du = d * s["y_scale"]
    dz = du
    if gate is not None:
        dg = du * z
        res["gate"] = (dg.sum(0) if s["gate"].dim() == 1 else dg.sum(1, keepdim=True) if s["gate"].shape[1] != dg.shape[1] else dg)
        if s["gate"].dim() == 2 and s["dim"] == 1:
            res["gate"] = dg
        res["gate"] = res["gate"].to(s["gate"].dtype)
        dz = du * gate
    if s["post"] != "none":
        res["post_weight"] = (dz * yh).sum(0).to(pt)
        if s["post_bias"] is not None:
            res["post_bias"] = dz.sum(0).to(pt)
        dz = _norm_back(s["post"], dz * s["post_weight"].float(), yh, yr)
    res["y"] = dz.to(dt)
    return res


def _norm_own(s):
    ops = _ops()
    total, out, post_mean, post_rstd, mean, rstd = ops._CAPI_residual_norm(
        s["x"], s["y"], s["gate"], s["post"], s["post_weight"], s["post_bias"], s["pre"], s["pre_weight"], s["pre_bias"], s["x_scale"],
        s["y_scale"], EPS)
    if s["pre"] == "none":
        out = None
    if not s["train"]:
        return total, out
    dx, dy, dgate, dpw, dpb, dw, db = ops._CAPI_residual_norm_backward(
        s["dsum"], s["dout"], total, s["y"], s["gate"], s["post"], s["post_weight"], s["post_bias"], s["pre"], s["pre_weight"],
        post_mean, post_rstd, mean, rstd, s["x_scale"], s["y_scale"])
    res = {"sum": total, "out": out, "x": dx, "y": dy}
    if s["gate"] is not None:
        res["gate"] = dgate
    if s["post"] != "none":
        res["post_weight"] = dpw
        if s["post_bias"] is not None:
            res["post_bias"] = dpb
    if s["pre"] != "none":
        res["pre_weight"] = dw
        if s["pre_bias"] is not None:
            res["pre_bias"] = db
    return res


def _values_plain(codes, scales):
    n, d = codes.shape
    r = torch.nn.functional.pad(codes.float(), (0, scales.shape[1] * GROUP - d)).view(n, -1, GROUP)
    return (r * scales[:, :, None]).view(n, -1)[:, :d]


def _kept_run_plain(s):
    if s["step"] == "keep":
        codes, scales = _kept_plain(s["x"])
        return (codes * scales).view(s["rows"], -1)[:, :s["dim"]].to(s["x"].dtype), scales[:, :, 0]
    g = s["grad"].float()
    dw = (g.t() @ _values_plain(s["codes"], s["scales"])).to(s["grad"].dtype)
    return (dw, g.sum(0).to(dw.dtype)) if s["bias"] else (dw,)


def _kept_run_own(s):
    ops = _ops()
    if s["step"] == "keep":
        codes, scales = ops._CAPI_keep_8bit(s["x"])
        return ops._CAPI_kept_8bit_values(codes, scales, s["x"].dtype), scales
    dw, db = ops._CAPI_kept_8bit_weight_grad(s["grad"], s["codes"], s["scales"], s["bias"])
    return (dw, db) if s["bias"] else (dw,)


_PLAIN = {"attention": _attention_plain, "norm": _norm_plain, "kept": _kept_run_plain}
_OWN = {"attention": _attention_own, "norm": _norm_own, "kept": _kept_run_own}


def run(state):
    return (_OWN if own else _PLAIN)[state["kind"]](state)


# ---------------------------------------------------------------------------
# what a pass cannot do without, and its result in 64 bits
# ---------------------------------------------------------------------------
def work(case):
    e = ESZ[case["dtype"]]
    if case["kind"] == "attention":
        q_lens, k_lens = _lengths(case)
        q, kv = sum(q_lens) * case["heads"] * case["dim"] * e, 2 * sum(k_lens) * case["kv_heads"] * case["dim"] * e
        rest = 4 * sum(q_lens) * case["heads"] + 16 * len(q_lens)
        pairs = _pairs(case) * case["heads"] * case["dim"]
        if not case["train"]:
            return {"bytes": 2 * q + kv + rest, "flops": 4 * pairs}
        return {"bytes": 4 * q + 2 * kv + rest, "flops": 14 * pairs}
    if case["kind"] == "norm":
        n, d = case["rows"], case["dim"]
        gate = {"none": 0, "column": d, "row": n, "element": n * d}[case["gate"]] * e
        params = sum(d * ESZ[case["params"]] * {"none": 0, "rms": 1, "layer": 2}[case[w]] for w in ("post", "pre"))
        moved = 3 + (case["pre"] != "none")  # x, y, the sum, the normed rows
        if not case["train"]:
            return {"bytes": moved * n * d * e + gate + params, "flops": 20 * n * d}
        # and the gradients of the sum and of the normed rows in, those of x and y out
        return {"bytes": 2 * moved * n * d * e + 2 * gate + 2 * params, "flops": 60 * n * d}
    n, d, o = case["rows"], case["dim"], case["out"]
    groups = -(-d // GROUP)
    if case["step"] == "keep":
        # rows in, codes out and in, values out, scales
        return {"bytes": 2 * n * d * e + 2 * n * d + 8 * n * groups, "flops": 6 * n * d}
    return {"bytes": n * d + 4 * n * groups + n * o * e + o * d * e + (o * e if case["bias"] else 0), "flops": 2 * n * d * o}


def _attention_exact(case, s):
    q_lens, k_lens = _lengths(case)
    h, hk, d, train = case["heads"], case["kv_heads"], case["dim"], case["train"]
    g, scale = h // hk, s["scale"]
    pairs = sum(a * b for a, b in zip(q_lens, k_lens))
    few = len(q_lens) <= 2500
    if pairs * h * d * (3.5 if train else 1.0) > 2.5e12 or (not few and pairs * h * d > 4e8):
        return None
    q, k, v = s["q"].double(), s["k"].double(), s["v"].double()
    nq, nk = q.shape[0], k.shape[0]
    if train:
        do = s["dout"].double()
    if not few:
        # every pair on its own, sums over the pairs of a query or of a key
        dev = "cuda"
        ql, kl = torch.tensor(q_lens, device=dev), torch.tensor(k_lens, device=dev)
        seq = torch.repeat_interleave(torch.arange(len(q_lens), device=dev), ql * kl)
        nth = torch.arange(seq.numel(), device=dev) - torch.repeat_interleave((ql * kl).cumsum(0) - ql * kl, ql * kl)
        i, j = nth // kl[seq], nth % kl[seq]
        if case["causal"]:
            keep = j - i <= (kl - ql)[seq]
            seq, i, j = seq[keep], i[keep], j[keep]
        i, j = i + s["q_offsets"][seq], j + s["k_offsets"][seq]
        out, lse = torch.zeros_like(q), torch.full((h, nq), -math.inf, device=dev, dtype=torch.float64)
        grads = [torch.zeros_like(t) for t in (q, k, v)]
        for a in range(h):
            c = a // g
            x = (q[i, a] * k[j, c]).sum(1) * scale
            top = torch.full((nq,), -math.inf, device=dev, dtype=torch.float64).scatter_reduce(0, i, x, "amax")
            w = torch.exp(x - top[i])
            under = torch.zeros(nq, device=dev, dtype=torch.float64).index_add_(0, i, w)
            lse[a] = top + torch.log(under)
            w = w / under[i]
            out[:, a] = torch.zeros_like(q[:, a]).index_add_(0, i, w[:, None] * v[j, c])
            if train:
                grads[2][:, c].index_add_(0, j, w[:, None] * do[i, a])
                dw = (do[i, a] * v[j, c]).sum(1)
                dx = w * (dw - torch.zeros_like(under).index_add_(0, i, w * dw)[i]) * scale
                grads[0][:, a].index_add_(0, i, dx[:, None] * k[j, c])
                grads[1][:, c].index_add_(0, j, dx[:, None] * q[i, a])
        return (out, lse, *grads) if train else (out, lse)
    out, lse = torch.zeros_like(q), torch.full((h, nq), -math.inf, device="cuda", dtype=torch.float64)
    dq, dk, dv = (torch.zeros_like(t) for t in (q, k, v)) if train else (None, None, None)
    a = c = 0
    for lq, lk in zip(q_lens, k_lens):
        qs, ks = slice(a, a + lq), slice(c, c + lk)
        a, c = a + lq, c + lk
        if lq == 0 or lk == 0:
            continue
        if case["causal"]:
            hidden = torch.ones((lq, lk), dtype=torch.bool, device="cuda").triu_(lk - lq + 1)
            blind = max(0, lq - lk)  # queries in front of the first key
        for n in range(hk):
            hs = slice(n * g, (n + 1) * g)
            Q, K, V = q[qs, hs].transpose(0, 1), k[ks, n], v[ks, n]
            x = torch.matmul(Q, K.t()) * scale
            if case["causal"]:
                x.masked_fill_(hidden, -math.inf)
            L = torch.logsumexp(x, 2)
            w = torch.softmax(x, 2)
            del x
            if case["causal"] and blind:
                w[:, :blind] = 0.0
            out[qs, hs] = torch.matmul(w, V).transpose(0, 1)
            lse[hs, qs] = L
            if train:
                dO = do[qs, hs].transpose(0, 1)
                dv[ks, n] = torch.einsum("hij,hid->jd", w, dO)
                dw = torch.matmul(dO, V.t())
                dw = w * (dw - (w * dw).sum(2, keepdim=True)) * scale
                dq[qs, hs] = torch.matmul(dw, K).transpose(0, 1)
                dk[ks, n] = torch.einsum("hij,hid->jd", dw, Q)
    return (out, lse, dq, dk, dv) if train else (out, lse)


def _norm_exact(case, s):
    train, dt = case["train"], s["x"].dtype
    leaf = {k: s[k].double().requires_grad_(train) for k in ("x", "y", "gate", "post_weight", "post_bias", "pre_weight", "pre_bias")
            if s[k] is not None}

    def norm(which, t):
        c = t - t.mean(1, keepdim=True) if case[which] == "layer" else t
        t = c * torch.rsqrt((c * c).mean(1, keepdim=True) + EPS) * leaf[which + "_weight"]
        return t + leaf[which + "_bias"] if which + "_bias" in leaf else t

    z = norm("post", leaf["y"]) if case["post"] != "none" else leaf["y"]
    total = s["x_scale"] * leaf["x"] + s["y_scale"] * (z * leaf["gate"] if "gate" in leaf else z)
    # stored rows: the rounding to their type has the derivative 1
    stored = total + (total.detach().to(dt).double() - total.detach())
    out = norm("pre", stored) if case["pre"] != "none" else None
    if not train:
        return total, out
    loss = (stored * s["dsum"].double()).sum()
    if out is not None:
        loss = loss + (out * s["dout"].double()).sum()
    loss.backward()
    res = {"sum": total.detach(), "out": out.detach() if out is not None else None}
    res.update({k: t.grad for k, t in leaf.items()})
    return res


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "attention":
        return _attention_exact(case, s)
    if case["kind"] == "norm":
        return _norm_exact(case, s)
    if case["step"] == "keep":
        # (a value next to a border between two codes has the one that the arithmetic in 32 bits gives)
        x = s["x"].double().abs()
        tops = [x[:, a:a + GROUP].amax(1) for a in range(0, case["dim"], GROUP)]
        return None, torch.stack(tops, 1) / 127
    g = s["grad"].double()
    x = s["codes"].double()
    x *= s["scales"].double().repeat_interleave(GROUP, 1)[:, :case["dim"]]
    dw = torch.einsum("no,nd->od", g, x)
    return (dw, torch.einsum("no->o", g)) if case["bias"] else (dw,)
