"""The operators of a training step behind the sampler, as measurable cases.

Three kinds, each in a plain form (elementary torch operations in 32 bits) and through torch.ops.dgs_ops:

  norm   layer norm of feature or hidden rows, forward alone or with its backward pass
  loss   softmax cross entropy of hidden rows against a weight row per class, the logits not kept; forward alone or
         with the gradients of the hidden rows and of the weight
  adamw  one AdamW step over a list of tensors, moments in 32 or in 8 bits, optionally with the low-precision copy
         of the parameters that the model reads

Moments and parameters lie in flat buffers in which every tensor begins at a multiple of 256 elements.
"""
import importlib
import itertools
import math
import random

import torch

own = False

DTYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}
ESZ = {"float32": 4, "bfloat16": 2, "float16": 2, "": 0}
EPS = 1e-5
IGNORE = -100
LR, BETA1, BETA2, ADAM_EPS, DECAY = 1e-3, 0.9, 0.999, 1e-8, 0.01
BLOCK = 256  # elements that share a scale


def listed():
    return [
        # hidden rows of one batch's seeds at inference: the smallest call there is, all latency
        dict(name="norm_batch_256", kind="norm", rows=1024, dim=256, dtype="float32", params="float32", pad=0, train=False),
        # the gathered features of one batch's input nodes, Products-shaped
        dict(name="norm_features_100", kind="norm", rows=430_000, dim=100, dtype="float32", params="float32", pad=0, train=True),
        # wide rows in mixed precision
        dict(name="norm_wide_4096", kind="norm", rows=16_384, dim=4096, dtype="bfloat16", params="float32", pad=0, train=True),
        # an odd width, rows that are part of a wider table
        dict(name="norm_odd_75", kind="norm", rows=33_333, dim=75, dtype="float16", params="float16", pad=6, train=True),
        # node classification: one batch's seeds against 172 classes, some of the seeds without a label
        dict(name="loss_classes", kind="loss", rows=1024, dim=256, vocab=172, dtype="bfloat16", pad=0, ignored=0.1, train=True),
        # a few rows against a large vocabulary: reading the weight once
        dict(name="loss_few_rows", kind="loss", rows=8, dim=512, vocab=50_000, dtype="bfloat16", pad=0, ignored=0.0, train=False),
        # link prediction judged against every node of the Products-shaped graph
        dict(name="loss_all_nodes", kind="loss", rows=1024, dim=128, vocab=2_449_029, dtype="bfloat16", pad=0, ignored=0.0, train=False),
        # a large training step
        dict(name="loss_train_large", kind="loss", rows=8192, dim=1024, vocab=65_537, dtype="bfloat16", pad=0, ignored=0.05, train=True),
        # odd sizes throughout
        dict(name="loss_train_odd", kind="loss", rows=4099, dim=203, vocab=30_011, dtype="float16", pad=3, ignored=0.3, train=True),
        # the layers of a small graph model, 32 bits throughout
        dict(name="adamw_small_model", kind="adamw", sizes="25600,25600,256,256,256,65536,65536,256,256,256,12032,12032,47",
             count=13, total=207_919, spread=0, grads="float32", copies="", bits=32),
        # an embedding row for every node, gradients in 16 bits, the 16-bit copy that the model reads
        dict(name="adamw_node_embedding", kind="adamw", sizes="313475712,25600,256,65536,256,12032,47", count=7, total=313_579_439,
             spread=0, grads="bfloat16", copies="bfloat16", bits=32),
        # many tensors of odd sizes, moments in 8 bits
        dict(name="adamw_8bit_many", kind="adamw", sizes="", count=120, total=60_000_000, spread=7, grads="bfloat16",
             copies="bfloat16", bits=8),
    ]


def _log(rng, lo, hi):
    """A whole number from lo to hi, spread over its logarithm."""
    return min(hi, max(lo, int(round(lo * (hi / lo) ** rng.random()))))


def draw(rng):
    kind = rng.choice(["norm", "loss", "loss", "adamw"])
    if kind == "norm":
        dtype = rng.choice(["float32", "bfloat16", "float16"])
        dim = _log(rng, 2, 8192)
        rows = _log(rng, 1, max(1, min(430_000, 67_000_000 // dim)))
        return dict(kind=kind, rows=rows, dim=dim, dtype=dtype, params=rng.choice([dtype, "float32"]),
                    pad=rng.choice([0, 0, 0, 1, 8]), train=rng.random() < 0.7)
    if kind == "loss":
        train = rng.random() < 0.6
        dim = _log(rng, 8, 1024)
        if rng.random() < 0.5:
            dim = -(-dim // 8) * 8
        vocab = _log(rng, 2, min(2_449_029, 180_000_000 // dim))
        rows = _log(rng, 1, max(1, min(8192, (500_000_000 if train else 2_000_000_000) // vocab)))
        return dict(kind=kind, rows=rows, dim=dim, vocab=vocab, dtype=rng.choice(["bfloat16", "bfloat16", "float16"]),
                    pad=rng.choice([0, 0, 0, 3]), ignored=rng.choice([0.0, 0.05, 0.5]), train=train)
    count = _log(rng, 1, 150)
    return dict(kind=kind, sizes="", count=count, total=_log(rng, max(1000, count * 40), 200_000_000), spread=rng.randrange(1 << 20),
                grads=rng.choice(["float32", "bfloat16", "float16"]), copies=rng.choice(["", "bfloat16", "float16"]),
                bits=rng.choice([8, 32]))


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------
def _tensor_sizes(case):
    if case["sizes"]:
        return [int(n) for n in case["sizes"].split(",")]
    rng = random.Random(case["spread"])
    shares = [math.exp(rng.uniform(0.0, 7.0)) for _ in range(case["count"])]
    return [max(1, int(case["total"] * s / sum(shares))) for s in shares]


def _slots(sizes):
    """Where each tensor begins in a flat buffer, and the buffer's length."""
    ends = list(itertools.accumulate((-(-n // BLOCK) * BLOCK for n in sizes), initial=0))
    return ends[:-1], ends[-1]


def _views(flat, sizes):
    return [flat[a:a + n] for a, n in zip(_slots(sizes)[0], sizes)]


def _strided(rows, dim, pad, dtype, g, scale, shift):
    """[rows, dim], the first columns of a table that is `pad` wider."""
    t = torch.randn((rows, dim + pad), device="cuda", generator=g)
    return t.mul_(scale).add_(shift).to(dtype)[:, :dim]


def _codes8(m, v):
    """8-bit codes and scales of both moments, a scale for each block: m = a sgn(c) (c/127)^2, sqrt(v) = a (c/255)^2."""
    m, r = m.view(-1, BLOCK), v.sqrt().view(-1, BLOCK)
    ma, ra = m.abs().amax(1), r.amax(1)
    t = torch.where(ma[:, None] > 0, m.abs() / ma[:, None], 0.0)
    mc = torch.round(t.sqrt() * 127.0) * m.sign()
    t = torch.where(ra[:, None] > 0, r / ra[:, None], 0.0)
    rc = torch.round(t.sqrt() * 255.0)
    rc = torch.where((r > 0) & (rc < 1), 1.0, rc)  # a second moment that is not zero stays so
    return mc.to(torch.int8).view(-1), ma, rc.to(torch.uint8).view(-1), ra


def _values8(mc, ma, rc, ra):
    c = mc.view(-1, BLOCK).float() * (1.0 / 127.0)
    m = c * c.abs() * ma[:, None]
    c = rc.view(-1, BLOCK).float() * (1.0 / 255.0)
    r = c * c * ra[:, None]
    return m.view(-1), (r * r).view(-1)


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    s = dict(case)
    if case["kind"] == "norm":
        n, d, dt, pt = case["rows"], case["dim"], DTYPES[case["dtype"]], DTYPES[case["params"]]
        s["x"] = _strided(n, d, case["pad"], dt, g, 1.5, 0.5)
        s["weight"] = torch.randn(d, device="cuda", generator=g).mul_(0.1).add_(1.0).to(pt)
        s["bias"] = torch.randn(d, device="cuda", generator=g).mul_(0.1).to(pt)
        if case["train"]:
            s["dy"] = torch.randn((n, d), device="cuda", generator=g).to(dt)
    elif case["kind"] == "loss":
        n, d, v, dt = case["rows"], case["dim"], case["vocab"], DTYPES[case["dtype"]]
        s["hidden"] = _strided(n, d, case["pad"], dt, g, 1.0, 0.0)
        s["weight"] = torch.randn((v, d), device="cuda", generator=g).mul_(2.0 / math.sqrt(d)).to(dt)
        t = torch.randint(0, v, (n,), device="cuda", generator=g)
        off = torch.rand(n, device="cuda", generator=g) < case["ignored"]
        s["target"] = torch.where(off, IGNORE, t)
        # the gradient of the rows' mean, times a weight that each row has
        s["dloss"] = torch.rand(n, device="cuda", generator=g).add_(0.5).div_(n)
    else:
        sizes = _tensor_sizes(case)
        total = _slots(sizes)[1]

        def flat(scale, dtype):
            f = torch.zeros(total, device="cuda")
            for x in _views(f, sizes):
                x.normal_(0.0, scale, generator=g)
            return f.to(dtype)

        s["params"], s["grads"] = flat(0.05, torch.float32), flat(1e-3, DTYPES[case["grads"]])
        s["copies"] = s["params"].to(DTYPES[case["copies"]]) if case["copies"] else None
        m = flat(3e-4, torch.float32)
        v = flat(1e-3, torch.float32).square_()
        if case["bits"] == 8:
            s["exp_avg"], s["exp_avg_scale"], s["exp_avg_sq"], s["exp_avg_sq_scale"] = _codes8(m, v)
        else:
            s["exp_avg"], s["exp_avg_sq"] = m, v
        s["step"] = 100
        # the tensors that the model and its backward pass hold
        s["param_list"], s["grad_list"] = _views(s["params"], sizes), _views(s["grads"], sizes)
        s["copy_list"] = _views(s["copies"], sizes) if case["copies"] else []
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


def _norm_plain(s):
    x, w = s["x"].float(), s["weight"].float()
    mean = x.mean(1, keepdim=True)
    c = x - mean
    rstd = 1.0 / (c.square().mean(1, keepdim=True) + EPS).sqrt()
    h = c * rstd
    y = (h * w + s["bias"].float()).to(s["x"].dtype)
    if not s["train"]:
        return y, mean[:, 0], rstd[:, 0]
    dy = s["dy"].float()
    g = dy * w
    dx = rstd * (g - g.mean(1, keepdim=True) - h * (g * h).mean(1, keepdim=True))
    return y, dx.to(s["x"].dtype), (dy * h).sum(0).to(s["weight"].dtype), dy.sum(0).to(s["weight"].dtype)


def _norm_own(s):
    ops = _ops()
    y, mean, rstd = ops._CAPI_layer_norm(s["x"], s["weight"], s["bias"], EPS)
    if not s["train"]:
        return y, mean, rstd
    dx, dw, db = ops._CAPI_layer_norm_backward(s["dy"], s["x"], s["weight"], mean, rstd, True, True)
    return y, dx, dw, db


def _loss_plain(s):
    h, w, target = s["hidden"].float(), s["weight"].float(), s["target"]
    logits = h @ w.t()
    top = logits.amax(1, keepdim=True)
    e = (logits - top).exp_()
    total = e.sum(1, keepdim=True)
    lse = (top + total.log())[:, 0]
    valid = target != IGNORE
    at = torch.where(valid, target, 0)[:, None]
    loss = torch.where(valid, lse - logits.gather(1, at)[:, 0], 0.0)
    if not s["train"]:
        return loss, lse * valid
    g = e.div_(total)
    g.scatter_add_(1, at, torch.full_like(total, -1.0))
    g.mul_((s["dloss"] * valid)[:, None])
    return loss, lse * valid, (g @ w).to(s["hidden"].dtype), (g.t() @ h).to(s["weight"].dtype)


def _loss_own(s):
    ops = _ops()
    loss, lse = ops._CAPI_linear_cross_entropy(s["hidden"], s["weight"], s["target"], IGNORE)
    if not s["train"]:
        return loss, lse
    dh, dw = ops._CAPI_linear_cross_entropy_backward(s["dloss"], s["hidden"], s["weight"], s["target"], lse, IGNORE, True, True)
    return loss, lse, dh, dw


def _adamw_plain(s):
    g, p = s["grads"].float(), s["params"]
    m, v = (s["exp_avg"], s["exp_avg_sq"]) if s["bits"] == 32 else \
        _values8(s["exp_avg"], s["exp_avg_scale"], s["exp_avg_sq"], s["exp_avg_sq_scale"])
    m = m * BETA1 + g * (1.0 - BETA1)
    v = v * BETA2 + g * g * (1.0 - BETA2)
    under = v.sqrt() * (1.0 / math.sqrt(1.0 - BETA2 ** s["step"])) + ADAM_EPS
    p = p * (1.0 - LR * DECAY) - m / under * (LR / (1.0 - BETA1 ** s["step"]))
    s["params"] = p
    if s["copies"] is not None:
        s["copies"] = p.to(s["copies"].dtype)
    if s["bits"] == 32:
        s["exp_avg"], s["exp_avg_sq"] = m, v
    else:
        s["exp_avg"], s["exp_avg_scale"], s["exp_avg_sq"], s["exp_avg_sq_scale"] = _codes8(m, v)
        m, v = _values8(s["exp_avg"], s["exp_avg_scale"], s["exp_avg_sq"], s["exp_avg_sq_scale"])
    s["step"] += 1
    return s["params"], s["copies"], m, v


def _adamw_own(s):
    ops = _ops()
    if s["bits"] == 32:
        ops._CAPI_adamw_step(s["param_list"], s["grad_list"], s["copy_list"], s["exp_avg"], s["exp_avg_sq"], LR, BETA1, BETA2,
                             ADAM_EPS, DECAY, s["step"])
        m, v = s["exp_avg"], s["exp_avg_sq"]
    else:
        ops._CAPI_adamw_step_8bit(s["param_list"], s["grad_list"], s["copy_list"], s["exp_avg"], s["exp_avg_scale"], s["exp_avg_sq"],
                                  s["exp_avg_sq_scale"], LR, BETA1, BETA2, ADAM_EPS, DECAY, s["step"])
        m = ops._CAPI_adamw_state_values(s["exp_avg"], s["exp_avg_scale"])
        v = ops._CAPI_adamw_state_values(s["exp_avg_sq"], s["exp_avg_sq_scale"])
    s["step"] += 1
    return s["params"], s["copies"], m, v


_PLAIN = {"norm": _norm_plain, "loss": _loss_plain, "adamw": _adamw_plain}
_OWN = {"norm": _norm_own, "loss": _loss_own, "adamw": _adamw_own}


def run(state):
    return (_OWN if own else _PLAIN)[state["kind"]](state)


# ---------------------------------------------------------------------------
# what a pass cannot do without, and its result in 64 bits
# ---------------------------------------------------------------------------
def work(case):
    if case["kind"] == "norm":
        n, d, e, p = case["rows"], case["dim"], ESZ[case["dtype"]], ESZ[case["params"]]
        if not case["train"]:
            return {"bytes": 2 * n * d * e + 2 * d * p + 8 * n, "flops": 8 * n * d}
        return {"bytes": 4 * n * d * e + 4 * d * p, "flops": 22 * n * d}
    if case["kind"] == "loss":
        n, d, v, e = case["rows"], case["dim"], case["vocab"], ESZ[case["dtype"]]
        live = n * (1.0 - case["ignored"])
        if not case["train"]:
            return {"bytes": (n + v) * d * e + 16 * n, "flops": 2 * live * v * d}
        return {"bytes": 2 * (n + v) * d * e + 20 * n, "flops": 6 * live * v * d}
    n = sum(_tensor_sizes(case))
    each = 8 + ESZ[case["grads"]] + ESZ[case["copies"]]
    # moments: read and written; from 8 bits the values they stand for are written too
    each += 16 if case["bits"] == 32 else 4 + 16.0 / BLOCK + 8
    return {"bytes": each * n, "flops": 16 * n}


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "norm":
        x = s["x"].double().requires_grad_(case["train"])
        w = s["weight"].double().requires_grad_(case["train"])
        b = s["bias"].double().requires_grad_(case["train"])
        y = torch.nn.functional.layer_norm(x, (case["dim"],), w, b, EPS)
        if not case["train"]:
            return y, x.mean(1), (x.var(1, unbiased=False) + EPS).rsqrt()
        y.backward(s["dy"].double())
        return y.detach(), x.grad, w.grad, b.grad
    if case["kind"] == "loss":
        h, w, target = s["hidden"].double(), s["weight"].double(), s["target"]
        rows = max(1, 400_000_000 // case["vocab"])
        loss, lse, dh, dw = [], [], [], None
        for a in range(0, case["rows"], rows):
            t = target[a:a + rows]
            z = h[a:a + rows] @ w.t()
            live = t != IGNORE
            lse.append(torch.logsumexp(z, 1) * live)
            loss.append(torch.nn.functional.cross_entropy(z, t, ignore_index=IGNORE, reduction="none"))
            if case["train"]:
                z = torch.softmax(z, 1)
                i = live.nonzero()[:, 0]
                z[i, t[i]] -= 1.0
                z *= (s["dloss"][a:a + rows].double() * live)[:, None]
                dh.append(z @ w)
                part = z.t() @ h[a:a + rows]
                dw = part if dw is None else dw.add_(part)
        if not case["train"]:
            return torch.cat(loss), torch.cat(lse)
        return torch.cat(loss), torch.cat(lse), torch.cat(dh), dw
    g = s["grads"].double()
    if case["bits"] == 32:
        m, v = s["exp_avg"].double(), s["exp_avg_sq"].double()
    else:
        c = s["exp_avg"].double().view(-1, BLOCK) / 127
        m = (torch.sign(c) * c ** 2 * s["exp_avg_scale"].double()[:, None]).view(-1)
        c = s["exp_avg_sq"].double().view(-1, BLOCK) / 255
        v = ((c ** 2 * s["exp_avg_sq_scale"].double()[:, None]) ** 2).view(-1)
    m.mul_(BETA1).add_(g, alpha=1 - BETA1)
    v.mul_(BETA2).addcmul_(g, g, value=1 - BETA2)
    t = s["step"]
    p = s["params"].double()
    p -= LR * DECAY * p
    p -= LR * (m / (1 - BETA1 ** t)) / ((v / (1 - BETA2 ** t)).sqrt() + ADAM_EPS)
    return p, (p if case["copies"] else None), (m if case["bits"] == 32 else None), (v if case["bits"] == 32 else None)
