"""The end of a block (norm, gate, residual, norm), forward and backward, against the definition in 64 bits.

Tolerances follow from the arithmetic: U = 2^-24, r = eps / 2 of the element type (one rounding).  A row's sums run over 8 values a
thread, 5 levels of shuffles and up to 32 warps, each step off by U of the sum of magnitudes: g = 64 U for a mean or a mean square, and
twice that for what is divided by its root.  In units of a row's deviation an error of the mean of g times the average magnitude counts
with rstd: off = 4 g (average |v| rstd + 1).  The second norm is of the stored sum, so the definition takes the sum that came back.
Errors go through the backward formulas by absolute values; column sums over n rows add (n + 64) U of their magnitudes."""
import itertools

import pytest
import torch

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
G = 64 * U
ROUND = {torch.float32: U, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
TINY = 2.0 ** -24
EPS = 1e-6


def make(n, D, dtype, ptype, post, pre, gate, pad=0, seed=0, bias=True):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def rand(*shape, scale=1.0, shift=0.0, t=dtype):
        return (torch.randn(shape, device="cuda", generator=g) * scale + shift).to(t)

    s = {k: rand(n, D + pad, scale=1.5, shift=0.4)[:, :D] for k in ("x", "y")}
    s["gate"] = {"none": lambda: None, "column": lambda: rand(D, t=ptype), "row": lambda: rand(n, 1),
                 "element": lambda: rand(n, D + pad)[:, :D]}[gate]()
    for k, kind in (("post", post), ("pre", pre)):
        s[k + "_weight"] = rand(D, scale=0.3, shift=1.0, t=ptype) if kind != "none" else None
        s[k + "_bias"] = rand(D, t=ptype) if kind != "none" and bias else None
    s["dsum"], s["dout"] = rand(n, D + pad)[:, :D], rand(n, D + pad)[:, :D] if pre != "none" else None
    return s


def normed(v, kind):
    """h, rstd and how far h may be off."""
    c = v - v.mean(-1, keepdim=True) if kind == "layer" else v
    rr = 1.0 / (c.square().mean(-1, keepdim=True) + EPS).sqrt()
    h = c * rr
    off = 4 * G * (v.abs().mean(-1, keepdim=True) * rr + 1) if kind == "layer" else 4 * G
    return h, rr, off * (h.abs() + (1 if kind == "layer" else 0))


def back(kind, d, w, h, rr, tol_h, tol_d):
    """The norm's gradient for d, and how far it may be off when d is off by tol_d and h by tol_h."""
    avg = lambda t: t.mean(-1, keepdim=True)  # noqa: E731
    e, te = d * w, tol_d * w.abs()
    res = rr * (e - h * avg(e * h) - (avg(e) if kind == "layer" else 0))
    size = e.abs() + h.abs() * avg((e * h).abs()) + avg(e.abs())
    tol = rr * (te + h.abs() * avg(te * h.abs()) + avg(te) + tol_h * avg((e * h).abs()) + h.abs() * avg(e.abs() * tol_h) + 8 * G * size)
    return res, tol


def check(ops, s, post, pre, xs=0.9, ys=-0.7):
    dt = s["x"].dtype
    r = ROUND[dt]
    D = s["x"].shape[-1]
    n = s["x"].numel() // D
    total, out, pm, pr, m, rs = ops._CAPI_residual_norm(s["x"], s["y"], s["gate"], post, s["post_weight"], s["post_bias"], pre,
                                                        s["pre_weight"], s["pre_bias"], xs, ys, EPS)
    one = torch.ones(D, device="cuda", dtype=torch.float64)
    wide = lambda k, absent: absent if s[k] is None else s[k].double()  # noqa: E731
    x, y, gate = s["x"].double(), s["y"].double(), wide("gate", one)
    z, tol_z = y, torch.zeros_like(y)
    if post != "none":
        yh, yr, tol_yh = normed(y, post)
        pw = wide("post_weight", one)
        z = yh * pw + wide("post_bias", 0 * one)
        tol_z = tol_yh * pw.abs() + 2 * U * (z.abs() + (yh * pw).abs())
    want = xs * x + ys * gate * z
    tol = abs(ys) * gate.abs() * tol_z + 4 * U * (abs(xs) * x.abs() + abs(ys) * (gate * z).abs()) + r * want.abs() + TINY
    assert ((total.double() - want).abs() <= tol).all()
    tol_g = torch.zeros_like(x)
    d = s["dsum"].double() if s["dsum"] is not None else torch.zeros_like(x)
    col = []
    if pre != "none":
        h, rr, tol_h = normed(total.double(), pre)
        w = wide("pre_weight", one)
        want = h * w + wide("pre_bias", 0 * one)
        assert ((out.double() - want).abs() <= tol_h * w.abs() + 2 * U * (want.abs() + (h * w).abs()) + r * want.abs() + TINY).all()
        if s["dout"] is not None:
            do = s["dout"].double()
            more, tol_g = back(pre, do, w, h, rr, tol_h, torch.zeros_like(x))
            d = d + more
            col += [("dw", do * h, do.abs() * tol_h), ("db", do, 0 * do)]
    else:
        assert out.numel() == 0
    tol_g = tol_g + 2 * U * d.abs()
    grads = ops._CAPI_residual_norm_backward(s["dsum"], s["dout"], total, s["y"], s["gate"], post, s["post_weight"], s["post_bias"], pre,
                                             s["pre_weight"], pm, pr, m, rs, xs, ys)
    got = dict(zip(("dx", "dy", "dgate", "dpw", "dpb", "dw", "db"), grads))
    assert ((got["dx"].double() - xs * d).abs() <= abs(xs) * (tol_g + 2 * U * d.abs()) + r * abs(xs) * d.abs() + TINY).all()
    du, tol_u = ys * d, abs(ys) * (tol_g + 2 * U * d.abs())
    if s["gate"] is not None:
        terms, tol = du * z, tol_u * z.abs() + du.abs() * tol_z + 2 * U * (du * z).abs()
        if s["gate"].shape == x.shape:
            assert ((got["dgate"].double() - terms).abs() <= tol + r * terms.abs() + TINY).all()
        elif s["gate"].dim() > 1:
            want = terms.sum(-1, keepdim=True)
            assert ((got["dgate"].double() - want).abs() <= tol.sum(-1, keepdim=True) + 64 * U * terms.abs().sum(-1, keepdim=True)
                    + r * want.abs() + TINY).all()
        else:
            col.append(("dgate", terms, tol))
    dz, tol_dz = du * gate, (tol_u + 2 * U * du.abs()) * gate.abs()
    if post != "none":
        col += [("dpw", dz * yh, tol_dz * yh.abs() + dz.abs() * tol_yh), ("dpb", dz, tol_dz)]
        dz, tol_dz = back(post, dz, pw, yh, yr, tol_yh, tol_dz)
    assert ((got["dy"].double() - dz).abs() <= tol_dz + r * dz.abs() + TINY).all()
    for name, terms, tol in col:
        if got[name].numel() == 0:
            continue
        flat = lambda t: t.reshape(-1, D)  # noqa: E731
        want = flat(terms).sum(0)
        tol = flat(tol).sum(0) + (n + 64) * U * flat(terms.abs()).sum(0) + ROUND[got[name].dtype] * want.abs() + TINY
        assert ((got[name].double() - want).abs() <= tol).all(), name
    return (total, out) + tuple(grads)


FORMS = [(p, q) for p in ("none", "rms", "layer") for q in ("none", "rms", "layer")]


@pytest.mark.parametrize("post,pre", FORMS)
@pytest.mark.parametrize("gate", ["none", "column", "row", "element"])
def test_all_forms(ops, post, pre, gate):
    for (n, D, dtype, pad), bias in zip([(37, 64, torch.float32, 0), (19, 75, torch.float16, 6), (9, 1024, torch.bfloat16, 8),
                                         (5, 2500, torch.float32, 1), (3, 4104, torch.bfloat16, 0)], itertools.cycle([True, False])):
        check(ops, make(n, D, dtype, dtype, post, pre, gate, pad, seed=D, bias=bias), post, pre)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("D", [1, 2, 7, 8, 31, 32, 33, 100, 128, 129, 255, 256, 257, 1000, 1024, 1032, 4095, 4096, 4097, 8191, 8192])
def test_widths(ops, D, dtype):
    for n in (1, 2, 33):
        check(ops, make(n, D, dtype, torch.float32, "layer", "rms", "column", seed=D + n), "layer", "rms")


@pytest.mark.parametrize("n,D", [(3001, 100), (5000, 256), (1200, 4096), (20000, 16)])
def test_many_rows(ops, n, D):
    """Every CTA takes several rows."""
    check(ops, make(n, D, torch.bfloat16, torch.float32, "rms", "layer", "element"), "rms", "layer")
    check(ops, make(n, D, torch.float32, torch.float32, "none", "rms", "row"), "none", "rms")


def test_absent_parts(ops):
    s = make(40, 96, torch.float32, torch.float32, "rms", "layer", "column")
    full = check(ops, s, "rms", "layer")
    for gone in ("dsum", "dout"):
        check(ops, dict(s, **{gone: None}), "rms", "layer")
    check(ops, dict(s, dsum=None, dout=None), "rms", "layer")
    # without weights: ones
    bare = dict(s, post_weight=None, post_bias=None, pre_weight=None, pre_bias=None)
    check(ops, bare, "rms", "layer")
    ones = torch.ones(96, device="cuda")
    a = check(ops, dict(bare, post_weight=ones, pre_weight=ones), "rms", "layer")
    b = check(ops, bare, "rms", "layer")
    assert all(torch.equal(p, q) for p, q in zip(a[:5], b[:5])) and b[5].numel() == 0
    assert full[0].shape == s["x"].shape


def test_shapes_and_strides(ops):
    s = make(24, 64, torch.bfloat16, torch.bfloat16, "rms", "rms", "element")
    base = check(ops, s, "rms", "rms")
    three = {k: v.reshape(2, 12, 64) if v is not None and v.dim() == 2 else v for k, v in s.items()}
    got = check(ops, three, "rms", "rms")
    assert got[0].shape == (2, 12, 64) and all(torch.equal(a.reshape(-1), b.reshape(-1)) for a, b in zip(base, got))
    turned = {k: v.t().contiguous().t() if v is not None and v.dim() == 2 else v for k, v in s.items()}
    assert all(torch.equal(a, b) for a, b in zip(base, check(ops, turned, "rms", "rms")))
    one = dict(s, dsum=s["dsum"][:1].expand(24, 64), dout=s["dout"][:1, :1].expand(24, 64))
    check(ops, one, "rms", "rms")
    off = torch.empty(24 * 64 + 1, dtype=torch.bfloat16, device="cuda")[1:].view(24, 64).copy_(s["y"])
    check(ops, dict(s, y=off), "rms", "rms")


def test_no_rows(ops):
    s = make(0, 32, torch.float32, torch.float32, "rms", "layer", "column")
    got = check(ops, s, "rms", "layer")
    assert got[0].shape == (0, 32) and all((t == 0).all() and t.shape == (32,) for t in got[4:])


def test_rows_that_are_not_finite_leave_the_others(ops):
    s = make(300, 256, torch.float32, torch.float32, "layer", "rms", "row")
    base = check(ops, s, "layer", "rms")
    bad = {k: v.clone() if v is not None else None for k, v in s.items()}
    bad["x"][7, 3], bad["y"][250, 9] = float("nan"), float("inf")
    total, out, *stats = ops._CAPI_residual_norm(bad["x"], bad["y"], bad["gate"], "layer", s["post_weight"], s["post_bias"], "rms",
                                                 s["pre_weight"], s["pre_bias"], 0.9, -0.7, EPS)
    grads = ops._CAPI_residual_norm_backward(s["dsum"], s["dout"], total, bad["y"], s["gate"], "layer", s["post_weight"], s["post_bias"], "rms",
                                             s["pre_weight"], *stats, 0.9, -0.7)
    rows = [i for i in range(300) if i not in (7, 250)]
    assert all(torch.equal(a[rows], b[rows]) for a, b in zip((total, out, *grads[:3]), base[:5]))


def test_the_same_inputs_give_the_same_bits(ops):
    s = make(7000, 100, torch.bfloat16, torch.float32, "layer", "layer", "column")
    base = check(ops, s, "layer", "layer")
    for _ in range(3):
        assert all(torch.equal(a, b) for a, b in zip(base, check(ops, s, "layer", "layer")))


def test_a_value_far_from_zero(ops):
    """Variances are of centred values: rows around 1000 with a deviation of 1."""
    s = make(64, 512, torch.float32, torch.float32, "layer", "layer", "none")
    s["x"], s["y"] = s["x"] + 1000.0, s["y"] + 1000.0
    check(ops, s, "layer", "layer")


def test_autograd(pkg):
    s = make(30, 48, torch.float32, torch.float32, "rms", "layer", "element")
    names = ("x", "y", "gate", "post_weight", "post_bias", "pre_weight", "pre_bias")
    mine = {k: s[k].clone().requires_grad_() for k in names}
    total, out = pkg.residual_norm(mine["x"], mine["y"], mine["gate"], "rms", mine["post_weight"], mine["post_bias"], "layer",
                                   mine["pre_weight"], mine["pre_bias"], 0.9, 0.7, EPS)
    ((total * s["dsum"]).sum() + (out * s["dout"]).sum()).backward()
    ref = {k: s[k].double().requires_grad_() for k in names}
    z = ref["y"] * torch.rsqrt(ref["y"].square().mean(-1, keepdim=True) + EPS) * ref["post_weight"] + ref["post_bias"]
    t = 0.9 * ref["x"] + 0.7 * ref["gate"] * z
    o = torch.nn.functional.layer_norm(t, (48,), ref["pre_weight"], ref["pre_bias"], EPS)
    ((t * s["dsum"]).sum() + (o * s["dout"]).sum()).backward()
    for k in names:
        # sums of 30 rows of gradients of some 10, all in 32 bits: 2^-24 times some hundred steps
        assert (mine[k].grad.double() - ref[k].grad).abs().amax() <= 256 * U * ref[k].grad.abs().amax() + 256 * U
    # one output alone, and neither
    for which in (0, 1):
        x = s["x"].clone().requires_grad_()
        pkg.residual_norm(x, s["y"], norm="rms", weight=s["pre_weight"])[which].sum().backward()
        assert x.grad is not None
    total, none = pkg.residual_norm(s["x"], s["y"], norm=None)
    assert none is None and torch.equal(total, s["x"] + s["y"])
    with pytest.raises(ValueError, match="norm"):
        pkg.residual_norm(s["x"], s["y"], norm="batch")


def test_differences(pkg):
    """The gradient along random directions against central differences in 32 bits."""
    s = make(6, 16, torch.float32, torch.float32, "layer", "rms", "row", seed=9)
    names = ("x", "y", "gate", "post_weight", "pre_weight")
    leaf = {k: s[k].clone().requires_grad_() for k in names}

    def loss(t):
        total, out = pkg.residual_norm(t["x"], t["y"], t["gate"], "layer", t["post_weight"], s["post_bias"], "rms", t["pre_weight"],
                                       s["pre_bias"])
        return (total.double() * s["dsum"].double()).sum() + (out.double() * s["dout"].double()).sum()

    loss(leaf).backward()
    g = torch.Generator(device="cuda").manual_seed(4)
    h = 2.0 ** -7
    with torch.no_grad():
        size = sum(s[k].abs().sum().double() for k in ("dsum", "dout")) * 4
        for k in names:
            way = torch.randn(s[k].shape, device="cuda", generator=g)
            way /= way.norm()
            ends = [loss(dict(s, **{k: s[k] + sign * h * way})) for sign in (1, -1)]
            slope = (ends[0] - ends[1]) / (2 * h)
            # third derivatives of some hundred (rows of 16 with deviations near 1) leave 100 h^2, rounding 2^-22 of the sums over h
            assert (slope - (leaf[k].grad.double() * way.double()).sum()).abs() <= 100 * h * h + 2.0 ** -22 * size / h


def test_recorded_and_on_another_stream(ops):
    s = make(500, 200, torch.bfloat16, torch.bfloat16, "rms", "layer", "column")
    args = (s["gate"], "rms", s["post_weight"], s["post_bias"], "layer", s["pre_weight"], s["pre_bias"], 0.9, -0.7, EPS)

    def both():
        total, out, *stats = ops._CAPI_residual_norm(s["x"], s["y"], *args)
        return (total, out) + tuple(ops._CAPI_residual_norm_backward(s["dsum"], s["dout"], total, s["y"], s["gate"], "rms", s["post_weight"],
                                                                     s["post_bias"], "layer", s["pre_weight"], *stats, 0.9, -0.7))

    both()
    torch.cuda.synchronize()
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            graphs.append((g, both()))
    s["x"].mul_(0.5)
    want = both()
    for g, _ in graphs:
        g.replay()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        more = both()
    torch.cuda.synchronize()
    for res in [r for _, r in graphs] + [more]:
        assert all(torch.equal(a, b) for a, b in zip(res, want))


def test_refusals(ops):
    s = make(4, 16, torch.float32, torch.float32, "rms", "layer", "column")

    def call(post="rms", pre="layer", **kw):
        a = dict(s, **kw)
        return ops._CAPI_residual_norm(a["x"], a["y"], a["gate"], post, a["post_weight"], a["post_bias"], pre, a["pre_weight"], a["pre_bias"],
                                       1.0, 1.0, EPS)

    total, out, *stats = call()
    for kw, text in ((dict(y=s["y"].half()), "one shape and type"), (dict(y=s["y"][:3]), "one shape"), (dict(x=s["x"].double()), "one shape|float32"),
                     (dict(post="none"), "without its norm"), (dict(pre="none"), "without its norm"), (dict(pre="batch"), "'none', 'rms' or 'layer'"),
                     (dict(post_weight=None), "needs a weight"), (dict(pre_weight=None), "needs a weight"),
                     (dict(pre_weight=s["pre_weight"][:3]), "elements of a row"), (dict(pre_weight=s["pre_weight"].half()), "share one type"),
                     (dict(gate=s["x"][:3]), "the gate"), (dict(gate=s["x"].half()), "type of x"), (dict(gate=s["gate"].cpu()), "must be on")):
        with pytest.raises(RuntimeError, match=text):
            call(**kw)
    wide = torch.zeros(2, 8200, device="cuda")
    with pytest.raises(RuntimeError, match="8192"):
        ops._CAPI_residual_norm(wide, wide, None, "none", None, None, "rms", None, None, 1.0, 1.0, EPS)
    with pytest.raises(RuntimeError, match="scales finite"):
        ops._CAPI_residual_norm(s["x"], s["y"], None, "none", None, None, "rms", None, None, float("inf"), 1.0, EPS)

    def back(ds=s["dsum"], do=s["dout"], st=stats, pre="layer"):
        return ops._CAPI_residual_norm_backward(ds, do, total, s["y"], s["gate"], "rms", s["post_weight"], s["post_bias"], pre,
                                                s["pre_weight"] if pre != "none" else None, *st, 1.0, 1.0)

    for kw, text in ((dict(ds=s["dsum"][:2]), "shape and type of sum"), (dict(do=s["dout"].half()), "shape and type of sum"),
                     (dict(st=stats[:3] + [stats[3][:2]]), "rstd must be what"), (dict(pre="none", st=stats[:2] + [stats[0], stats[0]]), "without its norm")):
        with pytest.raises(RuntimeError, match=text):
            back(**kw)
