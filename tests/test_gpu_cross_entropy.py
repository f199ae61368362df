"""Softmax cross entropy against a large vocabulary, forward and backward, against the definition in 64 bits.

Tolerances follow from the arithmetic.  With u = 2^-24: a logit is a sum of D exact (16-bit types) or rounded (32-bit)
products in 32 bits, each addition rounded or cut, so it is within e = 2 (D + 8) u sum |h w| of its value; the exponentials
are good to a few units, the sum over V of them to (V + 64) u.  A gradient is a sum over V (or n) of products of G, which
carries the type's rounding r (2^-8, 2^-11, or u) and the error of exp, in 32 bits, and is rounded once to the type."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
ROUND = {torch.float32: U, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
TYPES = [torch.float32, torch.bfloat16, torch.float16]
SIZES = [(1, 1, 1), (1, 8, 2), (3, 5, 7), (2, 64, 300), (127, 64, 255), (128, 64, 256), (129, 72, 257), (200, 16, 513),
         (257, 200, 129), (300, 203, 1000), (5, 1000, 3001), (1000, 100, 47), (64, 256, 5000), (385, 264, 1537)]


def make(n, D, V, dtype, ignored=0.0, seed=0, pad=0, wpad=0, scale=2.0, ids=torch.int64):
    g = torch.Generator(device="cuda").manual_seed(seed)
    h = torch.randn((n, D + pad), device="cuda", generator=g).to(dtype)[:, :D]
    w = (torch.randn((V, D + wpad), device="cuda", generator=g) * (scale / math.sqrt(D))).to(dtype)[:, :D]
    t = torch.randint(0, V, (n,), device="cuda", generator=g)
    t[torch.rand(n, device="cuda", generator=g) < ignored] = -100
    dl = torch.rand(n, device="cuda", generator=g) + 0.5
    return h, w, t.to(ids), dl


def check(ops, h, w, t, dl, ignore=-100):
    n, D, V, r = h.shape[0], h.shape[1], w.shape[0], ROUND[h.dtype]
    hd, wd, live = h.double(), w.double(), t != ignore
    hd = torch.where(live[:, None], hd, 0.0)
    s = hd @ wd.t()
    e = 2 * (D + 8) * U * (hd.abs() @ wd.abs().t()).amax(1)
    lse = torch.logsumexp(s, 1)
    at = torch.where(live, t, 0).long()[:, None]
    loss = (lse - s.gather(1, at)[:, 0]) * live
    got_loss, got_lse = ops._CAPI_linear_cross_entropy(h, w, t, ignore)
    assert got_loss.dtype == got_lse.dtype == torch.float32
    tol = 2 * e + (V + 64) * U + 8 * U * (lse.abs() + s.abs().amax(1))
    assert ((got_lse.double() - lse * live).abs() <= tol * live).all()
    assert ((got_loss.double() - loss).abs() <= 2 * tol * live).all()
    dh, dw = ops._CAPI_linear_cross_entropy_backward(dl, h, w, t, got_lse, ignore, True, True)
    p = torch.softmax(s, 1)
    G = p.clone()
    G[torch.arange(n, device="cuda"), at[:, 0]] -= 1.0
    scale = torch.where(live, dl, 0.0).double()[:, None]
    G, p = G * scale, p * scale
    # what each entry of G may be off by: the exponential of a logit and an lse that are off, the type's rounding, and for
    # float16 the distance of the smallest steps, 2^-24 of the largest factor
    dG = p.abs() * (4 * e + tol + 32 * U)[:, None] + G.abs() * r + (2.0 ** -24 * dl.max() if h.dtype == torch.float16 else 0.0)
    dG = torch.where(live[:, None], dG, 0.0)
    for got, ref, lim, k in ((dh, G @ wd, dG @ wd.abs() + 2 * (V + 8) * U * (G.abs() @ wd.abs()), V),
                             (dw, G.t() @ hd, dG.t() @ hd.abs() + 2 * (n + 8) * U * (G.abs().t() @ hd.abs()), n)):
        small = 2.0 ** -25 if h.dtype == torch.float16 else 2.0 ** -126
        assert got.dtype == h.dtype and ((got.double() - ref).abs() <= lim + r * ref.abs() + small).all()
    assert (dh[~live] == 0).all()
    return got_loss, got_lse, dh, dw


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,D,V", SIZES)
def test_sizes(ops, n, D, V, dtype):
    check(ops, *make(n, D, V, dtype))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("n", [1, 2, 7, 8, 9])
@pytest.mark.parametrize("D", [1, 4, 75, 256, 260, 1030, 1100])
def test_few_rows(ops, dtype, n, D):
    for V, ignored in ((129, 0.0), (1003, 0.4), (20_011, 0.0), (140_011, 0.4)):
        h, w, t, dl = make(n, D, V, dtype, ignored, seed=n)
        _, lse, dh, dw = check(ops, h, w, t, dl)
        alone = [ops._CAPI_linear_cross_entropy_backward(dl, h, w, t, lse, -100, a, not a)[0 if a else 1] for a in (True, False)]
        assert torch.equal(alone[0], dh) and torch.equal(alone[1], dw)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("ignored", [0.3, 0.97, 1.0])
def test_ignored_rows(ops, dtype, ignored):
    h, w, t, dl = make(300, 96, 700, dtype, ignored)
    clean = check(ops, h, w, t, dl)
    bad = h.clone()
    bad[t == -100] = float("nan")                                     # what stands in an ignored row reaches nothing
    bad[:, 3][t == -100] = float("inf")
    dl2 = torch.where(t == -100, float("inf"), dl)
    loss, lse = ops._CAPI_linear_cross_entropy(bad, w, t, -100)
    dh, dw = ops._CAPI_linear_cross_entropy_backward(dl2, bad, w, t, lse, -100, True, True)
    assert all(torch.equal(p, q) for p, q in zip(clean, (loss, lse, dh, dw)))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("pad,wpad", [(1, 0), (8, 0), (0, 1), (0, 8), (3, 5)])
def test_strides(ops, dtype, pad, wpad):
    check(ops, *make(150, 104, 333, dtype, 0.1, pad=pad, wpad=wpad))
    h, w, t, dl = make(150, 104, 333, dtype, 0.1)
    base = ops._CAPI_linear_cross_entropy(h, w, t, -100)
    for hh, ww in ((h.t().contiguous().t(), w), (h, w.t().contiguous().t())):
        assert all(torch.equal(p, q) for p, q in zip(base, ops._CAPI_linear_cross_entropy(hh, ww, t, -100)))
    flat = torch.cat([w.reshape(-1)[:1], w.reshape(-1)])[1:].view(333, 104)   # a weight that begins off 16 bytes
    assert all(torch.equal(p, q) for p, q in zip(base, ops._CAPI_linear_cross_entropy(h, flat, t, -100)))


@pytest.mark.parametrize("dtype", TYPES)
def test_sharp_and_flat_rows(ops, dtype):
    check(ops, *make(140, 64, 900, dtype, scale=40.0))                # logits to +-150: exponentials that under- and overflow
    h, w, t, dl = make(140, 64, 900, dtype)
    w.zero_()                                                         # all logits equal
    loss, lse, dh, dw = check(ops, h, w, t, dl)
    assert (loss - math.log(900)).abs().max() <= 1e-5
    check(ops, *make(140, 64, 900, dtype)[:3], torch.zeros(140, device="cuda"))
    check(ops, *make(140, 64, 900, dtype)[:3], torch.full((140,), 1e-6, device="cuda"))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_classes_out_of_reach(ops, dtype):
    """Classes switched off by a logit of minus infinity or the type's lowest value have probability and gradient zero."""
    for low in (-float("inf"), torch.finfo(dtype).min):
        h, w, t, dl = make(70, 32, 400, dtype)
        h, w = h.clone(), w.clone()
        h[:, 0], w[:, 0] = 1.0, 0.0
        w[300:, 0] = low
        w[300:, 1:] = 0.0
        t = t % 300
        loss, lse = ops._CAPI_linear_cross_entropy(h, w, t, -100)
        want_loss, want_lse = ops._CAPI_linear_cross_entropy(h, w[:300].contiguous(), t, -100)
        assert torch.allclose(lse, want_lse, rtol=1e-6, atol=1e-6) and torch.allclose(loss, want_loss, rtol=1e-6, atol=1e-6)
        _, dw = ops._CAPI_linear_cross_entropy_backward(dl, h, w, t, lse, -100, False, True)
        assert (dw[300:] == 0).all()


def test_a_row_that_is_no_number_stays_alone(ops):
    for dtype in TYPES:
        h, w, t, dl = make(200, 48, 500, dtype)
        loss, lse = ops._CAPI_linear_cross_entropy(h, w, t, -100)
        bad = h.clone()
        bad[77, 5] = float("nan")
        l2, e2 = ops._CAPI_linear_cross_entropy(bad, w, t, -100)
        rows = torch.arange(200, device="cuda") != 77
        assert torch.equal(loss[rows], l2[rows]) and l2[77].isnan() and e2[77].isnan()
        dh, _ = ops._CAPI_linear_cross_entropy_backward(dl, bad, w, t, e2, -100, True, False)
        want, _ = ops._CAPI_linear_cross_entropy_backward(dl, h, w, t, lse, -100, True, False)
        assert torch.equal(dh[rows], want[rows]) and dh[77].isnan().all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_id_types_and_ignore_index(ops, dtype):
    h, w, t, dl = make(90, 40, 300, dtype, 0.2)
    base = check(ops, h, w, t, dl)
    assert all(torch.equal(p, q) for p, q in zip(base, check(ops, h, w, t.int(), dl)))
    t2 = torch.where(t == -100, 7, torch.where(t == 7, 8, t))         # an index inside the vocabulary
    check(ops, h, w, t2, dl, ignore=7)


def test_targets_out_of_range(ops):
    h, w, t, dl = make(64, 32, 100, torch.bfloat16)
    for wrong in (100, -1, 1 << 40):
        bad = t.clone()
        bad[9] = wrong
        loss, lse = ops._CAPI_linear_cross_entropy(h, w, bad, -100)
        torch.cuda.synchronize()
        with pytest.raises(RuntimeError, match="out-of-range"):      # noticed by the next call
            ops._CAPI_linear_cross_entropy(h, w, t, -100)
        assert loss[9] == 0 and lse[9] == 0 and loss.isfinite().all()
    ops._CAPI_linear_cross_entropy(h, w, t, -100)


@pytest.mark.parametrize("dtype", TYPES)
def test_no_rows_and_wanted_gradients(ops, dtype):
    h, w, t, dl = make(0, 32, 50, dtype)
    loss, lse = ops._CAPI_linear_cross_entropy(h, w, t, -100)
    dh, dw = ops._CAPI_linear_cross_entropy_backward(dl, h, w, t, lse, -100, True, True)
    assert loss.shape == lse.shape == (0,) and dh.shape == (0, 32) and dw.shape == (50, 32) and (dw == 0).all()
    h, w, t, dl = make(160, 72, 310, dtype)
    _, lse = ops._CAPI_linear_cross_entropy(h, w, t, -100)
    dh, dw = ops._CAPI_linear_cross_entropy_backward(dl, h, w, t, lse, -100, True, True)
    a, none = ops._CAPI_linear_cross_entropy_backward(dl, h, w, t, lse, -100, True, False)
    assert torch.equal(a, dh) and none.numel() == 0
    none, b = ops._CAPI_linear_cross_entropy_backward(dl, h, w, t, lse, -100, False, True)
    assert torch.equal(b, dw) and none.numel() == 0


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("n,D,V", [(1024, 128, 60_001), (4096, 192, 9000), (20_000, 64, 3000), (33, 512, 200_000)])
def test_many_pieces_and_same_bits_again(ops, dtype, n, D, V):
    args = make(n, D, V, dtype, 0.1)
    first = check(ops, *args)
    h, w, t, dl = args
    for _ in range(2):
        loss, lse = ops._CAPI_linear_cross_entropy(h, w, t, -100)
        again = (loss, lse) + tuple(ops._CAPI_linear_cross_entropy_backward(dl, h, w, t, lse, -100, True, True))
        assert all(torch.equal(p, q) for p, q in zip(first, again))


def test_autograd_against_the_formula_and_differences(pkg, ops):
    h, w, t, _ = make(30, 24, 65, torch.float32, 0.3)
    for reduction in ("mean", "sum", "none"):
        a, b = h.clone().requires_grad_(), w.clone().requires_grad_()
        out = pkg.linear_cross_entropy(a, b, t, reduction=reduction)
        ha, wb = h.double().requires_grad_(), w.double().requires_grad_()
        ref = torch.nn.functional.cross_entropy(ha @ wb.t(), t, ignore_index=-100, reduction=reduction)
        weight = torch.linspace(0.5, 2.0, out.numel(), device="cuda").view(out.shape)
        out.backward(weight)
        ref.backward(weight.double())
        for got, want in ((out, ref), (a.grad, ha.grad), (b.grad, wb.grad)):
            # 24 products and 65 classes (30 rows): under 200 roundings of sums whose terms are below 50 in all
            assert (got.double() - want).abs().max().item() <= 200 * U * 50
    a, b = h.clone().requires_grad_(), w.clone().requires_grad_()
    pkg.linear_cross_entropy(a, b, t).backward()
    g = torch.Generator(device="cuda").manual_seed(3)

    def f(hh, ww):
        return torch.nn.functional.cross_entropy(hh @ ww.t(), t, ignore_index=-100)
    for leaf, i in ((a, 0), (b, 1)):
        d = torch.randn(leaf.shape, device="cuda", generator=g, dtype=torch.float64)
        x = [h.double(), w.double()]
        up = f(*[v + 1e-6 * d if i == j else v for j, v in enumerate(x)])
        down = f(*[v - 1e-6 * d if i == j else v for j, v in enumerate(x)])
        terms = leaf.grad.double() * d
        assert abs(terms.sum().item() - ((up - down) / 2e-6).item()) <= 2e3 * U * terms.abs().sum().item() + 1e-7
    assert pkg.linear_cross_entropy(h, w, torch.full_like(t, -100)).isnan()
    assert pkg.linear_cross_entropy(h, w, torch.full_like(t, -100), reduction="sum") == 0


def test_other_stream(ops):
    h, w, t, dl = make(700, 128, 5000, torch.bfloat16)
    loss, lse = ops._CAPI_linear_cross_entropy(h, w, t, -100)
    want = ops._CAPI_linear_cross_entropy_backward(dl, h, w, t, lse, -100, True, True)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        l2, e2 = ops._CAPI_linear_cross_entropy(h, w, t, -100)
        got = ops._CAPI_linear_cross_entropy_backward(dl, h, w, t, e2, -100, True, True)
    s.synchronize()
    assert torch.equal(loss, l2) and all(torch.equal(p, q) for p, q in zip(want, got))


def test_offsets_beyond_32_bits(ops):
    D, V = 1024, 2_200_000                                            # 2.25e9 elements of the weight
    h, _, _, dl = make(3, D, 2, torch.bfloat16)
    w = torch.zeros((V, D), dtype=torch.bfloat16, device="cuda")
    w[-1] = h[1] / 16
    t = torch.tensor([V - 1, V - 1, 0], device="cuda")
    s = h.double() @ w[-1].double()
    lse = torch.log((V - 1) + torch.exp(s))
    loss, got = ops._CAPI_linear_cross_entropy(h, w, t, -100)
    want = lse - torch.stack([s[0], s[1], 0 * s[2]])
    # the logit's products, and V equal terms added in chains of at most V / 100
    tol = 2 * (D + 8) * U * (h.double().abs() @ w[-1].double().abs()).max() + V / 100 * U
    assert (got.double() - lse).abs().max() <= tol and (loss.double() - want).abs().max() <= 2 * tol
    _, dw = ops._CAPI_linear_cross_entropy_backward(dl, h, w, t, got, -100, False, True)
    p = torch.exp(s - lse)
    ref = (dl.double() * (p - torch.tensor([1.0, 1.0, 0.0], device="cuda"))) @ h.double()
    assert (dw[-1].double() - ref).abs().max() <= 2.0 ** -7 * (dl.double() @ h.double().abs()).max()


def test_refusals(ops):
    h, w, t, dl = make(8, 16, 20, torch.bfloat16)
    lse = torch.zeros(8, device="cuda")
    for args, why in (((h.double(), w.double(), t, -100), "float32"), ((h, w.half(), t, -100), "share one type"),
                      ((h, w[:, :15], t, -100), "one length"), ((h[0], w, t, -100), "matrices"),
                      ((h, w, t[:7], -100), "one id for each row"), ((h, w, t.float(), -100), "int32 or int64"),
                      ((h, w.cpu(), t, -100), "must be on"), ((h, w[:0], t, -100), "at least one class")):
        with pytest.raises(RuntimeError, match=why):
            ops._CAPI_linear_cross_entropy(*args)
    for gl, e in ((dl[:7], lse), (dl.double(), lse), (dl, lse.half()), (dl[:, None], lse)):
        with pytest.raises(RuntimeError, match="one value for each row"):
            ops._CAPI_linear_cross_entropy_backward(gl, h, w, t, e, -100, True, True)
