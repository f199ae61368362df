"""Layer norm, forward and backward, against the definition in 64 bits.

Tolerances follow from the arithmetic: u = 2^-24 is the unit roundoff of the sums.  A row's sums run over at most 64 values
a thread and 13 levels of a tree (wider rows: D / 256 values and 13 levels), each step off by u of the sum of magnitudes, so
mean and variance are within g = (80 + D / 256) u of theirs; a result in fewer bits is rounded once (r = 2^-8 or 2^-11)."""
import pytest
import torch

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
ROUND = {torch.float32: U, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
SHAPES = [(1, 1), (1, 7), (3, 2), (5, 16), (1000, 4), (257, 31), (64, 33), (31, 75), (100, 100), (9, 128), (33, 255), (17, 256),
          (1025, 257), (11, 600), (7, 1000), (5, 1024), (6, 2048), (3, 2051), (4, 4096), (2, 8192), (2, 8200), (3, 16384),
          (2, 16390), (2, 20001), (1, 40000)]


def make(n, D, dtype, ptype, pad=0, seed=0, shift=0.5):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = (torch.randn((n, D + pad), device="cuda", generator=g) * 1.5 + shift).to(dtype)[:, :D]
    dy = torch.randn((n, D + pad), device="cuda", generator=g).to(dtype)[:, :D]
    w = (torch.randn(D, device="cuda", generator=g) * 0.3 + 1.0).to(ptype)
    b = torch.randn(D, device="cuda", generator=g).to(ptype)
    return x, dy, w, b


def definition(x, w, b, eps):
    x = x.double()
    mean = x.mean(-1, keepdim=True)
    rstd = 1.0 / ((x - mean).square().mean(-1, keepdim=True) + eps).sqrt()
    h = (x - mean) * rstd
    return h * (1.0 if w is None else w.double()) + (0.0 if b is None else b.double()), mean, rstd, h


def check(x, dy, w, b, ops, eps=1e-5):
    D, n = x.shape[-1], x.numel() // x.shape[-1]
    g_u = (80 + D / 256) * U
    y, mean, rstd = ops._CAPI_layer_norm(x, w, b, eps)
    ry, rm, rr, rh = definition(x, w, b, eps)
    wd = torch.ones(D, device="cuda", dtype=torch.float64) if w is None else w.double()
    spread = x.double().abs().mean(-1, keepdim=True)
    # what an error of g_u in the mean does to the centred values, in units of the row's deviation
    off = 4 * g_u * (spread * rr + 1)
    assert ((mean.double().unsqueeze(-1) - rm).abs() <= g_u * spread + U * rm.abs()).all()
    assert ((rstd.double().unsqueeze(-1) / rr - 1).abs() <= off + 4 * U).all()
    tol = off * (rh.abs() + 1) * wd.abs() + 4 * U * ry.abs() + ROUND[x.dtype] * ry.abs() + 2.0 ** -25
    assert ((y.double() - ry).abs() <= tol).all()
    # backward
    dx, dw, db = ops._CAPI_layer_norm_backward(dy, x, w, mean, rstd, True, w is not None)
    d = dy.double()
    g = d * wd
    rdx = rr * (g - g.mean(-1, keepdim=True) - rh * (g * rh).mean(-1, keepdim=True))
    size = rr * (g.abs() + g.abs().mean(-1, keepdim=True) + rh.abs() * (g * rh).abs().mean(-1, keepdim=True))
    slack = rr * (1 + rh.abs()) * g.abs().mean(-1, keepdim=True)
    tol = (off + 2 * g_u) * (3 * size + 3 * slack) + ROUND[x.dtype] * rdx.abs() + 2.0 ** -25
    assert ((dx.double() - rdx).abs() <= tol).all()
    if w is not None:
        flat = lambda t: t.reshape(-1, D)  # noqa: E731
        for got, terms, more in ((dw, d * rh, (d.abs() * off * (rh.abs() + 1))), (db, d, 0 * d)):
            ref = flat(terms).sum(0)
            tol = (n + 16) * U * flat(terms.abs()).sum(0) + flat(more).sum(0) + ROUND[w.dtype] * ref.abs() + 2.0 ** -25
            assert ((got.double() - ref).abs() <= tol).all()
    return y, dx, dw, db


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("n,D", SHAPES)
def test_shapes(ops, n, D, dtype):
    check(*make(n, D, dtype, dtype), ops)


@pytest.mark.parametrize("D", [75, 100, 256, 4096, 20001])
@pytest.mark.parametrize("pad", [1, 8, 6])
@pytest.mark.parametrize("ptype", [torch.float32, torch.bfloat16])
def test_strides_and_parameter_types(ops, D, pad, ptype):
    check(*make(65, D, torch.bfloat16, ptype, pad), ops)
    x, dy, w, b = make(65, D, torch.float32, ptype, pad)
    check(x, dy.contiguous(), w, b, ops)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_without_parameters_and_other_layouts(ops, dtype):
    x, dy, w, b = make(24, 48, dtype, dtype)
    check(x, dy, None, None, ops)
    y0, _, _ = ops._CAPI_layer_norm(x, w, None, 1e-5)
    assert torch.equal(y0, ops._CAPI_layer_norm(x, w, torch.zeros_like(b), 1e-5)[0])
    y, m, r = ops._CAPI_layer_norm(x.view(2, 3, 4, 48), w, b, 1e-5)
    assert y.shape == (2, 3, 4, 48) and m.shape == r.shape == (2, 3, 4)
    assert torch.equal(y.view(24, 48), ops._CAPI_layer_norm(x, w, b, 1e-5)[0])
    t = x.t().contiguous().t()                                        # columns are the contiguous direction
    assert torch.equal(ops._CAPI_layer_norm(t, w, b, 1e-5)[0], ops._CAPI_layer_norm(x, w, b, 1e-5)[0])
    e = x[:1].expand(5, 48)                                           # the same row five times
    assert torch.equal(ops._CAPI_layer_norm(e, w, b, 1e-5)[0], ops._CAPI_layer_norm(e.contiguous(), w, b, 1e-5)[0])
    v = x[3]                                                          # one row, no leading dimension
    y, m, r = ops._CAPI_layer_norm(v, w, b, 1e-5)
    assert y.shape == (48,) and m.shape == () and torch.equal(y, ops._CAPI_layer_norm(x, w, b, 1e-5)[0][3])
    off = torch.randn(48 * 8 + 1, device="cuda").to(dtype)[1:].view(8, 48)  # not 16-byte aligned
    check(off, off.flip(0), w, b, ops)


def test_values_at_the_edges(ops):
    w, b = torch.ones(64, device="cuda"), torch.zeros(64, device="cuda")
    x = torch.full((4, 64), 3.25, device="cuda")                      # a row without spread: the eps alone
    y, m, r = ops._CAPI_layer_norm(x, w, b, 1e-5)
    assert (y == 0).all() and (m == 3.25).all()
    check(*make(16, 256, torch.float32, torch.float32, shift=1000.0), ops)   # spread far below the mean
    x, dy, w, b = make(40, 64, torch.float32, torch.float32)
    clean = ops._CAPI_layer_norm(x, w, b, 1e-5)
    bad = x.clone()
    bad[7, 3], bad[20, 0] = float("nan"), float("inf")
    y, m, r = ops._CAPI_layer_norm(bad, w, b, 1e-5)
    rows = torch.ones(40, dtype=torch.bool, device="cuda")
    rows[7] = rows[20] = False
    assert torch.equal(y[rows], clean[0][rows]) and y[7].isnan().all() and y[20].isnan().all()
    dx, _, _ = ops._CAPI_layer_norm_backward(dy, bad, w, m, r, True, True)
    assert torch.equal(dx[rows], ops._CAPI_layer_norm_backward(dy, x, w, clean[1], clean[2], True, True)[0][rows])


def test_no_rows(ops):
    x, w = torch.empty(0, 32, device="cuda"), torch.ones(32, device="cuda")
    y, m, r = ops._CAPI_layer_norm(x, w, w, 1e-5)
    assert y.shape == (0, 32) and m.numel() == 0
    dx, dw, db = ops._CAPI_layer_norm_backward(x, x, w, m, r, True, True)
    assert dx.shape == (0, 32) and (dw == 0).all() and (db == 0).all() and dw.shape == (32,)


def test_wanted_gradients(ops):
    x, dy, w, b = make(50, 96, torch.float32, torch.float32)
    _, m, r = ops._CAPI_layer_norm(x, w, b, 1e-5)
    dx, dw, db = ops._CAPI_layer_norm_backward(dy, x, w, m, r, True, True)
    only, none, _ = ops._CAPI_layer_norm_backward(dy, x, w, m, r, True, False)
    assert torch.equal(only, dx) and none.numel() == 0
    none, dw2, db2 = ops._CAPI_layer_norm_backward(dy, x, w, m, r, False, True)
    assert none.numel() == 0 and torch.equal(dw, dw2) and torch.equal(db, db2)


@pytest.mark.parametrize("D", [20, 100, 256, 1024, 4096])
@pytest.mark.parametrize("rows", [8, 16, 32, 64, 128, 256, 512, 1024])
def test_about_one_cluster_of_rows(ops, rows, D):
    for n in (rows - 1, rows, rows + 1):
        check(*make(n, D, torch.bfloat16, torch.float32), ops)
        check(*make(n, D, torch.float32, torch.float32, pad=1), ops)


@pytest.mark.parametrize("n,D", [(5000, 100), (3001, 1024), (700, 4096)])
def test_same_bits_again(ops, n, D):
    x, dy, w, b = make(n, D, torch.bfloat16, torch.float32)
    _, m, r = ops._CAPI_layer_norm(x, w, b, 1e-5)
    first = ops._CAPI_layer_norm_backward(dy, x, w, m, r, True, True)
    for _ in range(3):
        assert all(torch.equal(p, q) for p, q in zip(first, ops._CAPI_layer_norm_backward(dy, x, w, m, r, True, True)))


def test_autograd_against_the_formula_and_differences(pkg, ops):
    x, dy, w, b = make(6, 40, torch.float32, torch.float32)
    leaves = [t.clone().requires_grad_() for t in (x, w, b)]
    pkg.layer_norm(*leaves, eps=1e-3).backward(dy)
    direct = ops._CAPI_layer_norm_backward(dy, x, w, *ops._CAPI_layer_norm(x, w, b, 1e-3)[1:], True, True)
    assert all(torch.equal(t.grad, d) for t, d in zip(leaves, direct))
    # central differences of the definition in 64 bits along random directions: step 1e-6, error below 1e-8
    g = torch.Generator(device="cuda").manual_seed(5)
    for i, leaf in enumerate(leaves):
        for _ in range(3):
            d = torch.randn(leaf.shape, device="cuda", generator=g, dtype=torch.float64)
            f = []
            for sign in (1e-6, -1e-6):
                args = [t.detach().double() for t in leaves]
                args[i] = args[i] + sign * d
                f.append((definition(*args, 1e-3)[0] * dy.double()).sum())
            want = ((f[0] - f[1]) / 2e-6).item()
            terms = leaf.grad.double() * d
            assert abs(terms.sum().item() - want) <= 2e3 * U * terms.abs().sum().item() + 1e-6


def test_other_stream(ops):
    x, dy, w, b = make(4000, 512, torch.bfloat16, torch.bfloat16)
    want = ops._CAPI_layer_norm(x, w, b, 1e-5)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        got = ops._CAPI_layer_norm(x, w, b, 1e-5)
    s.synchronize()
    assert all(torch.equal(p, q) for p, q in zip(want, got))


def test_offsets_beyond_32_bits(ops):
    n, D = 2_200_000, 1000                                            # 2.2e9 elements
    x = torch.zeros((n, D), dtype=torch.bfloat16, device="cuda")
    tail = torch.randn(5, D, device="cuda").bfloat16()
    x[-5:] = tail
    w, b = torch.ones(D, device="cuda"), torch.zeros(D, device="cuda")
    y, m, r = ops._CAPI_layer_norm(x, w, b, 1e-5)
    small = ops._CAPI_layer_norm(tail, w, b, 1e-5)
    assert torch.equal(y[-5:], small[0]) and torch.equal(m[-5:], small[1]) and (y[:5] == 0).all()
    dx, dw, db = ops._CAPI_layer_norm_backward(x, x, w, m, r, True, True)
    sd = ops._CAPI_layer_norm_backward(tail, tail, w, small[1], small[2], True, True)
    assert torch.equal(dx[-5:], sd[0]) and torch.allclose(dw, sd[1], rtol=1e-5, atol=1e-5)


def test_refusals(ops):
    x, w = torch.zeros(4, 8, device="cuda"), torch.ones(8, device="cuda")
    m = torch.zeros(4, device="cuda")
    for args, why in (((x.double(), None, None, 1e-5), "float32"), ((x, w[:7], None, 1e-5), "elements of a row"),
                      ((x, w, w.bfloat16(), 1e-5), "shape and type"), ((x, None, w, 1e-5), "needs a weight"),
                      ((x, w.cpu(), None, 1e-5), "must be on"), ((x[:, :0], None, None, 1e-5), "at least one element"),
                      ((x, w, w, -1.0), "eps")):
        with pytest.raises(RuntimeError, match=why):
            ops._CAPI_layer_norm(*args)
    for args, why in (((x[:3], x, w, m, m, True, True), "shape and type"), ((x.half(), x, w, m, m, True, True), "shape and type"),
                      ((x, x, None, m, m, True, True), "without a weight"), ((x, x, w, m[:3], m, True, True), "mean and rstd"),
                      ((x, x, w, m.double(), m, True, True), "mean and rstd")):
        with pytest.raises(RuntimeError, match=why):
            ops._CAPI_layer_norm_backward(*args)
