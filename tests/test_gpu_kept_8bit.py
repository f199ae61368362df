"""Rows kept in 8 bits and the weight's gradient from them, against the definition.

Codes, scales and values are IEEE arithmetic in 32 bits, operation by operation, and have to be equal.  The gradient: the products of
16-bit operands (the values rounded to the type) are exact in 32 bits, and every addition of n of them, in any order, is off by at most
2^-23 of the sum of magnitudes so far (a truncated one; a rounded one 2^-24): (n + 64) 2^-23 sum |g||v|, plus one rounding of the result."""
import pytest
import torch

pytestmark = pytest.mark.gpu
ROUND = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
TINY = {torch.float32: 2.0 ** -126, torch.bfloat16: 2.0 ** -126, torch.float16: 2.0 ** -24}
TYPES = [torch.float32, torch.bfloat16, torch.float16]


def rows(n, D, dtype, pad=0, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn((n, D + pad), device="cuda", generator=g) * torch.exp(torch.randn((n, 1), device="cuda", generator=g))
    return x.to(dtype)[:, :D]


def definition(x):
    n, D = x.shape
    groups = -(-D // 128)
    r = torch.nn.functional.pad(x.float(), (0, groups * 128 - D)).view(n, groups, 128)
    top = r.abs().amax(2, keepdim=True)
    by = torch.where(top > 0, torch.div(torch.full_like(top, 127.0), top), 0.0)
    codes = torch.round(r * by).clamp(-127, 127)
    scales = torch.div(top, torch.full_like(top, 127.0))
    return codes.view(n, -1)[:, :D].to(torch.int8), scales[:, :, 0], (codes * scales).view(n, -1)[:, :D]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,D,pad", [(1, 1, 0), (3, 7, 0), (5, 8, 0), (100, 100, 0), (33, 75, 6), (17, 127, 1), (9, 128, 0), (9, 129, 0),
                                     (40, 256, 8), (7, 1000, 0), (3, 4096, 0), (2, 5001, 3), (20000, 16, 0), (3001, 384, 0)])
def test_codes_and_values(ops, n, D, pad, dtype):
    x = rows(n, D, dtype, pad)
    codes, scales = ops._CAPI_keep_8bit(x)
    want_codes, want_scales, want = definition(x)
    assert torch.equal(codes, want_codes) and torch.equal(scales, want_scales)
    for t in TYPES:
        assert torch.equal(ops._CAPI_kept_8bit_values(codes, scales, t), want.to(t))
    # within half a step of what was kept (and its rounding in 32 bits)
    top = torch.repeat_interleave(scales * 127, 128, 1)[:, :D]
    assert ((want.double() - x.double()).abs() <= top.double() * (0.5 / 127 + 2.0 ** -22)).all()


@pytest.mark.parametrize("dtype", TYPES)
def test_special_rows(ops, dtype):
    x = rows(12, 300, dtype)
    x[0] = 0.0
    x[1, :128], x[1, 5] = 0.0, -0.0
    x[2, 130], x[3, 0], x[4, 299] = float("nan"), float("inf"), float("-inf")
    x[5] = torch.finfo(dtype).max
    x[6] = torch.finfo(dtype).smallest_normal
    codes, scales = ops._CAPI_keep_8bit(x)
    v = ops._CAPI_kept_8bit_values(codes, scales, torch.float32)
    assert (v[0] == 0).all() and (scales[0] == 0).all() and (v[1, :128] == 0).all()
    # the groups that hold them are lost, the others are not
    groups = [(2, 1), (3, 0), (4, 2)]
    want_codes, want_scales, want = definition(x)
    for r in range(12):
        for g in range(3):
            c = slice(g * 128, min(300, g * 128 + 128))
            if (r, g) in groups:
                assert not scales[r, g].isfinite() and not v[r, c].isfinite().any()
            elif r != 6:  # (127 / a is no finite number there)
                assert torch.equal(v[r, c], want[r, c])
    # the largest number of 32 bits: 127 rn(max / 127) is max (1 + e) with |e| <= 2^-24, which for e > 0 is infinity; of 16 bits it is a number
    assert torch.equal(v[5], want[5]) and (dtype == torch.float32 or ((v[5] / x[5].float() - 1).abs() <= 2.0 ** -23).all())
    assert v[6].isfinite().all()


def check_grad(ops, n, O, D, dtype, pad=0, codes_pad=0, seed=0, bias=True):
    g = torch.Generator(device="cuda").manual_seed(seed)
    grad = torch.randn((n, O + pad), device="cuda", generator=g).to(dtype)[:, :O]
    codes, scales = ops._CAPI_keep_8bit(rows(n, D, torch.float32, seed=seed + 1))
    if codes_pad:
        wide = torch.full((n, D + codes_pad), 77, dtype=torch.int8, device="cuda")
        wide[:, :D] = codes
        codes = wide[:, :D]
    dw, db = ops._CAPI_kept_8bit_weight_grad(grad, codes, scales, bias)
    v = ops._CAPI_kept_8bit_values(codes, scales, dtype).double()
    d = grad.double()
    want, size = d.t() @ v, d.abs().t() @ v.abs()
    tol = (n + 64) * 2.0 ** -23 * size + ROUND[dtype] * want.abs() + TINY[dtype]
    assert ((dw.double() - want).abs() <= tol).all(), ((dw.double() - want).abs() / tol).amax().item()
    # what many additions are off by goes with the root of their number: a tile or a share of the rows left out would be far beyond it
    rms = ((dw.double() - want - 0.0).square().mean().sqrt() / want.square().mean().sqrt().clamp_min(1e-30)).item()
    assert rms <= ROUND[dtype] + 1e-4, rms
    if bias:
        want = d.sum(0)
        assert ((db.double() - want).abs() <= (n + 64) * 2.0 ** -23 * d.abs().sum(0) + ROUND[dtype] * want.abs() + TINY[dtype]).all()
    else:
        assert db.numel() == 0
    return grad, codes, scales, dw, db


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,O,D", [(1, 1, 1), (2, 3, 5), (63, 47, 75), (64, 64, 64), (65, 128, 128), (300, 129, 257), (1000, 8, 100),
                                   (777, 256, 256), (2000, 47, 256), (129, 300, 1000), (5000, 2, 8), (40000, 16, 24)])
def test_weight_gradient(ops, n, O, D, dtype):
    check_grad(ops, n, O, D, dtype, seed=n)
    check_grad(ops, n, O, D, dtype, pad=3, codes_pad=5, seed=n + 1, bias=False)


@pytest.mark.parametrize("n,O,D", [(4096, 1024, 512), (100_000, 172, 100), (3000, 700, 3000)])
def test_larger_weight_gradients(ops, n, O, D):
    check_grad(ops, n, O, D, torch.bfloat16)
    check_grad(ops, n, O, D, torch.float16, pad=8)


def test_the_same_inputs_give_the_same_bits(ops):
    grad, codes, scales, dw, db = check_grad(ops, 50_000, 100, 200, torch.bfloat16)
    for _ in range(3):
        again = ops._CAPI_kept_8bit_weight_grad(grad, codes, scales, True)
        assert torch.equal(again[0], dw) and torch.equal(again[1], db)


def test_values_behind_the_rows_do_not_count(ops):
    """Rows of a longer buffer, columns of a wider one, whose rest holds anything."""
    n, O, D = 333, 40, 90
    grad, codes, scales, dw, db = check_grad(ops, n, O, D, torch.bfloat16)
    g2 = torch.full((n + 50, O + 24), float("nan"), device="cuda", dtype=torch.bfloat16)
    c2 = torch.full((n + 50, D + 38), -128, device="cuda", dtype=torch.int8)
    s2 = torch.full((n + 50, 1), float("nan"), device="cuda")
    g2[:n, :O], c2[:n, :D], s2[:n] = grad, codes, scales
    got = ops._CAPI_kept_8bit_weight_grad(g2[:n, :O], c2[:n, :D], s2[:n], True)
    assert torch.equal(got[0], dw) and torch.equal(got[1], db)


def test_no_rows(ops):
    x = torch.zeros(0, 200, device="cuda", dtype=torch.bfloat16)
    codes, scales = ops._CAPI_keep_8bit(x)
    assert codes.shape == (0, 200) and scales.shape == (0, 2)
    assert ops._CAPI_kept_8bit_values(codes, scales, torch.float16).shape == (0, 200)
    dw, db = ops._CAPI_kept_8bit_weight_grad(torch.zeros(0, 5, device="cuda"), codes, scales, True)
    assert dw.shape == (5, 200) and (dw == 0).all() and (db == 0).all()


def test_linear(pkg, ops):
    g = torch.Generator(device="cuda").manual_seed(2)
    for dtype in TYPES:
        x = torch.randn((3, 50, 60), device="cuda", generator=g).to(dtype).requires_grad_()
        w = torch.randn((20, 60), device="cuda", generator=g).to(dtype).requires_grad_()
        b = torch.randn(20, device="cuda", generator=g).to(dtype).requires_grad_()
        dy = torch.randn((3, 50, 20), device="cuda", generator=g).to(dtype)
        y = pkg.linear_8bit(x, w, b)
        assert torch.equal(y, torch.nn.functional.linear(x, w, b))
        y.backward(dy)
        codes, scales = pkg.keep_8bit(x.detach().view(150, 60))
        want = ops._CAPI_kept_8bit_weight_grad(dy.view(150, 20), codes, scales, True)
        assert torch.equal(w.grad, want[0]) and torch.equal(b.grad, want[1])
        assert torch.equal(x.grad, (dy.view(150, 20) @ w.detach()).view(3, 50, 60))
        # near the gradient of the rows themselves: half a step of 127 for each value, random in sign
        exact = dy.double().view(150, 20).t() @ x.detach().double().view(150, 60)
        assert (w.grad.double() - exact).norm() <= (0.5 / 127 * 3.5 + 2 * ROUND[dtype]) * exact.norm()
        # what is kept: codes, scales and the weight
        saved = []
        with torch.autograd.graph.saved_tensors_hooks(lambda t: saved.append(t) or t, lambda t: t):
            pkg.linear_8bit(x, w, b)
        assert sorted((tuple(t.shape), t.dtype) for t in saved) == sorted([((20, 60), dtype), ((150, 60), torch.int8), ((150, 1), torch.float32)],
                                                                            key=lambda p: p[0]) or len(saved) == 3
        assert not any(t.dtype == dtype and t.numel() == x.numel() for t in saved)
        # frozen weights keep nothing
        saved.clear()
        with torch.autograd.graph.saved_tensors_hooks(lambda t: saved.append(t) or t, lambda t: t):
            pkg.linear_8bit(x, w.detach(), b).sum().backward()
        assert len(saved) == 1
    with pytest.raises(ValueError, match="one type"):
        pkg.linear_8bit(x.float(), w)


def test_recorded_and_on_another_stream(ops):
    x, grad = rows(3000, 200, torch.bfloat16), rows(3000, 60, torch.bfloat16, seed=3)

    def both():
        codes, scales = ops._CAPI_keep_8bit(x)
        return (ops._CAPI_kept_8bit_values(codes, scales, torch.bfloat16), *ops._CAPI_kept_8bit_weight_grad(grad, codes, scales, True))

    both()
    torch.cuda.synchronize()
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            graphs.append((g, both()))
    x.mul_(-0.5)
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
    x = torch.zeros(4, 130, device="cuda")
    codes, scales = ops._CAPI_keep_8bit(x)
    with pytest.raises(RuntimeError, match="rows of at least one element"):
        ops._CAPI_keep_8bit(x[0])
    with pytest.raises(RuntimeError, match="float32, bfloat16 or float16"):
        ops._CAPI_keep_8bit(x.double())
    for c, s, text in ((codes.float(), scales, "int8 rows"), (codes[0], scales, "int8 rows"), (codes, scales[:, :1], "every 128 codes"),
                       (codes, scales.half(), "every 128 codes"), (codes, scales[:3], "every 128 codes"), (codes, scales.cpu(), "must be on")):
        with pytest.raises(RuntimeError, match=text):
            ops._CAPI_kept_8bit_values(c, s, torch.float32)
        with pytest.raises(RuntimeError, match=text):
            ops._CAPI_kept_8bit_weight_grad(x, c, s, True)
    with pytest.raises(RuntimeError, match="the type must be"):
        ops._CAPI_kept_8bit_values(codes, scales, torch.float64)
    for g, text in ((x[:3], "one row for each"), (x[0], "one row for each"), (x.double(), "float32, bfloat16 or float16"), (x.cpu(), "must be on")):
        with pytest.raises(RuntimeError, match=text):
            ops._CAPI_kept_8bit_weight_grad(g, codes, scales, False)
