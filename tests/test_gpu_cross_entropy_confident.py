"""Losses of rows that are right already: the target's logit stands far above the others, and the loss is the logarithm of a sum
just above one.

Rows have one element that is not zero, so a logit is one product of two 16-bit values and exact in 32 bits, and what is left
is the sum.  Its largest term is one, exactly; x = what the others add has their errors (differences of logits up to 30, rounded
to 2^-24 of themselves twice and times log2(e) in 32 bits, and 2^-22 of the exponential: 2^-18 of x in all), and each addition to a
sum that holds the one rounds to u = 2^-24: a term for every 128 classes, six within 32 of them, three to join groups of columns,
13 to join slices.  So a loss is never negative, and of one class it is zero."""
import pytest
import torch

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


def rows(n, V, top, dtype):
    g = torch.Generator(device="cuda").manual_seed(n + V)
    h, w = torch.zeros(n, 72, device="cuda"), torch.zeros(V, 72, device="cuda")
    h[:, 5] = 1 + torch.rand(n, device="cuda", generator=g)
    w[:, 5] = top - 8 - torch.randint(0, 16, (V,), device="cuda", generator=g) / 2
    at = (V * 2) // 3
    w[at, 5] = top
    return h.bfloat16().to(dtype), w.to(dtype), torch.full((n,), at, dtype=torch.int64, device="cuda")


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("n", [1, 32, 33, 300])
@pytest.mark.parametrize("V", [1, 2, 50, 128, 129, 500, 5000])
@pytest.mark.parametrize("top", [20.0, 50.0, 100.0])
def test_losses(ops, n, V, top, dtype):
    h, w, t = rows(n, V, top, dtype)
    s = h.double() @ w.double().t()
    x = torch.exp(s - s.gather(1, t[:, None])).sum(1) - 1
    loss, lse = ops._CAPI_linear_cross_entropy(h, w, t, -100)
    assert (loss >= 0).all()
    if V == 1:
        assert (loss == 0).all()
    tol = (V / 128 + 14 + (13 if V > 256 else 0)) * U + x * 2.0 ** -18
    assert ((loss.double() - torch.log1p(x)).abs() <= tol).all()
    assert ((lse.double() - torch.logsumexp(s, 1)).abs() <= tol + U * lse.double().abs()).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_the_same_rows_beside_one_another(ops, dtype):
    """As many rows as take one kernel and one more, which take another: the loss of a row hardly changes."""
    h, w, t = rows(33, 700, 50.0, dtype)
    one, _ = ops._CAPI_linear_cross_entropy(h, w, t, -100)
    other, _ = ops._CAPI_linear_cross_entropy(h[:32].contiguous(), w, t[:32], -100)
    assert (one[:32] - other).abs().max() <= 64 * U


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("n", [1, 32, 33, 300])
@pytest.mark.parametrize("V", [2, 50, 128, 129, 500])
@pytest.mark.parametrize("top", [20.0, 100.0])
def test_the_targets_entry_of_the_gradient(ops, pkg, n, V, top, dtype):
    """A column of the weight that only the target's class has, against a column of zeros of the rows: dh there is p - 1, out of one
    entry.  It has the loss's error, and two roundings to the type."""
    h, w, t = rows(n, V, top, dtype)
    w[t[0], 7] = 1.0
    s = h.double() @ w.double().t()
    x = torch.exp(s - s.gather(1, t[:, None])).sum(1) - 1
    h.requires_grad_()
    pkg.linear_cross_entropy(h, w, t, reduction="sum").backward()
    want = -x / (1 + x)
    r = {torch.float32: 8 * U, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}[dtype]
    tol = (V / 128 + 14 + (13 if V > 256 else 0)) * U + x * 2.0 ** -18 + 2 * r * want.abs() + 2.0 ** -24
    assert ((h.grad[:, 7].double() - want).abs() <= tol).all()
    # without the loss: lse and the logit in 32 bits, a rounding of each
    loss, lse = ops._CAPI_linear_cross_entropy(h.detach(), w, t, -100)
    dh, _ = ops._CAPI_linear_cross_entropy_backward(torch.ones(n, device="cuda"), h.detach(), w, t, lse, -100, True, False)
    assert ((dh[:, 7].double() - want).abs() <= tol + 2 * U * lse.double().abs() + 8 * U).all()


def test_a_loss_that_does_not_fit(ops):
    h, w, t = rows(8, 20, 20.0, torch.bfloat16)
    loss, lse = ops._CAPI_linear_cross_entropy(h, w, t, -100)
    for bad, why in ((loss[:7], "one value"), (loss.double(), "one value"), (loss[:, None], "one value"), (loss.cpu(), "must be on")):
        with pytest.raises(RuntimeError, match=why):
            ops._CAPI_linear_cross_entropy_backward(torch.ones(8, device="cuda"), h, w, t, lse, bad, -100, True, True)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_ignored_rows_with_the_loss_at_hand(ops, dtype):
    g = torch.Generator(device="cuda").manual_seed(0)
    for n in (20, 300):
        h, w = torch.randn(n, 40, device="cuda", generator=g).to(dtype), torch.randn(700, 40, device="cuda", generator=g).to(dtype)
        t = torch.randint(0, 700, (n,), device="cuda", generator=g)
        t[::3] = -100
        loss, lse = ops._CAPI_linear_cross_entropy(h, w, t, -100)
        dl = torch.ones(n, device="cuda")
        clean = ops._CAPI_linear_cross_entropy_backward(dl, h, w, t, lse, loss, -100, True, True)
        bad = h.clone()
        bad[::3] = float("nan")
        loss[::3] = float("nan")
        dl[::3] = float("inf")
        again = ops._CAPI_linear_cross_entropy_backward(dl, bad, w, t, lse, loss, -100, True, True)
        assert all(torch.equal(p, q) for p, q in zip(clean, again)) and (clean[0][::3] == 0).all()


def test_losses_changed_in_place(pkg):
    h, w, t = rows(40, 60, 20.0, torch.bfloat16)
    a, b = h.clone().requires_grad_(), h.clone().requires_grad_()
    loss = pkg.linear_cross_entropy(a, w, t, reduction="none")
    loss *= 2.0
    loss.sum().backward()
    (2.0 * pkg.linear_cross_entropy(b, w, t, reduction="none")).sum().backward()
    assert torch.equal(a.grad, b.grad)
