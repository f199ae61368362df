"""AdamW where some tensors have no gradient for a while, against torch's AdamW in 64 bits, which counts a tensor's own steps."""
import pytest
import torch

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("late", [1, 9, 300])
def test_a_gradient_that_comes_late(pkg, bits, late):
    """The first step of a tensor is lr against the gradient's sign, whenever it comes."""
    g = torch.Generator(device="cuda").manual_seed(late)
    p = [torch.randn(n, device="cuda", generator=g) for n in (300, 1000)]
    first = p[1].clone()
    opt = pkg.AdamW(p, lr=1e-2, bits=bits, weight_decay=0.0)
    for _ in range(late):
        opt.step([torch.randn(300, device="cuda", generator=g), None])
    assert torch.equal(first, p[1])
    grad = torch.randn(1000, device="cuda", generator=g)
    opt.step([torch.randn(300, device="cuda", generator=g), grad])
    # m / sqrt(v) is the sign but for eps = 1e-8 of a gradient that is hardly below 1e-4, and some ten roundings; the sum's own
    moved = first.double() - p[1].double()
    assert ((moved - 1e-2 * grad.double().sign()).abs() <= 1e-2 * (1e-8 / grad.double().abs() + 16 * U) + U * 8).all()


def test_gradients_that_come_and_go_like_torch(pkg):
    g = torch.Generator(device="cuda").manual_seed(1)
    p = [torch.randn(n, device="cuda", generator=g) for n in (300, 40, 1000, 7)]
    ref = [x.double().requires_grad_() for x in p]
    opt, want = pkg.AdamW(p, lr=1e-2, weight_decay=0.05), torch.optim.AdamW(ref, lr=1e-2, weight_decay=0.05)
    for step in range(40):
        grads = [torch.randn(x.shape, device="cuda", generator=g) if (step >> i) % 2 == 0 or i == 0 else None for i, x in enumerate(p)]
        for y, d in zip(ref, grads):
            y.grad = None if d is None else d.double()
        opt.step(grads)
        want.step()
    for x, y in zip(p, ref):
        # 40 steps of at most some 3e-2, each within a few dozen roundings, added to values below 8 with a rounding of 2^-22 each
        assert (x.double() - y.detach()).abs().max() <= 40 * (3e-2 * 64 * U + 2.0 ** -22)
