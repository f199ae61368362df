"""linear_8bit where nothing will ask for a gradient: nothing is kept, and nothing is quantised on the way."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("mode", [torch.no_grad, torch.inference_mode])
def test_without_gradients(pkg, mode):
    n, D, O = 100_000, 256, 8
    x = torch.randn(n, D, device="cuda", dtype=torch.bfloat16)
    w = torch.randn(O, D, device="cuda", dtype=torch.bfloat16).requires_grad_()
    b = torch.randn(O, device="cuda", dtype=torch.bfloat16).requires_grad_()
    with mode():
        pkg.linear_8bit(x, w, b)  # (workspaces of torch's product)
        torch.cuda.synchronize()
        before = torch.cuda.memory_allocated()
        torch.cuda.reset_peak_memory_stats()
        y = pkg.linear_8bit(x, w, b)
        torch.cuda.synchronize()
        taken = torch.cuda.max_memory_allocated() - before
        assert not y.requires_grad and torch.equal(y, torch.nn.functional.linear(x, w, b))
    # the result has n O elements of two bytes; codes would take n D bytes
    assert taken < n * D // 2, taken
    y = pkg.linear_8bit(x, w, b)
    assert y.requires_grad
    y.float().sum().backward()
    assert w.grad is not None and b.grad is not None


def test_a_frozen_weight(pkg):
    x = torch.randn(50, 20, device="cuda", requires_grad=True)
    w = torch.randn(10, 20, device="cuda")
    pkg.linear_8bit(x, w).sum().backward()
    assert torch.allclose(x.grad, w.sum(0).expand(50, 20))
