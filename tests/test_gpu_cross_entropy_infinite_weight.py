"""A row whose loss has an infinite gradient (a loss scale that overflowed, say) takes no other row's gradient away."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("n,V", [(1, 400), (20, 500), (40, 90), (200, 500), (300, 20_000)])
@pytest.mark.parametrize("bad", [float("inf"), -float("inf"), float("nan")])
def test_the_other_rows(ops, n, V, bad, dtype):
    g = torch.Generator(device="cuda").manual_seed(n)
    h = torch.randn(n, 64, device="cuda", generator=g).to(dtype)
    w = (torch.randn(V, 64, device="cuda", generator=g) / 4).to(dtype)
    t = torch.randint(0, V, (n,), device="cuda", generator=g)
    dl = torch.full((n,), 1e-3, device="cuda")
    loss, lse = ops._CAPI_linear_cross_entropy(h, w, t, -100)
    clean, _ = ops._CAPI_linear_cross_entropy_backward(dl, h, w, t, lse, -100, True, True)
    at = n // 2
    dl[at] = bad
    for more in ((), (loss,)):
        dh, dw = ops._CAPI_linear_cross_entropy_backward(dl, h, w, t, lse, *more, -100, True, True)
        rows = torch.arange(n, device="cuda") != at
        if not more:
            assert torch.equal(dh[rows], clean[rows])
        assert dh[rows].isfinite().all() and ((dh[rows].double() - clean[rows].double()).norm() <= 1e-2 * clean[rows].double().norm())
        assert not dh[at].isfinite().any() and not dw.isfinite().any()
