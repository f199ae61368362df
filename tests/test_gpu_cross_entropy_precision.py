"""How far the cross entropy's results are off as a whole: G travels to the products in 16 bits (two planes of them where few rows
or results would not average its rounding), so gradients may be off by sqrt(2) times what rounding the exact ones costs; the
statistics are in 32 bits, so losses are within 1e-6 of theirs also where a tensor core's accumulator would not be."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu


def rel(a, b):
    return ((a.double() - b).norm() / b.norm()).item()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("weights", ["varied", "equal", "spread"])
@pytest.mark.parametrize("n,D,V", [(1, 64, 2), (1, 700, 5000), (3, 500, 7), (100, 64, 1000), (128, 200, 300), (129, 200, 300),
                                   (275, 335, 2641), (613, 52, 137), (2000, 8, 3), (1000, 1000, 4), (300, 96, 20_000)])
def test_gradients_as_a_whole(ops, n, D, V, weights, dtype):
    g = torch.Generator(device="cuda").manual_seed(n + D)
    h = torch.randn(n, D, device="cuda", generator=g).to(dtype)
    w = (torch.randn(V, D, device="cuda", generator=g) * (2.0 / math.sqrt(D))).to(dtype)
    t = torch.randint(0, V, (n,), device="cuda", generator=g)
    dl = torch.full((n,), 1.0 / n, device="cuda")
    if weights == "varied":
        dl = (torch.rand(n, device="cuda", generator=g) + 0.5) / n
    if weights == "spread":
        dl = torch.exp(torch.randn(n, device="cuda", generator=g) * 2)
    loss, lse = ops._CAPI_linear_cross_entropy(h, w, t, -100)
    dh, dw = ops._CAPI_linear_cross_entropy_backward(dl, h, w, t, lse, -100, True, True)
    s = h.double() @ w.double().t()
    assert rel(loss, torch.logsumexp(s, 1) - s[torch.arange(n), t]) <= (1e-6 if n >= 100 else 1e-5)
    G = torch.softmax(s, 1)
    G[torch.arange(n), t] -= 1.0
    G *= dl.double()[:, None]
    for got, want in ((dh, G @ w.double()), (dw, G.t() @ h.double())):
        assert rel(got, want) <= 1.5 * rel(want.to(dtype), want)
