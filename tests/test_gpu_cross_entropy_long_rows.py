"""How far losses are off where rows are long: a tensor core cuts what it adds to an accumulator, so logits lose a little with
every 16 of k.  Up to rows of 1 024 that leaves losses within 1e-6 of theirs as a whole, and beyond grows with the length; with no
more than 128 classes and more than 32 rows the parts are added in registers and it does not grow."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("n,D,V", [(1000, 1000, 129), (1000, 1000, 172), (1000, 1024, 5000), (32, 1024, 172), (256, 8192, 100), (256, 8192, 200),
                                   (1000, 4096, 5000), (32, 8192, 200), (300, 2500, 129)])
def test_losses_as_a_whole(ops, n, D, V, dtype):
    g = torch.Generator(device="cuda").manual_seed(n + D)
    h = torch.randn(n, D, device="cuda", generator=g).to(dtype)
    w = (torch.randn(V, D, device="cuda", generator=g) * (2.0 / math.sqrt(D))).to(dtype)
    t = torch.randint(0, V, (n,), device="cuda", generator=g)
    s = h.double() @ w.double().t()
    want = torch.logsumexp(s, 1) - s[torch.arange(n), t]
    loss, _ = ops._CAPI_linear_cross_entropy(h, w, t, -100)
    limit = 1e-6 if V <= 128 and n > 32 else 1e-6 * max(1.0, D / 1024)
    assert (loss.double() - want).norm() <= limit * want.norm()
