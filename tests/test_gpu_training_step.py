"""The operators together, behind the sampler: the example trains, and one step of it is the step that torch's own operators make."""
import importlib

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("bits", [32, 8])
def test_the_example_learns(bits, capsys):
    example = importlib.import_module("dist-gpu-sampling_b200.train_nodes")
    losses = example.main(["--nodes", "20000", "--steps", "60", "--batch", "512", "--classes", "12", "--hidden", "64", "--dim", "36",
                           "--fanouts", "5,5", "--bits", str(bits)])
    assert all(torch.isfinite(torch.tensor(losses)))
    # it begins near log 12 = 2.48; the classes can be told from the neighbours' features
    assert sum(losses[-5:]) / 5 < 0.6 * sum(losses[:3]) / 3
    assert "step   59" in capsys.readouterr().out


def test_one_step_like_torch(pkg):
    """Layer norm, head and AdamW in float32 against torch in float64: tolerances are a few hundred roundings of 2^-24 of values of
    the size met here (rows of 40, 90 classes, gradients below 1)."""
    g = torch.Generator(device="cuda").manual_seed(0)
    x = torch.randn(300, 40, device="cuda", generator=g)
    t = torch.randint(0, 90, (300,), device="cuda", generator=g)
    t[::7] = -100
    p = [torch.randn(s, device="cuda", generator=g) * 0.2 for s in ((40,), (40,), (90, 40))]
    mine = [v.clone().requires_grad_() for v in p]
    ref = [v.double().requires_grad_() for v in p]
    opt, want = pkg.AdamW(mine, lr=1e-2), torch.optim.AdamW(ref, lr=1e-2)
    for _ in range(3):
        loss = pkg.linear_cross_entropy(pkg.layer_norm(x, mine[0], mine[1]), mine[2], t)
        other = torch.nn.functional.cross_entropy(torch.nn.functional.layer_norm(x.double(), (40,), ref[0], ref[1]) @ ref[2].t(), t)
        assert abs(loss.item() - other.item()) <= 300 * 2.0 ** -24 * 10
        loss.backward()
        other.backward()
        for a, b in zip(mine, ref):
            assert (a.grad.double() - b.grad).abs().max() <= 300 * 2.0 ** -24 * max(1.0, b.grad.abs().max().item())
        # the same gradients for both, so that m / sqrt(v) of tiny ones does not decide
        for a, b in zip(mine, ref):
            b.grad.copy_(a.grad.double())
        opt.step()
        want.step()
        opt.zero_grad()
        want.zero_grad()
        for a, b in zip(mine, ref):
            assert (a.detach().double() - b.detach()).abs().max() <= 64 * 2.0 ** -24
            b.data.copy_(a.detach().double())
