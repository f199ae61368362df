"""What a step of AdamW leaves alone stays usable: autograd may go on with what it saved of tensors that had no gradient."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("bits", [32, 8])
def test_versions_of_what_was_not_written(pkg, bits):
    p = [torch.randn(300, device="cuda"), torch.randn(40, device="cuda"), torch.zeros(0, device="cuda")]
    copies = [x.bfloat16() for x in p]
    before = [t._version for t in p + copies]
    pkg.AdamW(p, bits=bits, copies=copies).step([torch.randn(300, device="cuda"), None, torch.zeros(0, device="cuda")])
    moved = [t._version > v for t, v in zip(p + copies, before)]
    assert moved == [True, False, False] * 2


def test_backward_through_a_frozen_weight_after_a_step(pkg):
    frozen, w = torch.randn(8, 8, device="cuda"), torch.randn(8, 8, device="cuda", requires_grad=True)
    opt = pkg.AdamW([frozen, w.detach()])
    other = torch.randn(5, 8, device="cuda", requires_grad=True)
    loss = (other @ frozen).square().sum()                            # saved `frozen`
    before = frozen.clone()
    opt.step([None, torch.randn(8, 8, device="cuda")])
    loss.backward()
    assert torch.equal(frozen, before) and other.grad is not None
    loss = (other @ w).square().sum()                                 # one that a step has written is refused, as ever
    pkg.AdamW([w]).step([torch.ones(8, 8, device="cuda")])
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()
