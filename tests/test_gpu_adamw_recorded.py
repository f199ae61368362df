"""A step counts on the host, so one that a CUDA graph recorded would be the same step for ever: the optimizer refuses it."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("bits", [32, 8])
def test_a_step_is_not_recorded(pkg, bits):
    p, g = torch.ones(300, device="cuda"), torch.ones(300, device="cuda")
    opt = pkg.AdamW([p], bits=bits)
    opt.step([g])
    before, moments = p.clone(), [t.clone() for t in opt.state.values()]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = g * 1.0
        with pytest.raises(RuntimeError, match="recorded"):
            opt.step([held])
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(p, before) and opt.steps == 1 and opt.tensor_steps == [1]
    assert all(torch.equal(a, b) for a, b in zip(moments, opt.state.values()))
    opt.step([g])
    assert opt.steps == 2 and not torch.equal(p, before)


def test_the_operator_itself_may_be(ops):
    """Its count is the caller's: one step, replayed as it is."""
    p, g, m = torch.ones(300, device="cuda"), torch.ones(300, device="cuda"), torch.zeros(2, 512, device="cuda")
    q, n = p.clone(), m.clone()
    args = (1e-3, 0.9, 0.999, 1e-8, 0.0, 5)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops._CAPI_adamw_step([p], [g], [], m[0], m[1], *args)
    for _ in range(3):
        graph.replay()
        ops._CAPI_adamw_step([q], [g], [], n[0], n[1], *args)
    torch.cuda.synchronize()
    assert torch.equal(p, q) and torch.equal(m, n)
