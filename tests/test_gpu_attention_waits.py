"""A wait of the attention kernels that runs out: the call gives up as a whole, is reported by the next one, and leaves nothing behind."""
import pytest
import torch

from test_gpu_attention import make, offsets

pytestmark = pytest.mark.gpu


@pytest.fixture
def no_waiting(abi):
    def off():
        assert abi.dgs_set_wait_limit(0) == 2_000_000_000
    yield off
    abi.dgs_set_wait_limit(2_000_000_000)


@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("dtype,heads,kv_heads,d", [(torch.bfloat16, 4, 2, 64), (torch.float16, 3, 3, 128), (torch.float16, 2, 2, 40)])
def test_a_wait_that_runs_out_is_reported(ops, abi, no_waiting, dtype, heads, kv_heads, d, causal):
    lens = [1000, 1, 40, 600]
    q, k, v, do = make(lens, lens, heads, kv_heads, d, dtype)
    o, scale = offsets(lens), d ** -0.5
    out, lse = ops._CAPI_attention(q, k, v, o, o, causal, scale)
    base = ops._CAPI_attention_backward(do, q, k, v, out, lse, o, o, causal, scale, True, True)
    torch.cuda.synchronize()
    no_waiting()
    ops._CAPI_attention(q, k, v, o, o, causal, scale)
    torch.cuda.synchronize()
    with pytest.raises(RuntimeError, match="earlier _CAPI_attention call reported an error"):
        ops._CAPI_attention(q, k, v, o, o, causal, scale)
    ops._CAPI_attention_backward(do, q, k, v, out, lse, o, o, causal, scale, True, True)
    torch.cuda.synchronize()
    assert abi.dgs_set_wait_limit(2_000_000_000) == 0
    with pytest.raises(RuntimeError, match="earlier _CAPI_attention_backward call reported an error"):
        ops._CAPI_attention(q, k, v, o, o, causal, scale)
    again = ops._CAPI_attention(q, k, v, o, o, causal, scale)
    assert torch.equal(again[0], out) and torch.equal(again[1], lse)
    for a, b in zip(ops._CAPI_attention_backward(do, q, k, v, out, lse, o, o, causal, scale, True, True), base):
        assert torch.equal(a, b)
