"""A wait of the weight gradient's kernel that runs out: the status word has it, the next call reports it, and no result of that call
looks like a number, with or without a status word."""
import ctypes

import pytest
import torch

pytestmark = pytest.mark.gpu
ERR_CUDA = 2


# (one share of the rows and several; few results and several tiles)
@pytest.mark.parametrize("n,O,D", [(300, 40, 100), (300, 300, 600), (20_000, 47, 256), (20_000, 300, 300)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_a_wait_that_runs_out_is_reported(ops, abi, dtype, n, O, D):
    g = torch.Generator(device="cuda").manual_seed(n + O)
    grad = torch.randn((n, O), device="cuda", generator=g).to(dtype)
    codes, scales = ops._CAPI_keep_8bit(torch.randn((n, D), device="cuda", generator=g))
    dw, db = ops._CAPI_kept_8bit_weight_grad(grad, codes, scales, True)
    code = 1 if dtype == torch.bfloat16 else 2
    ws = torch.empty(abi.dgs_kept_8bit_weight_grad_workspace_bytes(n, O, D, code), dtype=torch.uint8, device="cuda")
    p = lambda t: ctypes.c_void_p(t.data_ptr())  # noqa: E731

    def direct(status):
        w, b = torch.zeros_like(dw), torch.zeros_like(db)
        rc = abi.dgs_kept_8bit_weight_grad_reported(p(grad), O, code, p(codes), D, p(scales), n, O, D, p(w), p(b), p(ws), ws.numel(),
                                                    p(status) if status is not None else None,
                                                    ctypes.c_void_p(torch.cuda.current_stream().cuda_stream))
        torch.cuda.synchronize()
        assert rc == 0
        return w, b

    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    torch.cuda.synchronize()
    assert abi.dgs_set_wait_limit(0) == 2_000_000_000
    try:
        for s in (status, None):
            w, b = direct(s)
            assert w.isnan().all() and b.isnan().all()
        assert status.item() == ERR_CUDA
        ops._CAPI_kept_8bit_weight_grad(grad, codes, scales, True)
        torch.cuda.synchronize()
    finally:
        assert abi.dgs_set_wait_limit(2_000_000_000) == 0
    with pytest.raises(RuntimeError, match="earlier _CAPI_kept_8bit_weight_grad call reported an error"):
        ops._CAPI_kept_8bit_weight_grad(grad, codes, scales, True)
    again = ops._CAPI_kept_8bit_weight_grad(grad, codes, scales, True)
    assert torch.equal(again[0], dw) and torch.equal(again[1], db)
    status.zero_()
    w, b = direct(status)
    assert torch.equal(w, dw) and torch.equal(b, db) and status.item() == 0
