"""The weight's gradient from 8-bit rows where a warp's 32 results end inside of it, over several blocks of 32 columns: every result is
there, in one share of the rows and in many, and nothing is written behind the last one.  Tolerances: test_gpu_kept_8bit.py."""
import ctypes

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("n", [70, 3000])
@pytest.mark.parametrize("O", [1, 2, 31, 33, 47, 95, 97, 127, 129, 161, 255, 257, 290])
@pytest.mark.parametrize("D", [33, 100, 256, 300])
def test_results_that_end_inside_a_warp(ops, O, D, n, dtype):
    g = torch.Generator(device="cuda").manual_seed(O)
    grad = torch.randn((n, O), device="cuda", generator=g).to(dtype)
    codes, scales = ops._CAPI_keep_8bit(torch.randn((n, D), device="cuda", generator=g))
    dw, db = ops._CAPI_kept_8bit_weight_grad(grad, codes, scales, True)
    v, d = ops._CAPI_kept_8bit_values(codes, scales, dtype).double(), grad.double()
    r = torch.finfo(dtype).eps / 2
    want, size = d.t() @ v, d.abs().t() @ v.abs()
    assert ((dw.double() - want).abs() <= (n + 64) * 2.0 ** -23 * size + r * want.abs() + 2.0 ** -24).all()
    want = d.sum(0)
    assert ((db.double() - want).abs() <= (n + 64) * 2.0 ** -23 * d.abs().sum(0) + r * want.abs() + 2.0 ** -24).all()


@pytest.mark.parametrize("n,O,D", [(70, 47, 100), (3000, 33, 300), (3000, 300, 33)])
def test_nothing_behind_the_results(pkg, abi, ops, n, O, D):
    g = torch.Generator(device="cuda").manual_seed(n)
    grad = torch.randn((n, O), device="cuda", generator=g).bfloat16()
    codes, scales = ops._CAPI_keep_8bit(torch.randn((n, D), device="cuda", generator=g))
    dw, db = ops._CAPI_kept_8bit_weight_grad(grad, codes, scales, True)
    wb = abi.dgs_kept_8bit_weight_grad_workspace_bytes(n, O, D, 1)
    ws = torch.empty(wb + 1024, dtype=torch.uint8, device="cuda")
    ws[wb:] = 123
    more_w, more_b = (torch.full((m + 64,), 3.0, dtype=torch.bfloat16, device="cuda") for m in (O * D, O))
    p = lambda t: ctypes.c_void_p(t.data_ptr())  # noqa: E731
    rc = abi.dgs_kept_8bit_weight_grad(p(grad), O, 1, p(codes), D, p(scales), n, O, D, p(more_w), p(more_b), p(ws), wb,
                                       ctypes.c_void_p(torch.cuda.current_stream().cuda_stream))
    torch.cuda.synchronize()
    assert rc == 0
    assert torch.equal(more_w[:O * D].view(O, D), dw) and torch.equal(more_b[:O], db)
    assert (more_w[O * D:] == 3).all() and (more_b[O:] == 3).all() and (ws[wb:] == 123).all()
