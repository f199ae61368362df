"""Attention, residual norms and 8-bit kept rows without a GPU: schemas, refusals before any launch, sizes of workspaces."""
import ctypes

import pytest
import torch

SCHEMAS = {
    "_CAPI_attention": "(Tensor _0, Tensor _1, Tensor _2, Tensor _3, Tensor _4, bool _5, float _6) -> (Tensor _0, Tensor _1)",
    "_CAPI_attention_backward":
        "(Tensor _0, Tensor _1, Tensor _2, Tensor _3, Tensor _4, Tensor _5, Tensor _6, Tensor _7, bool _8, float _9, bool _10, bool _11) "
        "-> (Tensor _0, Tensor _1, Tensor _2)",
}
INVALID, UNSUPPORTED = 1, 5
A = 0x10000  # never dereferenced on the host


def test_schemas(ops):
    for name, sig in SCHEMAS.items():
        assert str(torch._C._get_schema("dgs_ops::" + name, "")) == "dgs_ops::" + name + sig


def test_tensors_on_the_host_are_refused(ops, pkg):
    x, o = torch.zeros(4, 2, 8), torch.tensor([0, 4])
    with pytest.raises(RuntimeError, match="CUDA tensor"):
        ops._CAPI_attention(x, x, x, o, o, False, 1.0)
    with pytest.raises(RuntimeError, match="CUDA tensor"):
        ops._CAPI_attention_backward(x, x, x, x, x, x[0], o, o, False, 1.0, True, True)
    with pytest.raises(RuntimeError, match="CUDA tensor"):
        pkg.attention(x, x, x, o)


def problem(pkg, **kw):
    p = pkg.Attention(A, A, A, 256, 64, 128, 64, 128, 64, A, A, 100, 200, 7, 4, 2, 64, 1, 1, 0, 0.125)
    for k, v in kw.items():
        setattr(p, k, v)
    return p


def test_attention_argument_errors(pkg, abi):
    def forward(out=A, lse=A, ws=A, wb=1 << 40, **kw):
        return abi.dgs_attention_forward(ctypes.byref(problem(pkg, **kw)), out, lse, ws, wb, None, None)

    def backward(dout=A, row=256, head=64, out=A, lse=A, dq=A, dk=A, dv=A, ws=A, wb=1 << 40, **kw):
        return abi.dgs_attention_backward(ctypes.byref(problem(pkg, **kw)), dout, row, head, out, lse, dq, dk, dv, ws, wb, None, None)

    for call in (forward, backward):
        assert call(dtype=3) == UNSUPPORTED and call(dtype=-1) == UNSUPPORTED
        assert call(d=136) == UNSUPPORTED and b"128" in abi.dgs_last_error()
        assert call(d=60) == UNSUPPORTED and call(d=0) == UNSUPPORTED and call(d=62, dtype=0) == UNSUPPORTED
        assert call(heads=3) == INVALID and call(kv_heads=0) == INVALID and call(heads=0) == INVALID
        assert call(n_q=-1) == INVALID and call(n_k=1 << 30) == INVALID and call(seqs=-1) == INVALID
        assert call(q=A + 8) == INVALID and b"16-byte" in abi.dgs_last_error()
        assert call(k_row=132) == INVALID and call(v_head=4) == INVALID and call(q_row=-256) == INVALID
        assert call(scale=float("inf")) == INVALID and call(scale=float("nan")) == INVALID
        assert call(q=None) == INVALID and call(k=None) == INVALID and call(k_offsets=None) == INVALID
        assert call(ws=None) == INVALID and call(ws=A + 16) == INVALID and call(wb=100) == INVALID
        assert b"workspace" in abi.dgs_last_error()
        assert call(lse=None) == INVALID and call(out=None) == INVALID and call(out=A + 8) == INVALID
    assert backward(dv=None) == INVALID and b"together" in abi.dgs_last_error()
    assert backward(dout=None) == INVALID and backward(row=250) == INVALID and backward(dq=A + 2) == INVALID
    assert abi.dgs_attention_forward(None, A, A, A, 1 << 40, None, None) == INVALID
    # nothing to do needs nothing
    assert forward(n_q=0, q=None) == 0 and backward(dq=None, dk=None, dv=None) == 0


def test_attention_workspace(pkg, abi):
    size = lambda back=0, **kw: abi.dgs_attention_workspace_bytes(ctypes.byref(problem(pkg, **kw)), back)  # noqa: E731
    assert abi.dgs_attention_workspace_bytes(None, 0) == 0 and size(heads=0) == 0 and size(n_q=-1) == 0
    # a place and a map entry for what is there, delta for the backward pass; parts of rows only where a row can have many keys
    assert 0 < size() < 64 * 1024 and size(1) >= size() + 4 * 4 * 100
    assert size(n_k=256) < 64 * 1024 < size(n_k=1 << 20, n_q=16)
    # it grows with rows and keys, not with their product
    assert size(1, n_q=1 << 20, n_k=1 << 20, seqs=1) < 200 << 20
