"""Attention, residual norms and 8-bit kept rows without a GPU: schemas, refusals before any launch, sizes of workspaces."""
import ctypes

import pytest
import torch

SCHEMAS = {
    "_CAPI_attention": "(Tensor _0, Tensor _1, Tensor _2, Tensor _3, Tensor _4, bool _5, float _6) -> (Tensor _0, Tensor _1)",
    "_CAPI_attention_backward":
        "(Tensor _0, Tensor _1, Tensor _2, Tensor _3, Tensor _4, Tensor _5, Tensor _6, Tensor _7, bool _8, float _9, bool _10, bool _11) "
        "-> (Tensor _0, Tensor _1, Tensor _2)",
    "_CAPI_residual_norm":
        "(Tensor _0, Tensor _1, Tensor? _2, str _3, Tensor? _4, Tensor? _5, str _6, Tensor? _7, Tensor? _8, float _9, float _10, float _11) "
        "-> (Tensor _0, Tensor _1, Tensor _2, Tensor _3, Tensor _4, Tensor _5)",
    "_CAPI_residual_norm_backward":
        "(Tensor? _0, Tensor? _1, Tensor _2, Tensor _3, Tensor? _4, str _5, Tensor? _6, Tensor? _7, str _8, Tensor? _9, Tensor _10, "
        "Tensor _11, Tensor _12, Tensor _13, float _14, float _15) "
        "-> (Tensor _0, Tensor _1, Tensor _2, Tensor _3, Tensor _4, Tensor _5, Tensor _6)",
    "_CAPI_keep_8bit": "(Tensor _0) -> (Tensor _0, Tensor _1)",
    "_CAPI_kept_8bit_values": "(Tensor _0, Tensor _1, int _2) -> Tensor _0",
    "_CAPI_kept_8bit_weight_grad": "(Tensor _0, Tensor _1, Tensor _2, bool _3) -> (Tensor _0, Tensor _1)",
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
    x = x[0]
    with pytest.raises(RuntimeError, match="CUDA tensor"):
        pkg.residual_norm(x, x)
    with pytest.raises(RuntimeError, match="CUDA tensor"):
        ops._CAPI_residual_norm_backward(x, x, x, x, None, "none", None, None, "rms", None, x, x, x, x, 1.0, 1.0)
    with pytest.raises(RuntimeError, match="CUDA tensor"):
        pkg.keep_8bit(x)
    codes = x.to(torch.int8)
    with pytest.raises(RuntimeError, match="CUDA tensor"):
        pkg.kept_8bit_values(codes, x)
    with pytest.raises(RuntimeError, match="CUDA tensor"):
        ops._CAPI_kept_8bit_weight_grad(x, codes, x, False)
    with pytest.raises(ValueError, match="norm"):
        pkg.residual_norm(x, x, post="batch")


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


def norm_problem(pkg, **kw):
    p = pkg.ResidualNorm(A, 64, None, 0, A, A, A, A, 10, 64, 0, 0, 0, 1, 2, 1.0, 1.0, 1e-6)
    for k, v in kw.items():
        setattr(p, k, v)
    return ctypes.byref(p)


def test_residual_norm_argument_errors(pkg, abi):
    def forward(x=A, stride=64, total=A, out=A, stats=(None, A, A, A), **kw):
        return abi.dgs_residual_norm_forward(norm_problem(pkg, **kw), x, stride, total, out, *stats, None)

    def backward(total=A, ds=A, ds_stride=64, do=A, do_stride=64, stats=(None, A, A, A), grads=(A, A, None, A, A, A, A), ws=A, wb=1 << 40, **kw):
        return abi.dgs_residual_norm_backward(norm_problem(pkg, **kw), total, ds, ds_stride, do, do_stride, *stats, *grads, ws, wb, None)

    for call in (forward, backward):
        assert call(dtype=3) == UNSUPPORTED and call(param_dtype=-1) == UNSUPPORTED
        assert call(D=0) == INVALID and call(n=-1) == INVALID and call(D=8193) == UNSUPPORTED and b"8192" in abi.dgs_last_error()
        assert call(post=3) == INVALID and call(pre=-1) == INVALID and call(gate_kind=4) == INVALID
        assert call(gate_kind=1) == INVALID and call(gate=A) == INVALID and b"gate" in abi.dgs_last_error()
        assert call(post=0) == INVALID and call(pre=0) == INVALID and b"without its norm" in abi.dgs_last_error()
        assert call(weight=None) == INVALID and call(post_weight=None) == INVALID and b"bias" in abi.dgs_last_error()
        assert call(y_stride=63) == INVALID and call(gate=A, gate_kind=3, gate_stride=63) == INVALID
        assert call(eps=-1.0) == INVALID and call(x_scale=float("nan")) == INVALID and call(y_scale=float("inf")) == INVALID
        assert call(y=None) == INVALID and call(stats=(None, None, A, A)) == INVALID and call(stats=(None, A, None, A)) == INVALID
        assert call(post=2) == INVALID
    assert forward(x=None) == INVALID and forward(total=None) == INVALID and forward(out=None) == INVALID and forward(stride=63) == INVALID
    assert backward(ds_stride=63) == INVALID and backward(do_stride=0) == INVALID and backward(total=None) == INVALID
    assert backward(ws=None) == INVALID and backward(wb=16) == INVALID and b"workspace" in abi.dgs_last_error()
    assert backward(grads=(A, A, A, A, A, A, A)) == INVALID and b"absent" in abi.dgs_last_error()
    assert forward(n=0, y=None) == 0 and backward(grads=(None,) * 7) == 0 and backward(n=0, grads=(None,) * 7) == 0
    assert abi.dgs_residual_norm_backward_workspace_bytes(0, 64) == 0 and abi.dgs_residual_norm_backward_workspace_bytes(1, 64) == 4 * 64 * 4


def test_kept_argument_errors(abi):
    def keep(x=A, stride=100, dtype=1, n=7, D=100, codes=A, scales=A):
        return abi.dgs_keep_8bit(x, stride, dtype, n, D, codes, scales, None)

    def values(codes=A, stride=100, scales=A, n=7, D=100, dtype=1, out=A):
        return abi.dgs_kept_8bit_values(codes, stride, scales, n, D, dtype, out, None)

    def grad(g=A, g_stride=47, dtype=1, codes=A, stride=100, scales=A, n=7, O=47, D=100, dw=A, db=A, ws=A, wb=1 << 40):
        return abi.dgs_kept_8bit_weight_grad(g, g_stride, dtype, codes, stride, scales, n, O, D, dw, db, ws, wb, None)

    for call in (keep, values, grad):
        assert call(dtype=3) == UNSUPPORTED and call(D=0) == INVALID and call(n=-1) == INVALID and call(D=1 << 23) == INVALID
        assert call(stride=99) == INVALID and b"overlap" in abi.dgs_last_error()
        assert call(codes=None) == INVALID and call(scales=None) == INVALID
    assert keep(x=None) == INVALID and values(out=None) == INVALID
    assert grad(O=0) == INVALID and grad(g=None) == INVALID and grad(dw=None) == INVALID and grad(g_stride=46) == INVALID
    assert grad(ws=None) == INVALID and grad(wb=8) == INVALID and grad(ws=A + 8) == INVALID and b"workspace" in abi.dgs_last_error()
    # weights whose tiles a grid cannot have
    for dtype in (0, 1, 2):
        assert grad(O=1 << 22, g_stride=1 << 22, dtype=dtype) == INVALID and grad(O=1 << 20, D=1 << 20, g_stride=1 << 20, stride=1 << 20, dtype=dtype) == INVALID
        assert b"a weight of" in abi.dgs_last_error()
    assert keep(n=0, x=None) == 0 and values(n=0, out=None) == 0
    size = abi.dgs_kept_8bit_weight_grad_workspace_bytes
    assert size(0, 4, 4, 0) == 0 and size(4, 4, 4, 7) == 0 and 0 < size(1, 4, 4, 1) and size(430_000, 47, 256, 1) < 64 << 20
