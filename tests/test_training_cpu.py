"""The operators of a training step without a GPU: schemas, refusals before any launch, sizes of workspaces and slots."""
import ctypes

import pytest
import torch

SCHEMAS = {
    "_CAPI_layer_norm": "(Tensor _0, Tensor? _1, Tensor? _2, float _3) -> (Tensor _0, Tensor _1, Tensor _2)",
    "_CAPI_layer_norm_backward":
        "(Tensor _0, Tensor _1, Tensor? _2, Tensor _3, Tensor _4, bool _5, bool _6) -> (Tensor _0, Tensor _1, Tensor _2)",
    "_CAPI_linear_cross_entropy": "(Tensor _0, Tensor _1, Tensor _2, int _3) -> (Tensor _0, Tensor _1)",
    "_CAPI_linear_cross_entropy_backward":
        "(Tensor _0, Tensor _1, Tensor _2, Tensor _3, Tensor _4, int _5, bool _6, bool _7) -> (Tensor _0, Tensor _1)",
    "_CAPI_adamw_step":
        "(Tensor[] _0, Tensor?[] _1, Tensor[] _2, Tensor _3, Tensor _4, float _5, float _6, float _7, float _8, float _9, "
        "int _10) -> ()",
    "_CAPI_adamw_step_8bit":
        "(Tensor[] _0, Tensor?[] _1, Tensor[] _2, Tensor _3, Tensor _4, Tensor _5, Tensor _6, float _7, float _8, float _9, "
        "float _10, float _11, int _12) -> ()",
    "_CAPI_adamw_state_values": "(Tensor _0, Tensor _1) -> Tensor _0",
}


def test_schemas(ops):
    for name, sig in SCHEMAS.items():
        assert str(torch._C._get_schema("dgs_ops::" + name, "")) == "dgs_ops::" + name + sig


def test_tensors_on_the_host_are_refused(ops, pkg):
    x = torch.zeros(4, 8)
    with pytest.raises(RuntimeError, match="CUDA tensor"):
        ops._CAPI_layer_norm(x, None, None, 1e-5)
    with pytest.raises(RuntimeError, match="CUDA tensor"):
        ops._CAPI_layer_norm_backward(x, x, None, x[:, 0], x[:, 0], True, False)
    with pytest.raises(RuntimeError, match="CUDA tensor"):
        ops._CAPI_linear_cross_entropy(x, x, torch.zeros(4, dtype=torch.int64), -100)
    with pytest.raises(RuntimeError, match="CUDA tensor"):
        ops._CAPI_adamw_step([x], [x], [], x, x, 1e-3, 0.9, 0.999, 1e-8, 0.0, 1)
    with pytest.raises(RuntimeError, match="CUDA tensor"):
        ops._CAPI_adamw_state_values(torch.zeros(256, dtype=torch.int8), torch.zeros(1))
    with pytest.raises(ValueError, match="reduction"):
        pkg.linear_cross_entropy(x, x, torch.zeros(4, dtype=torch.int64), reduction="avg")
    with pytest.raises(ValueError, match="bits"):
        pkg.AdamW([x], bits=16)
    with pytest.raises(ValueError, match="no parameters"):
        pkg.AdamW([])


INVALID, UNSUPPORTED = 1, 5
A = 0x10000  # never dereferenced on the host


def test_layer_norm_argument_errors(abi):
    def call(x=A, stride=8, dtype=0, w=A, b=A, pd=0, n=4, D=8, eps=1e-5, y=A):
        return abi.dgs_layer_norm(x, stride, dtype, w, b, pd, n, D, eps, y, A, A, None)
    assert call(D=0) == INVALID and call(n=-1) == INVALID
    assert call(stride=7) == INVALID and b"apart" in abi.dgs_last_error()
    assert call(dtype=3) == UNSUPPORTED and call(pd=-1) == UNSUPPORTED
    assert call(w=None) == INVALID and b"bias" in abi.dgs_last_error()
    assert call(eps=-1.0) == INVALID and call(eps=float("nan")) == INVALID
    assert call(x=None) == INVALID and call(y=None) == INVALID
    assert call(n=0, x=None) == 0

    def back(n=4, dw=A, db=A, ws=A, wb=1 << 20, dy=A, stride=8):
        return abi.dgs_layer_norm_backward(dy, stride, A, 8, 0, A, 0, A, A, n, 8, A, dw, db, ws, wb, None)
    assert back(dw=None) == INVALID and back(ws=None) == INVALID and back(wb=8) == INVALID
    assert b"workspace" in abi.dgs_last_error()
    assert back(dy=None) == INVALID and back(stride=3) == INVALID
    assert abi.dgs_layer_norm_backward_workspace_bytes(0, 8) == 0
    assert abi.dgs_layer_norm_backward_workspace_bytes(3, 8) >= 3 * 2 * 8 * 4


def test_cross_entropy_argument_errors(abi):
    def call(h=A, hs=8, ws=8, dtype=1, n=4, D=8, V=10, loss=A, work=A, wb=1 << 30):
        return abi.dgs_linear_cross_entropy(h, hs, A, ws, dtype, A, 1, n, D, V, -100, loss, A, work, wb, None, None)
    assert call(dtype=7) == UNSUPPORTED
    assert call(n=-1) == INVALID and call(D=0) == INVALID and call(V=0) == INVALID
    assert call(V=1 << 31) == UNSUPPORTED and call(D=(1 << 20) + 8, hs=1 << 21, ws=1 << 21) == UNSUPPORTED
    assert call(hs=7) == INVALID and call(ws=7) == INVALID
    assert call(h=None) == INVALID and call(loss=None) == INVALID
    assert call(work=None) == INVALID and call(wb=0) == INVALID and call(work=A + 16) == INVALID
    assert b"workspace" in abi.dgs_last_error()
    assert call(n=0, h=None) == 0

    def back(dloss=A, dh=A, dw=A, work=A, wb=1 << 40):
        return abi.dgs_linear_cross_entropy_backward(dloss, A, 8, A, 8, 1, A, 1, A, 4, 8, 10, -100, dh, dw, work, wb, None, None)
    assert back(dloss=None) == INVALID and back(work=None) == INVALID and back(wb=64) == INVALID
    assert back(dh=None, dw=None) == 0
    for dtype in (0, 1, 2):
        for fn in (abi.dgs_linear_cross_entropy_workspace_bytes, abi.dgs_linear_cross_entropy_backward_workspace_bytes):
            assert fn(100, 64, 1000, dtype) > 0 and fn(0, 64, 1000, dtype) == 0 and fn(100, 64, 1000, 9) == 0
    # the logits are never all held: 8 192 rows against 2^20 classes would be 32 GB of them
    assert abi.dgs_linear_cross_entropy_workspace_bytes(8192, 1024, 1 << 20, 1) < 1 << 28
    assert abi.dgs_linear_cross_entropy_backward_workspace_bytes(8192, 1024, 1 << 20, 1) < 1 << 30


def test_adamw_argument_errors(abi, pkg):
    def call(lr=1e-3, b1=0.9, b2=0.999, eps=1e-8, wd=0.0, step=1, m=A, count=1, **kw):
        t = (pkg.AdamWTensor * 1)()
        for k, v in dict(dict(param=A, grad=A, n=5, at=0), **kw).items():
            setattr(t[0], k, v)
        return abi.dgs_adamw_step(t, count, m, A, lr, b1, b2, eps, wd, step, None)
    assert call(lr=-1.0) == INVALID and call(lr=float("nan")) == INVALID and call(eps=-1.0) == INVALID
    assert call(b1=1.0) == INVALID and call(b2=-0.1) == INVALID and call(wd=-1.0) == INVALID
    assert call(step=0) == INVALID and b"steps" in abi.dgs_last_error()
    assert call(m=None) == INVALID and call(m=A + 4) == INVALID
    assert call(at=100) == INVALID and b"slot" in abi.dgs_last_error()
    assert call(grad=None) == INVALID and call(n=-1) == INVALID
    assert call(param_dtype=5) == UNSUPPORTED and call(copy=A, copy_dtype=5) == UNSUPPORTED
    assert call(count=-1) == INVALID
    assert abi.dgs_adamw_step(None, 0, None, None, 1e-3, 0.9, 0.999, 1e-8, 0.0, 1, None) == 0
    assert abi.dgs_adamw_step_8bit(None, 1, A, A, A, A, 1e-3, 0.9, 0.999, 1e-8, 0.0, 1, None) == INVALID
    assert abi.dgs_adamw_step_8bit(None, 1, A, None, A, A, 1e-3, 0.9, 0.999, 1e-8, 0.0, 1, None) == INVALID
    assert abi.dgs_adamw_state_values(A, 0, A, 100, A, None) == INVALID
    assert abi.dgs_adamw_state_values(None, 0, A, 256, A, None) == INVALID
    assert abi.dgs_adamw_state_values(None, 0, None, 0, None, None) == 0
    assert [abi.dgs_adamw_slot_elems(n) for n in (0, 1, 256, 257)] == [0, 256, 256, 512]
    assert ctypes.sizeof(pkg.AdamWTensor) == 56
