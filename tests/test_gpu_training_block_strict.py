"""What the operators of a block hand back and keep, exactly: which gradients there are, what linear_8bit saves, and the weight's gradient
against the rows that codes and scales stand for before their rounding to 16 bits."""
import pytest
import torch

pytestmark = pytest.mark.gpu
ROUND = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


@pytest.mark.parametrize("dtype", list(ROUND))
def test_what_linear_8bit_saves(pkg, dtype):
    x = torch.randn(3, 50, 260, device="cuda").to(dtype).requires_grad_()
    w = torch.randn(20, 260, device="cuda").to(dtype).requires_grad_()
    b = torch.randn(20, device="cuda").to(dtype).requires_grad_()
    saved = []
    with torch.autograd.graph.saved_tensors_hooks(lambda t: saved.append((tuple(t.shape), str(t.dtype))) or t, lambda t: t):
        pkg.linear_8bit(x, w, b)
    assert sorted(saved) == sorted([((20, 260), str(dtype)), ((150, 260), "torch.int8"), ((150, 3), "torch.float32")])


@pytest.mark.parametrize("post,pre", [(p, q) for p in ("none", "rms", "layer") for q in ("none", "rms", "layer")])
@pytest.mark.parametrize("gate", ["none", "column", "row", "element"])
def test_which_gradients_a_residual_norm_returns(ops, post, pre, gate):
    n, D, dt, pt = 6, 40, torch.bfloat16, torch.float32
    x, y, ds = (torch.randn(n, D, device="cuda").to(dt) for _ in range(3))
    g = {"none": None, "column": torch.randn(D, device="cuda"), "row": torch.randn(n, 1, device="cuda").to(dt),
         "element": torch.randn(n, D, device="cuda").to(dt)}[gate]
    for weights in (True, False):
        w = {k: torch.randn(D, device="cuda") if weights and kind != "none" else None for k, kind in (("post", post), ("pre", pre))}
        total, out, *stats = ops._CAPI_residual_norm(x, y, g, post, w["post"], w["post"], pre, w["pre"], w["pre"], 0.9, 0.7, 1e-6)
        do = torch.randn(n, D, device="cuda").to(dt) if pre != "none" else None
        grads = ops._CAPI_residual_norm_backward(ds, do, total, y, g, post, w["post"], w["post"], pre, w["pre"], *stats, 0.9, 0.7)
        there = lambda k: ((D,), pt) if w[k] is not None else ((0,), None)  # noqa: E731
        want = [((n, D), dt), ((n, D), dt), (tuple(g.shape), g.dtype) if g is not None else ((0,), None), there("post"), there("post"),
                there("pre"), there("pre")]
        for t, (shape, kind) in zip(grads, want):
            assert tuple(t.shape) == shape and (kind is None or t.dtype == kind) and t.isfinite().all()


@pytest.mark.parametrize("dtype", list(ROUND))
@pytest.mark.parametrize("n,O,D", [(65, 128, 128), (2000, 47, 256), (5000, 300, 75)])
def test_the_weights_gradient_against_unrounded_rows(ops, n, O, D, dtype):
    """In 16 bits each value is rounded once before its product: r sum |g||v| besides the sums' own error (n + 64) 2^-23 of that."""
    g = torch.Generator(device="cuda").manual_seed(n)
    grad = torch.randn((n, O), device="cuda", generator=g).to(dtype)
    codes, scales = ops._CAPI_keep_8bit(torch.randn((n, D), device="cuda", generator=g))
    dw, _ = ops._CAPI_kept_8bit_weight_grad(grad, codes, scales, False)
    v = codes.double() * scales.double().repeat_interleave(128, 1)[:, :D]
    want, size = grad.double().t() @ v, grad.double().abs().t() @ v.abs()
    r = ROUND[dtype]
    # (float32: code times scale is rounded as well; fp16: below its normal numbers by half of 2^-24 a value)
    room = ((n + 64) * 2.0 ** -23 + r) * size + r * want.abs() + 2.0 ** -25 * grad.double().abs().sum(0)[:, None] + 2.0 ** -25
    assert ((dw.double() - want).abs() <= room).all()
