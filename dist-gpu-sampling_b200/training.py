"""A training step on the batches that the samplers deliver: layer norm, softmax cross entropy against a large vocabulary
(the classes of a data set, or every node of the graph), AdamW.

    for input_nodes, blocks, n_edges, x in sampler(seed_batches):
        h = model(blocks, layer_norm(x, w, b))                   # the model's own layers
        loss = linear_cross_entropy(h.bfloat16(), head, labels)  # the logits are never held
        loss.backward()
        optimizer.step()

Autograd functions and an optimizer over torch.ops.dgs_ops._CAPI_layer_norm*, _CAPI_linear_cross_entropy* and
_CAPI_adamw_step*, which may be called directly as well (without autograd).  No counterparts in the reference, whose trainers take these from
torch (oppo_bench/single_node/chunktensor.py:120-172).  torch is imported with the first call, as in the rest of the package.
"""
import importlib

_functions = {}


def _ops():
    import torch
    importlib.import_module(__package__).load_ops()
    return torch.ops.dgs_ops


def _define():
    """The autograd functions, made at the first call."""
    import torch
    ops = _ops()

    class LayerNorm(torch.autograd.Function):
        @staticmethod
        def forward(ctx, x, weight, bias, eps):
            y, mean, rstd = ops._CAPI_layer_norm(x, weight, bias, eps)
            ctx.save_for_backward(x, weight, mean, rstd)
            return y

        @staticmethod
        @torch.autograd.function.once_differentiable
        def backward(ctx, grad):
            x, weight, mean, rstd = ctx.saved_tensors
            want_x, want_w, want_b, _ = ctx.needs_input_grad
            dx, dw, db = ops._CAPI_layer_norm_backward(grad, x, weight, mean, rstd, want_x, want_w or want_b)
            return dx if want_x else None, dw if want_w else None, db if want_b else None, None

    class LinearCrossEntropy(torch.autograd.Function):
        @staticmethod
        def forward(ctx, hidden, weight, target, ignore_index, shown):
            loss, lse = ops._CAPI_linear_cross_entropy(hidden, weight, target, ignore_index)
            # (a caller who sees the rows' losses may change them in place)
            ctx.save_for_backward(hidden, weight, target, lse, loss.clone() if shown else loss)
            ctx.ignore_index = ignore_index
            return loss

        @staticmethod
        @torch.autograd.function.once_differentiable
        def backward(ctx, grad):
            hidden, weight, target, lse, loss = ctx.saved_tensors
            want_h, want_w = ctx.needs_input_grad[:2]
            dh, dw = ops._CAPI_linear_cross_entropy_backward.from_loss(grad, hidden, weight, target, lse, loss, ctx.ignore_index, want_h, want_w)
            return dh if want_h else None, dw if want_w else None, None, None, None

    class Attention(torch.autograd.Function):
        @staticmethod
        def forward(ctx, q, k, v, q_offsets, k_offsets, causal, scale):
            out, lse = ops._CAPI_attention(q, k, v, q_offsets, k_offsets, causal, scale)
            ctx.save_for_backward(q, k, v, out, lse, q_offsets, k_offsets)
            ctx.causal, ctx.scale = causal, scale
            ctx.mark_non_differentiable(lse)
            return out, lse

        @staticmethod
        @torch.autograd.function.once_differentiable
        def backward(ctx, grad, _):
            q, k, v, out, lse, q_offsets, k_offsets = ctx.saved_tensors
            want_q, want_k, want_v = ctx.needs_input_grad[:3]
            dq, dk, dv = ops._CAPI_attention_backward(grad, q, k, v, out, lse, q_offsets, k_offsets, ctx.causal, ctx.scale, want_q,
                                                      want_k or want_v)
            return dq if want_q else None, dk if want_k else None, dv if want_v else None, None, None, None, None

    class ResidualNorm(torch.autograd.Function):
        @staticmethod
        def forward(ctx, x, y, gate, post, post_weight, post_bias, pre, weight, bias, x_scale, y_scale, eps):
            total, out, *stats = ops._CAPI_residual_norm(x, y, gate, post, post_weight, post_bias, pre, weight, bias, x_scale, y_scale, eps)
            ctx.save_for_backward(total, y, gate, post_weight, post_bias, weight, *stats)
            ctx.forms, ctx.scales = (post, pre), (x_scale, y_scale)
            ctx.set_materialize_grads(False)
            return (total, out) if pre != "none" else (total, None)

        @staticmethod
        @torch.autograd.function.once_differentiable
        def backward(ctx, dsum, dout):
            total, y, gate, post_weight, post_bias, weight, *stats = ctx.saved_tensors
            if dsum is None and dout is None:
                return (None,) * 12
            dx, dy, dgate, dpw, dpb, dw, db = ops._CAPI_residual_norm_backward(
                dsum, dout, total, y, gate, ctx.forms[0], post_weight, post_bias, ctx.forms[1], weight, *stats, *ctx.scales)
            grads = (dx, dy, dgate, None, dpw, dpb, None, dw, db, None, None, None)
            return tuple(g if want else None for g, want in zip(grads, ctx.needs_input_grad))

    class Linear8bit(torch.autograd.Function):
        @staticmethod
        def forward(ctx, x, weight, bias, recorded):
            ctx.shape = x.shape
            # (needs_input_grad is true of a trainable weight where nothing is recorded, too)
            keep = recorded and ctx.needs_input_grad[1]
            ctx.save_for_backward(weight, *ops._CAPI_keep_8bit(x.reshape(-1, x.shape[-1])) if keep else ())
            with torch.autocast("cuda", enabled=False):  # (the caller's types, here and in the backward pass)
                return torch.nn.functional.linear(x, weight, bias)

        @staticmethod
        @torch.autograd.function.once_differentiable
        def backward(ctx, grad):
            weight, *kept = ctx.saved_tensors
            want_x, want_w, want_b, _ = ctx.needs_input_grad
            rows = grad.reshape(-1, grad.shape[-1])
            dw = db = None
            if want_w:
                dw, db = ops._CAPI_kept_8bit_weight_grad(rows, *kept, want_b)
            elif want_b:
                db = rows.sum(0, dtype=torch.float32).to(grad.dtype)
            with torch.autocast("cuda", enabled=False):
                dx = (rows @ weight).view(ctx.shape) if want_x else None
            return dx, dw, db if want_b else None, None

    _functions.update(norm=LayerNorm, loss=LinearCrossEntropy, attention=Attention, residual=ResidualNorm, linear=Linear8bit)


def layer_norm(x, weight=None, bias=None, eps=1e-5):
    """(x - mean) / sqrt(var + eps) * weight + bias over x's last dimension, with gradients for x, weight and bias.
    x: float32, bfloat16 or float16; weight and bias of one type, x's or another of the three (a bias needs a weight)."""
    if not _functions:
        _define()
    return _functions["norm"].apply(x, weight, bias, float(eps))


def linear_cross_entropy(hidden, weight, target, ignore_index=-100, reduction="mean"):
    """Softmax cross entropy of the logits hidden @ weight.T against `target`, with gradients for hidden and weight.

    hidden [n, D] and weight [V, D] share one type (16 bits run on the tensor cores; float32 runs on the CUDA cores, at about half the
    speed of torch with the logits held); target holds n ids (int64 or int32).  Rows whose target is ignore_index
    count as nothing: loss 0, no gradient, whatever their hidden values are.  reduction: "mean" over the other rows (no such
    row: nan, as torch's cross_entropy has it), "sum", or "none" for one float32 loss per row."""
    if reduction not in ("mean", "sum", "none"):
        raise ValueError("linear_cross_entropy: reduction must be 'mean', 'sum' or 'none', got %r" % (reduction,))
    if not _functions:
        _define()
    loss = _functions["loss"].apply(hidden, weight, target, int(ignore_index), reduction == "none")
    if reduction == "none":
        return loss
    if reduction == "sum":
        return loss.sum()
    return loss.sum() / (target != ignore_index).sum()


def attention(q, k, v, q_offsets, k_offsets=None, causal=False, scale=None, return_lse=False):
    """Softmax attention of packed sequences of different lengths, with gradients for q, k and v.

    q [n_q, heads, d], k and v [n_k, key heads, d] share one type (float32, bfloat16 or float16; heads a multiple of key heads, d up
    to 128) and may be parts of a wider tensor.  Sequence s is the query rows q_offsets[s] to q_offsets[s + 1] and the key rows of
    k_offsets (default: the same) likewise.  Every node of a block over its sampled neighbours, `indptr, indices = block_csc(row, col, n_dst)`:

        attention(q, k[indices], v[indices], torch.arange(n_dst + 1, device="cuda"), indptr)

    causal: query i of Lq sees the keys j <= i + Lk - Lq (the last query sees all of them).  scale: 1 / sqrt(d) by default.  A query that
    sees no key gives zeros, and so do rows outside of all sequences.  return_lse: also the logarithm of the sum of exponentials
    [heads, n_q] (float32, without a gradient; -inf where no key is seen).  Sequences of 24 queries and more (8 over
    many keys) run on the tensor cores in 16 bits; float32 runs on the CUDA cores.  Gradients are added in a fixed order (those of `k[indices]`
    back into k are torch's, by atomics).  A number that is not finite reaches what depends on it: other sequences, and causal queries
    that do not see it, keep their results."""
    if k_offsets is None:
        k_offsets = q_offsets
    if not _functions:
        _define()
    scale = q.shape[-1] ** -0.5 if scale is None else float(scale)
    out, lse = _functions["attention"].apply(q, k, v, q_offsets, k_offsets, bool(causal), scale)
    return (out, lse) if return_lse else out


def residual_norm(x, y, gate=None, post=None, post_weight=None, post_bias=None, norm="rms", weight=None, bias=None, x_scale=1.0,
                  y_scale=1.0, eps=1e-6):
    """The end of a block and the norm in front of the next one, with gradients for all tensors:

        sum = x_scale * x + y_scale * gate * post(y),   out = norm(sum)        -> (sum, out)

    x (the residual rows) and y (the block's output) have one shape and type.  post and norm: "rms", "layer" or None, over the last
    dimension (up to 8192 elements), each with a weight and a bias where they are given; norm=None gives None for out.  gate: a value for
    each column [D], for each row [..., 1] or for each element.  The norm is of the sum as it is stored, in x's type."""
    if not _functions:
        _define()
    for name in (post, norm):
        if name not in (None, "rms", "layer"):
            raise ValueError("residual_norm: a norm must be 'rms', 'layer' or None, got %r" % (name,))
    return _functions["residual"].apply(x, y, gate, post or "none", post_weight, post_bias, norm or "none", weight, bias, float(x_scale),
                                        float(y_scale), float(eps))


def keep_8bit(x):
    """Rows [n, D] in 8 bits: (codes [n, D] int8, scales [n, ceil(D / 128)] float32).  A code is the nearest of 255 even steps between minus
    and plus the largest magnitude a among its row's 128 columns: within a / 254 of the value."""
    return _ops()._CAPI_keep_8bit(x)


def kept_8bit_values(codes, scales, dtype=None):
    """The rows that keep_8bit's codes and scales stand for (dtype: float32 by default)."""
    import torch
    return _ops()._CAPI_kept_8bit_values(codes, scales, dtype or torch.float32)


def linear_8bit(x, weight, bias=None):
    """x @ weight.T + bias whose input is kept for the backward pass in 8 bits (keep_8bit) instead of its own type: half the memory of
    16-bit activations, a quarter of 32-bit ones.  The result and the gradient of x are those of torch's linear; the weight's gradient is
    taken from the kept rows, in one pass over their codes.  x [..., D], weight [O, D] and bias [O] of one type (16 bits run on the tensor
    cores).  Nothing is kept without gradients (torch.no_grad, a weight that needs none).  Where another operator keeps x anyway (attention
    keeps its result), or two layers read it, the codes come on top, once for each layer."""
    import torch
    if not _functions:
        _define()
    if x.dtype != weight.dtype or (bias is not None and bias.dtype != weight.dtype):
        raise ValueError("linear_8bit: x, weight and bias must share one type")
    return _functions["linear"].apply(x, weight, bias, torch.is_grad_enabled())


class AdamW:
    """AdamW over a list of tensors, one launch a step (for lists of up to 512), moments in 32 or in 8 bits.

        optimizer = AdamW([p for p in model.parameters()], lr=1e-3)
        optimizer = AdamW(masters, copies=model_params, bits=8)      # 32-bit parameters, 16-bit model

    params are written in place (contiguous; float32, bfloat16 or float16).  copies, if given, receive every new parameter in
    their own type, and gradients are taken from them: 16-bit model parameters with 32-bit masters.  A tensor without a
    gradient stays as it is, and the step does not count for it: the bias corrections go by the steps that a tensor's own
    moments have seen (`tensor_steps`; a launch for each of the counts that a step meets).  The moments lie in two flat
    buffers, a slot of whole 256-element blocks for each tensor.

    bits=8: a moment's code is rounded down or up at random so that the moment keeps its mean over the steps.  The root of a second
    moment whose code is c (255 for its block's largest, 255 sqrt(root / largest) for the others) then stands within some
    sqrt(1 / (2 c)) of its value: 5 % beside the largest, 15 % at a hundredth of it.  seed: of that rounding; with the same seed the
    same steps give the same bits."""

    def __init__(self, params, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=1e-2, bits=32, copies=None, seed=0):
        import torch
        if bits not in (32, 8):
            raise ValueError("AdamW: bits must be 32 or 8, got %r" % (bits,))
        self.params = list(params)
        self.copies = list(copies) if copies is not None else []
        if not self.params:
            raise ValueError("AdamW: no parameters")
        if self.copies and len(self.copies) != len(self.params):
            raise ValueError("AdamW: %d parameters and %d copies" % (len(self.params), len(self.copies)))
        self.lr, self.betas, self.eps, self.weight_decay, self.bits, self.steps = lr, tuple(betas), eps, weight_decay, bits, 0
        self.tensor_steps, self.seed = [0] * len(self.params), int(seed)
        self._ops = _ops()
        blocks = sum(-(-p.numel() // 256) for p in self.params)
        dev = self.params[0].device

        def zeros(n, dtype):
            return torch.zeros(n, dtype=dtype, device=dev)

        if bits == 32:
            self.state = {"exp_avg": zeros(blocks * 256, torch.float32), "exp_avg_sq": zeros(blocks * 256, torch.float32)}
        else:
            self.state = {"exp_avg": zeros(blocks * 256, torch.int8), "exp_avg_scale": zeros(blocks, torch.float32),
                          "exp_avg_sq": zeros(blocks * 256, torch.uint8), "exp_avg_sq_scale": zeros(blocks, torch.float32)}

    def zero_grad(self):
        for p in self.params + self.copies:
            p.grad = None

    def step(self, grads=None):
        """One step with `grads` (None in the place of a gradient that is absent), or with the tensors' own .grad."""
        import torch
        if self.params[0].is_cuda and torch.cuda.is_current_stream_capturing():
            raise RuntimeError("AdamW: a step that a CUDA graph recorded would repeat its count for ever; call step() outside of it")
        if grads is None:
            grads = [p.grad for p in self.copies or self.params]
        grads = list(grads)
        if len(grads) != len(self.params):
            raise ValueError("AdamW: %d parameters and %d gradients" % (len(self.params), len(grads)))
        counts = [n if g is None else n + 1 for n, g in zip(self.tensor_steps, grads)]
        due = {n for n, g in zip(counts, grads) if g is not None}
        for n in sorted(due):
            now = grads if len(due) == 1 else [g if c == n else None for c, g in zip(counts, grads)]
            self._step(now, n)
            self.tensor_steps = [t if g is None else n for t, g in zip(self.tensor_steps, now)]
        self.steps += 1

    def _step(self, grads, step):
        st, (b1, b2) = self.state, self.betas
        if self.bits == 32:
            self._ops._CAPI_adamw_step(self.params, grads, self.copies, st["exp_avg"], st["exp_avg_sq"], self.lr, b1, b2, self.eps,
                                       self.weight_decay, step)
        else:
            self._ops._CAPI_adamw_step_8bit.unbiased(self.params, grads, self.copies, st["exp_avg"], st["exp_avg_scale"], st["exp_avg_sq"],
                                                     st["exp_avg_sq_scale"], self.lr, b1, b2, self.eps, self.weight_decay, step, self.seed)

    def moments(self):
        """(first, second) moments as two flat float32 tensors, laid out like the state."""
        st = self.state
        if self.bits == 32:
            return st["exp_avg"], st["exp_avg_sq"]
        return (self._ops._CAPI_adamw_state_values(st["exp_avg"], st["exp_avg_scale"]),
                self._ops._CAPI_adamw_state_values(st["exp_avg_sq"], st["exp_avg_sq_scale"]))

    def state_dict(self):
        return {"steps": self.steps, "tensor_steps": list(self.tensor_steps), "bits": self.bits, "sizes": [p.numel() for p in self.params],
                "state": {k: v.clone() for k, v in self.state.items()}}

    def load_state_dict(self, saved):
        if saved["bits"] != self.bits or saved["sizes"] != [p.numel() for p in self.params]:
            raise ValueError("AdamW: the saved state is of other tensors or another number of bits")
        for k, v in self.state.items():
            v.copy_(saved["state"][k])
        self.steps = saved["steps"]
        # (a state without counts of its own is of the time when one stood for all tensors)
        self.tensor_steps = list(saved.get("tensor_steps", [self.steps] * len(self.params)))
