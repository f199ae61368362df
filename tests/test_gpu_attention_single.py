"""Gradients of single queries over a few keys (a seed over its sampled neighbours).

Everything but the results is in 32 bits, so in 16 bits the error of dq, dk and dv is that of rounding the exact gradients and little
besides.  In the 2-norm: rounding leaves 2^-9 / sqrt(3) (bf16; fp16 2^-12 / sqrt(3)) of a value or more than half of that.  A slope
p (e - delta) is off by some sqrt(d) 2^-24 |do| |v| in the mean: with a common mean of 3 in v and do and d = 64 that is 8 * 2^-24 * 640 against
slopes of 25, 1.2e-5 of them, while half of 2^-12 / sqrt(3) is 7e-5: at most sqrt(1 + 0.17^2) = 1.015 times; exp2, its argument and lse leave
2^-21 of a weight, less than that.  1.05 is asked for."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu


def gradients(q, k, v, do, seqs, keys, group, scale):
    """dq, dk, dv in 64 bits of `seqs` single queries over as many keys each."""
    d = q.shape[2]
    q, do = (t.double().view(seqs, -1, group, d) for t in (q, do))  # [seq, key head, of the group, d]
    k, v = (t.double().view(seqs, keys, -1, d) for t in (k, v))
    p = (torch.einsum("scgd,sjcd->scgj", q, k) * scale).softmax(-1)
    e = torch.einsum("scgd,sjcd->scgj", do, v)
    ds = p * (e - (p * e).sum(-1, keepdim=True)) * scale
    return (torch.einsum("scgj,sjcd->scgd", ds, k).reshape(seqs, -1, d), torch.einsum("scgj,scgd->sjcd", ds, q).reshape(seqs * keys, -1, d),
            torch.einsum("scgj,scgd->sjcd", p, do).reshape(seqs * keys, -1, d))


@pytest.mark.parametrize("mean", [0.0, 1.0, 3.0])
@pytest.mark.parametrize("keys", [1, 2, 4, 15, 16, 17, 33, 64, 65, 130, 512])
@pytest.mark.parametrize("dtype,heads,kv_heads,d", [(torch.bfloat16, 4, 4, 64), (torch.bfloat16, 4, 2, 64), (torch.float16, 4, 1, 64),
                                                    (torch.float16, 2, 2, 128), (torch.bfloat16, 3, 1, 32)])
def test_rounded_once(ops, dtype, heads, kv_heads, d, keys, mean):
    seqs, scale = max(40, 2000 // keys), d ** -0.5
    g = torch.Generator(device="cuda").manual_seed(keys)

    def rand(rows, h, shift=0.0):
        return (torch.randn((rows, h, d), device="cuda", generator=g) + shift).to(dtype)

    q, k, v, do = rand(seqs, heads), rand(seqs * keys, kv_heads), rand(seqs * keys, kv_heads, mean), rand(seqs, heads, mean)
    qo, ko = torch.arange(seqs + 1, device="cuda"), torch.arange(seqs + 1, device="cuda") * keys
    out, lse = ops._CAPI_attention(q, k, v, qo, ko, False, scale)
    got = ops._CAPI_attention_backward(do, q, k, v, out, lse, qo, ko, False, scale, True, True)
    for name, t, want in zip(("dq", "dk", "dv"), got, gradients(q, k, v, do, seqs, keys, heads // kv_heads, scale)):
        if keys == 1 and name != "dv":
            # one key has the weight 1 and no slope: e - delta is at most what 32 bits leave of sum |do||v| ((d + 4) roundings of each)
            bound = (2 * d + 40) * 2.0 ** -24 * (do.double().abs().amax() * v.double().abs().amax() * d) * scale
            assert t.double().abs().amax() <= bound * (k if name == "dq" else q).double().abs().amax() * (heads // kv_heads)
            continue
        # (fp16: what is below its normal numbers is rounded by half of 2^-24, here as there)
        rounded = want.to(dtype).double()
        if torch.equal(rounded, want):  # (dv of one key and one head is do: its weight 1 within 2^-20, so the nearest number is do itself)
            assert torch.equal(t.double(), want), name
            continue
        ratio = ((t.double() - want).norm() / (rounded - want).norm()).item()
        assert ratio <= 1.05, "%s: %.3f" % (name, ratio)


@pytest.mark.parametrize("lengths", [[0, 1, 513, 2, 512, 100], [3] * 300 + [400], [20] * 50 + [0] * 50])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("heads,kv_heads", [(8, 8), (6, 2), (4, 1), (5, 5)])
def test_mixed_lengths_and_either_gradient_alone(ops, lengths, dtype, heads, kv_heads):
    d, n = 24, len(lengths)
    g = torch.Generator(device="cuda").manual_seed(n)

    def rand(rows, h):
        return torch.randn((rows, h, d), device="cuda", generator=g).to(dtype)

    q, k, v, do = rand(n, heads), rand(sum(lengths), kv_heads), rand(sum(lengths), kv_heads), rand(n, heads)
    qo = torch.arange(n + 1, device="cuda")
    ko = torch.tensor([0] + lengths, device="cuda").cumsum(0)
    out, lse = ops._CAPI_attention(q, k, v, qo, ko, False, 0.3)
    args = (do, q, k, v, out, lse, qo, ko, False, 0.3)
    dq, dk, dv = ops._CAPI_attention_backward(*args, True, True)
    assert torch.equal(ops._CAPI_attention_backward(*args, True, False)[0], dq)
    for a, b in zip(ops._CAPI_attention_backward(*args, False, True)[1:], (dk, dv)):
        assert torch.equal(a, b)
    at = 0
    for i, m in enumerate(lengths):
        s = slice(at, at + m)
        at += m
        if m == 0:
            assert (dq[i] == 0).all()
            continue
        # sums of up to 512 terms of some 24 products each, in 32 bits, and one rounding (2^-8 in bf16)
        room = (512 + 64) * 2.0 ** -24 + (2.0 ** -8 if dtype == torch.bfloat16 else 0.0)
        for t, want in zip((dq[i:i + 1], dk[s], dv[s]), gradients(q[i:i + 1], k[s], v[s], do[i:i + 1], 1, m, heads // kv_heads, 0.3)):
            assert (t.double() - want).abs().amax() <= room * max(1.0, want.abs().amax().item())
