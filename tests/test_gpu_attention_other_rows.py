"""What a row of attention may depend on: its own sequence, in tiles too, which come whole from memory with the rows behind a sequence's
end (the next sequence's, or padding) in them.  The bits of a sequence are the same whatever numbers those rows hold."""
import pytest
import torch

from test_gpu_attention import make, offsets

pytestmark = pytest.mark.gpu


def both(ops, q, k, v, do, qo, ko, causal):
    scale = q.shape[2] ** -0.5
    out, lse = ops._CAPI_attention(q, k, v, qo, ko, causal, scale)
    return (out, lse, *ops._CAPI_attention_backward(do, q, k, v, out, lse, qo, ko, causal, scale, True, True))


def parts(res, nq, nk):
    out, lse, dq, dk, dv = res
    return out[:nq], lse[:, :nq], dq[:nq], dk[:nk], dv[:nk]


@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("heads,kv_heads", [(4, 2), (3, 3), (6, 2)])
@pytest.mark.parametrize("dtype,d", [(torch.bfloat16, 64), (torch.float16, 64), (torch.bfloat16, 128), (torch.float16, 100)])
def test_rows_behind_a_sequence(ops, dtype, d, heads, kv_heads, causal):
    nq, nk, behind = 300, 700, 150
    q, k, v, do = make([nq], [nk], heads, kv_heads, d, dtype, pad=behind)
    for padded in (True, False):  # rows of nobody; of another sequence
        lens = ([nq], [nk]) if padded else ([nq, behind], [nk, behind])
        qo, ko = (offsets(x) for x in lens)
        found = []
        for size in (0.0, 1.0, 40.0):
            # (fp16 scales slopes by a bound over all rows of the call: the largest gradients are those of the sequence itself)
            for t, n, most in ((q, nq, size), (k, nk, size), (v, nk, min(size, 0.5)), (do, nq, min(size, 0.5))):
                g = torch.Generator(device="cuda").manual_seed(3)
                t[n:] = (torch.randn(t[n:].shape, device="cuda", generator=g) * most).to(dtype)
            found.append([t.clone() for t in parts(both(ops, q, k, v, do, qo, ko, causal), nq, nk)])
        for other in found[1:]:
            for name, a, b in zip(("out", "lse", "dq", "dk", "dv"), found[0], other):
                assert torch.equal(a, b), (name, padded)
