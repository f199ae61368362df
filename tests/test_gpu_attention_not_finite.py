"""A sequence with numbers that are not finite, beside others: their bits are what they are without it, in float16 too, whose slopes are scaled by
a bound over all rows of a call."""
import math

import pytest
import torch

from test_gpu_attention import make, offsets

pytestmark = pytest.mark.gpu


def both(ops, q, k, v, do, qo, ko, causal):
    scale = q.shape[2] ** -0.5
    out, lse = ops._CAPI_attention(q, k, v, qo, ko, causal, scale)
    return (out, lse, *ops._CAPI_attention_backward(do, q, k, v, out, lse, qo, ko, causal, scale, True, True))


@pytest.mark.parametrize("bad", [math.inf, -math.inf, math.nan])
@pytest.mark.parametrize("dtype,d", [(torch.float16, 64), (torch.float16, 128), (torch.bfloat16, 64)])
@pytest.mark.parametrize("size", [1e-4, 1.0])
def test_a_sequence_that_is_not_finite(ops, dtype, d, bad, size):
    """A gradient or value of one sequence that is not finite changes no bit of the others', small gradients in fp16 included."""
    lens = [200, 130, 64, 500]
    q, k, v, do = make(lens, lens, 4, 2, d, dtype)
    do = (do.float() * size).to(dtype)
    v[200:330] *= 0.5
    do[200:330] *= 0.5
    o = offsets(lens)
    base = both(ops, q, k, v, do, o, o, True)
    for which in range(4):
        t = [x.clone() for x in (q, k, v, do)]
        t[which][250, 1, 3] = bad
        got = both(ops, *t, o, o, True)
        for name, a, b in zip(("out", "dq", "dk", "dv"), (got[0], *got[2:]), (base[0], *base[2:])):
            assert torch.equal(a[:200], b[:200]) and torch.equal(a[330:], b[330:]), (name, which)
