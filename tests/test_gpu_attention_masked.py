"""Causal sequences with numbers that are not finite at places that a query does not see: results that do not depend on them by the
definition are what they are without them (within the tolerances of test_gpu_attention.py)."""
import math

import pytest
import torch

from test_gpu_attention import definition, make, offsets

pytestmark = pytest.mark.gpu


def within(got, want, tol, rows, what):
    off = (got.double() - want).abs() / tol.clamp_min(1e-300)
    off = torch.where(torch.isinf(want), torch.where(got.double() == want, 0.0, math.nan), off)[rows]
    bad = off.amax().item() if off.numel() else 0.0  # (nan, where a value is, fails too)
    assert bad <= 1.0, "%s: %.3f of the tolerance" % (what, bad)


@pytest.mark.parametrize("bad", [math.inf, math.nan])
@pytest.mark.parametrize("dtype,heads,kv_heads,d", [(torch.bfloat16, 4, 2, 64), (torch.float16, 3, 3, 128), (torch.bfloat16, 2, 1, 40),
                                                    (torch.float32, 2, 1, 32)])
@pytest.mark.parametrize("lq,lk", [(300, 300), (40, 40), (129, 400), (400, 129), (8, 100)])
def test_what_a_query_does_not_see(ops, dtype, heads, kv_heads, d, lq, lk, bad):
    q_lens, k_lens = [30, lq, 1], [30, lk, 5]
    q, k, v, do = make(q_lens, k_lens, heads, kv_heads, d, dtype)
    if dtype == torch.float16:  # (the bound by which slopes are scaled is that of the first sequence, with or without the bad number)
        v[:30] *= 2.0
        do[:30] *= 2.0
    qo, ko, scale = offsets(q_lens), offsets(k_lens), d ** -0.5
    want, tol = definition(q, k, v, do, q_lens, k_lens, True, scale)
    i, j = torch.arange(lq, device="cuda"), torch.arange(lk, device="cuda")
    n, m = 31 + lq, 35 + lk
    for at in (0, 1, 7, 64, 100, 127, 128, 200, 299):
        for which in range(4):
            if at >= (lq if which in (0, 3) else lk):
                continue
            t = [x.clone() for x in (q, k, v, do)]
            t[which][30 + at, 0, 2] = bad
            out, lse = ops._CAPI_attention(*t[:3], qo, ko, True, scale)
            grads = ops._CAPI_attention_backward(t[3], *t[:3], out, lse, qo, ko, True, scale, True, True)
            rows, keys = torch.ones(n, dtype=torch.bool, device="cuda"), torch.ones(m, dtype=torch.bool, device="cuda")
            own_q, own_k = slice(30, 30 + lq), slice(30, 30 + lk)
            if which in (0, 3):  # of a query: its own row, and the keys that it sees
                rows[30 + at] = False
                keys[own_k] = j > at + lk - lq
            else:  # of a key: the queries that see it, and the keys that those see (the last one sees all)
                rows[own_q] = i + lk - lq < at
                keys[own_k] = False
            all_rows, all_keys = torch.ones_like(rows), torch.ones_like(keys)
            within(out, want["out"], tol["out"], all_rows if which == 3 else rows, ("out", at, which))
            seen = (all_rows if which > 1 else rows).expand(heads, n)
            within(lse, want["lse"], tol["lse"], seen, ("lse", at, which))
            for name, g, r in zip(("dq", "dk", "dv"), grads, (rows, keys, all_keys if which == 2 else keys)):
                within(g, want[name], tol[name], r, (name, at, which))
            # and what does depend on it shows it
            if which == 2 and 30 + at - (lk - lq) + 1 < 30 + lq:
                assert not out[30 + lq - 1].isfinite().all()
            # the same call gives the same bits
            again = ops._CAPI_attention_backward(t[3], *t[:3], out, lse, qo, ko, True, scale, True, True)
            for a, b in zip(grads, again):
                assert torch.equal(a.nan_to_num(7.0), b.nan_to_num(7.0))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_queries_that_see_no_key(ops, dtype):
    """Zeros for them, whatever they and the keys hold, and they give nothing to any gradient."""
    lq, lk = 200, 70
    q, k, v, do = make([lq], [lk], 4, 2, 64, dtype)
    want, tol = definition(q, k, v, do, [lq], [lk], True, 0.125)
    qo, ko = offsets([lq]), offsets([lk])
    for bad in (math.inf, math.nan):
        t = [x.clone() for x in (q, k, v, do)]
        t[0][:lq - lk], t[3][:lq - lk] = bad, bad
        out, lse = ops._CAPI_attention(*t[:3], qo, ko, True, 0.125)
        grads = ops._CAPI_attention_backward(t[3], *t[:3], out, lse, qo, ko, True, 0.125, True, True)
        assert (out[:lq - lk] == 0).all() and (lse[:, :lq - lk] == -math.inf).all() and (grads[0][:lq - lk] == 0).all()
        for name, x in zip(("out", "dq", "dk", "dv"), (out, *grads)):
            within(x, want[name], tol[name], torch.ones(x.shape[0], dtype=torch.bool, device="cuda"), name)
        # keys and values that are not finite leave them at zero
        t = [q, k.clone(), v.clone(), do]
        t[1][:], t[2][:] = bad, bad
        out, lse = ops._CAPI_attention(*t[:3], qo, ko, True, 0.125)
        dq = ops._CAPI_attention_backward(do, *t[:3], out, lse, qo, ko, True, 0.125, True, True)[0]
        assert (out[:lq - lk] == 0).all() and (lse[:, :lq - lk] == -math.inf).all() and (dq[:lq - lk] == 0).all()
        assert out[lq - lk:].isnan().any()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_a_step_that_went_wrong_altogether(ops, dtype):
    """Nothing but nan in one of the sequences: its results are nan, the others' bits are what they were."""
    lens = [100, 600, 40]
    q, k, v, do = make(lens, lens, 4, 2, 64, dtype)
    o = offsets(lens)

    def both(q, k, v, do):
        out, lse = ops._CAPI_attention(q, k, v, o, o, True, 0.125)
        return (out, *ops._CAPI_attention_backward(do, q, k, v, out, lse, o, o, True, 0.125, True, True))

    v[:100] *= 2.0  # (the bound by which float16 slopes are scaled is the first sequence's)
    do[:100] *= 2.0
    base = both(q, k, v, do)
    for which in ((0, 1, 2, 3), (0, 2), (2,), (3,)):
        t = [x.clone() for x in (q, k, v, do)]
        for i in which:
            t[i][100:700] = math.nan
        got = both(*t)
        for a, b in zip(got, base):
            assert torch.equal(a[:100], b[:100]) and torch.equal(a[700:], b[700:])
        assert got[1][100:700].isnan().all() and got[2][100:700].isnan().all()
        assert got[0][100:700].isnan().all() == (which != (3,)) and got[3][100:700].isnan().all() == (which != (2,))
