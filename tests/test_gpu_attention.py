"""Attention over packed sequences, forward and backward, against the definition in 64 bits.

Tolerances follow from the arithmetic.  r = eps / 2 of the element type (one rounding), U = 2^-24.  A score is a sum of d products of
exact inputs, scaled: off by at most (d + 4) U scale sum |q||k|, and so are lse and, relative to it, p (call it s for the largest
of a row, with 16 U for exp2 and its argument's own rounding, |x| U).
  out   each p may be rounded to the element type before its product:        r |o| + (r + 2 s + n U) sum p |v|
  dv    likewise over the queries:                                           r |dv| + (r + 2 s + n U) sum p |do|
  ds    = p (e - delta); delta may come from the rounded out:  E = sum |do| (r |o| + (r + 2 s + n U) sum p |v|); rounded itself:
        dev = (r + 2 s + n U) p (|e| + |delta|) + p (E + n U sum|do||v|max)
  dq    r |dq| + scale sum_j dev |k|,  dk  r |dk| + scale sum_i dev |q|
(float32 operands and delta taken in 32 bits are held to the same, with r = U.)
Below the normal numbers roundings are absolute.  exp2 flushes weights under F = 2^-126 to 0, so every p may be off by F.  In fp16
half a step is 2^-25 at the most: the forward pass holds weights lifted by 2^4 or more (the row's largest is at least that), which leaves
2^-29 of p; the backward pass lifts them by 2^12, which leaves 2^-37, and scales ds so that its bound 2 B 2^12 s / 4 is between 2^14 and 2^15,
B the largest |do| times the largest |v| (norms of rows) of all sequences: 2^-25 of that is at most B 2^-40.  One smallest step for the
results' own rounding."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
ROUND = {torch.float32: U, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
TINY = {torch.float32: 2.0 ** -126, torch.bfloat16: 2.0 ** -126, torch.float16: 2.0 ** -24}


def offsets(lens, first=0, dtype=torch.int64):
    return torch.tensor([first] + lens, device="cuda").cumsum(0).to(dtype)


def make(q_lens, k_lens, heads, kv_heads, d, dtype, seed=0, pad=0, fused=False, spread=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    nq, nk = sum(q_lens) + pad, sum(k_lens) + pad

    def rand(*shape):
        return (torch.randn(shape, device="cuda", generator=g) * spread).to(dtype)

    if fused:
        both = rand(nq, heads + 2 * kv_heads, d)
        q, k, v = both[:, :heads], both[:, heads:heads + kv_heads], both[:, heads + kv_heads:]
    else:
        q, k, v = rand(nq, heads, d), rand(nk, kv_heads, d), rand(nk, kv_heads, d)
    return q, k, v, rand(nq, heads, d)


def definition(q, k, v, do, q_lens, k_lens, causal, scale):
    """Results and how far they may be off, in 64 bits."""
    r, dt = ROUND[q.dtype], q.dtype
    q, k, v, do = (t.double() for t in (q, k, v, do))
    (nq, h, d), (nk, hk, _) = q.shape, k.shape
    g = h // hk
    res = {n: torch.zeros_like(t) for n, t in (("out", q), ("dq", q), ("dk", k), ("dv", v))}
    tol = {n: torch.zeros_like(t) for n, t in res.items()}
    res["lse"] = torch.full((h, nq), -math.inf, device="cuda", dtype=torch.float64)
    tol["lse"] = torch.zeros_like(res["lse"])
    half = dt == torch.float16
    nq, nk = sum(q_lens), sum(k_lens)
    F = 2.0 ** -126
    floor_out, floor_p = F + 2.0 ** -29 * half, F + 2.0 ** -37 * half
    floor_ds = 2.0 ** -40 * half * do[:nq].norm(dim=2).amax() * v[:nk].norm(dim=2).amax() if nq and nk else 0.0
    a = c = 0
    for lq, lk in zip(q_lens, k_lens):
        A, C = slice(a, a + lq), slice(c, c + lk)
        a, c = a + lq, c + lk
        if lq == 0 or lk == 0:
            continue
        see = torch.ones(lq, lk, dtype=torch.bool, device="cuda")
        if causal:
            see = see.tril(lk - lq)
        live = see.any(1)
        for x in range(h):
            Q, K, V, D = q[A, x], k[C, x // g], v[C, x // g], do[A, x]
            s = (Q @ K.t()) * scale
            s = torch.where(see, s, -math.inf)
            top = torch.where(live, s.amax(1), 0.0)[:, None]
            p = torch.exp(s - top)
            under = p.sum(1, keepdim=True)
            p = torch.where(live[:, None], p / under, 0.0)
            lse = torch.where(live, top[:, 0] + under[:, 0].log(), -math.inf)
            o = p @ V
            e = D @ V.t()
            delta = (p * e).sum(1, keepdim=True)
            ds = p * (e - delta)
            off = ((d + 6) * U * abs(scale) * (Q.abs() @ K.abs().t()) * see).amax(1, keepdim=True) + 16 * U
            off = off + U * torch.where(live, lse.abs(), 0.0)[:, None]
            step = r + 2 * off
            res["out"][A, x], res["lse"][x, A] = o, lse
            tol["out"][A, x] = r * o.abs() + ((step + lk * U) * p + floor_out) @ V.abs()
            tol["lse"][x, A] = off[:, 0] * 2 + U * torch.where(live, lse.abs(), 0.0)
            res["dq"][A, x] = ds @ K * scale
            res["dk"][C, x // g] += ds.t() @ Q * scale
            res["dv"][C, x // g] += p.t() @ D
            tol["dv"][C, x // g] += ((step + (lq + 8) * U) * p + floor_p).t() @ D.abs()
            E = (D.abs() * (r * o.abs() + (step + (lk + d) * U) * (p @ V.abs()))).sum(1, keepdim=True)
            dev = ((step + (lk + lq + 8) * U) * p + floor_p) * (e.abs() + delta.abs()) + floor_ds + p * (E + (d + 4) * U * (D.abs() @ V.abs().t()))
            tol["dq"][A, x] = abs(scale) * (dev @ K.abs())
            tol["dk"][C, x // g] += abs(scale) * (dev.t() @ Q.abs())
    for n in ("dq", "dk", "dv"):
        tol[n] += r * res[n].abs()
    for n in ("out", "dq", "dk", "dv"):
        tol[n] += TINY[dt] * 2
    return res, tol


def compare(got, want, tol, what):
    inf = torch.isinf(want)
    assert torch.equal(torch.isinf(got), inf), what
    got, want = torch.where(inf, 0.0, got.double()), torch.where(inf, 0.0, want)
    over = (got - want).abs() / tol.clamp_min(1e-300)
    bad = over.amax().item() if over.numel() else 0.0  # (nan, where a value is, fails too)
    assert bad <= 1.0, "%s: %.3f of the tolerance" % (what, bad)


def check(ops, q, k, v, do, q_lens, k_lens, causal, scale=None, id_type=torch.int64):
    scale = q.shape[2] ** -0.5 if scale is None else scale
    qo, ko = offsets(q_lens, dtype=id_type), offsets(k_lens, dtype=id_type)
    out, lse = ops._CAPI_attention(q, k, v, qo, ko, causal, scale)
    dq, dk, dv = ops._CAPI_attention_backward(do, q, k, v, out, lse, qo, ko, causal, scale, True, True)
    torch.cuda.synchronize()
    want, tol = definition(q, k, v, do, q_lens, k_lens, causal, scale)
    for n, t in (("out", out), ("lse", lse), ("dq", dq), ("dk", dk), ("dv", dv)):
        compare(t, want[n], tol[n], n)
    return out, lse, dq, dk, dv


LENGTHS = {
    "one token": ([1], [1]),
    "seeds over neighbours": ([1] * 9, [0, 1, 2, 3, 15, 16, 17, 10, 5]),
    "short": ([3, 0, 7, 1, 16], [3, 4, 0, 1, 40]),
    "few queries, many keys": ([1, 2, 16, 1], [257, 1500, 300, 5000]),
    "around a tile": ([47, 48, 49, 127, 128, 129, 255, 256, 257], [47, 48, 49, 127, 128, 129, 255, 256, 257]),
    "queries and keys of other lengths": ([100, 300, 64, 500, 48], [130, 7, 500, 64, 1]),
    "long": ([700, 1], [700, 1]),
}


@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("lengths", list(LENGTHS))
@pytest.mark.parametrize("dtype,heads,kv_heads,d", [(torch.bfloat16, 4, 2, 64), (torch.float16, 2, 2, 128), (torch.float32, 3, 1, 32),
                                                    (torch.bfloat16, 6, 1, 40), (torch.float16, 8, 2, 16), (torch.float32, 2, 2, 100)])
def test_against_the_definition(ops, lengths, causal, dtype, heads, kv_heads, d):
    q_lens, k_lens = LENGTHS[lengths]
    check(ops, *make(q_lens, k_lens, heads, kv_heads, d, dtype), q_lens, k_lens, causal)


@pytest.mark.parametrize("d", [1, 3, 7, 33, 75, 127])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_odd_heads(ops, d, dtype):
    q_lens, k_lens = [5, 60, 1], [9, 70, 300]
    got = check(ops, *make(q_lens, k_lens, 2, 1, d, dtype, seed=d), q_lens, k_lens, True, id_type=torch.int32)
    assert all(t.is_contiguous() for t in got)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_parts_of_a_wider_tensor(ops, dtype):
    lens = [33, 150, 1, 8]
    q, k, v, do = make(lens, lens, 4, 2, 64, dtype, fused=True)
    got = check(ops, q, k, v, do, lens, lens, True)
    same = check(ops, q.contiguous(), k.contiguous(), v.contiguous(), do, lens, lens, True)
    assert all(torch.equal(a, b) for a, b in zip(got, same))
    # heads first in memory, an address off the 16-byte grid, one gradient for all rows
    turned = [t.transpose(0, 1).contiguous().transpose(0, 1) for t in (q, k, v, do)]
    same = check(ops, *turned, lens, lens, True)
    assert all(torch.equal(a, b) for a, b in zip(got, same))
    off = torch.empty(q.numel() + 1, dtype=dtype, device="cuda")[1:].view(q.shape).copy_(q)
    same = check(ops, off, k, v, do, lens, lens, True)
    assert all(torch.equal(a, b) for a, b in zip(got, same))
    check(ops, q, k, v, do[:1].expand_as(do), lens, lens, True)
    check(ops, q, k, v, do[:1, :1, :1].expand_as(do), lens, lens, True)


@pytest.mark.parametrize("dtype,d", [(torch.bfloat16, 64), (torch.float32, 32), (torch.float16, 128)])
@pytest.mark.parametrize("q_lens,k_lens", [([20, 130, 3], [20, 130, 3]), ([1, 1, 1], [40, 700, 2])])
def test_rows_outside_of_all_sequences(ops, dtype, d, q_lens, k_lens):
    """Padding rows hold anything; results there are 0 and no other row sees them."""
    q, k, v, do = make(q_lens, k_lens, 2, 1, d, dtype, pad=9)
    base = check(ops, q, k, v, do, q_lens, k_lens, False)
    for bad in (math.nan, math.inf):
        q2, k2, v2, do2 = (t.clone() for t in (q, k, v, do))
        for t in (q2, k2, v2, do2):
            t[-9:] = bad
        scale = d ** -0.5
        qo, ko = offsets(q_lens), offsets(k_lens)
        out, lse = ops._CAPI_attention(q2, k2, v2, qo, ko, False, scale)
        grads = ops._CAPI_attention_backward(do2, q2, k2, v2, out, lse, qo, ko, False, scale, True, True)
        assert all(torch.equal(a, b) for a, b in zip(base, (out, lse, *grads)))
        assert (out[-9:] == 0).all() and (lse[:, -9:] == -math.inf).all() and all((t[-9:] == 0).all() for t in grads)
    # sequences that begin behind rows of nobody
    shift = lambda t: torch.cat([torch.full_like(t[:5], math.nan), t[:-9]])  # noqa: E731
    out, lse = ops._CAPI_attention(shift(q), shift(k), shift(v), offsets(q_lens, 5), offsets(k_lens, 5), False, d ** -0.5)
    grads = ops._CAPI_attention_backward(shift(do), shift(q), shift(k), shift(v), out, lse, offsets(q_lens, 5), offsets(k_lens, 5), False,
                                         d ** -0.5, True, True)
    for a, b in zip((out, *grads), (base[0], *base[2:])):
        assert torch.equal(a[5:], b[:-9]) and (a[:5] == 0).all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_a_sequence_that_is_not_finite_leaves_the_others(ops, dtype):
    lens = [30, 100, 64, 2]
    q, k, v, do = make(lens, lens, 2, 2, 64, dtype)
    base = check(ops, q, k, v, do, lens, lens, True)
    bad = [t.clone() for t in (q, k, v, do)]
    for t in bad:
        t[30:130] = math.nan
    qo = offsets(lens)
    out, lse = ops._CAPI_attention(*bad[:3], qo, qo, True, 0.125)
    grads = ops._CAPI_attention_backward(bad[3], *bad[:3], out, lse, qo, qo, True, 0.125, True, True)
    for a, b in zip((out, *grads), (base[0], *base[2:])):
        assert torch.equal(a[:30], b[:30]) and torch.equal(a[130:], b[130:]) and a[30:130].isnan().any()


@pytest.mark.parametrize("dtype,d", [(torch.bfloat16, 64), (torch.float32, 64), (torch.float16, 128)])
def test_large_scores(ops, dtype, d):
    """Scores of hundreds: the largest of a row grows from tile to tile, most weights vanish."""
    lens = [300, 20, 1]
    q, k, v, do = make(lens, lens, 2, 1, d, dtype, spread=6.0)
    k = (k.double() * torch.linspace(0.1, 2.0, k.shape[0], device="cuda")[:, None, None]).to(dtype)
    check(ops, q, k, v, do, lens, lens, False)
    check(ops, q, k, v, do, lens, lens, True, scale=0.5)
    check(ops, q, k, v, do, lens, lens, False, scale=0.0)
    check(ops, q, k, v, do, lens, lens, False, scale=-0.1)


@pytest.mark.parametrize("size", [1e-6, 1e-3, 1e3])
def test_small_and_large_gradients_in_fp16(ops, size):
    lens = [200, 20, 600]
    q, k, v, do = make(lens, lens, 2, 1, 64, torch.float16)
    do = (do.double() * size).half()
    check(ops, q, k, v, do, lens, lens, False)


def test_the_same_inputs_give_the_same_bits(ops):
    q_lens, k_lens = [1, 300, 20, 1, 129], [3000, 300, 20, 7, 1000]
    q, k, v, do = make(q_lens, k_lens, 4, 2, 64, torch.bfloat16)
    qo, ko = offsets(q_lens), offsets(k_lens)

    def both():
        out, lse = ops._CAPI_attention(q, k, v, qo, ko, False, 0.125)
        return (out, lse, *ops._CAPI_attention_backward(do, q, k, v, out, lse, qo, ko, False, 0.125, True, True))

    base = both()
    for _ in range(5):
        assert all(torch.equal(a, b) for a, b in zip(base, both()))
    # either gradient alone
    dq, dk, dv = ops._CAPI_attention_backward(do, q, k, v, base[0], base[1], qo, ko, False, 0.125, True, False)
    assert torch.equal(dq, base[2]) and dk.shape[0] == 0 and dv.shape[0] == 0
    dq, dk, dv = ops._CAPI_attention_backward(do, q, k, v, base[0], base[1], qo, ko, False, 0.125, False, True)
    assert dq.shape[0] == 0 and torch.equal(dk, base[3]) and torch.equal(dv, base[4])


@pytest.mark.parametrize("dtype,d", [(torch.bfloat16, 64), (torch.float16, 128)])
@pytest.mark.parametrize("causal", [False, True])
def test_either_gradient_alone(ops, dtype, d, causal):
    """In tiles of which none, some and all rows see one tile of keys at the most: the same bits as both together."""
    q_lens, k_lens = [24, 128, 129, 130, 300, 40, 200, 256, 30], [24, 128, 127, 140, 300, 400, 0, 128, 1]
    q, k, v, do = make(q_lens, k_lens, 4, 2, d, dtype)
    qo, ko = offsets(q_lens), offsets(k_lens)
    out, lse, dq, dk, dv = check(ops, q, k, v, do, q_lens, k_lens, causal)
    args = (do, q, k, v, out, lse, qo, ko, causal, d ** -0.5)
    assert torch.equal(ops._CAPI_attention_backward(*args, True, False)[0], dq)
    for got, want in zip(ops._CAPI_attention_backward(*args, False, True)[1:], (dk, dv)):
        assert torch.equal(got, want)


@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("length", [24, 40, 100, 128])
def test_gradients_of_short_sequences_are_rounded_twice_at_most(ops, dtype, length, causal):
    """dq and dk in the 2-norm.  Two independent roundings, dS's and the result's, are sqrt(2) = 1.414 times the error of rounding the exact
    gradients; over the 40 * 4 * length * 64 values here the ratio's own spread is below 1 %: at most 1.45."""
    lens = [length] * 40
    q, k, v, do = make(lens, lens, 4, 4, 64, dtype)
    o = offsets(lens)
    out, lse = ops._CAPI_attention(q, k, v, o, o, causal, 0.125)
    got = ops._CAPI_attention_backward(do, q, k, v, out, lse, o, o, causal, 0.125, True, True)
    w = [t.double().view(40, length, 4, 64).transpose(1, 2) for t in (q, k, v, do)]
    x = w[0] @ w[1].transpose(2, 3) * 0.125
    if causal:
        x = x.masked_fill(torch.ones(length, length, dtype=torch.bool, device="cuda").triu(1), -math.inf)
    p = x.softmax(-1)
    e = w[3] @ w[2].transpose(2, 3)
    ds = p * (e - (p * e).sum(-1, keepdim=True)) * 0.125
    for t, want in ((got[0], ds @ w[1]), (got[1], ds.transpose(2, 3) @ w[0])):
        want = want.transpose(1, 2).reshape(t.shape)
        assert (t.double() - want).norm() <= 1.45 * (want.to(dtype).double() - want).norm()


def test_many_sequences(ops):
    """More than one CTA makes the plan of; a long one among them."""
    g = torch.Generator().manual_seed(1)
    k_lens = torch.randint(0, 16, (5000,), generator=g).tolist()
    q_lens = [1] * 5000
    q_lens[777], k_lens[777], k_lens[4000] = 60, 90, 2500
    q, k, v, do = make(q_lens, k_lens, 2, 2, 32, torch.bfloat16)
    qo, ko = offsets(q_lens), offsets(k_lens)
    out, lse = ops._CAPI_attention(q, k, v, qo, ko, False, 0.2)
    dq, dk, dv = ops._CAPI_attention_backward(do, q, k, v, out, lse, qo, ko, False, 0.2, True, True)
    # the same sequences in pieces that one CTA plans
    for a, b in ((0, 700), (700, 900), (3900, 4100)):
        A, C = slice(qo[a], qo[b]), slice(ko[a], ko[b])
        got = check(ops, q[A], k[C], v[C], do[A], q_lens[a:b], k_lens[a:b], False, scale=0.2)
        for x, y in zip(got, (out[A], lse[:, A], dq[A], dk[C], dv[C])):
            assert torch.equal(x, y)


@pytest.mark.parametrize("n", [255, 257, 511, 512, 513, 1000, 1024, 1025, 2500])
def test_a_row_is_split_by_its_own_keys(ops, n):
    """One long row among short ones, in batches of which one is twice the other: as both have few keys a sequence on average, lanes are
    shared out alike, and in 32 bits, where the order of a sum shows, its values and gradients are the same bits."""
    found = []
    for seqs in (1501, 3001):
        q_lens, k_lens = [1] * seqs, [i % 7 for i in range(seqs)]
        k_lens[700] = n
        g = torch.Generator(device="cuda").manual_seed(n)
        q, k, v, do = make(q_lens, k_lens, 4, 2, 32, torch.float32, seed=seqs)
        at = sum(k_lens[:700])
        for t, rows in ((q, slice(700, 701)), (k, slice(at, at + n)), (v, slice(at, at + n)), (do, slice(700, 701))):
            t[rows] = torch.randn(t[rows].shape, device="cuda", generator=g)
        qo, ko = offsets(q_lens), offsets(k_lens)
        out, lse = ops._CAPI_attention(q, k, v, qo, ko, False, 0.2)
        dq, dk, dv = ops._CAPI_attention_backward(do, q, k, v, out, lse, qo, ko, False, 0.2, True, True)
        found.append((out[700], lse[:, 700], dq[700], dk[at:at + n], dv[at:at + n]))
    for x, y in zip(*found):
        assert torch.equal(x, y)


def test_nothing_to_do(ops):
    q, k, v, do = make([3, 2], [4, 1], 2, 1, 16, torch.float32)
    none = torch.zeros(1, dtype=torch.int64, device="cuda")
    out, lse = ops._CAPI_attention(q, k, v, none, none, False, 1.0)
    assert (out == 0).all() and (lse == -math.inf).all()
    for t in ops._CAPI_attention_backward(do, q, k, v, out, lse, none, none, False, 1.0, True, True):
        assert (t == 0).all()
    o = offsets([0, 0])
    out, lse = ops._CAPI_attention(q[:0], k, v, o, o, True, 1.0)
    assert out.shape == (0, 2, 16) and lse.shape == (2, 0)
    dq, dk, dv = ops._CAPI_attention_backward(do[:0], q[:0], k, v, out, lse, o, o, True, 1.0, True, True)
    assert dq.shape[0] == 0 and (dk == 0).all() and (dv == 0).all()
    out, lse = ops._CAPI_attention(q, k[:0], v[:0], offsets([3, 2]), o, False, 1.0)
    assert (out == 0).all()
    dq, dk, dv = ops._CAPI_attention_backward(do, q, k[:0], v[:0], out, lse, offsets([3, 2]), o, False, 1.0, True, True)
    assert (dq == 0).all() and dk.shape == (0, 1, 16)


def test_autograd_and_differences(pkg):
    lens = [7, 1, 12]
    q, k, v, do = (t.requires_grad_(i < 3) for i, t in enumerate(make(lens, lens, 4, 2, 8, torch.float32)))
    o = offsets(lens)
    out, lse = pkg.attention(q, k, v, o, causal=True, return_lse=True)
    assert not lse.requires_grad
    out.backward(do)
    want, tol = definition(q.detach(), k.detach(), v.detach(), do, lens, lens, True, 8 ** -0.5)
    for t, n in ((q, "dq"), (k, "dk"), (v, "dv")):
        compare(t.grad, want[n], tol[n], n)
    # central differences of the loss along random directions; third derivatives of some 10 leave 10 h^2, rounding 2^-22 |loss| / h
    g = torch.Generator(device="cuda").manual_seed(5)
    with torch.no_grad():
        for t in (q, k, v):
            way = torch.randn(t.shape, device="cuda", generator=g)
            way /= way.norm()
            h = 2.0 ** -6
            ends = []
            for sign in (1, -1):
                at = [x if x is not t else x + sign * h * way for x in (q, k, v)]
                ends.append((pkg.attention(*at, o, causal=True).double() * do.double()).sum())
            slope = (ends[0] - ends[1]) / (2 * h)
            size = (pkg.attention(q, k, v, o, causal=True).double() * do.double()).abs().sum()
            assert (slope - (t.grad.double() * way.double()).sum()).abs() <= 10 * h * h + 2.0 ** -20 * size / h
    # only what wants a gradient gets one
    a = v.detach().clone().requires_grad_()
    pkg.attention(q.detach(), k.detach(), a, o, causal=True).backward(do)
    assert torch.equal(a.grad, v.grad)


def test_a_blocks_neighbours(pkg, ops):
    """The seeds of a sampled block over their neighbours, from its CSC form."""
    n_dst, n_src = 40, 90
    g = torch.Generator().manual_seed(3)
    row = torch.randint(0, n_dst, (300,), generator=g).sort().values.cuda()
    col = torch.randint(0, n_src, (300,), generator=g).cuda()
    indptr, indices = pkg.block_csc(row, col, n_dst)
    q, k, v, do = make([n_dst], [n_src], 2, 2, 32, torch.float32)
    out = pkg.attention(q, k[indices], v[indices], torch.arange(n_dst + 1, device="cuda"), indptr)
    lens = (indptr[1:] - indptr[:-1]).tolist()
    want, tol = definition(q, k[indices], v[indices], do, [1] * n_dst, lens, False, 32 ** -0.5)
    compare(out, want["out"], tol["out"], "out")


def test_bad_offsets_are_reported(ops, monkeypatch):
    q, k, v, do = make([4, 4], [6, 6], 1, 1, 16, torch.float32)
    good, ko = offsets([4, 4]), offsets([6, 6])
    for bad in ([0, 4, 9], [0, 6, 4], [-1, 4, 8], [0, 4, 1 << 40]):
        b = torch.tensor(bad, device="cuda")
        out, lse = ops._CAPI_attention(q, k, v, b, ko, False, 0.25)
        torch.cuda.synchronize()
        with pytest.raises(RuntimeError, match="_CAPI_attention"):
            ops._CAPI_attention(q, k, v, good, ko, False, 0.25)
        assert out.isfinite().all()
    out, lse = ops._CAPI_attention(q, k, v, good, ko, False, 0.25)
    ops._CAPI_attention_backward(do, q, k, v, out, lse, good, torch.tensor([0, 6, 13], device="cuda"), False, 0.25, True, True)
    torch.cuda.synchronize()
    with pytest.raises(RuntimeError, match="_CAPI_attention_backward"):
        ops._CAPI_attention(q, k, v, good, ko, False, 0.25)
    ops._CAPI_attention(q, k, v, good, ko, False, 0.25)


def test_recorded_and_replayed(ops):
    """Forward and backward in a CUDA graph, with offsets and values that change between replays; two graphs and an eager call at once."""
    q_lens, k_lens = [1, 300, 20, 1], [3000, 300, 20, 7]
    q, k, v, do = make(q_lens, k_lens, 4, 2, 64, torch.bfloat16)
    qo, ko = offsets(q_lens), offsets(k_lens)

    def both():
        out, lse = ops._CAPI_attention(q, k, v, qo, ko, False, 0.125)
        return (out, lse, *ops._CAPI_attention_backward(do, q, k, v, out, lse, qo, ko, False, 0.125, True, True))

    both()
    torch.cuda.synchronize()
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            res = both()
        graphs.append((g, res))
    for seed, lens in ((1, [20, 1, 300, 1]), (2, [300, 20, 1, 1])):
        for t, n in zip((q, k, v, do), make(q_lens, k_lens, 4, 2, 64, torch.bfloat16, seed=seed)):
            t.copy_(n)
        qo.copy_(offsets(lens))
        want = both()
        for g, res in graphs:
            g.replay()
        torch.cuda.synchronize()
        for g, res in graphs:
            assert all(torch.equal(a, b) for a, b in zip(res, want))


def test_many_calls_in_flight(ops):
    """Calls queued one behind the other, each with several tiles for every SM: no wait of theirs may run out."""
    lens = [2048] * 4
    q, k, v, do = make(lens, lens, 8, 4, 128, torch.bfloat16)
    o = offsets(lens)
    out, lse = ops._CAPI_attention(q, k, v, o, o, True, 0.1)
    base = ops._CAPI_attention_backward(do, q, k, v, out, lse, o, o, True, 0.1, True, True)
    for _ in range(100):
        last = ops._CAPI_attention_backward(do, q, k, v, out, lse, o, o, True, 0.1, True, True)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(base, last))
    again = ops._CAPI_attention(q, k, v, o, o, True, 0.1)  # (an error of an earlier call would be raised here)
    assert torch.equal(again[0], out)


def test_on_another_stream(ops):
    lens = [200, 3, 1]
    q, k, v, do = make(lens, lens, 2, 2, 64, torch.bfloat16)
    o = offsets(lens)
    base = ops._CAPI_attention(q, k, v, o, o, True, 0.1)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = ops._CAPI_attention(q, k, v, o, o, True, 0.1)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(base, got))


def test_refusals(ops):
    q, k, v, do = make([4], [6], 4, 2, 16, torch.float32)
    o = offsets([4])
    good = dict(q=q, k=k, v=v, qo=o, ko=offsets([6]), scale=0.25)

    def call(**kw):
        a = dict(good, **kw)
        return ops._CAPI_attention(a["q"], a["k"], a["v"], a["qo"], a["ko"], False, a["scale"])

    for kw, text in ((dict(k=k.bfloat16()), "one type"), (dict(q=q.double()), "float32, bfloat16 or float16"), (dict(k=k[:5]), "one shape"),
                     (dict(k=k[..., :8], v=v[..., :8]), "same number"), (dict(q=q[:, :3]), "multiple of the key heads"),
                     (dict(q=q[0]), r"\[rows, heads, d\]"), (dict(qo=o.float(), ko=o.float()), "int"), (dict(qo=offsets([4, 0])), "each sequence"),
                     (dict(qo=o.int()), "share one type"), (dict(qo=o[:0], ko=o[:0]), "each sequence"), (dict(scale=math.inf), "finite"),
                     (dict(qo=o.cpu()), "must be on"), (dict(k=k.cpu()), "must be on")):
        with pytest.raises(RuntimeError, match=text):
            call(**kw)
    wide = torch.zeros(4, 1, 136, device="cuda")
    with pytest.raises(RuntimeError, match="1 to 128"):
        ops._CAPI_attention(wide, wide, wide, o, o, False, 0.1)
    out, lse = call()
    for g, o2, l2 in ((do[:3], out, lse), (do.half(), out, lse), (do, out[:, :1], lse), (do, out, lse[:, :3]), (do, out, lse.double())):
        with pytest.raises(RuntimeError, match="must"):
            ops._CAPI_attention_backward(g, q, k, v, o2, l2, o, offsets([6]), False, 0.25, True, True)
