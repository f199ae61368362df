"""AdamW over lists of tensors against the definition: in 64 bits with derived tolerances, and operation by operation in 32
bits on the host, whose bits the kernel has to give (every operation is rounded to nearest on both sides)."""
import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
ROUND = {torch.float32: U, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
HYPER = (1e-2, 0.9, 0.99, 1e-8, 0.1)
SIZES = [[1], [255, 256, 257], [7, 2048, 2049, 1, 100_003], [5000] * 3 + [0, 12], [33] * 70, [300] * 600, [1_000_001]]


def slots(sizes):
    starts, at = [], 0
    for n in sizes:
        starts.append(at)
        at += -(-n // 256) * 256
    return starts, at


def make(sizes, ptype, gtype, ctype, seed=0, odd=0):
    """Tensors of a list; odd: each begins that many elements into its own allocation."""
    g = torch.Generator(device="cuda").manual_seed(seed)

    def rand(n, scale, dtype):
        return (torch.randn(n + odd, device="cuda", generator=g) * scale).to(dtype)[odd:]
    p = [rand(n, 0.1, ptype) for n in sizes]
    gr = [rand(n, 0.01, gtype) for n in sizes]
    c = [torch.full((n + odd,), 7.0, device="cuda", dtype=ctype)[odd:] for n in sizes] if ctype is not None else []
    starts, total = slots(sizes)
    m, v = torch.zeros(total, device="cuda"), torch.zeros(total, device="cuda")
    for a, n in zip(starts, sizes):
        m[a:a + n] = rand(n, 0.005, torch.float32)
        v[a:a + n] = rand(n, 0.01, torch.float32).square()
    return p, gr, c, m, v


def step32(p, g, m, v, step, hyper=HYPER):
    """The formula in float32, an operation at a time, on the host."""
    lr, b1, b2, eps, wd = hyper
    f = np.float32
    p, g, m, v = (x.float().cpu().numpy() for x in (p, g, m, v))
    m = m * f(b1) + g * f(1 - b1)
    v = v * f(b2) + g * g * f(1 - b2)
    under = np.sqrt(v) * f(1 / math.sqrt(1 - b2 ** step)) + f(eps)
    return p * f(1 - lr * wd) - m / under * f(lr / (1 - b1 ** step)), m, v


def same(t, a):
    return torch.equal(t.cpu(), torch.from_numpy(np.ascontiguousarray(a)).to(t.dtype))


@pytest.mark.parametrize("sizes", SIZES)
@pytest.mark.parametrize("types", [(torch.float32, torch.float32, None), (torch.float32, torch.bfloat16, torch.bfloat16),
                                   (torch.bfloat16, torch.float16, torch.float32), (torch.float16, torch.float16, None)])
@pytest.mark.parametrize("odd", [0, 1])
def test_step_32bit(ops, sizes, types, odd):
    p, g, c, m, v = make(sizes, *types, odd=odd)
    want = [step32(x, y, m[a:a + x.numel()], v[a:a + x.numel()], 3) for x, y, a in zip(p, g, slots(sizes)[0])]
    old = [x.double() for x in p], m.double(), v.double()
    ops._CAPI_adamw_step(p, g, c, m, v, *HYPER, 3)
    lr, b1, b2, eps, wd = HYPER
    for i, (x, a) in enumerate(zip(p, slots(sizes)[0])):
        n = x.numel()
        assert same(x, want[i][0]) and same(m[a:a + n], want[i][1]) and same(v[a:a + n], want[i][2])
        if c:
            assert same(c[i], want[i][0])
        # 64 bits: a handful of roundings, each u of its own operands, and the type's rounding
        gd = g[i].double()
        md = old[1][a:a + n] * b1 + gd * (1 - b1)
        vd = old[2][a:a + n] * b2 + gd * gd * (1 - b2)
        upd = lr / (1 - b1 ** 3) * md / (vd.sqrt() / math.sqrt(1 - b2 ** 3) + eps)
        pd = old[0][i] * (1 - lr * wd) - upd
        size = (old[1][a:a + n].abs() * b1 + gd.abs() * (1 - b1)) / md.abs().clamp_min(1e-300)
        tol = 12 * U * (pd.abs() + old[0][i].abs()) + 12 * U * upd.abs() * (1 + size) + ROUND[x.dtype] * pd.abs() + 2.0 ** -25
        assert ((x.double() - pd).abs() <= tol).all()
    assert all((m[a + n:b] == 0).all() for a, n, b in zip(slots(sizes)[0], sizes, slots(sizes)[0][1:] + [m.numel()]))


def codes32(m, v):
    """8-bit codes and scales of one block's moments, in float32 on the host."""
    f = np.float32
    r = np.sqrt(v)
    ma, ra = np.abs(m).max(), r.max()
    with np.errstate(divide="ignore", invalid="ignore"):
        tm = np.sqrt(np.abs(m) / ma) if ma > 0 else np.zeros_like(m)
        tv = np.sqrt(r / ra) if ra > 0 else np.zeros_like(r)
    cm = np.rint(tm * f(127)) * np.sign(m)
    cv = np.rint(tv * f(255))
    cv = np.where((r > 0) & (cv < 1), f(1), cv)
    return cm.astype(np.int8), ma, cv.astype(np.uint8), ra


def values32(mc, ma, vc, ra):
    f = np.float32
    c = mc.astype(f) * f(1.0 / 127.0)
    d = vc.astype(f) * f(1.0 / 255.0)
    r = d * d * f(ra)
    return c * np.abs(c) * f(ma), r * r


@pytest.mark.parametrize("sizes", [[1], [255, 256, 257], [7, 2048, 2049, 1, 20_003], [33] * 70, [0, 300]])
@pytest.mark.parametrize("types", [(torch.float32, torch.float32, None), (torch.float32, torch.bfloat16, torch.bfloat16),
                                   (torch.bfloat16, torch.bfloat16, None)])
@pytest.mark.parametrize("odd", [0, 3])
def test_steps_8bit(ops, sizes, types, odd):
    p, g, c, _, _ = make(sizes, *types, odd=odd)
    starts, total = slots(sizes)
    mc, vc = torch.zeros(total, dtype=torch.int8, device="cuda"), torch.zeros(total, dtype=torch.uint8, device="cuda")
    ms, vs = torch.zeros(total // 256, device="cuda"), torch.zeros(total // 256, device="cuda")
    hp = [x.float().cpu() for x in p]
    hm, hv = np.zeros(total, np.float32), np.zeros(total, np.float32)
    for step in (1, 2, 3):
        if step == 2:
            g = [x * 0.3 for x in g]
        ops._CAPI_adamw_step_8bit(p, g, c, mc, ms, vc, vs, *HYPER, step)
        for i, (a, n) in enumerate(zip(starts, sizes)):
            new, m, v = step32(hp[i], g[i], torch.from_numpy(hm[a:a + n]), torch.from_numpy(hv[a:a + n]), step)
            assert same(p[i], new)
            hp[i] = p[i].float().cpu()
            hm[a:a + n], hv[a:a + n] = m, v
        for b in range(total // 256):
            at = slice(b * 256, b * 256 + 256)
            want = codes32(hm[at], hv[at])
            assert np.array_equal(mc[at].cpu().numpy(), want[0]) and np.array_equal(vc[at].cpu().numpy(), want[2])
            assert ms[b].item() == want[1] and vs[b].item() == want[3]
            hm[at], hv[at] = values32(*want)
        assert same(ops._CAPI_adamw_state_values(mc, ms), hm) and same(ops._CAPI_adamw_state_values(vc, vs), hv)


def test_8bit_holds_the_moments(ops):
    """How near the codes are: half a step of the squares' scale, (|c| + 1/2) / 127^2 of the largest value (255 for v's root)."""
    n = 50_000
    p, g, _, m, v = make([n], torch.float32, torch.float32, None)
    total = m.numel()
    mc, vc = torch.zeros(total, dtype=torch.int8, device="cuda"), torch.zeros(total, dtype=torch.uint8, device="cuda")
    ms, vs = torch.zeros(total // 256, device="cuda"), torch.zeros(total // 256, device="cuda")
    ops._CAPI_adamw_step_8bit(p, g, [], mc, ms, vc, vs, *HYPER, 1)
    want_m = torch.zeros(total, device="cuda", dtype=torch.float64)
    want_m[:n] = g[0].double() * (1 - HYPER[1])
    r = torch.zeros(total, device="cuda", dtype=torch.float64)
    r[:n] = g[0].double().abs() * math.sqrt(1 - HYPER[2])
    got = ops._CAPI_adamw_state_values(mc, ms).double()
    lim = ms.repeat_interleave(256).double() * (mc.double().abs() + 0.5) / 127 ** 2
    assert ((got - want_m).abs() <= lim * 1.0001 + 1e-12).all()
    root = ops._CAPI_adamw_state_values(vc, vs).double().sqrt()
    lim = vs.repeat_interleave(256).double() * (vc.double() + 1) / 255 ** 2
    assert ((root - r).abs() <= lim * 1.0001 + 1e-12).all()
    assert ((vc != 0) == (r > 0)).all()


def test_edges(ops):
    # zero gradients from the start: moments stay zero, parameters only decay; a gradient that is no number stays where it is
    for bits in (32, 8):
        p = torch.ones(600, device="cuda")
        g = torch.zeros(600, device="cuda")
        g[300] = float("nan")
        if bits == 32:
            m, v = torch.zeros(768, device="cuda"), torch.zeros(768, device="cuda")
            ops._CAPI_adamw_step([p], [g], [], m, v, *HYPER, 1)
            assert m.isnan().sum() == 1 and v.isnan().sum() == 1
        else:
            mc, vc = torch.zeros(768, dtype=torch.int8, device="cuda"), torch.zeros(768, dtype=torch.uint8, device="cuda")
            ms, vs = torch.zeros(3, device="cuda"), torch.zeros(3, device="cuda")
            ops._CAPI_adamw_step_8bit([p], [g], [], mc, ms, vc, vs, *HYPER, 1)
            assert ms.isnan().tolist() == vs.isnan().tolist() == [False, True, False]
            assert ms[0] == ms[2] == 0 and (mc == 0).all()
        rest = torch.arange(600, device="cuda") != 300
        assert p[300].isnan() and (p[rest] == float(np.float32(1 - HYPER[0] * HYPER[4]))).all()


def test_absent_gradients_and_the_optimizer(pkg):
    torch.manual_seed(0)
    for bits in (32, 8):
        p = [torch.randn(n, device="cuda").requires_grad_() for n in (300, 40, 1000)]
        ref = [x.detach().double().clone().requires_grad_() for x in p]
        opt = pkg.AdamW(p, lr=1e-2, bits=bits, weight_decay=0.05)
        want = torch.optim.AdamW(ref, lr=1e-2, weight_decay=0.05)
        for step in range(4):
            for i, (x, y) in enumerate(zip(p, ref)):
                g = torch.randn(x.shape, device="cuda")
                x.grad, y.grad = (None, None) if i == 1 else (g, g.double())
            before = p[1].detach().clone()
            version = p[0]._version
            opt.step()
            want.step()
            assert torch.equal(before, p[1].detach()) and p[0]._version > version
        # 4 steps of up to lr = 1e-2 each: 32 bits to some roundings of values below 5; 8 bits hold most moments to a few
        # hundredths (their bits are checked above), so the steps differ by less than a tenth on average and never by more than
        # two steps in opposite directions
        for x, y in zip(p, ref):
            diff = (x.detach().double() - y.detach()).abs()
            assert diff.max() <= (64 * U * 5 if bits == 32 else 8e-2) and (bits == 32 or diff.mean() <= 4e-3)
        saved = opt.state_dict()
        again = pkg.AdamW(p, lr=1e-2, bits=bits)
        again.load_state_dict(saved)
        assert again.steps == 4 and all(torch.equal(a, b) for a, b in zip(opt.moments(), again.moments()))
        with pytest.raises(ValueError, match="other tensors"):
            pkg.AdamW(p[:2], bits=bits).load_state_dict(saved)


def test_other_stream(ops):
    p, g, c, m, v = make([100_000, 333], torch.float32, torch.bfloat16, torch.bfloat16)
    q = [t.clone() for t in p], [t.clone() for t in c], m.clone(), v.clone()
    ops._CAPI_adamw_step(p, g, c, m, v, *HYPER, 5)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        ops._CAPI_adamw_step(q[0], g, q[1], q[2], q[3], *HYPER, 5)
    s.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(p + c + [m, v], q[0] + q[1] + [q[2], q[3]]))


def test_offsets_beyond_32_bits(ops):
    n = (1 << 32) + 1000
    p = torch.ones(n, dtype=torch.bfloat16, device="cuda")
    g = torch.zeros(n, dtype=torch.bfloat16, device="cuda")
    total = -(-n // 256) * 256
    mc, vc = torch.zeros(total, dtype=torch.int8, device="cuda"), torch.zeros(total, dtype=torch.uint8, device="cuda")
    ms, vs = torch.zeros(total // 256, device="cuda"), torch.zeros(total // 256, device="cuda")
    g[-3:] = 1.0
    ops._CAPI_adamw_step_8bit([p], [g], [], mc, ms, vc, vs, 0.5, 0.9, 0.99, 1e-8, 0.0, 1)
    assert p[-3:].float().tolist() == [0.5] * 3 and (p[:4096] == 1).all() and (p[n - 1000:n - 3] == 1).all()
    assert mc[n - 3:n].tolist() == [127] * 3 and vc[n - 3:n].tolist() == [255] * 3 and (mc[n:] == 0).all()
    assert mc[:-1024].any().item() is False


def test_refusals(ops):
    p, g, _, m, v = make([300, 20], torch.float32, torch.float32, None)
    h = (1e-3, 0.9, 0.999, 1e-8, 0.0, 1)
    wide = torch.zeros(300, 2, device="cuda")[:, 0]
    for args, why in ((([wide, p[1]], g, [], m, v), "contiguous"), ((p, g[:1], [], m, v), "gradients"), ((p, g, [p[0]], m, v), "copies"),
                      ((p, [g[1], g[0]], [], m, v), "elements"), ((p, g, [], m[:300], v), "at least"),
                      ((p, g, [], m.double(), v), "type"), ((p, g, [], m, v.cpu()), "must be on"),
                      (([x.double() for x in p], g, [], m, v), "float32"), ((p, [g[0].cpu(), g[1]], [], m, v), "must be on")):
        before = [x.clone() for x in p]
        with pytest.raises(RuntimeError, match=why):
            ops._CAPI_adamw_step(*args, *h)
        assert all(torch.equal(a, b) for a, b in zip(before, p))
    with pytest.raises(RuntimeError, match="steps count from 1"):
        ops._CAPI_adamw_step(p, g, [], m, v, 1e-3, 0.9, 0.999, 1e-8, 0.0, 0)
    mc, s = torch.zeros(768, dtype=torch.int8, device="cuda"), torch.zeros(3, device="cuda")
    with pytest.raises(RuntimeError, match="exp_avg_sq"):
        ops._CAPI_adamw_step_8bit(p, g, [], mc, s, mc, s, *h)
    with pytest.raises(RuntimeError, match="exp_avg_scale"):
        ops._CAPI_adamw_step_8bit(p, g, [], mc, s[:1], mc.byte(), s, *h)
    with pytest.raises(RuntimeError, match="int8"):
        ops._CAPI_adamw_state_values(s, s)
