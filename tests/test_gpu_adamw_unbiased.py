"""8-bit moments over many steps: codes rounded at random keep the moments their mean, where the nearest code would hold them fast."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu
H = (1e-2, 0.9, 0.99, 1e-8, 0.1)


def state(total):
    return [torch.zeros(total, dtype=torch.int8, device="cuda"), torch.zeros(total // 256, device="cuda"),
            torch.zeros(total, dtype=torch.uint8, device="cuda"), torch.zeros(total // 256, device="cuda")]


def start(ops, n=1500, dtype=torch.float32, seed=0):
    """A state two steps old, and a third gradient."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    s = state(-(-n // 256) * 256)
    p = torch.randn(n, device="cuda", generator=g).to(dtype)
    for step in (1, 2):
        ops._CAPI_adamw_step_8bit([p], [torch.randn(n, device="cuda", generator=g)], [], *s, *H, step)
    return p, s, torch.randn(n, device="cuda", generator=g) * 0.5


def test_a_code_is_one_of_two_and_its_mean_is_the_moment(ops):
    p0, s0, g = start(ops)
    n = p0.numel()
    m = ops._CAPI_adamw_state_values(s0[0], s0[1])[:n].double() * H[1] + g.double() * (1 - H[1])
    v = ops._CAPI_adamw_state_values(s0[2], s0[3])[:n].double() * H[2] + g.double().square() * (1 - H[2])
    p1, s1 = p0.clone(), [t.clone() for t in s0]
    ops._CAPI_adamw_step_8bit([p1], [g], [], *s1, *H, 3)
    N = 400
    sums = [torch.zeros(n, device="cuda", dtype=torch.float64) for _ in range(2)]
    for seed in range(N):
        p, s = p0.clone(), [t.clone() for t in s0]
        ops._CAPI_adamw_step_8bit([p], [g], [], *s, *H, 3, seed - 200)
        assert torch.equal(p, p1) and torch.equal(s[1], s1[1]) and torch.equal(s[3], s1[3])     # the step and the scales are the same
        a, b = s[1].repeat_interleave(256)[:n].double(), s[3].repeat_interleave(256)[:n].double()
        cm, cv = 127 * (m.abs() / a).sqrt(), 255 * (v.sqrt() / b).sqrt()
        # the code below or above (a value within 2^-20 of a code may count as the one before or after it)
        for c, got in ((cm, s[0][:n].double().abs()), (cv, s[2][:n].double())):
            lo = (c * (1 - 2.0 ** -20)).floor()
            assert ((got >= lo.clamp_min(0)) & (got <= (c * (1 + 2.0 ** -20)).floor() + 1)).all()
        assert (s[0][:n].double() * m >= 0).all() and (s[2][:n][v > 0] > 0).all() and not s[0][n:].any() and not s[2][n:].any()
        for t, x in zip(sums, (ops._CAPI_adamw_state_values(s[0], s[1]), ops._CAPI_adamw_state_values(s[2], s[3]))):
            t += x[:n].double()
    # a mean of N values one step of the codes apart has a standard deviation of at most half a step / sqrt(N); six of them
    step_m = a * (2 * cm + 3) / 127 ** 2
    step_v = b.square() * ((cv + 2) ** 4 - cv ** 4) / 255 ** 4
    assert ((sums[0] / N - m).abs() <= 3 * step_m / N ** 0.5 + 2.0 ** -20 * m.abs()).all()
    keeps = cv >= 1                                                   # (below it the code one is kept)
    assert ((sums[1] / N - v).abs() <= 3 * step_v / N ** 0.5 + 2.0 ** -20 * v)[keeps].all()
    # and together: the errors of 1500 elements average, in units of their steps
    assert ((sums[0] / N - m) / step_m).mean().abs() <= 3 / (N * n) ** 0.5
    assert ((sums[1] / N - v) / step_v)[keeps].mean().abs() <= 3 / (N * n) ** 0.5


def test_the_same_call_gives_the_same_bits(ops):
    """Whatever the list looks like: the words go by the place in the buffers."""
    p0, s0, g = start(ops, 4096 + 300)

    def run(cut, step=3, seed=7):
        p, s = p0.clone(), [t.clone() for t in s0]
        ops._CAPI_adamw_step_8bit([p[:cut], p[cut:]], [g[:cut], g[cut:]], [], *s, *H, step, seed)
        return [p] + s
    first = run(256)
    assert all(torch.equal(a, b) for a, b in zip(first, run(256))) and all(torch.equal(a, b) for a, b in zip(first, run(4096)))
    for other in (run(256, step=4), run(256, seed=8)):
        assert (first[1] != other[1]).float().mean() > 0.2 and (first[3] != other[3]).float().mean() > 0.2


@pytest.mark.parametrize("change", ["cut", "grow"])
def test_long_runs_follow_the_moments(pkg, change):
    """The gradients of half a block change after 2 000 steps, and 2 000 steps later the stored roots are the exact ones: a root of
    code c wanders about by sqrt(1 / (2 c)) of itself (each step it moves by 4 / c of the moment with probability at most
    c / 1000 and falls back by a thousandth).  At a tenth of the largest c is some 80 and that is 8 %."""
    rng = np.random.default_rng(5)
    p = torch.zeros(256, device="cuda")
    opt = pkg.AdamW([p], lr=1e-4, bits=8)
    v = np.zeros(256)
    grads = rng.standard_normal((4000, 256)).astype(np.float32)
    if change == "cut":
        grads[2000:, 128:] *= 0.1
    else:
        grads[2000:, :128] *= 3
    on = torch.from_numpy(grads).cuda()
    for i in range(4000):
        v = 0.999 * v + 0.001 * grads[i].astype(np.float64) ** 2
        opt.step([on[i]])
    ratio = (opt.moments()[1].cpu().numpy().astype(np.float64) / v) ** 0.5
    assert ratio.min() > 0.5 and ratio.max() < 1.5
    for half in (ratio[:128], ratio[128:]):
        assert abs(np.median(half) - 1) < 0.06


def test_gradients_that_are_no_numbers_and_empty_blocks(ops):
    for bad in (float("nan"), float("inf"), -float("inf")):
        p, g, s = torch.ones(600, device="cuda"), torch.zeros(600, device="cuda"), state(768)
        g[300] = bad
        ops._CAPI_adamw_step_8bit([p], [g], [], *s, *H, 1, 0)
        assert s[1].isfinite().tolist() == s[3].isfinite().tolist() == [True, False, True] and s[1][0] == s[1][2] == 0
        assert (s[0][:256] == 0).all() and (s[2][:256] == 0).all() and not ops._CAPI_adamw_state_values(s[0], s[1])[300].isfinite()
        assert not p[300].isfinite() and (p[torch.arange(600, device="cuda") != 300] == float(np.float32(1 - H[0] * H[4]))).all()
    p, s = torch.ones(300, device="cuda"), state(512)
    tiny = torch.full((300,), 1e-22, device="cuda")                   # second moments and their roots below the smallest normal numbers
    ops._CAPI_adamw_step_8bit([p], [tiny], [], *s, *H, 1, 0)
    assert (s[0][:300] == 127).all() and p.isfinite().all()
