"""AdamW refuses lists in which two writers would meet: nothing is launched, nothing changes."""
import pytest
import torch

pytestmark = pytest.mark.gpu
H = (1e-3, 0.9, 0.999, 1e-8, 0.0, 1)


def step(ops, bits, p, g, copies, total=1024):
    if bits == 32:
        m = torch.zeros(2, total, device="cuda")
        ops._CAPI_adamw_step(p, g, copies, m[0], m[1], *H)
    else:
        c, s = torch.zeros(2, total, dtype=torch.uint8, device="cuda"), torch.zeros(2, total // 256, device="cuda")
        ops._CAPI_adamw_step_8bit(p, g, copies, c[0].view(torch.int8), s[0], c[1], s[1], *H)


@pytest.mark.parametrize("bits", [32, 8])
def test_tensors_that_overlap(ops, pkg, bits):
    flat = torch.ones(1000, device="cuda")
    a, b, inside, behind = flat[:300], flat[299:500], flat[100:200], flat[300:600]
    other, g = torch.ones(300, device="cuda"), torch.ones(300, device="cuda")
    cases = [([a, a], []), ([a, b], []), ([a, inside], []), ([other, a], [a, other]),
             ([a, other], [torch.ones(300, device="cuda"), flat[250:550]]), ([a], [a.view(torch.bfloat16)[:300]])]
    for p, copies in cases:
        before = [t.clone() for t in p + copies + [flat]]
        grads = [g[:t.numel()] for t in p]
        with pytest.raises(RuntimeError, match="overlap"):
            step(ops, bits, p, grads, copies)
        assert all(torch.equal(x, y) for x, y in zip(before, p + copies + [flat]))
    with pytest.raises(RuntimeError, match="overlap"):
        pkg.AdamW([a, a], bits=bits).step([g, g])
    step(ops, bits, [a, behind], [g, g], [])                          # neighbours
    step(ops, bits, [a, a], [g, None], [])                            # one of them is not written
    first = a.clone()
    step(ops, bits, [a], [g], [a])                                    # a copy that is the parameter itself
    assert (a != first).all()


def test_moments_that_overlap(ops):
    p, g = torch.ones(300, device="cuda"), torch.ones(300, device="cuda")
    m, c, s = torch.zeros(1024, device="cuda"), torch.zeros(1024, dtype=torch.uint8, device="cuda"), torch.zeros(8, device="cuda")
    for args in ((m, m), (m, m[256:]), (m[:512], p.new_zeros(0).set_(m.untyped_storage(), 511, (513,)))):
        with pytest.raises(RuntimeError, match="overlap|16-byte"):
            ops._CAPI_adamw_step([p], [g], [], *args, *H)
    with pytest.raises(RuntimeError, match="overlap"):
        ops._CAPI_adamw_step([m[:300]], [g], [], m, torch.zeros(1024, device="cuda"), *H)
    with pytest.raises(RuntimeError, match="overlap"):
        ops._CAPI_adamw_step_8bit([p], [g], [], c.view(torch.int8), s, c, s[4:], *H)
    with pytest.raises(RuntimeError, match="overlap"):
        ops._CAPI_adamw_step_8bit([p], [g], [], torch.zeros(1024, dtype=torch.int8, device="cuda"), s, c, s, *H)
    assert (p == 1).all() and (m == 0).all() and (c == 0).all()
    ops._CAPI_adamw_step([p], [g], [], m, m[512:], *H)                # one buffer for both, the slots apart
    assert (m[:300] != 0).all() and (m[512:812] != 0).all() and (m[300:512] == 0).all() and (m[812:] == 0).all()
