"""The optimizer's count of steps, a tensor at a time, without a GPU: a stand-in for the operators records what they are called with."""
import importlib

import pytest
import torch


@pytest.fixture()
def calls(pkg, monkeypatch):
    made = []

    class Ops:
        @staticmethod
        def _CAPI_adamw_step(params, grads, copies, m, v, lr, b1, b2, eps, wd, step):
            made.append((step, [i for i, g in enumerate(grads) if g is not None]))

        _CAPI_adamw_step_8bit = None
    monkeypatch.setattr(importlib.import_module("dist-gpu-sampling_b200.training"), "_ops", lambda: Ops)
    return made


def test_a_step_counts_for_the_tensors_that_have_a_gradient(pkg, calls):
    p = [torch.zeros(n) for n in (3, 300, 5)]
    opt = pkg.AdamW(p)
    g = [torch.ones(n) for n in (3, 300, 5)]
    opt.step(g)
    opt.step([g[0], None, None])
    opt.step([g[0], None, None])
    opt.step(g)                                     # counts 4, 2, 2: one launch for each of the two
    opt.step([None, g[1], None])
    assert calls == [(1, [0, 1, 2]), (2, [0]), (3, [0]), (2, [1, 2]), (4, [0]), (3, [1])]
    opt.step([None, None, None])
    assert len(calls) == 6 and opt.steps == 6 and opt.tensor_steps == [4, 3, 2]


def test_counts_are_saved(pkg, calls):
    p, g = [torch.zeros(4), torch.zeros(4)], [torch.ones(4)] * 2
    opt = pkg.AdamW(p)
    opt.step([g[0], None])
    opt.step([g[0], None])
    saved = opt.state_dict()
    opt.step(g)                                     # (what was saved stays what it was)
    again = pkg.AdamW(p)
    again.load_state_dict(saved)
    assert again.steps == 2 and again.tensor_steps == [2, 0]
    del calls[:]
    again.step(g)
    assert calls == [(1, [1]), (3, [0])]
    del saved["tensor_steps"]                       # a state saved when one count stood for all tensors
    again.load_state_dict(saved)
    assert again.tensor_steps == [2, 2]


def test_a_step_that_fails_is_not_counted(pkg, calls, monkeypatch):
    opt = pkg.AdamW([torch.zeros(4)])

    def fail(*_):
        raise RuntimeError("refused")
    monkeypatch.setattr(opt._ops, "_CAPI_adamw_step", fail)
    with pytest.raises(RuntimeError, match="refused"):
        opt.step([torch.ones(4)])
    assert opt.steps == 0 and opt.tensor_steps == [0]
