"""What the optimizers do with a clip scale of the caller's, seen from the host:
stand-ins for CUDA tensors, and the native calls recorded in place of run."""
import contextlib
import ctypes

import numpy as np
import pytest
import torch

import tikun_b200
from tikun_b200 import _native
from tikun_b200.optimizer import AdamW as TorchAdamW


class OnDevice(torch.Tensor):
    """A host tensor that says it is a CUDA tensor; `dev` stands for its device."""
    is_cuda = property(lambda self: True)
    device = property(lambda self: getattr(self, "dev", torch.device("cpu")))


def on_device(data, dev=None):
    t = torch.as_tensor(data, dtype=torch.float32).clone().as_subclass(OnDevice)
    if dev is not None:
        t.dev = torch.device(dev)
    return t


def leaf(*shape, dev=None):
    p = on_device(torch.randn(*shape)).requires_grad_()
    p.grad = torch.ones(*shape).as_subclass(OnDevice)
    if dev is not None:
        p.dev = torch.device(dev)
    return p


class Calls(list):
    """(entry point, address that it reads or writes its scale at) of each call."""

    def record(self, name):
        def call(*args, **kw):
            at = kw["clip_scale_ptr"] if "clip_scale_ptr" in kw else args[-1]
            self.append((name, at))

        return call


@pytest.fixture
def calls(monkeypatch):
    got = Calls()
    for name in ("apply_pointwise", "step_fast_buffers_async", "muon_step"):
        monkeypatch.setattr(_native, name, got.record(name))
    monkeypatch.setattr(torch.cuda, "device", lambda dev: contextlib.nullcontext())
    return got


FORMS = {
    "universal": lambda ps: tikun_b200.AdamW(ps),
    "lion": lambda ps: tikun_b200.Lion(ps),
    "torch": lambda ps: TorchAdamW(ps),
}


def set_max_norm(opt, value):
    if isinstance(opt, TorchAdamW):
        opt.param_groups[0]["max_norm"] = value
    else:
        opt.max_norm = value


@pytest.mark.parametrize("max_norm", [0.0, 1.0])
@pytest.mark.parametrize("form", FORMS)
def test_a_step_without_a_scale_writes_none_of_the_callers(calls, form, max_norm):
    opt = FORMS[form]([leaf(5), leaf(2, 3)])
    scale = on_device(0.25)
    opt.step(clip_scale=scale)
    assert calls == [("apply_pointwise", scale.data_ptr())] and opt.clip_scale is scale
    set_max_norm(opt, max_norm)
    opt.step()
    name, at = calls[-1]
    assert name == "step_fast_buffers_async" and at != scale.data_ptr()
    assert opt.clip_scale is not scale and opt.clip_scale.data_ptr() == at
    own = opt.clip_scale
    opt.step()
    assert calls[-1][1] == own.data_ptr() and opt.clip_scale is own


@pytest.mark.parametrize("form", ["muon", "muon_nd"])
def test_muon_hands_its_adamw_no_buffer_of_the_callers(calls, form):
    w, b = leaf(4, 6), leaf(6)
    opt = tikun_b200.Muon([w], [b]) if form == "muon" else tikun_b200.MuonND([w, b])
    scale = on_device(0.25)
    opt.step(clip_scale=scale)
    assert sorted(calls) == [("apply_pointwise", scale.data_ptr()), ("muon_step", scale.data_ptr())]
    assert opt.clip_scale is scale
    calls.clear()
    opt.step()
    assert opt.clip_scale is None
    got = dict(calls)
    assert got["muon_step"] == 0 and got["step_fast_buffers_async"] != scale.data_ptr()


def test_host_and_device_leaves_in_one_in_backward_optimizer(calls, monkeypatch):
    """The scale of a host leaf is a number, which no device step takes for its buffer."""
    monkeypatch.setattr(_native, "step_fast_buffers", lambda *args, **kw: 1.0)
    host, dev = torch.nn.Parameter(torch.ones(3)), leaf(4)
    opt = tikun_b200.AdamW([host, dev], in_backward=True)
    host.sum().backward()
    assert opt.clip_scale == 1.0
    opt._step_single_tensor(dev)
    assert calls[-1] == ("step_fast_buffers_async", opt.clip_scale.data_ptr())


def state_of(opt, params):
    inner = [o for o in (opt, getattr(opt, "adamw", None), getattr(opt, "_adamw", None)) if o]
    return ([o.step_count for o in inner], opt.clip_scale, [p.detach().clone() for p in params])


@pytest.mark.parametrize("odd", ["first", "last"])
@pytest.mark.parametrize("form", [*FORMS, "muon", "muon_nd"])
def test_a_scale_on_another_device_is_refused_before_anything_changes(calls, form, odd):
    """Also where it is on the device of some of the leaves only."""
    ps = [leaf(4, 6), leaf(6, 2), leaf(6), leaf(3)]
    build = {**FORMS, "muon": lambda ps: tikun_b200.Muon(ps[:2], ps[2:]),
             "muon_nd": lambda ps: tikun_b200.MuonND(ps)}[form]
    opt = build(ps)
    ps[0 if odd == "first" else -1].dev = torch.device("cuda", 1)
    before = state_of(opt, ps)
    for scale in (on_device(0.5), on_device(0.5, "cuda:1"), on_device(0.5, "cuda:2")):
        with pytest.raises(ValueError, match="on the device of the parameters"):
            opt.step(clip_scale=scale)
    assert calls == []
    after = state_of(opt, ps)
    assert after[:2] == before[:2] and all(torch.equal(x, y) for x, y in zip(after[2], before[2]))
    assert not getattr(opt, "m1_state", None) and not getattr(opt, "momentum_state", None)
    # a leaf that is not stepped may be anywhere
    if form != "torch":  # which refuses a missing gradient
        ps[0 if odd == "first" else -1].grad = None
        opt.step(clip_scale=on_device(0.5))
        assert calls and opt.step_count == before[0][0] + 1


def test_a_scale_is_refused_for_host_leaves(calls):
    """Arrays and address pairs too, with the gradients given."""
    w = np.ones(4, np.float32)
    g = np.ones(4, np.float32)
    opt = tikun_b200.AdamW([w, (w.ctypes.data, 4)])
    with pytest.raises(ValueError, match="on the device of the parameters"):
        opt.step([g, g], clip_scale=on_device(0.5))
    p = torch.nn.Parameter(torch.ones(4))
    p.grad = torch.ones(4)
    for opt in (tikun_b200.SGD([p]), tikun_b200.MuonND([p]), TorchAdamW([p])):
        with pytest.raises(ValueError, match="on the device of the parameters"):
            opt.step(clip_scale=on_device(0.5, "cuda:0"))
        assert opt.step_count == 0
    assert calls == []


def test_an_arena_takes_no_gradients_with_a_refused_scale(calls, monkeypatch):
    from tikun_b200 import universal

    copied = []

    class Arena:
        def __init__(self, params):
            self.device = torch.device("cpu")

        def moments(self):
            return []

        def step(self, opt, grads, clip_scale):
            copied.append(grads)

    monkeypatch.setattr(universal, "_ArenaState", Arena)
    p = leaf(4)
    opt = tikun_b200.AdamW([p], arena=True)
    with pytest.raises(ValueError, match="on the device of the parameters"):
        opt.step([torch.ones(4)], clip_scale=on_device(0.5, "cuda:1"))
    assert copied == [] and opt.step_count == 0
    opt.step([torch.ones(4)], clip_scale=on_device(0.5))
    assert len(copied) == 1 and opt.step_count == 1


def test_a_closure_and_a_scale_are_refused_together(calls):
    """The closure makes new gradients, and the scale belongs to those before."""
    p = leaf(4)
    opt = TorchAdamW([p])
    ran = []
    with pytest.raises(ValueError, match="closure"):
        opt.step(lambda: ran.append(1), clip_scale=on_device(0.5))
    assert not ran and not calls and opt.step_count == 0
    opt.step(lambda: ran.append(1))
    opt.step(clip_scale=on_device(0.5))
    assert ran == [1] and [c[0] for c in calls] == ["step_fast_buffers_async", "apply_pointwise"]


@pytest.mark.parametrize("at,text", [(0, "scale_dev is NULL"), (4097, "not aligned"), (4098, "not aligned")])
def test_the_clipped_muon_step_refuses_an_address(at, text):
    """A kernel would fault on it; refused before any CUDA call."""
    hp = _native.TkMuonHParams(0.02, 0.95, 1, 5, _native.TK_NS_F16)
    L = _native.lib()
    assert L.tk_muon_step_clipped(None, 0, ctypes.byref(hp), at or None, None) == _native.TK_ERR_INVALID
    assert text in L.tk_last_error().decode()


@pytest.mark.parametrize("form", ["muon", "muon_nd"])
def test_a_step_that_forms_no_norm_shows_none(calls, monkeypatch, form):
    """grad_norm is the last step's, so none of an earlier step's is left there."""
    from tikun_b200 import grads, muon

    formed = [(on_device(float(k)), on_device(0.5)) for k in range(3)]
    left = iter(formed)
    for module, name in ((grads, "clip_scale"), (muon, "scale_of")):
        monkeypatch.setattr(module, name, lambda gs, max_norm: next(left))
    w, b = leaf(4, 6), leaf(6)
    opt = tikun_b200.Muon([w], [b]) if form == "muon" else tikun_b200.MuonND([w, b])
    given = on_device(0.25)
    for max_norm, scale, want in ((1.0, None, formed[0]), (0.0, None, (None, None)),
                                  (1.0, None, formed[1]), (0.0, given, (None, given)),
                                  (2.0, None, formed[2])):
        opt.max_norm = max_norm
        opt.step(clip_scale=scale)
        assert opt.grad_norm is want[0] and opt.clip_scale is want[1]
