"""Host logic of spn4cir_amd.optim.AdamW on the CPU: the device calls are stand-ins that count and move the parameters by one."""
import copy
import gc
import warnings
import weakref

import pytest
import torch

from spn4cir_amd import optim as O

HP = dict(lr=1e-2, betas=(0.9, 0.999), eps=1e-8, weight_decay=0.02)


class OnGpu(torch.nn.Parameter):
    """A host tensor that says it lies on the GPU."""
    is_cuda = property(lambda self: True)


class Plan:
    def __init__(self, params, state_bits=32, groups=None, state=None):
        self.params, self.state_bits, self.groups, self.own_moments = params, state_bits, groups, state
        self.addresses, self.numels = [p.data_ptr() for p in params], [p.numel() for p in params]
        at, self.offsets = 0, []
        for n in self.numels:
            self.offsets.append(at)
            at += (n + 127) // 128 * 128
        if state_bits == 8:
            self.m, self.v, self.m_scale, self.v_scale = state or [torch.zeros(k, dtype=torch.uint8) for k in (at, at, at // 128, at // 128)]


class Device:
    """What the stand-ins saw: `fail`: plans that raise before one is built, `ticks`, `calls` = (plan, gradients, hyper) of each launch."""

    def __init__(self):
        self.fail, self.ticks, self.calls, self.capturing, self.singles = 0, 0, [], False, 0

    def plan(self, *args, **kwargs):
        if self.fail:
            self.fail -= 1
            raise torch.OutOfMemoryError("stand-in")
        return Plan(*args, **kwargs)

    def multi(self, plan, grads, step, hyper, **kwargs):
        self.calls.append((plan, grads, hyper))
        for p, g in zip(plan.params, grads):
            if g is not None:
                p.data.add_(1.0)

    def spn_adamw_tick(self, *args):
        self.ticks += 1
        return 0

    def spn_adamw_step_dev(self, *args):
        self.singles += 1
        return 0


@pytest.fixture
def device(monkeypatch):
    d = Device()
    monkeypatch.setattr(O, "AdamWPlan", d.plan)
    monkeypatch.setattr(O, "adamw_multi", d.multi)
    monkeypatch.setattr(O, "lib", lambda: d)
    monkeypatch.setattr(O, "_stream", lambda: None)
    monkeypatch.setattr(O, "_p", lambda t: None)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: d.capturing)
    return d


def make(n=4):
    ps = [OnGpu(torch.zeros(5 + i)) for i in range(n)]
    for p in ps:
        p.grad = torch.ones(p.numel())
    return ps


@pytest.mark.parametrize("bits", [8, 32])
@pytest.mark.parametrize("groups,before", [(2, 1), (20, 1), (20, 2)])
def test_a_failed_first_step_is_not_the_end(device, bits, groups, before):
    """The construction of the first or second of the plans raises once: that step counts nothing and updates nothing, the next one updates
    every parameter."""
    ps = make(groups)
    o = O.AdamW([dict(params=[p]) for p in ps], state_bits=bits, **HP)
    real = device.plan
    made = []

    def plan(*args, **kwargs):
        made.append(1)
        if len(made) == before:
            raise torch.OutOfMemoryError("stand-in")
        return real(*args, **kwargs)
    O.AdamWPlan = plan
    with pytest.raises(torch.OutOfMemoryError):
        o.step()
    assert device.ticks == 0 and not device.calls and not any(bool(p.any()) for p in ps)
    for k in (1.0, 2.0):
        o.step()
        assert device.ticks == k and all(bool((p == k).all()) for p in ps)


@pytest.mark.parametrize("bits", [8, 32])
def test_a_failed_rebuild_is_not_the_end(device, bits):
    """The same for a plan that is rebuilt because a parameter's data was replaced."""
    ps = make()
    o = O.AdamW(ps, state_bits=bits, **HP)
    o.step()
    ps[1].data = ps[1].data.clone()
    device.fail = 1
    with pytest.raises(torch.OutOfMemoryError):
        o.step()
    assert device.ticks == 1 and len(device.calls) == 1
    o.step()
    assert device.ticks == 2 and all(bool((p == 2).all()) for p in ps) and ps[1].data_ptr() in device.calls[-1][0].addresses


def test_a_first_step_under_capture(device):
    """8 bits: refused before anything is built or counted, and the next step outside works.  32 bits: a warning (the graph would zero the state
    at every replay).  After init_state() neither."""
    ps = make()
    o = O.AdamW(ps, state_bits=8, **HP)
    device.capturing = True
    with pytest.raises(RuntimeError, match="init_state"):
        o.step()
    assert device.ticks == 0 and not device.calls and not o.state
    device.capturing = False
    o.step()
    assert device.ticks == 1 and all(bool((p == 1).all()) for p in ps)
    device.capturing = True
    with pytest.warns(UserWarning, match="init_state"):
        O.AdamW(make(), **HP).step()
    for bits in (8, 32):
        o = O.AdamW(make(), state_bits=bits, **HP)
        device.capturing = False
        o.init_state()
        state = {p: dict(st) for p, st in o.state.items()}
        o.init_state()
        device.capturing = True
        with warnings.catch_warnings():
            warnings.simplefilter("error")
            o.step()
        assert all(o.state[p][k] is t for p, st in state.items() for k, t in st.items())


@pytest.mark.parametrize("bits", [8, 32])
def test_every_updated_parameter_gets_a_new_version(device, bits):
    """Parameters re-pointed into one buffer (p.data = a slice) share memory but not a counter; one without a gradient, a frozen one and what the
    optimizer never touched keep theirs."""
    ps, flat = make(5), torch.zeros(64)
    for i, p in enumerate(ps[:3]):
        p.data = flat[i * 16:(i + 1) * 16]
        p.grad = torch.ones(16)
    ps[3].grad = None
    ps[4].requires_grad_(False)
    o = O.AdamW(ps, state_bits=bits, **HP)
    for _ in range(2):
        before = [p._version for p in ps]
        o.step()
        assert [p._version > v for p, v in zip(ps, before)] == [True, True, True, False, False]


@pytest.mark.parametrize("bits", [8, 32])
def test_views_of_one_buffer_bump_the_buffer(device, bits):
    """The models' form: parameters that are views of one flat tensor; its counter moves with theirs, also where one gradient buffer serves all."""
    flat, grad = torch.zeros(64), torch.ones(64)
    ps = [OnGpu(flat[i * 16:(i + 1) * 16]) for i in range(4)]
    for i, p in enumerate(ps):
        p.grad = grad[i * 16:(i + 1) * 16]
    o = O.AdamW(ps, state_bits=bits, **HP)
    for _ in range(2):
        before = flat._version
        o.step()
        assert flat._version > before
    assert device.singles == (2 if bits == 32 else 0)


@pytest.mark.parametrize("bits", [8, 32])
def test_what_a_captured_step_used_lives_on(device, bits):
    """A graph holds addresses only: the plan (its table above all), the moments and the counter of a captured step survive a replaced p.data
    and a loaded state."""
    ps = make()
    o = O.AdamW(ps, state_bits=bits, **HP)
    o.step()
    device.capturing = True
    o.step()
    device.capturing = False
    plan, step, runs = weakref.ref(device.calls[-1][0]), o._step_dev.data_ptr(), o._runs
    moments = weakref.ref(runs[0][0]["m"] if bits == 32 else plan().m)
    del runs
    device.calls.clear()
    ps[1].data = ps[1].data.clone()
    o.step()
    assert device.calls[-1][0] is not plan()
    o.load_state_dict(copy.deepcopy(o.state_dict()))
    o.step()
    device.calls.clear()
    gc.collect()
    assert plan() is not None and moments() is not None and o._captured[0][0].data_ptr() == step


def test_a_capture_after_replaced_data(device):
    """No plan is built inside a capture: 32 bits go tensor by tensor, 8 bits are refused."""
    for bits in (32, 8):
        device.capturing, device.singles = False, 0
        ps = make()
        o = O.AdamW(ps, state_bits=bits, **HP)
        o.step()
        n = len(device.calls)
        ps[2].data = ps[2].data.clone()
        device.capturing, device.fail = True, 1
        if bits == 32:
            o.step()
            assert device.singles == 4 and len(device.calls) == n
        else:
            with pytest.raises(RuntimeError, match="one step"):
                o.step()
        device.capturing, device.fail = False, 0
        o.step()
        assert len(device.calls) == n + 1


@pytest.mark.parametrize("bits,why", [(8, "other bits"), (32, "other bits"), (8, "size"), (32, "size"), (8, "memory")])
def test_a_refused_state_changes_nothing(device, bits, why):
    """A state of the other width, of another parameter's size, or one that finds no memory: the optimizer goes on with its own."""
    ps, other = make(), make(5)[1:]
    o, q = O.AdamW(ps, state_bits=bits, **HP), O.AdamW(make() if why != "size" else other, state_bits=40 - bits if why == "other bits" else bits, **HP)
    o.step(), q.step()
    sd = q.state_dict()
    if why == "size":                                                # 8 bits: one more block of codes; 32 bits: as torch, one element more
        for st in sd["state"].values():
            st["exp_avg"] = torch.zeros(300)
    sd["param_groups"][0]["lr"] = 5.0
    state, groups = {p: dict(st) for p, st in o.state.items()}, o.param_groups
    if why == "memory":
        device.fail = 1
    with pytest.raises((ValueError, RuntimeError)):
        o.load_state_dict(sd)
    assert o.param_groups is groups and groups[0]["lr"] == HP["lr"] and set(o.state) == set(state)
    assert all(o.state[p][k] is t for p, st in state.items() for k, t in st.items())
    o.step()
    assert all(bool((p == 2).all()) for p in ps) and device.calls[-1][2][0]["lr"] == HP["lr"]
    o.load_state_dict(copy.deepcopy(o.state_dict()))                 # and a state that fits is taken
    o.step()
    assert all(bool((p == 3).all()) for p in ps)


@pytest.mark.parametrize("bits", [8, 32])
def test_replaced_groups_count(device, bits):
    """param_groups[i] = another dict after the first step (what a program that rebuilds its schedule does): the next step takes its values."""
    ps = make()
    o = O.AdamW([dict(params=ps[:2]), dict(params=ps[2:])], state_bits=bits, **HP)
    o.step()
    o.param_groups[1] = dict(o.param_groups[1], lr=0.5)
    o.step()
    assert [h["lr"] for h in device.calls[-1][2]] == [HP["lr"], 0.5]


@pytest.mark.parametrize("bits", [8, 32])
def test_launches_go_to_the_parameters_device(device, bits, monkeypatch):
    """Parameters on another device than the current one: every launch of the step, the counter's among them, finds theirs current."""
    current, seen = [0], []

    class Guard:
        def __init__(self, di):
            self.di = di

        def __enter__(self):
            self.old, current[0] = current[0], self.di

        def __exit__(self, *args):
            current[0] = self.old
    monkeypatch.setattr(O.AdamW, "_device", lambda self: torch.device("cuda", 3))
    real_zeros = torch.zeros
    monkeypatch.setattr(torch, "zeros", lambda *a, device=None, **k: real_zeros(*a, **k))
    monkeypatch.setattr(torch.cuda, "current_device", lambda: current[0])
    monkeypatch.setattr(torch.cuda, "device", Guard)
    monkeypatch.setattr(O, "_stream", lambda: seen.append(current[0]))
    real = device.multi
    monkeypatch.setattr(O, "adamw_multi", lambda *a, **k: (seen.append(current[0]), real(*a, **k)))
    flat, grad = torch.zeros(64), torch.ones(64)
    ps = make(2) + [OnGpu(flat[i * 32:(i + 1) * 32]) for i in range(2)]
    for i, p in enumerate(ps[2:]):
        p.grad = grad[i * 32:(i + 1) * 32]
    o = O.AdamW(ps, state_bits=bits, on_step=lambda: seen.append(-current[0]), **HP)
    o.step()
    assert seen == ([3, 3, 0] if bits == 8 else [3, 3, 3, 0])        # counter, (the flat run,) the plan; the callback sees the caller's device


def test_one_tensor_alone(device):
    """32 bits: a single tensor needs no plan; a gradient of another type, or a second tensor, goes through one; its data may be replaced, but not by
    another size, and not by columns of something wider."""
    p, q = make(2)
    q.grad = None
    o = O.AdamW([p, q], **HP)
    device.fail = 1
    o.step()
    assert device.singles == 1 and not device.calls and device.fail == 1
    device.fail = 0
    p.data = p.data.clone()
    o.step()
    assert device.singles == 2
    q.grad = torch.ones(q.numel())
    o.step()
    assert device.singles == 2 and len(device.calls) == 1
    q.grad = None
    for data, error in ((torch.zeros(50), ValueError), (torch.zeros(5, 2)[:, 0], TypeError)):
        p.grad, p.data = None, data
        p.grad = torch.ones_like(data)
        ticks = device.ticks
        with pytest.raises(error):
            o.step()
        assert device.ticks == ticks and device.singles == 2 and len(device.calls) == 1


def test_a_flat_run_whose_data_is_replaced(device):
    """One of the views of a flat buffer moves (p.data = a copy): the step goes to its new memory, the others to theirs; with all of them back in one
    buffer the old one is left alone."""
    flat, grad = torch.zeros(64), torch.ones(64)
    ps = [OnGpu(flat[i * 16:(i + 1) * 16]) for i in range(4)]
    for i, p in enumerate(ps):
        p.grad = grad[i * 16:(i + 1) * 16]
    o = O.AdamW(ps, **HP)
    o.step()
    assert device.singles == 1 and not device.calls
    ps[2].data = ps[2].data.clone()
    o.step()
    assert device.singles == 1 and [p.data_ptr() for p in device.calls[-1][0].params] == [p.data_ptr() for p in ps]
    other = torch.zeros(64)
    for i, p in enumerate(ps):
        p.data = other[i * 16:(i + 1) * 16]
    o.step()
    assert device.singles == 1 and bool((other == 1).all()) and len(device.calls) == 2


def test_gradients_that_are_neighbours_by_chance(device):
    """Consecutive addresses count only within one buffer; another order, a missing one and another type do not count either."""
    flat, grad = torch.zeros(64), torch.ones(64)
    ps = [OnGpu(flat[i * 16:(i + 1) * 16]) for i in range(4)]
    o = O.AdamW(ps, **HP)

    def step(grads):
        for p, g in zip(ps, grads):
            p.grad = g
        before = device.singles
        o.step()
        return device.singles - before
    whole = [grad[i * 16:(i + 1) * 16] for i in range(4)]
    assert step(whole) == 1
    assert step(whole[::-1]) == 0 and step(whole[:3] + [torch.ones(16)]) == 0 and step(whole[:3] + [None]) == 0
    import numpy as np
    raw = np.ones(64, np.float32)
    assert step([torch.from_numpy(raw[i * 16:(i + 1) * 16]) for i in range(4)]) == 0          # four tensors that each own a part of it


@pytest.mark.parametrize("bits", [8, 32])
def test_nothing_to_train(device, bits):
    ps = make()
    for p in ps:
        p.requires_grad_(False)
    o = O.AdamW(ps, state_bits=bits, **HP)
    o.step()
    assert device.ticks == 1 and not device.calls and not any(bool(p.any()) for p in ps)


@pytest.mark.parametrize("capturing", [False, True])
@pytest.mark.parametrize("what", ["type", "size"])
def test_replaced_data_that_no_longer_fits(device, capturing, what):
    """p.data of another type, or a gradient of another size than the data: refused before anything is launched, by itself and among others, also where
    a capture goes tensor by tensor."""
    for n in (1, 3):
        device.capturing = False
        ps = make(n)
        o = O.AdamW(ps, **HP)
        o.init_state()
        p = ps[0]
        if what == "type":
            p.grad = None
            p.data = p.data.half()
            p.grad = torch.ones(p.numel(), dtype=torch.float16)
        else:
            data = p.data
            p.data, p.grad = torch.zeros(3), None
            p.grad = torch.ones(3)
            p.data = data
        device.capturing, ticks, singles, calls = capturing, device.ticks, device.singles, len(device.calls)
        with pytest.raises((TypeError, ValueError)):
            o.step()
        assert (device.ticks, device.singles, len(device.calls)) == (ticks, singles, calls)
