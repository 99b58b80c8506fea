"""What the optimizer class does on the host, without a GPU: its kernels are replaced by plain operations that note what they were
given, a capture by a stream that says it is capturing."""
import math

import pytest

torch = pytest.importorskip("torch")


class Kernels:
    """Stands in for the entry points: notes each launch's step and rate, and makes the step."""

    def __init__(self):
        self.steps, self.fail = [], None

    def step(self, params, grads, step, lr, betas, eps, weight_decay, norm, max_norm, moments):
        if self.fail is not None and self.fail in [id(p) for p in params]:
            raise ValueError("refused")
        t, rate = int(step), float(lr)
        self.steps.append((t, rate, len(params)))
        c = 1.0 if norm is None else min(1.0, max_norm / (float(norm) + 1e-6))
        for p, g, (m, v) in zip(params, grads, moments):
            m.mul_(betas[0]).add_(g * c, alpha=1 - betas[0])
            v.mul_(betas[1]).add_((g * c).square(), alpha=1 - betas[1])
            p.mul_(1 - rate * weight_decay)
            p.sub_(rate / (1 - betas[0] ** t) * m / (v.sqrt() / math.sqrt(1 - betas[1] ** t) + eps))

    def adamw_step(self, params, grads, ms, vs, step, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=0.01, norm=None,
                   max_norm=1.0, copies=None):
        self.step(params, grads, step, lr, betas, eps, weight_decay, norm, max_norm, list(zip(ms, vs)))

    def adamw8_step(self, params, grads, states, step, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=0.01, norm=None,
                    max_norm=1.0, copies=None, seed=0):
        for s in states:
            s[0].add_(1)
        zeros = [(torch.zeros_like(p), torch.zeros_like(p)) for p in params]
        self.step(params, grads, step, lr, betas, eps, weight_decay, norm, max_norm, zeros)


@pytest.fixture
def kernels(monkeypatch):
    from cswap_b200 import optim
    k = Kernels()
    monkeypatch.setattr(optim, "adamw_step", k.adamw_step)
    monkeypatch.setattr(optim, "adamw8_step", k.adamw8_step)
    monkeypatch.setattr(optim, "gradient_norm", lambda ts: torch.stack([t.norm() for t in ts]).norm())
    return k


@pytest.fixture
def capture(monkeypatch):
    """A switch: whether the current stream says that it is capturing."""
    on = [False]
    monkeypatch.setattr(torch.cuda, "is_available", lambda: True)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: on[0])

    def switch(value):
        on[0] = value
    return switch


def AdamW(*args, **kw):
    import cswap_b200
    return cswap_b200.AdamW(*args, **kw)


def parameters(n=3, seed=0):
    gen = torch.Generator().manual_seed(seed)
    return [torch.nn.Parameter(torch.randn(4 + i, generator=gen)) for i in range(n)]


def set_gradients(params, t):
    for i, p in enumerate(params):
        p.grad = torch.randn(p.shape, generator=torch.Generator().manual_seed(100 * t + i))


@pytest.mark.parametrize("bits", [32, 8])
def test_a_group_without_gradients_does_not_keep_a_step_from_being_captured(kernels, capture, bits):
    params, frozen = parameters(2), parameters(2, seed=1)
    opt = AdamW([dict(params=frozen), dict(params=params)], bits=bits, capturable=True)
    set_gradients(params, 1)
    capture(True)
    with pytest.raises(RuntimeError, match="captured"):
        opt.step()  # none has been made yet
    capture(False)
    opt.step()
    capture(True)
    opt.step()
    assert [s[0] for s in kernels.steps] == [1, 2]
    set_gradients(frozen, 1)  # and now it has gradients, but no state
    with pytest.raises(RuntimeError, match="captured"):
        opt.step()
    capture(False)
    assert all(not opt.state.get(p) for p in frozen)


def steps_of(opt, params):
    return [opt.state[p].get("step") for p in params]


def test_a_step_that_is_refused_is_not_counted(kernels):
    """Two groups, the second one refused: the first one's step has been made and counts, the other's does not."""
    first, second = parameters(2), parameters(2, seed=1)
    opt = AdamW([dict(params=first), dict(params=second)])
    for t in (1, 2):
        set_gradients(first + second, t)
        opt.step()
    kernels.fail = id(second[0])
    before = [p.detach().clone() for p in second]
    with pytest.raises(ValueError, match="refused"):
        opt.step()
    assert steps_of(opt, first) == [3, 3] and steps_of(opt, second) == [2, 2]
    assert all(torch.equal(p, b) for p, b in zip(second, before))
    kernels.fail = None
    kernels.steps.clear()
    opt.step()
    assert [s[0] for s in kernels.steps] == [4, 3]


def test_a_step_that_is_refused_is_not_counted_on_the_device(kernels, capture):
    first, second = parameters(2), parameters(2, seed=1)
    opt = AdamW([dict(params=first), dict(params=second)], capturable=True)
    set_gradients(first + second, 1)
    kernels.fail = id(second[0])
    for _ in range(2):  # also of a group that has made no step yet
        with pytest.raises(ValueError, match="refused"):
            opt.step()
    assert steps_of(opt, first) == [2, 2] and steps_of(opt, second) == [0, 0]
    kernels.fail = None
    kernels.steps.clear()
    opt.step()
    assert [s[0] for s in kernels.steps] == [3, 1]


def test_a_norm_that_is_refused_counts_no_step(kernels, monkeypatch):
    from cswap_b200 import optim
    params = parameters(2)
    opt = AdamW(params, max_norm=1.0)
    set_gradients(params, 1)
    good = optim.gradient_norm

    def bad(tensors):
        raise ValueError("refused")
    monkeypatch.setattr(optim, "gradient_norm", bad)
    with pytest.raises(ValueError, match="refused"):
        opt.step()
    monkeypatch.setattr(optim, "gradient_norm", good)
    opt.step()
    assert [s[0] for s in kernels.steps] == [1] and steps_of(opt, params) == [1, 1]


def replay(opt, times):
    """What replays of a captured step do to the counts on the device."""
    for group in opt.param_groups:
        if "device_step" in group:
            group["device_step"].add_(times)


def saved(opt):
    """A checkpoint as a program loads it: through a file, into the host's memory."""
    import io
    f = io.BytesIO()
    torch.save(opt.state_dict(), f)
    f.seek(0)
    return torch.load(f, map_location="cpu")


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("capturable", [True, False])
def test_replayed_steps_are_saved(kernels, capture, bits, capturable):
    """Steps that replays made count in a checkpoint, wherever it goes on."""
    params = parameters(2)
    opt = AdamW([dict(params=params[:1]), dict(params=params[1:])], bits=bits, capturable=True)
    set_gradients(params, 1)
    opt.step()
    capture(True)
    opt.step()  # on the device a capture counts nothing, but this stream only says that it captures: step 2
    capture(False)
    replay(opt, 98)
    state = opt.state_dict()
    assert [s["step"] for s in state["state"].values()] == [100, 100]
    again = [torch.nn.Parameter(p.detach().clone()) for p in params]
    other = AdamW([dict(params=again[:1]), dict(params=again[1:])], bits=bits, capturable=capturable)
    other.load_state_dict(saved(opt))
    kernels.steps.clear()
    for ps, o in ((params, opt), (again, other)):
        set_gradients(ps, 2)
        o.step()
    assert [s[0] for s in kernels.steps] == [101] * 4
    assert all(torch.equal(p, q) for p, q in zip(params, again))


def test_a_step_is_counted_where_it_runs(kernels, capture):
    """Capturing a step makes none."""
    params = parameters(2)
    opt = AdamW(params, capturable=True)
    set_gradients(params, 1)
    opt.step()
    capture(True)
    opt.step()
    assert steps_of(opt, params) == [1, 1]


@pytest.mark.parametrize("bits", [32, 8])
def test_a_checkpoint_holds_nothing_that_lies_on_the_device_in_its_groups(kernels, capture, bits):
    """What is counted on the device is made anew where the parameters are, so that a step may be captured right away."""
    params = parameters(2)
    opt = AdamW(params, lr=0.5, bits=bits, capturable=True)
    set_gradients(params, 1)
    opt.step()
    replay(opt, 6)
    state = saved(opt)
    assert all(not isinstance(v, torch.Tensor) for g in state["param_groups"] for v in g.values())
    assert "device_step" in opt.param_groups[0]  # the optimizer itself goes on as it was
    again = [torch.nn.Parameter(p.detach().clone()) for p in params]
    other = AdamW(again, lr=0.1, bits=bits, capturable=True)
    other.load_state_dict(state)
    set_gradients(again, 2)
    capture(True)
    kernels.steps.clear()
    other.step()
    assert [s[:2] for s in kernels.steps] == [(8, 0.5)]


def test_a_checkpoint_with_the_device_s_numbers_in_its_groups(kernels, capture):
    """As they were saved before: its count is the one that counts, and the checkpoint stays as it is."""
    params = parameters(2)
    opt = AdamW(params, lr=0.5, capturable=True)
    set_gradients(params, 1)
    opt.step()
    state = saved(opt)
    group = state["param_groups"][0]
    group["device_step"], group["device_lr"], group["told_lr"] = torch.tensor([41]), torch.tensor([0.5]), 0.5
    for capturable in (True, False):
        again = [torch.nn.Parameter(p.detach().clone()) for p in params]
        other = AdamW(again, capturable=capturable)
        other.load_state_dict(state)
        set_gradients(again, 2)
        kernels.steps.clear()
        other.step()
        assert [s[:2] for s in kernels.steps] == [(42, 0.5)]
        assert capturable or "device_step" not in other.param_groups[0]
    assert int(group["device_step"]) == 41 and "told_lr" in group
    assert [s["step"] for s in state["state"].values()] == [1, 1]


@pytest.mark.parametrize("how", ["deepcopy", "pickle"])
@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("capturable", [False, True])
def test_a_copy_steps_as_the_original(kernels, how, bits, capturable):
    import copy
    import pickle
    params = parameters(2)
    opt = AdamW(params, lr=0.1, bits=bits, max_norm=0.5, seed=7, capturable=capturable)
    set_gradients(params, 1)
    opt.step()
    other = copy.deepcopy(opt) if how == "deepcopy" else pickle.loads(pickle.dumps(opt))
    assert (other.bits, other.max_norm, other.seed, other.capturable) == (bits, 0.5, 7, capturable)
    again = other.param_groups[0]["params"]
    assert not any(p is q for p, q in zip(params, again))
    kernels.steps.clear()
    for ps, o in ((params, opt), (again, other)):
        set_gradients(ps, 2)
        o.step()
    assert [s[0] for s in kernels.steps] == [2, 2] and all(torch.equal(p, q) for p, q in zip(params, again))
