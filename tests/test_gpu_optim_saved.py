"""Checkpoints and copies of the optimizer: what goes on from them makes the steps that the original makes."""
import io

import pytest

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

both = pytest.mark.parametrize("bits", [32, 8])


@pytest.fixture(scope="module")
def cs():
    import cswap_b200
    assert torch.cuda.is_available()
    cswap_b200.lib()
    return cswap_b200


def normal(*shape, seed=0):
    return torch.randn(*shape, generator=torch.Generator(device="cuda").manual_seed(seed), device="cuda")


def parameters():
    return [torch.nn.Parameter(normal(*s, seed=i)) for i, s in enumerate([(40, 30), (40,), (300,), (1,)])]


def groups(params):
    return [dict(params=params[:2], lr=1e-2), dict(params=params[2:], weight_decay=0.1)]


def set_gradients(params, t):
    for i, p in enumerate(params):
        g = normal(*p.shape, seed=100 * t + i)
        if p.grad is None:
            p.grad = g
        else:
            p.grad.copy_(g)


def captured(opt):
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        opt.step()
    return graph


def through_a_file(state, where):
    f = io.BytesIO()
    torch.save(state, f)
    f.seek(0)
    return torch.load(f, map_location=where)


# A step by scalars of the device and one by scalars of the host, which differ in their last bits: float32's size, root and decay of
# the step by 2^-23 each, a rate that is float32 on the device by 2^-24 of the size; with the roundings that follow, less than
# 2^-21 of the parameter and of the move, which is 3.2 lr = 0.032 at most.
APART = 2.0 ** -21


def near(p, q, steps):
    p, q = p.detach(), q.detach()
    assert float((p - q).abs().max()) <= steps * APART * (float(p.abs().max()) + 0.032)


def same(opt, other, params, again):
    assert all(torch.equal(p, q) for p, q in zip(params, again))
    for p, q in zip(params, again):
        for name, value in opt.state[p].items():
            held = other.state[q][name]
            assert torch.equal(value, held) and value.device == held.device if isinstance(value, torch.Tensor) else value == held


@both
@pytest.mark.parametrize("capturable", [False, True])
def test_replays_count_in_a_checkpoint(cs, bits, capturable):
    """Ten replays between a checkpoint and the step before them: the next step is the twelfth, also of an optimizer that counts
    on the host."""
    params = parameters()
    opt = cs.AdamW(groups(params), bits=bits, max_norm=1.0, capturable=True, seed=5)
    set_gradients(params, 1)
    opt.step()
    graph = captured(opt)
    for t in range(2, 12):
        set_gradients(params, t)
        graph.replay()
    state = opt.state_dict()
    assert [s["step"] for s in state["state"].values()] == [11] * 4
    again = [torch.nn.Parameter(p.detach().clone()) for p in params]
    other = cs.AdamW(groups(again), bits=bits, max_norm=1.0, capturable=capturable, seed=5)
    other.load_state_dict(through_a_file(state, "cuda"))
    for ps, o in ((params, opt), (again, other)):
        set_gradients(ps, 12)
        o.step()
    if capturable:
        same(opt, other, params, again)
        return
    for p, q in zip(params, again):
        near(p, q, 1)
        for name, value in opt.state[p].items():
            assert not isinstance(value, torch.Tensor) or torch.equal(value, other.state[q][name])


@both
def test_a_capture_makes_no_step(cs, bits):
    params = parameters()
    opt = cs.AdamW(params, bits=bits, capturable=True)
    set_gradients(params, 1)
    opt.step()
    graph = captured(opt)
    assert [opt.state[p]["step"] for p in params] == [1] * 4
    graph.replay()
    assert [s["step"] for s in opt.state_dict()["state"].values()] == [2] * 4


@both
@pytest.mark.parametrize("where", ["cpu", "cuda"])
def test_a_capturable_optimizer_goes_on_from_the_host_s_memory(cs, bits, where):
    """Captured right after loading, and replayed: the steps of the original, bit by bit."""
    params = parameters()
    opt = cs.AdamW(groups(params), bits=bits, max_norm=1.0, capturable=True, seed=5)
    for t in (1, 2, 3):
        set_gradients(params, t)
        opt.step()
    state = through_a_file(opt.state_dict(), where)
    again = [torch.nn.Parameter(p.detach().clone()) for p in params]
    other = cs.AdamW(groups(again), lr=1.0, bits=bits, max_norm=1.0, capturable=True, seed=5)
    other.load_state_dict(state)
    set_gradients(again, 4)
    graph = captured(other)
    for t in (4, 5):
        set_gradients(params, t)
        opt.step()
        set_gradients(again, t)
        graph.replay()
    assert [s["step"] for s in opt.state_dict()["state"].values()] == [s["step"] for s in other.state_dict()["state"].values()] == [5] * 4
    same(opt, other, params, again)


@both
def test_a_checkpoint_of_an_optimizer_that_is_not_capturable(cs, bits):
    params = parameters()
    opt = cs.AdamW(groups(params), bits=bits, seed=5)
    for t in (1, 2):
        set_gradients(params, t)
        opt.step()
    again = [torch.nn.Parameter(p.detach().clone()) for p in params]
    other = cs.AdamW(groups(again), bits=bits, capturable=True, seed=5)
    other.load_state_dict(through_a_file(opt.state_dict(), "cpu"))
    for t in (3, 4):
        for ps, o in ((params, opt), (again, other)):
            set_gradients(ps, t)
            o.step()
    for p, q in zip(params, again):
        near(p, q, 2)
        for name, value in opt.state[p].items():
            assert not isinstance(value, torch.Tensor) or torch.equal(value, other.state[q][name])


@both
@pytest.mark.parametrize("capturable", [False, True])
def test_a_copy_makes_the_same_steps(cs, bits, capturable):
    import copy
    params = parameters()
    opt = cs.AdamW(groups(params), bits=bits, max_norm=1.0, capturable=capturable, seed=9)
    set_gradients(params, 1)
    opt.step()
    other = copy.deepcopy(opt)
    again = [p for g in other.param_groups for p in g["params"]]
    for ps, o in ((params, opt), (again, other)):
        set_gradients(ps, 2)
        o.step()
    same(opt, other, params, again)


def test_a_step_that_is_refused_is_not_counted(cs):
    """Averages of another type stand for what a call refuses."""
    for capturable in (False, True):
        params = parameters()
        opt = cs.AdamW(params, capturable=capturable)
        set_gradients(params, 1)
        opt.step()
        good = opt.state[params[0]]["exp_avg"]
        opt.state[params[0]]["exp_avg"] = good.half()
        before = [p.detach().clone() for p in params]
        with pytest.raises(ValueError, match="float32"):
            opt.step()
        assert all(torch.equal(p, b) for p, b in zip(params, before))
        opt.state[params[0]]["exp_avg"] = good
        set_gradients(params, 2)
        opt.step()
        assert [s["step"] for s in opt.state_dict()["state"].values()] == [2] * 4


def test_a_frozen_group_beside_a_captured_step(cs):
    params, frozen = parameters(), parameters()
    opt = cs.AdamW([dict(params=frozen), dict(params=params)], capturable=True)
    set_gradients(params, 1)
    opt.step()
    graph = captured(opt)
    graph.replay()
    assert [opt.state_dict()["state"][i]["step"] for i in range(4, 8)] == [2] * 4
    assert all(torch.equal(p, q) for p, q in zip(frozen, parameters()))


@both
def test_gradients_that_lie_in_another_order(cs, bits):
    """A parameter in one order in memory and its gradient in another, in a captured step too: the class puts them in order."""
    shape = (8, 6, 5, 4)
    first = torch.nn.Parameter(normal(*shape, seed=1))
    last = torch.nn.Parameter(normal(*shape, seed=1).to(memory_format=torch.channels_last))
    opts = [cs.AdamW([p], bits=32 if p is first else bits, capturable=True, seed=1) for p in (first, last)]
    plain = torch.nn.Parameter(normal(*shape, seed=1).to(memory_format=torch.channels_last))
    opts.append(cs.AdamW([plain], bits=bits, capturable=True, seed=1))
    g = normal(*shape, seed=2)
    first.grad, last.grad = g.to(memory_format=torch.channels_last), g.clone()
    plain.grad = g.to(memory_format=torch.channels_last)
    for o in opts:
        o.step()
    graph = captured(opts[1])
    graph.replay()
    opts[0].step()
    opts[2].step()
    assert last.stride() == plain.stride() != first.stride()
    assert torch.equal(last, plain) and (bits == 8 or torch.equal(last, first))
