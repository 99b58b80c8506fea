"""The lists that the optimizer's step takes: what else than a list may stand there, and which tensors may share memory."""
import pytest

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

import step_reference as R  # noqa: E402

both = pytest.mark.parametrize("bits", [32, 8])


@pytest.fixture(scope="module")
def cs():
    import cswap_b200
    assert torch.cuda.is_available()
    cswap_b200.lib()
    return cswap_b200


def normal(*shape, seed=0, kind=torch.float32):
    return torch.randn(*shape, generator=torch.Generator(device="cuda").manual_seed(seed), device="cuda").to(kind)


def made(cs, bits, sizes=(1000, 7, 300)):
    """(parameters, gradients, the state's lists) of a step."""
    ps, gs = [normal(n, seed=i) for i, n in enumerate(sizes)], [normal(n, seed=10 + i) for i, n in enumerate(sizes)]
    if bits == 8:
        return ps, gs, ([cs.adamw8_state(p) for p in ps],)
    return ps, gs, ([torch.zeros_like(p) for p in ps], [torch.zeros_like(p) for p in ps])


def step(cs, bits, ps, gs, state, **kw):
    (cs.adamw8_step if bits == 8 else cs.adamw_step)(ps, gs, *state, 1, **kw)


@both
def test_what_can_be_gone_through_once(cs, bits):
    """Generators, whose tensors nobody else holds: the step reads them while they live, and autograd learns of what it wrote."""
    want, gs, state = made(cs, bits)
    copies = [torch.empty_like(p, dtype=torch.bfloat16) for p in want]
    step(cs, bits, want, gs, state, copies=copies)
    ps, gs, state = made(cs, bits)
    others = [torch.empty_like(p, dtype=torch.bfloat16) for p in ps]
    versions = [t._version for t in others]
    once = lambda ts: (t for t in ts)
    state = tuple(once([once(s) for s in l]) if bits == 8 else once(l) for l in state)
    step(cs, bits, once(ps), (g.clone() for g in gs), state, copies=once(others))
    torch.empty(1 << 20, device="cuda").fill_(3.0)
    assert all(R.bits_equal(a, b) for a, b in zip(ps, want)) and all(R.bits_equal(a, b) for a, b in zip(others, copies))
    assert [t._version - v for t, v in zip(others, versions)] == [1] * 3
    assert float(cs.gradient_norm(g.clone() for g in gs)) == float(cs.gradient_norm(gs))
