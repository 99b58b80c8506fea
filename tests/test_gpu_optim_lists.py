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


@both
def test_gradients_where_something_is_written(cs, bits):
    """A gradient beside, or in the very place of, what its own entry writes; one that lies half there is refused, and so is one in
    the place of another entry's."""
    whole = normal(4000, seed=1)
    want, gs = whole[:1000].clone(), whole[1000:2000].clone()
    state = lambda n: ([cs.adamw8_state(torch.empty(n, device="cuda"))],) if bits == 8 else ([torch.zeros(n, device="cuda")], [torch.zeros(n, device="cuda")])
    step(cs, bits, [want], [gs], state(1000))
    p, g = whole[:1000], whole[1000:2000]
    step(cs, bits, [p], [g], state(1000), copies=[g])  # the copy goes where the gradient was
    assert R.bits_equal(p, want) and R.bits_equal(g, want)
    old = whole.clone()
    for bad in (whole[500:1500], whole[999:1999], whole[1:1001]):
        with pytest.raises(ValueError, match="overlap"):
            step(cs, bits, [p], [bad], state(1000))
    q = whole[2000:3000]
    for gs in ([whole[3000:], q], [q, whole[3000:]]):  # in place, and of the other entry
        call = lambda: step(cs, bits, [p, q], gs, tuple(a + b for a, b in zip(state(1000), state(1000))))
        if gs[0] is q:
            with pytest.raises(ValueError, match="overlap"):
                call()
            continue
        call()
    assert R.bits_equal(old[1000:2000], whole[1000:2000]) and R.bits_equal(old[3000:], whole[3000:])
    shared = normal(1000, seed=7)  # a gradient of two parameters
    step(cs, bits, [p, q], [shared, shared], tuple(a + b for a, b in zip(state(1000), state(1000))))


def test_averages_where_their_codes_are(cs):
    room = torch.zeros(4096, dtype=torch.uint8, device="cuda")
    m, v = room[:2000].view(torch.float32), normal(500).abs()
    state = tuple(room[at:at + n] for at, n in ((1900, 500), (2400, 500), (2900, 4), (2904, 4)))
    for call in (cs.adamw8_pack, cs.adamw8_unpack):
        with pytest.raises(ValueError, match="overlap"):
            call([state], [m], [v])


@pytest.mark.parametrize("count", [51, 52, 53, 105, 433])
@both
def test_a_list_is_its_parts(cs, bits, count):
    """Lists around what the kernels' parameters of one launch hold: in 32 bits what the step of each tensor on its own gives."""
    sizes = [(5 * i + 3) % 200 for i in range(count)]
    ps, gs, state = made(cs, bits, sizes)
    alone = [p.clone() for p in ps]
    step(cs, bits, ps, gs, state, lr=0.1)
    if bits == 8:  # their random bits go by the place in the lists, their parameters do not: the first step's averages are exact
        held = [(cs.adamw8_state(p),) for p in alone]
    else:
        held = [(torch.zeros_like(p), torch.zeros_like(p)) for p in alone]
    for p, q, g, s in zip(ps, alone, gs, held):
        step(cs, bits, [q], [g], tuple([t] for t in s), lr=0.1)
        assert R.bits_equal(p, q)
    if bits == 32:
        for l, own in zip(state, zip(*held)):
            assert all(R.bits_equal(a, b) for a, b in zip(l, own))
    want = torch.cat([g.double() for g in gs]).norm()
    assert abs(float(cs.gradient_norm(gs)) - float(want)) <= float(want) * 2.0 ** -23
