"""The optimizer's step in 32 and 8 bits, the norm of the gradients and the optimizer class, against their definitions."""
import math

import numpy as np
import pytest

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

import step_reference as R  # noqa: E402

KINDS = [torch.float32, torch.float16, torch.bfloat16]
kinds = pytest.mark.parametrize("kind", KINDS, ids=["fp32", "fp16", "bf16"])
SIZES = [1, 7, 8, 127, 128, 129, 1000, 2047, 2048, 2049, 5000, 0, 16384, 3]


@pytest.fixture(scope="module")
def cs():
    import cswap_b200
    assert torch.cuda.is_available()
    cswap_b200.lib()
    return cswap_b200


def normal(*shape, seed=0, kind=torch.float32):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn(*shape, generator=gen, device="cuda").to(kind)


def npy(t):
    return t.detach().float().cpu().numpy()


def gradients(n, seed, kind):
    return (normal(n, seed=seed) * torch.exp(2 * normal(n, seed=seed + 1)) * 1e-2).to(kind)


def apart(sizes, make, gap):
    """Tensors behind one another in one buffer, `gap` values between them."""
    whole = make(sum(sizes) + gap * len(sizes))
    at, views = 0, []
    for n in sizes:
        views.append(whole[at:at + n])
        at += n + gap
    return whole, views


OPTIONS = dict(lr=3e-3, betas=(0.8, 0.95), eps=1e-6, weight_decay=0.1)


# ---- 32 bits -------------------------------------------------------------------------------------------------------

@kinds
@pytest.mark.parametrize("grad", KINDS, ids=["fp32", "fp16", "bf16"])
@pytest.mark.parametrize("gap", [0, 16], ids=["packed", "apart"])
def test_step_in_32_bits(cs, kind, grad, gap):
    """Averages are 32-bit operations one by one: equal bits; parameters are within their roundings."""
    _, params = apart(SIZES, lambda n: normal(n, seed=1, kind=kind), gap)
    _, grads = apart(SIZES, lambda n: gradients(n, 2, grad), gap)
    _, ms = apart(SIZES, lambda n: normal(n, seed=4) * 1e-2, gap)
    _, vs = apart(SIZES, lambda n: normal(n, seed=5).square() * 1e-4, gap)
    copies = [torch.empty(n, dtype=torch.bfloat16, device="cuda") if i % 2 else None for i, n in enumerate(SIZES)]
    before = [[npy(t) for t in l] for l in (params, grads, ms, vs)]
    olds = [p.clone() for p in params]
    cs.adamw_step(params, grads, ms, vs, 3, copies=copies, **OPTIONS)
    plain = R.Adamw(3, **OPTIONS)
    for i in range(len(SIZES)):
        p, g, m, v = (b[i] for b in before)
        m, v = plain.averages(g, m, v)
        assert np.array_equal(npy(ms[i]), m) and np.array_equal(npy(vs[i]), v)
        want, move = plain.param(p, m, v)
        t = torch.from_numpy
        R.close(params[i], t(want), R.param_bound(t(want), t(move), olds[i].double().cpu(), 3e-3, kind))
        if copies[i] is not None:
            R.close(copies[i], t(want), R.param_bound(t(want), t(move), olds[i].double().cpu(), 3e-3, torch.bfloat16))


def test_what_lies_between_the_tensors_stays(cs):
    for bits in (32, 8):
        buffers = [apart(SIZES, lambda n: torch.full((n,), 7.0, device="cuda"), 3) for _ in range(4)]
        (_, params), (_, grads), (_, ms), (_, vs) = buffers
        if bits == 32:
            cs.adamw_step(params, grads, ms, vs, 1)
            written = [buffers[0], buffers[2], buffers[3]]
        else:
            codes = [apart(SIZES, lambda n: torch.full((n,), 7, dtype=torch.uint8, device="cuda"), 3) for _ in range(2)]
            scales = [apart([-(-n // 128) for n in SIZES], lambda n: torch.full((n,), 7, dtype=torch.uint8, device="cuda"), 1)
                      for _ in range(2)]
            for c in codes:
                for view in c[1]:
                    view.zero_()
            cs.adamw8_step(params, grads, list(zip(codes[0][1], codes[1][1], scales[0][1], scales[1][1])), 1)
            written = [buffers[0]] + codes
            for whole, views in scales:
                inside = torch.zeros(whole.numel(), dtype=torch.bool, device="cuda")
                for view in views:
                    inside[view.storage_offset():view.storage_offset() + view.numel()] = True
                assert (whole[~inside] == 7).all()
        for whole, views in written:
            inside = torch.zeros(whole.numel(), dtype=torch.bool, device="cuda")
            for view in views:
                inside[view.storage_offset():view.storage_offset() + view.numel()] = True
            assert (whole[~inside] == 7).all()
        assert (buffers[1][0] == 7).all()


@kinds
@pytest.mark.parametrize("offsets", [(1, 1, 1, 1, 1), (3, 3, 3, 3, 3), (1, 1, 1, 1, 0), (0, 2, 0, 0, 0), (2, 0, 1, 3, 2)])
@pytest.mark.parametrize("n", [1, 2, 3, 4, 5, 2047, 2049, 4095, 6000])
def test_tensors_off_their_alignment(cs, kind, offsets, n):
    """Parameter, gradient, both averages and copy so many values behind a boundary, all alike or each in its own way; their
    neighbours stay."""
    room = [torch.full((n + 9,), 5.0, device="cuda", dtype=k) for k in (kind, kind, torch.float32, torch.float32, torch.bfloat16)]
    p, g, m, v, c = (r[o + 4:o + 4 + n] for r, o in zip(room, offsets))
    p.copy_(normal(n, seed=1))
    g.copy_(normal(n, seed=2))
    m.copy_(normal(n, seed=3))
    v.copy_(normal(n, seed=4).square())
    mine = [t.clone() for t in (p, g, m, v, c)]
    cs.adamw_step([p], [g], [m], [v], 7, copies=[c], norm=cs.gradient_norm([g]), max_norm=0.5)
    cs.adamw_step([mine[0]], [mine[1]], [mine[2]], [mine[3]], 7, copies=[mine[4]], norm=cs.gradient_norm([mine[1]]), max_norm=0.5)
    for r, o, t, want in zip(room, offsets, (p, g, m, v, c), mine):
        assert R.bits_equal(t, want) and (r[:o + 4] == 5).all() and (r[o + 4 + n:] == 5).all()


# ---- 8 bits --------------------------------------------------------------------------------------------------------

def some_state(cs, n, seed):
    """A state as a few steps leave it, and the float32 averages that it holds."""
    m, v = gradients(n, seed, torch.float32), gradients(n, seed + 5, torch.float32).square() * 0.1
    state = cs.adamw8_state(m)
    cs.adamw8_pack([state], [m], [v])
    held = [torch.empty_like(m) for _ in range(2)]
    cs.adamw8_unpack([state], held[:1], held[1:])
    return state, npy(held[0]), npy(held[1])


def check_state(state, m, v, bits):
    codes = [t.cpu().numpy() for t in state]
    want_m, scale_m = R.encode(m, bits[0], 4)
    want_v, scale_v = R.encode(v, bits[1], 5)
    for got, want in zip(codes, (want_m, want_v, scale_m, scale_v)):
        assert np.array_equal(got, want)


@pytest.mark.parametrize("n", [n for n in SIZES if n])
def test_packing_rounds_to_the_nearest(cs, n):
    m, v = gradients(n, n, torch.float32), gradients(n, n + 1, torch.float32).square()
    state = cs.adamw8_state(m)
    assert [t.numel() for t in state] == [n, n, -(-n // 128), -(-n // 128)]
    cs.adamw8_pack([state], [m], [v])
    half = np.full(n, 1 << 19)
    check_state(state, npy(m), npy(v), (half, half))
    back = [torch.empty(n, device="cuda") for _ in range(2)]
    cs.adamw8_unpack([state], back[:1], back[1:])
    codes = [t.cpu().numpy() for t in state]
    assert np.array_equal(npy(back[0]), R.decode(codes[0], codes[2], 4)) and np.array_equal(npy(back[1]), R.decode(codes[1], codes[3], 5))
    # half a step of a code: a sixteenth of a number that has a leading one, else of the least step
    for got, want, least in ((back[0], m, 2.0 ** -17), (back[1], v, 2.0 ** -33)):
        scale = torch.nn.functional.pad(want.abs(), (0, -n % 128)).view(-1, 128).amax(1).repeat_interleave(128)[:n] * 2
        R.close(got, want, want.abs() / 16 + scale * least * (1 if least == 2.0 ** -33 else 0.5))


@kinds
@pytest.mark.parametrize("grad", [torch.float32, torch.bfloat16], ids=["fp32", "bf16"])
@pytest.mark.parametrize("gap", [0, 16], ids=["packed", "apart"])
def test_step_in_8_bits(cs, kind, grad, gap):
    """Codes and scales follow from the definition bit by bit, whatever lies at the ends of groups and tensors."""
    _, params = apart(SIZES, lambda n: normal(n, seed=1, kind=kind), gap)
    _, grads = apart(SIZES, lambda n: gradients(n, 2, grad), gap)
    held = [some_state(cs, n, 10 + i) for i, n in enumerate(SIZES)]
    states = [h[0] for h in held]
    before, ps, olds = [npy(t) for t in grads], [npy(t) for t in params], [p.clone() for p in params]
    copies = [torch.empty(n, dtype=torch.float16, device="cuda") for n in SIZES]
    cs.adamw8_step(params, grads, states, 5, seed=99, copies=copies, **OPTIONS)
    plain = R.Adamw(5, **OPTIONS)
    for i, n in enumerate(SIZES):
        m, v = plain.averages(before[i], held[i][1], held[i][2])
        bits = [b.astype(np.int64) * 16 + 8 for b in R.random_bits(99, 5, i, n)]
        check_state(states[i], m, v, bits)
        want, move = (torch.from_numpy(x) for x in plain.param(ps[i], m, v))
        R.close(params[i], want, R.param_bound(want, move, olds[i].double().cpu(), 3e-3, kind))
        R.close(copies[i], want, R.param_bound(want, move, olds[i].double().cpu(), 3e-3, torch.float16))


def test_a_state_of_zeros_and_groups_without_a_gradient(cs):
    p, g = normal(384, seed=1), torch.zeros(384, device="cuda")
    g[300] = 1e-3
    old = p.clone()
    state = cs.adamw8_state(p)
    cs.adamw8_step([p], [g], [state], 1, lr=0.1, weight_decay=0.0)
    assert torch.equal(p[:300], old[:300]) and torch.equal(p[301:], old[301:])
    assert abs(float(old[300] - p[300]) - 0.1) < 1e-5
    assert (state[2][:2] == 0).all() and (state[3][:2] == 0).all() and (state[0][:256] == 0).all() and (state[1][:256] == 0).all()
    # of a group that has anything no v is held as zero, so that no later step divides by nothing
    assert (state[1][256:] >= 1).all() and int(state[0].bitwise_and(127).ne(0).sum()) == 1


def test_weights_beside_much_larger_ones_move_by_bounded_steps(cs):
    """Gradients of 1 beside gradients of 2^-20: the small ones' averages are below what m's codes resolve and are rounded up now
    and then, which v's least code keeps from becoming a leap."""
    n = 128 * 64
    p = torch.zeros(n, device="cuda")
    state = cs.adamw8_state(p)
    gen = torch.Generator(device="cuda").manual_seed(3)
    size = torch.where(torch.arange(n, device="cuda") % 128 == 0, 1.0, 2.0 ** -20)
    for t in range(1, 41):
        before = p.clone()
        g = size * torch.randn(n, generator=gen, device="cuda")
        cs.adamw8_step([p], [g], [state], t, lr=1.0, weight_decay=0.0)
        # a step of Adam is below (1 - b1) / sqrt(1 - b2) = 3.2, its first ones below 1; a code's rounding lets m be twice what it
        # is and sqrt(v) sqrt(7 / 8) at the least, corrected by (1 - b1^t) and sqrt(1 - b2^t)
        assert float((p - before).abs().max()) < 8.0


def test_rounding_is_right_in_the_mean(cs):
    """The averages of a constant gradient: m reaches it, v creeps up by a thousandth of its square each step, a twentieth of a
    code's step.  Rounded to the nearest v would stay at a sixtieth; rounded at random 65536 values' mean is within five of its
    standard deviations: each step's rounding has a variance of a quarter of a step's square at most, a step is an eighth of v at
    most, and what is left of it after later steps sums to less than 1 / (1 - b2^2) of that."""
    n, steps = 65536, 400
    p, g = torch.zeros(n, device="cuda"), torch.full((n,), 0.3, device="cuda")
    state = cs.adamw8_state(p)
    for t in range(1, steps + 1):
        cs.adamw8_step([p], [g], [state], t, seed=7)
    m, v = torch.empty_like(p), torch.empty_like(p)
    cs.adamw8_unpack([state], [m], [v])
    for got, beta, value in ((m, 0.9, 0.3), (v, 0.999, 0.09)):
        want = value * (1 - beta ** steps)
        sigma = value / 8 / 2 * math.sqrt(min(steps, 1 / (1 - beta * beta)))
        # 2^-17 of a step is the truncation of the 16 random bits, 2^-23 a step float32's own
        assert abs(float(got.double().mean()) - want) < 5 * sigma / math.sqrt(n) + steps * value * 2.0 ** -19


def test_numbers_that_are_not(cs):
    """A gradient's NaN or infinity shows in its parameter, and from then on in its group's."""
    for bits in (32, 8):
        p, g = normal(512, seed=1), normal(512, seed=2)
        g[200], g[300] = math.nan, math.inf
        state = cs.adamw8_state(p)
        m, v = torch.zeros_like(p), torch.zeros_like(p)
        step = (lambda t: cs.adamw8_step([p], [g], [state], t)) if bits == 8 else (lambda t: cs.adamw_step([p], [g], [m], [v], t))
        step(1)
        assert torch.isnan(p).nonzero().flatten().tolist() == [200, 300]
        if bits == 8:
            assert state[2].tolist()[1:3] == [255, 255] and state[3].tolist()[1:3] == [255, 255]
            cs.adamw8_unpack([state], [m], [v])
            for t in (m, v):
                assert torch.isnan(t[128:384]).all() and torch.isfinite(t[:128]).all() and torch.isfinite(t[384:]).all()
        g[200], g[300] = 0.0, 0.0
        step(2)
        where = torch.zeros(512, dtype=torch.bool, device="cuda")
        if bits == 8:
            where[128:384] = True
        else:
            where[200] = where[300] = True
        assert torch.equal(torch.isnan(p), where)


def test_averages_at_the_ends_of_the_range(cs):
    """The smallest and largest averages that a scale can hold, and beyond."""
    for top in (2.0 ** -149, 2.0 ** -130, 1.75 * 2.0 ** -126, 1.75 * 2.0 ** 126, 1.751 * 2.0 ** 126, 3e38):
        m = normal(128, seed=1).clamp(-1, 1) * float(np.float32(top))
        m[5] = float(np.float32(top))
        v = m.abs()
        state = cs.adamw8_state(m)
        cs.adamw8_pack([state], [m], [v])
        half = np.full(128, 1 << 19)
        check_state(state, npy(m), npy(v), (half, half))
        back = [torch.empty_like(m) for _ in range(2)]
        cs.adamw8_unpack([state], back[:1], back[1:])
        c = [t.cpu().numpy() for t in state]
        assert np.array_equal(npy(back[0]), R.decode(c[0], c[2], 4), equal_nan=True)
        assert np.array_equal(npy(back[1]), R.decode(c[1], c[3], 5), equal_nan=True)
        assert bool(torch.isnan(back[0]).all()) == (top > 1.75 * 2.0 ** 126)


# ---- the norm, clipping, numbers on the device ---------------------------------------------------------------------

@kinds
def test_gradient_norm(cs, kind):
    """Squares and sums in float64: half a step of float32 is all that is lost."""
    for gap in (0, 16):
        _, grads = apart(SIZES, lambda n: gradients(n, 3, kind), gap)
        norm = cs.gradient_norm(grads)
        assert norm.dtype == torch.float32 and norm.shape == ()
        want = torch.cat([g.double() for g in grads]).norm()
        assert abs(float(norm) - float(want)) <= float(want) * 2.0 ** -23
        assert float(norm) == float(cs.gradient_norm(grads))
    assert float(cs.gradient_norm([torch.empty(0, device="cuda", dtype=kind)])) == 0.0
    big = torch.full((1000,), 3e38 if kind == torch.float32 else 6e4, device="cuda").to(kind)
    if kind == torch.float32:
        assert float(cs.gradient_norm([big])) == math.inf and float(cs.gradient_norm([big[:1]])) == float(big[0])
    big[7] = math.nan
    assert math.isnan(float(cs.gradient_norm([big])))


@pytest.mark.parametrize("bits", [32, 8])
def test_clipping(cs, bits):
    """The gradients times min(1, max_norm / (norm + 1e-6)), as float32 operations have it."""
    for max_norm in (1.0, 1e6, 0.0):
        ps = [normal(n, seed=n) for n in (1000, 64)]
        gs = [normal(n, seed=n + 1) for n in (1000, 64)]
        norm = cs.gradient_norm(gs)
        c = min(np.float32(1), np.float32(max_norm) / (np.float32(float(norm)) + np.float32(1e-6)))
        plain = R.Adamw(1, factor=c)
        olds = [npy(p) for p in ps]
        if bits == 32:
            ms, vs = ([torch.zeros_like(p) for p in ps] for _ in range(2))
            cs.adamw_step(ps, gs, ms, vs, 1, norm=norm, max_norm=max_norm)
        else:
            states = [cs.adamw8_state(p) for p in ps]
            cs.adamw8_step(ps, gs, states, 1, norm=norm, max_norm=max_norm)
        for i in range(2):
            zero = np.zeros(ps[i].numel(), np.float32)
            m, v = plain.averages(npy(gs[i]), zero, zero)
            if bits == 32:
                assert np.array_equal(npy(ms[i]), m) and np.array_equal(npy(vs[i]), v)
            else:
                check_state(states[i], m, v, [b.astype(np.int64) * 16 + 8 for b in R.random_bits(0, 1, i, zero.size)])
            want, move = (torch.from_numpy(x) for x in plain.param(olds[i], m, v))
            R.close(ps[i], want, R.param_bound(want, move, torch.from_numpy(olds[i]).double(), 1e-3, torch.float32))


@pytest.mark.parametrize("eps", [0.0, 1e-30, 2.0 ** -40, 1e-12, 1.0])
def test_epsilons(cs, eps):
    """Down to nothing, with averages of squares among float32's smallest numbers: the root of one is taken exactly there, and from
    2^-40 on what lies below 2^-126 moves the sum by less than 2^-23 of it."""
    g = torch.cat([normal(500, seed=1), normal(500, seed=2) * 1e-15, normal(500, seed=3) * 1e-19, normal(500, seed=4) * 1e15])
    p, m, v = torch.zeros_like(g), torch.zeros_like(g), torch.zeros_like(g)
    cs.adamw_step([p], [g], [m], [v], 1, eps=eps)
    plain = R.Adamw(1, eps=eps)
    zero = np.zeros(2000, np.float32)
    a, b = plain.averages(npy(g), zero, zero)
    assert np.array_equal(npy(m), a) and np.array_equal(npy(v), b)
    want, move = (torch.from_numpy(x) for x in plain.param(zero, a, b))
    R.close(p, want, R.param_bound(want, move, torch.zeros(2000).double(), 1e-3, torch.float32) + move.abs() * 2.0 ** -23)


def test_large_and_small_gradients_in_8_bits(cs):
    """Averages that are scaled in two steps, among others: 2^-110 to 2^60."""
    for power in (-55, -40, -20, 10, 16, 30, 60):
        p, g = normal(1000, seed=1), normal(1000, seed=2) * 2.0 ** power
        state, zero = cs.adamw8_state(p), np.zeros(1000, np.float32)
        plain, m, v = R.Adamw(1), zero, zero
        for t in (1, 2):
            plain.step = t
            cs.adamw8_step([p], [g], [state], t, seed=9)
            m, v = plain.averages(npy(g), m, v)
            check_state(state, m, v, [b.astype(np.int64) * 16 + 8 for b in R.random_bits(9, t, 0, 1000)])
            codes = [c.cpu().numpy() for c in state]
            m, v = R.decode(codes[0], codes[2], 4), R.decode(codes[1], codes[3], 5)


def test_clipping_by_a_norm_that_is_no_number(cs):
    p, g = normal(10), normal(10, seed=1)
    m, v = torch.zeros_like(p), torch.zeros_like(p)
    cs.adamw_step([p], [g], [m], [v], 1, norm=torch.tensor(math.nan, device="cuda"))
    assert torch.isnan(p).all() and torch.isnan(m).all()


@pytest.mark.parametrize("bits", [32, 8])
def test_step_and_rate_on_the_device(cs, bits):
    """The same as from the host, to the rounding of a float32 rate."""
    lr = float(np.float32(2e-3))
    for t in (1, 2, 1000, 123456):
        runs = []
        for step, rate in ((t, lr), (torch.tensor([t], device="cuda"), torch.tensor([lr], device="cuda")),
                           (torch.tensor(t, device="cuda"), lr), (t, torch.tensor(lr, device="cuda"))):
            p, g = normal(3000, seed=1), normal(3000, seed=2)
            if bits == 32:
                state = [torch.zeros_like(p), torch.zeros_like(p)]
                cs.adamw_step([p], [g], state[:1], state[1:], step, rate, betas=(0.9, 0.99))
            else:
                state = list(cs.adamw8_state(p))
                cs.adamw8_step([p], [g], [state], step, rate, betas=(0.9, 0.99), seed=5)
            runs.append([p] + state)
        for r in runs[1:]:
            assert all(torch.equal(a, b) for a, b in zip(r[1:], runs[0][1:]))
            # the device's logarithm and expm1 may differ in their last bits, and with them the scalars' rounding
            R.close(r[0], runs[0][0], runs[0][0].abs() * 2.0 ** -23 + lr * 10 * 2.0 ** -22)


# ---- lists ---------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("count", [1, 39, 40, 41, 380, 381, 1000])
@pytest.mark.parametrize("bits", [32, 8])
def test_many_tensors(cs, count, bits):
    """As many as one launch takes, and more; a tensor's place in the lists counts, not its launch."""
    sizes = [(7 * i + 5) % 300 for i in range(count)]
    make = lambda seed: [normal(n, seed=seed + i) for i, n in enumerate(sizes)]
    ps, gs = make(1), make(2)
    olds = [npy(p) for p in ps]
    plain = R.Adamw(2)
    norm = cs.gradient_norm(gs)
    want = math.sqrt(sum(float(g.double().square().sum()) for g in gs))
    assert abs(float(norm) - want) <= want * 2.0 ** -23
    if bits == 32:
        ms, vs = ([torch.zeros_like(p) for p in ps] for _ in range(2))
        cs.adamw_step(ps, gs, ms, vs, 2)
    else:
        states = [cs.adamw8_state(p) for p in ps]
        cs.adamw8_step(ps, gs, states, 2, seed=3)
    for i in sorted({0, count // 3, count // 2, min(count - 1, 379), min(count - 1, 380), count - 1}):
        zero = np.zeros(sizes[i], np.float32)
        m, v = plain.averages(npy(gs[i]), zero, zero)
        if bits == 32:
            assert np.array_equal(npy(ms[i]), m) and np.array_equal(npy(vs[i]), v)
        else:
            check_state(states[i], m, v, [b.astype(np.int64) * 16 + 8 for b in R.random_bits(3, 2, i, sizes[i])])
        w, move = (torch.from_numpy(x) for x in plain.param(olds[i], m, v))
        R.close(ps[i], w, R.param_bound(w, move, torch.from_numpy(olds[i]).double(), 1e-3, torch.float32))


def test_orders_in_memory(cs):
    """A parameter in another dense order than row by row, its gradient and averages in the same."""
    p = normal(8, 6, 5, 4).to(memory_format=torch.channels_last)
    g = normal(8, 6, 5, 4, seed=1).to(memory_format=torch.channels_last)
    m, v = torch.zeros_like(p), torch.zeros_like(p)
    q, h = p.contiguous(), g.contiguous()
    n, w = torch.zeros_like(q), torch.zeros_like(q)
    cs.adamw_step([p], [g], [m], [v], 1)
    cs.adamw_step([q], [h], [n], [w], 1)
    assert torch.equal(p, q) and torch.equal(m, n) and not p.is_contiguous()
    with pytest.raises(ValueError, match="order"):
        cs.adamw_step([p], [h], [m], [v], 1)


def test_refusals(cs):
    p, g, m, v = (normal(300, seed=i) for i in range(4))
    s = cs.adamw8_state(p)
    whole = normal(600)
    for call in (lambda: cs.adamw_step([p], [g], [m], [v], 0), lambda: cs.adamw_step([p], [g, g], [m], [v], 1),
                 lambda: cs.adamw_step([p], [g], [m], [], 1), lambda: cs.adamw_step([p], [g[:299]], [m], [v], 1),
                 lambda: cs.adamw_step([p], [g], [m.half()], [v], 1), lambda: cs.adamw_step([p.double()], [g], [m], [v], 1),
                 lambda: cs.adamw_step([p], [g.cpu()], [m], [v], 1), lambda: cs.adamw_step([p], [g], [m], [v], 1, lr=-1.0),
                 lambda: cs.adamw_step([p], [g], [m], [v], 1, lr=math.nan), lambda: cs.adamw_step([p], [g], [m], [v], 1, betas=(1.0, 0.9)),
                 lambda: cs.adamw_step([p], [g], [m], [v], 1, eps=-1e-8), lambda: cs.adamw_step([p], [g], [m], [v], 1, weight_decay=math.inf),
                 lambda: cs.adamw_step([p], [g], [m], [v], 1, norm=torch.ones(2, device="cuda")),
                 lambda: cs.adamw_step([p], [g], [m], [v], 1, norm=torch.ones((), device="cuda"), max_norm=-1.0),
                 lambda: cs.adamw_step([p], [g], [m], [v], torch.ones(1, device="cuda")),
                 lambda: cs.adamw_step([p], [g], [m], [v], 1, lr=torch.ones(1, device="cuda", dtype=torch.float64)),
                 lambda: cs.adamw_step([p], [g], [m], [v], 1, copies=[p]), lambda: cs.adamw_step([p], [g], [m], [m], 1),
                 lambda: cs.adamw_step([p, p], [g, g], [m, m.clone()], [v, v.clone()], 1),
                 lambda: cs.adamw_step([whole[:300], whole[299:599]], [g, g], [m, m.clone()], [v, v.clone()], 1),
                 lambda: cs.adamw_step([p, p.clone()], [g, g], [m, m], [v, v.clone()], 1),
                 lambda: cs.adamw_step([whole[::2]], [g], [m], [v], 1), lambda: cs.adamw_step([p], [g], [m], [v], 1, copies=[None, None]),
                 lambda: cs.adamw8_step([p], [g], [s[:3]], 1), lambda: cs.adamw8_step([p], [g], [(s[0], s[1], s[2], s[3][:2])], 1),
                 lambda: cs.adamw8_step([p], [g], [(s[0].float(), s[1], s[2], s[3])], 1),
                 lambda: cs.adamw8_step([p], [g], [(s[0], s[0], s[2], s[3])], 1), lambda: cs.adamw8_step([p], [g], [s], 1, seed=1 << 32),
                 lambda: cs.adamw8_step([p, p.clone()], [g, g], [s, s], 1), lambda: cs.adamw8_unpack([s], [m], [m]),
                 lambda: cs.adamw8_unpack([s], [m.half()], [v]), lambda: cs.adamw8_pack([s, s], [m, m], [v, v]),
                 lambda: cs.adamw8_pack([s], [m[:200]], [v[:200]]), lambda: cs.gradient_norm([]), lambda: cs.gradient_norm([whole[::2]]),
                 lambda: cs.gradient_norm([p.double()])):
        with pytest.raises(ValueError):
            call()
    for call in (lambda: cs.adamw_step([p], [None], [m], [v], 1), lambda: cs.adamw_step(p, [g], [m], [v], "1"),
                 lambda: cs.gradient_norm(3), lambda: cs.adamw8_step([p], [g], [3], 1)):
        with pytest.raises((TypeError, ValueError)):
            call()
    cs.adamw_step([], [], [], [], 1)
    cs.adamw8_step([], [], [], 1)


def test_autograd_learns_of_the_change(cs):
    """A parameter that a graph has kept is not to be changed before its backward pass."""
    p = normal(64).requires_grad_(True)
    y = (p * p).sum()
    g = normal(64, seed=1)
    with torch.no_grad():
        cs.adamw_step([p], [g], [torch.zeros(64, device="cuda")], [torch.zeros(64, device="cuda")], 1)
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        y.backward()


# ---- the optimizer -------------------------------------------------------------------------------------------------

def parameters(seed=0):
    return [torch.nn.Parameter(normal(*s, seed=seed + i)) for i, s in enumerate([(40, 30), (40,), (3, 5, 7), (1,)])]


def set_gradients(params, t):
    for i, p in enumerate(params):
        p.grad = None if (t == 2 and i == 1) else normal(*p.shape, seed=100 * t + i)


def test_optimizer_follows_torch(cs):
    """In 32 bits: ten steps, two groups, a parameter that misses one, clipping.  Both round some twenty times a step, each time
    by 2^-24 of a parameter or of a move of at most lr (1 - b1) / sqrt(1 - b2) = 3.2 lr."""
    mine, theirs = parameters(), parameters()
    groups = lambda ps: [dict(params=ps[:2], lr=1e-2), dict(params=ps[2:], weight_decay=0.1, betas=(0.8, 0.99))]
    a, b = cs.AdamW(groups(mine), max_norm=3.0), torch.optim.AdamW(groups(theirs), lr=1e-3)
    for t in range(1, 11):
        set_gradients(mine, t)
        set_gradients(theirs, t)
        torch.nn.utils.clip_grad_norm_(theirs, 3.0)
        a.step()
        b.step()
        for p, q in zip(mine, theirs):
            R.close(p.detach(), q.detach(), (q.detach().abs() + 0.032) * (t * 40 * 2.0 ** -24))


def test_optimizer_in_8_bits_is_the_step(cs):
    params, other = parameters(), parameters()
    opt = cs.AdamW(params, lr=1e-2, bits=8, seed=11)
    states = [cs.adamw8_state(p) for p in other]
    for t in (1, 3, 4):  # every parameter has its gradient
        set_gradients(params, t)
        opt.step()
    for k, t in enumerate((1, 3, 4)):
        cs.adamw8_step([p.detach() for p in other], [normal(*p.shape, seed=100 * t + i) for i, p in enumerate(other)], states, k + 1,
                       lr=1e-2, seed=11)
    assert all(torch.equal(p, q) for p, q in zip(params, other))


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("kind", [torch.float32, torch.bfloat16], ids=["fp32", "bf16"])
def test_a_saved_optimizer_goes_on(cs, bits, kind):
    make = lambda: [torch.nn.Parameter(p.detach().to(kind)) for p in parameters()]
    params = make()
    opt = cs.AdamW(params, lr=1e-2, bits=bits)
    for t in (1, 2):
        for i, p in enumerate(params):
            p.grad = normal(*p.shape, seed=100 * t + i, kind=kind)
        opt.step()
    again = [torch.nn.Parameter(p.detach().clone()) for p in params]
    other = cs.AdamW(again, lr=1.0, bits=bits)
    import io
    f = io.BytesIO()
    torch.save(opt.state_dict(), f)
    f.seek(0)
    other.load_state_dict(torch.load(f))
    for i, (p, q) in enumerate(zip(params, again)):
        p.grad = normal(*p.shape, seed=300 + i, kind=kind)
        q.grad = p.grad.clone()
    opt.step()
    other.step()
    assert all(torch.equal(p, q) for p, q in zip(params, again))
    for p, q in zip(params, again):
        for name, value in opt.state[p].items():
            assert not isinstance(value, torch.Tensor) or torch.equal(value, other.state[q][name])


@pytest.mark.parametrize("bits", [32, 8])
def test_a_captured_step(cs, bits):
    """Replays count their steps on the device, take new gradients and a new rate, and give what steps one by one give."""
    params, other = parameters(), parameters()
    opt = cs.AdamW(params, lr=1e-2, bits=bits, max_norm=2.0, capturable=True, seed=4)
    plain = cs.AdamW(other, lr=1e-2, bits=bits, max_norm=2.0, capturable=True, seed=4)
    for p, q in zip(params, other):
        p.grad, q.grad = torch.zeros_like(p), torch.zeros_like(q)
    fill = lambda ps, t: [p.grad.copy_(normal(*p.shape, seed=100 * t + i)) for i, p in enumerate(ps)]
    fill(params, 1)
    g = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match="capturable"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            opt.step()
    opt.step()
    with torch.cuda.graph(g):
        opt.step()
    for t in (2, 3, 4):
        if t == 4:
            opt.set_lr(1e-3)
        fill(params, t)
        g.replay()
    for t in (1, 2, 3, 4):
        if t == 4:
            plain.set_lr(1e-3)
        fill(other, t)
        plain.step()
    assert all(torch.equal(p, q) for p, q in zip(params, other))


@pytest.mark.parametrize("capturable", [False, True])
def test_a_scheduler_changes_the_rate(cs, capturable):
    params, other = parameters(), parameters()
    opt = cs.AdamW(params, lr=1e-2, capturable=capturable)
    plan = torch.optim.lr_scheduler.StepLR(opt, step_size=1, gamma=0.5)
    for t in (1, 3, 4):
        set_gradients(params, t)
        opt.step()
        plan.step()
    ms, vs = ([torch.zeros_like(p) for p in other] for _ in range(2))
    for k, t in enumerate((1, 3, 4)):
        cs.adamw_step([p.detach() for p in other], [normal(*p.shape, seed=100 * t + i) for i, p in enumerate(other)], ms, vs, k + 1,
                      lr=1e-2 * 0.5 ** k)
    for p, q in zip(params, other):
        R.close(p.detach(), q.detach(), q.detach().abs() * 3 * 2.0 ** -23 + 0.07 * 2.0 ** -20)  # a rate rounded to float32


def test_optimizer_refuses(cs):
    for bad in (dict(bits=16), dict(seed=-1), dict(seed=1 << 32), dict(max_norm=-1.0), dict(max_norm=math.nan)):
        with pytest.raises(ValueError):
            cs.AdamW(parameters(), **bad)
    opt = cs.AdamW(parameters(), lr=1e-3)
    opt.step()  # nothing has a gradient
    table = torch.nn.Embedding(10, 4, sparse=True).cuda()
    table(torch.tensor([1], device="cuda")).sum().backward()
    with pytest.raises(ValueError, match="dense"):
        cs.AdamW(table.parameters()).step()
