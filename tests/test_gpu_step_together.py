"""Linear layers in 8 bits and the optimizer's step as a program uses them: in the encoder, with the other training operators,
on other streams, captured and replayed, between kernels that rewrite their inputs, and where a wait runs out."""
import math

import pytest

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

import step_reference as R  # noqa: E402

LIMIT, SHORT = 1 << 32, -1000000  # two seconds, half a millisecond without copies


@pytest.fixture(scope="module")
def cs():
    import cswap_b200
    assert torch.cuda.is_available()
    cswap_b200.lib()
    return cswap_b200


def normal(*shape, seed=0, kind=torch.float32):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn(*shape, generator=gen, device="cuda").to(kind)


# A block of linear layers, norm and activation on the operators, and the same in 64 bits with the operands of its products
# rounded as the layer rounds them.
ROWS, H, FF = 150, 96, 200


def parameters(seed=0):
    shapes = dict(a=(FF, H), ab=(FF,), b=(H, FF), bb=(H,), w=(H,), wb=(H,))
    return {n: (normal(*s, seed=seed + i) / math.sqrt(s[-1]) if len(s) == 2 else normal(*s, seed=seed + i) * 0.1 + (n == "w")
                ).requires_grad_(True) for i, (n, s) in enumerate(shapes.items())}


def block(cs, p, x):
    h = cs.gelu(cs.fp8_linear(x, p["a"], p["ab"]))
    return cs.layer_norm(cs.fp8_linear(h, p["b"], p["bb"]), p["w"], p["wb"], residual=x)


class Rounded(torch.autograd.Function):
    @staticmethod
    def forward(ctx, cs, x, w, b):
        hold = lambda t: R.held_of(*cs.fp8_quantize(t.float()))
        x, w = hold(x), hold(w)
        ctx.save_for_backward(x, w)
        ctx.hold = hold
        return x @ w.t() + b

    @staticmethod
    def backward(ctx, dy):
        x, w = ctx.saved_tensors
        g = ctx.hold(dy)
        return None, g @ w, g.t() @ x, dy.sum(0)


def plain_block(cs, p, x):
    F = torch.nn.functional
    h = F.gelu(Rounded.apply(cs, x, p["a"], p["ab"]))
    return F.layer_norm(x + Rounded.apply(cs, h, p["b"], p["bb"]), (H,), p["w"], p["wb"])


def run(f, p, x, dy):
    y = f(p, x)
    return [y] + list(torch.autograd.grad(y, [x] + list(p.values()), dy))


def test_a_block_of_layers(cs):
    """Forward and every gradient.  The two differ where float32 and 64 bits fall on different sides of a code's border (a share of
    2^-17 of the values, each by a sixteenth) and by GELU's gradient on 254 steps of its group, half a percent of the largest of 128
    values: 2 % of a result's norm bounds both."""
    p, x, dy = parameters(), normal(ROWS, H, seed=50).requires_grad_(True), normal(ROWS, H, seed=51)
    got = run(lambda q, t: block(cs, q, t), p, x, dy)
    wide = {n: t.detach().double().requires_grad_(True) for n, t in p.items()}
    want = run(lambda q, t: plain_block(cs, q, t), wide, x.detach().double().requires_grad_(True), dy.double())
    for name, g, w in zip(["y", "x"] + list(p), got, want):
        assert g.dtype == torch.float32 and g.shape == w.shape
        assert float((g.detach().double() - w.detach()).norm() / w.detach().norm()) < 0.02, name
    for g, a in zip(got, run(lambda q, t: block(cs, q, t), p, x, dy)):
        assert torch.equal(g, a)


@pytest.mark.parametrize("lean", [True, False])
def test_the_encoder_in_8_bits(cs, lean):
    """Against the encoder as it is.  A value's rounding to e4m3 is 2^-5.2 of it at the mean, a product's two operands 0.038 of its
    result; four products one behind the other in each of two layers, there and back, and a gradient's own: 0.16 of a gradient's
    norm if they added like noise, and twice that for what norms and softmax make of it.  A missing term is 1 or more off."""
    from cswap_b200.workloads import BertEncoder

    torch.manual_seed(0)
    kw = dict(vocab=100, hidden=128, layers=2, heads=4, ffn=512, max_seq=128, dropout=0.0)
    plain, eight = BertEncoder(**kw).cuda(), BertEncoder(lean=lean, fp8=True, **kw).cuda()
    eight.load_state_dict(plain.state_dict())
    ids, target = torch.randint(0, 100, (8, 128), device="cuda"), torch.randint(0, 2, (8,), device="cuda")
    exe = cs.Execution(cs.SwapManager(pinned_bytes=1 << 26, staging_bytes=1 << 26))
    exe.init_(64)
    grads = [torch.autograd.grad(model.forward_with(exe, ids, target), list(model.parameters())) for model in (plain, eight)]
    scale = max(float(g.norm()) for g in grads[0])
    for (name, p), a, b in zip(eight.named_parameters(), *grads):
        assert b.dtype == p.dtype and torch.isfinite(b).all()
        assert float((a - b).norm()) < 0.32 * float(a.norm()) + 0.02 * scale, name


def test_a_training_step_with_the_optimizer(cs):
    """timed_steps with an optimizer in 8 bits: every parameter that has a gradient moves, by less than 2.2 lr a step (the first
    four steps of Adam: |m| is at most sqrt(v) corrected, times what a code's rounding adds, and the weight decay)."""
    from cswap_b200.workloads import BertEncoder, timed_steps

    torch.manual_seed(0)
    model = BertEncoder(vocab=50, hidden=64, layers=1, heads=2, ffn=128, max_seq=32, dropout=0.0, lean=True, fp8=True).cuda()
    exe = cs.Execution(cs.SwapManager(pinned_bytes=1 << 26, staging_bytes=1 << 26))
    exe.init_(40)
    opt = cs.AdamW(model.parameters(), lr=1e-3, bits=8, max_norm=1.0)
    before = [p.detach().clone() for p in model.parameters()]
    batch = lambda: (torch.randint(0, 50, (4, 32)).pin_memory(), torch.randint(0, 2, (4,)).pin_memory())
    out = timed_steps(model, exe, batch, steps=3, warmup=1, optimizer=opt)
    assert math.isfinite(out["loss"])
    for old, (name, p) in zip(before, model.named_parameters()):
        moved = float((p.detach() - old).abs().max())
        assert moved <= 4 * 2.2e-3 and (moved > 0 or p.grad is None or not p.grad.any()), name


def test_other_streams(cs):
    """Two streams at once, each with its own tensors: the results of one after the other."""
    sets = [(parameters(seed=10 * i), normal(ROWS, H, seed=60 + i).requires_grad_(True), normal(ROWS, H, seed=70 + i)) for i in range(2)]

    def step(p, x, dy):
        r = run(lambda q, t: block(cs, q, t), p, x, dy)
        new, states = [t.detach().clone() for t in p.values()], [cs.adamw8_state(t) for t in p.values()]
        cs.adamw8_step(new, r[2:], states, 1, norm=cs.gradient_norm(r[2:]), max_norm=0.1)
        return r + new + [c for s in states for c in s]

    want = [step(*s) for s in sets]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in sets]
    for _ in range(5):
        got = []
        for st, s in zip(streams, sets):
            with torch.cuda.stream(st):
                got.append(step(*s))
        torch.cuda.synchronize()
        for g, w in zip(got, want):
            assert all(torch.equal(a, b) for a, b in zip(g, w))


@pytest.mark.parametrize("bits", [32, 8])
def test_a_captured_training_step(cs, bits):
    """Forward, backward, clipping and the optimizer in a graph, replayed on new inputs: what the same steps do one by one."""
    def make():
        p = parameters(seed=30)
        opt = cs.AdamW(list(p.values()), lr=1e-2, bits=bits, max_norm=0.5, capturable=True, seed=3)
        return p, opt

    def step(p, opt, x, dy):
        y = block(cs, p, x)
        for q, g in zip(p.values(), torch.autograd.grad(y, list(p.values()), dy)):
            q.grad = g
        opt.step()
        return y.detach()

    xs, dys = [normal(ROWS, H, seed=80 + i) for i in range(4)], [normal(ROWS, H, seed=90 + i) for i in range(4)]
    p, opt = make()
    want = [step(p, opt, x, dy) for x, dy in zip(xs, dys)]
    q, other = make()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        first = step(q, other, xs[0], dys[0])
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(first, want[0])
    x, dy = xs[0].clone(), dys[0].clone()
    for t in q.values():
        t.grad = None
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        y = step(q, other, x, dy)
    for i in (1, 2, 3):
        x.copy_(xs[i])
        dy.copy_(dys[i])
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, want[i])
    for a, b in zip(p.values(), q.values()):
        assert torch.equal(a, b)


@pytest.mark.parametrize("which", ["x", "weight", "bias"])
def test_a_captured_layer_whose_leaf_has_a_live_graph(cs, which):
    """A leaf whose gradient belongs to a live graph of another stream, behind a view, too, is refused in a capture; without that
    graph the layer is captured, and its replay gives the gradient that the eager layer gave."""
    sets = {"x": normal(64, 40, seed=1), "weight": normal(64, 24, seed=2), "bias": normal(24, seed=3)}
    leaf = sets[which].requires_grad_(True)
    call = lambda: cs.fp8_linear(sets["x"].t(), sets["weight"].t(), sets["bias"].view(24))
    dy = normal(40, 24, seed=4)
    alive = call()
    ones = torch.ones(4, device="cuda")
    g, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    raised = None
    with torch.cuda.stream(side):
        g.capture_begin()
        try:
            call()
        except RuntimeError as err:
            raised = str(err)
        finally:
            keep = ones + 1  # the capture itself goes on
            g.capture_end()
    assert raised is not None and "live graph" in raised and keep.shape == (4,)
    grad, = torch.autograd.grad(alive, leaf, dy)
    del alive
    with torch.cuda.graph(g2 := torch.cuda.CUDAGraph()):
        again, = torch.autograd.grad(call(), leaf, dy)
    g2.replay()
    torch.cuda.synchronize()
    assert torch.equal(again, grad)


@pytest.mark.parametrize("m,n,k", [(77, 96, 200), (1, 4096, 4096), (2048, 2048, 512)])
def test_between_kernels_that_rewrite_the_inputs(cs, m, n, k):
    """A kernel that writes x right before the call and one that overwrites it right behind: the results of the call alone."""
    w = cs.fp8_quantize(normal(n, k, seed=1))
    buffer = torch.empty(1 << 26, device="cuda")
    x = buffer[-m * k:].view(m, k)
    src = normal(m, k, seed=2)
    want = cs.fp8_linear(src, w)
    for _ in range(5):
        buffer.fill_(7.0)  # 40 us of work in front
        x.copy_(src)
        got = cs.fp8_linear(x, w)
        buffer.fill_(-3.0)
        assert torch.equal(got, want)


def test_offsets_beyond_32_bits(cs):
    """A matrix of more than 2^32 values: its last rows' codes and their products are those of the rows on their own."""
    rows, cols = 1 << 17, (1 << 15) + 16
    x = torch.empty(rows, cols, dtype=torch.bfloat16, device="cuda")
    x[:128] = normal(128, cols, seed=1)
    x[-128:] = normal(128, cols, seed=2)
    x[128:-128] = 0.0
    codes, scales = cs.fp8_quantize(x)
    for part, rows_of in ((slice(0, 128), slice(0, 1)), (slice(rows - 128, rows), slice(-1, None))):
        c, s = cs.fp8_quantize(x[part].contiguous())
        assert torch.equal(codes[part].view(torch.uint8), c.view(torch.uint8))
        assert torch.equal(scales[rows_of].view(torch.uint8), s.view(torch.uint8))
        assert torch.equal(cs.fp8_dequantize(codes, scales, torch.bfloat16)[part], cs.fp8_dequantize(c, s, torch.bfloat16))
        w = cs.fp8_quantize(normal(8, cols, seed=3))
        assert torch.equal(cs.fp8_matmul(codes, scales, *w, transpose_b=True)[part], cs.fp8_matmul(c, s, *w, transpose_b=True))
    del x, codes, scales


# ---- waits ---------------------------------------------------------------------------------------------------------

@pytest.fixture
def limit(cs):
    yield lambda clocks: cs.check(cs.lib().csw_attention_wait_limit(clocks), "csw_attention_wait_limit")
    cs.lib().csw_attention_wait_limit(LIMIT)
    torch.cuda.synchronize()
    cs.lib().csw_device_status(None)  # what is left of it


def raises(cs):
    return pytest.raises(cs.CswapError, match="wait ran out")


@pytest.mark.parametrize("kind", [torch.float32, torch.bfloat16], ids=["fp32", "bf16"])
# a tile; operands exchanged, parts of the reduction; parts of a square result; tiles of pairs, several to a pair; more tiles than SMs
@pytest.mark.parametrize("m,n,k", [(5, 7, 64), (3, 4096, 4096), (128, 200, 4096), (2048, 5120, 300), (3000, 80, 200)])
def test_results_are_nan_and_the_status_is_told_once(cs, limit, kind, m, n, k):
    a, b = cs.fp8_quantize(normal(m, k, seed=1)), cs.fp8_quantize(normal(n, k, seed=2))
    product = lambda: cs.fp8_matmul(*a, *b, transpose_b=True, dtype=kind)
    want = product()
    cs.device_status()
    limit(SHORT)
    assert torch.isnan(product()).all()
    with raises(cs):
        cs.device_status()
    cs.device_status()
    limit(LIMIT)
    assert torch.equal(product(), want)
    cs.device_status()


def test_a_layer_of_a_few_rows_is_nan_too(cs, limit):
    x, w = normal(3, 2000), cs.fp8_quantize(normal(600, 2000, seed=1))
    want = cs.fp8_linear(x, w)
    limit(SHORT)
    assert torch.isnan(cs.fp8_linear(x, w)).all()
    limit(LIMIT)
    with raises(cs):
        cs.fp8_linear(x, w)
    assert torch.equal(cs.fp8_linear(x, w), want)


def test_the_next_call_raises(cs, limit):
    """Also in a backward pass, where autograd's thread makes the call."""
    x, w = normal(40, 64).requires_grad_(True), normal(30, 64, seed=1).requires_grad_(True)
    y = cs.fp8_linear(x, w)
    limit(SHORT)
    cs.fp8_linear(x, w)
    torch.cuda.synchronize()
    limit(LIMIT)
    with raises(cs):
        torch.autograd.grad(y.sum(), (x, w), retain_graph=True)
    assert all(torch.isfinite(g).all() for g in torch.autograd.grad(y.sum(), (x, w)))
