"""The training operators as a program uses them: several in a row, on other streams, captured and replayed, under the
engine's policies, in the encoder."""
import math

import pytest

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

import ops_reference as R  # noqa: E402


@pytest.fixture(scope="module")
def cs():
    import cswap_b200
    assert torch.cuda.is_available()
    cswap_b200.lib()
    return cswap_b200


def normal(*shape, seed=0, kind=torch.float32):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn(*shape, generator=gen, device="cuda").to(kind)


# One encoder layer on the operators, and the same in torch's own functions in any type.  Sizes small enough for 64 bits.
B, S, H, NH, FF = 2, 70, 64, 4, 160


def parameters(seed=0, kind=torch.float32):
    shapes = dict(q=(H, H), k=(H, H), v=(H, H), o=(H, H), f1=(FF, H), f2=(H, FF), w1=(H,), b1=(H,), w2=(H,), b2=(H,))
    p = {n: (normal(*s, seed=seed + i) / math.sqrt(s[-1]) if len(s) == 2 else normal(*s, seed=seed + i) * 0.1 + (n[0] == "w"))
         for i, (n, s) in enumerate(shapes.items())}
    return {n: t.to(kind).requires_grad_(True) for n, t in p.items()}


def split(t):
    return t.view(B, S, NH, H // NH).transpose(1, 2)


def layer(cs, p, x, lens):
    lin = torch.nn.functional.linear
    half = lambda t: split(t).to(torch.bfloat16)
    a = cs.attention(half(lin(x, p["q"])), half(lin(x, p["k"])), half(lin(x, p["v"])), kv_lens=lens)
    a = lin(a.transpose(1, 2).reshape(B, S, H).to(x.dtype), p["o"])
    x = cs.layer_norm(a, p["w1"], p["b1"], residual=x)
    h = cs.gelu_linear(lin(x, p["f1"]), p["f2"])
    return cs.layer_norm(h, p["w2"], p["b2"], residual=x)


def plain_layer(p, x, lens):
    F = torch.nn.functional
    lin = F.linear
    q, k, v = (split(lin(x, p[n])) for n in "qkv")
    s = (q @ k.transpose(2, 3) * (H // NH) ** -0.5).masked_fill(~R.seen(S, S, False, lens, x.device), -math.inf)
    a = lin((torch.softmax(s, 3) @ v).transpose(1, 2).reshape(B, S, H), p["o"])
    x = F.layer_norm(x + a, (H,), p["w1"], p["b1"])
    h = lin(F.gelu(lin(x, p["f1"])), p["f2"])
    return F.layer_norm(x + h, (H,), p["w2"], p["b2"])


def run(f, p, x, dy):
    y = f(p, x)
    return [y] + list(torch.autograd.grad(y, [x] + list(p.values()), dy))


LENS = [70, 41]


def test_a_layer_of_all_operators(cs):
    """Forward and every gradient against the layer in 64 bits.  The operands of attention are rounded to bfloat16 (2^-9
    of them at the mean, through four products), the feed-forward activation to 254 steps of its group (0.4 % of the
    largest of 128 values, in backward alone): a norm of the error of 2 % of the result's bounds both; a missing or
    doubled term is off by far more."""
    lens = torch.tensor(LENS, dtype=torch.int32, device="cuda")
    p, x, dy = parameters(), normal(B, S, H, seed=50).requires_grad_(True), normal(B, S, H, seed=51)
    got = run(lambda q, t: layer(cs, q, t, lens), p, x, dy)
    wide = {n: t.detach().double().requires_grad_(True) for n, t in p.items()}
    xd = x.detach().double().requires_grad_(True)
    want = run(lambda q, t: plain_layer(q, t, lens), wide, xd, dy.double())
    for name, g, w in zip(["y", "x"] + list(p), got, want):
        assert g.dtype == torch.float32 and g.shape == w.shape
        assert float((g.double() - w).norm() / w.norm()) < 0.02, name
    again = run(lambda q, t: layer(cs, q, t, lens), p, x, dy)
    for g, a in zip(got, again):
        assert torch.equal(g, a)  # nothing is added in the order in which it happens to come


def test_other_streams(cs):
    """Two streams at once, each with its own tensors: the results of one after the other."""
    lens = torch.tensor(LENS, dtype=torch.int32, device="cuda")
    sets = [(parameters(seed=i), normal(B, S, H, seed=60 + i).requires_grad_(True), normal(B, S, H, seed=70 + i))
            for i in range(2)]
    want = [run(lambda q, t: layer(cs, q, t, lens), *s) for s in sets]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in sets]
    for _ in range(5):
        got = []
        for st, s in zip(streams, sets):
            with torch.cuda.stream(st):
                got.append(run(lambda q, t: layer(cs, q, t, lens), *s))
        torch.cuda.synchronize()
        for g, w in zip(got, want):
            assert all(torch.equal(a, b) for a, b in zip(g, w))


def test_captured_and_replayed(cs):
    """A step and its backward pass in a CUDA graph, replayed on new values; two graphs of the same step do not share
    memory that one would overwrite for the other."""
    lens = torch.tensor(LENS, dtype=torch.int32, device="cuda")
    p = parameters()
    xs = [normal(B, S, H, seed=80 + i) for i in range(2)]
    dy = normal(B, S, H, seed=82)
    eager = [run(lambda q, t: layer(cs, q, t, lens), p, x.clone().requires_grad_(True), dy) for x in xs]
    eager = [[t.detach().clone() for t in e] for e in eager]
    graphs = []
    for _ in range(2):
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        mine = {n: t.detach().clone().requires_grad_(True) for n, t in p.items()}
        x = xs[0].clone().requires_grad_(True)
        with torch.cuda.stream(side):
            run(lambda q, t: layer(cs, q, t, lens), mine, x, dy)  # products pick their kernels outside of the capture
        torch.cuda.current_stream().wait_stream(side)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = run(lambda q, t: layer(cs, q, t, lens), mine, x, dy)
        graphs.append((g, x, [t.detach() for t in out]))
    for i in (0, 1):
        graphs[i][1].data.copy_(xs[i])
    for g, _, _ in graphs + graphs[::-1]:
        g.replay()
    torch.cuda.synchronize()
    for i in (0, 1):
        for a, b in zip(graphs[i][2], eager[i]):
            assert float((a - b).abs().max()) <= 1e-5 * float(b.abs().max())  # torch's products may choose otherwise


def test_a_capture_beside_a_live_graph_of_the_same_leaves_is_refused(cs):
    w = torch.ones(64, device="cuda").requires_grad_(True)
    x = normal(8, 64)
    alive = cs.layer_norm(x, w)  # holds w's accumulator, of this stream
    g = torch.cuda.CUDAGraph()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        g.capture_begin()
        try:
            with pytest.raises(RuntimeError, match="live graph"):
                cs.layer_norm(x, w)
            y = x + 1  # the capture itself goes on
        finally:
            g.capture_end()
    assert torch.autograd.grad(alive.sum(), w)[0].shape == w.shape
    del alive
    with torch.cuda.graph(g2 := torch.cuda.CUDAGraph()):
        gw, = torch.autograd.grad(cs.layer_norm(x, w), w, torch.ones_like(x))
    g2.replay()
    torch.cuda.synchronize()
    assert torch.isfinite(gw).all() and y.shape == x.shape


def test_policy_8_is_the_step_on_held_values(cs):
    """The engine under policy 8: outputs as without it, gradients those of a step whose saved activations are replaced
    by what their checkpoints hold, a quarter of the memory."""
    from cswap_b200 import Execution, LayerType

    torch.manual_seed(0)
    layers = [torch.nn.Linear(96, 128), torch.nn.Tanh(), torch.nn.Linear(128, 96), torch.nn.Tanh(), torch.nn.Linear(96, 8)]
    layers = [l.cuda() for l in layers]
    x = normal(64, 96, seed=1)

    def step(exe, hold):
        pre = x.clone().requires_grad_(True)
        exe.preforward()
        first = pre
        for l in layers:
            exe.pre(pre, LayerType.FC)
            out = l(pre)
            exe.post(pre, out, LayerType.FC)
            pre = out
        exe.postforward()
        params = [q for l in layers for q in l.parameters()]
        return pre.detach(), torch.autograd.grad(pre.square().sum(), [first] + params)

    def engine(pol):
        exe = Execution(cs.SwapManager(pinned_bytes=1 << 24, staging_bytes=1 << 24), min_numel=1)
        exe.init_(8)
        for i in range(8):
            exe.begin_stage[i], exe.policy[i] = i + 1, pol
        return exe

    plain = step(engine(cs.POLICY_KEEP), False)
    exe = engine(cs.POLICY_Q8)
    held = step(exe, True)
    # what is kept: each tanh keeps its output, which is the next linear layer's input; nothing keeps a linear one's
    assert exe.held_tensors == 2 and exe.swapped_tensors == 0 and torch.equal(held[0], plain[0])

    def pack(t):
        if t.is_cuda and t.dtype == torch.float32 and not (t.is_leaf and t.requires_grad) and t.grad_fn is not None and t.shape[0] == 64:
            return cs.q8_compress(t.contiguous()), t.shape
        return t

    def unpack(v):
        return v if isinstance(v, torch.Tensor) else cs.q8_decompress(v[0], math.prod(v[1])).view(v[1])

    pre = first = x.clone().requires_grad_(True)
    with torch.autograd.graph.saved_tensors_hooks(pack, unpack):
        for l in layers:
            pre = l(pre)
    want = torch.autograd.grad(pre.square().sum(), [first] + [q for l in layers for q in l.parameters()])
    for a, b, c in zip(held[1], want, plain[1]):
        assert torch.equal(a, b) and float((a - c).norm() / c.norm()) < 0.02
    import cswap_b200.compat as compat
    compat.cswapinit_(cs.SwapManager(pinned_bytes=1 << 24, staging_bytes=1 << 24))
    compat.execution().min_numel = 1
    compat.cswapinit()
    a = x.clone().requires_grad_(True)
    compat.cswappre(a)
    h = layers[0](a)
    compat.cswappost(a, h)
    compat.cswappre(h, cs.POLICY_Q8)
    y = layers[2](h)
    compat.cswappost(h, y)
    compat.execution().postforward()
    assert compat.execution().held_tensors == 1
    torch.autograd.grad(y.sum(), a)


def test_lean_encoder(cs):
    """The encoder on the operators against itself without: loss and gradients, and what backward has to keep."""
    from cswap_b200.workloads import BertEncoder

    class Numbers:
        index = -1

        def preforward(self):
            self.index = -1

        def postforward(self):
            pass

        def pre(self, x, lt=None):
            self.index += 1

        def post(self, x, y, lt=None, omit=False, forward=None):
            y.tensor_id = self.index

    torch.manual_seed(0)
    kw = dict(vocab=100, hidden=128, layers=2, heads=4, ffn=512, max_seq=128, dropout=0.0)
    plain, lean = BertEncoder(**kw).cuda(), BertEncoder(lean=True, **kw).cuda()
    lean.load_state_dict(plain.state_dict())
    ids = torch.randint(0, 100, (8, 128), device="cuda")
    target = torch.randint(0, 2, (8,), device="cuda")

    def step(model):
        kept = {}

        def pack(t):
            if not (t.is_leaf and t.requires_grad):
                kept[t.untyped_storage().data_ptr()] = t.untyped_storage().nbytes()
            return t

        with torch.autograd.graph.saved_tensors_hooks(pack, lambda t: t):
            loss = model.forward_with(Numbers(), ids, target)
        return loss, torch.autograd.grad(loss, [p for p in model.parameters()]), sum(kept.values())

    l0, g0, k0 = step(plain)
    l1, g1, k1 = step(lean)
    assert abs(float(l0 - l1)) < 0.01
    scale = max(float(g.norm()) for g in g0)
    for (name, _), a, b in zip(plain.named_parameters(), g0, g1):
        # a key's bias changes no softmax: its gradient is rounding alone
        assert float((a - b).norm()) < 0.03 * float(a.norm()) + 1e-3 * scale, name
    assert k1 < 0.6 * k0
    exe = cs.Execution(cs.SwapManager(pinned_bytes=1 << 26, staging_bytes=1 << 26))
    exe.init_(64)
    for i in range(64):
        exe.begin_stage[i], exe.policy[i] = i + 1, cs.POLICY_Q8
    loss = lean.forward_with(exe, ids, target)
    got = torch.autograd.grad(loss, list(lean.parameters()))
    assert torch.equal(loss, l1) and exe.held_tensors > 4
    for a, b in zip(got, g1):
        assert float((a - b).norm()) < 0.05 * float(b.norm()) + 2e-3 * scale


def test_autocast(cs):
    x, w = normal(5, 7, 64, seed=1).requires_grad_(True), normal(32, 64, seed=2).requires_grad_(True)
    with torch.autocast("cuda", dtype=torch.bfloat16):
        y = cs.gelu_linear(x, w)
    assert y.dtype == torch.bfloat16
    gx, gw = torch.autograd.grad(y.float().sum(), [x, w])
    assert gx.dtype == gw.dtype == torch.float32
    want = torch.autograd.grad(cs.gelu_linear(x, w).sum(), [x, w])
    for a, b in zip((gx, gw), want):
        assert float((a - b).norm() / b.norm()) < 0.02  # products of 7-bit values: 2^-8 each of their two operands


def test_the_current_device_need_not_be_the_tensors(cs):
    if torch.cuda.device_count() < 2:
        pytest.skip("one device")
    x = torch.randn(8, 64, device="cuda:1")
    assert cs.layer_norm(x).device == x.device
