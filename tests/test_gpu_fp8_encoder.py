"""The encoder with its layers in 8 bits against the one without, whose layers are made of quantizing and products one by one."""
import pytest

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

import step_reference as R  # noqa: E402

LAYERS = ("q", "k", "v", "o", "f1", "f2")


@pytest.fixture(scope="module")
def cs():
    import cswap_b200
    assert torch.cuda.is_available()
    cswap_b200.lib()
    return cswap_b200


@pytest.fixture
def deterministic():
    torch.use_deterministic_algorithms(True, warn_only=True)  # an embedding's gradient is a sum by atomics else
    yield
    torch.use_deterministic_algorithms(False)


class ByParts(torch.autograd.Function):
    """y = x w^T + b and its gradients by the operators that the layer is made of, each result within the bound of its product in
    64 bits; `seen` notes that a layer's backward pass has come by."""

    @staticmethod
    def forward(ctx, cs, seen, x, w, b):
        ctx.cs, ctx.seen = cs, seen
        qx, qw = cs.fp8_quantize(x), cs.fp8_quantize(w)
        ctx.save_for_backward(*qx, *qw)
        ctx.shape = x.shape
        y = cs.fp8_matmul(*qx, *qw, transpose_b=True, bias=b, dtype=x.dtype)
        R.close(y, *R.product(R.held_of(*qx), R.held_of(*qw).t(), b, x.dtype))
        return y.view(*x.shape[:-1], w.shape[0])

    @staticmethod
    def backward(ctx, dy):
        cs, saved = ctx.cs, ctx.saved_tensors
        qx, qw = saved[:2], saved[2:]
        *g, sums = cs.fp8_quantize(dy.contiguous(), sums=True)
        dx = cs.fp8_matmul(*g, *qw, dtype=dy.dtype)
        dw = cs.fp8_matmul(*g, *qx, transpose_a=True, dtype=dy.dtype)
        G = R.held_of(*g)
        R.close(dx, *R.product(G, R.held_of(*qw), None, dy.dtype))
        R.close(dw, *R.product(G.t(), R.held_of(*qx), None, dy.dtype))
        rows = G.shape[0]
        wide = dy.double().flatten(0, -2)
        R.close(sums, wide.sum(0), wide.abs().sum(0) * ((rows / 8 + 24) * 2.0 ** -24))
        ctx.seen.append(1)
        return None, None, dx.view(ctx.shape), dw, sums


@pytest.mark.parametrize("lean", [True, False])
def test_every_parameter_s_gradient(cs, deterministic, monkeypatch, lean):
    """Loss and every gradient have the same bits: nothing but the layers' own node is another way, and whatever it left out or
    mixed up, in any layer, would show in its parameters' gradients."""
    from cswap_b200 import workloads

    torch.manual_seed(0)
    kw = dict(vocab=100, hidden=144, layers=2, heads=3, ffn=520, max_seq=80, dropout=0.0, lean=lean)
    eight, plain = workloads.BertEncoder(fp8=True, **kw).cuda(), workloads.BertEncoder(**kw).cuda()
    for p in eight.parameters():  # biases and norms' weights, which begin at 0 and 1, as they are after some steps
        if p.dim() == 1:
            p.data.add_(torch.randn_like(p) * 0.1)
    plain.load_state_dict(eight.state_dict())
    seen = []
    for name in LAYERS:
        for m in getattr(plain, name):
            m.forward = lambda x, m=m: ByParts.apply(cs, seen, x, m.weight, m.bias)
    # the lean encoder's second product has its activation with it
    monkeypatch.setattr(workloads, "gelu_linear", lambda t, w, b: ByParts.apply(cs, seen, cs.gelu(t), w, b))
    ids, target = torch.randint(0, 100, (5, 77), device="cuda"), torch.randint(0, 2, (5,), device="cuda")
    exe = cs.Execution(cs.SwapManager(pinned_bytes=1 << 26, staging_bytes=1 << 26))
    exe.init_(80)
    losses = [m.forward_with(exe, ids, target) for m in (eight, plain)]
    grads = [torch.autograd.grad(l, list(m.parameters())) for l, m in zip(losses, (eight, plain))]
    assert len(seen) == 2 * len(LAYERS)
    assert R.bits_equal(losses[0].detach(), losses[1].detach())
    for (name, p), a, b in zip(eight.named_parameters(), *grads):
        assert float(a.norm()) > 0 and R.bits_equal(a, b), name
