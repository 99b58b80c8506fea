"""The linear layer in 8 bits under saved-tensor hooks that give back other tensors than they were given."""
import pytest

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

import step_reference as R  # noqa: E402

hooks = torch.autograd.graph.saved_tensors_hooks


@pytest.fixture(scope="module")
def cs():
    import cswap_b200
    assert torch.cuda.is_available()
    cswap_b200.lib()
    return cswap_b200


def normal(*shape, seed=0, kind=torch.float32):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn(*shape, generator=gen, device="cuda").to(kind)


def as_bytes(f):
    """A tensor's values moved by f as bytes."""
    def moved(t):
        return f(t.view(torch.uint8)).view(t.dtype)
    return moved


def apart(t):
    """Rows 32 bytes further apart than they have to be, and 16 bytes behind the beginning."""
    room = torch.full((t.shape[0] + 1, (t.shape[1] + 15) // 16 * 16 + 32), 0x7f, dtype=torch.uint8, device="cuda")
    room[:t.shape[0], 16:16 + t.shape[1]] = t
    return room[:t.shape[0], 16:16 + t.shape[1]]


def off_alignment(t):
    flat = torch.empty(t.numel() + 1, dtype=torch.uint8, device="cuda")[1:]
    return flat.view(t.shape).copy_(t)


MOVES = {
    "the same": lambda t: t,
    "dense": as_bytes(lambda t: t.contiguous().clone()),
    "apart": as_bytes(apart),
    "off its alignment": as_bytes(off_alignment),
    "columns first": as_bytes(lambda t: t.t().contiguous().t()),
    "through the host": lambda t: t.cpu().cuda(),
}


def gradients(cs, context, x, w, b, dy):
    with context:
        y = cs.fp8_linear(x, w, b)
    return [y.detach()] + list(torch.autograd.grad(y, (x, w, b), dy))


# widths that are padded to a multiple of 16, and one that is not; a single row, whose distance to the next one nobody tells
@pytest.mark.parametrize("shape,out", [((100, 515), 40), ((2, 60, 130), 257), ((3, 50), 64), ((1, 50), 7), ((200, 64), 33), ((5, 1), 3)])
def test_what_hooks_give_back_may_lie_otherwise(cs, shape, out):
    x, w, b = (normal(*s, seed=i).requires_grad_(True) for i, s in enumerate((shape, (out, shape[-1]), (out,))))
    dy = normal(*shape[:-1], out, seed=9)
    want = [cs.fp8_linear(x, w, b).detach()] + list(torch.autograd.grad(cs.fp8_linear(x, w, b), (x, w, b), dy))
    contexts = [torch.autograd.graph.save_on_cpu(pin_memory=pin) for pin in (False, True)]
    contexts += [hooks(lambda t: t, move) for move in MOVES.values()]
    for context in contexts:
        for got, t in zip(gradients(cs, context, x, w, b, dy), want):
            assert R.bits_equal(got, t)


def test_a_graph_that_is_kept_gives_the_same_again(cs):
    x, w = normal(70, 50, seed=1).requires_grad_(True), normal(30, 50, seed=2).requires_grad_(True)
    dy = normal(70, 30, seed=3)
    with torch.autograd.graph.save_on_cpu():
        y = cs.fp8_linear(x, w)
    first, second = (torch.autograd.grad(y, (x, w), dy, retain_graph=True) for _ in range(2))
    for a, b in zip(first, second):
        assert R.bits_equal(a, b)


@pytest.mark.parametrize("other", [lambda t: t.cpu(), lambda t: t.view(torch.uint8), lambda t: t.float(), lambda t: t[:, :-1],
                                   lambda t: t.reshape(-1), lambda t: t[:-1]],
                         ids=["on the host", "bytes", "float32", "a column less", "flat", "a row less"])
@pytest.mark.parametrize("which", [0, 1, 2, 3])
def test_another_tensor_is_refused(cs, other, which):
    """One of what the layer keeps: the input's codes and scales, the weight's codes and scales."""
    x, w = normal(140, 150, seed=1).requires_grad_(True), normal(130, 150, seed=2).requires_grad_(True)
    count = iter(range(4))
    with hooks(lambda t: (next(count), t), lambda p: other(p[1]) if p[0] == which else p[1]):
        y = cs.fp8_linear(x, w)
    with pytest.raises(RuntimeError, match="saved-tensor hook"):
        torch.autograd.grad(y.sum(), (x, w))
    assert all(torch.isfinite(g).all() for g in torch.autograd.grad(cs.fp8_linear(x, w).sum(), (x, w)))


@pytest.mark.parametrize("reentrant", [False, True])
def test_a_layer_that_is_computed_again(cs, reentrant):
    """torch's checkpoints, which keep the input alone and run the layers a second time in backward."""
    from torch.utils.checkpoint import checkpoint

    x, v, w = normal(70, 50, seed=1).requires_grad_(True), normal(130, 50, seed=2).requires_grad_(True), normal(30, 130, seed=3).requires_grad_(True)
    dy = normal(70, 30, seed=4)
    two = lambda t: cs.fp8_linear(cs.gelu(cs.fp8_linear(t, v)), w)
    want = torch.autograd.grad(two(x), (x, v, w), dy)
    for t in (x, v, w):
        t.grad = None
    checkpoint(two, x, use_reentrant=reentrant).backward(dy)
    for t, g in zip((x, v, w), want):
        assert R.bits_equal(t.grad, g)
