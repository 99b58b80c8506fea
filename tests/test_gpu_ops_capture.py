"""Captures beside a live graph of the same leaf on another stream, where the operator is given the leaf in another form
than the leaf itself.  The backward pass of such a capture would end the process; the call in front of it raises."""
import pytest

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


@pytest.fixture(scope="module")
def cs():
    import cswap_b200
    assert torch.cuda.is_available()
    cswap_b200.lib()
    return cswap_b200


def normal(*shape, kind=torch.float32):
    gen = torch.Generator(device="cuda").manual_seed(3)
    return torch.randn(*shape, generator=gen, device="cuda").to(kind)


def half_heads(t):
    return t.view(2, 9, 4, 16).transpose(1, 2).to(torch.bfloat16)


# the leaf, another operand, the call
CALLS = {
    "gelu of a transposed leaf": ((24, 8), None, lambda cs, x, o: cs.gelu(x.t())),
    "gelu_linear of a transposed leaf": ((64, 8), (5, 64), lambda cs, x, o: cs.gelu_linear(x.t(), o)),
    "layer_norm of a transposed leaf": ((64, 8), None, lambda cs, x, o: cs.layer_norm(x.t())),
    "layer_norm with a transposed residual": ((64, 8), (8, 64), lambda cs, x, o: cs.layer_norm(o, residual=x.t())),
    "layer_norm of a part of a leaf": ((9, 64), None, lambda cs, x, o: cs.layer_norm(x[1:])),
    "layer_norm of a leaf that is not contiguous": ((64, 64), None, lambda cs, x, o: cs.layer_norm(x)),
    "attention on heads of a leaf": ((2, 9, 64), None, lambda cs, x, o: cs.attention(*[half_heads(x)] * 3)),
}


@pytest.mark.parametrize("name", list(CALLS))
def test_a_leaf_behind_a_view_or_a_copy_is_found(cs, name):
    shape, other, f = CALLS[name]
    leaf = normal(*shape)
    leaf = (leaf.t() if "not contiguous" in name else leaf).requires_grad_(True)
    other = other and normal(*other)
    call = lambda cs, x: f(cs, x, other)
    assert leaf.is_leaf
    alive = call(cs, leaf)  # its graph holds the leaf's accumulator, of this stream
    ones = torch.ones(4, device="cuda")
    g, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    raised = None
    with torch.cuda.stream(side):
        g.capture_begin()
        try:
            call(cs, leaf)
        except RuntimeError as err:
            raised = str(err)  # its traceback would keep the copy that was made, and with it the accumulator
        finally:
            keep = ones + 1  # the capture itself goes on
            g.capture_end()
    assert raised is not None and "live graph" in raised
    grad, = torch.autograd.grad(alive.float().sum(), leaf)
    del alive
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):  # products pick their kernels outside of the capture
        torch.autograd.grad(call(cs, leaf).float().sum(), leaf)
    torch.cuda.current_stream().wait_stream(side)
    with torch.cuda.graph(g2 := torch.cuda.CUDAGraph()):
        again, = torch.autograd.grad(call(cs, leaf).float().sum(), leaf)
    g2.replay()
    torch.cuda.synchronize()
    assert keep.shape == (4,) and float((again - grad).abs().max()) <= 1e-3 * (1 + float(grad.abs().max()))
