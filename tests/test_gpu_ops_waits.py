"""What a program sees of attention's kernels where a wait for their own copies runs out.  A negative limit leaves the
copies out, so that the waits end without them; nothing else on the device is disturbed."""
import os
import subprocess
import sys

import pytest

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
LIMIT, SHORT = 1 << 32, -1000000  # two seconds, half a millisecond without copies
halves = pytest.mark.parametrize("kind", [torch.float16, torch.bfloat16], ids=["fp16", "bf16"])
# one tile; heads of 128, ragged, two tiles of queries a CTA; more pieces than SMs; keys' work split into parts
shapes = pytest.mark.parametrize("b,h,hk,ql,kl,dim,causal", [
    (1, 1, 1, 5, 7, 64, False), (2, 4, 2, 300, 333, 128, True), (8, 12, 12, 260, 260, 40, False), (1, 8, 1, 700, 200, 64, True)])


@pytest.fixture(scope="module")
def cs():
    import cswap_b200
    assert torch.cuda.is_available()
    cswap_b200.lib()
    return cswap_b200


@pytest.fixture
def limit(cs):
    yield lambda clocks: cs.check(cs.lib().csw_attention_wait_limit(clocks), "csw_attention_wait_limit")
    cs.lib().csw_attention_wait_limit(LIMIT)
    torch.cuda.synchronize()
    cs.lib().csw_device_status(None)  # what is left of it


def operands(b, h, hk, ql, kl, dim, kind):
    gen = torch.Generator(device="cuda").manual_seed(1)
    return [torch.randn(b, heads, n, dim, generator=gen, device="cuda").to(kind)
            for heads, n in ((h, ql), (hk, kl), (hk, kl), (h, ql))]


def raises(cs):
    return pytest.raises(cs.CswapError, match="wait ran out")


@halves
@shapes
def test_results_are_nan_and_the_status_is_told_once(cs, limit, kind, b, h, hk, ql, kl, dim, causal):
    q, k, v, do = operands(b, h, hk, ql, kl, dim, kind)
    want = cs.attention_forward(q, k, v, causal=causal)
    grads = cs.attention_backward(do, q, k, v, *want, causal=causal)
    cs.device_status()
    limit(SHORT)
    for t in cs.attention_forward(q, k, v, causal=causal):
        assert torch.isnan(t).all()
    with raises(cs):
        cs.device_status()
    cs.device_status()
    for t in cs.attention_backward(do, q, k, v, *want, causal=causal):
        assert torch.isnan(t).all()
    with raises(cs):
        cs.device_status("cuda")
    limit(LIMIT)
    again = cs.attention_forward(q, k, v, causal=causal)
    for a, w in zip(again + cs.attention_backward(do, q, k, v, *again, causal=causal), want + grads):
        assert torch.equal(a, w)
    cs.device_status()


def test_the_next_call_raises(cs, limit):
    """A program that never asks: the next pass, also one that autograd runs, raises in place of a launch."""
    q, k, v, do = (t.requires_grad_(True) for t in operands(2, 2, 2, 40, 50, 64, torch.bfloat16))
    y = cs.attention(q, k, v)
    limit(SHORT)
    cs.attention(q, k, v)
    torch.cuda.synchronize()
    limit(LIMIT)
    with raises(cs):
        torch.autograd.grad(y, (q, k, v), do, retain_graph=True)
    assert all(torch.isfinite(g).all() for g in torch.autograd.grad(y, (q, k, v), do))
    limit(SHORT)
    cs.attention(q, k, v)
    torch.cuda.synchronize()
    limit(LIMIT)
    with raises(cs):
        cs.attention(q, k, v)
    assert torch.equal(cs.attention(q, k, v), y)


def test_a_replayed_graph_tells(cs, limit):
    """The limit is that of the capture; the status of a replay is told to whoever calls next."""
    q, k, v, _ = operands(1, 2, 2, 40, 50, 64, torch.float16)
    cs.attention_forward(q, k, v)
    limit(SHORT)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        o, _ = cs.attention_forward(q, k, v)
    limit(LIMIT)
    g.replay()
    torch.cuda.synchronize()
    assert torch.isnan(o).all()
    with raises(cs):
        cs.attention_forward(q, k, v)


def test_the_first_call_of_a_process_may_be_captured():
    """The word of host memory that the kernels write is taken then, which a capture would refuse."""
    code = ("import torch, cswap_b200 as cs\n"
            "q = torch.randn(1, 2, 9, 64, device='cuda').half()\n"
            "g = torch.cuda.CUDAGraph()\n"
            "with torch.cuda.graph(g):\n"
            "    o, lse = cs.attention_forward(q, q, q)\n"
            "g.replay()\n"
            "cs.device_status()\n"
            "assert torch.equal(o, cs.attention_forward(q, q, q)[0])\n"
            "print('fine')\n")
    run = subprocess.run([sys.executable, "-c", code], cwd=ROOT, capture_output=True, text=True, timeout=300)
    assert run.returncode == 0 and run.stdout.strip() == "fine", run.stderr[-2000:]
