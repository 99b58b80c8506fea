"""Layers in 8 bits under the swap engine's policies: what they keep is codes, which no policy touches, so that a policy finds
nothing of theirs to move; what other layers keep beside them moves as ever."""
import pytest

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


@pytest.fixture(scope="module")
def cs():
    import cswap_b200
    assert torch.cuda.is_available()
    cswap_b200.lib()
    return cswap_b200


@pytest.fixture
def mgr(cs):
    m = cs.SwapManager(pinned_bytes=1 << 28, staging_bytes=1 << 28, zfp_maxbits=512)
    yield m
    m.close()


@pytest.fixture
def deterministic():
    torch.use_deterministic_algorithms(True, warn_only=True)  # an embedding's gradient is a sum by atomics else
    yield
    torch.use_deterministic_algorithms(False)


def engine(cs, mgr, n, policy):
    exe = cs.Execution(mgr)
    exe.init_(n)
    for i in range(n):
        exe.begin_stage[i] = i + 1
        exe.policy[i] = policy
    return exe


def normal(*shape, seed=0):
    return torch.randn(*shape, generator=torch.Generator(device="cuda").manual_seed(seed), device="cuda")


WIDTHS = [144, 130, 200, 72, 96]


def chain(cs, exe, x, weights, biases):
    """Layers one behind the other, each wrapped as the drivers wrap theirs."""
    if exe is not None:
        exe.preforward()
    for w, b in zip(weights, biases):
        layer = lambda t, w=w, b=b: cs.fp8_linear(t, w, b)
        if exe is not None:
            exe.pre(x)
        y = layer(x)
        if exe is not None:
            exe.post(x, y, forward=layer)
        x = y
    if exe is not None:
        exe.postforward()
    return x


@pytest.mark.parametrize("policy", ["POLICY_KEEP", "POLICY_DROP", "POLICY_RAW", "POLICY_SPARSE", "POLICY_ZFP", "POLICY_Q8"])
def test_a_chain_of_layers_is_passed_by(cs, mgr, policy):
    """Lossy policies, too, leave every gradient's bits: they would change an activation that a layer kept."""
    x = normal(60, WIDTHS[0], seed=1).requires_grad_(True)
    weights = [normal(b, a, seed=2 + i).requires_grad_(True) for i, (a, b) in enumerate(zip(WIDTHS, WIDTHS[1:]))]
    biases = [normal(b, seed=20 + i).requires_grad_(True) for i, b in enumerate(WIDTHS[1:])]
    dy = normal(60, WIDTHS[-1], seed=30)
    leaves = [x] + weights + biases
    want = torch.autograd.grad(chain(cs, None, x, weights, biases), leaves, dy)
    exe = engine(cs, mgr, 8, getattr(cs, policy))
    got = torch.autograd.grad(chain(cs, exe, x, weights, biases), leaves, dy)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    assert exe.swapped_tensors == exe.held_tensors == exe.recomputed_tensors == 0
    if policy not in ("POLICY_KEEP", "POLICY_DROP"):
        assert exe.skipped_unsaved == len(weights) - 1  # the outputs that a next layer takes


@pytest.mark.parametrize("lean", [True, False])
def test_the_encoder_under_every_policy(cs, mgr, deterministic, lean):
    """Loss and gradients: lossless policies leave their bits, lossy ones those of the loss, which is formed before."""
    from cswap_b200.workloads import BertEncoder

    torch.manual_seed(0)
    model = BertEncoder(vocab=100, hidden=128, layers=2, heads=4, ffn=512, max_seq=128, dropout=0.0, lean=lean, fp8=True).cuda()
    ids, target = torch.randint(0, 100, (8, 128), device="cuda"), torch.randint(0, 2, (8,), device="cuda")

    def run(policy):
        exe = engine(cs, mgr, 80, policy)
        loss = model.forward_with(exe, ids, target)
        return exe, loss.detach(), torch.autograd.grad(loss, list(model.parameters()))

    _, loss, grads = run(cs.POLICY_KEEP)
    _, again, more = run(cs.POLICY_KEEP)
    assert torch.equal(loss, again) and all(torch.equal(a, b) for a, b in zip(grads, more))
    for policy in (cs.POLICY_RAW, cs.POLICY_SPARSE):
        exe, l, g = run(policy)
        assert exe.swapped_tensors > 0
        assert torch.equal(l, loss) and all(torch.equal(a, b) for a, b in zip(g, grads))
    for policy in (cs.POLICY_ZFP, cs.POLICY_Q8):
        exe, l, g = run(policy)
        assert exe.swapped_tensors + exe.held_tensors > 0
        assert torch.equal(l, loss) and all(torch.isfinite(a).all() for a in g)
