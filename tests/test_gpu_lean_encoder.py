"""The encoder on the training operators where its products run in another type than its sums."""
import pytest

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


@pytest.mark.parametrize("kind", [torch.bfloat16, torch.float16], ids=["bf16", "fp16"])
def test_lean_encoder_under_autocast(kind):
    """As the encoder without under the same autocast.  Some 24 products in a row round both of their operands, 2^-9 of
    them at the mean in bfloat16, and another 24 on the way back: 0.02 of a gradient's norm in each of the two models, and
    0.02 for the activations held in 8 bits."""
    import cswap_b200 as cs
    from cswap_b200.workloads import BertEncoder

    torch.manual_seed(0)
    kw = dict(vocab=100, hidden=128, layers=2, heads=4, ffn=512, max_seq=128, dropout=0.0)
    plain, lean = BertEncoder(**kw).cuda(), BertEncoder(lean=True, **kw).cuda()
    lean.load_state_dict(plain.state_dict())
    ids, target = torch.randint(0, 100, (8, 128), device="cuda"), torch.randint(0, 2, (8,), device="cuda")
    exe = cs.Execution(cs.SwapManager(pinned_bytes=1 << 26, staging_bytes=1 << 26))
    exe.init_(64)

    def step(model):
        with torch.autocast("cuda", dtype=kind):
            loss = model.forward_with(exe, ids, target)
        return loss, torch.autograd.grad(loss, list(model.parameters()))

    (l0, g0), (l1, g1) = step(plain), step(lean)
    assert l1.dtype == torch.float32 and abs(float(l0 - l1)) < 0.02
    scale = max(float(g.norm()) for g in g0)
    for (name, p), a, b in zip(lean.named_parameters(), g0, g1):
        assert b.dtype == p.dtype == torch.float32
        # a key's bias changes no softmax: its gradient is rounding alone
        assert float((a - b).norm()) < 0.06 * float(a.norm()) + 2e-3 * scale, name


def test_lean_encoder_in_16_bits():
    """A model whose parameters are 16-bit themselves."""
    import cswap_b200 as cs
    from cswap_b200.workloads import BertEncoder

    torch.manual_seed(0)
    lean = BertEncoder(vocab=100, hidden=128, layers=1, heads=4, ffn=512, max_seq=128, dropout=0.0, lean=True).cuda().bfloat16()
    exe = cs.Execution(cs.SwapManager(pinned_bytes=1 << 26, staging_bytes=1 << 26))
    exe.init_(64)
    loss = lean.forward_with(exe, torch.randint(0, 100, (2, 50), device="cuda"), torch.tensor([0, 1], device="cuda"))
    for g in torch.autograd.grad(loss, list(lean.parameters())):
        assert g.dtype == torch.bfloat16 and torch.isfinite(g).all()
