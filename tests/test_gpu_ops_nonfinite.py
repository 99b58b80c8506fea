"""Attention on operands that hold a NaN or an infinity where queries see it: what the 64-bit form cannot compute must not
come out as a number, whichever position of a tile it stands at."""
import math

import pytest

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

import ops_reference as R  # noqa: E402

halves = pytest.mark.parametrize("kind", [torch.float16, torch.bfloat16], ids=["fp16", "bf16"])
COLUMN = 3


@pytest.fixture(scope="module")
def cs():
    import cswap_b200
    assert torch.cuda.is_available()
    cswap_b200.lib()
    return cswap_b200


def normal(*shape, seed=0, kind=torch.float32):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn(*shape, generator=gen, device="cuda").to(kind)


def definition(q, k, v, do, causal=False, lens=None):
    """(o, lse, dq, dk, dv) in 64 bits, every product taken, those with a probability of zero as well; rows that see
    nothing are zero, keys behind a sequence do not count."""
    q, k, v, do = (t.double() for t in (q, k, v, do))
    share, scale = q.shape[1] // k.shape[1], q.shape[3] ** -0.5
    if lens is not None:
        dead = (torch.arange(k.shape[2], device=k.device)[None, :] >= lens.long()[:, None])[:, None, :, None]
        k, v = k.masked_fill(dead, 0.0), v.masked_fill(dead, 0.0)
    k, v = k.repeat_interleave(share, 1), v.repeat_interleave(share, 1)
    seen = R.seen(q.shape[2], k.shape[2], causal, lens, q.device)
    s = (q @ k.transpose(2, 3) * scale).masked_fill(~seen, -math.inf)
    p = torch.softmax(s, 3).masked_fill(~seen, 0.0)
    o = p @ v
    ds = p * (do @ v.transpose(2, 3) - (do * o).sum(3, keepdim=True))

    def group(t):  # keys behind a sequence have no gradient
        t = t.unflatten(1, (-1, share)).sum(2)
        return t if lens is None else t.masked_fill(dead, 0.0)

    return o, torch.logsumexp(s, 3), ds @ k * scale, group(ds.transpose(2, 3) @ q * scale), group(p.transpose(2, 3) @ do)


def passes(cs, q, k, v, do, **kw):
    o, lse = cs.attention_forward(q, k, v, **kw)
    return (o, lse) + tuple(cs.attention_backward(do, q, k, v, o, lse, **kw))


def check(got, want, v):
    for name, g, w in zip(("o", "lse", "dq", "dk", "dv"), got, want):
        assert torch.equal(torch.isnan(g), torch.isnan(w)), name
        assert torch.equal(torch.isinf(g), torch.isinf(w)), name
    # a row that can be computed is a mean of values: each probability and the result rounded once, 2^-10 of both for float32
    most = v.masked_fill(~torch.isfinite(v), 0.0).double().abs().max()
    fine = torch.isfinite(want[0])
    off = (got[0].double() - want[0]).abs()[fine]
    assert off.numel() == 0 or float(off.max()) <= 2.5 * R.U[v.dtype] * float(most)
    fine = torch.isfinite(want[1])
    off = ((got[1].double() - want[1]).abs() / (1 + want[1].abs()))[fine]
    assert off.numel() == 0 or float(off.max()) <= 2.0 ** -10


@halves
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("ql,kl,first", [(150, 150, 40), (300, 520, 256)])
@pytest.mark.parametrize("which", ["q", "k", "v", "do"])
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf], ids=["nan", "inf", "minus_inf"])
def test_one_value_at_each_of_eight_positions(cs, kind, dim, ql, kl, first, which, bad):
    """Batch entry b holds the value at token first + b, with two tiles of keys and with five."""
    t = {n: normal(8, 2, ql if n in ("q", "do") else kl, dim, seed=i, kind=kind) for i, n in enumerate(("q", "k", "v", "do"))}
    for b in range(8):
        t[which][b, :, first + b, COLUMN] = bad
    check(passes(cs, **t), definition(**t), t["v"])


@halves
@pytest.mark.parametrize("dim", [64, 128])
def test_a_bad_key_within_its_sequence_and_nan_behind(cs, kind, dim):
    """Shared heads, sequences of every length: the keys behind them are NaN, the last one in front of the end as well, but
    for every other entry."""
    n = 300
    lens = torch.tensor([0, 1, 6, 7, 8, 100, 135, 136, 200, 262, 263, 300], dtype=torch.int32, device="cuda")
    t = dict(q=normal(12, 4, 200, dim, seed=1, kind=kind), do=normal(12, 4, 200, dim, seed=2, kind=kind),
             k=normal(12, 2, n, dim, seed=3, kind=kind), v=normal(12, 2, n, dim, seed=4, kind=kind))
    for b, m in enumerate(lens.tolist()):
        t["k"][b, :, m:], t["v"][b, :, m:] = math.nan, math.nan
        if m and b % 2:
            t["k"][b, :, m - 1, COLUMN] = math.nan
    check(passes(cs, **t, kv_lens=lens), definition(**t, lens=lens), t["v"])


@halves
@pytest.mark.parametrize("dim", [64, 128])
def test_rows_whose_scores_are_all_minus_infinity(cs, kind, dim):
    """Seen keys whose probabilities nobody can tell are not a row that sees nothing."""
    t = {n: normal(1, 1, 140, dim, seed=i, kind=kind) for i, n in enumerate(("q", "k", "v", "do"))}
    t["k"][..., COLUMN], t["q"][..., COLUMN] = -math.inf, 1.0
    t["q"][:, :, 5, COLUMN] = -1.0  # +inf all along
    got = passes(cs, **t)
    assert torch.isnan(got[0]).all() and (got[1][:, :, 6:] == -math.inf).all() and (got[1][:, :, 5] == math.inf).all()
    for g in got[2:]:
        assert torch.isnan(g).all()


@halves
@pytest.mark.parametrize("dim", [64, 128])
def test_a_bad_key_under_a_causal_mask(cs, kind, dim):
    """Every query that sees it shows it; so does every key that such a query sees."""
    for at in (0, 6, 7, 130, 199):
        t = {n: normal(1, 2, 200, dim, seed=i, kind=kind) for i, n in enumerate(("q", "k", "v", "do"))}
        t["k"][:, :, at, COLUMN] = math.nan
        o, lse, dq, dk, dv = passes(cs, **t, causal=True)
        for g in (o, lse, dq, dk, dv):
            assert torch.isnan(g[:, :, at:]).all()
        assert torch.isnan(dk).all() and torch.isnan(dv).all()  # the last query sees all of them
        assert torch.isfinite(lse[:, :, :at]).all()


@halves
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("ql,kl", [(200, 70), (130, 128), (400, 9), (129, 1)])
@pytest.mark.parametrize("bad", [math.nan, math.inf])
def test_queries_that_see_nothing_may_hold_anything(cs, kind, dim, ql, kl, bad):
    """No gradient passes through them: the same bits as with zeros in their place, of q and of the gradient of o."""
    t = {n: normal(2, 4, ql, dim, seed=i, kind=kind) for i, n in enumerate(("q", "do"))}
    t.update({n: normal(2, 2, kl, dim, seed=5 + i, kind=kind) for i, n in enumerate("kv")})
    dead = ql - kl
    zero = {n: x.clone() for n, x in t.items()}
    for n in ("q", "do"):
        zero[n][:, :, :dead], t[n][:, :, :dead] = 0.0, bad
    got, want = passes(cs, **t, causal=True), passes(cs, **zero, causal=True)
    for g, w in zip(got, want):
        assert torch.equal(g, w)
    assert not got[0][:, :, :dead].any() and not got[2][:, :, :dead].any() and (got[1][:, :, :dead] == -math.inf).all()


@halves
def test_gradients_of_an_overflow_are_seen(cs, kind):
    """Through autograd: a step that has diverged shows in the gradient of every operand that it went through."""
    q, k, v = (normal(1, 2, 40, 64, seed=i, kind=kind).requires_grad_(True) for i in range(3))
    with torch.no_grad():
        k[0, 0, 14, 0] = math.inf
        q[..., 0] = 1.0
    grads = torch.autograd.grad(cs.attention(q, k, v).float().sum(), (q, k, v))
    for g in grads:
        assert torch.isnan(g[:, 0]).all() and torch.isfinite(g[:, 1]).all()
