"""How near the operators come, beside the worst cases of test_gpu_ops.py: the norm of the error over a whole result, where
the roundings of many values average out."""
import math

import pytest

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

import ops_reference as R  # noqa: E402


def normal(*shape, seed=0, kind=torch.float32):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn(*shape, generator=gen, device="cuda").to(kind)


@pytest.mark.parametrize("kind,bound", [(torch.bfloat16, 0.003), (torch.float16, 0.0004)], ids=["bf16", "fp16"])
@pytest.mark.parametrize("dim", [40, 64, 128])
@pytest.mark.parametrize("b,h,hk,ql,kl,causal", [(4, 4, 4, 200, 200, False), (2, 8, 2, 500, 700, True),
                                                 (1, 4, 4, 1100, 1100, True), (2, 2, 2, 130, 2000, False)])
def test_attention_error_in_the_norm(kind, bound, dim, b, h, hk, ql, kl, causal):
    """A rounding to u = 2^-8 or 2^-11 is off by u / m at most, m the mantissa in 1 ... 2: with m spread as 1 / m, by
    u sqrt(3 / (8 ln 2)) / sqrt(3) = 0.425 u at the mean.  A result carries its own and, over independent values, as much
    from the rounded probabilities or score gradients of its product: 0.6 u = 0.0023 and 0.0003, of which the bounds leave
    a quarter to spare for small probabilities in float16 and for what float32 sums leave."""
    import cswap_b200 as cs
    q, do = normal(b, h, ql, dim, seed=1, kind=kind), normal(b, h, ql, dim, seed=2, kind=kind)
    k, v = normal(b, hk, kl, dim, seed=3, kind=kind), normal(b, hk, kl, dim, seed=4, kind=kind)
    o, lse = cs.attention_forward(q, k, v, causal=causal)
    want = R.Attention(q, k, v, do, causal, None, dim ** -0.5)
    assert float((lse.double() - want.lse).abs().max()) < 1e-4
    for name, got in zip(("o", "dq", "dk", "dv"), (o,) + cs.attention_backward(do, q, k, v, o, lse, causal=causal)):
        w = getattr(want, name)
        assert float((got.double() - w).norm() / w.norm()) < bound, name


def test_gelu_in_float32_is_near_the_function():
    """Phi is off by 6e-9 (the fit) and by the rounding of its factors: 2^-23 for the reciprocal and 2^-24 for what it is
    taken of, as much again for the exponential and for its argument (whose rounding, 2^-23 of x^2 / 2, is largest against
    exp(-x^2 / 2) at x^2 = 2), and 2^-24 of at most a half for each of seven steps: 2^-21 covers them, of |x| for x Phi(x)."""
    import cswap_b200 as cs
    x = torch.cat([normal(1 << 20, seed=5) * 2, torch.linspace(-12, 12, 100001, device="cuda")])
    y, packed = cs.gelu_forward(x)
    wide = x.double()
    off = (y.double() - wide * R.phi(wide)).abs()
    assert bool((off <= 2.0 ** -21 * wide.abs() + 2.0 ** -24 * y.double().abs()).all())
    held = cs.q8_decompress(packed, x.numel()).double()
    dy = normal(x.numel(), seed=6)
    slope = R.phi(held) + held * R.density(held)
    off = (cs.gelu_backward(dy, packed).double() - dy.double() * slope).abs()
    # the slope's second term is the bell, with its 2^-22, times |x| / sqrt(2 pi), of 0.25 at most
    assert bool((off <= (2.0 ** -21 + 2.0 ** -23) * dy.double().abs()).all())
    assert math.isfinite(float(off.max()))
