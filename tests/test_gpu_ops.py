"""The training operators against their definitions in 64 bits, at the sizes, masks and layouts where they can go
wrong.  Bounds follow from the roundings that each operator makes (ops_reference.py)."""
import math

import pytest

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

import ops_reference as R  # noqa: E402

KINDS = [torch.float32, torch.float16, torch.bfloat16]
kinds = pytest.mark.parametrize("kind", KINDS, ids=["fp32", "fp16", "bf16"])
halves = pytest.mark.parametrize("kind", KINDS[1:], ids=["fp16", "bf16"])


@pytest.fixture(scope="module")
def cs():
    import cswap_b200
    assert torch.cuda.is_available()
    cswap_b200.lib()
    return cswap_b200


def normal(*shape, seed=0, kind=torch.float32):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn(*shape, generator=gen, device="cuda").to(kind)


def same(a, b):
    """The same bits (NaNs of one pattern included)."""
    view = {4: torch.int32, 2: torch.int16, 1: torch.uint8}[a.element_size()]
    return torch.equal(a.contiguous().view(view), b.contiguous().view(view))


# ---- 8-bit checkpoints ---------------------------------------------------------------------------------------------

def check_q8(cs, x, packed):
    codes, scales, values = R.q8(x)
    n = x.numel()
    at = (n + 15) // 16 * 16
    host = packed.cpu()
    assert torch.equal(host[:n].view(torch.int8).float(), codes.float())
    got = host[at:at + 4 * scales.numel()].view(torch.float32)
    assert torch.equal(torch.nan_to_num(got, nan=-1.0), torch.nan_to_num(scales, nan=-1.0))
    return values


@kinds
@pytest.mark.parametrize("n", [0, 1, 3, 4, 127, 128, 129, 515, 4096, 100003, (1 << 20) - 1, (1 << 20) + 131])
def test_q8_round_trip(cs, kind, n):
    x = normal(n, seed=n, kind=kind)
    packed = cs.q8_compress(x)
    assert packed.numel() == cs.q8_bytes(n)
    values = check_q8(cs, x, packed)
    for out in KINDS:
        back = cs.q8_decompress(packed, n, dtype=out)
        assert back.dtype == out and torch.equal(back.cpu(), values.to(out))


@kinds
def test_q8_awkward_groups(cs, kind):
    """Zeros, one spike, values on the rounding's ties, the smallest and largest numbers, infinities and NaN."""
    x = normal(128 * 10, seed=3).cpu()
    x[128:256] = 0.0
    x[256:384] = 0.0
    x[300] = -7.0
    x[384:512] = torch.arange(128) - 64.0  # m = 64
    x[511] = 127.0                         # scale 1: halves are ties
    x[400:420] = torch.arange(20) + 0.5
    x[512:640] *= 2.0 ** -130
    x[640:768] *= 3e38 if kind == torch.float32 else 6e4
    x[768] = math.inf
    x[900] = math.nan
    x[1030] = -math.inf
    x[1152:1280] *= 2.0 ** -118
    x = x.to(kind).cuda()
    if kind == torch.float16:
        x[640:768] = x[640:768].clamp(-65504, 65504)
    if kind != torch.float32:  # the sixth group holds numbers, whatever the type makes of them
        x[640:768] = torch.nan_to_num(x[640:768], posinf=65504.0, neginf=-65504.0)
    packed = cs.q8_compress(x)
    values = check_q8(cs, x, packed)
    back = cs.q8_decompress(packed, x.numel(), dtype=torch.float32).cpu()
    assert torch.equal(torch.nan_to_num(back, nan=-1.0), torch.nan_to_num(values, nan=-1.0))
    assert torch.isnan(back[768:896]).all() and torch.isnan(back[896:1024]).all() and torch.isnan(back[1024:1152]).all()
    assert torch.isfinite(back[:640]).all() and (kind == torch.float32 or torch.isfinite(back[640:768]).all())


@kinds
def test_q8_and_gelu_of_views_off_their_alignment(cs, kind):
    """A contiguous tensor may begin anywhere in its storage; what lies in front and behind stays."""
    n = 1000
    for shift in (1, 2, 3):
        x = normal(n + 8, seed=shift, kind=kind)[shift:shift + n]
        packed = cs.q8_compress(x)
        values = check_q8(cs, x, packed)
        room = torch.full((n + 8,), 9.0, dtype=kind, device="cuda")
        cs.q8_decompress(packed, n, out=room[shift:shift + n])
        assert torch.equal(room[shift:shift + n].cpu(), values.to(kind))
        assert (room[:shift] == 9).all() and (room[shift + n:] == 9).all()
        y, again = cs.gelu_forward(x)
        assert torch.equal(again[:n], packed[:n])
        y0, _ = cs.gelu_forward(x.clone())
        assert torch.equal(y, y0)
        dy = normal(n + 8, seed=9, kind=kind)[shift:shift + n]
        assert torch.equal(cs.gelu_backward(dy, packed), cs.gelu_backward(dy.clone(), packed))


def test_q8_writes_nothing_behind_its_bytes(cs):
    for n in (1, 5, 130, 4097):
        need = cs.q8_bytes(n)
        room = torch.full((need + 64,), 77, dtype=torch.uint8, device="cuda")
        out = cs.q8_compress(normal(n), out=room)
        assert out.data_ptr() == room.data_ptr() and (room[need:] == 77).all()
        pad = room[n:(n + 15) // 16 * 16]
        assert (pad == 77).all()


def test_q8_refusals(cs):
    x = normal(256)
    packed = cs.q8_compress(x)
    for call in (lambda: cs.q8_compress(x.double()), lambda: cs.q8_compress(x.view(16, 16).t()),
                 lambda: cs.q8_compress(x, out=torch.empty(1000, device="cuda")),
                 lambda: cs.q8_decompress(packed, 256, dtype=torch.float64),
                 lambda: cs.q8_decompress(packed, -1), lambda: cs.q8_decompress(packed.view(torch.int8), 256),
                 lambda: cs.q8_decompress(packed, 256, out=torch.empty(255, device="cuda")),
                 lambda: cs.gelu_backward(x, packed.float()), lambda: cs.gelu_forward(x.long())):
        with pytest.raises(ValueError):
            call()
    for call in (lambda: cs.q8_compress(x, out=packed[:-1]), lambda: cs.q8_decompress(packed[:-1].clone(), 256),
                 lambda: cs.q8_decompress(packed, 1 << 40), lambda: cs.gelu_backward(normal(300), packed),
                 lambda: cs.q8_compress(normal(64), out=torch.empty(500, dtype=torch.uint8, device="cuda")[8:])):
        with pytest.raises(cs.CswapError):
            call()


# ---- GELU ------------------------------------------------------------------------------------------------------------

@kinds
@pytest.mark.parametrize("n", [0, 1, 130, 4099, (1 << 20) + 77])
def test_gelu_passes(cs, kind, n):
    """x Phi(x) to 2^-19 of |x| before it is rounded; the checkpoint as q8_compress writes it; the gradient on it."""
    x = normal(n, seed=n + 1, kind=kind) * 3
    dy = normal(n, seed=n + 2, kind=kind)
    y, packed = cs.gelu_forward(x)
    u, e = R.U[kind], 2.0 ** -19
    tiny = 2.0 ** -24 if kind == torch.float16 else 2.0 ** -133
    wide = x.double()
    want = wide * R.phi(wide)
    R.close(y, want, u * want.abs() + e * wide.abs().clamp(max=8.0) + tiny)
    held = check_q8(cs, x, packed).cuda().double() if n else wide
    dx, again = cs.gelu_backward(dy, packed, recompute=True)
    assert same(dx, cs.gelu_backward(dy, packed))
    slope = R.phi(held) + held * R.density(held)
    g = dy.double()
    R.close(dx, g * slope, u * (g * slope).abs() + e * g.abs() * 4 + tiny)
    R.close(again, held * R.phi(held), u * (held * R.phi(held)).abs() + e * held.abs().clamp(max=8.0) + tiny)


def test_gelu_of_extremes(cs):
    x = torch.zeros(128 * 4, device="cuda")
    x[:6] = torch.tensor([30.0, -30.0, 1e-30, -1e-30, 100.0, -100.0])
    x[128], x[256], x[384] = math.inf, math.nan, 3e38
    y, packed = cs.gelu_forward(x)
    assert y[0] == 30 and y[4] == 100 and abs(float(y[1])) < 1e-20 and abs(float(y[5])) < 1e-20
    assert y[128] == math.inf and math.isnan(float(y[256])) and y[384] == x[384]
    assert float(y[2]) == pytest.approx(5e-31, rel=1e-5)
    dx, again = cs.gelu_backward(torch.ones_like(x), packed, recompute=True)
    assert torch.isfinite(dx[:128]).all() and torch.isnan(dx[128:384]).all() and torch.isfinite(dx[384:]).all()
    assert dx[4] == 1 and dx[5] == 0 and dx[384] == 1 and again[384] == cs.q8_decompress(packed, 512)[384]


@kinds
def test_gelu_gradient_follows_the_held_values(cs, kind):
    x = normal(3, 5, 37, seed=4, kind=kind).requires_grad_(True)
    dy = normal(3, 5, 37, seed=5, kind=kind)
    y = cs.gelu(x)
    saved = sum(t.numel() * t.element_size() for t in y.grad_fn.saved_tensors)
    assert saved == cs.q8_bytes(x.numel())
    dx, = torch.autograd.grad(y, x, dy)
    y0, packed = cs.gelu_forward(x.detach())
    assert same(y, y0) and same(dx, cs.gelu_backward(dy, packed))
    # and by differences: values that are their own checkpoint (codes over a scale of a power of two)
    z = (torch.arange(-64, 64, device="cuda").float() / 32)
    z[0] = -127 / 32
    z.requires_grad_(True)
    g, = torch.autograd.grad(cs.gelu(z).sum(), z)
    h = 2.0 ** -10
    wide = z.detach().double()
    diff = ((wide + h) * R.phi(wide + h) - (wide - h) * R.phi(wide - h)) / (2 * h)
    # the third derivative of x Phi(x) is below 1.2: 1.2 / 6 h^2 of the difference, and 2^-20 of the kernel
    R.close(g, diff, torch.full_like(diff, 0.2 * h * h + 2.0 ** -20))


@pytest.mark.parametrize("bias", [True, False])
def test_gelu_linear(cs, bias):
    """The layer's output is torch's on gelu(x); its gradients are those on the held values, and nothing but the
    checkpoint (and the weight) is kept."""
    x = normal(2, 33, 64, seed=1).requires_grad_(True)
    w = normal(24, 64, seed=2).requires_grad_(True)
    b = normal(24, seed=3).requires_grad_(True) if bias else None
    dy = normal(2, 33, 24, seed=4)
    y = cs.gelu_linear(x, w, b)
    kept = [t for t in y.grad_fn.saved_tensors if t.data_ptr() != w.data_ptr()]
    assert [t.numel() for t in kept] == [cs.q8_bytes(x.numel())]
    got = torch.autograd.grad(y, [t for t in (x, w, b) if t is not None], dy)
    held = R.q8(x)[2].cuda().double().view_as(x)
    a, xd = held * R.phi(held), x.detach().double()
    want_y = xd * R.phi(xd) @ w.detach().double().t() + (b.detach().double() if bias else 0)
    g = dy.double()
    slope = R.phi(held) + held * R.density(held)
    wd = w.detach().double()
    e = 2.0 ** -15  # products of up to 66 terms, in float32, or in torch's own choice of steps for it
    R.close(y, want_y, e * ((xd * R.phi(xd)).abs() @ wd.abs().t() + 1))
    R.close(got[0], g @ wd * slope, e * (g.abs() @ wd.abs() * (slope.abs() + 1)))
    R.close(got[1], g.flatten(0, 1).t() @ a.flatten(0, 1), e * (g.abs().flatten(0, 1).t() @ (a.abs().flatten(0, 1) + 1)))
    if bias:
        R.close(got[2], g.sum((0, 1)), e * g.abs().sum((0, 1)))
    some = torch.autograd.grad(cs.gelu_linear(x.detach(), w, b), w, dy)[0]
    assert torch.allclose(some, got[1], rtol=1e-4, atol=1e-4)


# ---- layer norm --------------------------------------------------------------------------------------------------------

NORM_SHAPES = [(1, 1), (3, 2), (5, 7), (1001, 8), (70000, 8), (999, 13), (3001, 16), (777, 40), (513, 63), (300, 64), (77, 768), (33, 8), (130, 255), (65, 256), (9, 257), (40, 512), (31, 769),
               (7, 1001), (600, 1024), (6, 1025), (5, 2048), (9, 2051), (3, 4096), (5, 4097), (4, 8192), (3, 10000),
               (3, 8191), (5, 8193), (2, 12001), (2, 16380), (3, 16383), (2, 16384), (37, 1022), (3, 16385), (70, 20000), (1300, 40)]


def norm_bounds(x, h, rstd, dy, w, b, kind, param_kind):
    """Sums over c columns in float32 err by c 2^-24 of their terms' magnitudes at most (and far less as they are
    summed, in 32 to 512 strands)."""
    c, rows = x.shape[-1], x.numel() // x.shape[-1]
    e = 2.0 ** -24 * (c / 32 + 40)
    wa = w.abs() if w is not None else torch.ones(c, device=x.device, dtype=torch.float64)
    ba = b.abs() if b is not None else 0.0
    big = (x.abs().mean(-1, keepdim=True) + x.abs()) * rstd[..., None]  # what is subtracted, in units of the norm
    he = e * (big + h.abs() * (1 + big.square().mean(-1, keepdim=True)))
    y = (h.abs() * wa + ba) * (R.U[kind] + 2.0 ** -22) + he * wa
    g = dy.abs() * wa
    gh = (g * (h.abs() + he)).mean(-1, keepdim=True)
    dx0 = rstd[..., None] * (g + g.mean(-1, keepdim=True) + h.abs() * gh)
    dx = (R.U[kind] + 2 * e) * dx0 + rstd[..., None] * (he * gh + (g * he).mean(-1, keepdim=True) * (h.abs() + 1))
    e_rows = 2.0 ** -24 * (rows + 8)
    flat = lambda t: t.reshape(-1, c)
    dw = flat(dy.abs() * he).sum(0) + (e_rows + R.U[param_kind]) * flat(dy.abs() * h.abs()).sum(0)
    db = (e_rows + R.U[param_kind]) * flat(dy.abs()).sum(0)
    tiny = 2.0 ** -24 if torch.float16 in (kind, param_kind) else 2.0 ** -133
    return y + tiny, dx + tiny, dw + tiny, db + tiny, he


@kinds
@pytest.mark.parametrize("rows,cols", NORM_SHAPES)
@pytest.mark.parametrize("summed,wide_params", [(False, False), (True, True)])
def test_layer_norm_passes(cs, kind, rows, cols, summed, wide_params):
    param_kind = torch.float32 if wide_params else kind
    x = (normal(rows, cols, seed=rows) + 0.5).to(kind)
    r = normal(rows, cols, seed=cols, kind=kind) if summed else None
    w = (normal(cols, seed=5) * 0.2 + 1).to(param_kind)
    b = (normal(cols, seed=6) * 0.2).to(param_kind)
    dy = normal(rows, cols, seed=7, kind=kind)
    eps = 1e-5
    y, s, mean, rstd = cs.layer_norm_forward(x, w, b, eps, r)
    if summed:
        assert torch.equal(s, (x.float() + r.float()).to(kind))
    else:
        assert s.data_ptr() == x.data_ptr()
    wide = s.double()
    want, m, d, h = R.layer_norm(wide, w.double(), b.double(), eps)
    dx, dw, db = cs.layer_norm_backward(dy, s, mean, rstd, w)
    yb, dxb, dwb, dbb, he = norm_bounds(wide, h, d, dy.double(), w.double(), b.double(), kind, param_kind)
    R.close(y, want, yb)
    R.close(mean, m, 2.0 ** -24 * (cols / 32 + 40) * wide.abs().mean(-1) + 2.0 ** -140)
    # relative to rstd as he is to h
    R.close(rstd, d, d * (2.0 ** -22 + 2.0 ** -24 * (cols / 32 + 40) * (1 + (wide.abs() * d[:, None]).square().mean(-1) * 4)))
    gx, gw, gb = R.layer_norm_grads(dy.double(), h, d, w.double())
    R.close(dx, gx, dxb)
    R.close(dw, gw, dwb)
    R.close(db, gb, dbb)
    assert dw.dtype == db.dtype == param_kind
    again = cs.layer_norm_backward(dy, s, mean, rstd, w)
    assert same(again[0], dx) and same(again[1], dw) and same(again[2], db)
    only, none_w, none_b = cs.layer_norm_backward(dy, s, mean, rstd, w, sums=False)
    assert same(only, dx) and none_w is None and none_b is None


@kinds
def test_layer_norm_without_parameters(cs, kind):
    x = normal(4, 3, 100, seed=1, kind=kind)
    y, s, mean, rstd = cs.layer_norm_forward(x)
    want, m, d, h = R.layer_norm(x.double(), None, None, 1e-5)
    dy = normal(4, 3, 100, seed=2, kind=kind)
    yb, dxb, *_ = norm_bounds(x.double(), h, d, dy.double(), None, None, kind, kind)
    R.close(y, want, yb)
    assert mean.shape == (12,) and y.shape == x.shape
    dx, dw, db = cs.layer_norm_backward(dy, x, mean, rstd)
    R.close(dx, R.layer_norm_grads(dy.double(), h, d, None)[0], dxb)
    assert dw is None and db is None
    w = torch.ones(100, device="cuda", dtype=kind)
    y1, *_ = cs.layer_norm_forward(x, w)
    assert same(y1, y)


def test_layer_norm_far_from_zero_and_constant_rows(cs):
    """The variance is summed from the centred values: rows about 1000 keep their digits; a constant row gives b."""
    x = normal(8, 768, seed=1) + 1000
    x[3] = 42.0
    w, b = normal(768, seed=2), normal(768, seed=3)
    y, _, mean, rstd = cs.layer_norm_forward(x, w, b)
    want, m, d, h = R.layer_norm(x.double(), w.double(), b.double(), 1e-5)
    assert torch.equal(y[3], b) and float(mean[3]) == 42
    rest = [i for i in range(8) if i != 3]
    # the mean is off by a few steps of 1000 * 2^-24 = 6e-5, which shifts every value of its row alike
    R.close(y[rest], want[rest], (8 * 6e-5 * w.abs().double() + 1e-5).expand(7, 768))


def test_layer_norm_empty_and_refused(cs):
    w = torch.ones(16, device="cuda")
    x = torch.empty(0, 16, device="cuda")
    y, s, mean, rstd = cs.layer_norm_forward(x, w, w)
    dx, dw, db = cs.layer_norm_backward(x, x, mean, rstd, w)
    assert y.shape == (0, 16) and dx.shape == (0, 16) and (dw == 0).all() and (db == 0).all()
    x = normal(4, 16)
    y, s, mean, rstd = cs.layer_norm_forward(x, w, w)
    for call in (lambda: cs.layer_norm_forward(x.t()), lambda: cs.layer_norm_forward(x.double()),
                 lambda: cs.layer_norm_forward(x, None, w), lambda: cs.layer_norm_forward(x, w[:8]),
                 lambda: cs.layer_norm_forward(x, w.half(), w.half()), lambda: cs.layer_norm_forward(x, w, w.half()),
                 lambda: cs.layer_norm_forward(x, w, w, -1.0), lambda: cs.layer_norm_forward(x, w, w, 1e-5, x[:2]),
                 lambda: cs.layer_norm_forward(x, w, w, 1e-5, x.half()), lambda: cs.layer_norm_forward(torch.zeros((), device="cuda")),
                 lambda: cs.layer_norm_forward(torch.empty(3, 0, device="cuda")),
                 lambda: cs.layer_norm_backward(x.half(), x, mean, rstd, w),
                 lambda: cs.layer_norm_backward(x, x, mean[:2], rstd, w),
                 lambda: cs.layer_norm_backward(x, x, mean, rstd.half(), w)):
        with pytest.raises(ValueError):
            call()


def test_layer_norm_through_autograd(cs):
    x, r = (normal(6, 10, 96, seed=i).requires_grad_(True) for i in (1, 2))
    w, b = (normal(96, seed=i).requires_grad_(True) for i in (3, 4))
    dy = normal(6, 10, 96, seed=5)
    y = cs.layer_norm(x, w, b, 1e-5, residual=r)
    got = torch.autograd.grad(y, [x, r, w, b], dy)
    leaves = [t.detach().double().requires_grad_(True) for t in (x, r, w, b)]
    want = torch.autograd.grad(torch.nn.functional.layer_norm(leaves[0] + leaves[1], (96,), leaves[2], leaves[3]), leaves,
                               dy.double())
    for g, t in zip(got, want):
        R.close(g, t, 2.0 ** -17 * (t.abs() + t.abs().mean() * 4 + 1))
    # a gradient by differences, along one direction, of the same 64-bit function
    v = normal(6, 10, 96, seed=6).double()
    f = lambda t: (torch.nn.functional.layer_norm(leaves[0].detach() + t * v + leaves[1].detach(), (96,),
                                                  leaves[2].detach(), leaves[3].detach()) * dy.double()).sum()
    diff = float((f(1e-5) - f(-1e-5)) / 2e-5)
    assert float((got[0].double() * v).sum()) == pytest.approx(diff, rel=1e-4, abs=1e-3)
    # the same tensor as both terms; a transposed one; an expanded gradient
    z = normal(8, 32, seed=7).requires_grad_(True)
    g, = torch.autograd.grad(cs.layer_norm(z, residual=z).sum(0)[3], z)
    zd = z.detach().double().requires_grad_(True)
    t, = torch.autograd.grad(torch.nn.functional.layer_norm(2 * zd, (32,)).sum(0)[3], zd)
    R.close(g, t, 2.0 ** -18 * (t.abs() + 4))
    g, = torch.autograd.grad(cs.layer_norm(z.t()).mean(), z)
    assert g.shape == z.shape and float(g.abs().max()) < 1e-6


# ---- attention -----------------------------------------------------------------------------------------------------------

def operands(kind, b, h, hk, ql, kl, d, seed=0, tokens_first=True):
    def one(heads, n, i):
        if tokens_first:
            return normal(b, n, heads, d, seed=seed + i, kind=kind).transpose(1, 2)
        return normal(b, heads, n, d, seed=seed + i, kind=kind)
    return one(h, ql, 1), one(hk, kl, 2), one(hk, kl, 3), one(h, ql, 4)


def check_attention(cs, q, k, v, do, causal=False, lens=None, scale=None):
    want = R.Attention(q, k, v, do, causal, lens, scale if scale is not None else q.shape[3] ** -0.5)
    o, lse = cs.attention_forward(q, k, v, causal, lens, scale)
    R.close(o, want.o, want.o_bound)
    R.close(lse, want.lse, want.lse_bound)
    assert lse.dtype == torch.float32 and o.dtype == q.dtype
    dq, dk, dv = cs.attention_backward(do, q, k, v, o, lse, causal, lens, scale)
    R.close(dq, want.dq, want.dq_bound)
    R.close(dk, want.dk, want.dk_bound)
    R.close(dv, want.dv, want.dv_bound)
    again = cs.attention_backward(do, q, k, v, o, lse, causal, lens, scale)
    assert same(again[0], dq) and same(again[1], dk) and same(again[2], dv)
    return o, lse, dq, dk, dv


LENGTHS = [(1, 1), (1, 300), (5, 3), (64, 64), (63, 129), (128, 128), (129, 127), (200, 333), (512, 512), (257, 640),
           (700, 65)]


@halves
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("ql,kl", LENGTHS)
def test_attention_lengths(cs, kind, dim, causal, ql, kl):
    check_attention(cs, *operands(kind, 2, 2, 2, ql, kl, dim, seed=ql + kl), causal=causal)


@halves
@pytest.mark.parametrize("dim", [8, 16, 24, 40, 72, 80, 96, 104, 120])
def test_attention_dims(cs, kind, dim):
    check_attention(cs, *operands(kind, 1, 3, 1, 150, 170, dim, seed=dim), causal=True)


@halves
@pytest.mark.parametrize("heads,kv_heads", [(1, 1), (6, 2), (8, 1), (5, 5), (12, 3)])
@pytest.mark.parametrize("tokens_first", [True, False])
def test_attention_shared_heads(cs, kind, heads, kv_heads, tokens_first):
    check_attention(cs, *operands(kind, 2, heads, kv_heads, 100, 140, 64, seed=heads, tokens_first=tokens_first))


@halves
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("dim", [64, 128])
def test_attention_padded_batch(cs, kind, causal, dim):
    """Lengths of zero, one, inside a tile, at its end, all, and out of range; what lies behind them is NaN or
    infinite and counts for nothing."""
    lens = torch.tensor([0, 1, 127, 128, 129, 300, 1000, -5], dtype=torch.int32, device="cuda")
    q, k, v, do = operands(kind, 8, 2, 1, 260, 300, dim, seed=8)
    taken = lens.clamp(0, 300)
    for i in range(8):
        n = int(taken[i])
        k[i, :, n:] = math.nan
        v[i, :, n:] = math.inf
        if n < 300:
            v[i, :, -1] = math.nan
    o, lse, dq, dk, dv = check_attention(cs, q, k, v, do, causal=causal, lens=taken)
    raw = cs.attention_forward(q, k, v, causal, lens)
    assert same(raw[0], o) and same(raw[1], lse)
    assert (o[0] == 0).all() and (lse[0] == -math.inf).all() and (dq[0] == 0).all()
    for i in range(8):
        n = int(taken[i])
        assert (dk[i, :, n:] == 0).all() and (dv[i, :, n:] == 0).all()


@halves
@pytest.mark.parametrize("dim,causal", [(64, False), (64, True), (128, True)])
def test_attention_many_pieces(cs, kind, dim, causal):
    """More tiles of heads than a device runs at once, some without any key, others with one tile or two: a CTA goes
    through a dozen, and none of them waits for another."""
    lens = torch.randint(0, 261, (70,), generator=torch.Generator().manual_seed(dim), dtype=torch.int32)
    lens[::3] = 0
    lens[1::5] = 128
    q, k, v, do = operands(kind, 70, 16, 4, 130, 260, dim, seed=30)
    check_attention(cs, q, k, v, do, causal=causal, lens=lens.cuda())
    assert cs.lib().csw_device_status(torch.cuda.current_stream().cuda_stream) == 0


@halves
@pytest.mark.parametrize("heads,kv_heads,ql,kl,dim,causal", [(4, 1, 700, 700, 80, True), (8, 1, 1000, 70, 64, False),
                                                             (2, 2, 1500, 300, 40, True), (6, 1, 300, 900, 128, True)])
def test_attention_few_keys_and_many_queries(cs, kind, heads, kv_heads, ql, kl, dim, causal):
    """Where there are few tiles of keys their queries are split, and the parts' sums added up."""
    lens = torch.tensor([kl - kl // 3], dtype=torch.int32, device="cuda")
    ops = operands(kind, 1, heads, kv_heads, ql, kl, dim, seed=ql)
    check_attention(cs, *ops, causal=causal)
    check_attention(cs, *ops, causal=causal, lens=lens)


@halves
def test_attention_rows_that_see_nothing(cs, kind):
    """Causal with more queries than keys: the first rows see no key."""
    q, k, v, do = operands(kind, 1, 2, 2, 300, 20, 64, seed=2)
    o, lse, dq, dk, dv = check_attention(cs, q, k, v, do, causal=True)
    assert (o[:, :, :280] == 0).all() and (lse[:, :, :280] == -math.inf).all() and (dq[:, :, :280] == 0).all()
    assert (lse[:, :, 280:] > -math.inf).all()


@halves
@pytest.mark.parametrize("ql,kl", [(0, 5), (5, 0), (0, 0)])
def test_attention_empty(cs, kind, ql, kl):
    q, k, v, do = operands(kind, 2, 4, 2, ql, kl, 32)
    o, lse = cs.attention_forward(q, k, v)
    assert o.shape == q.shape and (o == 0).all() and (lse == -math.inf).all()
    dq, dk, dv = cs.attention_backward(do, q, k, v, o, lse)
    assert (dq == 0).all() and (dk == 0).all() and (dv == 0).all() and dk.shape == k.shape
    e = cs.attention_forward(q[:0], k[:0], v[:0])[0]
    assert e.shape == (0, 4, ql, 32)


@halves
@pytest.mark.parametrize("scale", [0.0, 1.0, -0.3, 0.02])
def test_attention_scales(cs, kind, scale):
    check_attention(cs, *operands(kind, 1, 2, 2, 130, 150, 64, seed=11), scale=scale)


@halves
def test_attention_large_scores(cs, kind):
    """Scores of some thousands: each row is all but one key, and the running maximum moves a long way."""
    q, k, v, do = operands(kind, 1, 2, 2, 140, 400, 64, seed=12)
    ramp = torch.linspace(-1, 1, 400, device="cuda")[None, None, :, None].to(kind)
    check_attention(cs, q.abs() * 4, (k * 0.1 + ramp * 3).to(kind), v, do, scale=1.0)


@halves
def test_attention_layouts(cs, kind):
    """Slices of one projection, heads in front, odd strides, a view off its alignment, an expanded tensor, a
    transposed head: the same results as of plain copies."""
    b, n, h, d = 2, 90, 3, 40
    packed = normal(b, n, 3, h, d, seed=1, kind=kind)
    q, k, v = (packed[:, :, i].transpose(1, 2) for i in range(3))
    do = normal(b, h, n, d, seed=2, kind=kind)
    plain = [t.contiguous() for t in (q, k, v)]
    o, lse = cs.attention_forward(*plain, causal=True)
    grads = cs.attention_backward(do, *plain, o, lse, causal=True)

    def check(q, k, v, do):
        got, l = cs.attention_forward(q, k, v, causal=True)
        assert torch.equal(got, o) and torch.equal(l, lse)
        for a, g in zip(cs.attention_backward(do, q, k, v, got, l, causal=True), grads):
            assert torch.equal(a, g)

    check(q, k, v, do)
    off = torch.empty(b * h * n * d + 1, dtype=kind, device="cuda")[1:].view(b, h, n, d)
    off.copy_(plain[0])
    check(off, k, v, do)
    wide = torch.zeros(b, h, n, d + 3, dtype=kind, device="cuda")
    wide[..., :d] = plain[1]
    check(q, wide[..., :d], v, do)
    turned = plain[2].transpose(2, 3).contiguous().transpose(2, 3)
    check(q, k, turned, do.transpose(1, 2).contiguous().transpose(1, 2))
    one = normal(1, 1, n, d, seed=3, kind=kind)
    e = one.expand(b, h, n, d)
    for a, g in zip(cs.attention_forward(q, e, e), cs.attention_forward(q, e.contiguous(), e.contiguous())):
        assert torch.equal(a, g)
    assert torch.equal(cs.attention_backward(torch.ones_like(o[..., :1]).expand_as(o), *plain, o, lse, causal=True)[0],
                       cs.attention_backward(torch.ones_like(o), *plain, o, lse, causal=True)[0])


@halves
def test_attention_through_autograd(cs, kind):
    q, k, v, do = (t.detach() for t in operands(kind, 1, 4, 2, 60, 70, 32, seed=21))
    leaves = [t.requires_grad_(True) for t in (q, k, v)]
    o = cs.attention(*leaves, causal=True)
    got = torch.autograd.grad(o, leaves, do)
    want = R.Attention(q, k, v, do, True, None, 32 ** -0.5)
    for g, w, b in zip(got, (want.dq, want.dk, want.dv), (want.dq_bound, want.dk_bound, want.dv_bound)):
        R.close(g, w, b)
    # the formula's gradient is the function's: by differences, in 64 bits, along one direction of each operand
    for i, name in enumerate(("dq", "dk", "dv")):
        step = torch.randn(leaves[i].shape, device="cuda", dtype=torch.float64,
                           generator=torch.Generator(device="cuda").manual_seed(i))
        f = []
        for t in (1e-4, -1e-4):
            args = [a.detach().double() for a in leaves]
            args[i] = args[i] + t * step
            K, V = (a.repeat_interleave(2, 1) for a in args[1:])
            s = (args[0] @ K.transpose(2, 3) * 32 ** -0.5).masked_fill(~R.seen(60, 70, True, None, "cuda"), -math.inf)
            f.append((torch.softmax(s, 3) @ V * do.double()).sum())
        diff = float((f[0] - f[1]) / 2e-4)
        assert float((getattr(want, name) * step).sum()) == pytest.approx(diff, rel=1e-5, abs=1e-5)


def test_attention_refusals(cs):
    q, k, v, do = operands(torch.float16, 2, 4, 2, 10, 12, 32)
    lens = torch.tensor([3, 4], dtype=torch.int32, device="cuda")
    o, lse = cs.attention_forward(q, k, v)
    for call in (lambda: cs.attention(q.float(), k.float(), v.float()), lambda: cs.attention(q, k.bfloat16(), v),
                 lambda: cs.attention(q[0], k[0], v[0]), lambda: cs.attention(q, k, v[:, :, :5]),
                 lambda: cs.attention(q[:1], k, v), lambda: cs.attention(q[..., :24], k, v),
                 lambda: cs.attention(q[..., :12], k[..., :12], v[..., :12]), lambda: cs.attention(q[:, :3], k, v),
                 lambda: cs.attention(q[:, :0], k, v), lambda: cs.attention(q, k, v, kv_lens=lens.long()),
                 lambda: cs.attention(q, k, v, kv_lens=lens[:1]), lambda: cs.attention(q, k, v, kv_lens=lens.cpu()),
                 lambda: cs.attention(q, k, v, scale=math.nan), lambda: cs.attention(q, k, v, scale=math.inf),
                 lambda: cs.attention(*(torch.zeros(1, 1, 4, 136, device="cuda", dtype=torch.half),) * 3),
                 lambda: cs.attention_backward(do, q, k, v, o, lse[:1]),
                 lambda: cs.attention_backward(do.float(), q, k, v, o, lse),
                 lambda: cs.attention_backward(do, q, k, v, o[:, :2], lse)):
        with pytest.raises(ValueError):
            call()


# ---- offsets beyond 32 bits ------------------------------------------------------------------------------------------------

def test_offsets_beyond_32_bits(cs):
    """More than 2^31 values, or as many bytes between two entries: the last ones are as right as the first."""
    n = (1 << 31) + 1000
    x = torch.zeros(n, dtype=torch.bfloat16, device="cuda")
    for at in (0, n - 5000):
        x[at:at + 5000] = normal(5000, seed=at % 7, kind=torch.bfloat16)
    y, packed = cs.gelu_forward(x)
    assert torch.equal(packed[:n], cs.q8_compress(x)[:n])
    dx, again = cs.gelu_backward(y, packed, recompute=True)
    start = (n - 5000 + 127) // 128 * 128  # a tail that begins with a group stands for itself
    tail = x[start:].clone()
    y1, p1 = cs.gelu_forward(tail)
    d1, a1 = cs.gelu_backward(y1, p1, recompute=True)
    assert torch.equal(y[start:], y1) and torch.equal(packed[start:n], p1[:n - start])
    assert torch.equal(dx[start:], d1) and torch.equal(again[start:], a1)
    assert torch.equal(cs.q8_decompress(packed, n, dtype=torch.bfloat16)[start:],
                       cs.q8_decompress(p1, n - start, dtype=torch.bfloat16))
    del packed, dx, again
    rows = n // 1000
    x2 = x[:rows * 1000].view(rows, 1000)
    x2[-7:] = normal(7, 1000, seed=5, kind=torch.bfloat16)
    z, _, mean, rstd = cs.layer_norm_forward(x2)
    z1, _, m1, r1 = cs.layer_norm_forward(x2[-7:].clone())
    assert torch.equal(z[-7:], z1) and torch.equal(mean[-7:], m1) and torch.equal(rstd[-7:], r1)
    g, _, _ = cs.layer_norm_backward(x2, x2, mean, rstd)
    assert torch.equal(g[-7:], cs.layer_norm_backward(x2[-7:].clone(), x2[-7:].clone(), m1, r1)[0])
    del z, g, y
    far = (1 << 31) - 8192  # between two batch entries: more than 2^32 bytes
    t = normal(2, 2, 100, 32, seed=3, kind=torch.bfloat16)
    apart = torch.as_strided(x, (2, 2, 100, 32), (far, 3200, 32, 1))
    apart.copy_(t)
    want, got = cs.attention_forward(t, t, t), cs.attention_forward(apart, apart, apart)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    for a, b in zip(cs.attention_backward(apart, apart, apart, apart, *got), cs.attention_backward(t, t, t, t, *want)):
        assert torch.equal(a, b)
