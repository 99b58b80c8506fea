"""Matrices in 8-bit floating point, their products and the linear layer on them, against their definitions."""
import math

import pytest

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

import step_reference as R  # noqa: E402

KINDS = [torch.float32, torch.float16, torch.bfloat16]
kinds = pytest.mark.parametrize("kind", KINDS, ids=["fp32", "fp16", "bf16"])


@pytest.fixture(scope="module")
def cs():
    import cswap_b200
    assert torch.cuda.is_available()
    cswap_b200.lib()
    return cswap_b200


def normal(*shape, seed=0, kind=torch.float32):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn(*shape, generator=gen, device="cuda").to(kind)


def check_codes(x, codes, scales):
    want, powers, held = R.fp8(x)
    assert codes.dtype == torch.float8_e4m3fn and scales.dtype == torch.float8_e8m0fnu
    assert tuple(codes.shape) == tuple(x.shape) and tuple(scales.shape) == powers.shape
    assert torch.equal(scales.view(torch.uint8).cpu(), torch.from_numpy(powers))
    got = codes.contiguous().view(torch.uint8).cpu()
    nan = torch.isnan(held)
    assert torch.equal(got[~nan], torch.from_numpy(want)[~nan]) and ((got[nan] & 127) == 127).all()
    return held


# ---- quantizing ----------------------------------------------------------------------------------------------------

@kinds
@pytest.mark.parametrize("rows,cols", [(1, 1), (1, 128), (3, 7), (77, 768), (128, 128), (129, 16), (130, 127), (257, 40),
                                       (2, 5000), (1000, 129)])
def test_quantize_and_back(cs, kind, rows, cols):
    x = (normal(rows, cols, seed=rows) * torch.exp(3 * normal(cols, seed=cols))).to(kind)
    codes, scales = cs.fp8_quantize(x)
    held = check_codes(x, codes, scales)
    for to in KINDS:
        back = cs.fp8_dequantize(codes, scales, dtype=to)
        assert back.dtype == to and torch.equal(back.cpu(), held.to(to))


@kinds
def test_quantize_awkward_blocks(cs, kind):
    """Zeros, a spike, ties of every exponent, values on the border of a scale, the smallest and largest numbers, NaN and
    infinities."""
    x = normal(256, 128 * 6, seed=1)
    x[:128, :128] = 0.0
    x[:128, 128:256] = 0.0
    x[5, 200] = -3.0
    ties = torch.from_numpy((R.e4m3_values()[:126] + R.e4m3_values()[1:127]) / 2).float().cuda()
    x[:128, 256:384] = ties.repeat(2)[:128]
    x[0, 256] = 448.0
    x[:128, 384:512] *= 2.0 ** -130  # below the least scale; 0 in 16 bits
    x[:128, 512:640] = x[:128, 512:640].sign() * torch.finfo(kind).max
    x[7, 640], x[8, 641], x[9, 642] = math.nan, math.inf, -math.inf
    for j in range(6):  # the largest at, just above and just below 1.75 2^j
        x[128:, 128 * j:128 * j + 128] = x[128:, 128 * j:128 * j + 128].clamp(-1, 1)
        x[128, 128 * j] = 1.75 * 2.0 ** j * (1 + (j % 3 - 1) * 2.0 ** -7)
    x[200, 5] = -0.0
    x = x.to(kind)
    codes, scales = cs.fp8_quantize(x)
    held = check_codes(x, codes, scales)
    assert torch.isnan(held).sum() == 3
    for to in KINDS:
        back = cs.fp8_dequantize(codes, scales, dtype=to).cpu()
        assert R.bits_equal(torch.nan_to_num(back, nan=-1.0), torch.nan_to_num(held.to(to), nan=-1.0))


def test_every_code_and_scale(cs):
    """All 256 codes under all 256 scales, as torch converts both types."""
    codes = torch.arange(256, dtype=torch.uint8, device="cuda").view(2, 128).repeat(128 * 128, 1)[:128 * 256].contiguous()
    scales = torch.arange(256, dtype=torch.uint8, device="cuda").view(256, 1)
    c, s = codes.view(torch.float8_e4m3fn), scales.view(torch.float8_e8m0fnu)
    got = cs.fp8_dequantize(c, s)
    want = (c.double() * s.double().repeat_interleave(128, 0)).float()
    assert torch.equal(torch.isnan(got), torch.isnan(want)) and torch.equal(torch.nan_to_num(got), torch.nan_to_num(want))


@kinds
def test_quantize_of_rows_apart_and_off_their_alignment(cs, kind):
    whole = normal(140, 300, seed=2, kind=kind)
    for view in (whole[:, :137], whole[3:, 1:200], whole[:, 160:], whole[:1, 5:21]):
        codes, scales = cs.fp8_quantize(view)
        again, powers = cs.fp8_quantize(view.contiguous())
        assert torch.equal(codes.contiguous().view(torch.uint8), again.contiguous().view(torch.uint8))
        assert torch.equal(scales.view(torch.uint8), powers.view(torch.uint8))
        assert codes.data_ptr() % 16 == 0 and (codes.shape[0] == 1 or codes.stride(0) % 16 == 0)
    flat = normal(1001, seed=3, kind=kind)[1:].view(10, 100)
    check_codes(flat, *cs.fp8_quantize(flat))
    deep = normal(3, 5, 64, seed=4, kind=kind)
    codes, scales = cs.fp8_quantize(deep)
    assert tuple(codes.shape) == (15, 64)
    check_codes(deep.view(15, 64), codes, scales)


@kinds
@pytest.mark.parametrize("rows,cols", [(1, 5), (128, 40), (300, 257), (5000, 33)])
def test_column_sums(cs, kind, rows, cols):
    """A column's sum goes through rows / 8 + 24 additions in float32 at most, in an order that does not change."""
    x = normal(rows, cols, seed=rows + cols, kind=kind)
    codes, scales, sums = cs.fp8_quantize(x, sums=True)
    check_codes(x, codes, scales)
    wide = x.double()
    assert sums.dtype == torch.float32
    R.close(sums, wide.sum(0), wide.abs().sum(0) * ((rows / 8 + 24) * 2.0 ** -24))
    assert R.bits_equal(sums, cs.fp8_quantize(x, sums=True)[2])


def test_empty_matrices(cs):
    for shape in ((0, 5), (5, 0), (0, 0)):
        x = torch.empty(shape, device="cuda")
        codes, scales, sums = cs.fp8_quantize(x, sums=True)
        assert tuple(codes.shape) == shape and sums.shape == (shape[1],) and (sums == 0).all()
        assert cs.fp8_dequantize(codes, scales).shape == shape
    q = lambda *shape: cs.fp8_quantize(normal(*shape))
    bias = normal(7)
    for ta, tb in ((False, False), (True, True)):
        a, b = (q(0, 5), q(7, 0)) if ta else (q(5, 0), q(0, 7))
        got = cs.fp8_matmul(*a, *b, transpose_a=ta, transpose_b=tb, bias=bias, dtype=torch.float32)
        assert torch.equal(got, bias.expand(5, 7))
    assert cs.fp8_matmul(*q(0, 5), *q(5, 3)).shape == (0, 3) and cs.fp8_matmul(*q(4, 5), *q(5, 0)).shape == (4, 0)


# ---- products ------------------------------------------------------------------------------------------------------

def operands(cs, m, n, k, ta, tb, seed=0):
    """Matrices whose blocks differ in scale, as codes, and what they hold."""
    def one(rows, cols, s):
        x = normal(rows, cols, seed=s)
        x = x * torch.exp2(torch.randint(-6, 7, (-(-rows // 128), -(-cols // 128)), device="cuda",
                                         generator=torch.Generator(device="cuda").manual_seed(s)).float()
                           ).repeat_interleave(128, 0).repeat_interleave(128, 1)[:rows, :cols]
        q = cs.fp8_quantize(x)
        return q, R.held_of(*q)
    a, A = one(*((k, m) if ta else (m, k)), seed + 1)
    b, B = one(*((n, k) if tb else (k, n)), seed + 2)
    return a, b, A.t() if ta else A, B.t() if tb else B


SHAPES = [(1, 1, 1), (1, 300, 200), (300, 1, 130), (17, 40, 515), (64, 520, 129), (65, 64, 128), (128, 128, 128), (130, 257, 384),
          (256, 512, 96), (333, 515, 1001), (1000, 96, 2048), (257, 1030, 40), (32, 4096, 4096), (96, 96, 9000)]


@pytest.mark.parametrize("ta,tb", [(False, True), (False, False), (True, False), (True, True)],
                         ids=["nt", "nn", "tn", "tt"])
@pytest.mark.parametrize("m,n,k", SHAPES)
def test_products(cs, m, n, k, ta, tb):
    """Every direction and type, with and without a bias; few and many tiles, rows and columns that end inside one, parts of
    the reduction that are joined."""
    a, b, A, B = operands(cs, m, n, k, ta, tb)
    for kind in KINDS:
        for bias in (None, normal(n, seed=9, kind=kind)):
            got = cs.fp8_matmul(*a, *b, transpose_a=ta, transpose_b=tb, bias=bias, dtype=kind)
            want, bound = R.product(A, B, bias, kind)
            assert got.dtype == kind and got.shape == (m, n)
            if kind == torch.float16:  # what half precision cannot hold
                bound = bound.masked_fill(want.abs() > 65000, math.inf)
                got, want = got.clamp(-65504, 65504), want.clamp(-65504, 65504)
            R.close(got, want, bound)
            assert R.bits_equal(got, cs.fp8_matmul(*a, *b, transpose_a=ta, transpose_b=tb, bias=bias, dtype=kind
                                                   ).clamp(-65504, 65504) if kind == torch.float16 else
                                cs.fp8_matmul(*a, *b, transpose_a=ta, transpose_b=tb, bias=bias, dtype=kind))


def test_product_with_a_bias_of_another_type(cs):
    a, b, A, B = operands(cs, 70, 33, 60, False, True)
    for kind in KINDS:
        bias = normal(33, seed=5, kind=kind)
        want, bound = R.product(A, B, bias, torch.bfloat16)
        R.close(cs.fp8_matmul(*a, *b, transpose_b=True, bias=bias), want, bound)


@pytest.mark.parametrize("m,n,k", [(200, 300, 260), (5, 700, 2000)])
def test_numbers_that_are_not_show_where_they_go_in(cs, m, n, k):
    x, w = normal(m, k, seed=1), normal(n, k, seed=2)
    x[3, 150], x[4, 5], w[130, 200] = math.nan, math.inf, -math.inf
    y = cs.fp8_matmul(*cs.fp8_quantize(x), *cs.fp8_quantize(w), transpose_b=True, dtype=torch.float32)
    want = torch.zeros(m, n, dtype=torch.bool, device="cuda")
    want[3], want[4], want[:, 130] = True, True, True
    assert torch.equal(torch.isnan(y), want) and torch.isfinite(y[~want]).all()


def test_scales_at_both_ends(cs):
    """The least and the greatest scales: products of 2^-252 vanish, of 2^-6 and 2^16 do not."""
    tiny, huge = normal(64, 128, seed=1) * 2.0 ** -124, normal(64, 128, seed=2) * 2.0 ** 118
    one = normal(32, 128, seed=3)
    for x in (tiny, huge):
        q, o = cs.fp8_quantize(x), cs.fp8_quantize(one)
        want, bound = R.product(R.held_of(*q), R.held_of(*o).t(), None, torch.float32)
        R.close(cs.fp8_matmul(*q, *o, transpose_b=True, dtype=torch.float32), want, bound + 2.0 ** -140)
    q, h = cs.fp8_quantize(tiny), cs.fp8_quantize(huge)
    want, bound = R.product(R.held_of(*q), R.held_of(*h).t(), None, torch.float32)
    R.close(cs.fp8_matmul(*q, *h, transpose_b=True, dtype=torch.float32), want, bound)
    assert (cs.fp8_matmul(*q, *q, transpose_b=True, dtype=torch.float32) == 0).all()


def test_codes_of_a_program_that_pads_its_rows_otherwise(cs):
    """Codes with more room behind their rows than quantizing leaves; what lies there is not used."""
    x, w = normal(40, 50, seed=1), normal(30, 50, seed=2)
    codes, scales = cs.fp8_quantize(x)
    room = torch.full((40, 160), 0x7f, dtype=torch.uint8, device="cuda")  # NaN
    room[:, :50] = codes.contiguous().view(torch.uint8)
    wide = room.view(torch.float8_e4m3fn)[:, :50]
    q = cs.fp8_quantize(w)
    for t in (True, False):
        b = q if t else cs.fp8_quantize(w.t().contiguous())
        assert R.bits_equal(cs.fp8_matmul(wide, scales, *b, transpose_b=t), cs.fp8_matmul(codes, scales, *b, transpose_b=t))
    assert R.bits_equal(cs.fp8_dequantize(wide, scales), cs.fp8_dequantize(codes, scales))


# ---- the layer -----------------------------------------------------------------------------------------------------

def keeping(f):
    """What f() returns, and the tensors that autograd keeps for it."""
    kept = []
    with torch.autograd.graph.saved_tensors_hooks(lambda t: kept.append(t) or t, lambda t: t):
        y = f()
    return y, kept


@kinds
@pytest.mark.parametrize("bias", [True, False])
@pytest.mark.parametrize("shape,out", [((3, 33, 64), 40), ((300, 130), 257), ((1, 1000), 200)])
def test_linear_and_its_gradients(cs, kind, bias, shape, out):
    """Each result is the product of the quantized operands; nothing but codes is kept."""
    x, w = normal(*shape, seed=1, kind=kind).requires_grad_(True), normal(out, shape[-1], seed=2, kind=kind).requires_grad_(True)
    b = normal(out, seed=3, kind=kind).requires_grad_(True) if bias else None
    dy = normal(*shape[:-1], out, seed=4, kind=kind)
    y, kept = keeping(lambda: cs.fp8_linear(x, w, b))
    kept = sum(t.numel() * t.element_size() for t in kept)
    blocks = lambda r, c: -(-r // 128) * -(-c // 128)
    rows, cols = x.numel() // shape[-1], shape[-1]
    assert kept == rows * cols + out * cols + blocks(rows, cols) + blocks(out, cols)
    grads = torch.autograd.grad(y, [x, w] + ([b] if bias else []), dy)
    X, W, G = (R.held_of(*cs.fp8_quantize(t.detach())) for t in (x, w, dy))
    for got, want, bound in ((y, *R.product(X, W.t(), b.detach() if bias else None, kind)),
                             (grads[0], *R.product(G, W, None, kind)), (grads[1], *R.product(G.t(), X, None, kind))):
        assert got.dtype == kind
        R.close(got.detach().reshape(want.shape), want, bound)
    assert grads[0].shape == x.shape and grads[1].shape == w.shape
    if bias:
        wide = dy.double().flatten(0, -2)
        R.close(grads[2], wide.sum(0), wide.abs().sum(0) * ((rows / 8 + 24) * 2.0 ** -24) + wide.sum(0).abs() * R.U[kind])


def test_linear_gradients_by_differences(cs):
    """Small whole numbers are their own codes: the layer is then the linear map itself, and a loss's difference over a step of
    1 in one value is its gradient."""
    whole = lambda *s, seed: torch.randint(-3, 4, s, device="cuda", generator=torch.Generator(device="cuda").manual_seed(seed)).float()
    x, w, dy = whole(20, 24, seed=1).requires_grad_(True), whole(17, 24, seed=2).requires_grad_(True), whole(20, 17, seed=3)
    loss = lambda a, b: float((cs.fp8_linear(a, b) * dy).sum())
    dx, dw = torch.autograd.grad((cs.fp8_linear(x, w) * dy).sum(), (x, w))
    with torch.no_grad():
        base = loss(x, w)
        for i, j in ((0, 0), (7, 23), (19, 5), (16, 11)):
            for t, d in ((x, dx), (w, dw)):
                if i < t.shape[0]:
                    moved = t.clone()
                    moved[i, j] += 1
                    assert (loss(moved, w) if t is x else loss(x, moved)) - base == float(d[i, j])


def test_linear_keeps_what_its_gradients_need(cs):
    x, w = normal(9, 64), normal(5, 64, seed=1)
    for gx, gw in ((True, False), (False, True)):
        y, kept = keeping(lambda: cs.fp8_linear(x.clone().requires_grad_(gx), w.clone().requires_grad_(gw)))
        assert len(kept) == 2 and kept[0].numel() == (w.numel() if gx else x.numel())
    assert cs.fp8_linear(x, w).grad_fn is None


def test_linear_is_differentiable_once(cs):
    x, w = normal(9, 64).requires_grad_(True), normal(5, 64, seed=1).requires_grad_(True)
    dx, = torch.autograd.grad(cs.fp8_linear(x, w).square().sum(), x, create_graph=True)
    with pytest.raises(RuntimeError, match="differentiable once"):
        dx.sum().backward()


def test_linear_of_nothing(cs):
    w, b = normal(5, 64, seed=1).requires_grad_(True), normal(5).requires_grad_(True)
    x = torch.empty(2, 0, 64, device="cuda").requires_grad_(True)
    y = cs.fp8_linear(x, w, b)
    dx, dw, db = torch.autograd.grad(y.sum(), (x, w, b))
    assert y.shape == (2, 0, 5) and dx.shape == x.shape and (dw == 0).all() and (db == 0).all()
    y = cs.fp8_linear(torch.empty(2, 3, 0, device="cuda"), torch.empty(5, 0, device="cuda"), b)
    assert torch.equal(y, b.expand(2, 3, 5))


def test_linear_of_a_weight_quantized_before(cs):
    w, b = normal(300, 136, seed=1, kind=torch.bfloat16), normal(300, seed=2)
    q = cs.fp8_quantize(w)
    for shape in ((1, 136), (3, 4, 136), (200, 136)):
        x = normal(*shape, seed=3, kind=torch.bfloat16)
        assert R.bits_equal(cs.fp8_linear(x, q, b), cs.fp8_linear(x, w, b).detach())
    with pytest.raises(ValueError, match="no gradient"):
        cs.fp8_linear(normal(2, 136).requires_grad_(True), q)


@kinds
@pytest.mark.parametrize("rows,cols,out", [(1, 4096, 4096), (1, 1, 2), (2, 127, 300), (7, 515, 1030), (32, 2000, 640), (33, 300, 520),
                                           (5, 9000, 130), (31, 640, 31), (3, 70000, 40), (1, 0, 5)])
def test_linear_of_a_few_rows(cs, kind, rows, cols, out):
    """What quantizing and the product give one after the other, bit by bit, also where one launch does both; rows that lie
    apart, and off their alignment."""
    w = cs.fp8_quantize(normal(out, cols, seed=1, kind=kind))
    whole = (normal(rows, cols + 9, seed=2) * torch.exp(2 * normal(cols + 9, seed=3))).to(kind)
    for x in (whole[:, :cols].contiguous(), whole[:, :cols], whole[:, 3:cols + 3]):
        for bias in (None, normal(out, seed=4, kind=kind)):
            want = cs.fp8_matmul(*cs.fp8_quantize(x.contiguous()), *w, transpose_b=True, bias=bias, dtype=kind)
            assert R.bits_equal(cs.fp8_linear(x, w, bias), want)


def test_linear_of_a_few_rows_that_hold_no_numbers(cs):
    x, w = normal(4, 300, seed=1), cs.fp8_quantize(normal(200, 300, seed=2))
    x[1, 200], x[2, 5], x[3, :] = math.nan, -math.inf, 0.0
    y = cs.fp8_linear(x, w)
    assert torch.isfinite(y[0]).all() and torch.isnan(y[1]).all() and torch.isnan(y[2]).all() and (y[3] == 0).all()


def test_linear_under_autocast_and_of_a_transposed_input(cs):
    x, w = normal(24, 10, seed=1).requires_grad_(True), normal(6, 24, seed=2).requires_grad_(True)
    y = cs.fp8_linear(x.t(), w)
    want = cs.fp8_linear(x.detach().t().contiguous().requires_grad_(True), w)
    assert R.bits_equal(y, want)
    with torch.autocast("cuda", torch.bfloat16):
        z = cs.fp8_linear(x.t(), w)
        torch.autograd.grad(z.sum(), (x, w))
    assert R.bits_equal(z, y)


# ---- refusals ------------------------------------------------------------------------------------------------------

def test_refusals(cs):
    x = normal(40, 64)
    c, s = cs.fp8_quantize(x)
    odd, powers = cs.fp8_quantize(normal(40, 50))
    tight = odd.contiguous()  # rows of 50 bytes
    for call in (lambda: cs.fp8_quantize(x.double()), lambda: cs.fp8_quantize(x.t()), lambda: cs.fp8_quantize(torch.zeros((), device="cuda")),
                 lambda: cs.fp8_quantize(normal(4, 6, 8)[:, ::2]),
                 lambda: cs.fp8_dequantize(x, s), lambda: cs.fp8_dequantize(c, s.float()), lambda: cs.fp8_dequantize(c, s, torch.float64),
                 lambda: cs.fp8_dequantize(c.view(torch.uint8), s), lambda: cs.fp8_dequantize(tight, powers),
                 lambda: cs.fp8_dequantize(c, s.view(-1)), lambda: cs.fp8_dequantize(c[:, 1:33], s),
                 lambda: cs.fp8_dequantize(c.t(), s), lambda: cs.fp8_dequantize(c.cpu(), s),
                 lambda: cs.fp8_matmul(c, s, c, s), lambda: cs.fp8_matmul(c, s, c, s, transpose_a=True, transpose_b=True),
                 lambda: cs.fp8_matmul(c, s, c, s, transpose_b=True, bias=normal(64)),
                 lambda: cs.fp8_matmul(c, s, c, s, transpose_b=True, bias=normal(40).double()),
                 lambda: cs.fp8_matmul(c, s, c, s, transpose_b=True, bias=normal(80)[::2]),
                 lambda: cs.fp8_matmul(c, s, c, s, transpose_b=True, dtype=torch.int32),
                 lambda: cs.fp8_linear(x, normal(5, 40)), lambda: cs.fp8_linear(normal(64), normal(5, 64)),
                 lambda: cs.fp8_linear(x, (odd, powers)), lambda: cs.fp8_linear(x.double(), normal(5, 64)),
                 lambda: cs.fp8_linear(x, normal(5, 64, 1))):
        with pytest.raises(ValueError):
            call()
    with pytest.raises(TypeError):
        cs.fp8_dequantize(c, s, "float32")


def test_a_last_row_without_its_padding_is_refused(cs):
    """50 codes at the end of their storage: the kernels read and write a row's padding."""
    codes, scales = cs.fp8_quantize(normal(3, 50))
    short = torch.empty(2 * 64 + 50, dtype=torch.uint8, device="cuda").as_strided((3, 50), (64, 1)).view(torch.float8_e4m3fn)
    with pytest.raises(ValueError, match="padded"):
        cs.fp8_dequantize(short, scales)
    one = torch.zeros(1, 50, dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn)
    with pytest.raises(ValueError, match="padded"):
        cs.fp8_dequantize(one, scales)


@pytest.mark.parametrize("ta,tb", [(False, True), (False, False), (True, False), (True, True)],
                         ids=["nt", "nn", "tn", "tt"])
@pytest.mark.parametrize("m,n,k", [(2304, 2048, 640), (3000, 1700, 300), (2500, 1801, 4500), (1025, 5000, 100)])
def test_products_of_many_tiles(cs, m, n, k, ta, tb):
    """Tiles that two CTAs share, one behind the other on the same pair; results whose rows begin on 16 bytes and anywhere."""
    a, b, A, B = operands(cs, m, n, k, ta, tb)
    for kind in KINDS:
        bias = normal(n, seed=9, kind=kind)
        got = cs.fp8_matmul(*a, *b, transpose_a=ta, transpose_b=tb, bias=bias, dtype=kind)
        want, bound = R.product(A, B, bias, kind)
        if kind == torch.float16:  # what half precision cannot hold
            bound = bound.masked_fill(want.abs() > 65000, math.inf)
            got, want = got.clamp(-65504, 65504), want.clamp(-65504, 65504)
        R.close(got, want, bound)
