"""What the 8-bit floating-point matrices and the optimizer's step refuse, without a GPU: bad arguments of the C ABI end in a
status before any launch (a launch would return CSW_ERR_CUDA here), bad tensors in an exception."""
import ctypes as C

import pytest

ARG, SIZE = 1, 2
F32, F16, BF16 = 0, 1, 2


@pytest.fixture(scope="module")
def L():
    from cswap_b200 import build
    build.build()
    import cswap_b200
    return cswap_b200.lib()


@pytest.fixture(scope="module")
def mem():
    buf = (C.c_char * (1 << 16))()
    base = (C.addressof(buf) + 255) // 256 * 256
    yield base
    del buf


def test_quantize_arguments(L, mem):
    x, codes, scales, sums, ws = (mem + 8192 * i for i in range(5))

    def quantize(x=x, t=F32, rows=200, cols=5, stride=5, codes=codes, ld=16, scales=scales, sums=None, st=F32, ws=ws,
                 size=1 << 12):
        return L.csw_fp8_quantize(x, t, rows, cols, stride, codes, ld, scales, sums, st, ws, size, None)

    for bad in (dict(t=3), dict(x=None), dict(x=x + 2), dict(stride=4), dict(codes=None), dict(codes=codes + 8), dict(ld=8),
                dict(ld=24), dict(cols=17, stride=17), dict(scales=None), dict(sums=sums + 2), dict(sums=sums, st=3),
                dict(sums=sums + 1, st=BF16), dict(sums=sums, ws=None),
                dict(sums=sums, ws=ws + 2), dict(rows=1 << 31), dict(cols=1 << 31, stride=1 << 31, ld=1 << 31),
                dict(ld=(1 << 39) + 16), dict(stride=1 << 42),
                dict(rows=(1 << 31) - 1, cols=(1 << 31) - 1, stride=1 << 31, ld=1 << 31)):
        assert quantize(**bad) == ARG, bad
    assert quantize(sums=sums, size=39) == SIZE
    assert quantize(rows=0, x=None, codes=None, scales=None, ld=0) == 0 and quantize(cols=0, x=None, codes=None, scales=None) == 0
    b = C.c_size_t()
    for rows, cols, need in ((128, 5, 0), (129, 5, 40), (0, 7, 0), (16384, 768, 128 * 768 * 4)):
        assert L.csw_fp8_quantize_workspace(rows, cols, C.byref(b)) == 0 and b.value == need
    assert L.csw_fp8_quantize_workspace(1, 1, None) == ARG and L.csw_fp8_quantize_workspace(1 << 31, 1, C.byref(b)) == ARG


def test_dequantize_arguments(L, mem):
    codes, scales, out = mem, mem + 8192, mem + 16384

    def dequantize(codes=codes, ld=16, scales=scales, rows=3, cols=5, out=out, t=F16):
        return L.csw_fp8_dequantize(codes, ld, scales, rows, cols, out, t, None)

    for bad in (dict(t=9), dict(codes=None), dict(codes=codes + 4), dict(ld=20), dict(cols=40), dict(scales=None), dict(out=None),
                dict(out=out + 1), dict(t=F32, out=out + 2)):
        assert dequantize(**bad) == ARG, bad
    assert dequantize(rows=0, codes=None, scales=None, out=None) == 0


def test_matmul_arguments(L, mem):
    from cswap_b200._lib import Fp8Matrix
    p, s, out = mem, mem + 16384, mem + 32768

    def matrix(codes=p, scales=s, rows=4, cols=6, ld=16, t=0):
        return Fp8Matrix(codes, scales, rows, cols, ld, t)

    def matmul(a=matrix(), b=matrix(rows=6, cols=3), bias=None, bias_type=F32, out=out, t=BF16):
        r = [C.byref(m) if m is not None else None for m in (a, b)]
        return L.csw_fp8_matmul(*r, bias, bias_type, out, t, None)

    for bad in (dict(a=None), dict(b=None), dict(t=4), dict(out=None), dict(out=out + 1), dict(bias=p, bias_type=5),
                dict(bias=p + 2), dict(b=matrix()), dict(b=matrix(cols=5, t=1)), dict(a=matrix(t=1)), dict(a=matrix(codes=None)),
                dict(a=matrix(codes=p + 8)), dict(a=matrix(scales=None)), dict(a=matrix(ld=8)), dict(a=matrix(ld=4)),
                dict(a=matrix(rows=1 << 31)), dict(a=matrix(ld=1 << 40)),
                dict(a=matrix(rows=(1 << 31) - 8, cols=1), b=matrix(rows=1, cols=1)),
                dict(a=matrix(rows=1 << 30, cols=1), b=matrix(rows=1, cols=1 << 30, ld=1 << 30))):
        assert matmul(**bad) == ARG, bad
    empty = matrix(codes=None, scales=None, rows=0, cols=6)
    assert matmul(a=empty, out=None) == 0


def test_linear_arguments(L, mem):
    from cswap_b200._lib import Fp8Matrix
    x, p, s, out, ws = (mem + 8192 * i for i in range(5))

    def linear(x=x, t=F32, rows=40, stride=6, w=Fp8Matrix(p, s, 9, 6, 16, 0), bias=None, bt=F32, out=out, ot=BF16, ws=ws, size=4096):
        return L.csw_fp8_linear(x, t, rows, stride, C.byref(w) if w is not None else None, bias, bt, out, ot, ws, size, None)

    for bad in (dict(x=None), dict(x=x + 2), dict(t=3), dict(stride=5), dict(w=None), dict(w=Fp8Matrix(p, s, 9, 6, 16, 1)),
                dict(w=Fp8Matrix(p + 4, s, 9, 6, 16, 0)), dict(w=Fp8Matrix(p, None, 9, 6, 16, 0)), dict(w=Fp8Matrix(p, s, 9, 6, 8, 0)),
                dict(bias=p + 2), dict(bias=p, bt=4), dict(out=None), dict(out=out + 1), dict(ot=9), dict(ws=None), dict(ws=ws + 8),
                dict(rows=1 << 31), dict(rows=(1 << 31) - 8), dict(stride=1 << 42)):
        assert linear(**bad) == ARG, bad
    assert linear(size=40 * 16) == SIZE and linear(rows=0, x=None, out=None, ws=None, size=0) == 0
    b = C.c_size_t()
    for rows, cols, outs, need in ((40, 6, 9, 40 * 16 + 1), (32, 6, 33, 0), (1, 4096, 4096, 0), (32, 6, 32, 513), (0, 6, 9, 0),
                                   (1, 65537, 9, 65552 + 513), (300, 130, 5, 300 * 144 + 6)):
        assert L.csw_fp8_linear_workspace(rows, cols, outs, C.byref(b)) == 0 and b.value == need
    assert L.csw_fp8_linear_workspace(1, 1, 1, None) == ARG and L.csw_fp8_linear_workspace(1 << 31, 1, 1, C.byref(b)) == ARG


def test_step_arguments(L, mem):
    from cswap_b200._lib import AdamwOptions, AdamwTensor
    at = [mem + 4096 * i for i in range(8)]

    def tensor(p=at[0], g=at[1], c=None, m=at[2], v=at[3], ms=None, vs=None, n=9, pt=F32, gt=F32, ct=F32):
        return AdamwTensor(p, g, c, m, v, ms, vs, n, pt, gt, ct)

    def options(bits=32, step=1, lr=1e-3, b1=0.9, b2=0.999, eps=1e-8, wd=0.0, top=1.0, ds=None, dl=None, dn=None):
        return AdamwOptions(bits, 0, step, lr, b1, b2, eps, wd, top, ds, dl, dn)

    def step(t=tensor(), o=options(), count=1):
        return L.csw_adamw_step(C.byref(t) if t is not None else None, count, C.byref(o) if o is not None else None, None)

    eight = dict(ms=at[4], vs=at[5])
    for bad in (dict(t=None), dict(o=None), dict(count=1 << 25), dict(t=tensor(p=None)), dict(t=tensor(g=None)), dict(t=tensor(p=at[0] + 2)),
                dict(t=tensor(pt=3)), dict(t=tensor(gt=-1)), dict(t=tensor(c=at[6], ct=3)), dict(t=tensor(c=at[6] + 1, ct=F16)),
                dict(t=tensor(m=None)), dict(t=tensor(v=at[3] + 1)), dict(t=tensor(n=(1 << 41) + 1)), dict(t=tensor(**eight)),
                dict(o=options(bits=8)), dict(t=tensor(ms=at[4]), o=options(bits=8)), dict(o=options(bits=16)),
                dict(o=options(step=0)), dict(o=options(lr=-1.0)), dict(o=options(lr=float("nan"))), dict(o=options(b1=1.0)),
                dict(o=options(b2=-0.1)), dict(o=options(b2=float("nan"))), dict(o=options(eps=-1.0)), dict(o=options(wd=float("inf"))),
                dict(o=options(ds=at[6] + 4)), dict(o=options(dl=at[6] + 2)), dict(o=options(dn=at[6] + 1)),
                dict(o=options(dn=at[6], top=-1.0)), dict(o=options(dn=at[6], top=float("nan")))):
        assert step(**bad) == ARG, bad
    assert step(t=None, count=0) == 0 and step(t=tensor(p=None, g=None, m=None, v=None, n=0)) == 0
    for f in (L.csw_adamw8_pack, L.csw_adamw8_unpack):
        good = dict(c=at[6], **eight)
        for bad in (tensor(**eight), tensor(c=at[6]), tensor(p=at[0] + 2, **good), tensor(**{**good, "m": None}), tensor(n=1 << 42, **good),
                    tensor(pt=BF16, **good), tensor(ct=F16, **good)):
            assert f(C.byref(bad), 1, None) == ARG
        assert f(None, 1, None) == ARG and f(None, 0, None) == 0
    b = C.c_size_t()
    assert L.csw_gradient_norm_workspace(None, 0, C.byref(b)) == 0 and b.value == 0
    assert L.csw_gradient_norm_workspace(C.byref(tensor()), 1, C.byref(b)) == 0 and b.value == 8
    assert L.csw_gradient_norm_workspace(C.byref(tensor()), 1, None) == ARG
    norm = lambda t=tensor(), to=at[6], ws=at[7], size=8: L.csw_gradient_norm(C.byref(t), 1, to, ws, size, None)
    assert norm(size=7) == SIZE
    for bad in (dict(to=None), dict(to=at[6] + 2), dict(ws=None), dict(ws=at[7] + 4), dict(t=tensor(g=None)), dict(t=tensor(gt=7))):
        assert norm(**bad) == ARG, bad


def test_cpu_tensors_are_refused(L):
    import torch
    import cswap_b200 as cs
    x = torch.zeros(4, 16)
    c, s = x.to(torch.float8_e4m3fn), torch.zeros(1, 1, dtype=torch.uint8).view(torch.float8_e8m0fnu)
    state = cs.adamw8_state(x)
    for call in (lambda: cs.fp8_quantize(x), lambda: cs.fp8_dequantize(c, s), lambda: cs.fp8_matmul(c, s, c, s, transpose_b=True),
                 lambda: cs.fp8_linear(x, x), lambda: cs.fp8_linear(x, (c, s)), lambda: cs.gradient_norm([x]),
                 lambda: cs.adamw_step([x], [x], [x], [x], 1), lambda: cs.adamw8_step([x], [x], [state], 1),
                 lambda: cs.adamw8_pack([state], [x], [x]), lambda: cs.adamw8_unpack([state], [x], [x])):
        with pytest.raises(ValueError, match="CUDA"):
            call()


def test_the_mixing_of_the_rounding_spreads_every_bit():
    """Flipping a bit of the input flips each bit of the output in 40 to 60 % of 65536 cases, and counting through the inputs
    gives every value of 8 bits about as often: within six standard deviations."""
    import numpy as np
    import step_reference as R
    x = np.arange(1 << 16, dtype=np.uint32)
    for start in (0, 0x9e3779b9, 0xffff0000):
        at = x + np.uint32(start)
        base = R.mix(at)
        for bit in range(32):
            flipped = base ^ R.mix(at ^ np.uint32(1 << bit))
            for out in range(32):
                assert 0.4 < ((flipped >> np.uint32(out)) & 1).mean() < 0.6
        for shift in (0, 8, 16, 24):
            counts = np.bincount((base >> np.uint32(shift)) & 255, minlength=256)
            assert abs(counts - 256).max() < 6 * 16
