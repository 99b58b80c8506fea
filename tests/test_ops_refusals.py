"""What the training operators refuse, without a GPU: bad arguments of the C ABI end in a status before any launch
(there is no device here that a launch could run on: it would return CSW_ERR_CUDA), bad tensors in an exception."""
import ctypes as C

import pytest

ARG, SIZE, CUDA = 1, 2, 3
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


def test_q8_sizes(L):
    import cswap_b200 as cs
    assert [cs.q8_bytes(n) for n in (0, 1, 16, 17, 128, 129, 50331648)] == \
        [0, 16 + 4, 16 + 4, 32 + 4, 128 + 4, 144 + 8, 50331648 + 4 * 393216]
    with pytest.raises(ValueError):
        cs.q8_bytes(-1)
    b = C.c_size_t()
    assert L.csw_q8_bytes(1 << 43, C.byref(b)) == ARG and L.csw_q8_bytes(5, None) == ARG


def test_q8_and_gelu_arguments(L, mem):
    p, q = mem, mem + 4096
    need = 144 + 8
    assert L.csw_q8_compress(p, 3, 129, q, need, None) == ARG           # no such type
    assert L.csw_q8_compress(None, F32, 129, q, need, None) == ARG
    assert L.csw_q8_compress(p + 2, F32, 129, q, need, None) == ARG     # a float between floats
    assert L.csw_q8_compress(p, F32, 129, q + 8, need, None) == ARG     # the checkpoint lies on 16 bytes
    assert L.csw_q8_compress(p, F32, 129, q, need - 1, None) == SIZE
    assert L.csw_q8_compress(None, F32, 0, None, 0, None) == 0          # nothing to do
    assert L.csw_q8_decompress(q, need - 1, 129, p, F32, None) == SIZE
    assert L.csw_q8_decompress(q, need, 129, None, F32, None) == ARG
    assert L.csw_q8_decompress(q, need, 129, p + 1, BF16, None) == ARG
    assert L.csw_q8_decompress(None, 0, 0, None, F16, None) == 0
    assert L.csw_gelu_forward(p, F32, 129, None, q, need, None) == ARG
    assert L.csw_gelu_forward(p, F32, 129, p, q, need - 1, None) == SIZE
    assert L.csw_gelu_backward(p, F32, q, need, 129, None, None, None) == ARG
    assert L.csw_gelu_backward(p, F32, q, need, 129, p, p + 2, None) == ARG
    assert L.csw_gelu_backward(p, F32, q, need - 1, 129, p, None, None) == SIZE


def test_layer_norm_arguments(L, mem):
    p = [mem + 4096 * i for i in range(8)]

    def forward(x=p[0], r=None, w=p[1], b=p[2], t=BF16, pt=BF16, rows=3, cols=5, y=p[3], s=None, mean=p[4], rstd=p[5]):
        return L.csw_layer_norm_forward(x, r, w, b, t, pt, rows, cols, 1e-5, y, s, mean, rstd, None)

    for bad in (dict(t=3), dict(pt=F16), dict(t=F32, pt=BF16), dict(cols=0), dict(rows=1 << 31), dict(cols=1 << 31),
                dict(x=None), dict(y=None), dict(mean=None), dict(rstd=p[5] + 2), dict(x=p[0] + 1), dict(w=p[1] + 1),
                dict(pt=F32, b=p[2] + 2), dict(r=p[6]), dict(r=p[6] + 1, s=p[7])):
        assert forward(**bad) == ARG, bad
    assert forward(rows=0, x=None, y=None) == 0

    def backward(dy=p[0], x=p[1], mean=p[2], rstd=p[3], w=p[4], t=BF16, pt=F32, rows=3, cols=5, dx=p[5], dw=p[6],
                 db=p[7], ws=mem + 32768, size=1 << 15):
        return L.csw_layer_norm_backward(dy, x, mean, rstd, w, t, pt, rows, cols, dx, dw, db, ws, size, None)

    for bad in (dict(t=7), dict(pt=F16), dict(cols=0), dict(dy=None), dict(x=p[1] + 1), dict(dx=None), dict(mean=None),
                dict(rstd=p[3] + 1), dict(w=p[4] + 2), dict(dw=p[6] + 2), dict(ws=None), dict(ws=mem + 32770)):
        assert backward(**bad) == ARG, bad
    assert backward(size=3) == SIZE
    b = C.c_size_t()
    assert L.csw_layer_norm_workspace(0, 768, C.byref(b)) == 0 and b.value == 0
    assert L.csw_layer_norm_workspace(1, 768, C.byref(b)) == 0 and b.value == 2 * 4 * 768
    assert L.csw_layer_norm_workspace(1, 0, C.byref(b)) == ARG


def test_attention_arguments(L, mem):
    from cswap_b200._lib import AttentionOperand, AttentionShape

    def shape(**kw):
        d = dict(type=BF16, causal=0, batch=1, heads=4, kv_heads=2, q_len=8, k_len=8, dim=16, scale=0.25, kv_lens=None)
        d.update(kw)
        return AttentionShape(**d)

    def operand(data=mem, b=512, h=128, t=16):
        return AttentionOperand(data, b, h, t)

    o = operand()

    def forward(s, q=o, k=o, v=o, out=o, lse=mem):
        r = [C.byref(x) if x is not None else None for x in (s, q, k, v, out)]
        return L.csw_attention_forward(*r, lse, None)

    for bad in (dict(type=F32), dict(type=5), dict(dim=0), dict(dim=12), dict(dim=136), dict(heads=3), dict(heads=0),
                dict(kv_heads=0), dict(batch=1 << 20), dict(q_len=1 << 31), dict(kv_lens=mem + 2),
                dict(batch=65535, heads=65534, q_len=1 << 30)):
        assert forward(shape(**bad)) == ARG, bad
    assert forward(None) == ARG
    for bad in (operand(data=None), operand(data=mem + 8), operand(b=4), operand(h=9), operand(t=-16), operand(h=0), operand(t=0),
                None):
        for place in ("q", "k", "v", "out"):
            assert forward(shape(batch=2), **{place: bad}) == ARG
    assert forward(shape(), lse=None) == ARG
    # the stride of an axis of one step is not looked at: one token of one head, refused for its missing lse
    assert forward(shape(heads=1, kv_heads=1, q_len=1, k_len=1), *[operand(b=0, h=0, t=0)] * 4, lse=None) == ARG
    assert forward(shape(q_len=(1 << 29) + 1)) == ARG
    empty = operand(data=None, b=0, h=0, t=0)
    assert forward(shape(q_len=0), q=empty, out=empty, lse=None) == 0
    size = C.c_size_t()
    assert L.csw_attention_workspace(C.byref(shape()), C.byref(size)) == 0 and size.value >= 4 * 8 * 4
    assert L.csw_attention_workspace(C.byref(shape(dim=7)), C.byref(size)) == ARG
    refs = [C.byref(o)] * 4
    s = C.byref(shape())
    assert L.csw_attention_backward(s, *refs, mem, *refs, mem, size.value - 1, None) == SIZE
    assert L.csw_attention_backward(s, *refs, None, *refs, mem, size.value, None) == ARG
    assert L.csw_attention_backward(s, *refs, mem, *refs, None, size.value, None) == ARG
    assert L.csw_attention_backward(s, *refs, mem, None, *refs[1:], mem, size.value, None) == ARG


def test_operators_refuse_cpu_tensors(L):
    import torch
    import cswap_b200 as cs
    x, h = torch.zeros(4, 8), torch.zeros(1, 2, 4, 8, dtype=torch.float16)
    lse = torch.zeros(1, 2, 4)
    for call in (lambda: cs.q8_compress(x), lambda: cs.q8_decompress(torch.zeros(64, dtype=torch.uint8), 32),
                 lambda: cs.gelu(x), lambda: cs.gelu_linear(x, torch.zeros(3, 8)), lambda: cs.gelu_forward(x),
                 lambda: cs.gelu_backward(x, torch.zeros(64, dtype=torch.uint8)), lambda: cs.layer_norm(x),
                 lambda: cs.layer_norm_forward(x), lambda: cs.layer_norm_backward(x, x, x[:, 0], x[:, 0]),
                 lambda: cs.attention(h, h, h), lambda: cs.attention_forward(h, h, h),
                 lambda: cs.attention_backward(h, h, h, h, h, lse)):
        with pytest.raises(ValueError, match="CUDA"):
            call()
    with pytest.raises(TypeError):
        cs.q8_compress([1.0])
    with pytest.raises(TypeError):
        cs.layer_norm_forward(x, "weight")
