"""Matrices in 8-bit floating point and the optimizer's step by their definitions, in 64 bits and numpy's 32-bit operations."""
import numpy as np
import torch

U = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
# half the distance of the numbers below the type's normal ones
SMALL = {torch.float32: 2.0 ** -150, torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -134}


def e4m3_values():
    """The value of each of the 256 codes."""
    c = np.arange(256)
    x, f = c >> 3 & 15, c & 7
    v = np.where(x == 0, f / 8 * 2.0 ** -6, (1 + f / 8) * 2.0 ** (x - 7.0))
    v = np.where(c & 127 == 127, np.nan, v)
    return np.where(c & 128, -v, v)


def fp8(x):
    """(codes, scale bytes, the values held) of a matrix, by comparing with every number of the format."""
    x = x.detach().double().cpu().numpy()
    rows, cols = x.shape
    rb, cb = -(-rows // 128), -(-cols // 128)
    codes, scales, held = np.zeros((rows, cols), np.uint8), np.zeros((rb, cb), np.uint8), np.zeros((rows, cols))
    positive = e4m3_values()[:127]
    middle = (positive[1:] + positive[:-1]) / 2
    for i in range(rb):
        for j in range(cb):
            at = (slice(128 * i, 128 * i + 128), slice(128 * j, 128 * j + 128))
            b = x[at]
            size = np.abs(b)
            top = size[np.isfinite(size)].max(initial=0.0)
            e = -126
            while top > 448 * 2.0 ** e:
                e += 1
            t = np.where(np.isfinite(size), size, 0.0) * 2.0 ** -e
            # the nearest: how many middles lie below; on a middle, the even one
            below, upto = np.searchsorted(middle, t, "left"), np.searchsorted(middle, t, "right")
            c = np.where((below != upto) & (below % 2 == 1), upto, below)
            v = positive[c] * 2.0 ** e
            bad = ~np.isfinite(size)
            codes[at] = np.where(bad, 127, c | np.where(np.signbit(b), 128, 0))
            held[at] = np.where(bad, np.nan, np.where(np.signbit(b), -v, v))
            scales[i, j] = e + 127
    return codes, scales, torch.from_numpy(held)


def held_of(codes, scales):
    """The values that a program's codes and scales stand for, in float64."""
    v = torch.from_numpy(e4m3_values()).to(codes.device)[codes.view(torch.uint8).long()]
    s = torch.exp2(scales.view(torch.uint8).double() - 127).repeat_interleave(128, 0).repeat_interleave(128, 1)
    return v * s[:v.shape[0], :v.shape[1]]


def product(a, b, bias, kind):
    """(a b + bias, how far a result may be off) of float64 operands: products are exact; a step of the tensor cores adds 32 of
    them and the sum so far, each cut off at 2^-24 of the largest, k / 32 steps; the bias and the rounding to the type."""
    want, size = a @ b, a.abs() @ b.abs()
    off = size * ((33.0 * (a.shape[1] // 32 + 2)) * 2.0 ** -24)
    if bias is not None:
        want = want + bias.double()
        off = off + want.abs() * 2.0 ** -24
    return want, off + want.abs() * U[kind] + SMALL[kind]


# ---- the optimizer's step ------------------------------------------------------------------------------------------

def mix(x):
    x = x.astype(np.uint32)
    with np.errstate(over="ignore"):
        x = x ^ (x >> np.uint32(16))
        x = x * np.uint32(0x9e3779b1)
        x = x ^ (x >> np.uint32(15))
        x = x * np.uint32(0x85ebca77)
        return x ^ (x >> np.uint32(16))


def random_bits(seed, step, place, n):
    """(for m, for v) of a tensor's values: 16 bits each."""
    odd, word = 0x9e3779b9, 0xffffffff
    call = int(mix(np.array([seed + step * odd & word]))[0])
    key = int(mix(np.array([call + place * odd & word]))[0])
    r = mix((key + np.arange(n, dtype=np.uint64)) & np.uint64(word))
    return r >> np.uint32(16), r & np.uint32(0xffff)


def code_values(exponents):
    """The values of the codes without a sign, at a scale of 1."""
    c = np.arange(1 << exponents + 3)
    x, f = c >> 3, c & 7
    top = (1 << exponents) - 1
    return np.where(x == 0, f / 8 * 2.0 ** (1 - top), (1 + f / 8) * 2.0 ** (x - top))


def encode(x, bits, exponents):
    """(codes, scale bytes) of float32 values: codes without a sign by their definition as numbers; `bits` of 2^20 are added to
    the part of a step that a value is above its code."""
    n = x.size
    groups = -(-n // 128)
    wide = np.zeros(groups * 128)
    wide[:n] = x
    extra = np.zeros(groups * 128)
    extra[:n] = bits
    wide, extra = wide.reshape(groups, 128), extra.reshape(groups, 128)
    table = code_values(exponents)
    codes, scales = np.zeros((groups, 128), np.uint8), np.zeros(groups, np.uint8)
    for i in range(groups):
        size = np.abs(wide[i])
        top = size.max()
        if top == 0:
            continue
        if not np.isfinite(top) or top > 1.75 * 2.0 ** 126:
            scales[i] = 255
            continue
        e = -126
        while top > 1.75 * 2.0 ** e:
            e += 1
        scales[i] = e + 127
        t = size * 2.0 ** -e
        below = np.searchsorted(table, t, "right") - 1  # the largest code whose value is not above
        step = np.diff(table)[np.minimum(below, table.size - 2)]
        part = np.rint((t - table[below]) / step * 2.0 ** 20)  # the foot of float32's range: 20 bits below the code
        code = below + (part + extra[i] >= 2.0 ** 20)
        if exponents == 5:
            code = np.maximum(code, 1)
        else:
            code = code | np.where(np.signbit(wide[i]), 128, 0)
        codes[i] = code
    return codes.reshape(-1)[:n], scales


def decode(codes, scales, exponents):
    """The float32 values that codes and scales stand for, in float64."""
    table = code_values(exponents)
    size = table[codes & (127 if exponents == 4 else 255)]
    power = np.where(scales == 255, np.nan, np.where(scales == 0, 0.0, 2.0 ** (scales.astype(np.float64) - 127)))
    v = size * np.repeat(power, 128)[:codes.size]
    v = np.where((exponents == 4) & (codes >= 128), -v, v)
    return v.astype(np.float32)


class Adamw:
    """One step on numpy arrays: 64 bits for the parameter, 32-bit operations one by one for the averages."""

    def __init__(self, step, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=0.01, factor=1.0):
        self.step, self.lr, self.betas, self.eps, self.decay = step, lr, betas, eps, weight_decay
        self.factor = np.float32(factor)

    def averages(self, g, m, v):
        b1, r1, b2, r2 = (np.float32(x) for x in (self.betas[0], 1 - self.betas[0], self.betas[1], 1 - self.betas[1]))
        with np.errstate(all="ignore"):
            g = g.astype(np.float32) * self.factor
            return m * b1 + g * r1, v * b2 + g * r2 * g

    def param(self, p, m, v):
        b1, b2 = self.betas
        with np.errstate(all="ignore"):
            m_hat, v_hat = m.astype(np.float64) / (1 - b1 ** self.step), v.astype(np.float64) / (1 - b2 ** self.step)
            move = self.lr * m_hat / (np.sqrt(v_hat) + self.eps)
            return p.astype(np.float64) * (1 - self.lr * self.decay) - move, move


def param_bound(want, move, p, lr, kind):
    """Six float32 roundings of the move (its size, the root's product, the sum with eps, the root, the quotient, the product)
    and its scalars', a rounding of the decay, of its product, and of the difference; then the type's."""
    return move.abs() * (10 * 2.0 ** -24) + p.abs() * (3 * 2.0 ** -24) + want.abs() * 2.0 ** -24 + want.abs() * U[kind] + SMALL[kind]


def close(got, want, bound):
    got, want = got.double().cpu(), want.double().cpu()
    bound = bound.double().cpu() if isinstance(bound, torch.Tensor) else torch.full_like(want, bound)
    assert torch.equal(torch.isnan(got), torch.isnan(want)), "NaN where none belongs, or none where one does"
    fine = ~torch.isnan(want)
    off = ((got - want).abs() - bound)[fine & (got != want)]
    assert off.numel() == 0 or float(off.max()) <= 0, f"off by {float(off.max()):.3e} more than allowed"


def bits_equal(a, b):
    view = {4: torch.int32, 2: torch.int16, 1: torch.uint8}[a.element_size()]
    return torch.equal(a.contiguous().view(view), b.contiguous().view(view))
