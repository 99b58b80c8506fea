"""The operators of a training step in 8 bits, as timed passes through their entry points: linear layers whose products
take 8-bit floating-point operands, and the optimizer's step over all parameters with its state in 8 bits or in 32.

Kinds of pass ("op"):

  quantize   a matrix into 8-bit floating point and back, and the sums of its columns.  Blocks of 128 x 128 values share a
             scale 2^E, E the least for which the block's largest magnitude is at most 448 2^E (but -126 at least); a
             value's code is the e4m3 number nearest to x / 2^E, ties to even.
  linear     y = x W^T + b for a weight that was quantized before, x quantized in the call: serving.
  train      the same for a weight as it is, and its backward pass: y, and the gradients dx = dy W, dW = dy^T x, db, each
             product on quantized operands (dy, too).
  adamw      one step over many tensors: m = b1 m + (1 - b1) g, v = b2 v + (1 - b2) g^2,
             p = p (1 - lr wd) - lr (m / (1 - b1^t)) / (sqrt(v / (1 - b2^t)) + eps), the gradients scaled first so that
             their norm over all tensors is at most max_norm where that is given, and a 16-bit copy of the parameters
             written where one is kept.  In 8 bits, groups of 128 consecutive values of a tensor share a scale 2^E, E the
             least for which the largest magnitude is at most 1.75 2^E; m has a sign, 4 bits of exponent and 3 of mantissa,
             v 5 and 3, both with gradual underflow, rounded up or down by random bits from a seed, v never to zero.

Sizes: the parameters and token matrices of a BERT-base-shaped encoder at batch 32 x 512 (hidden 768), the parameters of
the VGG16 workload, wider layers, single tokens, and small and ragged ones of each kind.
"""
import math
import random

import torch

own = False

TYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
BYTES = {"fp32": 4, "bf16": 2, "fp16": 2, "": 0}
BLOCK = 128
GROUP = 128
BETAS, EPS, LR, DECAY, STEP, MAX_NORM = (0.9, 0.999), 1e-8, 1e-3, 0.01, 10, 1.0
FAN = 4  # a feed-forward layer's width over the hidden one's


def listed():
    return [
        # a short sentence's hidden states: a call is launch latency
        {"name": "quantize_tokens_bf16", "op": "quantize", "type": "bf16", "rows": 77, "cols": 768},
        # a wide feed-forward activation
        {"name": "quantize_wide_fp32", "op": "quantize", "type": "fp32", "rows": 16384, "cols": 4096},
        # one token through a wide layer, as in generation: the weight is read once
        {"name": "linear_token_bf16", "op": "linear", "type": "bf16", "rows": 1, "cols": 4096, "out": 4096, "bias": False},
        # a projection of the encoder, in evaluation
        {"name": "linear_hidden_bf16", "op": "linear", "type": "bf16", "rows": 16384, "cols": 768, "out": 768, "bias": True},
        # and in training, with the float32 parameters that it has by default
        {"name": "train_hidden_fp32", "op": "train", "type": "fp32", "rows": 16384, "cols": 768, "out": 768, "bias": True},
        # a wide layer's training step
        {"name": "train_wide_bf16", "op": "train", "type": "bf16", "rows": 8192, "cols": 4096, "out": 8192, "bias": False},
        # sizes that are no multiple of anything
        {"name": "train_ragged_fp16", "op": "train", "type": "fp16", "rows": 1001, "cols": 515, "out": 333, "bias": True},
        # the encoder's parameters, everything in 32 bits
        {"name": "adamw_encoder_fp32", "op": "adamw", "bits": 32, "set": "encoder", "layers": 12, "hidden": 768,
         "type": "fp32", "grad": "fp32", "copy": "", "clip": False},
        # the same with the state in 8 bits, 16-bit gradients and a 16-bit copy for the next forward pass, clipped
        {"name": "adamw8_encoder_bf16", "op": "adamw", "bits": 8, "set": "encoder", "layers": 12, "hidden": 768,
         "type": "fp32", "grad": "bf16", "copy": "bf16", "clip": True},
        # the convolutional workload's parameters
        {"name": "adamw8_vgg16_fp32", "op": "adamw", "bits": 8, "set": "vgg16", "type": "fp32", "grad": "fp32", "copy": "",
         "clip": True},
        # a few small ragged tensors (norms, biases, an adapter), one behind the other: a call is launch latency
        {"name": "adamw_small_bf16", "op": "adamw", "bits": 32, "set": "ragged", "tensors": 40, "numel": 60000, "salt": 7,
         "type": "bf16", "grad": "bf16", "copy": "", "clip": True},
        {"name": "adamw8_small_fp32", "op": "adamw", "bits": 8, "set": "ragged", "tensors": 9, "numel": 20000, "salt": 3,
         "type": "fp32", "grad": "fp32", "copy": "", "clip": False},
    ]


def _log_between(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["quantize", "linear", "linear", "train", "train", "adamw", "adamw"])
    kind = rng.choice(["fp32", "bf16", "fp16"])
    if op == "quantize":
        cols = _log_between(rng, 1, 16384)
        return {"op": op, "type": kind, "rows": _log_between(rng, 1, max(1, (1 << 26) // cols)), "cols": cols}
    if op != "adamw":
        cols, out = _log_between(rng, 8, 8192), _log_between(rng, 8, 8192)
        # no more products than the wide listed case, no more values than a token matrix of it
        most = min(8192 * 4096 * 8192 // (cols * out), (1 << 26) // max(cols, out), 16384)
        return {"op": op, "type": kind, "rows": _log_between(rng, 1, max(1, most)), "cols": cols, "out": out,
                "bias": rng.random() < 0.5}
    bits = rng.choice([8, 32])
    grad = kind if rng.random() < 0.7 else "fp32" if kind != "fp32" else rng.choice(["bf16", "fp16"])
    return {"op": op, "bits": bits, "set": "ragged", "tensors": _log_between(rng, 1, 600),
            "numel": _log_between(rng, 600, 1 << 26), "salt": rng.randrange(1 << 20), "type": kind, "grad": grad,
            "copy": rng.choice(["", "bf16", "fp16"]) if kind == "fp32" else "", "clip": rng.random() < 0.5}


# ---- what a program has in hand --------------------------------------------------------------------------------

def _sizes(case):
    """Values of each parameter tensor."""
    if case["set"] == "encoder":
        h = case["hidden"]
        layer = 4 * [h * h, h] + [h, h] + [h * FAN * h, FAN * h, FAN * h * h, h] + [h, h]
        return [30522 * h, 512 * h, h, h] + case["layers"] * layer + [2 * h, 2]
    if case["set"] == "vgg16":
        widths = [3, 64, 64, 128, 128, 256, 256, 256, 512, 512, 512, 512, 512, 512]
        convs = [n for a, b in zip(widths, widths[1:]) for n in (9 * a * b, b, b, b)]
        return convs + [512 * 4096, 4096, 4096 * 4096, 4096, 10 * 4096, 10]
    rng = random.Random(case["salt"])
    shares = [math.exp(rng.uniform(0.0, 6.0)) for _ in range(case["tensors"])]
    return [max(1, int(case["numel"] * s / sum(shares))) for s in shares]


def _places(case):
    """Where each tensor begins in a flat buffer of all of them, and the buffer's values.  In 8 bits every tensor begins
    a group of its own; in 32 they lie one behind the other."""
    step = GROUP if case["bits"] == 8 else 1
    begins, at = [], 0
    for n in _sizes(case):
        begins.append(at)
        at += -(-n // step) * step
    return begins, -(-at // GROUP) * GROUP


def _prepare_adamw(case, gen):
    def normal(n):
        return torch.randn(n, generator=gen, device="cuda")

    sizes = _sizes(case)
    begins, total = _places(case)
    held = torch.zeros(total, device="cuda")  # 1 where a value of a tensor lies, 0 between tensors
    marks = torch.zeros(total + 1, device="cuda", dtype=torch.int32)
    marks[torch.tensor(begins, device="cuda")] += 1
    marks.index_add_(0, torch.tensor([b + n for b, n in zip(begins, sizes)], device="cuda"),
                     torch.full((len(sizes),), -1, device="cuda", dtype=torch.int32))
    held.copy_(torch.cumsum(marks, 0)[:total])
    del marks
    s = {"case": case, "seed": 1234567}
    # gradients of sizes that differ from weight to weight, and averages such as a few steps leave behind
    size = torch.exp(normal(total)).mul_(1e-4)
    s["g"] = (normal(total) * size * held).to(TYPES[case["grad"]])
    s["p"] = (normal(total).mul_(0.02) * held).to(TYPES[case["type"]])
    m = normal(total).mul_(0.3).mul_(size).mul_(held)
    v = normal(total).mul_(0.2).add_(1.0).mul_(size).square_().mul_(0.01).mul_(held)
    del size, held
    s["copy"] = s["p"].to(TYPES[case["copy"]]) if case["copy"] else None
    views = lambda t: [t[b:b + n] for b, n in zip(begins, sizes)]
    s["ps"], s["gs"] = views(s["p"]), views(s["g"])
    s["copies"] = views(s["copy"]) if case["copy"] else None
    if case["bits"] == 32:
        s["m"], s["v"] = m, v
        s["ms"], s["vs"] = views(m), views(v)
        return s
    half = torch.full((1,), 1 << 19, device="cuda", dtype=torch.int32)
    s["m_codes"], s["m_scales"] = _pack(m, half, True)
    s["v_codes"], s["v_scales"] = _pack(v, half, False)
    groups = lambda t: [t[b // GROUP:b // GROUP + -(-n // GROUP)] for b, n in zip(begins, sizes)]
    s["states"] = list(zip(views(s["m_codes"]), views(s["v_codes"]), groups(s["m_scales"]), groups(s["v_scales"])))
    # where the averages are handed out in 32 bits; which tensor a group belongs to, and which of its groups it is
    s["m"], s["v"] = m, v
    s["ms"], s["vs"] = views(m), views(v)
    count = torch.tensor([-(-n // GROUP) for n in sizes], device="cuda")
    s["tensor"] = torch.repeat_interleave(torch.arange(len(sizes), device="cuda"), count)
    s["index"] = torch.arange(total // GROUP, device="cuda") - torch.tensor(begins, device="cuda")[s["tensor"]] // GROUP
    s["left"] = (torch.tensor(sizes, device="cuda")[s["tensor"]] - s["index"] * GROUP).clamp_(max=GROUP)
    return s


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    if case["op"] == "adamw":
        return _prepare_adamw(case, gen)

    def normal(*shape):
        return torch.randn(*shape, generator=gen, device="cuda")

    rows, cols, kind = case["rows"], case["cols"], TYPES[case["type"]]
    # what a layer is given: normal, some channels larger than others
    s = {"case": case, "x": normal(rows, cols).mul_(torch.exp(normal(cols))).to(kind)}
    if case["op"] == "quantize":
        return s
    out = case["out"]
    w = normal(out, cols).div_(math.sqrt(cols)).to(kind)
    s["b"] = normal(out).mul_(0.1).to(kind) if case["bias"] else None
    if case["op"] == "linear":  # rows of codes begin on 16 bytes
        codes, scales = _quantize(w)
        s["codes"] = torch.zeros(out, -(-cols // 16) * 16, device="cuda", dtype=torch.uint8)
        s["codes"][:, :cols] = codes[:out, :cols].contiguous().view(torch.uint8)
        s["codes"] = s["codes"].view(torch.float8_e4m3fn)[:, :cols]
        s["scales"] = scales.view(torch.int32).bitwise_right_shift(23).to(torch.uint8).view(torch.float8_e8m0fnu)
        return s
    s["w"] = w
    s["dy"] = normal(rows, out).mul_(1e-3).to(kind)
    for name in ("x", "w", "b"):
        if s[name] is not None:
            s[name].requires_grad_(True)
    return s


# ---- plain forms ---------------------------------------------------------------------------------------------

def _power(e):
    """2^e for whole e from -126 to 127, exactly."""
    return (e + 127).bitwise_left_shift(23).view(torch.float32)


def _quantize(x):
    """Codes of whole blocks, and the scales."""
    rows, cols = x.shape
    x = torch.nn.functional.pad(x.float(), (0, -cols % BLOCK, 0, -rows % BLOCK))
    x = x.view(-(-rows // BLOCK), BLOCK, -(-cols // BLOCK), BLOCK)
    top = x.abs().amax((1, 3)).view(torch.int32)
    # 448 is 1.75 2^8
    e = (top.bitwise_right_shift(23) - 135 + (top.bitwise_and(0x7fffff) > 0x600000).int()).clamp_(min=-126)
    codes = (x * _power(-e)[:, None, :, None]).to(torch.float8_e4m3fn)
    return codes.view(codes.shape[0] * BLOCK, -1), _power(e)


def _values(codes, scales):
    rows, cols = codes.shape
    codes = torch.nn.functional.pad(codes.float(), (0, -cols % BLOCK, 0, -rows % BLOCK))
    return (codes.view(scales.shape[0], BLOCK, -1, BLOCK) * scales.float()[:, None, :, None]).view(codes.shape)[:rows, :cols]


def _held(x):
    return _values(*_quantize(x))[:x.shape[0], :x.shape[1]]


def _unpack(codes, scales, signed):
    """The 32-bit values of groups of 8-bit codes."""
    code = codes.view(-1, GROUP).int()
    size = (code.bitwise_and(127) if signed else code).bitwise_left_shift(20).view(torch.float32)
    size = size * 2.0 ** (112 if signed else 96) * _power(scales.int() - 127)[:, None]
    return torch.where(code > 127, -size, size) if signed else size


def _pack(x, bits, signed):
    """Codes and scales of 32-bit values, with the random bits that round them: up where the 20 bits that are left out
    and these come to 2^20 together."""
    x = x.view(-1, GROUP)
    top = x.abs().amax(1).view(torch.int32)
    e = (top.bitwise_right_shift(23) - 127 + (top.bitwise_and(0x7fffff) > 0x600000).int()).clamp_(min=-126)
    size = x.abs() * _power(-e)[:, None] * 2.0 ** (-112 if signed else -96)
    code = (size.view(torch.int32) + bits).bitwise_right_shift(20)
    code = torch.where(x < 0, code + 128, code) if signed else code.clamp_(min=1)
    some = top > 0
    return (code * some[:, None]).to(torch.uint8).view(-1), ((e + 127) * some).to(torch.uint8)


def _mix(x):
    """A 32-bit number from another, by shifts and products modulo 2^32 (held in 64 bits here)."""
    mask = 0xffffffff
    x = x ^ (x >> 16)
    x = x * 0x9e3779b1 & mask
    x = x ^ (x >> 15)
    x = x * 0x85ebca77 & mask
    return x ^ (x >> 16)


def _random(s):
    """32 random bits for each value: from the seed and the step for the call, from that and its place for a tensor, from
    that and the value's index."""
    mask, odd = 0xffffffff, 0x9e3779b9
    call = _mix(s["seed"] + STEP * odd & mask)
    tensor = _mix(call + s["tensor"] * odd & mask)
    at = s["index"][:, None] * GROUP + torch.arange(GROUP, device=s["index"].device)
    return _mix(tensor[:, None] + at & mask)


def _clip(s):
    """(norm of all gradients, what they are multiplied with)."""
    norm = s["g"].double().square().sum().sqrt().float()
    return norm, torch.clamp(torch.full_like(norm, MAX_NORM) / (norm + 1e-6), max=1.0)


def _adamw_plain(s):
    case = s["case"]
    g, norm = s["g"].float(), None
    if case["clip"]:
        norm, factor = _clip(s)
        g = g * factor
    if case["bits"] == 8:
        m, v = _unpack(s["m_codes"], s["m_scales"], True).view(-1), _unpack(s["v_codes"], s["v_scales"], False).view(-1)
    else:
        m, v = s["m"], s["v"]
    m = m * BETAS[0] + g * (1 - BETAS[0])
    v = v * BETAS[1] + g * (1 - BETAS[1]) * g
    root = v.sqrt() * (1 / math.sqrt(1 - BETAS[1] ** STEP)) + EPS
    p = s["p"].float() * (1 - LR * DECAY) - m / root * (LR / (1 - BETAS[0] ** STEP))
    s["p"].copy_(p)
    if case["copy"]:
        s["copy"].copy_(p)
    if case["bits"] == 8:
        bits = _random(s)
        # a tensor's last group is as long as the tensor
        inside = torch.arange(GROUP, device=m.device) < s["left"][:, None]
        for name, t, b, signed in (("m", m, bits >> 16, True), ("v", v, bits & 0xffff, False)):
            codes, scales = _pack(t, (b * 16 + 8).int(), signed)
            s[name + "_codes"].copy_(codes * inside.view(-1))
            s[name + "_scales"].copy_(scales)
            s[name].copy_(_unpack(s[name + "_codes"], scales, signed).view(-1))
    else:
        s["m"].copy_(m)
        s["v"].copy_(v)
    return norm


def _run_plain(s):
    case = s["case"]
    if case["op"] == "adamw":
        return (s["p"], s["copy"], s["m"], s["v"], _adamw_plain(s))
    kind = s["x"].dtype
    x = s["x"].detach()
    if case["op"] == "quantize":
        return _held(x).to(kind), x.float().sum(0)
    w = _values(s["codes"], s["scales"]) if case["op"] == "linear" else _held(s["w"].detach())
    x = _held(x)
    y = torch.matmul(x, w.t())
    if s["b"] is not None:
        y += s["b"].detach().float()
    if case["op"] == "linear":
        return y.to(kind)
    dy = _held(s["dy"])
    db = s["dy"].float().sum(0).to(kind) if s["b"] is not None else None
    return y.to(kind), torch.matmul(dy, w).to(kind), torch.matmul(dy.t(), x).to(kind), db


# ---- the framework's operators --------------------------------------------------------------------------------

def _adamw_own(cs, s):
    case = s["case"]
    norm = cs.gradient_norm(s["gs"]) if case["clip"] else None
    rest = dict(lr=LR, betas=BETAS, eps=EPS, weight_decay=DECAY, norm=norm, max_norm=MAX_NORM, copies=s["copies"])
    if case["bits"] == 32:
        cs.adamw_step(s["ps"], s["gs"], s["ms"], s["vs"], STEP, **rest)
    else:
        cs.adamw8_step(s["ps"], s["gs"], s["states"], STEP, seed=s["seed"], **rest)
        cs.adamw8_unpack(s["states"], s["ms"], s["vs"])
    return norm


def _run_own(s):
    import cswap_b200 as cs

    case = s["case"]
    if case["op"] == "adamw":
        return (s["p"], s["copy"], s["m"], s["v"], _adamw_own(cs, s))
    if case["op"] == "quantize":
        codes, scales, sums = cs.fp8_quantize(s["x"], sums=True)
        return cs.fp8_dequantize(codes, scales, dtype=s["x"].dtype), sums
    if case["op"] == "linear":
        return cs.fp8_linear(s["x"], (s["codes"], s["scales"]), s["b"])
    y = cs.fp8_linear(s["x"], s["w"], s["b"])
    leaves = [s["x"], s["w"]] + ([s["b"]] if s["b"] is not None else [])
    grads = torch.autograd.grad(y, leaves, s["dy"])
    return (y,) + grads if s["b"] is not None else (y,) + grads + (None,)


def run(s):
    return _run_own(s) if own else _run_plain(s)


# ---- what a pass cannot do without -----------------------------------------------------------------------------

def work(case):
    """Inputs read once and outputs written once, the averages in 32 bits among them where they are handed out."""
    e = BYTES[case["type"]]
    if case["op"] == "adamw":
        n = sum(_sizes(case))
        state = 16 if case["bits"] == 32 else 4 * (1 + 1 / GROUP) + 8
        clip = BYTES[case["grad"]] if case["clip"] else 0  # the norm is known before the first value is changed
        return {"bytes": n * (2 * e + BYTES[case["grad"]] + clip + BYTES[case["copy"]] + state), "flops": 16 * n}
    rows, cols = case["rows"], case["cols"]
    if case["op"] == "quantize":  # there and back
        return {"bytes": rows * cols * (2 * e + 2) + 4 * cols, "flops": 4 * rows * cols}
    out = case["out"]
    bias = out * e if case["bias"] else 0
    product = 2 * rows * cols * out
    if case["op"] == "linear":
        return {"bytes": e * rows * (cols + out) + cols * out + bias, "flops": product}
    return {"bytes": e * (2 * rows * cols + 2 * rows * out + 2 * cols * out) + 2 * bias, "flops": 3 * product}


# ---- the definitions in 64 bits --------------------------------------------------------------------------------

def _near(t, bits, least):
    """t >= 0 to the nearest number of `bits` bits of mantissa whose last one stands for 2^least at least."""
    _, e = torch.frexp(t)  # t = f 2^e, f in 1/2 ... 1
    unit = torch.ldexp(torch.ones_like(t), (e - 1 - bits).clamp(min=least))
    return torch.round(t / unit) * unit


def _power_above(t):
    """The least power of two that is not below t."""
    f, e = torch.frexp(t)
    return torch.ldexp(torch.ones_like(t), torch.where(f == 0.5, e - 1, e))


def _exact_held(x):
    rows, cols = x.shape
    wide = torch.zeros(-(-rows // BLOCK) * BLOCK, -(-cols // BLOCK) * BLOCK, dtype=torch.float64, device=x.device)
    wide[:rows, :cols] = x.detach().double()
    blocks = wide.unflatten(0, (-1, BLOCK)).unflatten(2, (-1, BLOCK))
    top = blocks.abs().amax((1, 3), keepdim=True)
    scale = _power_above((top / 448).clamp(min=2.0 ** -126))
    held = _near(blocks.abs() / scale, 3, -9) * scale * blocks.sign()
    return held.flatten(2, 3).flatten(0, 1)[:rows, :cols]


def _exact_codes(x, bits, exponents):
    """The values that groups of 32-bit numbers are held as: by their definition with quanta, not by their bits."""
    x = x.double()
    top = x.abs().amax(1, keepdim=True)
    scale = _power_above((top / 1.75).clamp(min=2.0 ** -126))
    t = x.abs() / scale
    least = 2 - 2 ** exponents  # the exponent of the numbers that have no leading one
    _, e = torch.frexp(t)
    unit = torch.ldexp(torch.ones_like(t), (e - 1).clamp(min=least) - 3)
    whole = torch.round(t / unit * 2.0 ** 20)  # small numbers are rounded to 32 bits in front of it
    code = torch.floor((whole + bits) * 2.0 ** -20)
    if exponents == 5:
        code = torch.where((code == 0) & (top > 0), torch.ones_like(code), code)
        unit = torch.where(t == 0, torch.full_like(unit, 2.0 ** (least - 3)), unit)
    return code * unit * scale * x.sign().where(x != 0, torch.ones_like(x))


def _exact_adamw(case, seed):
    s = prepare(case, seed)
    g, norm = s["g"].double(), None
    if case["clip"]:
        norm = torch.linalg.vector_norm(g)
        g = g * min(1.0, MAX_NORM / (float(norm) + 1e-6))
    m, v = s["m"].double(), s["v"].double()
    if case["bits"] == 8:
        m = _unpack(s["m_codes"], s["m_scales"], True).double().view(-1)
        v = _unpack(s["v_codes"], s["v_scales"], False).double().view(-1)
    wide_m, wide_v = BETAS[0] * m + (1 - BETAS[0]) * g, BETAS[1] * v + (1 - BETAS[1]) * g * g
    m_hat, v_hat = wide_m / (1 - BETAS[0] ** STEP), wide_v / (1 - BETAS[1] ** STEP)
    p = s["p"].double() * (1 - LR * DECAY) - LR * m_hat / (v_hat.sqrt() + EPS)
    copy = p if case["copy"] else None
    if case["bits"] == 32:
        return p, copy, wide_m, wide_v, norm
    # The format takes the averages as 32-bit operations leave them, products and sums rounded one by one.
    to = torch.float32
    c = (torch.tensor(MAX_NORM) / (norm.to(to).cpu() + 1e-6)).clamp(max=1.0).to(g.device) if case["clip"] else None
    step = s["g"].to(to) if c is None else (s["g"].double() * c.double()).to(to)
    b1, rest1, b2, rest2 = (torch.tensor(b, dtype=to).double().to(g.device)
                            for b in (BETAS[0], 1 - BETAS[0], BETAS[1], 1 - BETAS[1]))
    m = ((m * b1).to(to).double() + (step.double() * rest1).to(to).double()).to(to)
    v = ((v * b2).to(to).double() + ((step.double() * rest2).to(to).double() * step.double()).to(to).double()).to(to)
    bits = _random(s)
    keep = (torch.arange(GROUP, device=g.device) < s["left"][:, None]).double()
    m = _exact_codes(m.view(-1, GROUP), (bits >> 16) * 16 + 8, 4) * keep
    v = _exact_codes(v.view(-1, GROUP), (bits & 0xffff) * 16 + 8, 5) * keep
    return p, copy, m.view(-1), v.view(-1), norm


def exact(case, seed):
    if case["op"] == "adamw":
        return _exact_adamw(case, seed)
    s = prepare(case, seed)
    x = _exact_held(s["x"])
    if case["op"] == "quantize":
        return x, s["x"].double().sum(0)
    if case["op"] == "linear":
        w = s["codes"].float().double()
        scale = s["scales"].float().double().repeat_interleave(BLOCK, 0).repeat_interleave(BLOCK, 1)
        w = w * scale[:w.shape[0], :w.shape[1]]
    else:
        w = _exact_held(s["w"])
    y = torch.einsum("rc,oc->ro", x, w)
    if s["b"] is not None:
        y = y + s["b"].detach().double()
    if case["op"] == "linear":
        return y
    dy = _exact_held(s["dy"])
    db = torch.einsum("ro->o", s["dy"].double()) if s["b"] is not None else None
    return y, torch.einsum("ro,oc->rc", dy, w), torch.einsum("ro,rc->oc", dy, x), db
