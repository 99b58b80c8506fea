"""The operators of a training step that saves little for backward, as timed passes through their entry points.

Kinds of pass ("op"):

  q8         a tensor into its 8-bit checkpoint and back: groups of 128 values, m = max |x|, scale m / 127, code
             rint(x * (127 / m)), each step in 32 bits; a group below 2^-120 is held as zeros.
  gelu       y = x Phi(x) with x kept as an 8-bit checkpoint; backward on the checkpoint: the gradient, and y once more
             for the weight gradient of the product behind it.
  ln_fwd     layer norm of the sum of two tensors: y, the sum, and each row's mean and 1 / standard deviation.
  ln_bwd     its backward pass: gradients of the sum, the weight (summed over rows) and the bias.
  ln         both in a row.
  attn_fwd   softmax(scale Q K^T) V and the logarithm of each row's sum of exponentials.
  attn       that and its backward pass, which forms the probabilities again.

Sizes: the token matrices of a BERT-base-shaped encoder at batch 32 x 512 (hidden 768, 12 heads of 64), longer causal
sequences whose heads share keys and values, and small and ragged ones of each kind.
"""
import math

import torch

import numpy as np

own = False

TYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
BYTES = {"fp32": 4, "bf16": 2, "fp16": 2}
GROUP = 128


def listed():
    return [
        # a short sentence's hidden states, [77, 768]: a call is launch latency
        {"name": "q8_tokens_bf16", "op": "q8", "type": "bf16", "numel": 77 * 768},
        # the feed-forward activation of the encoder at batch 32 x 512
        {"name": "q8_ffn_fp32", "op": "q8", "type": "fp32", "numel": 50331648},
        # the same activation through GELU and back
        {"name": "gelu_ffn_fp32", "op": "gelu", "type": "fp32", "numel": 50331648},
        # a ragged half-precision activation
        {"name": "gelu_ragged_fp16", "op": "gelu", "type": "fp16", "numel": 1000003},
        # the encoder's residual sum and norm, [32 * 512, 768]
        {"name": "ln_fwd_hidden_fp32", "op": "ln_fwd", "type": "fp32", "rows": 16384, "cols": 768},
        # a wide model's backward pass
        {"name": "ln_bwd_wide_bf16", "op": "ln_bwd", "type": "bf16", "rows": 16384, "cols": 4096},
        # one sentence of the encoder, there and back
        {"name": "ln_tokens_fp32", "op": "ln", "type": "fp32", "rows": 77, "cols": 768},
        # rows that are no multiple of anything
        {"name": "ln_ragged_bf16", "op": "ln", "type": "bf16", "rows": 4099, "cols": 1001},
        # the encoder's attention over padded sentences: forward alone, as in evaluation
        {"name": "attn_fwd_encoder_bf16", "op": "attn_fwd", "type": "bf16", "batch": 32, "heads": 12, "kv_heads": 12,
         "q_len": 512, "k_len": 512, "dim": 64, "causal": False, "padded": True},
        # and a training step's use of it
        {"name": "attn_encoder_bf16", "op": "attn", "type": "bf16", "batch": 32, "heads": 12, "kv_heads": 12,
         "q_len": 512, "k_len": 512, "dim": 64, "causal": False, "padded": True},
        # a long causal sequence, four heads to a key head
        {"name": "attn_causal_long_bf16", "op": "attn", "type": "bf16", "batch": 1, "heads": 32, "kv_heads": 8,
         "q_len": 4096, "k_len": 4096, "dim": 128, "causal": True, "padded": False},
        # a short ragged one: the last 37 of 113 tokens, heads of 40
        {"name": "attn_ragged_fp16", "op": "attn", "type": "fp16", "batch": 2, "heads": 6, "kv_heads": 3,
         "q_len": 37, "k_len": 113, "dim": 40, "causal": True, "padded": True},
    ]


def _log_between(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["q8", "gelu", "ln_fwd", "ln_bwd", "ln", "attn_fwd", "attn", "attn"])
    if op in ("q8", "gelu"):
        return {"op": op, "type": rng.choice(["fp32", "bf16", "fp16"]), "numel": _log_between(rng, 1, 50331648)}
    if op.startswith("ln"):
        kind = rng.choice(["fp32", "bf16", "fp16"])
        cols = _log_between(rng, 8, 16384)
        # no more elements than the widest listed case, less where both directions run
        most = (1 << 26) // (BYTES[kind] // 2) // (2 if op == "ln" else 1)
        return {"op": op, "type": kind, "rows": _log_between(rng, 1, max(1, most // cols)), "cols": cols}
    kv_heads = rng.choice([1, 2, 3, 4, 8])
    share = rng.choice([1, 1, 2, 4])
    k_len = _log_between(rng, 1, 4096)
    q_len = k_len if rng.random() < 0.6 else _log_between(rng, 1, 4096)
    # no more pairs than half of the long listed case's square, all heads together
    most = 32 * 4096 * 4096 // 2
    batch = max(1, min(rng.choice([1, 2, 5, 8, 16]), most // (kv_heads * share * q_len * k_len)))
    return {"op": op, "type": rng.choice(["bf16", "fp16"]), "batch": batch, "heads": kv_heads * share,
            "kv_heads": kv_heads, "q_len": q_len, "k_len": k_len, "dim": rng.choice([32, 40, 64, 80, 96, 128]),
            "causal": rng.random() < 0.5, "padded": rng.random() < 0.4}


def prepare(case, seed):
    op, dtype = case["op"], TYPES[case["type"]]
    gen = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape):
        return torch.randn(*shape, generator=gen, device="cuda")

    s = {"case": case}
    if op in ("q8", "gelu"):
        # what a linear layer puts out: normal, some channels larger than others
        n = case["numel"]
        s["x"] = normal(n).mul_(torch.rand(n, generator=gen, device="cuda").add_(0.5)).to(dtype)
        if op == "gelu":
            s["dy"] = normal(n).to(dtype)
        return s
    if op.startswith("ln"):
        rows, cols = case["rows"], case["cols"]
        x = normal(rows, cols).add_(0.25 * normal(cols)).to(dtype)
        s["weight"] = normal(cols).mul_(0.1).add_(1.0).to(dtype)
        s["bias"] = normal(cols).mul_(0.1).to(dtype)
        if op != "ln_bwd":
            s["residual"] = normal(rows, cols).to(dtype)
        if op != "ln_fwd":
            s["dy"] = normal(rows, cols).to(dtype)
        s["x"] = x
        if op == "ln_bwd":  # what the forward pass left
            wide = x.float()
            s["mean"] = wide.mean(1)
            s["rstd"] = torch.rsqrt((wide - s["mean"][:, None]).square_().mean(1) + 1e-5)
        return s
    b, h, hk, d = case["batch"], case["heads"], case["kv_heads"], case["dim"]
    # heads split out of a projection's rows: [batch, tokens, heads, dim], seen with the heads in front
    s["q"] = normal(b, case["q_len"], h, d).to(dtype).transpose(1, 2)
    s["k"] = normal(b, case["k_len"], hk, d).to(dtype).transpose(1, 2)
    s["v"] = normal(b, case["k_len"], hk, d).to(dtype).transpose(1, 2)
    if op == "attn":
        s["do"] = normal(b, case["q_len"], h, d).to(dtype).transpose(1, 2)
    s["lens"] = None
    if case["padded"]:  # sentences from a quarter of the row to all of it
        least = max(1, case["k_len"] // 4)
        s["lens"] = torch.randint(least, case["k_len"] + 1, (b,), generator=gen, device="cuda", dtype=torch.int32)
    return s


# ---- plain forms ---------------------------------------------------------------------------------------------

def _q8_plain(x):
    n = x.numel()
    x = torch.nn.functional.pad(x.float(), (0, -n % GROUP)).view(-1, GROUP)
    top = x.abs().amax(1, keepdim=True)
    held = top >= 2.0 ** -120
    # divisors are tensors: a division by a number is computed as a product with its reciprocal
    largest = torch.full_like(top, 127.0)
    scale = torch.where(held, top / largest, torch.zeros_like(top))
    inverse = torch.where(held, largest / top, torch.zeros_like(top))
    return (torch.round(x * inverse) * scale).view(-1)[:n]


def _phi(x):  # the normal distribution's sum and density
    return 0.5 * torch.erfc(x * -math.sqrt(0.5)), torch.exp(-0.5 * x * x) * (1.0 / math.sqrt(2.0 * math.pi))


def _gelu_plain(x, dy):
    kind = x.dtype
    x32 = x.float()
    held = _q8_plain(x)
    total, density = _phi(held)
    return ((x32 * _phi(x32)[0]).to(kind), held.to(kind), (dy.float() * (total + held * density)).to(kind),
            (held * total).to(kind))


def _ln_forward_plain(x, residual, weight, bias):
    total = (x.float() + residual.float()).to(x.dtype)
    wide = total.float()
    mean = wide.mean(1)
    centred = wide - mean[:, None]
    rstd = torch.rsqrt(centred.square().mean(1) + 1e-5)
    y = centred * rstd[:, None] * weight.float() + bias.float()
    return y.to(x.dtype), total, mean, rstd


def _ln_backward_plain(dy, x, mean, rstd, weight):
    g = dy.float()
    normed = (x.float() - mean[:, None]) * rstd[:, None]
    gw = g * weight.float()
    dx = (gw - gw.mean(1, keepdim=True) - normed * (gw * normed).mean(1, keepdim=True)) * rstd[:, None]
    return dx.to(x.dtype), (g * normed).sum(0).to(weight.dtype), g.sum(0).to(weight.dtype)


def _mask(case, lens, device):
    """True where a query may look: [batch or 1, 1, q_len, k_len].  The last query stands at the last key."""
    keys = torch.arange(case["k_len"], device=device)
    seen = torch.ones(1, 1, case["q_len"], case["k_len"], dtype=torch.bool, device=device)
    if case["causal"]:
        rows = torch.arange(case["q_len"], device=device) + (case["k_len"] - case["q_len"])
        seen = seen & (keys[None, :] <= rows[:, None])
    if lens is not None:
        seen = seen & (keys[None, :] < lens[:, None].long())[:, None, None, :]
    return seen


def _attn_plain(s):
    case = s["case"]
    kind = s["q"].dtype
    share = case["heads"] // case["kv_heads"]
    scale = 1.0 / math.sqrt(case["dim"])
    b, hk, kl, d = s["k"].shape
    q, k, v = s["q"].float(), s["k"].float(), s["v"].float()
    if share > 1:
        k, v = k.repeat_interleave(share, 1), v.repeat_interleave(share, 1)
    scores = torch.matmul(q, k.transpose(2, 3)).mul_(scale)
    scores.masked_fill_(~_mask(case, s["lens"], q.device), float("-inf"))
    top = scores.amax(3, keepdim=True)
    top.masked_fill_(top == float("-inf"), 0.0)
    p = scores.sub_(top).exp_()
    total = p.sum(3, keepdim=True)
    lse = (total.log() + top).squeeze(3)
    p.div_(torch.where(total == 0, torch.ones_like(total), total))
    o = torch.matmul(p, v)
    if case["op"] == "attn_fwd":
        return o.to(kind), lse
    do = s["do"].float()
    dv = torch.matmul(p.transpose(2, 3), do)
    dot = (do * o).sum(3, keepdim=True)
    ds = torch.matmul(do, v.transpose(2, 3)).sub_(dot).mul_(p).mul_(scale)
    dq = torch.matmul(ds, k)
    dk = torch.matmul(ds.transpose(2, 3), q)
    if share > 1:
        dk, dv = dk.view(b, hk, share, kl, d).sum(2), dv.view(b, hk, share, kl, d).sum(2)
    return o.to(kind), lse, dq.to(kind), dk.to(kind), dv.to(kind)


def _run_plain(s):
    op = s["case"]["op"]
    if op == "q8":
        return _q8_plain(s["x"]).to(s["x"].dtype)
    if op == "gelu":
        return _gelu_plain(s["x"], s["dy"])
    if op == "ln_fwd":
        return _ln_forward_plain(s["x"], s["residual"], s["weight"], s["bias"])
    if op == "ln_bwd":
        return _ln_backward_plain(s["dy"], s["x"], s["mean"], s["rstd"], s["weight"])
    if op == "ln":
        y, total, mean, rstd = _ln_forward_plain(s["x"], s["residual"], s["weight"], s["bias"])
        return (y, total, mean, rstd) + _ln_backward_plain(s["dy"], total, mean, rstd, s["weight"])
    return _attn_plain(s)


# ---- the framework's operators --------------------------------------------------------------------------------

def _run_own(s):
    import cswap_b200 as cs

    case = s["case"]
    op = case["op"]
    if op == "q8":
        packed = cs.q8_compress(s["x"])
        return cs.q8_decompress(packed, case["numel"], dtype=s["x"].dtype)
    if op == "gelu":
        y, packed = cs.gelu_forward(s["x"])
        dx, again = cs.gelu_backward(s["dy"], packed, recompute=True)
        return y, cs.q8_decompress(packed, case["numel"], dtype=s["x"].dtype), dx, again
    if op == "ln_fwd":
        return cs.layer_norm_forward(s["x"], s["weight"], s["bias"], 1e-5, s["residual"])
    if op == "ln_bwd":
        return cs.layer_norm_backward(s["dy"], s["x"], s["mean"], s["rstd"], s["weight"])
    if op == "ln":
        y, total, mean, rstd = cs.layer_norm_forward(s["x"], s["weight"], s["bias"], 1e-5, s["residual"])
        return (y, total, mean, rstd) + tuple(cs.layer_norm_backward(s["dy"], total, mean, rstd, s["weight"]))
    o, lse = cs.attention_forward(s["q"], s["k"], s["v"], causal=case["causal"], kv_lens=s["lens"])
    if op == "attn_fwd":
        return o, lse
    return (o, lse) + tuple(cs.attention_backward(s["do"], s["q"], s["k"], s["v"], o, lse, causal=case["causal"],
                                                  kv_lens=s["lens"]))


def run(s):
    return _run_own(s) if own else _run_plain(s)


# ---- what a pass cannot do without -----------------------------------------------------------------------------

def work(case):
    """Inputs read once and outputs written once; products of the pairs that the masks leave (padding by its mean)."""
    op, e = case["op"], BYTES[case["type"]]
    if op in ("q8", "gelu"):
        n = case["numel"]
        packed = n + 4 * -(-n // GROUP)
        if op == "q8":  # there and back
            return {"bytes": 2 * (e * n + packed), "flops": 4 * n}
        # x, y, packed; packed, dy, dx, y; packed, the values that it stands for
        return {"bytes": (2 * e * n + packed) + (3 * e * n + packed) + (e * n + packed), "flops": 40 * n}
    if op.startswith("ln"):
        n, r, c = case["rows"] * case["cols"], case["rows"], case["cols"]
        forward = 4 * e * n + 8 * r + 2 * e * c
        backward = 3 * e * n + 8 * r + 3 * e * c
        b = {"ln_fwd": forward, "ln_bwd": backward, "ln": forward + backward}[op]
        f = {"ln_fwd": 8 * n, "ln_bwd": 14 * n, "ln": 22 * n}[op]
        return {"bytes": b, "flops": f}
    ql, kl, d = case["q_len"], case["k_len"], case["dim"]
    least = max(1, kl // 4)
    keys = int(round((least + kl) / 2)) if case["padded"] else kl
    pairs = ql * keys
    if case["causal"]:
        pairs = sum(min(max(kl - ql + i + 1, 0), keys) for i in range(ql))
    q = case["batch"] * case["heads"] * ql * d * e
    kv = case["batch"] * case["kv_heads"] * kl * d * e
    lse = 4 * case["batch"] * case["heads"] * ql
    product = 2 * case["batch"] * case["heads"] * pairs * d
    forward = {"bytes": 2 * q + 2 * kv + lse, "flops": 2 * product}
    if op == "attn_fwd":
        return forward
    return {"bytes": forward["bytes"] + 4 * q + 4 * kv + lse, "flops": forward["flops"] + 5 * product}


# ---- the definitions in 64 bits --------------------------------------------------------------------------------

def _exact_q8(x):
    """The format defines its codes by 32-bit steps; the values they stand for follow in 64."""
    flat = x.float().cpu().numpy()
    n = flat.size
    padded = np.zeros(-(-n // GROUP) * GROUP, dtype=np.float32)
    padded[:n] = flat
    groups = padded.reshape(-1, GROUP)
    top = np.max(np.abs(groups), axis=1, keepdims=True)
    safe = np.where(top >= np.float32(2.0 ** -120), top, np.float32(1.0))
    live = (top >= np.float32(2.0 ** -120)).astype(np.float32)
    codes = np.rint(groups * (np.float32(127.0) / safe) * live)
    values = codes.astype(np.float64) * (safe / np.float32(127.0) * live).astype(np.float64)
    return torch.from_numpy(values.reshape(-1)[:n]).to(x.device)


def _normal_sum(x):
    return torch.special.ndtr(x)


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "q8":
        return _exact_q8(s["x"])
    if op == "gelu":
        x, held, dy = s["x"].double(), _exact_q8(s["x"]), s["dy"].double()
        slope = _normal_sum(held) + held * torch.exp(-held.square() / 2) / math.sqrt(2 * math.pi)
        return x * _normal_sum(x), held, dy * slope, held * _normal_sum(held)
    if op.startswith("ln"):
        weight = s["weight"].double()
        out = ()
        if op == "ln_bwd":
            total, mean, rstd = s["x"].double(), s["mean"].double()[:, None], s["rstd"].double()[:, None]
        else:
            # the sum is held in the inputs' type, and normed as it is held
            total = (s["x"].double() + s["residual"].double()).to(s["x"].dtype).double()
            var, mean = torch.var_mean(total, dim=1, unbiased=False, keepdim=True)
            rstd = (var + 1e-5).pow(-0.5)
            out = ((total - mean) * rstd * weight + s["bias"].double(), total, mean[:, 0], rstd[:, 0])
        if op == "ln_fwd":
            return out
        dy = s["dy"].double()
        normed = (total - mean) * rstd
        c = case["cols"]
        inner = dy * weight
        dx = rstd / c * (c * inner - inner.sum(1, keepdim=True) - normed * (inner * normed).sum(1, keepdim=True))
        return out + (dx, torch.einsum("rc,rc->c", dy, normed), dy.sum(0))
    if case["batch"] * case["heads"] * case["q_len"] * case["k_len"] > 32 * 4096 * 4096:
        return None
    share = case["heads"] // case["kv_heads"]
    scale = case["dim"] ** -0.5
    q, k, v = s["q"].double(), s["k"].double(), s["v"].double()
    do = s["do"].double() if op == "attn" else None
    o, lse = torch.empty_like(q), torch.empty(q.shape[:3], dtype=torch.float64, device=q.device)
    dq, dk, dv = torch.zeros_like(q), torch.zeros_like(k), torch.zeros_like(v)
    i = torch.arange(case["q_len"], device=q.device)[:, None] + case["k_len"] - case["q_len"]
    j = torch.arange(case["k_len"], device=q.device)[None, :]
    for b in range(case["batch"]):
        hidden = torch.zeros(case["q_len"], case["k_len"], dtype=torch.bool, device=q.device)
        if case["causal"]:
            hidden = hidden | (j > i)
        if s["lens"] is not None:
            hidden = hidden | (j >= s["lens"][b])
        dead = hidden.all(1)
        for h in range(case["heads"]):
            g = h // share
            scores = (q[b, h] @ k[b, g].T * scale).masked_fill(hidden, -math.inf)
            lse[b, h] = torch.logsumexp(scores, 1)
            p = torch.softmax(scores, 1).masked_fill(dead[:, None], 0.0)
            o[b, h] = p @ v[b, g]
            if do is not None:
                slope = do[b, h] @ v[b, g].T
                ds = p * (slope - (p * slope).sum(1, keepdim=True))
                dv[b, g] += p.T @ do[b, h]
                dq[b, h] = ds @ k[b, g] * scale
                dk[b, g] += ds.T @ q[b, h] * scale
    return (o, lse) if do is None else (o, lse, dq, dk, dv)
