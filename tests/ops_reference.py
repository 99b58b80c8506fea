"""The training operators in 64 bits (torch, on any device), and how far a kernel may be off them.

A result that is rounded to a type is off by at most U[type] of its value, half a step.  What an operator rounds on the
way adds its own share; E32 stands for what sums in float32 leave, relative to the sum of magnitudes."""
import math

import numpy as np
import torch

U = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}


def close(got, want, bound):
    """|got - want| <= bound, elementwise; equal infinities are close."""
    got = got.double()
    same = got == want
    worst = ((got - want).abs() - bound).masked_fill(same, -1.0)
    assert not torch.isnan(got).logical_and(~torch.isnan(want)).any(), "NaN where a number belongs"
    assert worst.numel() == 0 or float(worst.max()) <= 0, f"off by {float(worst.max()):.3e} more than allowed"


def q8(x):
    """(codes as float64, scales, the values held) by the format's float32 steps."""
    flat = x.detach().float().cpu().numpy().reshape(-1)
    n = flat.size
    groups = np.zeros(-(-n // 128) * 128, dtype=np.float32)
    groups[:n] = flat
    groups = groups.reshape(-1, 128)
    with np.errstate(all="ignore"):
        top = np.abs(groups).max(axis=1, keepdims=True)
        scale = (top / np.float32(127)).astype(np.float32)
        inverse = (np.float32(127) / top).astype(np.float32)
        tiny = top < np.float32(2.0 ** -120)
        bad = ~np.isfinite(top)
        scale = np.where(tiny, np.float32(0), np.where(bad, np.float32(np.nan), scale))
        codes = np.rint(groups * np.where(tiny | bad, np.float32(0), inverse))
        codes = np.where(np.isnan(codes), np.float32(0), codes)
        values = (codes.astype(np.float32) * scale).astype(np.float32)
    pick = lambda a: torch.from_numpy(np.ascontiguousarray(a.reshape(-1)[:n]))
    return pick(codes), torch.from_numpy(scale.reshape(-1)), pick(values)


def phi(x):
    return torch.special.ndtr(x)


def density(x):
    return torch.exp(-0.5 * x * x) / math.sqrt(2 * math.pi)


def layer_norm(x, weight, bias, eps):
    """(y, mean, rstd, normed) of float64 rows."""
    mean = x.mean(-1, keepdim=True)
    rstd = 1 / torch.sqrt((x - mean).square().mean(-1, keepdim=True) + eps)
    h = (x - mean) * rstd
    y = h
    if weight is not None:
        y = y * weight
    if bias is not None:
        y = y + bias
    return y, mean.squeeze(-1), rstd.squeeze(-1), h


def layer_norm_grads(dy, h, rstd, weight):
    g = dy * weight if weight is not None else dy
    dx = rstd[..., None] * (g - g.mean(-1, keepdim=True) - h * (g * h).mean(-1, keepdim=True))
    flat = lambda t: t.reshape(-1, t.shape[-1])
    return dx, flat(dy * h).sum(0), flat(dy).sum(0)


def seen(q_len, k_len, causal, lens, device):
    """[batch or 1, 1, q_len, k_len], True where a query sees a key."""
    j = torch.arange(k_len, device=device)
    m = torch.ones(1, 1, q_len, k_len, dtype=torch.bool, device=device)
    if causal:
        i = torch.arange(q_len, device=device) + k_len - q_len
        m = m & (j[None, :] <= i[:, None])
    if lens is not None:
        m = m & (j[None, :] < lens.long()[:, None])[:, None, None, :]
    return m


class Attention:
    """Forward and backward of float64 copies of the operands, with the bounds of a kernel that rounds the
    probabilities and the scores' gradients to the operands' type before their products."""

    def __init__(self, q, k, v, do, causal, lens, scale):
        kind = q.dtype
        u = U[kind]
        share = q.shape[1] // k.shape[1]
        mask = seen(q.shape[2], k.shape[2], causal, lens, q.device)
        widen = lambda t: t.detach().double()
        Q, K, V, DO = widen(q), widen(k), widen(v), widen(do)
        if lens is not None:  # what lies behind a sequence counts for nothing, whatever it is
            dead = (torch.arange(k.shape[2], device=k.device)[None, :] >= lens.long()[:, None])[:, None, :, None]
            K, V = K.masked_fill(dead, 0.0), V.masked_fill(dead, 0.0)
        K, V = K.repeat_interleave(share, 1), V.repeat_interleave(share, 1)
        s = (Q @ K.transpose(2, 3) * scale).masked_fill(~mask, -math.inf)
        self.lse = torch.logsumexp(s, 3)
        p = torch.exp(s - self.lse[..., None].masked_fill(self.lse[..., None] == -math.inf, 0.0))
        self.o = p @ V
        dp = DO @ V.transpose(2, 3)
        D = (DO * self.o).sum(3, keepdim=True)
        ds = p * (dp - D)
        group = lambda t: t.view(k.shape[0], k.shape[1], share, k.shape[2], k.shape[3]).sum(2)
        self.dq = ds @ K * scale
        self.dk, self.dv = group(ds.transpose(2, 3) @ Q * scale), group(p.transpose(2, 3) @ DO)
        # a score is a sum of dim products in float32, the larger for its base-2 exponent's rounding
        es = (Q.abs() @ K.abs().transpose(2, 3) * abs(scale)).masked_fill(~mask, 0.0)
        es = es * (2.0 ** -24 * (q.shape[3] + 8)) + 2.0 ** -20
        small = 2.0 ** -25 if kind == torch.float16 else 0.0  # a number below 2^-14 is rounded to steps of 2^-24
        n = mask.sum(3, keepdim=True).clamp(min=1).double() * 2.0 ** -23
        pe = p * (es + es.amax(3, keepdim=True) + n)  # what a probability is off before it is rounded
        self.lse_bound = es.amax(3) + n[..., 0] + self.lse.abs().masked_fill(self.lse == -math.inf, 0.0) * 2.0 ** -22
        self.o_bound = u * self.o.abs() + (u * p + small + pe).masked_fill(~mask, 0.0) @ V.abs() + 2.0 ** -25
        # D is taken with o as it was rounded
        De = (DO.abs() * self.o_bound).sum(3, keepdim=True) + (DO * self.o).abs().sum(3, keepdim=True) * 2.0 ** -16
        dpe = DO.abs() @ V.abs().transpose(2, 3) * (2.0 ** -24 * (q.shape[3] + 8))
        dse = ((u * ds).abs() + small + pe * (dp - D).abs() + p * (De + dpe)).masked_fill(~mask, 0.0)
        dvp = (u * p + small + pe).masked_fill(~mask, 0.0)
        grow = 1 + 2.0 ** -10
        sums = 2.0 ** -24 * (q.shape[2] * share + 16)
        self.dq_bound = u * self.dq.abs() + grow * (dse @ K.abs() + ds.abs() @ K.abs() * n) * abs(scale) + 2.0 ** -25
        self.dk_bound = u * self.dk.abs() + 2.0 ** -25 + grow * group(
            (dse + ds.abs() * sums).transpose(2, 3) @ Q.abs()) * abs(scale)
        self.dv_bound = u * self.dv.abs() + 2.0 ** -25 + grow * group((dvp + p * sums).transpose(2, 3) @ DO.abs())
