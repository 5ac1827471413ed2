"""Attention, the 8-bit cache and logits processing from their definitions, in 64 bits: what the GPU tests compare with."""

import math

import torch


def visible(first: int, rows: int, keys: int, *, causal=True, window=None, prefix=0):
    """bool [rows, keys]: which keys queries first .. first + rows - 1 see."""
    i, j = torch.arange(first, first + rows)[:, None], torch.arange(keys)[None, :]
    seen = torch.ones((rows, keys), dtype=torch.bool)
    if causal:
        seen = (j <= i) | (j < prefix)
    if window:
        seen = seen & ((i - j).abs() < window)
    return seen


def attend(q, k, v, first=0, *, causal=True, window=None, prefix=0, scale=None, softcap=None, slopes=None):
    """q [n, heads, D] at positions first.. over k, v [L, kv, D] -> (output, bound): float64 [n, heads, D], and how far a
    kernel may be off that reads BF16, sums in fp32, rounds its weights to BF16 and its output to BF16.

    The bound, from the formula o = sum p v / sum p, with A = sum p |v| (p normalised):
      output rounded to BF16                         2^-8 |o|
      each weight rounded to BF16, 2^-8 p            2^-8 A
      a score off by d: a weight off by 2 d          4 d A (numerator and normalisation)
    d: products are exact in fp32; a sum of D of them in any order, adders that cut included, is off by at most
    D 2^-23 scale sum |q k|; exp2's argument and result, cap, bias and their constants by 2^-20 (1 + |s|)."""
    n, heads, D = q.shape
    L, kv = k.shape[0], k.shape[1]
    group = heads // kv
    scale = 1 / math.sqrt(D) if scale is None else scale
    qd, kd, vd = q.double(), k.double().repeat_interleave(group, 1), v.double().repeat_interleave(group, 1)
    seen = visible(first, n, L, causal=causal, window=window, prefix=prefix).to(q.device)[None]
    s = torch.einsum("nhd,lhd->hnl", qd, kd) * scale
    sums = torch.einsum("nhd,lhd->hnl", qd.abs(), kd.abs()) * abs(scale)
    if softcap:
        s = softcap * torch.tanh(s / softcap)
    if slopes is not None:
        gap = (torch.arange(first, first + n, device=q.device)[:, None] - torch.arange(L, device=q.device)[None, :]).abs()
        s = s - slopes.double()[:, None, None] * gap[None]
    off = D * 2.0**-23 * sums + 2.0**-20 * (1 + s.abs())
    s = s.masked_fill(~seen, -math.inf)
    p = torch.softmax(s, dim=-1)
    p = torch.where(seen.any(-1, keepdim=True), p, torch.zeros_like(p))
    o = torch.einsum("hnl,lhd->nhd", p, vd)
    size = torch.einsum("hnl,lhd->nhd", p, vd.abs())
    d = torch.where(seen & (s > s.amax(-1, keepdim=True) - 40), off, torch.zeros_like(off)).amax(-1)  # a weight below e^-40 carries no error that shows
    return o, 2.0**-8 * o.abs() + (2.0**-8 + 4 * d.T[:, :, None]) * size + 1e-30


def stored(x, kind: str, block: int):
    """Tokens x [n, kv, D] as a cache gives them back, float64."""
    x = x.double()
    out = x.clone()
    for t0 in range(0, x.shape[0] // block * block, block):
        rows = x[t0 : t0 + block]
        finite = torch.where(torch.isfinite(rows), rows, torch.zeros_like(rows))
        most = finite.abs().amax(dim=(0, 2))
        rows = torch.where(torch.isnan(rows), torch.zeros_like(rows), rows)
        if kind == "int8":
            step = (most / torch.full_like(most, 127.0)).float().clamp(min=2.0**-100).double()[None, :, None]  # a tensor: by a number torch multiplies with its reciprocal
            out[t0 : t0 + block] = (rows / step).round().clamp(-127, 127) * step
        else:
            e = torch.tensor([max(-100, math.ceil(math.log2(m / 448))) if m > 0 else -100 for m in most.tolist()], dtype=torch.float64, device=x.device)
            step = torch.exp2(e)[None, :, None]
            y = (rows / step).clamp(-448, 448)
            grid = torch.exp2(torch.floor(torch.log2(y.abs().clamp(min=2.0**-30))).clamp(min=-6) - 3)
            out[t0 : t0 + block] = (y / grid).round() * grid * step
    return out


def logits(x, seen, counts, repetition, presence, frequency, bias=None, mask=None):
    """float64 logits under the rules; seen and counts [batch, vocab]; mask bool or None."""
    x = x.double()
    r = repetition.double()[:, None]
    x = torch.where(seen, torch.where(x > 0, x / r, x * r), x)
    x = x - (frequency.double()[:, None] * counts + presence.double()[:, None] * (counts > 0))
    if bias is not None:
        x = x + bias.double()
    return x if mask is None else x.masked_fill(~mask, -math.inf)
