"""Operators around the linear layers of a decoder, timed and compared one call at a time: attention
of prompts, attention over a cache held in 8 bits, and what is done to the logits.

`own` false: the operators in their plain form, elementary torch operations in 32 bits. `own` true: the
calls that a program using the package makes. `exact` is the definition in 64 bits.

Values follow what the path meets: keys with a few channels several times larger than the rest, scores
of a few units, logits of a few units with a long tail, prompts whose tokens repeat.
"""

from __future__ import annotations

import math
import random

import torch

own = False

CAPACITY = 64  # a cache's capacity in tokens is a multiple of this in the cases below


def listed() -> list:
    return [
        # A short question as the first call of a conversation: latency. (Llama-class heads.)
        {"name": "prompt_33", "op": "prompt", "tokens": 33, "docs": 1, "heads": 32, "kv": 8, "dim": 128},
        # A long prompt of one sequence.
        {"name": "prompt_8192", "op": "prompt", "tokens": 8192, "docs": 1, "heads": 32, "kv": 8, "dim": 128},
        # Eleven prompts packed without padding, capped scores and a sliding window, heads of 256 (Gemma-class).
        {"name": "prompt_docs_cap_window", "op": "prompt", "tokens": 5003, "docs": 11, "heads": 16, "kv": 8, "dim": 256, "cap": 50.0, "window": 1024},
        # Seven packed documents with a distance bias, each behind a prefix that is seen from everywhere.
        {"name": "prompt_docs_bias_prefix", "op": "prompt", "tokens": 6001, "docs": 7, "heads": 12, "kv": 12, "dim": 64, "bias": True, "prefix": 300},
        # One sequence decoding one token: latency of a step's attention.
        {"name": "decode_1x300", "op": "decode", "batch": 1, "longest": 300, "new": 1, "heads": 32, "kv": 8, "dim": 128, "kind": "int8", "block": 32},
        # One long conversation: all of the card has to work on one sequence.
        {"name": "decode_1x131073", "op": "decode", "batch": 1, "longest": 131073, "new": 1, "heads": 32, "kv": 8, "dim": 128, "kind": "int8", "block": 32},
        # A serving batch of unequal lengths.
        {"name": "decode_64x8192", "op": "decode", "batch": 64, "longest": 8192, "new": 1, "heads": 32, "kv": 8, "dim": 128, "kind": "int8", "block": 64},
        # A draft of three tokens being verified, heads of 256, capped scores and a window, e4m3.
        {"name": "decode_17x4001_cap_window", "op": "decode", "batch": 17, "longest": 4001, "new": 3, "heads": 16, "kv": 8, "dim": 256, "kind": "e4m3", "block": 16, "cap": 50.0, "window": 1024},
        # A further turn of two conversations: a chunk of prompt over what the cache holds.
        {"name": "chunk_2x500x9000", "op": "chunk", "batch": 2, "longest": 9000, "new": 500, "heads": 32, "kv": 8, "dim": 128, "kind": "int8", "block": 32},
        # A prompt's keys and values going into the cache, and the cache read back.
        {"name": "append_4x2000", "op": "append", "batch": 4, "new": 2000, "kv": 8, "dim": 128, "kind": "int8", "block": 32},
        # One sequence's logits with penalties: latency.
        {"name": "logits_1x128256", "op": "logits", "batch": 1, "vocab": 128256, "said": 1000, "type": "bf16", "penalties": True},
        # A batch under grammars, with a shared bias, as sequences are admitted (their prompts counted first).
        {"name": "logits_64x151937_grammar", "op": "logits", "batch": 64, "vocab": 151937, "said": 3000, "type": "fp32", "penalties": True, "bias": True, "grammar": True, "admit": True},
    ]


def _log(rng, lo: int, hi: int) -> int:
    return int(round(lo * (hi / lo) ** rng.random()))


def draw(rng) -> dict:
    op = rng.choice(["prompt", "prompt", "prompt", "decode", "decode", "decode", "chunk", "append", "logits", "logits"])
    dim = rng.choice([64, 128, 128, 256])
    kv = rng.choice([1, 2, 4, 8, 8, 12])
    heads = kv * rng.choice([1, 2, 3, 4, 4, 8])
    case = {"op": op}
    options = {}
    if rng.random() < 0.3:
        options["cap"] = rng.choice([20.0, 30.0, 50.0])
    if rng.random() < 0.3:
        options["window"] = _log(rng, 16, 4096)
    if rng.random() < 0.25:
        options["bias"] = True
    if op == "prompt":
        if rng.random() < 0.3:
            options["prefix"] = _log(rng, 8, 1000)
        elif rng.random() < 0.15:
            options["causal"] = False
        tokens = _log(rng, 1, 8192)
        while tokens * tokens * heads * dim > 8192 * 8192 * 32 * 128 // 2:
            tokens = tokens * 2 // 3
        return {**case, "tokens": tokens, "docs": _log(rng, 1, max(1, min(40, tokens))), "heads": heads, "kv": kv, "dim": dim, **options}
    kind, block = rng.choice(["int8", "int8", "e4m3"]), rng.choice([16, 32, 64])
    if op == "append":
        batch, new = _log(rng, 1, 32), _log(rng, 1, 8192)
        while batch * new * kv * dim > 4 * 2000 * 8 * 128 * 4:
            batch, new = max(1, batch * 2 // 3), max(1, new * 2 // 3)
        return {**case, "batch": batch, "new": new, "kv": kv, "dim": dim, "kind": kind, "block": block}
    if op in ("decode", "chunk"):
        new = rng.choice([1, 1, 1, 2, 5]) if op == "decode" else _log(rng, 17, 1000)
        batch = _log(rng, 1, 64 if op == "decode" else 8)
        longest = _log(rng, 40, 131072 if op == "decode" else 16384) + new
        while batch * longest * kv * dim > 64 * 8192 * 8 * 128 // 2 or (op == "chunk" and batch * longest * new * heads * dim > 2 * 9000 * 500 * 32 * 128):
            longest = longest * 2 // 3
            if longest <= new + 20:
                batch, new, longest = max(1, batch // 2), max(1, new // 2), longest + 20
        return {**case, "batch": batch, "longest": longest, "new": new, "heads": heads, "kv": kv, "dim": dim, "kind": kind, "block": block, **options}
    batch, vocab = _log(rng, 1, 128), _log(rng, 5000, 262144)
    while batch * vocab > 64 * 151937:
        batch = max(1, batch * 2 // 3)
    flags = {k: True for k in ("penalties", "bias", "grammar", "admit") if rng.random() < 0.6}
    return {**case, "batch": batch, "vocab": vocab, "said": _log(rng, 1, 8192), "type": rng.choice(["bf16", "fp32"]), **flags}


# ----------------------------------------------------------------------------- sizes of a case
def _documents(case) -> list:
    """Lengths of a prompt case's documents, unequal, at least one token each."""
    n, total = case["docs"], case["tokens"]
    r = random.Random(f"{n} {total}")
    weights = [0.1 + r.random() ** 2 for _ in range(n)]
    lens = [1 + int((total - n) * w / sum(weights)) for w in weights]
    lens[-1] += total - sum(lens)
    return lens


def _prefixes(case) -> list:
    """The prefix of every document of a prompt case (some longer than their document)."""
    r = random.Random(case["tokens"])
    return [r.randint(0, case["prefix"]) for _ in range(case["docs"])]


def _held(case) -> list:
    """Tokens that the cache holds of every sequence before the call; the first sequence ends, with the
    new tokens, at the longest length. Decoding: no block of tokens fills up in the call, so that it can
    be repeated without moving on."""
    n, new, block = case["batch"], case["new"], case["block"]
    r = random.Random(f"{n} {case['longest']}")
    lens = []
    for i in range(n):
        held = case["longest"] - new if i == 0 else max(0, int((case["longest"] - new) * (0.05 + 0.95 * r.random())))
        if case["op"] == "decode" and held % block + new >= block:
            held -= held % block
        lens.append(held)
    return lens


def _capacity(case) -> int:
    need = case["longest"] if "longest" in case else case["new"]
    return -(-need // CAPACITY) * CAPACITY


def _scale(case) -> float:
    return 1.0 / math.sqrt(case["dim"])


def _pairs(case) -> int:
    """Visible (query, key) pairs of one head, over all documents or sequences of the case."""
    window = case.get("window") or (1 << 40)
    total = 0
    if case["op"] == "prompt":
        lens = _documents(case)
        prefixes = _prefixes(case) if "prefix" in case else [0] * len(lens)
        spans = [(0, n, n, p) for n, p in zip(lens, prefixes)]
    else:
        spans = [(held, case["new"], held + case["new"], 0) for held in _held(case)]
    for first, rows, keys, prefix in spans:
        i = torch.arange(first, first + rows, dtype=torch.int64)
        lo = (i - window + 1).clamp(min=0)
        hi = torch.full_like(i, keys) if case.get("causal") is False else (i + 1).clamp(min=prefix).clamp(max=keys)
        total += int((torch.minimum(hi, i + window) - lo).sum())
    return total


def work(case) -> dict:
    if case["op"] == "logits":
        cells = case["batch"] * case["vocab"]
        size = (2 if case["type"] == "bf16" else 4) + 4  # logits in, logits out
        total = cells * size + 8 * case["batch"]
        total += cells // 8 * bool(case.get("grammar")) + 4 * case["vocab"] * bool(case.get("bias"))
        if case.get("penalties"):
            total += cells // 8 + 4 * case["batch"] * case["said"]  # which tokens were said, and the counts of those
        if case.get("admit"):
            total += 4 * case["batch"] * case["said"] + cells * 4 + cells // 8  # the prompts, and the counts they give
        return {"bytes": total, "flops": 4 * cells}
    kv, d, heads = case["kv"], case["dim"], case.get("heads", 0)
    if case["op"] == "append":
        values = 2 * case["batch"] * case["new"] * kv * d
        dense = 2 * case["batch"] * _capacity(case) * kv * d
        return {"bytes": values * (2 + 1) + values + dense * 4, "flops": 4 * values}
    flops = 4 * d * heads * _pairs(case)
    if case["op"] == "prompt":
        return {"bytes": case["tokens"] * d * (2 * heads + 2 * kv) * 2, "flops": flops}
    window = case.get("window") or (1 << 40)
    keys = sum(min(held + case["new"], window + case["new"] - 1) for held in _held(case))
    rows = case["batch"] * case["new"]
    total = 2 * keys * kv * d + 2 * keys * kv * 4 // case["block"] + 2 * rows * heads * d * 2
    if case["op"] == "decode":
        total += 2 * 2 * rows * kv * d * 2  # the new keys and values, in and into the cache
    return {"bytes": total, "flops": flops}


# ----------------------------------------------------------------------------- inputs
def _normal(shape, g, scale=1.0) -> torch.Tensor:
    return (torch.randn(shape, generator=g, device="cuda", dtype=torch.float32) * scale).to(torch.bfloat16)


def _keys(shape, g) -> torch.Tensor:
    k = torch.randn(shape, generator=g, device="cuda", dtype=torch.float32)
    k[..., 3 :: shape[-1] // 2] *= 5.0  # the few channels that are larger than the rest
    return k.to(torch.bfloat16)


def _inputs(case, seed: int) -> dict:
    """Tensors of a case from the seed alone."""
    g = torch.Generator(device="cuda").manual_seed(1000003 * seed + 17)
    if case["op"] == "logits":
        b, v, n = case["batch"], case["vocab"], case["said"]
        x = torch.randn((b, v), generator=g, device="cuda") * 2.0 + 6.0 * torch.rand((b, v), generator=g, device="cuda") ** 40
        s = {"logits": x.to(torch.bfloat16) if case["type"] == "bf16" else x}
        # what was said: half of it from a small set of tokens, so that many repeat
        common = torch.randint(0, v, (b, 1 + n // 8), generator=g, device="cuda")
        said = torch.randint(0, v, (b, n), generator=g, device="cuda")
        again = torch.gather(common, 1, torch.randint(0, common.shape[1], (b, n), generator=g, device="cuda"))
        s["said"] = torch.where(torch.rand((b, n), generator=g, device="cuda") < 0.5, again, said)
        if case.get("penalties"):
            s["repetition"] = 1.0 + 0.5 * torch.rand(b, generator=g, device="cuda")
            s["presence"] = torch.rand(b, generator=g, device="cuda")
            s["frequency"] = 0.5 * torch.rand(b, generator=g, device="cuda")
        if case.get("bias"):
            s["bias"] = torch.randn(v, generator=g, device="cuda") * (torch.rand(v, generator=g, device="cuda") < 0.02)
        if case.get("grammar"):
            allowed = torch.rand((b, -(-v // 32), 1), generator=g, device="cuda") < 0.3  # grammars allow and forbid in runs
            bits = allowed & (torch.rand((b, -(-v // 32), 32), generator=g, device="cuda") < 0.7)
            weights = torch.tensor([1 << i for i in range(31)] + [-(1 << 31)], dtype=torch.int64, device="cuda")
            s["mask"] = (bits * weights).sum(-1).to(torch.int32)
        return s
    d, kv = case["dim"], case["kv"]
    if case["op"] == "prompt":
        t = case["tokens"]
        return {"q": _normal((t, case["heads"], d), g, 1.5), "k": _keys((t, kv, d), g), "v": _normal((t, kv, d), g)}
    b, new = case["batch"], case["new"]
    s = {"k": _keys((b, new, kv, d), g), "v": _normal((b, new, kv, d), g)}
    if case["op"] != "append":
        s["q"] = _normal((b, new, case["heads"], d), g, 1.5)
        s["past"] = [(_keys((n, kv, d), g), _normal((n, kv, d), g)) for n in _held(case)]
    return s


def _slopes(heads: int) -> torch.Tensor:
    return torch.tensor([2.0 ** (-8.0 * (h + 1) / heads) for h in range(heads)], dtype=torch.float32, device="cuda")


def _options(case) -> dict:
    """The score options of a case as keyword arguments."""
    o = {}
    if "cap" in case:
        o["softcap"] = case["cap"]
    if "window" in case:
        o["window"] = case["window"]
    if case.get("bias"):
        o["slopes"] = _slopes(case["heads"])
    return o


def prepare(case, seed: int) -> dict:
    s = _inputs(case, seed)
    s["case"] = case
    if case["op"] == "logits":
        b, v = case["batch"], case["vocab"]
        if own:
            from binade_b200.cuda.logits import TokenCounts

            s["counts"] = TokenCounts(b, v)
            if not case.get("admit"):  # some of what was said is the prompt, the rest the answer so far
                cut = case["said"] // 2
                if cut:
                    s["counts"].add(s["said"][:, :cut], prompt=True)
                s["counts"].add(s["said"][:, cut:])
        else:
            s["seen"] = torch.zeros((b, v), dtype=torch.bool, device="cuda")
            s["counts"] = torch.zeros((b, v), dtype=torch.int32, device="cuda")
            if not case.get("admit"):
                cut = case["said"] // 2
                s["seen"].scatter_(1, s["said"], True)
                answer = s["said"][:, cut:]
                s["counts"].scatter_add_(1, answer, torch.ones_like(answer, dtype=torch.int32))
        return s
    s["options"] = _options(case)
    if case["op"] == "prompt":
        lens = _documents(case)
        s["lens"] = lens
        s["offsets"] = torch.tensor([sum(lens[:i]) for i in range(len(lens) + 1)], dtype=torch.int32, device="cuda")
        if "prefix" in case:
            s["prefixes"] = _prefixes(case)
            s["options"]["prefix"] = torch.tensor(s["prefixes"], dtype=torch.int32, device="cuda")
        if case.get("causal") is False:
            s["options"]["causal"] = False
        return s
    b, kv, d, block = case["batch"], case["kv"], case["dim"], case["block"]
    s["held"] = _held(case) if case["op"] != "append" else [0] * b
    past = s.pop("past", None)
    if own:
        from binade_b200.cuda.attention import KV8Cache

        cache = s["cache"] = KV8Cache(1, b, kv, d, _capacity(case), kind=case["kind"], block=block)
        if past is not None:
            for i, (k, v) in enumerate(past):  # one sequence at a time: the others bring no token
                if k.shape[0]:
                    n = torch.zeros(b, dtype=torch.int32, device="cuda")
                    n[i] = k.shape[0]
                    cache.append(0, k[None].expand(b, -1, -1, -1), v[None].expand(b, -1, -1, -1), n)
                    cache.advance(n)
            if case["op"] == "chunk":  # the chunk is in the cache already: `run` attends
                cache.append(0, s["k"], s["v"])
    else:
        s["cache"] = _PlainCache(case)
        for i, (k, v) in enumerate(past or []):
            s["cache"].append(i, k, v)
        if case["op"] == "chunk":
            for i in range(b):
                s["cache"].append(i, s["k"][i], s["v"][i], move=False)
    return s


# ----------------------------------------------------------------------------- plain forms
def _quantise(x: torch.Tensor, kind: str):
    """x [..., block, D] float32 -> (codes as float32, scale [..., 1, 1]): one scale for the block."""
    finite = torch.where(torch.isfinite(x), x, torch.zeros_like(x))
    amax = finite.abs().amax(dim=(-1, -2), keepdim=True)
    most = torch.full_like(amax, 127.0 if kind == "int8" else 448.0)  # a tensor: by a number torch multiplies with the reciprocal
    if kind == "int8":
        scale = (amax / most).clamp(min=2.0**-100)
        # the quotient in 64 bits: next to the border between two codes 32 are too few
        q = torch.round((torch.nan_to_num(x, nan=0.0).double() / scale.double())).clamp(-127, 127).float()
        return q, scale
    mantissa, exponent = torch.frexp(amax / most)
    exponent = torch.where(mantissa == 0.5, exponent - 1, exponent)  # ceil(log2(.))
    scale = torch.exp2(torch.where(amax > 0, exponent, torch.full_like(exponent, -100)).clamp(min=-100).double()).float()
    q = (torch.nan_to_num(x, nan=0.0) / scale).clamp(-448, 448).to(torch.float8_e4m3fn).float()
    return q, scale


class _PlainCache:
    """Codes, scales and the rows of the incomplete block, of every sequence and head."""

    def __init__(self, case):
        b, kv, d, block, cap = case["batch"], case["kv"], case["dim"], case["block"], _capacity(case)
        self.kind, self.block, self.cap = case["kind"], block, cap
        code = torch.int8 if self.kind == "int8" else torch.float8_e4m3fn
        self.codes = [torch.zeros((b, kv, cap, d), dtype=code, device="cuda") for _ in range(2)]
        self.scales = [torch.zeros((b, kv, cap // block), dtype=torch.float32, device="cuda") for _ in range(2)]
        # two places for open blocks: the one that was open before a call stays as it is when the call opens another
        self.tails = [torch.zeros((b, kv, 2, block, d), dtype=torch.bfloat16, device="cuda") for _ in range(2)]
        self.held, self.side = [0] * b, [0] * b

    def append(self, i: int, k: torch.Tensor, v: torch.Tensor, move: bool = True):
        """Tokens k, v [n, kv, D] behind what sequence i holds; with `move` it holds them from now on."""
        first, block, n, side = self.held[i], self.block, k.shape[0], self.side[i]
        part = first % block
        for x, codes, scales, tails in zip((k, v), self.codes, self.scales, self.tails):
            rows = torch.cat([tails[i, :, side, :part], x.transpose(0, 1)], dim=1)  # [kv, part + n, D]
            full = rows.shape[1] // block
            tails[i, :, side, part : part + n] = rows[:, part:block]
            if full:
                whole = rows[:, : full * block].float().reshape(rows.shape[0], full, block, -1)
                q, scale = _quantise(whole, self.kind)
                at = first - part
                codes[i, :, at : at + full * block] = q.reshape(rows.shape[0], full * block, -1).to(codes.dtype)
                scales[i, :, at // block : at // block + full] = scale[..., 0, 0]
                tails[i, :, 1 - side, : rows.shape[1] - full * block] = rows[:, full * block :]
        if move:
            self.held[i] += n
            self.side[i] ^= self.held[i] // block != first // block

    def rows(self, i: int, n: int) -> list:
        """The first n tokens of sequence i as the cache holds them: K, V [kv, n, D] float32."""
        full = n // self.block * self.block
        side = self.side[i] ^ (n // self.block != self.held[i] // self.block)
        out = []
        for codes, scales, tails in zip(self.codes, self.scales, self.tails):
            whole = codes[i, :, :full].float() * scales[i, :, : full // self.block].repeat_interleave(self.block, dim=1)[..., None]
            out.append(torch.cat([whole, tails[i, :, side, : n - full].float()], dim=1))
        return out


def _attend(q, k, v, first: int, prefix: int, case, slopes) -> torch.Tensor:
    """Queries q [n, heads, D] at positions first.. over k, v [kv, L, D] float32 -> [n, heads, D] float32."""
    n, heads, _ = q.shape
    kv, keys, _ = k.shape
    out = torch.empty(q.shape, dtype=torch.float32, device=q.device)
    i = torch.arange(first, first + n, device=q.device)[:, None]
    j = torch.arange(keys, device=q.device)[None, :]
    gap = (i - j).abs()
    visible = torch.ones((n, keys), dtype=torch.bool, device=q.device) if case.get("causal") is False else (j <= i) | (j < prefix)
    if "window" in case:
        visible = visible & (gap < case["window"])
    group = heads // kv
    for h in range(kv):
        s = torch.matmul(q[:, h * group : (h + 1) * group].float().transpose(0, 1), k[h].T) * _scale(case)  # [group, n, keys]
        if "cap" in case:
            s = case["cap"] * torch.tanh(s / case["cap"])
        if slopes is not None:
            s = s - slopes[h * group : (h + 1) * group, None, None] * gap
        s = s.masked_fill(~visible, float("-inf"))
        p = torch.exp(s - s.amax(dim=-1, keepdim=True))
        o = torch.matmul(p, v[h]) / p.sum(dim=-1, keepdim=True)
        out[:, h * group : (h + 1) * group] = o.transpose(0, 1)
    return out


def _plain(s):
    case = s["case"]
    if case["op"] == "logits":
        x, seen, counts = s["logits"].float(), s["seen"], s["counts"]
        if case.get("admit"):
            seen.zero_().scatter_(1, s["said"], True)
            counts.zero_()
        if case.get("penalties"):
            r = s["repetition"][:, None]
            x = torch.where(seen, torch.where(x > 0, x / r, x * r), x)
            x = x - (s["frequency"][:, None] * counts + s["presence"][:, None] * (counts > 0))
        if case.get("bias"):
            x = x + s["bias"]
        if case.get("grammar"):
            bit = torch.arange(case["vocab"], device=x.device)
            allowed = (s["mask"][:, bit >> 5] >> (bit & 31).to(torch.int32)) & 1
            x = x.masked_fill(allowed == 0, float("-inf"))
        top = x.amax(dim=1, keepdim=True)
        place = torch.arange(case["vocab"], device=x.device).expand_as(x)
        token = torch.where(x == top, place, torch.full_like(place, case["vocab"])).amin(dim=1)
        token = torch.where(top[:, 0] > float("-inf"), token, torch.full_like(token, -1))
        if case.get("admit"):
            return [x, token, counts]
        return [x, token]
    slopes = s["options"].get("slopes")
    if case["op"] == "prompt":
        out, at = torch.empty_like(s["q"]), 0
        for i, n in enumerate(s["lens"]):
            prefix = s["prefixes"][i] if "prefix" in case else 0
            k, v = (s[x][at : at + n].float().transpose(0, 1) for x in ("k", "v"))
            out[at : at + n] = _attend(s["q"][at : at + n], k, v, 0, prefix, case, slopes).to(out.dtype)
            at += n
        return [out]
    cache = s["cache"]
    if case["op"] == "append":
        for i in range(case["batch"]):
            cache.append(i, s["k"][i], s["v"][i], move=False)
        dense = [torch.zeros((case["batch"], case["kv"], cache.cap, case["dim"]), dtype=torch.float32, device="cuda") for _ in range(2)]
        for i in range(case["batch"]):
            for whole, rows in zip(dense, cache.rows(i, case["new"])):
                whole[i, :, : case["new"]] = rows
        return dense
    out = torch.empty_like(s["q"])
    for i in range(case["batch"]):
        if case["op"] == "decode":
            cache.append(i, s["k"][i], s["v"][i], move=False)
        k, v = cache.rows(i, cache.held[i] + case["new"])
        out[i] = _attend(s["q"][i], k, v, cache.held[i], 0, case, slopes).to(out.dtype)
    return [out, *cache.tails] if case["op"] == "decode" else [out]


# ----------------------------------------------------------------------------- one pass
def run(s):
    if not own:
        return _plain(s)
    case = s["case"]
    if case["op"] == "prompt":
        from binade_b200.cuda.attention import attention

        return [attention(s["q"], s["k"], s["v"], s["offsets"], scale=_scale(case), **s["options"])]
    if case["op"] == "decode":
        out = s["cache"].attend(0, s["q"], s["k"], s["v"], scale=_scale(case), **s["options"])
        return [out, s["cache"].k_tail[0], s["cache"].v_tail[0]]
    if case["op"] == "chunk":
        return [s["cache"].attend(0, s["q"], scale=_scale(case), **s["options"])]
    if case["op"] == "append":
        s["cache"].append(0, s["k"], s["v"])
        s["cache"].advance(case["new"])
        dense = s["cache"].dense(0)
        s["cache"].advance(-case["new"])
        return list(dense)
    from binade_b200.cuda.logits import process_logits

    if case.get("admit"):
        s["counts"].clear()
        s["counts"].add(s["said"], prompt=True)
    x, token = process_logits(s["logits"], s["counts"], repetition=s.get("repetition"), presence=s.get("presence"), frequency=s.get("frequency"), bias=s.get("bias"), mask=s.get("mask"))
    return [x, token, s["counts"].counts] if case.get("admit") else [x, token]


# ----------------------------------------------------------------------------- the definition in 64 bits
def _exact_stored(x: torch.Tensor, kind: str, block: int) -> torch.Tensor:
    """Tokens x [n, kv, D] as a cache gives them back, float64: whole blocks through 8 bits, the rest as is."""
    x = x.double()
    out = x.clone()
    for t0 in range(0, x.shape[0] - block + 1, block):
        rows = x[t0 : t0 + block]
        most = rows.abs().amax(dim=(0, 2))  # per head
        share = most / torch.full_like(most, 127.0 if kind == "int8" else 448.0)  # (a quotient, not a product with 1 / 127)
        if kind == "int8":
            step = share.float().double().clamp(min=2.0**-100)[None, :, None]
            out[t0 : t0 + block] = (rows / step).round().clamp(-127, 127) * step
        else:
            step = torch.exp2(torch.log2(share).ceil().clamp(min=-100))[None, :, None]
            y = rows / step
            size = torch.floor(torch.log2(y.abs().clamp(min=2.0**-20))).clamp(min=-6)  # e4m3: 3 bits behind the first, exponents down to -6
            grid = torch.exp2(size - 3)
            out[t0 : t0 + block] = ((y / grid).round() * grid).clamp(-448, 448) * step
    return out


def _exact_rows(q, k, v, first, prefix, case) -> torch.Tensor:
    """As `_attend`, float64, over k, v [L, kv, D]."""
    n, heads, d = q.shape
    keys, kv, _ = k.shape
    slopes = _slopes(heads).double() if case.get("bias") else torch.zeros(heads, dtype=torch.float64, device=q.device)
    out = torch.empty((n, heads, d), dtype=torch.float64, device=q.device)
    where = torch.arange(keys, device=q.device)
    step = max(1, (1 << 26) // keys)
    for h in range(heads):
        kh, vh = k[:, h * kv // heads], v[:, h * kv // heads]
        for r0 in range(0, n, step):
            at = torch.arange(first + r0, first + min(n, r0 + step), device=q.device)
            dist = (at[:, None] - where[None, :]).abs().double()
            z = torch.einsum("nd,kd->nk", q[r0 : r0 + step, h].double(), kh) / math.sqrt(d)
            if "cap" in case:
                z = torch.tanh(z / case["cap"]) * case["cap"]
            z = z - slopes[h] * dist
            hidden = torch.zeros_like(z, dtype=torch.bool)
            if case.get("causal") is not False:
                hidden = (where[None, :] > at[:, None]) & (where[None, :] >= prefix)
            if "window" in case:
                hidden = hidden | (dist >= case["window"])
            z[hidden] = -math.inf
            out[r0 : r0 + step, h] = torch.einsum("nk,kd->nd", torch.exp(z - torch.logsumexp(z, dim=1, keepdim=True)), vh)
    return out


def exact(case, seed: int):
    s = _inputs(case, seed)
    if case["op"] == "logits":
        b, v, n = case["batch"], case["vocab"], case["said"]
        x = s["logits"].double()
        times = torch.zeros((b, v), dtype=torch.int64, device="cuda")
        seen = torch.zeros((b, v), dtype=torch.int64, device="cuda").scatter_add_(1, s["said"], torch.ones_like(s["said"]))
        if not case.get("admit"):
            answer = s["said"][:, n // 2 :]
            times.scatter_add_(1, answer, torch.ones_like(answer))
        if case.get("penalties"):
            factor = torch.where(x > 0, 1.0 / s["repetition"].double()[:, None], s["repetition"].double()[:, None])
            x = torch.where(seen > 0, x * factor, x)
            x = x - s["frequency"].double()[:, None] * times - s["presence"].double()[:, None] * times.clamp(max=1)
        if case.get("bias"):
            x = x + s["bias"].double()
        if case.get("grammar"):
            words = s["mask"].long() & 0xFFFFFFFF
            allowed = torch.stack([(words >> i) & 1 for i in range(32)], dim=-1).reshape(b, -1)[:, :v]
            x = torch.where(allowed == 1, x, torch.full_like(x, -math.inf))
        # the token hangs on the last bit where two logits are as good as equal: it has no value in 64 bits
        return [x, None, times.to(torch.int32)] if case.get("admit") else [x, None]
    if case["op"] == "prompt":
        out, at = torch.empty(s["q"].shape, dtype=torch.float64, device="cuda"), 0
        prefixes = _prefixes(case) if "prefix" in case else [0] * case["docs"]
        for n, prefix in zip(_documents(case), prefixes):
            k, v = s["k"][at : at + n].double(), s["v"][at : at + n].double()
            out[at : at + n] = _exact_rows(s["q"][at : at + n], k, v, 0, prefix, case)
            at += n
        return [out]
    if case["op"] == "append":
        dense = []
        for x in (s["k"], s["v"]):
            whole = torch.zeros((case["batch"], case["kv"], _capacity(case), case["dim"]), dtype=torch.float64, device="cuda")
            for i in range(case["batch"]):
                whole[i, :, : case["new"]] = _exact_stored(x[i], case["kind"], case["block"]).transpose(0, 1)
            dense.append(whole)
        return dense
    if sum(_held(case)) * case["kv"] * case["dim"] > 600_000_000:
        return None
    out = torch.empty(s["q"].shape, dtype=torch.float64, device="cuda")
    block = case["block"]
    tails = [torch.zeros((case["batch"], case["kv"], 2, block, case["dim"]), dtype=torch.float64, device="cuda") for _ in range(2)]
    for i, (pk, pv) in enumerate(s["past"]):
        k, v = torch.cat([pk, s["k"][i]]), torch.cat([pv, s["v"][i]])
        stored = [_exact_stored(x, case["kind"], block) for x in (k, v)]
        out[i] = _exact_rows(s["q"][i], stored[0], stored[1], pk.shape[0], 0, case)
        # two open blocks are kept: the first that the past began with, and, if it filled up, the one open now
        now = k.shape[0] // block
        for tail, x in zip(tails, (k, v)):
            tail[i, :, 0, : min(block, x.shape[0])] = x[:block].double().transpose(0, 1)
            if now:
                tail[i, :, 1, : x.shape[0] - now * block] = x[now * block :].double().transpose(0, 1)
    return [out, *tails] if case["op"] == "decode" else [out]
