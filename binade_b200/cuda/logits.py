"""What happens to logits before a token is chosen.

  TokenCounts(batch, vocab)      which tokens a batch of sequences has said, on the device
  process_logits(logits, ...)    penalties for repeated tokens, a bias, a grammar's mask; the greedy token
"""

from __future__ import annotations

import ctypes

import torch

from .. import _native
from . import kernels as ck
from .attention import narrow, overlap, refuse_gradient


class TokenCounts:
    """For every sequence of a batch: the tokens seen in its prompt or its answer (a bit each, `seen`), and how
    often each occurs in the answer (`counts`, int32 [batch, vocab]). Lives on the device; adding and clearing can be captured in a graph."""

    def __init__(self, batch: int, vocab: int, device=None):
        if not 1 <= batch <= 65535 or not 1 <= vocab < 1 << 30:
            raise ValueError("batch (below 65536) and vocab (below 2^30) have to be positive")
        dev = ck.require_cuda() if device is None else torch.device(device)
        if dev.type != "cuda":
            raise ValueError(f"token counts live on a CUDA device, not {dev}")
        self.batch, self.vocab = batch, vocab
        words = -(-vocab // 32)
        self._all = torch.zeros((batch, words + vocab), dtype=torch.int32, device=dev)  # one array: cleared in one go
        self.seen, self.counts = self._all[:, :words], self._all[:, words:]
        self.device = self._all.device

    def add(self, tokens: torch.Tensor, lengths: torch.Tensor | None = None, prompt: bool = False) -> None:
        """tokens int64 or int32 [batch, n] (or [batch]: one each); lengths (whole numbers [batch]): how many of
        each row are real, the first ones. prompt: seen, but not counted. Tokens outside the vocabulary are passed over."""
        if not isinstance(tokens, torch.Tensor) or tokens.dtype not in (torch.int64, torch.int32) or tokens.device != self.device:
            raise ValueError(f"tokens have to be int64 or int32 on {self.device}")
        if tokens.dim() == 1:
            tokens = tokens[:, None]
        if tokens.dim() != 2 or tokens.shape[0] != self.batch:
            raise ValueError(f"tokens {tuple(tokens.shape)} for a batch of {self.batch}")
        if torch._C._cuda_getDevice() != self.device.index:
            raise ValueError(f"the counts are on {self.device}, the current device is another one")
        if tokens.shape[1] > 1 and tokens.stride(1) != 1:
            tokens = tokens.contiguous()
        if lengths is not None:
            if not isinstance(lengths, torch.Tensor) or lengths.device != self.device or lengths.shape != (self.batch,) or lengths.is_floating_point():
                raise ValueError(f"lengths have to be {self.batch} whole numbers on {self.device}")
            lengths = (narrow(lengths) if lengths.dtype.itemsize > 4 else lengths.to(torch.int32)).contiguous()
        ck._call("bn_token_counts", ck._p(tokens), int(tokens.dtype == torch.int64), tokens.stride(0), self.batch, tokens.shape[1], ck._p(lengths), self.vocab, int(prompt), ck._p(self.seen), self._all.stride(0), ck._p(self.counts), self._all.stride(0))

    def clear(self, row=None) -> None:
        """Forgets everything, or one sequence's tokens (row: a number)."""
        if row is not None and (not isinstance(row, int) or isinstance(row, bool) or not 0 <= row < self.batch):
            raise ValueError(f"row {row!r} of {self.batch}")
        (self._all if row is None else self._all[row]).zero_()


def _penalty(p, name: str, batch: int, device):
    """(device array or None, value) of a penalty."""
    if isinstance(p, torch.Tensor):
        if p.device != device or p.shape != (batch,):
            raise ValueError(f"{name} has to be a number or a tensor of {batch} on {device}")
        refuse_gradient(p, name)
        return p if p.dtype is torch.float32 and p.is_contiguous() else p.to(torch.float32).contiguous(), 0.0
    return None, float(p)


def process_logits(logits: torch.Tensor, said: TokenCounts | None = None, *, repetition=None, presence=None, frequency=None, bias: torch.Tensor | None = None, mask: torch.Tensor | None = None, out: torch.Tensor | None = None):
    """logits [batch, vocab] (bfloat16 or float32) -> (logits float32 [batch, vocab], tokens int64 [batch]).

    In this order, each operation rounded to fp32: a token that `said` has seen is divided by `repetition` if its
    logit is positive, else multiplied by it; `frequency` times its count and, if it was counted, `presence` are
    subtracted; `bias` (float32 [vocab], or [batch, vocab]) is added; where a bit of `mask` (int32, 32 tokens a word,
    [ceil(vocab / 32)] or [batch, ceil(vocab / 32)], set = allowed) is clear the logit becomes -inf.
    Penalties are numbers or float tensors [batch]. tokens: each row's lowest index of its largest logit, -1 if
    nothing is left above -inf (NaN is never chosen). `out`: where to write the logits (may be `logits` itself if float32)."""
    if not isinstance(logits, torch.Tensor) or logits.dtype not in (torch.bfloat16, torch.float32) or logits.dim() != 2 or not logits.is_cuda or logits.get_device() != torch._C._cuda_getDevice():
        raise ValueError(f"logits have to be bfloat16 or float32 [batch, vocab] on the current device, {ck.require_cuda()}")
    dev = logits.device
    refuse_gradient(logits, "logits")
    batch, vocab = logits.shape
    if not 1 <= vocab < 1 << 30 or batch > 65535:
        raise ValueError(f"logits {tuple(logits.shape)}")
    if vocab > 1 and logits.stride(1) != 1 or batch > 1 and logits.stride(0) < vocab:
        logits = logits.contiguous()
    rules = _native.LogitRules(repetition_all=1.0)
    keep = []
    if repetition is not None or presence is not None or frequency is not None:
        if said is None:
            raise ValueError("penalties need the tokens that were said")
        for name, p, none in (("repetition", repetition, 1.0), ("presence", presence, 0.0), ("frequency", frequency, 0.0)):
            t, value = _penalty(none if p is None else p, name, batch, dev)
            keep.append(t)
            setattr(rules, name, ck._p(t))
            setattr(rules, name + "_all", value)
        if rules.repetition is None and not rules.repetition_all > 0:
            raise ValueError("repetition has to be positive")
        if said.batch != batch or said.vocab != vocab or said.device != dev:
            raise ValueError(f"counts of {said.batch} x {said.vocab} on {said.device} for logits {tuple(logits.shape)}")
        rules.seen, rules.counts, rules.seen_row, rules.counts_row = ck._p(said.seen), ck._p(said.counts), said._all.stride(0), said._all.stride(0)
    for name, t, width, dtype in (("bias", bias, vocab, torch.float32), ("mask", mask, -(-vocab // 32), torch.int32)):
        if t is None:
            continue
        if not isinstance(t, torch.Tensor) or t.dtype != dtype or t.device != dev or t.shape not in ((width,), (batch, width)):
            raise ValueError(f"{name} has to be {dtype} of [{width}] or [{batch}, {width}] on {dev}")
        refuse_gradient(t, name)
        t = t.contiguous()
        keep.append(t)
        setattr(rules, name, ck._p(t))
        setattr(rules, name + "_row", width if t.dim() == 2 else 0)
    if out is None:
        out = torch.empty(batch, vocab, dtype=torch.float32, device=dev)
    elif not isinstance(out, torch.Tensor) or out.dtype != torch.float32 or out.shape != logits.shape or out.device != dev or out.requires_grad or (vocab > 1 and out.stride(1) != 1) or (batch > 1 and out.stride(0) < vocab):
        raise ValueError("out has to be float32 of the logits' shape with rows of neighbouring elements that do not overlap")
    elif overlap(out, logits) and not (out.data_ptr() == logits.data_ptr() and out.dtype == logits.dtype and (batch == 1 or out.stride(0) == logits.stride(0))):
        raise ValueError("out may be logits (float32), but not lie across them")
    elif any(t is not None and overlap(out, t) for t in (*keep, said and said._all)):
        raise ValueError("out may not lie among the penalties, the bias, the mask or the counts")
    refuse_gradient(out, "out")
    tokens = torch.empty(batch, dtype=torch.int64, device=dev)
    if batch:
        ck._call("bn_logits", ck._p(logits), int(logits.dtype == torch.float32), logits.stride(0), batch, vocab, ctypes.byref(rules), ck._p(out), out.stride(0), ck._p(tokens))
    return out, tokens
