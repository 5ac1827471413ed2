"""Attention beside the R4 linear layers: of prompts, and of new tokens over a cache held in 8 bits.

  attention(q, k, v, offsets)      packed prompts: every query over the keys of its own document
  KV8Cache(layers, batch, ...)     keys and values of a batch of sequences as 8-bit codes with a scale for
                                   each block of tokens and head; append, attend, advance, dense

Scores take the options that models put on them: softcap (s = cap tanh(s / cap), caps from 2^-60 to 2^60), slopes (a bias
-slope |i - j| for each query head), window (keys at a distance below it), prefix (the first keys of a document,
seen from everywhere in it) and causal. Kernels, no gradients: tensors that ask for one are refused.
"""

from __future__ import annotations

import ctypes
import math
import operator

import torch
from torch.autograd import forward_ad

from .. import _native
from . import kernels as ck

HEAD_DIMS = (64, 128, 256)
BLOCKS = (16, 32, 64)
KINDS = {"int8": 0, "e4m3": 1}  # BN_KV8_INT8, BN_KV8_E4M3


def refuse_gradient(t: torch.Tensor, name: str) -> None:
    """The calls here have no gradients, backward or forward: what asks for one is told so."""
    if t.requires_grad and torch.is_grad_enabled() or forward_ad._current_level >= 0 and forward_ad.unpack_dual(t).tangent is not None:
        raise ValueError(f"{name} asks for a gradient: there is none here (use torch.no_grad)")


def _rows(t: torch.Tensor, name: str, dims: int, device, apart: bool = False):
    """Checks a BF16 tensor of rows (its last dimension a head's) on CUDA device number `device` and gives it with
    rows that the kernels can read (neighbouring elements, every row on 16 bytes; apart: no two the same), and the
    strides of its leading dimensions, 0 for one that is not stepped."""
    if not isinstance(t, torch.Tensor) or t.dtype is not torch.bfloat16 or t.dim() != dims:
        raise ValueError(f"{name} has to be a bfloat16 tensor of {dims} dimensions")
    if t.get_device() != device:
        raise ValueError(f"{name} is on {t.device}, the call on cuda:{device}")
    refuse_gradient(t, name)
    if t.is_contiguous() and t.data_ptr() % 16 == 0:
        steps, bits = t.stride()[:-1], 0
        for step in steps:
            bits |= step
        return t, _steps(t) if bits & 7 else steps  # (of a dimension of one element torch takes any stride for contiguous)
    steps = _steps(t)
    fits = t.stride(-1) == 1 and t.data_ptr() % 16 == 0
    for s, n in zip(steps, t.shape):
        fits = fits and not s % 8 and (s or n <= 1 or not apart)
    if not fits:
        t = t.contiguous() if not t.is_contiguous() else t.clone()
        steps = _steps(t)
    return t, steps


def _steps(t: torch.Tensor):
    """Strides of the leading dimensions; of one that is not stepped, 0."""
    return [s if n > 1 else 0 for s, n in zip(t.stride(), t.shape)][:-1]


def _numbers(t, name: str, n: int, device, dtype=torch.int32) -> torch.Tensor | None:
    if t is None:
        return None
    if not isinstance(t, torch.Tensor) or t.get_device() != device or t.dim() != 1 or t.numel() != n or (dtype == torch.int32 and t.is_floating_point()):
        raise ValueError(f"{name} has to be a tensor of {n} {'whole ' if dtype == torch.int32 else ''}numbers on cuda:{device}")
    if dtype == torch.float32:
        refuse_gradient(t, name)
    elif t.dtype.itemsize > 4:
        t = narrow(t)
    return t if t.dtype is dtype and t.is_contiguous() else t.to(dtype).contiguous()


def narrow(t: torch.Tensor) -> torch.Tensor:
    """64-bit whole numbers in 32: what lies beyond them as the nearest that they hold (a prefix of 2^40 keys is all of them)."""
    return t.clamp(-(1 << 31), (1 << 31) - 1).to(torch.int32)


def extent(t: torch.Tensor):
    """First and last byte address (the latter exclusive) that a tensor's elements lie in."""
    last = sum((n - 1) * s for n, s in zip(t.shape, t.stride())) if t.numel() else -1
    return t.data_ptr(), t.data_ptr() + (last + 1) * t.element_size()


def overlap(a: torch.Tensor, b: torch.Tensor) -> bool:
    (a0, a1), (b0, b1) = extent(a), extent(b)
    return a0 < b1 and b0 < a1


def _out(out, like: torch.Tensor, device, *inputs) -> torch.Tensor:
    if out is None:
        return torch.empty_like(like, memory_format=torch.contiguous_format)
    if not isinstance(out, torch.Tensor) or out.dtype != torch.bfloat16 or out.shape != like.shape or out.get_device() != device or out.requires_grad:
        raise ValueError("out has to be a bfloat16 tensor of q's shape on its device")
    refuse_gradient(out, "out")
    if out.stride(-1) != 1 or out.data_ptr() % 16 or any(s % 8 or s == 0 for s, n in zip(out.stride()[:-1], out.shape[:-1]) if n > 1):
        raise ValueError("out's rows have to lie apart, each of neighbouring elements from a 16-byte boundary on")
    if any(t is not None and overlap(out, t) for t in inputs):
        raise ValueError("out may not lie among the inputs")
    return out


_score_structs: dict = {}  # bn_scores of calls without slopes, by their options


def _scores(dim: int, heads: int, device, scale, softcap, window, slopes, causal):
    """The bn_scores of a call, and the slopes that it points at."""
    scale, softcap = None if scale is None else float(scale), None if softcap is None else float(softcap)
    window, causal = None if window is None else operator.index(window), bool(causal)
    options = (dim, scale, softcap, window, causal)  # (plain numbers: what a tensor holds may change)
    made = _score_structs.get(options) if slopes is None else None  # (one look: another thread may clear the table)
    if made is not None:
        return made, None
    if softcap is not None and not 2.0**-60 <= softcap <= 2.0**60:
        raise ValueError("softcap has to be a number in 2^-60 .. 2^60")
    if window is not None and not 1 <= window < 1 << 30:
        raise ValueError("window has to be at least 1")
    if scale is not None and not abs(scale) <= 3.4e38:
        raise ValueError("scale has to be a number that fp32 holds")
    slopes = _numbers(slopes, "slopes", heads, device, torch.float32)
    made = _native.Scores(1.0 / math.sqrt(dim) if scale is None else scale, softcap or 0.0, window or 0, ck._p(slopes), int(causal))
    if slopes is None:
        if len(_score_structs) >= 64:
            _score_structs.clear()
        _score_structs[options] = made
    return made, slopes


def _device(t) -> int:
    if not isinstance(t, torch.Tensor) or not t.is_cuda or t.get_device() != torch._C._cuda_getDevice():
        raise ValueError(f"q has to be a tensor on the current device, {ck.require_cuda()}")
    return t.get_device()


def attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, offsets: torch.Tensor | None = None, *, causal: bool = True, scale: float | None = None, softcap: float | None = None, window: int | None = None, slopes: torch.Tensor | None = None, prefix: torch.Tensor | None = None, out: torch.Tensor | None = None) -> torch.Tensor:
    """Softmax attention of packed prompts: q [T, heads, D], k and v [T, kv_heads, D] bfloat16 (views of a fused
    projection's output are read in place), D 64, 128 or 256, heads a multiple of kv_heads -> [T, heads, D].

    offsets: rising whole numbers [documents + 1] on the device: tokens offsets[n] .. offsets[n + 1] - 1 are
    document n, and queries see keys of their own document only (None: one document). Rows of tokens in no
    document come back as zeros, or, with `out` given, stay as they are. causal: a query sees no key behind
    it, but for the first prefix[n] of its document n. window: only keys at a distance below it. scale
    defaults to 1 / sqrt(D). Nothing is read on the host: the call can be captured in a graph."""
    dev = _device(q)
    q, q_steps = _rows(q, "q", 3, dev, apart=True)
    k, k_steps = _rows(k, "k", 3, dev, apart=True)
    v, v_steps = _rows(v, "v", 3, dev, apart=True)
    T, heads, D = q.shape
    kv = k.shape[1]
    if D not in HEAD_DIMS or k.shape != (T, kv, D) or v.shape != k.shape or kv < 1 or heads < 1 or heads % kv:
        raise ValueError(f"q {tuple(q.shape)}, k {tuple(k.shape)}, v {tuple(v.shape)}: heads of 64, 128 or 256, query heads a multiple of key heads, the same tokens")
    docs = 1
    if offsets is not None:
        if not isinstance(offsets, torch.Tensor) or offsets.numel() < 1:
            raise ValueError("offsets has to be a tensor of documents + 1 whole numbers")
        docs = offsets.numel() - 1
        offsets = _numbers(offsets, "offsets", docs + 1, dev)
    prefix = _numbers(prefix, "prefix", docs, dev)
    scores, slopes = _scores(D, heads, dev, scale, softcap, window, slopes, causal)
    y = _out(out, q, dev, q, k, v, offsets, prefix, slopes)
    if T:
        ck._call("bn_attention", q.data_ptr(), *q_steps, k.data_ptr(), *k_steps, v.data_ptr(), *v_steps, T, heads, kv, D, ck._p(offsets), docs, ck._p(prefix), ctypes.byref(scores), y.data_ptr(), *(y.stride()[:-1] if out is None else _steps(y)), int(out is None))
    return y


class KV8Cache:
    """Keys and values of `batch` sequences in `layers` layers, 8 bits a value: codes with one fp32 scale for each
    block of `block` tokens and head ("int8": amax / 127; "e4m3": a power of two). The tokens of a block that is
    not full yet stay in BF16 until it is, so what is held does not depend on how the tokens came.
    NaN is stored as 0 and an infinity as the largest code.

    A step of a model: for every layer `attend(layer, q, k, v)` (or `append` and later `attend`), then
    one `advance`. `length` (int32 [batch], on the device) is what each sequence holds; setting a sequence's to 0
    frees its place. Calls on one cache are ordered by the stream that they share."""

    def __init__(self, layers: int, batch: int, kv_heads: int, head_dim: int, max_seq: int, kind: str = "int8", block: int = 32, device=None):
        if min(layers, batch, kv_heads, max_seq) < 1 or batch > 65535 or kv_heads > 65535 or max_seq >= 1 << 30:
            raise ValueError("layers, batch, kv_heads and max_seq have to be positive (batch and kv_heads below 65536, max_seq below 2^30)")
        if head_dim not in HEAD_DIMS or block not in BLOCKS or kind not in KINDS:
            raise ValueError(f"head_dim {head_dim} (64, 128, 256), block {block} (16, 32, 64), kind {kind!r} (int8, e4m3)")
        dev = ck.require_cuda() if device is None else torch.device(device)
        if dev.type != "cuda":
            raise ValueError(f"the cache lives on a CUDA device, not {dev}")
        self.device = dev if dev.index is not None else ck.require_cuda()
        self._index, self._work = self.device.index, {}  # device number; workspace bytes by (tokens, heads)
        self.layers, self.batch, self.kv_heads, self.head_dim, self.max_seq, self.kind, self.block = layers, batch, kv_heads, head_dim, max_seq, kind, block
        rows = -(-max_seq // 64) * 64
        new = lambda *shape, dtype: torch.zeros((layers, batch, kv_heads, *shape), dtype=dtype, device=self.device)  # noqa: E731
        self.k, self.v = new(rows, head_dim, dtype=torch.uint8), new(rows, head_dim, dtype=torch.uint8)
        self.k_scale, self.v_scale = new(rows // block, dtype=torch.float32), new(rows // block, dtype=torch.float32)
        self.k_tail, self.v_tail = new(2, block, head_dim, dtype=torch.bfloat16), new(2, block, head_dim, dtype=torch.bfloat16)
        self.length, self._side = torch.zeros(batch, dtype=torch.int32, device=self.device), torch.zeros(batch, dtype=torch.int32, device=self.device)
        self._kept = torch.full((batch, 2), -1, dtype=torch.int32, device=self.device)
        self._tickets = torch.zeros(batch * kv_heads, dtype=torch.int32, device=self.device)
        self._structs = [_native.KV8Struct(*(t[i].data_ptr() for t in (self.k, self.v, self.k_scale, self.v_scale, self.k_tail, self.v_tail)), self.length.data_ptr(), self._side.data_ptr(), self._tickets.data_ptr(), batch, kv_heads, rows, head_dim, max_seq, block, KINDS[kind], self._kept.data_ptr()) for i in range(layers)]

    def bytes(self) -> int:
        """Device memory of the cache."""
        return sum(t.numel() * t.element_size() for t in (self.k, self.v, self.k_scale, self.v_scale, self.k_tail, self.v_tail, self.length, self._side, self._kept))

    def _layer(self, layer: int):
        if not 0 <= layer < self.layers:
            raise ValueError(f"layer {layer} of {self.layers}")
        if torch._C._cuda_getDevice() != self._index:
            raise ValueError(f"the cache is on {self.device}, the current device is another one")
        return ctypes.byref(self._structs[layer])

    def _new(self, t, name: str, heads: int | None = None, apart: bool = False):
        t, steps = _rows(t, name, 4, self._index, apart)
        if t.shape[0] != self.batch or t.shape[3] != self.head_dim or (heads is not None and t.shape[2] != heads):
            raise ValueError(f"{name} {tuple(t.shape)}: [batch {self.batch}, tokens, {'heads' if heads is None else heads}, {self.head_dim}] expected")
        return t, steps

    def append(self, layer: int, k: torch.Tensor, v: torch.Tensor, counts: torch.Tensor | None = None) -> None:
        """New tokens k, v [batch, tokens, kv_heads, D] bfloat16 behind what the sequences hold; counts (whole
        numbers [batch] on the device): how many of each sequence's are real, the first ones (None: all).
        `length` stays until `advance`: until then a second append writes the same places again. Tokens
        beyond max_seq are dropped, and bn_device_status tells (value 1 in bits 24..27)."""
        at = self._layer(layer)
        (k, k_steps), (v, v_steps) = self._new(k, "k", self.kv_heads), self._new(v, "v", self.kv_heads)
        if k.shape != v.shape:
            raise ValueError(f"k {tuple(k.shape)} and v {tuple(v.shape)} differ")
        counts = _numbers(counts, "counts", self.batch, self._index)
        if k.shape[1]:
            ck._call("bn_kv8_append", at, k.data_ptr(), *k_steps, v.data_ptr(), *v_steps, k.shape[1], ck._p(counts))

    def attend(self, layer: int, q: torch.Tensor, k: torch.Tensor | None = None, v: torch.Tensor | None = None, counts: torch.Tensor | None = None, *, causal: bool = True, scale: float | None = None, softcap: float | None = None, window: int | None = None, slopes: torch.Tensor | None = None, prefix: torch.Tensor | None = None, out: torch.Tensor | None = None) -> torch.Tensor:
        """Attention of new tokens q [batch, tokens, heads, D] bfloat16 over what their sequences hold and
        themselves -> [batch, tokens, heads, D]. With k and v the tokens are appended first; without, an `append`
        before did it. Query t of sequence b has position length[b] + t and sees the keys up to itself (all
        length[b] + counts[b] if not causal; options as in `attention`, prefix [batch]). Rows behind a sequence's
        counts come back as zeros, or, with `out` given, stay as they are."""
        at = self._layer(layer)
        q, q_steps = self._new(q, "q", apart=True)
        tokens, heads = q.shape[1], q.shape[2]
        if heads < 1 or heads % self.kv_heads:
            raise ValueError(f"{heads} query heads over {self.kv_heads} key heads")
        if (k is None) != (v is None):
            raise ValueError("k and v come together")
        counts = _numbers(counts, "counts", self.batch, self._index)
        prefix = _numbers(prefix, "prefix", self.batch, self._index)
        scores, slopes = _scores(self.head_dim, heads, self._index, scale, softcap, window, slopes, causal)
        y = _out(out, q, self._index, q, k, v, counts, prefix, slopes)
        if k is None:
            new = (None, 0, 0, 0, None, 0, 0, 0)
        else:
            (k, k_steps), (v, v_steps) = self._new(k, "k", self.kv_heads), self._new(v, "v", self.kv_heads)
            if k.shape[1] != tokens or v.shape[1] != tokens:
                raise ValueError(f"k {tuple(k.shape)} and v {tuple(v.shape)} for {tokens} tokens")
            new = (k.data_ptr(), *k_steps, v.data_ptr(), *v_steps)
        if tokens:
            need = self._work.get((tokens, heads))
            if need is None:
                need = self._work[tokens, heads] = _native.load("cuda").bn_kv8_workspace(at, tokens, heads)
            work = torch.empty(need, dtype=torch.uint8, device=self.device) if need else None
            ck._call("bn_kv8_attend", at, q.data_ptr(), *q_steps, *new, tokens, heads, ck._p(counts), ck._p(prefix), ctypes.byref(scores), y.data_ptr(), *(y.stride()[:-1] if out is None else _steps(y)), int(out is None), ck._p(work), need)
        return y

    def advance(self, n) -> None:
        """Moves `length` on by n tokens (a number, or whole numbers [batch] on the device), within 0 .. max_seq.
        Fewer than were appended may be kept (a draft whose end is rejected), and a sequence may go back. The new
        length has to lie on a border of blocks, or in a block whose rows are still held in BF16: the one that was
        open before the append, or the one that is open behind all its tokens. A sequence for which it does not
        stays where it is, and bn_device_status tells (value 2 in bits 24..27)."""
        at = self._layer(0)
        counts = _numbers(n, "n", self.batch, self._index) if isinstance(n, torch.Tensor) else None
        ck._call("bn_kv8_advance", at, 0 if counts is not None else n, ck._p(counts))

    def dense(self, layer: int):
        """What the layer holds as the values that its codes stand for: (K, V) float32 [batch, kv_heads,
        max_seq, D], zeros behind each sequence's length."""
        at = self._layer(layer)
        k, v = (torch.empty((self.batch, self.kv_heads, self.max_seq, self.head_dim), dtype=torch.float32, device=self.device) for _ in range(2))
        ck._call("bn_kv8_dense", at, ck._p(k), ck._p(v))
        return k, v
