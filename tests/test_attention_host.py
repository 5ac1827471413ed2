"""Refusals of the attention, cache and logits entry points on the host: no GPU is needed to be told no."""

import ctypes as C

import pytest
import torch

import attention_reference as ref
from binade_b200 import _native

BUF = 0x10000  # an aligned address that no call below gets to read


def cache(**change):
    c = _native.KV8Struct(*([BUF] * 9), 2, 2, 128, 128, 100, 32, 0)
    for k, v in change.items():
        setattr(c, k, v)
    return c


def scores(**change):
    s = _native.Scores(0.1, 0.0, 0, None, 1)
    for k, v in change.items():
        setattr(s, k, v)
    return s


def attention(q=BUF, qs=(512, 128), k=BUF, ks=(256, 128), v=BUF, vs=(256, 128), T=8, heads=4, kv=2, D=128, offsets=None, docs=1, s=None, out=BUF, os=(512, 128)):
    s = scores() if s is None else s
    return _native.call("cuda", "bn_attention", q, *qs, k, *ks, v, *vs, T, heads, kv, D, offsets, docs, None, C.byref(s), out, *os, 0, None)


@pytest.mark.parametrize("change", [dict(q=None), dict(out=None), dict(q=BUF + 2), dict(k=BUF + 8), dict(qs=(516, 128)), dict(vs=(256, 4)), dict(T=-1), dict(T=1 << 40), dict(heads=0), dict(heads=3), dict(kv=0), dict(D=96), dict(D=0), dict(docs=2), dict(docs=-1), dict(s=scores(window=-1)), dict(s=scores(softcap=-1.0)), dict(s=scores(softcap=float("nan")))])
def test_attention_refuses(change):
    with pytest.raises(_native.NativeError, match="bad argument: bn_attention"):
        attention(**change)


def test_attention_of_nothing():
    assert attention(T=0, q=None, k=None, v=None, out=None) == 0


BAD_CACHES = [dict(k=None), dict(v_scale=None), dict(length=None), dict(side=None), dict(tickets=None), dict(k=BUF + 4), dict(D=80), dict(block=8), dict(block=48), dict(kind=2), dict(batch=0), dict(kv_heads=0), dict(rows=64), dict(rows=100), dict(max_seq=0), dict(max_seq=1 << 31)]


@pytest.mark.parametrize("change", BAD_CACHES)
def test_caches_refused(change):
    c = C.byref(cache(**change))
    s = scores()
    for call in (
        lambda: _native.call("cuda", "bn_kv8_append", c, BUF, 256, 256, 128, BUF, 256, 256, 128, 1, None, None),
        lambda: _native.call("cuda", "bn_kv8_attend", c, BUF, 512, 512, 128, None, 0, 0, 0, None, 0, 0, 0, 1, 4, None, None, C.byref(s), BUF, 512, 512, 128, 0, None, 0, None),
        lambda: _native.call("cuda", "bn_kv8_advance", c, 1, None, None),
        lambda: _native.call("cuda", "bn_kv8_dense", c, BUF, BUF, None),
    ):
        with pytest.raises(_native.NativeError, match="bad argument: bn_kv8"):
            call()


def attend(c=None, q=BUF, qs=(512, 512, 128), k=None, tokens=1, heads=4, s=None, out=BUF, os=(512, 512, 128), work=BUF, bytes=1 << 40):
    c, s = cache() if c is None else c, scores() if s is None else s
    return _native.call("cuda", "bn_kv8_attend", C.byref(c), q, *qs, k, 256, 256, 128, None, 256, 256, 128, tokens, heads, None, None, C.byref(s), out, *os, 0, work, bytes, None)


@pytest.mark.parametrize("change", [dict(q=None), dict(k=BUF), dict(out=None), dict(q=BUF + 2), dict(qs=(512, 512, 4)), dict(os=(4, 512, 128)), dict(tokens=-1), dict(tokens=1 << 40), dict(heads=0), dict(heads=3), dict(heads=1 << 20), dict(s=scores(window=-1)), dict(s=scores(softcap=-1.0))])
def test_attend_refuses(change):
    with pytest.raises(_native.NativeError, match="bad argument: bn_kv8_attend"):
        attend(**change)


def test_cache_calls_of_nothing_and_sizes():
    assert attend(tokens=0, q=None, out=None) == 0
    c = C.byref(cache())
    assert _native.call("cuda", "bn_kv8_append", c, None, 256, 256, 128, None, 256, 256, 128, 0, None, None) == 0
    for args in ((None, 256, 256, 128, BUF, 256, 256, 128, 1), (BUF, 256, 256, 4, BUF, 256, 256, 128, 1), (BUF + 2, 256, 256, 128, BUF, 256, 256, 128, 1), (BUF, 256, 256, 128, BUF, 256, 256, 128, -1)):
        with pytest.raises(_native.NativeError, match="bad argument"):
            _native.call("cuda", "bn_kv8_append", c, *args, None, None)
    with pytest.raises(_native.NativeError, match="bad argument"):
        _native.call("cuda", "bn_kv8_advance", c, 1 << 40, None, None)
    with pytest.raises(_native.NativeError, match="bad argument"):
        _native.call("cuda", "bn_kv8_dense", c, BUF + 4, BUF, None)


def test_logits_refuse():
    r = _native.LogitRules(repetition_all=1.0)
    half = _native.LogitRules(seen=BUF, repetition_all=1.0)
    call = lambda x=BUF, batch=1, V=8, rules=r, out=BUF, token=BUF: _native.call("cuda", "bn_logits", x, 1, V, batch, V, C.byref(rules) if rules else None, out, V, token, None)  # noqa: E731
    for change in (dict(x=None), dict(out=None), dict(token=None), dict(batch=-1), dict(batch=1 << 20), dict(V=0), dict(V=1 << 31), dict(rules=None), dict(rules=half)):
        with pytest.raises(_native.NativeError, match="bad argument: bn_logits"):
            call(**change)
    assert call(batch=0, x=None, out=None, token=None) == 0
    count = lambda tokens=BUF, batch=1, n=4, V=8, seen=BUF, counts=BUF: _native.call("cuda", "bn_token_counts", tokens, 1, n, batch, n, None, V, 0, seen, 1, counts, V, None)  # noqa: E731
    for change in (dict(tokens=None), dict(seen=None), dict(counts=None), dict(batch=-1), dict(n=-1), dict(V=0)):
        with pytest.raises(_native.NativeError, match="bad argument: bn_token_counts"):
            count(**change)
    assert count(n=0, tokens=None) == 0


def test_without_a_device_the_calls_raise():
    if torch.cuda.is_available():
        pytest.skip("there is a CUDA device")
    from binade_b200.cuda.attention import KV8Cache
    from binade_b200.cuda.attention import attention as public
    from binade_b200.cuda.logits import TokenCounts, process_logits

    x = torch.zeros((1, 1, 64), dtype=torch.bfloat16)
    for call in (lambda: public(x, x, x), lambda: KV8Cache(1, 1, 1, 64, 64), lambda: TokenCounts(1, 8), lambda: process_logits(torch.zeros((1, 8)))):
        with pytest.raises(RuntimeError, match="needs a CUDA device"):
            call()


# ------------------------------------------------------------------------- the definition that the GPU tests compare with
def test_definition_of_what_is_visible():
    for causal in (True, False):
        for window in (None, 1, 3):
            for prefix in (0, 4):
                got = ref.visible(2, 4, 8, causal=causal, window=window, prefix=prefix)
                for r in range(4):
                    i = 2 + r
                    lo = max(0, i - window + 1) if window else 0
                    hi = min(8, i + window if window else 8, max(i + 1, prefix) if causal else 8)
                    assert got[r].tolist() == [lo <= j < hi for j in range(8)]


def test_definition_of_the_stored_values():
    x = torch.tensor([1.0, -127.0, 63.5, 0.0, 64.5, 2.5, float("nan"), float("inf")], dtype=torch.float64)
    rows = x.to(torch.bfloat16).repeat(16, 8).view(16, 1, 64)
    got = ref.stored(rows, "int8", 16)[0, 0, :8]
    assert got.tolist() == [1.0, -127.0, 64.0, 0.0, 64.0, 2.0, 0.0, 127.0]
    e4m3 = ref.stored(rows, "e4m3", 16)[0, 0, :8]
    scale = 2.0 ** -1
    assert torch.equal(e4m3.float(), (torch.nan_to_num(rows.float()[0, 0, :8], nan=0.0) / scale).clamp(-448, 448).to(torch.float8_e4m3fn).float() * scale)
