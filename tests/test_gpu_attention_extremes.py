"""Attention at the ends of its range: blocks of zeros, sinks, infinities beside masked NaN, caps of all sizes, rows that torch
calls contiguous whatever their stride. Against the definition in 64 bits (attention_reference.py)."""

import math

import pytest
import torch

import attention_reference as ref
from test_gpu_attention import close, gen, normal

pytestmark = pytest.mark.gpu


def status():
    import ctypes

    from binade_b200 import _native

    st = ctypes.c_int(-1)
    _native.call("cuda", "bn_device_status", ctypes.byref(st))
    return st.value


def constant(n, kv, D, value):
    return torch.full((n, kv, D), float(value), dtype=torch.bfloat16, device="cuda")


def check_decode(keys, values, heads, kind, block, new=1, batch=1, **options):
    """keys, values [L, kv, D]: all but the last `new` tokens are held; queries of ones (with scale = 1 / D a
    key's score is its mean) against the definition."""
    from binade_b200.cuda.attention import KV8Cache

    L, kv, D = keys.shape
    cache = KV8Cache(1, batch, kv, D, L, kind=kind, block=block)
    held = L - new
    many = lambda x: x[None].expand(batch, -1, -1, -1)  # noqa: E731
    if held:
        cache.append(0, many(keys[:held]), many(values[:held]))
        cache.advance(held)
    q = torch.ones((batch, new, heads, D), dtype=torch.bfloat16, device="cuda")
    got = cache.attend(0, q, many(keys[held:]), many(values[held:]), scale=1.0 / D, **options)
    want, bound = ref.attend(q[0], ref.stored(keys, kind, block), ref.stored(values, kind, block), held, scale=1.0 / D, **options)
    for b in range(batch):
        close(got[b], want, bound)


# ------------------------------------------------------------------------- values whose scales lie far apart
@pytest.mark.parametrize("kind", ["int8", "e4m3"])
@pytest.mark.parametrize("D,heads,kv,block", [(64, 4, 1, 16), (128, 8, 2, 32), (256, 2, 1, 64)])
@pytest.mark.parametrize("gap", [-20, -4, 0, 2, 3, 4, 8, 12, 20])
def test_decode_over_blocks_of_zero_values(kind, D, heads, kv, block, gap):
    """Keys of weight whose values are all zero stay in the sum of weights: before an open block, before, between and
    behind stored blocks, in one warp and in four, whole and cut into parts."""
    zeros, one = (lambda n: constant(n, kv, D, 0)), (lambda n: constant(n, kv, D, 1))
    for held, new in ((block, 1), (128, 1), (128, 3), (640, 2), (6000 // block * block, 1)):
        check_decode(torch.cat([zeros(held), constant(new, kv, D, gap)]), torch.cat([zeros(held), one(new)]), heads, kind, block, new=new)
    for before, behind in ((128, 0), (0, 256), (320, 704), (4096, 4096)):
        keys = torch.cat([zeros(before), constant(block, kv, D, gap), zeros(behind + 1)])
        values = torch.cat([zeros(before), one(block), zeros(behind + 1)])
        check_decode(keys, values, heads, kind, block)
        check_decode(keys, values, heads, kind, block, softcap=30.0)


@pytest.mark.parametrize("kind", ["int8", "e4m3"])
def test_decode_over_blocks_of_zero_values_in_many_parts_and_batches(kind):
    zeros = lambda n: constant(n, 8, 128, 0)  # noqa: E731
    for L, batch in ((70_016, 1), (2048, 3), (500, 40)):
        for gap in (-3, 3, 9, 15):
            keys = torch.cat([zeros(L), constant(2, 8, 128, gap)])
            values = torch.cat([zeros(L), constant(2, 8, 128, -2)])
            check_decode(keys, values, 32, kind, 32, new=1, batch=batch)
            keys[L // 64 * 32 : L // 64 * 32 + 32] = gap - 2
            values[L // 64 * 32 : L // 64 * 32 + 32] = 3
            check_decode(keys, values, 32, kind, 32, new=2, batch=batch)


@pytest.mark.parametrize("kind", ["int8", "e4m3"])
@pytest.mark.parametrize("D,heads,kv", [(64, 4, 2), (128, 12, 1), (256, 4, 1)])
def test_decode_values_from_the_smallest_to_the_largest(kind, D, heads, kv):
    """Neighbouring blocks of values from 1e-30 to 1e30 with scores that make up for the difference, or do not."""
    g = gen(70)
    for slope in (0.0, -1.0, 1.0):  # nats a factor of e
        keys, values = [], []
        for e in (0, -30, 20, -10, 30, 5, -20, 10, -5, 25):
            keys.append(constant(32, kv, D, slope * e * math.log(10)))
            values.append((normal((32, kv, D), g).float() * 10.0**e).to(torch.bfloat16))
        check_decode(torch.cat(keys + [constant(3, kv, D, 0)]), torch.cat(values + [normal((3, kv, D), g)]), heads, kind, 16, new=2)


@pytest.mark.parametrize("kind", ["int8", "e4m3"])
@pytest.mark.parametrize("D,heads,kv", [(64, 4, 2), (128, 12, 1), (256, 4, 1)])
@pytest.mark.parametrize("size", [1e-25, 1e-20, 1.0, 1e30])
def test_decode_small_values_behind_an_open_token_without_any(D, heads, kv, kind, size):
    """The open block takes the weight and has no values, or ones as small: stored blocks' stay beside it, however small."""
    g = gen(79)
    for gap in (10, 24, 40):
        for open_size in (0.0, size, 1e-3 * size):
            keys = torch.cat([constant(96, kv, D, 0), constant(3, kv, D, gap)])
            values = (torch.cat([normal((96, kv, D), g).abs().float() * size, normal((3, kv, D), g).abs().float() * open_size])).to(torch.bfloat16)
            check_decode(keys, values, heads, kind, 32, new=2)
            check_decode(keys, values, heads, kind, 32, new=2, softcap=100.0)


@pytest.mark.parametrize("kind", ["int8", "e4m3"])
@pytest.mark.parametrize("D,heads,kv,L", [(64, 4, 1, 4100), (128, 4, 1, 9001), (128, 24, 1, 4100), (256, 4, 2, 4100), (128, 4, 1, 300)])
@pytest.mark.parametrize("gap", [6.0, 12.0, 17.0, 18.0])
def test_decode_behind_a_sink(kind, D, heads, kv, L, gap):
    """The first key takes nearly all the weight and has no value: what the others add up to is the output."""
    g = gen(71)
    keys, values = normal((L, kv, D), g, 0.5), (normal((L, kv, D), g) + 1).to(torch.bfloat16)
    keys[0], values[0] = gap, 0
    for block in (16, 64):
        check_decode(keys, values, heads, kind, block)
    order = torch.arange(L, device="cuda").roll(L // 2)  # and in the middle
    check_decode(keys[order], values[order], heads, kind, 32)


@pytest.mark.parametrize("kind", ["int8", "e4m3"])
@pytest.mark.parametrize("D", [64, 128, 256])
def test_decode_values_beside_keys_that_rise_without_any(kind, D):
    """Every other block has zeros for values and, for one head, a score that rises from tile to tile by less than a power of two;
    for another head of the same warp the blocks between them rise by more. The first head's keep their bits."""
    from binade_b200.cuda.attention import KV8Cache

    g = gen(80)
    batch, kv, L = 60, 8, 100 * 128
    key = torch.arange(L, device="cuda")
    zero = key // 16 % 2 == 0
    none = torch.zeros_like(key, dtype=torch.float32)
    halves = torch.stack([torch.where(zero, 0.9 * (key // 128), none), torch.where(zero, none, 3.6 * (key // 128))], dim=1) * math.log(2)
    keys = halves.repeat_interleave(D // 2, 1)[:, None].expand(L, kv, D).to(torch.bfloat16)
    values = torch.where(zero[:, None, None], torch.zeros((), device="cuda"), normal((L, kv, D), g).float().abs()).to(torch.bfloat16)
    cache = KV8Cache(1, batch, kv, D, L + 1, kind=kind, block=16)
    many = lambda x: x[None].expand(batch, -1, -1, -1)  # noqa: E731
    cache.append(0, many(keys), many(values))
    cache.advance(L)
    q = (2 * torch.eye(2, device="cuda").repeat_interleave(D // 2, 1).repeat(kv, 1))[None, None].expand(batch, 1, 2 * kv, D).to(torch.bfloat16)
    last = torch.zeros((1, kv, D), dtype=torch.bfloat16, device="cuda")
    got = cache.attend(0, q, many(last), many(last), scale=1.0 / D)
    want, bound = ref.attend(q[0], ref.stored(torch.cat([keys, last]), kind, 16), ref.stored(torch.cat([values, last]), kind, 16), L, scale=1.0 / D)
    for b in range(batch):
        close(got[b], want, bound)


# ------------------------------------------------------------------------- rows that are computed again
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("softcap", [None, 20.0])
def test_a_score_of_minus_infinity_beside_masked_values_that_are_not_finite(D, softcap):
    """The first visible key has weight 0 whatever a key that is not seen holds."""
    from binade_b200.cuda.attention import KV8Cache, attention

    g = gen(72)
    T = 60
    q, k, v = normal((T, 24, D), g).abs() + 0.5, normal((T, 8, D), g), normal((T, 8, D), g)
    q = q.to(torch.bfloat16)
    k[0, :, 3] = -math.inf
    want, bound = ref.attend(q, k, v, softcap=softcap)
    first = 0 if softcap else 1  # (alone, that key has no weight to give; a cap makes its score finite)
    clean = v.clone()
    v[T - 1, :, 5], v[T - 1, :, D - 2] = math.nan, math.inf
    got = attention(q, k, v, softcap=softcap)
    close(got[first : T - 1], want[first : T - 1], bound[first : T - 1])
    close(attention(q, k, clean, softcap=softcap)[first:], want[first:], bound[first:])
    for batch in (1, 6):  # few rows a key head at a time, and many
        cache = KV8Cache(1, batch, 8, D, 64, block=64)
        got = cache.attend(0, *(x[None].expand(batch, -1, -1, -1).contiguous() for x in (q, k, v)), softcap=softcap)
        for b in range(batch):
            close(got[b, first : T - 1], want[first : T - 1], bound[first : T - 1])


def test_rows_computed_again_repeat_bit_for_bit():
    """Heads of 256: the halves of a row belong to two warps, and a masked infinity may show to one of them alone."""
    from binade_b200.cuda.attention import attention

    g = gen(73)
    T = 700
    q, k, v = normal((T, 4, 256), g), normal((T, 2, 256), g), normal((T, 2, 256), g)
    want, bound = ref.attend(q, k, v)
    v[T - 1, 0, 5], v[T - 1, 1, 200] = math.inf, math.nan
    first = attention(q, k, v)
    close(first[: T - 1], want[: T - 1], bound[: T - 1])
    for _ in range(50):
        assert torch.equal(first[: T - 1], attention(q, k, v)[: T - 1])


# ------------------------------------------------------------------------- caps
@pytest.mark.parametrize("D,heads,kv", [(64, 4, 2), (128, 8, 2), (256, 2, 1)])
@pytest.mark.parametrize("softcap", [2.0**-60, 1e-3, 300.0, 1000.0, 1e4, 1e6, 1e9, 2.0**60])
def test_caps_of_all_sizes(D, heads, kv, softcap):
    from binade_b200.cuda.attention import KV8Cache, attention

    g = gen(74)
    T = 300
    q, k, v = normal((T, heads, D), g, 2.0), normal((T, kv, D), g, 1.5), normal((T, kv, D), g)
    want, bound = ref.attend(q, k, v, softcap=softcap)
    close(attention(q, k, v, softcap=softcap), want, bound)
    stored = [ref.stored(x, "int8", 32) for x in (k, v)]
    for new, batch in ((2, 1), (120, 6)):
        cache = KV8Cache(1, batch, kv, D, T, block=32)
        many = [x[None].expand(batch, -1, -1, -1).contiguous() for x in (q, k, v)]
        cache.append(0, many[1][:, :-new], many[2][:, :-new])
        cache.advance(T - new)
        got = cache.attend(0, *(x[:, -new:] for x in many), softcap=softcap)
        want, bound = ref.attend(q[-new:], *stored, T - new, softcap=softcap)
        for b in range(batch):
            close(got[b], want, bound)


def test_caps_and_scales_that_fp32_does_not_hold_are_refused():
    from binade_b200.cuda.attention import attention

    x = torch.zeros((8, 4, 128), dtype=torch.bfloat16, device="cuda")
    for bad in (dict(softcap=1e-50), dict(softcap=1e39), dict(softcap=2.0**61), dict(softcap=2.0**-61), dict(scale=1e39), dict(scale=-1e39)):
        with pytest.raises(ValueError):
            attention(x, x, x, **bad)


# ------------------------------------------------------------------------- whole numbers
def test_whole_numbers_beyond_32_bits_do_not_wrap():
    from binade_b200.cuda.attention import KV8Cache, attention

    g = gen(75)
    q, k, v = normal((90, 4, 64), g), normal((90, 2, 64), g), normal((90, 2, 64), g)
    everything = torch.tensor([1 << 40], device="cuda")
    want, bound = ref.attend(q, k, v, prefix=1000)
    close(attention(q, k, v, prefix=everything), want, bound)
    offsets = torch.tensor([-(1 << 40), 1 << 33], device="cuda")
    want, bound = ref.attend(q, k, v)
    close(attention(q, k, v, offsets), want, bound)
    cache = KV8Cache(1, 1, 2, 64, 100, block=32)
    cache.append(0, k[None], v[None], torch.tensor([1 << 40], device="cuda"))
    cache.advance(torch.tensor([-(1 << 40)], device="cuda"))
    assert cache.length.tolist() == [0]
    cache.advance(90)
    stored = [ref.stored(x, "int8", 32) for x in (k, v)]
    want, bound = ref.attend(q[-1:], *stored, 89)
    cache.advance(-1)
    close(cache.attend(0, q[None, -1:], k[None, -1:], v[None, -1:], torch.tensor([(1 << 33) + 0], device="cuda"), prefix=everything)[0], want, bound)


# ------------------------------------------------------------------------- strides
def test_one_token_of_rows_with_an_odd_stride():
    """torch calls a tensor contiguous whatever the stride of a dimension of one element."""
    from binade_b200.cuda.attention import KV8Cache, attention

    g = gen(76)
    wide = normal((5, 260), g)
    x = wide[:, :256].unflatten(1, (2, 128))
    for n in (1, 2, 5):
        got = attention(x[:n], x[:n], x[:n])
        want, bound = ref.attend(x[:n], x[:n], x[:n])
        close(got, want, bound)
    for first in (x[:1], x[2:3]):
        cache = KV8Cache(1, 1, 2, 128, 64)
        new = first[None]
        got = cache.attend(0, new, new, new)
        assert torch.equal(got[0], first)
    one = x[:5, None]  # [5, 1, 2, 128]: a batch of single tokens, copied
    cache = KV8Cache(1, 5, 2, 128, 64)
    assert torch.equal(cache.attend(0, one, one, one), one)
    out = torch.empty((1, 260), dtype=torch.bfloat16, device="cuda")[:, :256].unflatten(1, (2, 128))
    attention(x[:1], x[:1], x[:1], out=out)
    assert torch.equal(out, x[:1])


# ------------------------------------------------------------------------- how far a cache moves on
def test_advance_into_a_block_that_is_not_held_is_refused():
    from binade_b200 import _native
    from binade_b200.cuda.attention import KV8Cache

    g = gen(77)
    k, v = normal((3, 60, 1, 64), g), normal((3, 60, 1, 64), g)
    for apart in (True, False):
        _native.call("cuda", "bn_device_status_reset")
        cache = KV8Cache(1, 3, 1, 64, 200, block=16)
        cache.append(0, k[:, :15], v[:, :15])
        cache.advance(15)
        n = 20 if apart else 16
        if apart:
            cache.append(0, k[:, 15:35], v[:, 15:35])
        else:
            cache.attend(0, k[:, 15:31], k[:, 15:31], v[:, 15:31])
        assert status() == 0
        if apart:
            cache.advance(torch.tensor([5, 17, 1], device="cuda"))  # into block 1, which went straight to codes; 2, open; a border
            assert cache.length.tolist() == [15, 32, 16] and status() >> 24 == 2
            _native.call("cuda", "bn_device_status_reset")
            cache.advance(torch.tensor([n, 0, 0], device="cuda"))
            assert cache.length.tolist() == [35, 32, 16] and status() == 0
            got = cache.dense(0)
            for b, L in enumerate((35, 32, 16)):
                for x, y in zip(got, (k, v)):
                    assert torch.equal(x[b, :, :L].transpose(0, 1), ref.stored(y[b, :L], "int8", 16).float())
        else:
            cache.advance(torch.tensor([5, 16, 1], device="cuda"))  # 20 and 31 lie in the open block behind 31 tokens
            assert cache.length.tolist() == [20, 31, 16] and status() == 0


def test_a_sequence_goes_back_as_far_as_its_rows_are_held():
    from binade_b200 import _native
    from binade_b200.cuda.attention import KV8Cache

    _native.call("cuda", "bn_device_status_reset")
    g = gen(78)
    k, v, again = normal((1, 100, 2, 128), g), normal((1, 100, 2, 128), g), normal((1, 100, 2, 128), g)
    cache = KV8Cache(2, 1, 2, 128, 200, block=32)
    at = 0
    for n in (20, 20, 30):  # 20, 40, 70 tokens: blocks 1 and 2 are held as they came, block 0 is codes
        for layer in range(2):
            cache.append(layer, k[:, at : at + n], v[:, at : at + n])
        cache.advance(n)
        at += n
    cache.advance(-20)  # 50, in block 1
    assert cache.length.item() == 50 and status() == 0
    cache.advance(-40)  # 10, in block 0: no
    assert cache.length.item() == 50 and status() >> 24 == 2
    _native.call("cuda", "bn_device_status_reset")
    for layer in range(2):
        cache.append(layer, again[:, :70], again[:, :70])  # 120: blocks 1 and 3 are held
    cache.advance(60)  # 110, in block 3
    assert cache.length.item() == 110
    cache.advance(-5)  # 105: the same
    cache.advance(-40)  # 65, in block 2, which went straight to codes
    assert cache.length.item() == 105 and status() >> 24 == 2
    _native.call("cuda", "bn_device_status_reset")
    cache.advance(-9)  # 96: a border
    assert cache.length.item() == 96
    cache.advance(-40)  # 56, in block 1
    assert cache.length.item() == 56 and status() == 0
    want = [torch.cat([x[0, :50], again[0, :6]]) for x in (k, v)]
    for layer in range(2):
        for got, w in zip(cache.dense(layer), want):
            assert torch.equal(got[0, :, :56].transpose(0, 1), ref.stored(w, "int8", 32).float())
    cache.advance(-24)  # 32, a border; then on, over what was there
    q = normal((1, 12, 4, 128), g)
    for layer in range(2):
        cache.attend(layer, q, again[:, 80:92], again[:, 80:92])
    cache.advance(7)
    want = [torch.cat([x[0, :32], again[0, 80:87]]) for x in (k, v)]
    assert cache.length.item() == 39 and status() == 0
    for got, w in zip(cache.dense(1), want):
        assert torch.equal(got[0, :, :39].transpose(0, 1), ref.stored(w, "int8", 32).float())
    cache.length.zero_()  # the place is free: a new sequence, behind which nothing of the old one may come back
    cache.append(0, k[:, :3], v[:, :3])
    cache.advance(3)
    assert cache.length.item() == 3 and status() == 0
