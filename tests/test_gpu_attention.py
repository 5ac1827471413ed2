"""Attention of prompts, the 8-bit cache and its attention, logits processing: through the public calls, against the
definitions in 64 bits (attention_reference.py, where the bounds are derived)."""

import math

import pytest
import torch

import attention_reference as ref

pytestmark = pytest.mark.gpu


def gen(seed: int):
    return torch.Generator(device="cuda").manual_seed(seed)


def normal(shape, g, scale=1.0):
    return (torch.randn(shape, generator=g, device="cuda") * scale).to(torch.bfloat16)


def slopes_of(heads):
    return torch.tensor([2.0 ** (-8.0 * (h + 1) / heads) for h in range(heads)], device="cuda")


def close(got, want, bound):
    bad = (got.double() - want).abs() > bound
    assert not bad.any(), f"{int(bad.sum())} of {bad.numel()} off, worst {((got.double() - want).abs() / bound).max().item():.2f} of the bound"
    assert torch.isfinite(got).all()


def check_prompt(lens, heads, kv, D, seed=0, prefixes=None, fused=False, behind=0, **options):
    g = gen(seed)
    T = sum(lens) + behind
    if fused:  # views of one projection's output
        qkv = normal((T, (heads + 2 * kv) * D), g, 1.3)
        q, k, v = (x.view(T, -1, D) for x in qkv.split([heads * D, kv * D, kv * D], dim=1))
    else:
        q, k, v = normal((T, heads, D), g, 1.5), normal((T, kv, D), g), normal((T, kv, D), g)
    from binade_b200.cuda.attention import attention

    offsets = torch.tensor([sum(lens[:i]) for i in range(len(lens) + 1)], device="cuda")
    prefix = None if prefixes is None else torch.tensor(prefixes, device="cuda")
    got = attention(q, k, v, offsets, prefix=prefix, **options)
    at = 0
    for n, doc in enumerate(lens):
        if doc:
            rows = slice(at, at + doc)
            want, bound = ref.attend(q[rows], k[rows], v[rows], prefix=prefixes[n] if prefixes else 0, **options)
            close(got[rows], want, bound)
        at += doc
    assert not got[at:].any()
    return q, k, v, offsets, got


# ------------------------------------------------------------------------------------------ prompts
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("heads,kv", [(1, 1), (4, 1), (6, 2), (8, 8), (40, 8)])
@pytest.mark.parametrize("lens", [[1], [2, 0, 3], [127], [128], [129, 64], [31, 300, 1, 7]])
def test_prompt_shapes(D, heads, kv, lens):
    check_prompt(lens, heads, kv, D, seed=D + heads + len(lens))


@pytest.mark.parametrize("options", [dict(softcap=5.0), dict(softcap=50.0, window=33), dict(window=1), dict(window=128), dict(causal=False), dict(causal=False, window=40), dict(scale=0.3), dict(scale=-0.05)])
@pytest.mark.parametrize("D,heads,kv", [(64, 4, 2), (128, 8, 2), (256, 3, 1)])
def test_prompt_options(options, D, heads, kv):
    check_prompt([257, 5, 190], heads, kv, D, seed=3, **options)


@pytest.mark.parametrize("D,heads,kv", [(64, 6, 6), (128, 8, 2), (256, 2, 2)])
@pytest.mark.parametrize("window", [None, 50])
def test_prompt_bias_and_prefix(D, heads, kv, window):
    check_prompt([300, 40, 129], heads, kv, D, seed=4, prefixes=[100, 1000, 0], slopes=slopes_of(heads), window=window)


@pytest.mark.parametrize("D", [64, 128, 256])
def test_prompt_long(D):
    check_prompt([1500, 777], 4, 2, D, seed=5)
    check_prompt([2100], 2, 1, D, seed=6, softcap=30.0, slopes=slopes_of(2), window=700)


def test_prompt_in_place_of_views_and_rows_behind():
    check_prompt([140, 33], 8, 2, 128, seed=7, fused=True, behind=60)
    check_prompt([40], 4, 4, 64, seed=8, fused=True, behind=3)
    from binade_b200.cuda.attention import attention

    g = gen(9)
    q, k, v = normal((200, 4, 128), g), normal((200, 2, 128), g), normal((200, 2, 128), g)
    k[150:], v[150:] = math.nan, math.inf
    offsets = torch.tensor([10, 150], device="cuda", dtype=torch.int32)
    out = torch.full((200, 4, 128), 7.0, dtype=torch.bfloat16, device="cuda")
    assert attention(q, k, v, offsets, out=out) is out
    want, bound = ref.attend(q[10:150], k[10:150], v[10:150])
    close(out[10:150], want, bound)
    assert (out[:10] == 7).all() and (out[150:] == 7).all()
    assert not attention(q, k, v, offsets)[150:].any()
    # offsets that leave the tokens, or fall, read and write nothing outside
    attention(q, k, v, torch.tensor([0, 50, 40, 500], device="cuda", dtype=torch.int32))
    attention(q, k, v, torch.tensor([-7, 50, 1 << 30], device="cuda", dtype=torch.int32), window=3)
    torch.cuda.synchronize()
    # rows that start on odd places: copied
    odd = normal((50, 4, 130), g)[..., 1:129]
    got = attention(odd, odd[:, :2], odd[:, 2:])
    want, bound = ref.attend(odd, odd[:, :2], odd[:, 2:])
    close(got, want, bound)


@pytest.mark.parametrize("D", [64, 128, 256])
def test_prompt_masked_keys_may_hold_anything(D):
    """A token of NaN or infinite keys and values shows only in the queries that see it."""
    from binade_b200.cuda.attention import attention

    g = gen(10)
    T, spoiled = 300, 200
    q, k, v = normal((T, 4, D), g), normal((T, 2, D), g), normal((T, 2, D), g)
    want, bound = ref.attend(q, k, v, window=64)
    k[spoiled, 0], v[spoiled, 0, 5], v[spoiled, 1, 7] = math.nan, math.nan, -math.inf
    got = attention(q, k, v, window=64)
    rows = torch.arange(T, device="cuda")
    sees = (rows >= spoiled) & (rows < spoiled + 64)
    close(got[~sees], want[~sees], bound[~sees])
    assert torch.isnan(got[sees][:, :2]).all()
    close(got[sees][:, 2:, 8:], want[sees][:, 2:, 8:], bound[sees][:, 2:, 8:])
    assert (got[sees][:, 2:, 7] == -math.inf).all()


def test_prompt_large_scores():
    """Scores of thousands, and all alike: the running maximum carries both."""
    from binade_b200.cuda.attention import attention

    g = gen(11)
    q, k, v = normal((260, 2, 128), g, 60.0), normal((260, 2, 128), g, 20.0), normal((260, 2, 128), g)
    got = attention(q, k, v)
    want, bound = ref.attend(q, k, v)
    close(got, want, bound)
    k[:] = 0
    want, bound = ref.attend(q, k, v)
    close(attention(q, k, v), want, bound)
    v[:] = 1e37
    want, bound = ref.attend(q, k, v)
    close(attention(q, k, v), want, bound)


def test_prompt_graph_stream_and_repeat():
    from binade_b200.cuda.attention import attention

    g = gen(12)
    q, k, v = normal((400, 8, 128), g), normal((400, 2, 128), g), normal((400, 2, 128), g)
    offsets = torch.tensor([0, 150, 400], device="cuda", dtype=torch.int32)
    first = attention(q, k, v, offsets)
    assert all(torch.equal(first, attention(q, k, v, offsets)) for _ in range(5))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = attention(q, k, v, offsets)
    graph.replay()
    assert torch.equal(y, first)
    offsets.copy_(torch.tensor([0, 399, 400], device="cuda"))
    q.mul_(0.5)
    graph.replay()
    want, bound = ref.attend(q[:399], k[:399], v[:399])
    close(y[:399], want, bound)
    assert torch.equal(y[399], v[399].repeat_interleave(4, 0))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        z = attention(q, k, v, offsets)
    side.synchronize()
    assert torch.equal(z, y)


# ------------------------------------------------------------------------------------------ the cache
class History:
    """A KV8Cache and the tokens that went into it."""

    def __init__(self, batch, kv, D, max_seq, kind="int8", block=32, layers=1):
        from binade_b200.cuda.attention import KV8Cache

        self.cache = KV8Cache(layers, batch, kv, D, max_seq, kind=kind, block=block)
        self.k = [torch.zeros((0, kv, D), dtype=torch.bfloat16, device="cuda") for _ in range(batch)]
        self.v = [torch.zeros((0, kv, D), dtype=torch.bfloat16, device="cuda") for _ in range(batch)]

    def tokens(self, counts, g, scale=1.0):
        n, c = max(counts), self.cache
        k, v = normal((c.batch, n, c.kv_heads, c.head_dim), g, scale), normal((c.batch, n, c.kv_heads, c.head_dim), g, scale)
        for b, have in enumerate(counts):
            self.k[b], self.v[b] = torch.cat([self.k[b], k[b, :have]]), torch.cat([self.v[b], v[b, :have]])
        return k, v, torch.tensor(counts, device="cuda", dtype=torch.int32)

    def append(self, counts, g, scale=1.0, layer=0):
        k, v, n = self.tokens(counts, g, scale)
        self.cache.append(layer, k, v, n)
        self.cache.advance(n)

    def stored(self, b):
        return tuple(ref.stored(x[b], self.cache.kind, self.cache.block) for x in (self.k, self.v))

    def check_attend(self, counts, heads, g, layer=0, prefixes=None, apart=False, qscale=1.5, **options):
        """New tokens through attend (or append, then attend) against the definition; moves on."""
        c = self.cache
        k, v, n = self.tokens(counts, g)
        q = normal((c.batch, max(counts), heads, c.head_dim), g, qscale)
        prefix = None if prefixes is None else torch.tensor(prefixes, device="cuda")
        if apart:
            c.append(layer, k, v, n)
            got = c.attend(layer, q, counts=n, prefix=prefix, **options)
        else:
            got = c.attend(layer, q, k, v, n, prefix=prefix, **options)
        for b, have in enumerate(counts):
            if have:
                ks, vs = self.stored(b)
                want, bound = ref.attend(q[b, :have], ks, vs, ks.shape[0] - have, prefix=prefixes[b] if prefixes else 0, **options)
                close(got[b, :have], want, bound)
            assert not got[b, have:].any()
        c.advance(n)
        return q, got


@pytest.mark.parametrize("kind", ["int8", "e4m3"])
@pytest.mark.parametrize("block", [16, 32, 64])
@pytest.mark.parametrize("D", [64, 128, 256])
def test_cache_holds_what_the_definition_says(kind, block, D):
    """Whatever way the tokens came: in one call, one by one, in odd pieces, ragged over the batch."""
    g = gen(D + block)
    h = History(3, 2, D, 300, kind, block)
    for counts in ([5, 0, 1], [block, block - 1, 2 * block], [1, 1, 1], [2, 0, block + 3], [70, 100, 40], [1, 1, 0], [17, 64, 63]):
        h.append(counts, g, scale=math.exp(counts[0] % 5 - 2))
        k, v = h.cache.dense(0)
        for b in range(3):
            n = h.k[b].shape[0]
            for got, want in zip((k, v), h.stored(b)):
                assert torch.equal(got[b, :, :n].transpose(0, 1).double().float(), want.float()), (counts, b)
                assert not got[b, :, n:].any()
    assert h.cache.length.tolist() == [x.shape[0] for x in h.k]


@pytest.mark.parametrize("kind", ["int8", "e4m3"])
def test_cache_codes_of_awkward_values(kind):
    """Zeros, subnormals, values near the largest, ties between codes, NaN and infinities, against the definition."""
    from binade_b200.cuda.attention import KV8Cache

    D, block = 64, 16
    every = torch.arange(1 << 16, dtype=torch.int32, device="cuda").to(torch.int16).view(torch.bfloat16)  # all BF16 values
    g = gen(20)
    blocks = [every.view(-1, block, D)[i] for i in range(64)]
    blocks += [torch.zeros((block, D), dtype=torch.bfloat16, device="cuda"), torch.full((block, D), 1e-40, device="cuda").to(torch.bfloat16), torch.full((block, D), 3.3e38, device="cuda").to(torch.bfloat16)]
    half = (torch.arange(block * D, device="cuda") % 255 - 127).float().view(block, D) * 0.5  # amax 63.5: codes and halves between them
    blocks += [half.to(torch.bfloat16), (half * 2).to(torch.bfloat16), torch.full((block, D), math.nan, device="cuda").to(torch.bfloat16)]
    mixed = normal((block, D), g)
    mixed[3, 5], mixed[4, 6], mixed[5, 7] = math.nan, math.inf, -math.inf
    blocks += [mixed] + [normal((block, D), g, 2.0 ** (i - 20)) for i in range(40)]
    x = torch.cat(blocks)[:, None, :]
    c = KV8Cache(1, 1, 1, D, x.shape[0], kind=kind, block=block)
    c.append(0, x[None], x[None].neg().contiguous())
    c.advance(x.shape[0])
    k, v = c.dense(0)
    want = ref.stored(x, kind, block)
    assert torch.equal(k[0, 0].double(), want[:, 0].float().double())
    assert torch.equal(v[0, 0].double(), -want[:, 0].float().double())


@pytest.mark.parametrize("kind", ["int8", "e4m3"])
@pytest.mark.parametrize("D,heads,kv", [(64, 4, 4), (128, 8, 2), (128, 32, 1), (256, 6, 2)])
@pytest.mark.parametrize("block", [16, 64])
def test_decode_over_the_cache(kind, D, heads, kv, block):
    g = gen(heads + D)
    h = History(4, kv, D, 700, kind, block)
    h.append([0, 1, block - 1, 515], g)
    h.check_attend([1, 1, 1, 1], heads, g)
    h.check_attend([1, 0, 1, 1], heads, g, apart=True)
    h.check_attend([3, 2, 0, 1], heads, g)
    h.append([100, 77, 64, 1], g)
    h.check_attend([1, 1, 1, 1], heads, g)
    h.check_attend([2, 5, 5, 1], heads, g, apart=True)


@pytest.mark.parametrize("options", [dict(softcap=4.0), dict(window=1), dict(window=50, softcap=30.0), dict(window=300), dict(scale=0.02), dict(causal=False), dict(causal=False, window=7)])
@pytest.mark.parametrize("D,heads,kv,kind", [(64, 3, 1, "e4m3"), (128, 8, 2, "int8"), (256, 4, 4, "int8")])
def test_decode_options(options, D, heads, kv, kind):
    g = gen(30)
    h = History(2, kv, D, 900, kind, 32)
    h.append([200, 777], g)
    h.check_attend([1, 1], heads, g, **options)
    h.check_attend([4, 3], heads, g, **options)
    h.check_attend([1, 1], heads, g, slopes=slopes_of(heads), prefixes=[0, 1000], **options)


@pytest.mark.parametrize("kind,D,heads,kv,block", [("int8", 128, 8, 2, 32), ("e4m3", 64, 6, 2, 16), ("int8", 256, 4, 2, 64), ("e4m3", 128, 4, 4, 64)])
@pytest.mark.parametrize("options", [{}, dict(softcap=20.0, window=100), dict(causal=False)])
def test_chunks_over_the_cache(kind, D, heads, kv, block, options):
    g = gen(31)
    h = History(3, kv, D, 1200, kind, block)
    h.check_attend([33, 1, 130], heads, g, **options)
    h.append([300, 0, 64], g)
    h.check_attend([17, 129, 200], heads, g, apart=True, **options)
    h.check_attend([256, 300, 0], heads, g, slopes=slopes_of(heads), prefixes=[10, 500, 3], **options)


@pytest.mark.parametrize("kind", ["int8", "e4m3"])
@pytest.mark.parametrize("D,block", [(64, 64), (128, 16), (256, 32)])
@pytest.mark.parametrize("options", [{}, dict(softcap=10.0), dict(window=90), dict(scale=-0.1)])
def test_wide_batches_of_chunks(kind, D, block, options):
    """Many rows, enough of them for the kernel that reads the keys once: blocks that end inside a tile of keys, sequences
    without tokens, heads of a group that is no power of two, and values that are not finite in the open block."""
    g = gen(D + block)
    h = History(5, 8, D, 900, kind, block)
    h.append([0, 3, 200, 129, 500], g)
    h.check_attend([150, 97, 1, 0, 64], 24, g, **options)
    h.check_attend([64, 130, 33, 200, 128], 24, g, apart=True, **options)
    h.check_attend([30, 100, 97, 10, 3], 8, g, **options)
    q, k, v = normal((5, 100, 16, D), g), normal((5, 100, 8, D), g), normal((5, 100, 8, D), g)
    held = h.cache.length.tolist()
    at = [max(0, (n + 100) // block * block - n) for n in held]  # the first token of each sequence that stays in the open block
    for b in range(5):
        if at[b] < 100:
            k[b, at[b], 2], v[b, at[b], 3, 5] = math.nan, math.inf
    got = h.cache.attend(0, q, k, v, **options)
    for b in range(5):
        if at[b] >= 100:
            continue
        clean = [torch.cat([x, y[b]]) for x, y in ((h.k[b], k), (h.v[b], v))]
        stored = [ref.stored(torch.nan_to_num(x.float(), nan=0.0, posinf=0.0).to(torch.bfloat16), kind, block) for x in clean]
        want, bound = ref.attend(q[b], *stored, held[b], **options)
        touched = torch.zeros((100, 16), dtype=torch.bool, device="cuda")
        end = at[b] + (options.get("window") or 1000)
        touched[at[b] : end, 4:8] = True  # heads of key heads 2 and 3
        close(got[b][~touched], want[~touched], bound[~touched])
        assert torch.isnan(got[b, at[b] : end, 4:6]).all() and (got[b, at[b] : end, 6:8, 5] == math.inf).all()
        close(got[b, at[b] : end, 6:8, 6:], want[at[b] : end, 6:8, 6:], bound[at[b] : end, 6:8, 6:])


@pytest.mark.parametrize("heads,kv", [(40, 1), (64, 1), (24, 2), (12, 12)])
def test_groups_of_many_sizes(heads, kv):
    check_prompt([70, 130], heads, kv, 128, seed=heads)
    g = gen(heads)
    h = History(2, kv, 128, 400, "int8", 32)
    h.append([70, 200], g)
    for counts in ([1, 1], [2, 1], [16, 9], [17, 3], [1, 0]):
        h.check_attend(counts, heads, g)


def test_steps_over_block_borders_equal_append_and_attend():
    """A step that appends inside the attention's launch gives what append and attend apart give, bit for bit in what
    is stored, at every place of a block, drafts that fill one among them."""
    from binade_b200.cuda.attention import KV8Cache

    g = gen(60)
    for block, D, kind in ((16, 64, "int8"), (64, 128, "e4m3"), (32, 256, "int8")):
        a, b = (KV8Cache(1, 3, 2, D, 600, kind=kind, block=block) for _ in range(2))
        for step in range(60):
            n = 1 + step * 7 % 16
            q, k, v = normal((3, n, 4, D), g), normal((3, n, 2, D), g), normal((3, n, 2, D), g)
            counts = torch.tensor([n, max(0, n - 3), step % 2], device="cuda")
            x = a.attend(0, q, k, v, counts)
            b.append(0, k, v, counts)
            y = b.attend(0, q, counts=counts)
            a.advance(counts), b.advance(counts)
            assert torch.allclose(x.float(), y.float(), atol=2e-2, rtol=2e-2)
            for s, t in ((a.k, b.k), (a.v, b.v), (a.k_scale, b.k_scale), (a.v_scale, b.v_scale), (a.k_tail, b.k_tail), (a.v_tail, b.v_tail), (a.length, b.length), (a._side, b._side)):
                assert torch.equal(s, t)
            assert not a._tickets.any()


def test_decode_long_and_wide():
    """A cache of more than 2^31 codes in one array, its last sequence behind that border."""
    g = gen(32)
    h = History(5, 8, 128, 500_000, "int8", 64)
    assert h.cache.k.numel() > 1 << 31
    h.append([1, 0, 64, 3, 3000], g)
    h.check_attend([1, 1, 1, 1, 1], 32, g)
    h.check_attend([1, 1, 70, 1, 100], 32, g)


def test_decode_values_of_all_sizes():
    """Blocks whose scales lie far apart, scores of thousands, keys all alike."""
    g = gen(33)
    h = History(1, 2, 128, 600, "int8", 16)
    for i in range(20):
        h.append([16], g, scale=10.0 ** (i % 7 - 3))
    h.append([13], g)
    h.check_attend([1], 8, g, qscale=1e-3)
    h.check_attend([1], 8, g, qscale=300.0)
    h.check_attend([1], 8, g, qscale=0.0)


def test_cache_values_that_are_not_finite():
    """In the open block, as they are, they show in the queries that see them and in no other; a stored
    block has none."""
    from binade_b200.cuda.attention import KV8Cache

    g = gen(34)
    for D, tokens in ((64, 40), (128, 3), (256, 21), (128, 70)):
        c = KV8Cache(1, 1, 2, D, 256, block=64)
        past = 120 if tokens < 64 else 3
        k, v = normal((1, past, 2, D), g), normal((1, past, 2, D), g)
        past_kv = (k, v)
        c.append(0, k, v)
        c.advance(past)
        q, k, v = normal((1, tokens, 4, D), g), normal((1, tokens, 2, D), g), normal((1, tokens, 2, D), g)
        whole = [ref.stored(torch.cat([a[0], b[0]]), "int8", 64) for a, b in zip(past_kv, (k, v))]
        want, bound = ref.attend(q[0], *whole, past)
        close(c.attend(0, q, k, v)[0], want, bound)
        at = tokens - 2
        k[0, at, 0], v[0, at, 1, 3] = math.nan, math.inf
        got = c.attend(0, q, k, v)[0]
        close(got[:at], want[:at], bound[:at])
        if past + at >= (past + tokens) // 64 * 64:
            assert torch.isnan(got[at:, :2]).all() and (got[at:, 2:, 3] == math.inf).all()
            close(got[at:, 2:, 4:], want[at:, 2:, 4:], bound[at:, 2:, 4:])


@pytest.mark.parametrize("block", [16, 64])
def test_cache_keeps_the_accepted_part_of_a_draft(block):
    """Drafts of up to a block of tokens, of which a part is kept, over block borders: as if only that part
    had come. Appending twice changes nothing."""
    from binade_b200.cuda.attention import KV8Cache

    g = gen(37)
    a, b = (KV8Cache(1, 2, 1, 64, 41 * block, block=block) for _ in range(2))
    r = torch.Generator().manual_seed(5)
    for step in range(40):
        n = int(torch.randint(1, block + 1, (1,), generator=r))
        keep = torch.randint(0, n + 1, (2,), generator=r).to(torch.int32).cuda()
        k, v, q = normal((2, n, 1, 64), g), normal((2, n, 1, 64), g), normal((2, n, 2, 64), g)
        for _ in range(1 + step % 2):
            a.append(0, k, v)
        a.advance(keep)
        b.append(0, k, v, keep)
        b.advance(keep)
        assert torch.equal(a.length, b.length)
        for x, y in zip(a.dense(0), b.dense(0)):
            assert torch.equal(x, y)
        assert torch.equal(a.attend(0, q, k, v), b.attend(0, q, k, v))


def test_cache_capacity_rows_left_alone_and_status():
    import ctypes

    from binade_b200 import _native
    from binade_b200.cuda.attention import KV8Cache

    def status():
        st = ctypes.c_int(-1)
        _native.call("cuda", "bn_device_status", ctypes.byref(st))
        return st.value

    g = gen(35)
    c = KV8Cache(1, 2, 1, 64, 70, block=32)
    k, v = normal((2, 80, 1, 64), g), normal((2, 80, 1, 64), g)
    counts = torch.tensor([70, 20], device="cuda")
    c.append(0, k, v, counts)
    c.advance(counts)
    assert status() == 0 and c.length.tolist() == [70, 20]
    q = normal((2, 3, 2, 64), g)
    out = torch.full((2, 3, 2, 64), 7.0, dtype=torch.bfloat16, device="cuda")
    c.attend(0, q, k[:, :3], v[:, :3], torch.tensor([2, 1], device="cuda"), out=out)
    assert (out[0] == 7).all() and (out[1, 1:] == 7).all()  # no room for a token of the first sequence
    whole = [ref.stored(torch.cat([x[1, :20], x[1, :1]]), "int8", 32) for x in (k, v)]
    want, bound = ref.attend(q[1, :1], *whole, 20)
    close(out[1, :1], want, bound)
    assert status() >> 24 & 1
    _native.call("cuda", "bn_device_status_reset")
    assert status() == 0
    c.advance(5)
    assert c.length.tolist() == [70, 25]
    # an empty cache and no new tokens: nothing is seen, zeros
    e = KV8Cache(1, 2, 1, 64, 64)
    assert not e.attend(0, q, k[:, :3], v[:, :3], torch.zeros(2, dtype=torch.int32, device="cuda")).any()


def test_cache_layers_streams_graphs():
    """Layers lie apart; a captured step replays as the sequences grow, over block borders; two graphs do not meet."""
    from binade_b200.cuda.attention import KV8Cache

    g = gen(36)
    B, kv, heads, D, steps = 3, 2, 8, 128, 40
    a, b = (KV8Cache(2, B, kv, D, 200, block=16) for _ in range(2))
    k, v, q = normal((steps, 2, B, 1, kv, D), g), normal((steps, 2, B, 1, kv, D), g), normal((steps, 2, B, 1, heads, D), g)
    want = []
    for s in range(steps):
        want.append([a.attend(l, q[s, l], k[s, l], v[s, l]) for l in range(2)])
        a.advance(1)
    buf = [torch.empty_like(x[0]) for x in (q, k, v)]
    graphs, outs = [], []
    for _ in range(2):  # two graphs of the same step
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append([b.attend(l, buf[0][l], buf[1][l], buf[2][l]) for l in range(2)])
            b.advance(1)
        graphs.append(graph)
    for s in range(steps):
        for x, y in zip(buf, (q, k, v)):
            x.copy_(y[s])
        graphs[s % 2].replay()
        assert all(torch.equal(x, y) for x, y in zip(outs[s % 2], want[s]))
    assert torch.equal(a.length, b.length) and torch.equal(a.k, b.k) and torch.equal(a.v_scale, b.v_scale)
    # attending again on another stream, without moving on
    a.advance(-1)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        again = a.attend(1, q[-1, 1])
    side.synchronize()
    assert torch.equal(again, want[-1][1])


def test_refusals():
    from binade_b200.cuda.attention import KV8Cache, attention
    from binade_b200.cuda.logits import TokenCounts, process_logits

    x = torch.zeros((8, 4, 128), dtype=torch.bfloat16, device="cuda")
    for bad in (
        lambda: attention(x.float(), x, x),
        lambda: attention(x, x[:, :3], x[:, :3]),
        lambda: attention(x, x[:7], x[:7]),
        lambda: attention(x[..., :96], x[..., :96], x[..., :96]),
        lambda: attention(x.cpu(), x, x),
        lambda: attention(x, x.cpu(), x),
        lambda: attention(x, x, x, torch.tensor([0, 8])),
        lambda: attention(x, x, x, torch.tensor([0.0, 8.0], device="cuda")),
        lambda: attention(x, x, x, softcap=0.0),
        lambda: attention(x, x, x, softcap=math.nan),
        lambda: attention(x, x, x, window=0),
        lambda: attention(x, x, x, scale=math.inf),
        lambda: attention(x, x, x, slopes=torch.ones(3, device="cuda")),
        lambda: attention(x, x, x, prefix=torch.ones(2, device="cuda", dtype=torch.int32)),
        lambda: attention(x, x, x, out=x),
        lambda: attention(x, x, x, out=torch.empty((8, 4, 128), device="cuda")),
        lambda: attention(x, x, x, out=torch.empty((1, 4, 128), dtype=torch.bfloat16, device="cuda").expand(8, 4, 128)),
        lambda: attention(x.clone().requires_grad_(), x, x),
        lambda: KV8Cache(1, 1, 1, 96, 64),
        lambda: KV8Cache(1, 1, 1, 64, 64, block=48),
        lambda: KV8Cache(1, 1, 1, 64, 64, kind="fp8"),
        lambda: KV8Cache(0, 1, 1, 64, 64),
        lambda: KV8Cache(1, 1, 1, 64, 64, device="cpu"),
    ):
        with pytest.raises(ValueError):
            bad()
    c = KV8Cache(2, 2, 2, 128, 64)
    t = torch.zeros((2, 3, 2, 128), dtype=torch.bfloat16, device="cuda")
    for bad in (
        lambda: c.append(2, t, t),
        lambda: c.append(-1, t, t),
        lambda: c.append(0, t[:1], t[:1]),
        lambda: c.append(0, t, t[:, :2]),
        lambda: c.append(0, t.half(), t.half()),
        lambda: c.append(0, t, t, torch.tensor([1, 1])),
        lambda: c.append(0, t, t, torch.tensor([1], device="cuda")),
        lambda: c.attend(0, t[:, :, :1]),
        lambda: c.attend(0, t, t),
        lambda: c.attend(0, t, t[:, :2], t[:, :2]),
        lambda: c.attend(0, t, t, t, out=t),
        lambda: c.advance(torch.ones(3, device="cuda", dtype=torch.int32)),
    ):
        with pytest.raises(ValueError):
            bad()
    assert attention(x[:0], x[:0], x[:0]).shape == (0, 4, 128)
    assert c.attend(0, t[:, :0]).shape == (2, 0, 2, 128)
    y = torch.zeros((2, 100), device="cuda")
    counts = TokenCounts(2, 100)
    for bad in (
        lambda: process_logits(y.double()),
        lambda: process_logits(y[0]),
        lambda: process_logits(y.cpu()),
        lambda: process_logits(y, repetition=1.2),
        lambda: process_logits(y, counts, repetition=0.0),
        lambda: process_logits(y, TokenCounts(3, 100), presence=1.0),
        lambda: process_logits(y, counts, presence=torch.ones(3, device="cuda")),
        lambda: process_logits(y, bias=torch.ones(99, device="cuda")),
        lambda: process_logits(y, bias=torch.ones(100, device="cuda", dtype=torch.bfloat16)),
        lambda: process_logits(y, mask=torch.ones(4, device="cuda")),
        lambda: process_logits(y, mask=torch.ones(3, device="cuda", dtype=torch.int32)),
        lambda: process_logits(y, out=torch.empty((2, 100), dtype=torch.bfloat16, device="cuda")),
        lambda: process_logits(y, out=y[:1].expand(2, 100)),
        lambda: process_logits(y[:, :99], out=y[:, 1:]),
        lambda: process_logits(y.clone().requires_grad_()),
        lambda: counts.add(torch.zeros((3, 1), dtype=torch.int64, device="cuda")),
        lambda: counts.add(torch.zeros((2, 1), device="cuda")),
        lambda: counts.add(torch.zeros((2, 1), dtype=torch.int64)),
        lambda: counts.add(torch.zeros((2, 1), dtype=torch.int64, device="cuda"), lengths=torch.ones(3, dtype=torch.int32, device="cuda")),
        lambda: counts.clear(2),
        lambda: counts.clear(torch.tensor([0])),
        lambda: TokenCounts(0, 5),
        lambda: TokenCounts(1, 5, device="cpu"),
    ):
        with pytest.raises(ValueError):
            bad()


# ------------------------------------------------------------------------------------------ logits
def bits_of(allowed: torch.Tensor) -> torch.Tensor:
    """bool [.., V] -> int32 words."""
    V = allowed.shape[-1]
    padded = torch.nn.functional.pad(allowed, (0, -V % 32)).reshape(*allowed.shape[:-1], -1, 32).long()
    words = (padded << torch.arange(32, device=allowed.device)).sum(-1)
    return torch.where(words >= 1 << 31, words - (1 << 32), words).to(torch.int32)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("batch,V", [(1, 1), (3, 2), (2, 31), (5, 33), (1, 2047), (2, 8192), (3, 50257), (4, 128256)])
@pytest.mark.parametrize("what", ["none", "penalties", "all", "rows"])
def test_logits(dtype, batch, V, what):
    """Bound: three roundings to fp32 on the way, each at most 2^-24 of what it rounds; the token is the first largest of what came out."""
    from binade_b200.cuda.logits import TokenCounts, process_logits

    g = gen(V + batch)
    x = (torch.randn((batch, V), generator=g, device="cuda") * 3).to(dtype)
    said = TokenCounts(batch, V)
    prompt = torch.randint(-2, V + 2, (batch, 50), generator=g, device="cuda")
    answer = torch.randint(0, max(1, V // 4), (batch, 70), generator=g, device="cuda").to(torch.int32)
    lengths = torch.tensor([(7 * b) % 71 for b in range(batch)], device="cuda")
    said.add(prompt, prompt=True)
    said.add(answer, lengths=lengths)
    said.add(answer[:, 0])
    seen, counts = torch.zeros((batch, V), dtype=torch.bool), torch.zeros((batch, V), dtype=torch.int64)
    for b in range(batch):
        for t in prompt[b].tolist():
            if 0 <= t < V:
                seen[b, t] = True
        for t in answer[b, : lengths[b]].tolist() + [answer[b, 0].item()]:
            seen[b, t] = True
            counts[b, t] += 1
    seen, counts = seen.cuda(), counts.cuda()
    assert torch.equal(said.counts, counts.int())
    r, p, f = (torch.rand(batch, generator=g, device="cuda") + o for o in (1.0, -0.3, 0.1))
    bias = mask = allowed = None
    kw = {}
    if what == "penalties":
        kw = dict(repetition=1.25, presence=0.5, frequency=0.25)
        r, p, f = (torch.full((batch,), c, device="cuda") for c in (1.25, 0.5, 0.25))
    elif what == "none":
        r, p, f = torch.ones_like(r), torch.zeros_like(p), torch.zeros_like(f)
    else:
        shape = (V,) if what == "all" else (batch, V)
        bias = torch.randn(shape, generator=g, device="cuda")
        allowed = torch.rand(shape, generator=g, device="cuda") < 0.5
        kw = dict(repetition=r, presence=p, frequency=f, bias=bias, mask=bits_of(allowed))
        if what == "rows" and batch > 1:
            allowed[1] = False  # nothing is left
            kw["mask"] = bits_of(allowed)
        allowed = allowed.expand(batch, V)
    got, token = process_logits(x, said if kw else None, **kw)
    want = ref.logits(x, seen, counts, r, p, f, bias, allowed)
    bound = 1.001 * 2.0**-24 * (3 * x.double().abs() * r.double()[:, None] + 4 * (f.abs()[:, None] * counts + p.abs()[:, None]) + (bias.abs().double() if bias is not None else 0) + 1e-30)
    assert torch.equal(torch.isinf(got), torch.isinf(want))
    ok = torch.isfinite(want)
    assert ((got.double() - want).abs() <= bound)[ok].all()
    top = got.amax(dim=1)
    for b in range(batch):
        expect = -1 if top[b] == -math.inf else int((got[b] == top[b]).nonzero()[0])
        assert token[b].item() == expect
    if dtype == torch.float32:
        inplace = x.clone()
        again, same = process_logits(inplace, said if kw else None, out=inplace, **kw)
        assert again is inplace and torch.equal(again, got) and torch.equal(same, token)


def test_logits_strides_nan_and_graph():
    from binade_b200.cuda.logits import TokenCounts, process_logits

    g = gen(50)
    wide = torch.randn((4, 1003), generator=g, device="cuda")
    x = wide[:, 1:1000]  # rows start anywhere
    got, token = process_logits(x)
    assert torch.equal(got, x) and torch.equal(token, x.argmax(1))
    out = torch.zeros((4, 1002), device="cuda")
    process_logits(x.to(torch.bfloat16), out=out[:, 2:1001])
    assert torch.equal(out[:, 2:1001], x.to(torch.bfloat16).float()) and not out[:, :2].any() and not out[:, 1001:].any()
    allowed = torch.ones((4, 999), dtype=torch.bool, device="cuda")
    allowed[:, 10] = False
    y = x.clone()
    y[:, 10], y[1, 20], y[2] = math.nan, math.inf, math.nan
    got, token = process_logits(y, mask=bits_of(allowed))
    assert (got[:, 10] == -math.inf).all() and token[1] == 20 and token[2] == -1 and torch.isnan(got[2, 11:]).all()
    assert torch.equal(token[[0, 3]], got[[0, 3]].argmax(1))
    equal = torch.zeros((2, 40000), device="cuda")
    equal[1, :39999] = -1
    assert process_logits(equal)[1].tolist() == [0, 39999]

    said = TokenCounts(4, 999)
    buf, nxt = y.clone(), torch.zeros(4, dtype=torch.int64, device="cuda")

    def step():
        z, t = process_logits(buf, said, frequency=0.5, repetition=1.1, mask=bits)
        nxt.copy_(t)
        said.add(nxt)
        return z

    bits = bits_of(allowed)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        z = step()
    said.clear()
    buf.copy_(torch.randn((4, 999), generator=g, device="cuda"))
    picks = []
    for _ in range(30):
        graph.replay()
        picks.append(nxt.clone())
    said.clear()
    for p in picks:
        step()
        assert torch.equal(nxt, p)
    assert torch.equal(said.counts.sum(1), torch.full((4,), 30, device="cuda"))
    said.clear(2)
    assert not said.counts[2].any() and not said.seen[2].any() and said.counts[1].any()
