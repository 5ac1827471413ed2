"""The decoder on a cache in 8 bits: prompts in one pass, steps, drafts of a second turn, and rules on the logits, run
together as a serving loop runs them; attention inside is compared with the definition in 64 bits."""

import pytest
import torch

import attention_reference as ref

pytestmark = pytest.mark.gpu


def tiny(max_seq=160):
    from binade_b200.cuda.llama import LlamaShape

    return LlamaShape(layers=2, hidden=256, ffn=512, heads=4, kv_heads=2, head_dim=64, vocab=512, max_seq=max_seq)


def prompt_of(n, seed=1):
    return torch.randint(0, 512, (n,), device="cuda", generator=torch.Generator(device="cuda").manual_seed(seed))


class PlainCache:
    """The calls that a decoder makes of a KV8Cache, from the definition."""

    def __init__(self, layers, kind, block):
        self.k, self.v, self.kind, self.block = [None] * layers, [None] * layers, kind, block
        self.held = 0
        self.length = torch.zeros(1, dtype=torch.int32, device="cuda")

    def append(self, layer, k, v):
        old = (self.k[layer][: self.held], self.v[layer][: self.held]) if self.k[layer] is not None else (k[0, :0], v[0, :0])
        self.k[layer], self.v[layer] = torch.cat([old[0], k[0]]), torch.cat([old[1], v[0]])

    def attend(self, layer, q, k, v):
        self.append(layer, k, v)
        ks, vs = (ref.stored(x[layer], self.kind, self.block) for x in (self.k, self.v))
        return ref.attend(q[0], ks, vs, self.held)[0].to(torch.bfloat16)[None]

    def advance(self, n):
        self.held += n
        self.length.fill_(self.held)


@pytest.mark.parametrize("cache", ["int8", "e4m3"])
def test_prompt_steps_and_second_turn_against_the_definition(cache, monkeypatch):
    """Logits agree as those of two summation orders do (the tolerance of the decoder's other test)."""
    from binade_b200.cuda import llama

    m = llama.Decoder(tiny(), kind="r4", cache=cache)
    p, follow, later = prompt_of(45), prompt_of(20, 2), prompt_of(37, 3)

    def run():
        got = [m.prefill(p)]
        for i in range(20):
            pos = torch.full((1,), 45 + i, dtype=torch.int64, device="cuda")
            got.append(m.step(follow[i : i + 1], pos))
        got.append(m.prefill(later, more=True))
        return torch.cat(got).float()

    a = run()
    assert m.cache.length.item() == 45 + 20 + 37
    assert torch.equal(run(), a)  # the first prompt empties the cache
    plain = PlainCache(2, cache, m.cache.block)
    monkeypatch.setattr(m, "cache", plain)
    monkeypatch.setattr(m, "reset", lambda: None)
    monkeypatch.setattr(llama, "attention", lambda q, k, v: ref.attend(q, k, v)[0].to(torch.bfloat16))
    with torch.no_grad():
        b = run()
    assert torch.allclose(a, b, atol=2e-2, rtol=2e-2)


def test_short_of_a_block_the_cache_is_exact():
    """Fewer tokens than a block are held in BF16: the same logits as the BF16 cache gives, to the order of sums; and
    graph and eager runs give the same tokens, before and behind a block's border."""
    from binade_b200.cuda.llama import Decoder

    a, b = Decoder(tiny(), kind="bf16", cache="int8"), Decoder(tiny(), kind="bf16")
    p = prompt_of(9)
    la = a.prefill(p).float()
    for i in range(9):
        lb = b.step(p[i : i + 1], torch.full((1,), i, dtype=torch.int64, device="cuda")).float()
    assert torch.allclose(la, lb, atol=2e-2, rtol=2e-2)
    eager, _ = a.generate(p, 70, use_graph=False)
    graphed, secs = a.generate(p, 70, use_graph=True)
    assert torch.equal(eager, graphed) and secs > 0
    with pytest.raises(ValueError):
        b.prefill(p)
    with pytest.raises(ValueError):
        a.prefill(prompt_of(161))


@pytest.mark.parametrize("cache", ["bf16", "int8"])
@pytest.mark.parametrize("use_graph", [False, True])
def test_rules_on_the_logits(cache, use_graph):
    from test_gpu_attention import bits_of

    from binade_b200.cuda.llama import Decoder

    m = Decoder(tiny(), kind="r4", cache=cache)
    p = prompt_of(12)
    free, _ = m.generate(p, 20, use_graph=use_graph)
    same, _ = m.generate(p, 20, use_graph=use_graph, rules={})
    assert torch.equal(free, same)
    allowed = torch.zeros(512, dtype=torch.bool, device="cuda")
    allowed[::7] = True
    masked, _ = m.generate(p, 30, use_graph=use_graph, rules=dict(mask=bits_of(allowed)))
    assert (masked % 7 == 0).all()
    fresh, _ = m.generate(p, 60, use_graph=use_graph, rules=dict(frequency=1e6, mask=bits_of(allowed)))
    assert len(set(fresh.tolist())) == 60  # every allowed token once before any twice
    none, _ = m.generate(p, 3, use_graph=use_graph, rules=dict(mask=bits_of(allowed & False)))
    assert none.tolist() == [-1, -1, -1]
    bias = torch.zeros(512, device="cuda")
    bias[77] = 1e6
    assert (m.generate(p, 4, use_graph=use_graph, rules=dict(bias=bias))[0] == 77).all()


def test_self_check_on_an_8_bit_cache():
    from binade_b200.cuda.llama import Decoder

    m = Decoder(tiny(), kind="r4", cache="int8")
    assert m.self_check()["linears_decoding_to_their_source"] == 9
    assert m.cache.length.item() == 0
