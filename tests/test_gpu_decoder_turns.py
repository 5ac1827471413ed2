"""The decoder on a cache in 8 bits at the end of its room: generation after generation, and a further turn."""

import pytest
import torch

from test_gpu_attention_extremes import status
from test_gpu_decoder_cache import prompt_of, tiny

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rules", [None, dict(repetition=1.2)])
def test_generations_that_fill_the_cache_leave_no_status(rules):
    from binade_b200 import _native
    from binade_b200.cuda.llama import Decoder

    _native.call("cuda", "bn_device_status_reset")
    m = Decoder(tiny(64), kind="bf16", cache="int8")
    p = prompt_of(20)
    first, _ = m.generate(p, 44, use_graph=True, rules=rules)
    assert m.cache.length.item() == 64
    again, _ = m.generate(p, 44, use_graph=True, rules=rules)
    assert torch.equal(first, again) and status() == 0


def test_a_further_turn_that_does_not_fit_is_refused():
    from binade_b200 import _native
    from binade_b200.cuda.llama import Decoder

    _native.call("cuda", "bn_device_status_reset")
    m = Decoder(tiny(64), kind="bf16", cache="e4m3")
    m.prefill(prompt_of(40))
    with pytest.raises(ValueError, match="behind 40"):
        m.prefill(prompt_of(25), more=True)
    assert m.cache.length.item() == 40 and status() == 0
    m.prefill(prompt_of(24), more=True)
    assert m.cache.length.item() == 64 and status() == 0
    with pytest.raises(ValueError, match="behind 64"):
        m.prefill(prompt_of(1), more=True)
    graph, p = torch.cuda.CUDAGraph(), prompt_of(9)
    m.prefill(prompt_of(20))
    want = m.prefill(p, more=True)
    m.cache.advance(-9)
    with torch.cuda.graph(graph):  # a capture of it still goes
        got = m.prefill(p, more=True)
    graph.replay()
    assert torch.equal(got, want) and m.cache.length.item() == 29
