"""What the attention calls refuse beside their sizes."""

import pytest
import torch

pytestmark = pytest.mark.gpu


def test_out_among_the_numbers_of_a_call_is_refused():
    """Blocks write rows while others still read the offsets, prefixes, counts and slopes there."""
    from binade_b200.cuda.attention import KV8Cache, attention

    q = torch.randn((8, 4, 64), device="cuda").to(torch.bfloat16)
    out = torch.zeros_like(q)
    words, floats = out.view(torch.int32).reshape(-1), out.view(torch.float32).reshape(-1)
    words[1], words[2] = 8, 8
    cache = KV8Cache(1, 1, 4, 64, 64)
    for call in (
        lambda: attention(q, q, q, words[:2], out=out),
        lambda: attention(q, q, q, prefix=words[3:4], out=out),
        lambda: attention(q, q, q, slopes=floats[8:12], out=out),
        lambda: cache.attend(0, q[None], q[None], q[None], words[1:2], out=out[None]),
        lambda: cache.attend(0, q[None], q[None], q[None], prefix=words[1:2], out=out[None]),
        lambda: cache.attend(0, q[None], q[None], q[None], slopes=floats[8:12], out=out[None]),
    ):
        with pytest.raises(ValueError, match="among the inputs"):
            call()
