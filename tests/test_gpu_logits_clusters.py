"""The joins of the logits kernel: blocks of a cluster that have next to nothing to do before they hand on their choice."""

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("V", [1, 2048, 2049, 4097, 8193, 16385, 32769])
@pytest.mark.parametrize("batch", [1, 8, 9, 1000])
def test_every_block_of_a_cluster_is_heard(V, batch):
    """The largest logit in each block's piece in turn, the first blocks and the last short ones among them, beside other
    work on the card, again and again."""
    from binade_b200.cuda.logits import process_logits

    g = torch.Generator(device="cuda").manual_seed(V + batch)
    x = torch.randn((batch, V), generator=g, device="cuda", dtype=torch.float32)
    at = torch.randint(0, V, (batch,), generator=g, device="cuda")
    at[0], at[-1] = V - 1, min(V - 1, 2047)
    x.scatter_(1, at[:, None], 100.0)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    busy = torch.zeros((1 << 20,), device="cuda")
    for _ in range(50):
        with torch.cuda.stream(side):
            busy.add_(1)
        got, token = process_logits(x)
        assert torch.equal(token, at)
    assert torch.equal(got, x)
    torch.cuda.current_stream().wait_stream(side)
