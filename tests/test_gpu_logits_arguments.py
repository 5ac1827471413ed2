"""What process_logits refuses beside its sizes."""

import pytest
import torch
from torch.autograd import forward_ad

pytestmark = pytest.mark.gpu


def test_what_asks_for_a_gradient_is_refused():
    from binade_b200.cuda.attention import attention
    from binade_b200.cuda.logits import TokenCounts, process_logits

    said = TokenCounts(2, 100)
    x = torch.zeros((2, 100), device="cuda")
    asks, rows = torch.ones(100, device="cuda", requires_grad=True), torch.ones(2, device="cuda", requires_grad=True)
    q = torch.zeros((8, 4, 64), dtype=torch.bfloat16, device="cuda")
    calls = (
        lambda: process_logits(x, bias=asks),
        lambda: process_logits(x, said, repetition=rows),
        lambda: process_logits(x, said, frequency=rows),
        lambda: attention(q, q, q, slopes=torch.ones(4, device="cuda", requires_grad=True)),
    )
    for call in calls:
        with pytest.raises(ValueError, match="gradient"):
            call()
        with torch.no_grad():
            call()
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(x, x)
        for call in (
            lambda: process_logits(dual),
            lambda: process_logits(x, bias=forward_ad.make_dual(asks.detach(), asks.detach())),
            lambda: process_logits(x, said, presence=forward_ad.make_dual(rows.detach(), rows.detach())),
            lambda: process_logits(x, out=forward_ad.make_dual(torch.empty_like(x), x)),
            lambda: attention(forward_ad.make_dual(q, q), q, q),
            lambda: attention(q, q, q, out=forward_ad.make_dual(torch.empty_like(q), q)),
        ):
            with pytest.raises(ValueError, match="gradient"):
                call()
        process_logits(x), attention(q, q, q)


def test_out_among_the_rules_is_refused():
    """A block writes its piece of a row while another still reads the bias, the mask or the penalties there."""
    from binade_b200.cuda.logits import TokenCounts, process_logits

    said = TokenCounts(2, 96)
    x, out = torch.randn((2, 96), device="cuda"), torch.zeros((2, 96), device="cuda")
    for call in (
        lambda: process_logits(x, bias=out, out=out),
        lambda: process_logits(x, bias=out[1], out=out),
        lambda: process_logits(x, said, presence=out[0, :2], out=out),
        lambda: process_logits(x, mask=out.view(-1).view(torch.int32)[:3], out=out),
        lambda: process_logits(x, said, presence=1.0, out=said.counts.view(torch.float32)),
    ):
        with pytest.raises(ValueError, match="out may not"):
            call()
    one = torch.randn((2, 96), device="cuda")
    got, _ = process_logits(one, said, presence=1.0, bias=out[0], out=one)  # the logits themselves, beside the others
    assert got is one


def test_lengths_beyond_32_bits_do_not_wrap():
    from binade_b200.cuda.logits import TokenCounts

    said = TokenCounts(2, 10)
    said.add(torch.tensor([[1, 2, 3], [4, 5, 6]], device="cuda"), lengths=torch.tensor([1 << 32, -(1 << 32) + 2], device="cuda"))
    assert said.counts.sum(1).tolist() == [3, 0]
