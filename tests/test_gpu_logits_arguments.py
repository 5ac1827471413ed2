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
