"""Checks of arguments that need no GPU: the helpers behind the attention and logits calls, on CPU tensors (whose device
number is -1)."""

import torch

from binade_b200.cuda import attention

CPU = -1


def test_rows_of_one_token_take_no_stride():
    """torch calls a tensor contiguous whatever the stride of a dimension of one element; the kernels read strides."""
    wide = torch.zeros((5, 260), dtype=torch.bfloat16)
    x = wide[:, :256].unflatten(1, (2, 128))
    for n in (1, 2, 5):
        t, steps = attention._rows(x[:n], "q", 3, CPU, apart=True)
        assert torch.equal(t, x[:n]) and all(s % 8 == 0 for s in steps)
    assert attention._rows(x[:1], "q", 3, CPU, apart=True)[0].data_ptr() == wide.data_ptr()  # and is read in place
