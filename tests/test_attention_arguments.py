"""Checks of arguments that need no GPU: the helpers behind the attention and logits calls, on CPU tensors (whose device
number is -1)."""

import pytest
import torch
from torch.autograd import forward_ad

from binade_b200.cuda import attention, logits

CPU = -1


def test_rows_of_one_token_take_no_stride():
    """torch calls a tensor contiguous whatever the stride of a dimension of one element; the kernels read strides."""
    wide = torch.zeros((5, 260), dtype=torch.bfloat16)
    x = wide[:, :256].unflatten(1, (2, 128))
    for n in (1, 2, 5):
        t, steps = attention._rows(x[:n], "q", 3, CPU, apart=True)
        assert torch.equal(t, x[:n]) and all(s % 8 == 0 for s in steps)
    assert attention._rows(x[:1], "q", 3, CPU, apart=True)[0].data_ptr() == wide.data_ptr()  # and is read in place


def test_options_of_a_call_survive_another_thread(monkeypatch):
    """Between a look and a read another thread may empty the table."""

    class Emptied(dict):
        def __contains__(self, key):
            there = super().__contains__(key)
            self.clear()
            return there

    monkeypatch.setattr(attention, "_score_structs", Emptied())
    for _ in range(3):
        made, _ = attention._scores(128, 4, CPU, None, 20.0, 7, None, True)
        assert (made.softcap, made.window, made.causal) == (20.0, 7, 1)


def test_what_asks_for_a_gradient_is_refused():
    asks = torch.ones(4, requires_grad=True)
    for bad in (
        lambda: attention._scores(128, 4, CPU, None, None, None, asks, True),
        lambda: logits._penalty(asks, "presence", 4, asks.device),
        lambda: logits._penalty(asks.double(), "presence", 4, asks.device),
    ):
        with pytest.raises(ValueError, match="gradient"):
            bad()
        with torch.no_grad():
            bad()


def test_what_carries_a_tangent_is_refused():
    x = torch.ones((4, 2, 64), dtype=torch.bfloat16)
    with forward_ad.dual_level():
        dual, p = forward_ad.make_dual(x, x), forward_ad.make_dual(torch.ones(4), torch.ones(4))
        for bad in (
            lambda: attention._rows(dual, "q", 3, CPU),
            lambda: attention._scores(128, 4, CPU, None, None, None, p, True),
            lambda: logits._penalty(p, "presence", 4, p.device),
        ):
            with pytest.raises(ValueError, match="gradient"):
                bad()
        attention._rows(x, "q", 3, CPU)
    attention._rows(x, "q", 3, CPU)


def test_whole_numbers_beyond_32_bits_do_not_wrap():
    got = attention._numbers(torch.tensor([1 << 40, -(1 << 40), (1 << 31) - 1, 5]), "prefix", 4, CPU)
    assert got.dtype is torch.int32 and got.tolist() == [(1 << 31) - 1, -(1 << 31), (1 << 31) - 1, 5]


@pytest.mark.parametrize("bad", [dict(softcap=1e-50), dict(softcap=1e39), dict(softcap=2.0**61), dict(softcap=2.0**-61), dict(scale=1e39)])
def test_caps_and_scales_that_fp32_does_not_hold_are_refused(bad):
    with pytest.raises(ValueError):
        attention._scores(128, 4, CPU, bad.get("scale"), bad.get("softcap"), None, None, True)


@pytest.mark.parametrize("bad", [dict(softcap=1e-30), dict(softcap=float("inf")), dict(softcap=2.0**61), dict(scale=float("inf")), dict(scale=float("nan"))])
def test_the_c_calls_refuse_them_too(bad):
    from test_attention_host import attend, attention, scores

    from binade_b200._native import NativeError

    for call in (attention, attend):
        with pytest.raises(NativeError, match="bad argument"):
            call(s=scores(**bad))


def test_advance_needs_to_know_which_blocks_are_held():
    import ctypes

    from test_attention_host import cache

    from binade_b200 import _native

    with pytest.raises(_native.NativeError, match="bad argument: bn_kv8_advance"):
        _native.call("cuda", "bn_kv8_advance", ctypes.byref(cache(kept=None)), 1, None, None)


def test_options_are_taken_by_value():
    """A number in a tensor may change between two calls; nothing is kept by an object's identity."""
    scale, cap, window, causal = torch.tensor(0.5), torch.tensor(20.0), torch.tensor(7), torch.tensor(True)
    for factor in (1, 2, 3):
        made, _ = attention._scores(128, 4, CPU, scale, cap, window, None, causal)
        assert (made.scale, made.softcap, made.window, made.causal) == (0.5 * factor, 20.0 * factor, 7, factor % 2)
        scale.add_(0.5), cap.add_(20.0), causal.logical_not_()


def test_out_among_the_inputs_is_refused():
    x = torch.zeros((2, 4, 64), dtype=torch.bfloat16)
    for t in (x, x.view(torch.int32)[0, 0], x.view(torch.float32)[1, 3, :2]):
        with pytest.raises(ValueError, match="among the inputs"):
            attention._out(x, torch.empty_like(x), CPU, None, t)
    assert attention._out(x, torch.empty_like(x), CPU, torch.zeros(4)) is x
