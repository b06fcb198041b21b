"""How the language-model operators allocate their results (lm._new): torch's
shortest way, its public one where that is missing or where someone has to see
the allocation."""
import pytest
import torch
from torch.utils._python_dispatch import TorchDispatchMode

from bafe_b200 import lm

SHAPES = [((7,), torch.float32), ((0,), torch.int32), ((3, 5), torch.int32), ((0, 4), torch.float32), ((2, 8), torch.bfloat16)]


class Seen(TorchDispatchMode):
    def __init__(self):
        super().__init__()
        self.names = []

    def __torch_dispatch__(self, func, types, args=(), kwargs=None):
        self.names.append(func.__name__)
        return func(*args, **(kwargs or {}))


def same(t, shape, dtype):
    return tuple(t.shape) == shape and t.dtype == dtype and t.is_contiguous() and t.is_cuda


def test_the_public_way_is_taken_where_it_has_to_be(monkeypatch):
    """No GPU: which of the two is called."""
    calls = []
    monkeypatch.setattr(torch, "empty", lambda shape, dtype, device: calls.append(("public", shape, dtype, device)))
    monkeypatch.setattr(lm, "_strided", lambda shape, stride, dtype: calls.append(("short", shape, stride, dtype)))
    lm._new((2, 3), torch.float32)
    assert calls.pop() == ("short", (2, 3), (3, 1), torch.float32)
    with Seen():
        lm._new((2, 3), torch.float32)
    assert calls.pop() == ("public", (2, 3), torch.float32, "cuda")
    torch.use_deterministic_algorithms(True)
    try:
        lm._new((4,), torch.int32)
        assert calls.pop()[0] == "public"
    finally:
        torch.use_deterministic_algorithms(False)
    monkeypatch.setattr(lm, "_strided", None)
    lm._new((4,), torch.int32)
    assert calls.pop() == ("public", (4,), torch.int32, "cuda")
    assert not calls


@pytest.mark.gpu
@pytest.mark.parametrize("shape,dtype", SHAPES)
def test_both_ways_give_the_same(cuda, monkeypatch, shape, dtype):
    assert same(lm._new(shape, dtype), shape, dtype)
    monkeypatch.setattr(lm, "_strided", None)
    assert same(lm._new(shape, dtype), shape, dtype)


@pytest.mark.gpu
def test_modes_see_the_results_of_a_call(cuda):
    x = torch.randn(6, 64, device="cuda").bfloat16()
    place = torch.arange(6, dtype=torch.int32, device="cuda")[:, None]
    with Seen() as seen:
        lm.dispatch(x, place)
    assert any("empty" in n for n in seen.names)


@pytest.mark.gpu
def test_deterministic_fill_reaches_what_a_call_leaves_unset(cuda):
    """Rows that no place names are unset: torch fills them with NaN where it is asked to."""
    x = torch.ones(6, 64, device="cuda")
    place = torch.full((6, 2), -1, dtype=torch.int32, device="cuda")
    place[:, 0] = torch.arange(6)
    torch.use_deterministic_algorithms(True)
    try:
        y = lm.dispatch(x, place)
    finally:
        torch.use_deterministic_algorithms(False)
    assert (y[:6] == 1).all() and y[6:].isnan().all()
