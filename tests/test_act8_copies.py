"""Copies of an Act8 (deepcopy, pickle, torch.save): its tensors, and nothing of the optimizer arena that its norm's parameters live in."""
import copy
import io
import pickle

import pytest
import torch

from hific_amd import act8, lib


class _Arena:
    epoch = 0

    def __reduce__(self):
        raise AssertionError("the arena was copied")


class _Slot:
    def __init__(self, arena):
        self.arena = arena


def _kept(arena):
    gamma, beta = torch.nn.Parameter(torch.rand(1, 3, 1, 1)), torch.nn.Parameter(torch.rand(1, 3, 1, 1))
    if arena is not None:
        gamma._hific_slot = beta._hific_slot = _Slot(arena)
    q, e = torch.randint(-127, 128, (2, 3, 4, 4), dtype=torch.int8), torch.full((2, 4, 4), 121, dtype=torch.uint8)
    return act8.Act8._of(q, e, gamma, beta, True), gamma


def _saved(a):
    f = io.BytesIO()
    torch.save(a, f)
    f.seek(0)
    return torch.load(f, weights_only=False)             # (written two lines above)


@pytest.mark.parametrize("how", [copy.deepcopy, lambda a: pickle.loads(pickle.dumps(a)), _saved])
@pytest.mark.parametrize("in_arena", [False, True])
def test_a_copy_holds_its_own_parameters(how, in_arena):
    a, gamma = _kept(_Arena() if in_arena else None)
    b = how(a)
    assert torch.equal(a.q, b.q) and torch.equal(a.e, b.e) and torch.equal(a.gamma, b.gamma) and torch.equal(a.beta, b.beta) and b.relu
    before = b.gamma.clone()
    with torch.no_grad():
        gamma.add_(1.0)
    assert torch.equal(b.gamma, before)
    b._current()                                         # still what it was a copy of
    with pytest.raises(lib.HificError, match="changed"):
        a._current()
    with pytest.raises(lib.HificError, match="changed"):
        how(a)


def test_a_shallow_copy_shares_the_tensors():
    a, _ = _kept(None)
    b = copy.copy(a)
    assert b.q.data_ptr() == a.q.data_ptr() and b.gamma.data_ptr() == a.gamma.data_ptr()
