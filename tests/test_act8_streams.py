"""conv2d(x8=) and the conv -> norm blocks in the backward pass, CPU side: which launches go to the side stream and which tensors are kept
for it.  The launches are recorded, not made."""
import types

import pytest
import torch

from hific_amd import act8, lib, ops


class _Slot:
    def __init__(self, like):
        self.grad, self.index = torch.zeros_like(like), 0

    def take(self):
        return 0

    def written(self):
        pass


@pytest.fixture
def launches(monkeypatch):
    """[(entry point, stream, pointers)], and what the side stream was told to keep."""
    log = types.SimpleNamespace(calls=[], kept=[], stream="main")

    class Side:
        def __init__(self, ev, *tensors, key=None):
            log.kept += [t for t in tensors if t is not None]

        def __enter__(self):
            log.stream = "side"

        def __exit__(self, *exc):
            log.stream = "main"

    def call(name, *args):
        log.calls.append((name, log.stream, args))
    monkeypatch.setattr(lib, "_cur_device", lambda: -1)
    monkeypatch.setattr(lib, "stream_obj", lambda *a: types.SimpleNamespace(record_event=lambda: None))
    monkeypatch.setattr(lib, "call", call)
    monkeypatch.setattr(act8, "stream", lambda: 0)
    monkeypatch.setattr(ops, "_ws", lambda t: (0, 0))
    monkeypatch.setattr(ops, "_SideLaunch", Side)
    monkeypatch.setattr(ops, "_SIDE_ON", True)
    monkeypatch.setattr(act8, "_conv_bwd_data", lambda dz, *a: call("data", dz.data_ptr()))
    monkeypatch.setattr(act8, "_conv_wgrad8", lambda saved, relu, dy, dw, *a: call("weight", *[lib.ptr(t) for t in saved], dw.data_ptr()))
    return log


def _ctx(weight, bias, w_slot, b_slot, q, e, gamma, beta):
    need = (True, False, False, False, False, False, True, True, False, False, False)
    return types.SimpleNamespace(saved_tensors=(q, e, gamma, beta, weight), needs_input_grad=need, has_bias=True, bias_grad=True, w_slot=w_slot,
                                 b_slot=b_slot, geom=(1, 1, 1, 1, 1, 0), xrelu=True, mode=lib.HIFIC_BF16, x_shape=q.shape, x_dtype=torch.bfloat16)


@pytest.mark.parametrize("w_in", [False, True])
@pytest.mark.parametrize("b_in", [False, True])
def test_gradients_handed_to_autograd_come_from_the_main_stream(launches, w_in, b_in):
    """A gradient that autograd accumulates (its parameter has no slot in an arena) is read on the main stream at once: only gradients
    that are written into an arena may be left to the side stream, which is joined at the end of the backward pass."""
    weight, bias = torch.zeros(6, 4, 3, 3), torch.zeros(6)
    q, e = torch.zeros(2, 4, 5, 5, dtype=torch.int8), torch.full((2, 5, 5), 127, dtype=torch.uint8)
    w_slot, b_slot = (_Slot(weight) if w_in else None), (_Slot(bias) if b_in else None)
    ctx = _ctx(weight, bias, w_slot, b_slot, q, e, None, None)
    with torch.no_grad():
        grads = act8.Conv8Fn.backward(ctx, torch.zeros(2, 6, 5, 5, dtype=torch.bfloat16))
    dw, db = grads[6], grads[7]
    assert (dw is None) == w_in and (db is None) == b_in
    by = {name: (stream, args) for name, stream, args in launches.calls}
    assert by["data"][0] == "main"
    if not w_in:
        assert by["weight"][0] == "main" and by["weight"][1][-1] == dw.data_ptr()
    if not b_in:
        assert by["hific_channel_sum"][0] == "main" and by["hific_channel_sum"][1][1] == db.data_ptr()
    if w_in and b_in:
        assert by["weight"][0] == by["hific_channel_sum"][0] == "side"


@pytest.mark.parametrize("arena", [False, True])
def test_the_side_stream_holds_everything_that_its_launches_read(launches, arena):
    """gamma and beta of an Act8 may be temporaries (a computed gamma) that the node alone holds: their memory must not go back to the
    allocator before the side stream has read them."""
    weight, bias = torch.zeros(6, 4, 3, 3), torch.zeros(6)
    q, e = torch.zeros(2, 4, 5, 5, dtype=torch.int8), torch.full((2, 5, 5), 127, dtype=torch.uint8)
    gamma, beta = torch.ones(4), torch.zeros(4)
    ctx = _ctx(weight, bias, _Slot(weight) if arena else None, _Slot(bias) if arena else None, q, e, gamma, beta)
    dy = torch.zeros(2, 6, 5, 5, dtype=torch.bfloat16)
    with torch.no_grad():
        act8.Conv8Fn.backward(ctx, dy)
    read = [args[:4] for name, stream, args in launches.calls if name == "weight" and stream == "side"]
    assert bool(read) == arena
    held = {t.data_ptr() for t in launches.kept}
    for ptrs in read:
        assert set(ptrs) <= held, "an operand of a side-stream launch is not recorded there"
    if arena:
        assert dy.data_ptr() in held
