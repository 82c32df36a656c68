"""Python descriptors of the 8-bit linear layer (no GPU): what the calls are told about a tensor stays inside its buffer."""
import os

import numpy as np
import pytest

from intel_gaudi3_software_amd import HipCalculator, MMEStackException, MmeSimTensor, abi


def told(t):
    """The strides that the 8-bit linear layer's entry points are given."""
    return list(t._ref._obj.strides)


def last(t, strides):
    return sum(st * (sz - 1) for st, sz in zip(strides, t.sizes))


def test_a_stride_of_zero_repeats_the_row():
    row = np.zeros(64, np.float32)
    t = MmeSimTensor([64, 9], 2, abi.FP32, row, strides=[1, 0])
    assert told(t)[:2] == [1, 0] and last(t, told(t)) == 63 and t._ref._obj.data == row.ctypes.data
    planes = np.zeros(64 * 3, np.float32)
    t = MmeSimTensor([64, 3, 5], 3, abi.FP32, planes, strides=[1, 64, 0])
    assert told(t)[:3] == [1, 64, 0] and last(t, told(t)) == 191
    t = MmeSimTensor([64, 5, 3], 3, abi.FP32, planes, strides=[1, 0, 64])
    assert told(t)[:3] == [1, 0, 64]
    # the other entry points take such strides for dense ones: not in a buffer that has no room for that
    t = MmeSimTensor([64, 9], 2, abi.FP32, row, strides=[1, 0])
    calc = HipCalculator.__new__(HipCalculator)
    with pytest.raises(MMEStackException) as e:
        calc._placement(t)
    assert e.value.status == abi.EINVAL
    t = MmeSimTensor([64, 9], 2, abi.FP32, np.zeros(64 * 9, np.float32), strides=[1, 0])
    assert calc._placement(t) is False and list(t.desc.strides)[:2] == [1, 64] and told(t)[:2] == [1, 0]
    # (a dimension of one index or none has no stride to speak of)
    t = MmeSimTensor([64, 9, 1], 3, abi.FP32, np.zeros(64 * 9, np.float32), strides=[1, 64, 0, 0, 0])
    assert told(t) == list(t.desc.strides) == [1, 64, 576, 576, 576]
    t = MmeSimTensor([64, 0], 2, abi.FP32)
    assert told(t) == list(t.desc.strides)


def test_overlapping_rows_stay_inside_the_buffer():
    """Input rows may share memory: the buffer has to hold the last element of the last row, which no single dimension shows."""
    for sizes, strides in (([64, 9, 9], [1, 8, 8]), ([16, 4, 4], [1, 16, 24]), ([8, 3, 1, 5], [1, 5, 15, 7])):
        need = 1 + sum(st * (sz - 1) for st, sz in zip(strides, sizes))
        assert need > max(st * sz for st, sz in zip(strides, sizes))
        t = MmeSimTensor(sizes, len(sizes), abi.FP32, np.zeros(need, np.float32), strides=strides)
        assert last(t, told(t)) == need - 1
        with pytest.raises(ValueError):
            MmeSimTensor(sizes, len(sizes), abi.FP32, np.zeros(need - 1, np.float32), strides=strides)
        assert MmeSimTensor(sizes, len(sizes), abi.FP32, strides=strides).data().size >= need


def test_own_stream_waits_for_the_stream_of_its_own_device(monkeypatch):
    """The operands are written on the current stream of their device, which need not be the current device's."""
    torch = pytest.importorskip("torch")
    seen = []

    class Event:
        def record(self, stream=None):
            seen.append(("record", stream))

    class External:
        def __init__(self, pointer, device=None):
            seen.append(("stream", pointer, device))

        def wait_event(self, event):
            seen.append(("wait", type(event)))

    monkeypatch.setattr(torch.cuda, "Event", Event)
    monkeypatch.setattr(torch.cuda, "ExternalStream", External)
    monkeypatch.setattr(torch.cuda, "current_stream", lambda device=None: "stream of device %s" % device)
    calc = HipCalculator.__new__(HipCalculator)
    calc._caller_stream, calc._in_flight, calc._gpu = False, [], 3
    monkeypatch.setattr(HipCalculator, "stream", lambda self: 77)
    calc._after_torch()
    assert seen == [("record", "stream of device 3"), ("stream", 77, 3), ("wait", Event)]


def test_windows_of_windows():
    """A window's address and strides, windows inside it, and those that leave the buffer."""
    t = MmeSimTensor([20, 3], 2, abi.FP32)
    w = t.window(10, [10, 3])
    assert w.desc.data == t.desc.data + 40 and list(w.desc.strides)[:2] == [1, 20] and w.getSizes()[:2] == [10, 3]
    assert w.window(3, [7, 3]).desc.data == t.desc.data + 52
    assert list(t.window(0, [20, 9], [1, 0, 0, 0, 0]).desc.strides) == [1, 0, 0, 0, 0]
    for bad in ((11, [10, 3]), (0, [20, 4]), (-1, [10, 3])):
        with pytest.raises(ValueError):
            t.window(*bad)
    with pytest.raises(ValueError):
        w.window(3, [8, 3])


def test_one_pitch_over_a_dimension_of_one_index():
    """The stride of a dimension of one index says nothing: rows behind it have to follow from the dimension before."""
    if not os.path.exists(abi.LIB_PATH):
        pytest.skip("libmme_hip.so has not been built (python -m intel_gaudi3_software_amd.build)")
    MIB = 1 << 20

    def one_pitch(sizes, strides, out_strides=None):
        o, x = (abi.make_tensor(at * MIB, sizes, t, 0, 0, None, dim=5) for at, t in ((2048, abi.INT8), (1, abi.BF16)))
        for t, st in ((x, strides), (o, out_strides or o.strides)):
            for d in range(5):
                t.strides[d] = st[d]
        return abi.plan_quantize_rows(o, 4096 * MIB, x)["one_pitch"]

    assert one_pitch([64, 3, 1, 4, 1], [1, 100, 300, 300, 1200]) == 1
    assert one_pitch([64, 3, 1, 4, 1], [1, 100, 700, 700, 2800]) == 0   # (planes 700 apart, three rows of pitch 100 in each)
    assert one_pitch([64, 3, 1, 1, 4], [1, 100, 5, 700, 700]) == 0
    assert one_pitch([64, 3, 1, 4, 1], [1, 64, 192, 192, 768], [1, 64, 1000, 1000, 4000]) == 0
    assert one_pitch([64, 1, 1, 5, 1], [1, 100, 100, 100, 500]) == 1
    assert one_pitch([64, 3, 4, 1, 1], [1, 0, 0, 0, 0]) == 1            # (one row for all)
    assert one_pitch([64, 3, 1, 4, 1], [1, 0, 100, 100, 400]) == 0      # (one row for the three of a plane)
