"""What the Python side of the operators on device arrays decides before it calls the library (no GPU)."""
import numpy as np
import pytest
import torch

from adhip import operators as ops


class Elsewhere:
    """As a tensor that has device memory, for the arrays beside the one in question."""
    is_cuda = True

    def __init__(self, *shape, dtype="float32"):
        self.shape, self.dtype = shape, dtype

    def stride(self):
        return tuple(1 for _ in self.shape)

    def data_ptr(self):
        return 256

    def numel(self):
        return 1

    def is_contiguous(self):
        return True


def test_host_tensors_are_refused():
    """A kernel that is handed an address of host memory faults: no such array gets as far as the library (there is none here)."""
    host, here = torch.zeros((1, 1, 1, 64)), Elsewhere(1, 1, 1, 64)
    lse, room = Elsewhere(1, 1, 1), Elsewhere(1 << 20, dtype="int32")
    table, at = Elsewhere(4, 32), Elsewhere(1, 1, dtype="int32")
    room.nbytes = 1 << 20

    def refused(call, *args, **how):
        with pytest.raises(ValueError, match="in device memory"):
            call(None, *args, **how)

    for i in range(5):
        args = [here, here, here, here, lse]
        args[i] = torch.zeros((1, 1, 1)) if i == 4 else host
        refused(ops.attention, *args, workspace=room)
    refused(ops.attention, here, here, here, here, lse, workspace=torch.zeros(1 << 20))
    for name in ("slopes", "lengths", "prefix", "query_documents", "key_documents"):
        refused(ops.attention, here, here, here, here, lse, workspace=room, **{name: torch.zeros(1)})
    for i in range(4):
        args = [here, here, here, here]
        args[i] = host
        refused(ops.attention_backward, here, here, here, here, lse, *args, workspace=room)
    for i, bad in enumerate((host, host, torch.zeros((4, 32)), torch.zeros((4, 32)), torch.zeros((1, 1), dtype=torch.int32))):
        args = [here, here, table, table, at]
        args[i] = bad
        refused(ops.rotary, *args)
    refused(ops.rotary, here, here, table, table, at, second=host, second_out=here)
    one, states = torch.zeros(1), [Elsewhere(1, 256, dtype="float8_e4m3fn")]
    how = dict(step=1, rate=0.1)
    for i in range(4):
        args = [[Elsewhere(1)] for _ in range(4)]
        args[i] = [one]
        refused(ops.adamw, *args, **how)
    for name in ("parameters_out", "first_out", "second_out"):
        refused(ops.adamw, *[[Elsewhere(1)] for _ in range(4)], **how, **{name: [one]})
    states[0].numel = lambda: 256
    for bad in range(4):
        scales = [[one] if i == bad else [Elsewhere(1)] for i in range(4)]
        refused(ops.adamw, [Elsewhere(1)], [Elsewhere(1)], states, states, first_scales=scales[0], second_scales=scales[1],
                first_scales_out=scales[2], second_scales_out=scales[3], **how)


def test_whole_numbers_keep_their_value():
    """Numbers of documents are often hashes of 64 bits: cut off to 32 they would meet others, or belong to none."""
    for values in ([2 ** 31], [-2 ** 31 - 1], [0, 2 ** 40]):
        with pytest.raises(ValueError, match="32 bits"):
            ops.DeviceArray.of(None, np.array(values))
    ends = [-2 ** 31, 0, 2 ** 31 - 1]
    kept = ops._host_values(np.array([ends, ends]).T, "int32")
    assert kept.dtype == np.int32 and kept.flags.c_contiguous and kept.tolist() == np.array([ends, ends]).T.tolist()
    assert ops._host_values(np.array([True, False]), "int32").tolist() == [1, 0]
    assert ops._host_values(7, "int32").tolist() == [7]
    for values in ([0.5], [2 ** 40]):
        with pytest.raises(ValueError, match="32 bits"):
            ops._host_values(values, "int32")
