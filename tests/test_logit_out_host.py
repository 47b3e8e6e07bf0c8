"""Where adjust_logits may write (checked before anything runs): the next check, of the
device, is what an allowed call on the CPU meets."""
import pytest
import torch

from specfit_amd import ops


def _meets(logits, out, **more):
    with pytest.raises(ValueError) as refused:
        ops.adjust_logits(logits, out=out, **more)
    message = str(refused.value)
    assert ("share no memory" in message) != ("device" in message), message
    return "share no memory" in message


def test_columns_of_one_buffer():
    buffer = torch.zeros((4, 30))
    logits = buffer[:, 5:15]
    assert not _meets(logits, buffer[:, 15:25])
    assert not _meets(buffer[:, 15:25], logits)
    assert not _meets(logits, logits)
    assert _meets(logits, buffer[:, 14:24]) and _meets(logits, buffer[:, 4:14])
    assert not _meets(buffer[:2, 5:15], buffer[2:, 3:13])      # one behind the other
    assert not _meets(buffer[:3, 20:30], buffer[1:, 0:10])     # side by side around the rows' end
    assert _meets(buffer[:2, 21:30], buffer.view(-1)[50:110].view(2, 30)[:, :9])
    bias = buffer[:, 15:25]
    assert not _meets(torch.zeros((4, 10)), buffer[:, 5:15], bias=bias)
    assert _meets(torch.zeros((4, 10)), buffer[:, 6:16], bias=bias)
    assert _meets(torch.zeros((4, 10)), buffer[:, 5:15], bias=buffer.view(-1)[60:70])


def test_other_strides_are_refused_where_they_meet():
    buffer = torch.zeros(400)
    out = buffer.as_strided((4, 10), (30, 1), 0)
    assert _meets(buffer.as_strided((4, 10), (29, 1), 12), out)
    assert not _meets(buffer.as_strided((4, 10), (29, 1), 100), out)
