"""CPU checks of how the discriminator's entry points send host lengths to the device."""
import pytest
import torch

from sad_amd import functional as Fn


@pytest.mark.parametrize("dtype", [torch.int16, torch.int32, torch.int64])
def test_host_lengths_are_copied_before_the_call_returns(dtype):
    """What goes to the device is no alias of the caller's buffer (with the host in the device's place it would show)."""
    buf = torch.tensor([3, 2, 2], dtype=dtype)
    sent = Fn._lengths_to_device(buf, 3, torch.device("cpu"))
    buf.fill_(1)
    assert sent.tolist() == [3, 2, 2] and sent.dtype == torch.int32
