"""GPU test of host lengths in pinned memory through the discriminator's entry points."""
import pytest

pytestmark = pytest.mark.gpu


def test_pinned_src_len_may_be_refilled_after_the_call():
    """The copy to the device waits behind earlier work on the stream; the caller's buffer is free as soon as the call is back."""
    import torch
    from sad_amd import functional as Fn
    dev = torch.device("cuda", torch.cuda.current_device())
    lengths = torch.tensor([40, 7, 3], dtype=torch.int32).pin_memory()
    a = torch.randn(4096, 4096, device="cuda")
    torch.cuda.synchronize()
    for _ in range(40):
        a = (a @ a) * 1e-3                       # some milliseconds of work in front
    sent = Fn._lengths_to_device(lengths, 3, dev)
    lengths.fill_(1)
    torch.cuda.synchronize()
    assert sent.tolist() == [40, 7, 3]
