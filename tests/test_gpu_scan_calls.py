"""GPU tests of calls to the gated scan and the 8-bit checkpoints beside the plain ones: what a program may do with their
arguments and results between and after the calls."""
import pytest

pytestmark = pytest.mark.gpu


def _t():
    import torch
    from sad_amd import functional as Fn
    return torch, Fn


def test_checkpoint_moved_to_the_host_and_back():
    torch, Fn = _t()
    x = torch.randn(37, 70, device="cuda")
    dy = torch.randn(37, 9, device="cuda")
    ck = Fn.checkpoint8(x)
    want, dw = ck.restore(), Fn.weight_grad8(dy, ck)
    ck.saved = ck.saved.cpu()
    with pytest.raises(RuntimeError, match="must be on the HIP device"):
        ck.restore()
    with pytest.raises(RuntimeError, match="checkpoint on cpu"):
        Fn.weight_grad8(dy, ck)
    ck.saved = ck.saved.cuda()
    assert torch.equal(ck.restore(), want) and torch.equal(Fn.weight_grad8(dy, ck), dw)
    for part in (ck.saved[:-1], ck.saved[1:], torch.cat([ck.saved, ck.saved])):
        with pytest.raises(RuntimeError, match="holds"):
            Fn.Checkpoint8(part, ck.shape, ck.dtype).restore()
        with pytest.raises(RuntimeError, match="holds"):
            Fn.weight_grad8(dy, Fn.Checkpoint8(part, ck.shape, ck.dtype))
    shifted = torch.cat([ck.saved[:1], ck.saved])[1:]
    with pytest.raises(RuntimeError, match="16-byte aligned"):
        Fn.Checkpoint8(shifted, ck.shape, ck.dtype).restore()
