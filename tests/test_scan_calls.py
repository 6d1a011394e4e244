"""CPU checks of what the gated scan's and the 8-bit checkpoints' entry points do with calls a user can make beside the plain
ones.  Refused calls raise before anything is launched, through functional and through torch.ops.sad_amd alike."""
import pytest
import torch

from sad_amd import functional as Fn
from sad_amd import lib

F32 = torch.float32


def _codes(n, **kw):
    return torch.zeros(n, dtype=torch.uint8, **kw)


@pytest.mark.parametrize("saved,shape,message", [
    (_codes(7 * 68), (7, 33), "must be on the HIP device"),                    # moved to the host
    (_codes(64), (1000, 33), "holds 68000 bytes, got 64"),                     # a slice of the codes
    (_codes(7 * 68 + 1), (7, 33), "holds 476 bytes"),
    (_codes(0), (7, 33), "holds 476 bytes"),
    (_codes(5), (0, 33), "holds 0 bytes"),
    (torch.zeros(7 * 68), (7, 33), "contiguous uint8"),
    (_codes(2 * 7 * 68)[::2], (7, 33), "contiguous uint8"),
    (_codes(34), (), "channel axis"),
])
def test_restore_takes_whole_checkpoints_on_the_device_only(saved, shape, message):
    with pytest.raises(RuntimeError, match=message):
        Fn.Checkpoint8(saved, shape, F32).restore()


@pytest.mark.parametrize("saved,message", [
    (_codes(4 * 34), "must be on the HIP device"),
    (_codes(4 * 34 - 1), "holds 136 bytes, got 135"),
    (_codes(4 * 34).view(torch.int8), "contiguous uint8"),
    (_codes(2 * 4 * 34)[::2], "contiguous uint8"),
])
def test_weight_gradient_takes_whole_checkpoints_on_the_device_only(saved, message):
    with pytest.raises(RuntimeError, match=message):
        lib.load_ops().weight_grad8(torch.zeros(4, 5), saved, 6, True)
    with pytest.raises(RuntimeError):
        Fn.weight_grad8(torch.zeros(4, 5), Fn.Checkpoint8(saved, (4, 6), F32), bias=True)


@pytest.mark.parametrize("which", ["z", "h0"])
def test_scan_refuses_dual_tensors(which):
    import torch.autograd.forward_ad as fa
    ops, args = lib.load_ops(), dict(z=torch.zeros(2, 3, 12), h0=torch.zeros(2, 4))
    with fa.dual_level():
        args[which] = fa.make_dual(args[which], torch.ones_like(args[which]))
        for grad in (False, True):
            with torch.set_grad_enabled(grad), pytest.raises(RuntimeError, match="gated_scan has no forward-mode derivative"):
                ops.gated_scan(args["z"], args["h0"], None, False, True, False)


@pytest.mark.parametrize("which", ["z", "h", "h_out"])
def test_step_refuses_dual_tensors(which):
    import torch.autograd.forward_ad as fa
    args = dict(z=torch.zeros(2, 12), h=torch.zeros(2, 4), h_out=torch.zeros(2, 4))
    with fa.dual_level(), torch.no_grad():
        args[which] = fa.make_dual(args[which], torch.ones_like(args[which]))
        with pytest.raises(RuntimeError, match="gated_scan_step has no forward-mode derivative"):
            lib.load_ops().gated_scan_step(args["z"], args["h"], None, True, args["h_out"])


def test_step_refuses_to_write_into_a_tensor_that_needs_a_gradient():
    h_out = torch.zeros(2, 4, requires_grad=True)
    with pytest.raises(RuntimeError, match="no gradient"):
        Fn.gated_scan_step(torch.zeros(2, 12), torch.zeros(2, 4), h_out=h_out)
    with torch.no_grad(), pytest.raises(RuntimeError, match="no CPU path"):      # past that check
        Fn.gated_scan_step(torch.zeros(2, 12), torch.zeros(2, 4), h_out=h_out)


@pytest.mark.parametrize("dtype", [torch.int16, torch.int32, torch.int64])
def test_host_lengths_are_copied_before_the_call_returns(dtype):
    """What goes to the device is no alias of the caller's buffer (with the host in the device's place it would show)."""
    buf = torch.tensor([3, 0, 2], dtype=dtype)
    sent = Fn._scan_lengths(buf, 3, 3, torch.device("cpu"))
    buf.zero_()
    assert sent.tolist() == [3, 0, 2] and sent.dtype == torch.int32


@pytest.mark.parametrize("dtype", [torch.complex32, torch.complex64, torch.complex128, torch.float64, torch.bool])
def test_lengths_are_integers(dtype):
    with pytest.raises(RuntimeError, match="must be 2 integers"):
        Fn.gated_scan(torch.zeros(2, 3, 12), lengths=torch.ones(2).to(dtype))


def _direct(device="cpu"):
    """Calls of the operators themselves, past functional's checks."""
    ops = lib.load_ops()
    f = lambda *shape, dtype=F32: torch.zeros(shape, dtype=dtype, device=device)
    return {
        "gated_scan": lambda: ops.gated_scan(f(2, 3, 12), f(2, 4), f(2, dtype=torch.int32), False, True, False),
        "gated_scan int8": lambda: ops.gated_scan(f(2, 3, 12).requires_grad_(True), None, None, False, True, True),
        "gated_scan_step": lambda: ops.gated_scan_step(f(2, 12), f(2, 4), None, True, f(2, 4)),
        "checkpoint8": lambda: ops.checkpoint8(f(3, 5)),
        "restore8": lambda: ops.restore8(f(3 * 34, dtype=torch.uint8), [3, 5], F32),
        "weight_grad8": lambda: ops.weight_grad8(f(3, 2), f(3 * 34, dtype=torch.uint8), 5, True),
        "linear8": lambda: ops.linear8(f(3, 5), f(2, 5), f(2)),
        "linear8 grad": lambda: ops.linear8(f(3, 5).requires_grad_(True), f(2, 5), f(2)),
    }


@pytest.mark.parametrize("name", sorted(_direct()))
def test_operators_refuse_host_tensors(name):
    with pytest.raises(RuntimeError, match="must be on the HIP device"):
        _direct()[name]()


@pytest.mark.parametrize("device", ["cuda", "cpu"])
@pytest.mark.parametrize("name", sorted(_direct()))
def test_operators_refuse_fake_tensors(name, device):
    """A tracer's tensors have no memory: nothing may follow their pointers or trace a call without its work."""
    from torch._subclasses.fake_tensor import FakeTensorMode
    with FakeTensorMode(), pytest.raises(RuntimeError, match="cannot be traced"):
        _direct(device=device)[name]()


@pytest.mark.parametrize("name", sorted(_direct()))
def test_operators_refuse_meta_tensors(name):
    with pytest.raises(RuntimeError, match="cannot be traced"):
        _direct(device="meta")[name]()


def test_operators_refuse_the_wrappers_of_function_transforms():
    ops = lib.load_ops()
    with pytest.raises(RuntimeError, match="cannot be traced"):
        torch.func.grad(lambda x: ops.linear8(x, torch.zeros(2, 5), None).sum())(torch.zeros(3, 5))
    with pytest.raises(RuntimeError, match="cannot be traced"):
        torch.func.grad(lambda z: ops.gated_scan(z, None, None, False, True, False)[0].sum())(torch.zeros(2, 3, 12))


def test_bind_takes_the_library_s_own_functions_only():
    import ctypes
    ops, l = lib.load_ops(), lib.load()
    names = ("sad_last_error", "sad_gated_scan_workspace_bytes", "sad_gated_scan_kept_bytes", "sad_gated_scan_codes_bytes",
             "sad_gated_scan_fwd", "sad_gated_scan_bwd", "sad_gated_scan_step", "sad_checkpoint8_bytes", "sad_checkpoint8_save",
             "sad_checkpoint8_restore", "sad_weight_grad8_workspace_bytes", "sad_weight_grad8")
    good = [ctypes.cast(getattr(l, n), ctypes.c_void_p).value for n in names]
    ops.bind(good)
    for i in range(12):
        for other in (0, 16, good[(i + 1) % 12], good[i] + 1, ctypes.cast(ctypes.CDLL(None).abort, ctypes.c_void_p).value):
            with pytest.raises(RuntimeError, match="address %d is not %s" % (i, names[i])):
                ops.bind(good[:i] + [other] + good[i + 1:])
    # what was bound stays
    with pytest.raises(RuntimeError, match="holds 34 bytes"):
        ops.restore8(torch.zeros(1, dtype=torch.uint8), [1, 5], F32)


def test_size_limits_are_those_of_a_launch():
    l = lib.load()
    most = (2 ** 32 - 1) // 64 // 4 * 4                          # waves of 64 threads in workgroups of four
    for B, D in ((most, 2), (most, 128), (most // 2, 129), (1, 1 << 24), (2 ** 25 + 100, 2)):
        assert l.sad_gated_scan_workspace_bytes(B, 1, D) == 16, (B, D)
        assert l.sad_gated_scan_kept_bytes(B, 1, D) == B * D * 4
    for B, D in ((most + 1, 2), (most // 2 + 1, 129), (2 ** 31 - 1, 2)):
        assert l.sad_gated_scan_workspace_bytes(B, 1, D) == 0 and "beyond the supported maximum" in lib.last_error()


def test_operators_without_the_library_raise():
    """The operator library loaded by itself has no functions to call: every operator says so instead of following NULL."""
    import subprocess
    import sys
    code = """
import sys, torch
torch.ops.load_library(sys.argv[1])
o, f, u = torch.ops.sad_amd, torch.zeros, torch.zeros(102, dtype=torch.uint8)
for call in (lambda: o.gated_scan(f(2, 3, 12), None, None, False, True, False), lambda: o.gated_scan_step(f(2, 12), f(2, 4), None, True, f(2, 4)),
             lambda: o.checkpoint8(f(3, 5)), lambda: o.restore8(u, [3, 5], torch.float32), lambda: o.weight_grad8(f(3, 2), u, 5, True),
             lambda: o.linear8(f(3, 5), f(2, 5), None)):
    try:
        call()
    except RuntimeError as e:
        assert "not bound" in str(e), e
    else:
        raise AssertionError("no error")
print("done")
"""
    r = subprocess.run([sys.executable, "-c", code, lib.OPS_PATH], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and r.stdout.split()[-1] == "done", (r.returncode, r.stderr[-400:])
