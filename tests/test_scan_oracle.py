"""CPU checks of the gated scan and of the 8-bit checkpoints: the 64-bit oracle against differences and hand-made values,
and the refusals of the Python and C entry points (nothing is launched)."""
import ctypes

import numpy as np
import pytest
import torch

from oracle import scan_oracle as O
from sad_amd import functional as Fn
from sad_amd import lib


@pytest.mark.parametrize("reverse", [False, True])
@pytest.mark.parametrize("gated", [False, True])
def test_oracle_gradient_matches_differences(reverse, gated):
    r = np.random.default_rng(3)
    B, T, D = 3, 7, 4
    z, h0 = r.normal(size=(B, T, (3 if gated else 2) * D)), r.normal(size=(B, D))
    dy, dh, lengths = r.normal(size=(B, T, D)), r.normal(size=(B, D)), [7, 0, 4]
    ref = O.scan(z, h0, lengths, reverse, gated, dy=dy, dh_last=dh)

    def loss(zz, hh):
        o = O.scan(zz, hh, lengths, reverse, gated)
        return (o["y"] * dy).sum() + (o["h_last"] * dh).sum()

    eps = 1e-5      # truncation ~ eps^2, rounding ~ 1e-16 * |loss| / eps: both below 1e-9
    for arr, grad in ((z, ref["dz"]), (h0, ref["dh0"])):
        for idx in np.ndindex(arr.shape):
            keep = arr[idx]
            arr[idx] = keep + eps
            up = loss(z, h0)
            arr[idx] = keep - eps
            down = loss(z, h0)
            arr[idx] = keep
            assert abs((up - down) / (2 * eps) - grad[idx]) < 1e-8, idx


def test_oracle_closed_form():
    """Constant input and decay: h_t = x (1 - a^t), and the gradient of its sum in x is sum (1 - a^t)."""
    T = 40
    z = np.zeros((1, T, 4))
    z[..., :2], z[..., 2:] = 1.5, 2.0
    a = 1.0 / (1.0 + np.exp(-2.0))
    o = O.scan(z, None, None, False, False, dy=np.ones((1, T, 2)))
    t = np.arange(1, T + 1)
    assert np.allclose(o["y"][0, :, 0], 1.5 * (1 - a ** t), rtol=0, atol=1e-13)
    assert np.allclose(o["dz"][0, :, 0].sum(), (1 - a ** t).sum(), rtol=1e-13)


def test_checkpoint_format_by_hand():
    x = np.zeros((1, 40))
    x[0, :4] = [127.0, 1.0, 0.5, -1.5]             # step 1: ties to even
    x[0, 32:36] = [127.5, np.nan, np.inf, 3.0]     # step 2 in the second block of channels, two entries lost
    v = O.code_values(x)
    assert v[0, :4].tolist() == [127.0, 1.0, 0.0, -2.0]
    assert v[0, 32] == 128.0 and np.isnan(v[0, 33:35]).all() and v[0, 35] == 4.0
    top = float(np.finfo(np.float32).max)
    assert O.code_values(np.array([[top, -top]])).tolist() == [[63 * 2.0 ** 122, -63 * 2.0 ** 122]]
    assert O.code_values(np.array([[65504.0, 2.0 ** -24]]), fp16=True).tolist() == [[63 * 2.0 ** 10, 0.0]]
    assert O.code_values(np.array([[3 * 2.0 ** -24, 2.0 ** -24]]), fp16=True).tolist() == [[3 * 2.0 ** -24, 2.0 ** -24]]


Z = torch.zeros(2, 3, 12)


@pytest.mark.parametrize("kw,message", [
    (dict(z=torch.zeros(2, 12)), "must be"),
    (dict(z=torch.zeros(2, 3, 13)), "13 columns"),
    (dict(z=torch.zeros(2, 3, 3)), "3 columns"),                               # one channel
    (dict(z=torch.zeros(2, 3, 12, dtype=torch.float64)), "float32, bfloat16 or float16"),
    (dict(z=Z, h0=torch.zeros(2, 5)), "h0 must be"),
    (dict(z=Z, h0=torch.zeros(2, 4, dtype=torch.float16)), "h0 must be"),
    (dict(z=Z, lengths=[1, 2, 3]), "lengths must be 2 integers"),
    (dict(z=Z, lengths=torch.tensor([1.0, 2.0])), "lengths must be 2 integers"),
    (dict(z=Z, lengths=torch.tensor([True, False])), "lengths must be 2 integers"),
    (dict(z=Z, lengths=[1, 4]), "0..3"),
    (dict(z=Z, lengths=[-1, 3]), "0..3"),
    (dict(z=Z, save="int4"), "save must be"),
    (dict(z=Z), "no CPU path"),
])
def test_scan_refusals(kw, message):
    with pytest.raises(RuntimeError, match=message):
        Fn.gated_scan(**kw)


S, H = torch.zeros(2, 12), torch.zeros(2, 4)


@pytest.mark.parametrize("args,kw,message", [
    ((Z, H), {}, "z must be"),
    ((torch.zeros(2, 13), H), {}, "13 columns"),
    ((S, torch.zeros(2, 4, dtype=torch.bfloat16)), {}, "h must be"),
    ((S, torch.zeros(2, 3)), {}, "h must be"),
    ((S, torch.zeros(4, 2).t()), {}, "h must be"),                             # channel stride 2
    ((S, H), dict(alive=torch.zeros(3, dtype=torch.bool)), "alive must be"),
    ((S, H), dict(alive=torch.zeros(2)), "alive must be"),
    ((S, H), dict(h_out=torch.zeros(2, 4, dtype=torch.float16)), "h_out must be"),
    ((S, H), dict(h_out=torch.zeros(1, 4).expand(2, 4)), "rows of h_out overlap"),
    ((S, torch.zeros(3, 4)[:2]), dict(h_out=None), "no CPU path"),
    ((S.clone().requires_grad_(True), H), {}, "no gradient"),
])
def test_step_refusals(args, kw, message):
    with pytest.raises(RuntimeError, match=message):
        Fn.gated_scan_step(*args, **kw)


def test_step_refuses_shifted_state():
    buf = torch.zeros(3, 4)
    with pytest.raises(RuntimeError, match="must not overlap"):
        Fn.gated_scan_step(S, buf[:2], h_out=buf[1:])
    flat = torch.zeros(24)
    with pytest.raises(RuntimeError, match="must not overlap z"):
        Fn.gated_scan_step(flat.view(2, 12), H, h_out=flat[:8].view(2, 4))


@pytest.mark.parametrize("call,message", [
    (lambda: Fn.checkpoint8(torch.zeros(3, 4, dtype=torch.int8)), "float32, bfloat16 or float16"),
    (lambda: Fn.checkpoint8(torch.tensor(1.0)), "channel axis"),
    (lambda: Fn.checkpoint8(torch.zeros(3, 4)), "no CPU path"),
    (lambda: Fn.weight_grad8(torch.zeros(3, 5), Fn.Checkpoint8(torch.zeros(1, dtype=torch.uint8), (4, 6), torch.float32)), "does not belong"),
    (lambda: Fn.weight_grad8(torch.zeros(4, 5), Fn.Checkpoint8(torch.zeros(1, dtype=torch.uint8), (4, 6), torch.float16)), "does not belong"),
    (lambda: Fn.weight_grad8(torch.zeros(4, 5), Fn.Checkpoint8(torch.zeros(1, dtype=torch.uint8), (4, 6), torch.float32)), "no CPU path"),
    (lambda: Fn.linear8(torch.zeros(4, 6), torch.zeros(5, 7)), "do not fit"),
    (lambda: Fn.linear8(torch.zeros(4, 6), torch.zeros(5, 6, dtype=torch.float16)), "weight must be"),
    (lambda: Fn.linear8(torch.zeros(4, 6), torch.zeros(5, 6), torch.zeros(6)), "bias must be"),
    (lambda: Fn.linear8(torch.zeros(4, 6), torch.zeros(5, 6)), "no CPU path"),
])
def test_checkpoint_refusals(call, message):
    with pytest.raises(RuntimeError, match=message):
        call()


def test_c_entries_refuse_without_a_launch():
    l = lib.load()
    assert l.sad_gated_scan_workspace_bytes(0, 4, 8) == 0 and "B >= 1" in lib.last_error()
    assert l.sad_gated_scan_kept_bytes(2, 33, 5) == 2 * 3 * 5 * 4
    assert l.sad_gated_scan_codes_bytes(2, 33, 33, 1) == 2 * 3 * (3 * (33 + 2) * 16 + 4)
    assert l.sad_checkpoint8_bytes(7, 33) == 7 * 68 and l.sad_checkpoint8_bytes(0, 3) == 0
    assert l.sad_checkpoint8_bytes(1 << 30, 1) > 0 and l.sad_checkpoint8_bytes((1 << 30) + 1, 1) == 0
    assert l.sad_weight_grad8_workspace_bytes(5, 0, 3, lib.SRC_BF16) == 0
    a = lib.SadScanArgs()
    one = ctypes.c_void_p(16)                                       # never followed: every call below is refused

    def refused(rc, text):
        assert rc == -1 and text in lib.last_error(), lib.last_error()

    refused(l.sad_gated_scan_fwd(None, one, None), "args is NULL")
    refused(l.sad_gated_scan_fwd(ctypes.byref(a), one, None), "B >= 1")
    a.B, a.T, a.D, a.kind = 2, 3, 4, 7
    refused(l.sad_gated_scan_fwd(ctypes.byref(a), one, None), "kind must be")
    a.kind = lib.SRC_F16
    refused(l.sad_gated_scan_fwd(ctypes.byref(a), one, None), "z is NULL")
    a.z = a.y = a.h_last = 16
    refused(l.sad_gated_scan_fwd(ctypes.byref(a), None, None), "workspace is NULL")
    a.codes = 16
    refused(l.sad_gated_scan_fwd(ctypes.byref(a), one, None), "codes need kept")
    a.kept, a.codes = 16, 20
    refused(l.sad_gated_scan_fwd(ctypes.byref(a), one, None), "16-byte aligned")
    refused(l.sad_gated_scan_bwd(ctypes.byref(a), one, None), "dz is NULL")
    a.z = a.codes = None
    refused(l.sad_gated_scan_bwd(ctypes.byref(a), one, None), "need z or codes")
    refused(l.sad_gated_scan_step(2, 4, lib.SRC_IDS, 1, one, 12, one, 4, None, one, 4, one, 4, None), "kind must be")
    refused(l.sad_gated_scan_step(2, 4, lib.SRC_F32, 1, None, 12, one, 4, None, one, 4, one, 4, None), "z is NULL")
    refused(l.sad_checkpoint8_save(1, 2, 3, lib.SRC_F32, one, 0, 3, ctypes.c_void_p(8), None), "16-byte aligned")
    refused(l.sad_checkpoint8_save(0, 2, 3, lib.SRC_F32, one, 0, 3, one, None), "rows must be positive")
    refused(l.sad_checkpoint8_save(1 << 20, 1 << 20, 3, lib.SRC_F32, one, 0, 3, one, None), "beyond the supported maximum")
    refused(l.sad_checkpoint8_restore(2, 3, lib.SRC_F32, None, one, None), "saved is NULL")
    refused(l.sad_weight_grad8(1, 2, 3, 4, 9, one, 0, 3, one, one, None, one, None), "kind must be")
    refused(l.sad_weight_grad8(1, 2, 3, 4, lib.SRC_F32, one, 0, 3, one, None, None, one, None), "dw is NULL")


def test_missing_operator_library_fails_loudly(monkeypatch):
    monkeypatch.setattr(lib, "_ops", None)
    monkeypatch.setattr(lib, "OPS_PATH", "/nonexistent/libsad_torch.so")
    with pytest.raises(RuntimeError, match="libsad_torch.so not found"):
        lib.load_ops()


def test_operators_are_registered():
    ops = lib.load_ops()
    for name in ("gated_scan", "gated_scan_step", "checkpoint8", "restore8", "weight_grad8", "linear8"):
        assert getattr(ops, name).default is not None
    with pytest.raises(RuntimeError, match="12 addresses"):
        ops.bind([0])
