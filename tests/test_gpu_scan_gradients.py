"""GPU: results and gradients of the gated scan in long sentences, every entry against the 64-bit oracle within the bound of its own
rounding errors (tests/scan_bounds.py, checked on the CPU in test_scan_bounds.py)."""
import numpy as np
import pytest

from oracle import scan_oracle as O
from tests import scan_bounds as SB

pytestmark = pytest.mark.gpu


def _np(t):
    return t.detach().double().cpu().numpy()


@pytest.mark.parametrize("gated,save", [(True, "input"), (False, "input"), (True, "int8"), (False, "int8")])
@pytest.mark.parametrize("reverse", [False, True], ids=["fwd", "rev"])
@pytest.mark.parametrize("dtype", ["bfloat16", "float16", "float32"])
@pytest.mark.parametrize("case", SB.CASES, ids=["%dx%dx%d" % c[:3] for c in SB.CASES])
def test_every_entry_within_its_own_error(case, dtype, reverse, gated, save):
    import torch
    from sad_amd import functional as Fn
    B, T, D, lengths = case
    dt = getattr(torch, dtype)
    z, h0, dy, dh = SB.make(case, gated, seed=B + T)
    zt, dyt = (torch.from_numpy(v).cuda().to(dt) for v in (z, dy))
    z, dy = _np(zt), _np(dyt)
    zt.requires_grad_(True)
    h0t = torch.from_numpy(h0).cuda().requires_grad_(True)
    y, last = Fn.gated_scan(zt, h0=h0t, lengths=lengths, reverse=reverse, gated_output=gated, save=save)
    dz, dh0 = torch.autograd.grad([y, last], [zt, h0t], [dyt, torch.from_numpy(dh).cuda()])
    int8 = O.part_values(z, gated, dtype == "float16") if save == "int8" else None
    ref = O.scan(z, h0, lengths, reverse, gated, int8=int8, dy=dy, dh_last=dh)
    tol = SB.bounds(z, h0, lengths, reverse, gated, dy, dh, ref, int8=int8)
    half, least = torch.finfo(dt).eps / 2, torch.finfo(dt).smallest_normal * torch.finfo(dt).eps / 2
    for name, got, h in (("y", y, (half, least)), ("h_last", last, ()), ("dz", dz, (half, least)), ("dh0", dh0, ())):
        bad = SB.misses(_np(got), ref[name], tol[name], *h)
        assert not bad.any(), (name, int(bad.sum()), float(np.max(np.abs(_np(got) - ref[name])[bad])))
