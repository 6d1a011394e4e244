"""GPU tests of infinite states, activations and gradients in the gated scan, against the 64-bit oracle.  The recurrence is
linear: with a finite token an infinite state stays what it is, and opposite infinities give NaN.  Every channel is a recurrence of
its own, so the finite channels beside it keep the bits of a call without infinities."""
import numpy as np
import pytest

from oracle import scan_oracle as O

pytestmark = pytest.mark.gpu
INF = float("inf")


def _t():
    import torch
    from sad_amd import functional as Fn
    return torch, Fn


def _np(t):
    return t.detach().double().cpu().numpy()


def _kinds(a):
    """0 finite, 1 / -1 infinite, 2 NaN."""
    return np.where(np.isnan(a), 2, np.where(np.isinf(a), np.sign(np.nan_to_num(a)), 0))


# B, T, D, lengths: one block; a few blocks; cut along time with empty and short sentences behind which whole chunks lie
SHAPES = [(1, 7, 4, None), (2, 40, 5, [40, 33]), (3, 600, 6, [600, 37, 0]), (2, 5000, 4, [4999, 16])]


@pytest.mark.parametrize("save", ["input", "int8"])
@pytest.mark.parametrize("reverse", [False, True], ids=["fwd", "rev"])
@pytest.mark.parametrize("dtype", ["float32", "bfloat16", "float16"])
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "%dx%dx%d" % s[:3])
@pytest.mark.parametrize("where", ["h0", "x", "x twice", "dh_last", "dy"])
def test_infinities_follow_the_definition(where, shape, dtype, reverse, save):
    torch, Fn = _t()
    if where.startswith("x") and save == "int8":
        where = "h0"                                        # 8-bit codes keep an infinite x as a lost entry
    B, T, D, lengths = shape
    dt = getattr(torch, dtype)
    r = np.random.default_rng(T + D)
    z = torch.from_numpy(r.uniform(-2, 2, size=(B, T, 3 * D))).to(dt)
    t = {"h0": r.uniform(1, 2, size=(B, D)), "dh_last": r.uniform(1, 2, size=(B, D)), "dy": r.uniform(1, 2, size=(B, T, D))}
    t = {k: torch.from_numpy(v).to(dt if k == "dy" else torch.float32) for k, v in t.items()}
    bad_z, bad = z.clone(), {k: v.clone() for k, v in t.items()}
    c = D - 2                                               # the channel; every sentence of the batch has one entry
    for b in range(B):
        n = T if lengths is None else lengths[b]
        if where.startswith("x") and n > 0:
            order = list(range(n - 1, -1, -1)) if reverse else list(range(n))
            bad_z[b, order[n // 2], c] = INF
            if where == "x twice" and n > 3:
                bad_z[b, order[n // 2 + 2], c] = -INF
        elif where in ("h0", "dh_last"):
            bad[where][b, c] = -INF if b % 2 else INF
        elif where == "dy" and n > 0:
            bad["dy"][b, n // 2, c] = INF
    out = []
    for zz, tt in ((z, t), (bad_z, bad)):
        zc, h0 = zz.cuda().requires_grad_(True), tt["h0"].cuda().requires_grad_(True)
        y, last = Fn.gated_scan(zc, h0=h0, lengths=lengths, reverse=reverse, save=save)
        dz, dh0 = torch.autograd.grad([y, last], [zc, h0], [tt["dy"].cuda(), tt["dh_last"].cuda()])
        out.append((y, last, dz.view(B, T, 3, D), dh0))
    zn = _np(bad_z)
    with np.errstate(all="ignore"):
        ref = O.scan(zn, _np(bad["h0"]), lengths, reverse, True, int8=O.part_values(zn, True, dtype == "float16") if save == "int8" else None,
                     dy=_np(bad["dy"]), dh_last=_np(bad["dh_last"]))
    assert not np.isfinite(np.concatenate([ref[k].ravel() for k in ("y", "h_last", "dz", "dh0")])).all()
    others = [k for k in range(D) if k != c]
    for got, clean, name in zip(out[1], out[0], ("y", "h_last", "dz", "dh0")):
        want = ref[name].reshape(got.shape)
        assert torch.equal(got[..., others], clean[..., others]), name
        assert np.array_equal(_kinds(_np(got)), _kinds(want)), (name, where)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16", "float16"])
def test_infinities_in_the_step(dtype):
    torch, Fn = _t()
    z = torch.zeros(5, 12, dtype=getattr(torch, dtype), device="cuda")
    z[3, 1], z[4, 1] = INF, -INF
    h = torch.ones(5, 4, device="cuda")
    h[0, 1], h[1, 1], h[3, 1], h[4, 1] = INF, -INF, INF, INF
    y, out = Fn.gated_scan_step(z, h)
    for got in (y, out):
        assert got[:4, 1].tolist()[0:2] == [INF, -INF] and got[3, 1] == INF and torch.isnan(got[4, 1])
        assert torch.isfinite(got[:, [0, 2, 3]]).all() and torch.isfinite(got[2]).all()
