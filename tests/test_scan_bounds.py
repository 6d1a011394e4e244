"""CPU checks of the error bounds the GPU's gradients are held against: float32 arithmetic of the kernels' kind stays within
them, and they are narrow enough to reject gradients that lost what a chunk's carry brings."""
import numpy as np
import pytest

from tests import scan_bounds as SB
from oracle import scan_oracle as O

F = np.float32
IDS = ["%dx%dx%d" % c[:3] for c in SB.CASES]


def _f32_scan(z, h0, lengths, reverse, gated, dy, dh):
    """The recurrence and its gradient step by step in float32, in the kernels' forms."""
    B, T, W = z.shape
    D = W // (3 if gated else 2)
    z, dy = z.astype(F), dy.astype(F)
    n = np.full(B, T) if lengths is None else np.asarray(lengths)
    L = F(1.4426950408889634)
    odds = np.exp2(L * z[..., D:2 * D])
    s = (F(1) / (F(1) + odds)).astype(F)
    u = np.exp2(-L * z[..., 2 * D:]) if gated else np.zeros_like(s)
    so = (F(1) / (F(1) + u)).astype(F)
    order = list(range(T - 1, -1, -1) if reverse else range(T))
    h, y = h0.astype(F), np.zeros((B, T, D), F)
    before, after, dz = np.zeros((B, T, D), F), np.zeros((B, T, D), F), np.zeros((B, T, W), F)
    for t in order:
        ok = (t < n)[:, None]
        before[:, t] = h
        h = np.where(ok, h + s[:, t] * (z[:, t, :D] - h), h)
        after[:, t] = h
        y[:, t] = np.where(ok, h * so[:, t] if gated else h, 0)
    last, carry = h, dh.astype(F)
    for t in reversed(order):
        ok = (t < n)[:, None]
        g0 = dy[:, t] * so[:, t] if gated else dy[:, t]
        g = g0 + carry
        dx = s[:, t] * g
        parts = [dx, -(odds[:, t] * s[:, t] * dx) * (z[:, t, :D] - before[:, t])]
        if gated:
            parts.append(g0 * after[:, t] * (u[:, t] * so[:, t]))
        dz[:, t] = np.where(ok, np.concatenate(parts, -1), 0)
        carry = np.where(ok, g - s[:, t] * g, carry)
    return dict(y=y, h_last=last, dz=dz, dh0=carry)


def _reference(case, gated, reverse, seed=3):
    z, h0, dy, dh = SB.make(case, gated, seed)
    z, dy = z.astype(F).astype(np.float64), dy.astype(F).astype(np.float64)
    ref = O.scan(z, h0, case[3], reverse, gated, dy=dy, dh_last=dh)
    return z, h0, dy, dh, ref, SB.bounds(z, h0, case[3], reverse, gated, dy, dh, ref)


@pytest.mark.parametrize("reverse", [False, True], ids=["fwd", "rev"])
@pytest.mark.parametrize("case", SB.CASES, ids=IDS)
@pytest.mark.parametrize("gated", [True, False])
def test_float32_arithmetic_stays_within_the_bounds(case, gated, reverse):
    z, h0, dy, dh, ref, tol = _reference(case, gated, reverse)
    got = _f32_scan(z, h0, case[3], reverse, gated, dy, dh)
    for k in ("y", "h_last", "dz", "dh0"):
        assert not SB.misses(got[k].astype(np.float64), ref[k], tol[k]).any(), k


@pytest.mark.parametrize("reverse", [False, True], ids=["fwd", "rev"])
@pytest.mark.parametrize("case", SB.CASES, ids=IDS)
def test_bounds_reject_wrong_carries(case, reverse):
    """The bound is far below the gradient, part by part; without the carry across one boundary of 16 steps, with one chunk's
    gradient in another's place, with the long channels' carry off by a hundredth, a gradient is rejected (in bfloat16 too)."""
    B, T, D, lengths = case
    z, h0, dy, dh, ref, tol = _reference(case, True, reverse)
    dz, half = ref["dz"], 2.0 ** -8
    for q in range(3):
        part = slice(q * D, (q + 1) * D)
        rms = lambda v: np.sqrt(np.mean(np.square(v)))
        assert rms(tol["dz"][..., part]) < 0.05 * rms(dz[..., part]), (q, rms(tol["dz"][..., part]), rms(dz[..., part]))
    assert np.mean(SB.misses(np.zeros_like(dz), dz, tol["dz"], half)) > 0.9 * np.mean(dz != 0)
    k = T // 2 // 16 * 16
    # the halves of the sequence, each for itself, with nothing carried from the later one into the earlier one's gradient
    first, second = (slice(k, T), slice(0, k)) if reverse else (slice(0, k), slice(k, T))
    ln = [T] * B if lengths is None else lengths
    cut = lambda sl: [min(max(n - sl.start, 0), sl.stop - sl.start) for n in ln]
    lost = dz.copy()
    lost[:, first] = O.scan(z[:, first], h0, cut(first), reverse, True, dy=dy[:, first], dh_last=np.zeros_like(dh))["dz"]
    wrong = SB.misses(lost, dz, tol["dz"], half)
    assert wrong[..., :2 * D].any() and not wrong[:, second].any()
    # the carry a hundredth too large
    enter = O.scan(z[:, first], h0, cut(first), reverse, True)["h_last"]
    carry = O.scan(z[:, second], enter, cut(second), reverse, True, dy=dy[:, second], dh_last=dh)["dh0"]
    right, off = (O.scan(z[:, first], h0, cut(first), reverse, True, dy=dy[:, first], dh_last=carry * m)["dz"] for m in (1.0, 1.01))
    assert not SB.misses(right, dz[:, first], tol["dz"][:, first]).any()
    assert SB.misses(off, dz[:, first], tol["dz"][:, first]).any()
    shifted = dz.copy()
    shifted[:, :T - 16] = dz[:, 16:]
    assert np.mean(SB.misses(shifted, dz, tol["dz"], half)) > 0.5 * np.mean(dz != 0)
