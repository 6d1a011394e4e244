"""Rounding error of the gated scan's kernels, entry by entry, from the recurrences of the errors themselves (float64).

u = 2^-24 is half a step of float32.  First-order bounds; the whole is multiplied by 1.05 for the higher orders.
  * A sigmoid is rcp(1 + exp2(L f)), L = log2 e as float32 (off by 0.22 u) times f (rounded): the exponential's relative error is
    1.22 |f| u from its argument and 2 u of its own, the sum adds u, the reciprocal 2 u.  A factor odds * sigmoid adds u.
        c(f) = (1.25 |f| + 8) u                                                          for s, a, so and 1 - so
  * h' = h + s (x - h): x - h and the sum are rounded once each:  e' = a e + (c + u) s |x - h| + u |h'|.
    Where a sentence is cut along time, h comes from maps (M, v): v is such a state from 0, M the same recurrence with x = 1,
    and h - M h + v is applied for at most 15 groups and 3 chunks, two roundings each, of a map composed of at most 4.  With
    A >= |h|, |v|, |x| over the channel's time, M and v together have at most twice the terms of one state:
        e'[t] = a e[t-1] + 2 ((c + u) s 2 A + u A)  ,  and 50 u A once for the joins
  * g[t] = dy so + a[t+1] g[t+1] likewise, with G >= the sum of |dy so| and |dh| under the same decays:
        e_g[t] = a e_g[t+1] + 2 (c s G + 2 u G) + (c(o) + u) |dy so|  ,  and 50 u G once
  * The backward pass recomputes states from the kept ones: at most twice e_h (with 8-bit codes the kept state's error, and
    that of states at the restored values).
  * dx = s g, df = -(a s g) (x - h), do = dy so h (1 - so): errors of g, h and of x - h (u |x - h| more) times the other
    factors, c for each sigmoid, u for each product."""
import numpy as np

from oracle import scan_oracle as O

U = 2.0 ** -24


def c(f):
    return (1.25 * np.abs(f) + 8) * U


def _order(T, reverse):
    return range(T - 1, -1, -1) if reverse else range(T)


def _state_error(x, f, h0, live, reverse):
    """Bounds [B,T+1,D] of the state's error after each step; index T: the state in front of the first one (exact)."""
    B, T, D = x.shape
    s, a = O.sigmoid(-f), O.sigmoid(f)
    A = np.abs(h0)
    top = A.copy()
    for t in _order(T, reverse):
        A = np.where(live[:, t], a[:, t] * A + s[:, t] * np.abs(x[:, t]), A)
        top = np.maximum(top, np.where(live[:, t], np.maximum(A, np.abs(x[:, t])), 0))
    e, out = np.zeros((B, D)), np.zeros((B, T + 1, D))
    for t in _order(T, reverse):
        e = np.where(live[:, t], a[:, t] * e + 2 * ((c(f[:, t]) + U) * s[:, t] * 2 * top + U * top), e)
        out[:, t] = e + 50 * U * top
    return out


def bounds(z, h0, lengths, reverse, gated, dy, dh, ref, int8=None):
    """Tolerances dict(y, h_last, dz, dh0) of float32 results for the oracle's ``ref`` (the arguments are the oracle's)."""
    B, T, W = z.shape
    D = W // (3 if gated else 2)
    n = np.full(B, T) if lengths is None else np.minimum(np.maximum(lengths, 0), T)
    live = (np.arange(T)[None] < n[:, None])[..., None]
    h0 = np.zeros((B, D)) if h0 is None else h0
    dh = np.zeros((B, D)) if dh is None else dh
    x, f = z[..., :D], z[..., D:2 * D]
    e_h = _state_error(x, f, h0, live, reverse)
    last = list(_order(T, reverse))[-1]
    out = {"h_last": e_h[:, last] * 1.05}
    so = O.sigmoid(z[..., 2 * D:]) if gated else np.ones_like(x)
    out["y"] = np.where(live, so * e_h[:, :T] + (c(z[..., 2 * D:]) + U if gated else 0) * np.abs(ref["y"]), 0) * 1.05
    # backward pass
    e_h = 2 * e_h
    if int8 is not None:
        z = int8
        x, f = z[..., :D], z[..., D:2 * D]
        e_h = e_h + _state_error(x, f, h0, live, reverse)
        so = O.sigmoid(z[..., 2 * D:]) if gated else so
    s, a = O.sigmoid(-f), O.sigmoid(f)
    dho = np.where(live, np.abs(dy) * so, 0.0)
    G = np.abs(dh)
    top = G.copy()
    for t in reversed(_order(T, reverse)):
        G = np.where(live[:, t], dho[:, t] + G, G)
        top = np.maximum(top, G)
        G = np.where(live[:, t], a[:, t] * G, G)
    dz = np.zeros((B, T, W))
    e = np.zeros((B, D))
    d = np.abs(ref["dz"])
    co = c(z[..., 2 * D:]) if gated else np.zeros_like(x)
    for t in reversed(_order(T, reverse)):
        ok = live[:, t]
        eg = e + (co[:, t] + U) * dho[:, t] + 50 * U * top
        with np.errstate(all="ignore"):
            g = np.where(s[:, t] > 0, d[:, t, :D] / s[:, t], top)
            diff = np.where(d[:, t, :D] > 0, d[:, t, D:2 * D] / (a[:, t] * d[:, t, :D]), np.inf)      # |h - x|
        diff = np.minimum(diff, np.abs(x[:, t]) + np.abs(h0) + np.abs(x).max(1))
        t_in = t + 1 if reverse else t - 1
        eh_in = e_h[:, t_in] if 0 <= t_in < T else 0.0
        dz[:, t, :D] = s[:, t] * eg + (c(f[:, t]) + U) * d[:, t, :D]
        dz[:, t, D:2 * D] = a[:, t] * s[:, t] * (eg * diff + g * (eh_in + U * diff)) + (2 * c(f[:, t]) + 4 * U) * d[:, t, D:2 * D]
        if gated:
            dz[:, t, 2 * D:] = np.abs(dy[:, t]) * so[:, t] * (1 - so[:, t]) * e_h[:, t] + (2 * co[:, t] + 5 * U) * d[:, t, 2 * D:]
        dz[:, t] = np.where(ok, dz[:, t], 0)
        step = 2 * (c(f[:, t]) * s[:, t] * top + 2 * U * top) + (co[:, t] + U) * dho[:, t]
        e = np.where(ok, a[:, t] * e + step, e)
    out["dz"] = dz * 1.05 + 1e-37
    out["dh0"] = (e + 50 * U * top) * 1.05
    return out


def misses(got, want, tol, half=0.0, least=0.0):
    """Entries beyond their bound.  ``half``: half a step of the type the results are rounded to, relative to the value;
    ``least``: half its smallest step.  Below the type's smallest normal number the step stays that of its subnormals (float16:
    2^-24 below 2^-14), so that rounding is off by up to 2^-25 there, more than 2^-11 of the value."""
    return ~(np.abs(got - want) <= tol + np.maximum(half * (np.abs(want) + tol), least))


# B, T, D, lengths, cut: what the gradient's carries have to cross.  63 chunks in 16 groups; 38 in 10; 25 in 7; 19 in 5; one
CASES = [(1, 5000, 6, None), (2, 1200, 300, [1200, 1111]), (3, 400, 130, [400, 17, 399]), (2, 300, 64, [300, 259]), (1, 2000, 34, None),
         (4, 45, 40, [45, 0, 33, 16])]


def make(case, gated, seed):
    """Inputs in float64 (to be rounded to their type by the caller): z, h0, dy, dh."""
    B, T, D, lengths = case
    r = np.random.default_rng(seed)
    z = r.normal(size=(B, T, (3 if gated else 2) * D))
    z[..., D:2 * D] += r.uniform(0, 6, size=D)
    return z, r.normal(size=(B, D)).astype(np.float32), r.normal(size=(B, T, D)), r.normal(size=(B, D)).astype(np.float32)
