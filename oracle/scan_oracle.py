"""Plain 64-bit implementations of the gated linear recurrence and of the 8-bit checkpoint format (numpy, step by step).
Test infrastructure only; written from the formulas, nothing of the package is imported."""
import numpy as np

KEPT = 16      # steps between the states a training call keeps
BLOCK = 32     # channels that share an exponent


def sigmoid(v):
    with np.errstate(over="ignore"):
        return 1.0 / (1.0 + np.exp(-v))


def code_values(x, fp16=False):
    """Values of an 8-bit checkpoint of x [..., C] (any float type), float64."""
    lo, hi = (-24, 10) if fp16 else (-126, 122)
    x = np.asarray(x, np.float64)
    out = np.empty_like(x)
    for c in range(0, x.shape[-1], BLOCK):
        v = x[..., c:c + BLOCK]
        finite = np.isfinite(v)
        top = np.where(finite, np.abs(v), 0.0).max(-1, keepdims=True) if v.size else np.zeros(v.shape[:-1] + (1,))
        e = np.full(top.shape, lo)
        for k in range(lo, hi):                       # the smallest exponent whose 127 steps reach the largest entry
            e = np.where(top > 127.0 * 2.0 ** k, k + 1, e)
        cap = np.where(e == hi, 63.0, 127.0)
        step = 2.0 ** e.astype(np.float64)
        q = np.clip(np.rint(np.where(finite, v, 0.0) / step), -cap, cap)
        out[..., c:c + BLOCK] = np.where(finite, q * step, np.nan)
    return out


def scan(z, h0, lengths, reverse, gated, int8=None, dy=None, dh_last=None):
    """z [B,T,3D|2D] float64; returns dict(y, h_last) and, with dy, dict(..., dz, dh0).  ``int8``: None, or the values the
    backward pass sees in place of z."""
    B, T, W = z.shape
    D = W // (3 if gated else 2)
    y, h_last = np.zeros((B, T, D)), np.zeros((B, D))
    dz, dh0 = np.zeros((B, T, W)), np.zeros((B, D))
    for b in range(B):
        n = T if lengths is None else min(max(int(lengths[b]), 0), T)
        order = range(n - 1, -1, -1) if reverse else range(n)
        h = np.zeros(D) if h0 is None else h0[b].astype(np.float64)
        before, after = np.zeros((T, D)), np.zeros((T, D))
        for t in order:
            x, f = z[b, t, :D], z[b, t, D:2 * D]
            before[t] = h
            h = sigmoid(f) * h + sigmoid(-f) * x
            after[t] = h
            y[b, t] = sigmoid(z[b, t, 2 * D:]) * h if gated else h
        h_last[b] = h
        if dy is None:
            continue
        w = z if int8 is None else int8
        if int8 is not None:                          # states inside a block of KEPT steps: recomputed from what was kept
            for t in order:
                starts = (t == n - 1 or t % KEPT == KEPT - 1) if reverse else t % KEPT == 0
                h = before[t] if starts else h
                before[t] = h
                h = sigmoid(w[b, t, D:2 * D]) * h + sigmoid(-w[b, t, D:2 * D]) * w[b, t, :D]
                after[t] = h
        g = np.zeros(D) if dh_last is None else dh_last[b].astype(np.float64)
        for t in reversed(order):
            x, f = w[b, t, :D], w[b, t, D:2 * D]
            a, s = sigmoid(f), sigmoid(-f)
            if gated:
                so = sigmoid(w[b, t, 2 * D:])
                dz[b, t, 2 * D:] = dy[b, t] * after[t] * so * sigmoid(-w[b, t, 2 * D:])
                g = g + dy[b, t] * so
            else:
                g = g + dy[b, t]
            dz[b, t, :D] = s * g
            dz[b, t, D:2 * D] = a * s * g * (before[t] - x)
            g = a * g
        dh0[b] = g
    out = dict(y=y, h_last=h_last)
    if dy is not None:
        out.update(dz=dz, dh0=dh0)
    return out


def part_values(z, gated, fp16=False):
    """What the backward pass of a call with 8-bit activations sees: x, f, o as checkpoints of their own."""
    return np.concatenate([code_values(p, fp16) for p in np.split(z, 3 if gated else 2, axis=-1)], axis=-1)
