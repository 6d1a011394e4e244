"""GPU tests of the gated scan and of the 8-bit activation checkpoints against the 64-bit oracle (oracle/scan_oracle.py).

Tolerances (fixed before the first run).  u = 2^-24 is half a step of float32, eps/2 half a step of the output type.
  * sigmoid as exp2 and reciprocal: the argument is rounded (|f| log2 e u absolute, ln 2 of it in the exponential), exp2,
    the sum and the reciprocal add two steps of 2 u each at most: relative error <= (|f| + 8) u.
  * state: the errors of s act on x - h, weighted with s and the decays, whose sum is at most one: (F + 8) u * 2 X with
    F = max|f|, X = max(|x|, |h0|) >= |h|; each step also rounds h twice (3 u X): T steps at most.
    => tol_h = (2 (F + 8) + 3 T) u X.   y adds (F + 8) u X and its own rounding.
  * g: the same recurrence on dy and dh: G = max|g| of the oracle: tol_g = (2 (F + 8) + 3 T) u G.  A gradient is a product
    of g (or dy <= G') with factors of at most 1 (dx), |h - x| / 4 <= X / 2 (df), |h| / 4 (do): its error is at most
    tol_g (1 + X) + G (1 + tol_h + 4 (F + 8) u (1 + X)), of which only the error terms count:
    => tol_dz = tol_g (1 + X) + G (tol_h + 4 (F + 8) u (1 + X)), plus eps/2 |dz|.
  * products of a weight gradient are exact (7 x 8, 7 x 11 significant bits, or three exact parts); m of them are added in
    float32 in some order: m u sum|terms| at most; the checkpoint's values are exact."""
import numpy as np
import pytest

from oracle import scan_oracle as O

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
TYPES = ["bf16", "fp16", "fp32"]


def _t():
    import torch
    return torch, {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def _dev(a, dt, layout="batch"):
    """numpy -> device tensor of type dt.  layout: batch [B,T,C]; time: [T,B,C] storage; wide: rows of a larger matrix,
    starting at an odd element."""
    torch, _ = _t()
    t = torch.from_numpy(np.ascontiguousarray(a)).to("cuda").to(dt)
    if layout == "time":
        return t.transpose(0, 1).contiguous().transpose(0, 1)
    if layout == "wide":
        big = torch.full(t.shape[:-1] + (t.shape[-1] + 5,), float("nan"), dtype=dt, device="cuda")
        big[..., 3:3 + t.shape[-1]] = t
        return big[..., 3:3 + t.shape[-1]]
    return t


def _np(t):
    return t.detach().double().cpu().numpy()


def _half(dt):
    torch, _ = _t()
    return torch.finfo(dt).eps / 2


def _check(got, ref, tol, half, what):
    bound = tol + half * (np.abs(ref) + tol)
    bad = ~(np.abs(got - ref) <= bound)
    assert not bad.any(), (what, int(bad.sum()), float(np.abs(got - ref).max()), float(np.min(bound)))


def _tols(z, D, h0, T):
    X = max(np.abs(z[..., :D]).max(), np.abs(h0).max() if h0 is not None else 0.0)
    F = np.abs(z[..., D:]).max()
    return X, F, (2 * (F + 8) + 3 * T) * U * X


def _case(B, T, D, dtype, gated, reverse, lengths, with_h0, save, layout="batch", seed=0, use_dy=True, use_dh=True):
    torch, DT = _t()
    from sad_amd import functional as Fn
    dt = DT[dtype]
    r = np.random.default_rng(seed)
    z = r.normal(size=(B, T, (3 if gated else 2) * D))
    z[..., D:2 * D] += r.uniform(0, 6, size=D)
    dy, dh = r.normal(size=(B, T, D)), r.normal(size=(B, D))
    h0 = r.normal(size=(B, D)).astype(np.float32) if with_h0 else None
    zt = _dev(z, dt, layout).requires_grad_(True)
    dyt = _dev(dy, dt, layout)
    h0t = torch.from_numpy(h0).cuda().requires_grad_(True) if with_h0 else None
    z, dy, dh = _np(zt), _np(dyt), dh.astype(np.float32).astype(np.float64)      # what the kernels see
    int8 = O.part_values(z, gated, dtype == "fp16") if save == "int8" else None
    ref = O.scan(z, h0, lengths, reverse, gated, int8=int8, dy=dy if use_dy else np.zeros_like(dy), dh_last=dh if use_dh else None)

    ln = None if lengths is None else torch.tensor(lengths, dtype=torch.int32, device="cuda")
    y, last = Fn.gated_scan(zt, h0=h0t, lengths=ln, reverse=reverse, gated_output=gated, save=save)
    assert y.dtype == dt and last.dtype == torch.float32 and tuple(y.shape) == (B, T, D) and tuple(last.shape) == (B, D)
    outs = ([y] if use_dy else []) + ([last] if use_dh else [])
    gout = ([dyt] if use_dy else []) + ([torch.from_numpy(dh.astype(np.float32)).cuda()] if use_dh else [])
    grads = torch.autograd.grad(outs, [zt] + ([h0t] if with_h0 else []), gout)

    X, F, tol_h = _tols(z, D, h0, T)
    _check(_np(last), ref["h_last"], tol_h, U, "h_last")
    _check(_np(y), ref["y"], tol_h + (F + 8) * U * X, _half(dt), "y")
    # largest |g|: |dy| and |dh| times the sum of the decays behind them; bounded from the data of the case
    z8 = z if int8 is None else int8
    X8, F8, tol8 = _tols(z8, D, h0, T)
    G = np.abs(ref["dh0"]).max() + np.abs(dh).max() + np.abs(dy).max() * min(T, 1.0 / (1.0 - O.sigmoid(F8)))
    X8 = max(X8, X)
    tol_g = (2 * (F8 + 8) + 3 * T) * U * G
    tol_dz = tol_g * (1 + X8) + G * (max(tol8, tol_h) + 4 * (F8 + 8) * U * (1 + X8))
    _check(_np(grads[0]), ref["dz"], tol_dz, _half(dt), "dz")
    if with_h0:
        _check(_np(grads[1]), ref["dh0"], tol_g, U, "dh0")
    if lengths is not None:      # rows behind a sentence
        for b, n in enumerate(lengths):
            assert (_np(y)[b, n:] == 0).all() and (_np(grads[0])[b, n:] == 0).all()
            if n == 0:
                assert np.array_equal(_np(last)[b], h0[b] if with_h0 else np.zeros(D))
    return y, last, grads


SHAPES = [
    (1, 1, 2, None), (3, 17, 5, [17, 0, 1]), (2, 16, 128, None), (4, 33, 130, [33, 16, 32, 15]), (5, 29, 331, [0, 29, 16, 17, 1]),
    (3, 50, 33, [50, 48, 2]),            # the last channel opens a block of 32 of its own
    (2, 47, 257, None), (2, 300, 64, [300, 259]), (1, 2000, 34, None), (40, 23, 300, None),
]


@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "%dx%dx%d" % s[:3])
@pytest.mark.parametrize("reverse", [False, True], ids=["fwd", "rev"])
@pytest.mark.parametrize("dtype", TYPES)
def test_scan_matches_oracle(shape, reverse, dtype):
    B, T, D, lengths = shape
    for gated, with_h0, save in ((True, True, "input"), (False, False, "input"), (True, False, "int8"), (False, True, "int8")):
        _case(B, T, D, dtype, gated, reverse, lengths, with_h0, save, seed=B + T + D)


@pytest.mark.parametrize("layout", ["time", "wide"])
@pytest.mark.parametrize("save", ["input", "int8"])
@pytest.mark.parametrize("dtype", TYPES)
def test_scan_strides(layout, save, dtype):
    y, _, grads = _case(4, 37, 45, dtype, True, False, [37, 3, 0, 20], True, save, layout=layout, seed=7)
    if layout == "time":
        assert y.transpose(0, 1).is_contiguous() and grads[0].transpose(0, 1).is_contiguous()


@pytest.mark.parametrize("use_dy,use_dh", [(True, False), (False, True)])
def test_scan_single_gradient(use_dy, use_dh):
    _case(3, 40, 66, "fp32", True, True, [40, 0, 31], True, "input", use_dy=use_dy, use_dh=use_dh, seed=9)


def test_scan_long_wide_batches():
    """The forms with and without a cut along time, at sizes with several chunks, and several sentences per workgroup."""
    _case(1, 5000, 6, "fp32", True, False, None, True, "input", seed=11)
    _case(2, 1200, 700, "bf16", True, True, [1200, 1111], False, "int8", seed=12)
    _case(300, 5, 520, "fp16", False, False, [5, 0, 3] * 100, True, "input", seed=13)


@pytest.mark.parametrize("save", ["input", "int8"])
@pytest.mark.parametrize("reverse", [False, True])
def test_scan_ignores_what_lies_behind_a_sentence(save, reverse):
    torch, _ = _t()
    from sad_amd import functional as Fn
    g = torch.Generator().manual_seed(5)
    z = torch.randn(3, 40, 3 * 70, generator=g)
    dy = torch.randn(3, 40, 70, generator=g)
    lengths = [21, 0, 40]
    zero, junk = z.clone(), z.clone()
    dzero, djunk = dy.clone(), dy.clone()
    for b, n in enumerate(lengths):
        zero[b, n:], dzero[b, n:] = 0.0, 0.0
        junk[b, n:], djunk[b, n:] = float("nan"), float("inf")
        junk[b, n:, ::2] = -float("inf")
    res = []
    for zz, dd in ((zero, dzero), (junk, djunk)):
        zt = zz.cuda().requires_grad_(True)
        y, last = Fn.gated_scan(zt, lengths=torch.tensor(lengths), reverse=reverse, save=save)      # host lengths
        dz, = torch.autograd.grad([y, last], [zt], [dd.cuda(), torch.ones_like(last)])
        res.append((y, last, dz))
    for a, b in zip(*res):
        assert torch.equal(a, b) and torch.isfinite(a).all()


def test_scan_extreme_gates():
    """Gates at and past the ends of the exponential: shares of exactly 0 and 1, no NaN; NaN in a token reaches its own
    channel only, from that token on."""
    torch, _ = _t()
    from sad_amd import functional as Fn
    z = torch.zeros(1, 6, 12)
    z[0, :, 0:4] = 2.0
    z[0, :, 4:8] = torch.tensor([-300.0, 300.0, float("-inf"), float("inf")])
    z[0, :, 8:12] = torch.tensor([300.0, -300.0, 0.0, float("inf")])
    zt = z.cuda().requires_grad_(True)
    h0 = torch.full((1, 4), 5.0, device="cuda")
    y, last = Fn.gated_scan(zt, h0=h0)
    assert last.tolist() == [[2.0, 5.0, 2.0, 5.0]]
    assert y[0, 3].tolist() == [2.0, 0.0, 1.0, 5.0]
    dz, = torch.autograd.grad([y, last], [zt], [torch.ones_like(y), torch.ones_like(last)])
    assert torch.isfinite(dz).all()
    z = torch.randn(1, 40, 12)
    z[0, 20, 1] = float("nan")
    y, last = Fn.gated_scan(z.cuda())
    bad = torch.isnan(y[0]).cpu()
    assert bad[20:, 1].all() and bad.sum() == 20 and torch.isnan(last[0]).tolist() == [False, True, False, False]


def test_scan_int8_keeps_nonfinite_tokens_to_themselves():
    """A NaN activation inside a sentence: the restored value is NaN, its neighbours in the block of 32 are unchanged."""
    torch, _ = _t()
    from sad_amd import functional as Fn
    z = torch.randn(1, 20, 3 * 40)
    clean = z.clone()
    z[0, 19, 3] = float("inf")          # the last token: only its own channel can be touched
    grads = []
    for t in (clean, z):
        zt = t.cuda().requires_grad_(True)
        y, _ = Fn.gated_scan(zt, save="int8")
        grads.append(torch.autograd.grad(y, zt, torch.ones_like(y))[0])
    same = torch.isclose(grads[0], grads[1], rtol=0, atol=0).reshape(20, 3, 40)
    assert same[..., :3].all() and same[..., 4:].all()
    assert torch.isnan(grads[1][0, 19]).any()


def test_scan_pieces_equal_the_whole():
    """Reading a text in pieces, state handed on, gives the whole's values up to the rounding of the states."""
    torch, _ = _t()
    from sad_amd import functional as Fn
    torch.manual_seed(2)
    z = torch.randn(3, 100, 3 * 36, device="cuda")
    y, last = Fn.gated_scan(z)
    h, parts = None, []
    for a, b in ((0, 1), (1, 17), (17, 64), (64, 100)):
        yp, h = Fn.gated_scan(z[:, a:b], h0=h)
        parts.append(yp)
    z64 = _np(z)
    _, _, tol = _tols(z64, 36, None, 100)
    assert (torch.cat(parts, 1) - y).abs().max() <= 2 * tol and (h - last).abs().max() <= 2 * tol
    hs, ys = torch.zeros(3, 36, device="cuda"), []
    for t in range(100):
        yt, hs = Fn.gated_scan_step(z[:, t], hs, h_out=hs)
        ys.append(yt)
    assert (torch.stack(ys, 1) - y).abs().max() <= 2 * tol and (hs - last).abs().max() <= 2 * tol


def test_scan_gradient_against_differences():
    """Directional differences of the kernels' own forward pass (float32).  The truncation at this step is computed with
    the oracle; the rounding is that of y and h_last divided by the step."""
    torch, _ = _t()
    from sad_amd import functional as Fn
    r = np.random.default_rng(8)
    B, T, D, step = 2, 30, 20, 2.0 ** -5
    z, d = r.normal(size=(B, T, 3 * D)).astype(np.float32), r.normal(size=(B, T, 3 * D)).astype(np.float32)
    dy, dh = r.normal(size=(B, T, D)).astype(np.float32), r.normal(size=(B, D)).astype(np.float32)
    lengths = [30, 13]

    def on_device(v):
        y, last = Fn.gated_scan(torch.from_numpy(v).cuda(), lengths=torch.tensor(lengths))
        return (_np(y) * dy).sum() + (_np(last) * dh).sum()

    def by_oracle(v):
        o = O.scan(v.astype(np.float64), None, lengths, False, True)
        return (o["y"] * dy).sum() + (o["h_last"] * dh).sum()

    up, down = (z + np.float32(step) * d), (z - np.float32(step) * d)
    zt = torch.from_numpy(z).cuda().requires_grad_(True)
    y, last = Fn.gated_scan(zt, lengths=torch.tensor(lengths))
    grad, = torch.autograd.grad([y, last], [zt], [torch.from_numpy(dy).cuda(), torch.from_numpy(dh).cuda()])
    along = (_np(grad) * (up.astype(np.float64) - down.astype(np.float64))).sum()
    ref = O.scan(z.astype(np.float64), None, lengths, False, True, dy=dy, dh_last=dh)
    exact_along = (ref["dz"] * (up.astype(np.float64) - down.astype(np.float64))).sum()
    truncation = abs((by_oracle(up) - by_oracle(down)) - exact_along)
    X, F, tol_h = _tols(np.abs(z.astype(np.float64)) + step * np.abs(d), D, None, T)
    rounding = 2 * (np.abs(dy).sum() + np.abs(dh).sum()) * (tol_h + (F + 9) * U * X)
    assert abs((on_device(up) - on_device(down)) - along) <= truncation + 2 * rounding


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("B,D", [(1, 2), (3, 45), (70, 512), (2, 1300)])
def test_step_matches_oracle(dtype, B, D):
    torch, DT = _t()
    from sad_amd import functional as Fn
    r = np.random.default_rng(B + D)
    for gated in (True, False):
        big = torch.from_numpy(r.normal(size=(B, 3 * D + 3))).cuda().to(DT[dtype])
        z = big[:, 1:1 + (3 if gated else 2) * D]
        h = torch.from_numpy(r.normal(size=(B, D)).astype(np.float32)).cuda()
        alive = torch.from_numpy(r.random(B) > 0.3).cuda()
        zz, hh = _np(z), _np(h)
        ref = O.scan(zz[:, None], hh, [int(v) for v in alive.cpu()], False, gated)
        X, F, tol = _tols(zz, D, hh, 1)
        y, out = Fn.gated_scan_step(z, h, alive=alive, gated_output=gated)
        _check(_np(out), ref["h_last"], tol, U, "h")
        _check(_np(y), ref["y"][:, 0], tol + (F + 8) * U * X, _half(DT[dtype]), "y")
        dead = ~alive
        assert torch.equal(out[dead], h[dead]) and (y[dead] == 0).all()
        kept, version = h.clone(), h._version
        y2, same = Fn.gated_scan_step(z, h, alive=alive, gated_output=gated, h_out=h)       # in place
        assert same is h and h._version > version and torch.equal(h, out) and torch.equal(y2, y) and not torch.equal(kept, h) or dead.all()


def test_empty_sizes():
    torch, _ = _t()
    from sad_amd import functional as Fn
    z = torch.zeros(2, 0, 12, device="cuda", requires_grad=True)
    h0 = torch.ones(2, 4, device="cuda", requires_grad=True)
    y, last = Fn.gated_scan(z, h0=h0)
    assert tuple(y.shape) == (2, 0, 4) and torch.equal(last, h0)
    assert torch.equal(torch.autograd.grad(last.sum(), h0)[0], torch.ones_like(h0))
    y, last = Fn.gated_scan(torch.zeros(0, 5, 12, device="cuda"))
    assert tuple(y.shape) == (0, 5, 4) and tuple(last.shape) == (0, 4)
    y, h = Fn.gated_scan_step(torch.zeros(0, 12, device="cuda"), torch.zeros(0, 4, device="cuda"))
    assert tuple(y.shape) == (0, 4)
    c = Fn.checkpoint8(torch.zeros(0, 7, device="cuda"))
    assert tuple(c.restore().shape) == (0, 7)
    dw, db = Fn.weight_grad8(torch.zeros(0, 3, device="cuda"), c, bias=True)
    assert tuple(dw.shape) == (3, 7) and not dw.any() and not db.any()


# ---- 8-bit checkpoints -----------------------------------------------------------------------------------------------
def _spread(r, rows, cols):
    """Rows of very different size, exact ties, zeros and block maxima just at and above 127 steps."""
    x = r.normal(size=(rows, cols)) * 2.0 ** r.integers(-12, 8, size=(rows, 1))
    x[rows // 2] = 0.0
    x[0] = r.integers(-254, 255, size=cols) * 0.5
    x[-1, 0] = 127.0
    return x


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,cols", [(1, 1), (5, 31), (3, 32), (7, 33), (70, 300), (3, 5001), (129, 64)])
def test_checkpoint_values_are_exact(dtype, rows, cols):
    torch, DT = _t()
    from sad_amd import functional as Fn
    r = np.random.default_rng(rows * cols)
    x = torch.from_numpy(_spread(r, rows, cols)).cuda().to(DT[dtype])
    got = Fn.checkpoint8(x).restore()
    assert got.dtype == x.dtype and np.array_equal(_np(got), O.code_values(_np(x), dtype == "fp16"))


@pytest.mark.parametrize("dtype", TYPES)
def test_checkpoint_ends_of_the_range(dtype):
    torch, DT = _t()
    from sad_amd import functional as Fn
    dt = DT[dtype]
    fi = torch.finfo(dt)
    x = torch.zeros(6, 40, dtype=dt, device="cuda")
    x[0, :3] = torch.tensor([fi.max, fi.min, fi.max / 2])
    x[1, :3] = torch.tensor([fi.tiny, -fi.tiny * 3, fi.tiny / 4])
    x[2, :4] = torch.tensor([float("nan"), float("inf"), -float("inf"), 1.0])
    x[3, 33] = float("nan")
    x[4] = float("inf")
    x[5, 5] = fi.smallest_subnormal if hasattr(fi, "smallest_subnormal") else fi.tiny
    want = O.code_values(_np(x), dtype == "fp16")
    got = _np(Fn.checkpoint8(x).restore())
    assert np.array_equal(got, want, equal_nan=True)
    assert np.isnan(got[2, :3]).all() and got[2, 3] == 1.0 and np.isnan(got[3]).sum() == 1 and np.isfinite(got[:2]).all()


def test_checkpoint_layouts():
    torch, _ = _t()
    from sad_amd import functional as Fn
    x = torch.randn(6, 5, 70, device="cuda")
    want = Fn.checkpoint8(x).restore()
    assert torch.equal(Fn.checkpoint8(x.transpose(0, 1).contiguous().transpose(0, 1)).restore(), want)
    assert torch.equal(Fn.checkpoint8(torch.cat([x, x], -1)[..., :70]).restore(), want)
    assert torch.equal(Fn.checkpoint8(x.permute(2, 0, 1).contiguous().permute(1, 2, 0)).restore(), want)      # channel stride 30
    assert torch.equal(Fn.checkpoint8(x.view(2, 3, 5, 70)).restore(), want.view(2, 3, 5, 70))
    assert torch.equal(Fn.checkpoint8(x[0, 0]).restore(), want[0, 0])
    assert torch.equal(Fn.checkpoint8(x[:1].expand(6, 5, 70)).restore(), want[:1].expand(6, 5, 70))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("M,N,K", [(1, 1, 1), (3, 5, 33), (64, 128, 128), (65, 129, 130), (1000, 77, 301), (4100, 300, 40), (700, 16, 640)])
def test_weight_grad(dtype, M, N, K):
    torch, DT = _t()
    from sad_amd import functional as Fn
    r = np.random.default_rng(M + N + K)
    x = torch.from_numpy(_spread(r, M, K)).cuda().to(DT[dtype])
    dy = torch.from_numpy(r.normal(size=(M, N))).cuda().to(DT[dtype])
    ck = Fn.checkpoint8(x)
    dw, db = Fn.weight_grad8(dy, ck, bias=True)
    xv, dv = O.code_values(_np(x), dtype == "fp16"), _np(dy)
    assert dw.dtype == torch.float32 and db.dtype == torch.float32
    bound = M * U * (np.abs(dv).T @ np.abs(xv)) * (3 if dtype == "fp32" else 1) + 1e-38
    assert (np.abs(_np(dw) - dv.T @ xv) <= bound).all()
    assert (np.abs(_np(db) - dv.sum(0)) <= M * U * np.abs(dv).sum(0)).all()
    again = Fn.weight_grad8(dy, ck)
    assert torch.equal(again, dw)
    # rows of another layout
    wide = torch.full((M, N + 3), float("nan"), dtype=dy.dtype, device="cuda")
    wide[:, 1:N + 1] = dy
    assert torch.equal(Fn.weight_grad8(wide[:, 1:N + 1], ck), dw)


def test_weight_grad_batched_rows_and_nonfinite():
    torch, _ = _t()
    from sad_amd import functional as Fn
    x, dy = torch.randn(7, 11, 50, device="cuda"), torch.randn(7, 11, 21, device="cuda")
    flat = Fn.weight_grad8(dy.view(77, 21), Fn.checkpoint8(x.view(77, 50)))
    t = lambda v: v.transpose(0, 1).contiguous().transpose(0, 1)
    assert torch.equal(Fn.weight_grad8(t(dy), Fn.checkpoint8(t(x))), flat)
    x[3, 4, 5] = float("inf")
    dw = Fn.weight_grad8(dy, Fn.checkpoint8(x))
    assert torch.isnan(dw[:, 5]).all() and torch.isfinite(dw[:, :5]).all() and torch.isfinite(dw[:, 6:]).all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("bias", [True, False])
def test_linear8(dtype, bias):
    """y and dx are the linear layer's own (its products of rounded operands, added in float32: k u sum|terms|, then
    rounded; a library that adds the bias after rounding rounds twice); dW, db from the restored input."""
    torch, DT = _t()
    from sad_amd import functional as Fn
    dt = DT[dtype]
    torch.manual_seed(4)
    B, T, K, N = 5, 9, 45, 70
    x = torch.randn(T, B, K, device="cuda").to(dt).transpose(0, 1).requires_grad_(True)
    w = (torch.randn(N, K, device="cuda") / K ** 0.5).requires_grad_(True)
    b = torch.randn(N, device="cuda").requires_grad_(True) if bias else None
    dy = torch.randn(B, T, N, device="cuda").to(dt)
    y = Fn.linear8(x, w, b)
    grads = torch.autograd.grad(y, [x, w] + ([b] if bias else []), dy)
    assert y.dtype == dt and grads[0].dtype == dt and grads[1].dtype == torch.float32
    xv, wv, dv = _np(x), _np(w.to(dt)), _np(dy)
    bv = _np(b.to(dt)) if bias else 0.0
    ref, mag = xv @ wv.T + bv, np.abs(xv) @ np.abs(wv).T + np.abs(bv)
    _check(_np(y), ref, (K + 1) * U * mag + _half(dt) * mag, _half(dt), "y")
    _check(_np(grads[0]), dv @ wv, N * U * (np.abs(dv) @ np.abs(wv)), _half(dt), "dx")
    xr = O.code_values(xv, dtype == "fp16").reshape(-1, K)
    d2 = dv.reshape(-1, N)
    assert (np.abs(_np(grads[1]) - d2.T @ xr) <= 3 * B * T * U * (np.abs(d2).T @ np.abs(xr))).all()
    if bias:
        assert (np.abs(_np(grads[2]) - d2.sum(0)) <= B * T * U * np.abs(d2).sum(0)).all()
    # frozen pieces, and parameters in the activations' type
    xf = x.detach()
    gw, = torch.autograd.grad(Fn.linear8(xf, w, b), w, dy)
    assert torch.equal(gw, grads[1])
    wd = w.detach().to(dt).requires_grad_(True)
    gd, = torch.autograd.grad(Fn.linear8(xf, wd), wd, dy)
    assert gd.dtype == dt and torch.equal(gd, grads[1].to(dt))
    gx, = torch.autograd.grad(Fn.linear8(x, w.detach(), b.detach() if bias else None), x, dy)
    assert torch.equal(gx, grads[0])
    with torch.no_grad():
        plain = Fn.linear8(x, w, b)
    assert not plain.requires_grad and torch.equal(plain, y) and plain.stride() == y.stride()
    with torch.autocast("cuda", dtype=torch.float16):                  # the type of x decides, inside autocast too
        assert torch.equal(Fn.linear8(x, w, b), y)
    one = Fn.linear8(xf[0, 0], wd)
    g1, = torch.autograd.grad(one, wd, dy[0, 0])
    assert tuple(one.shape) == (N,) and g1.abs().max() > 0


# ---- the operators together ------------------------------------------------------------------------------------------
def _layer(x, w, b, lengths):
    """A bidirectional recurrent layer as a user builds it: in-projections and scans, activations in 8 bits."""
    torch, _ = _t()
    from sad_amd import functional as Fn
    outs = []
    for d in range(2):
        z = Fn.linear8(x, w[d], b[d])
        y, last = Fn.gated_scan(z, lengths=lengths, reverse=d == 1, save="int8")
        outs.append((y, last))
    return torch.cat([o[0] for o in outs], -1), torch.cat([o[1] for o in outs], -1)


def test_layer_runs_and_trains():
    """Soft tokens -> embedding -> bidirectional layer -> loss: gradients reach the tokens and every parameter; a second
    identical run gives the same bits."""
    torch, _ = _t()
    from sad_amd import functional as Fn
    torch.manual_seed(6)
    B, T, V, E, H = 6, 19, 200, 48, 40
    emb = torch.randn(V, E, device="cuda").requires_grad_(True)
    S = torch.softmax(torch.randn(T, B, V, device="cuda"), -1).to(torch.bfloat16).transpose(0, 1).requires_grad_(True)
    w = [(torch.randn(3 * H, E, device="cuda") * 0.2).requires_grad_(True) for _ in range(2)]
    b = [torch.zeros(3 * H, device="cuda").requires_grad_(True) for _ in range(2)]
    lengths = torch.tensor([19, 19, 12, 5, 1, 0], device="cuda")
    leaves = [S, emb] + w + b

    def once():
        y, last = _layer(Fn.soft_embedding(S, emb), w, b, lengths)
        return torch.autograd.grad(y.float().square().mean() + last.square().mean(), leaves)

    first, second = once(), once()
    for i, (p, q) in enumerate(zip(first, second)):
        assert torch.isfinite(p).all() and p.abs().max() > 0, i
        if i != 1:                      # the embedding's own gradient is accumulated with atomics
            assert torch.equal(p, q), i
    assert not first[0][5].any() and first[0][0].any()      # the empty sentence


def test_other_stream_and_two_calls_at_once():
    torch, _ = _t()
    from sad_amd import functional as Fn
    torch.manual_seed(1)
    zs = [torch.randn(2, 900, 3 * 64, device="cuda") for _ in range(2)]
    want = [Fn.gated_scan(z) for z in zs]
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [None, None]
    for i, s in enumerate(streams):
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            got[i] = Fn.gated_scan(zs[i])
    for s in streams:
        torch.cuda.current_stream().wait_stream(s)
    for a, b in zip(got, want):
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


def test_captured_training_step_replays():
    """Forward and backward of projection and scan in one graph, replayed over new inputs with eager work in between."""
    torch, _ = _t()
    from sad_amd import functional as Fn
    torch.manual_seed(3)
    B, T, E, H = 3, 600, 64, 32
    x = torch.randn(B, T, E, device="cuda", dtype=torch.bfloat16)
    w = (torch.randn(3 * H, E, device="cuda") * 0.2).requires_grad_(True)
    dy = torch.randn(B, T, H, device="cuda", dtype=torch.bfloat16)
    lengths = torch.tensor([600, 77, 0], dtype=torch.int32, device="cuda")

    def step(xx):
        y, last = Fn.gated_scan(Fn.linear8(xx, w), lengths=lengths, save="int8")
        return y.detach(), last.detach(), torch.autograd.grad([y, last], [w], [dy, torch.ones_like(last)])[0]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            step(x)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(x)
    for k in range(4):
        x.copy_(torch.randn(B, T, E, device="cuda"))
        lengths.copy_(torch.tensor([600 - k, 77 + k, k], dtype=torch.int32, device="cuda"))
        graph.replay()
        torch.cuda.synchronize()
        kept = [o.clone() for o in out]
        for a, b in zip(kept, step(x)):
            assert torch.equal(a, b), k


def test_offsets_past_32_bits():
    """A tensor of more than 2^32 bytes: its last sentence equals the same sentence alone."""
    torch, _ = _t()
    from sad_amd import functional as Fn
    B, T, D = 1100, 650, 2048
    z = torch.zeros(B, T, 2 * D, dtype=torch.bfloat16, device="cuda")          # 5.9 GB
    z[-1].normal_()
    y, last = Fn.gated_scan(z, gated_output=False)
    y1, last1 = Fn.gated_scan(z[-1:], gated_output=False)
    X, F, tol = _tols(_np(z[-1:]), D, None, T)
    assert (last[-1] - last1[0]).abs().max() <= 2 * tol
    assert (y[-1].float() - y1[0].float()).abs().max() <= 2 * tol + 2 * X * 2.0 ** -8
    assert not y[0].any()
    ck = Fn.checkpoint8(z)
    assert torch.equal(ck.restore()[-1], Fn.checkpoint8(z[-1]).restore())


def test_gradient_of_an_expanded_output():
    """y.sum().backward() hands in an expanded gradient; a non-leaf z; gradients add up over two uses."""
    torch, _ = _t()
    from sad_amd import functional as Fn
    torch.manual_seed(9)
    z = torch.randn(2, 20, 3 * 8, device="cuda", requires_grad=True)
    y, _ = Fn.gated_scan(z * 1.0)
    g1, = torch.autograd.grad(y.sum(), z)
    y, _ = Fn.gated_scan(z)
    g2, = torch.autograd.grad(y, z, torch.ones_like(y))
    assert torch.equal(g1, g2)
    a, _ = Fn.gated_scan(z)
    b, _ = Fn.gated_scan(z)
    g3, = torch.autograd.grad(a.sum() + b.sum(), z)
    assert torch.equal(g3, g1 + g2)


def test_saved_input_may_not_change():
    torch, _ = _t()
    from sad_amd import functional as Fn
    z = torch.randn(2, 20, 3 * 8, device="cuda", requires_grad=True)
    zz = z * 1.0
    y, _ = Fn.gated_scan(zz)
    zz.add_(1.0)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()
    zz = z * 1.0
    y, _ = Fn.gated_scan(zz, save="int8")       # nothing of z is kept
    zz.add_(1.0)
    y.sum().backward()


def test_no_second_derivative():
    """create_graph works; differentiating the gradient again raises instead of returning something wrong."""
    torch, _ = _t()
    from sad_amd import functional as Fn
    z = torch.randn(2, 20, 3 * 8, device="cuda", requires_grad=True)
    y, _ = Fn.gated_scan(z)
    g, = torch.autograd.grad(y.sum(), z, create_graph=True)
    with pytest.raises(RuntimeError, match="no second derivative"):
        g.sum().backward()
    w = torch.randn(5, 24, device="cuda", requires_grad=True)
    g, = torch.autograd.grad(Fn.linear8(z, w).sum(), w, create_graph=True)
    with pytest.raises(RuntimeError, match="no second derivative"):
        g.sum().backward()


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("M,N,K", [(903, 4093, 3001), (705, 5101, 4001), (1503, 4001, 2001), (1311, 1501, 300), (2050, 128, 128)],
                         ids=["256x256", "192x256", "128x320", "128x128", "split"])
def test_weight_grad_tiles(dtype, M, N, K):
    """Every output tile of the kernel, at odd sizes with several stages, against a 64-bit product; then with lost entries in
    the first, a middle and the last stage: their columns are NaN, every other entry keeps its bits."""
    torch, DT = _t()
    from sad_amd import functional as Fn
    g = torch.Generator(device="cuda").manual_seed(M)
    x = torch.randn(M, K, device="cuda", generator=g).to(DT[dtype])
    dy = torch.randn(M, N, device="cuda", generator=g).to(DT[dtype])
    ck = Fn.checkpoint8(x)
    dw, db = Fn.weight_grad8(dy, ck, bias=True)
    xv, dv = ck.restore().double(), dy.double()
    assert ((dw.double() - dv.t() @ xv).abs() <= M * U * (dv.abs().t() @ xv.abs())).all()
    assert ((db.double() - dv.sum(0)).abs() <= M * U * dv.abs().sum(0)).all()
    bad = x.clone()
    cols = [0, K // 2, K - 1]
    for row, col in zip((5, M // 2, M - 1), cols):
        bad[row, col] = float("inf")
    dn = Fn.weight_grad8(dy, Fn.checkpoint8(bad))
    assert torch.isnan(dn[:, cols]).all()
    rest = [c for c in range(K) if c // 32 not in [c // 32 for c in cols]]
    assert torch.equal(dn[:, rest], dw[:, rest])
    assert torch.isfinite(dn).sum() == N * (K - 3)


@pytest.mark.parametrize("reverse", [False, True])
def test_scan_int8_lost_entries_in_long_sentences(reverse):
    """A lost forget gate in the middle of sentences cut along time: its own channel's gradient is NaN on the side the
    gradient flows to, every other channel keeps its bits."""
    torch, _ = _t()
    from sad_amd import functional as Fn
    torch.manual_seed(4)
    D = 96
    z = torch.randn(2, 1500, 3 * D)
    grads = []
    for lost in (False, True):
        zz = z.clone()
        if lost:
            zz[1, 700, D + 37] = float("nan")
        zt = zz.cuda().requires_grad_(True)
        y, last = Fn.gated_scan(zt, lengths=torch.tensor([1500, 1400]), reverse=reverse, save="int8")
        y = torch.where(torch.isnan(y), torch.zeros_like(y), y)
        grads.append(torch.autograd.grad(y.sum(), zt)[0].view(2, 1500, 3, D))
    other = [c for c in range(D) if c // 32 != 37 // 32]
    assert torch.equal(grads[0][..., other], grads[1][..., other]) and torch.equal(grads[0][0], grads[1][0])
    assert torch.isnan(grads[1][1, 700, :2, 37]).all()
    same_block = [c for c in range(32, 64) if c != 37]
    assert torch.isfinite(grads[1][..., same_block]).all()
