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


@pytest.mark.parametrize("save", ["input", "int8"])
@pytest.mark.parametrize("layout", ["time", "wide"])
def test_saved_tensors_kept_on_the_host(layout, save):
    """Hooks for saved tensors give z back in another layout than the forward pass saw (save_on_cpu: contiguous)."""
    torch, Fn = _t()
    torch.manual_seed(3)
    B, T, D = 5, 37, 40
    z = torch.randn(B, T, 3 * D, device="cuda")
    if layout == "time":
        z = z.transpose(0, 1).contiguous().transpose(0, 1)
    else:
        z = torch.cat([z, z], -1)[..., 7:7 + 3 * D]
    z.requires_grad_(True)
    lengths = torch.tensor([37, 0, 12, 36, 1], dtype=torch.int32, device="cuda")
    dy = torch.randn(B, T, D, device="cuda")

    def grad():
        y, last = Fn.gated_scan(z, lengths=lengths, save=save)
        return torch.autograd.grad([y, last], z, [dy, torch.ones_like(last)])[0]

    want = grad()
    with torch.autograd.graph.save_on_cpu():
        got = grad()
    assert torch.equal(got, want)
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t, lambda t: t.transpose(0, -1).contiguous().transpose(0, -1)):
        got = grad()                                                   # channel stride B, codes not contiguous
    assert torch.equal(got, want)


@pytest.mark.parametrize("unpack,message", [
    (lambda t: t[:1] if t.dim() == 3 else t, "saved z came back"),
    (lambda t: t.double() if t.dim() == 3 else t, "saved z came back"),
    (lambda t: t.cpu() if t.dim() == 3 else t, "saved z came back"),
    (lambda t: t[:-16] if t.element_size() == 1 else t, "kept states came back"),
    (lambda t: t.cpu() if t.element_size() == 1 else t, "came back"),
    (lambda t: t.cpu() if t.dtype.itemsize == 4 and t.dim() == 1 else t, "lengths came back"),
    (lambda t: t.long() if t.dtype.itemsize == 4 and t.dim() == 1 else t, "lengths came back"),
])
def test_saved_tensors_that_come_back_as_others_are_refused(unpack, message):
    torch, Fn = _t()
    z = torch.randn(2, 20, 3 * 8, device="cuda", requires_grad=True)
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t, unpack):
        y, _ = Fn.gated_scan(z, lengths=torch.tensor([20, 3], dtype=torch.int32, device="cuda"))
        with pytest.raises(RuntimeError, match=message):
            torch.autograd.grad(y.sum(), z)


@pytest.mark.parametrize("save", ["input", "int8"])
@pytest.mark.parametrize("layout", ["batch", "time"])
def test_scan_results_are_modified_in_place(layout, save):
    """A layer that goes on in place (dropout mask, residual) gives the gradients of the one that does not."""
    torch, Fn = _t()
    torch.manual_seed(5)
    B, T, D = 4, 21, 24
    z = torch.randn(B, T, 3 * D, device="cuda")
    if layout == "time":
        z = z.transpose(0, 1).contiguous().transpose(0, 1)
    z.requires_grad_(True)
    res = torch.randn(B, T, D, device="cuda", requires_grad=True)
    keep = (torch.rand(B, T, D, device="cuda") > 0.3).float()
    grads = []
    for inplace in (True, False):
        y, last = Fn.gated_scan(z, save=save)
        if inplace:
            y.mul_(keep)
            y += res
            last.mul_(2.0)
        else:
            y, last = y * keep + res, last * 2.0
        grads.append((y.detach(),) + torch.autograd.grad(y.square().sum() + last.square().sum(), [z, res]))
        assert (y.stride(0) < y.stride(1)) == (layout == "time")
    for a, b in zip(*grads):
        assert torch.equal(a, b)


@pytest.mark.parametrize("layout,shape", [("batch", (6, 20)), ("batch", (20,)), ("batch", (4, 6, 20)), ("time", (4, 6, 20)),
                                          ("batch", (2, 3, 5, 20))], ids=str)
def test_linear8_result_is_modified_in_place(layout, shape):
    torch, Fn = _t()
    torch.manual_seed(6)
    x = torch.randn(shape, device="cuda")
    if layout == "time":
        x = x.transpose(0, 1).contiguous().transpose(0, 1)
    x.requires_grad_(True)
    w, b = torch.randn(7, 20, device="cuda", requires_grad=True), torch.randn(7, device="cuda", requires_grad=True)
    res = torch.randn(shape[:-1] + (7,), device="cuda", requires_grad=True)
    grads = []
    for inplace in (True, False):
        y = Fn.linear8(x, w, b)
        if inplace:
            y.mul_(2.0)
            y += res
        else:
            y = y * 2.0 + res
        grads.append((y.detach(),) + torch.autograd.grad(y.square().sum(), [x, w, b, res]))
    for a, c in zip(*grads):
        assert torch.equal(a, c)
    with torch.no_grad():
        y = Fn.linear8(x, w, b)
    y += res                                            # made without a graph, modified with one
    assert torch.equal(torch.autograd.grad(y.sum(), res)[0], torch.ones_like(res))


@pytest.mark.parametrize("layout", ["batch", "time"])
def test_linear8_forward_derivative_without_a_graph(layout):
    """A dual tensor that needs no gradient: y is linear in it, and keeps its tangent."""
    torch, Fn = _t()
    import torch.autograd.forward_ad as fa
    g = torch.Generator().manual_seed(8)
    x, t = (torch.randint(-3, 4, (4, 6, 20), generator=g).float().cuda() for _ in range(2))      # exact in any order
    w = torch.randint(-3, 4, (7, 20), generator=g).float().cuda()
    if layout == "time":
        x, t = (v.transpose(0, 1).contiguous().transpose(0, 1) for v in (x, t))
    with fa.dual_level():
        y = fa.unpack_dual(Fn.linear8(fa.make_dual(x, t), w))
        assert torch.equal(y.primal, x @ w.t()) and torch.equal(y.tangent, t @ w.t())


@pytest.mark.parametrize("rows,K,N", [((2, 3), 0, 5), ((2, 3), 4, 0), ((), 0, 5), ((2, 0), 4, 5), ((0,), 0, 0)], ids=str)
def test_linear8_with_an_empty_axis(rows, K, N):
    """As the linear layer: no input channel gives the bias, no output channel and no row give empty results."""
    torch, Fn = _t()
    x, w = torch.ones(rows + (K,), device="cuda", requires_grad=True), torch.ones(N, K, device="cuda", requires_grad=True)
    b = torch.arange(N, dtype=torch.float32, device="cuda").requires_grad_(True)
    out = []
    for f in (Fn.linear8, torch.nn.functional.linear):
        y = f(x, w, b)
        out.append((y,) + torch.autograd.grad(y.sum(), [x, w, b]))
    for a, c in zip(*out):
        assert a.shape == c.shape and torch.equal(a, c)


def test_dual_tensors_are_refused_where_a_tangent_would_be_lost():
    torch, Fn = _t()
    import torch.autograd.forward_ad as fa
    with fa.dual_level():
        z = fa.make_dual(torch.zeros(2, 3, 12, device="cuda"), torch.ones(2, 3, 12, device="cuda"))
        h = torch.zeros(2, 4, device="cuda")
        with pytest.raises(RuntimeError, match="no forward-mode derivative"):
            Fn.gated_scan(z)
        with pytest.raises(RuntimeError, match="no forward-mode derivative"):
            Fn.gated_scan(z, save="int8")
        with pytest.raises(RuntimeError, match="no forward-mode derivative"):
            Fn.gated_scan_step(z[:, 0], h)
        assert not h.any()
        assert not Fn.gated_scan(fa.unpack_dual(z).primal)[0].any()


def test_pinned_lengths_may_be_refilled_after_the_call():
    """The copy to the device waits behind earlier work on the stream; the caller's buffer is free as soon as the call is back."""
    torch, Fn = _t()
    torch.manual_seed(7)
    z = torch.randn(3, 40, 3 * 16, device="cuda")
    lengths = torch.tensor([40, 7, 0], dtype=torch.int32).pin_memory()
    want = Fn.gated_scan(z, lengths=[40, 7, 0])
    a = torch.randn(4096, 4096, device="cuda")
    torch.cuda.synchronize()
    for _ in range(40):
        a = (a @ a) * 1e-3                       # some milliseconds of work in front
    got = Fn.gated_scan(z, lengths=lengths)
    lengths.fill_(1)
    torch.cuda.synchronize()
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


@pytest.mark.parametrize("dtype", ["uint8", "int16", "uint32", "int64"])
def test_device_lengths_of_any_integer_type_are_clamped(dtype):
    torch, Fn = _t()
    torch.manual_seed(2)
    z = torch.randn(3, 20, 3 * 8, device="cuda")
    top = {"uint8": 255, "int16": 2 ** 15 - 1, "uint32": 2 ** 32 - 1, "int64": 2 ** 40 + 1}[dtype]
    lengths = torch.tensor([top, 7, 0], dtype=torch.int64).to(getattr(torch, dtype)).cuda()
    for a, b in zip(Fn.gated_scan(z, lengths=lengths), Fn.gated_scan(z, lengths=[20, 7, 0])):
        assert torch.equal(a, b)


def test_operators_check_their_own_arguments():
    """torch.ops.sad_amd is public: what the kernels assume is checked there too."""
    torch, Fn = _t()
    from sad_amd import lib
    ops = lib.load_ops()
    f = lambda *shape, dtype=torch.float32: torch.zeros(shape, dtype=dtype, device="cuda")
    scan = lambda z=f(2, 3, 12), h0=None, lengths=None: ops.gated_scan(z, h0, lengths, False, True, False)
    step = lambda z=f(2, 12), h=f(2, 4), alive=None, h_out=f(2, 4): ops.gated_scan_step(z, h, alive, True, h_out)
    scan(), step()
    for call, message in (
        (lambda: scan(f(2, 3, 13)), "parts of two channels"), (lambda: scan(f(2, 12)), "parts of two channels"),
        (lambda: scan(f(2, 12, 3).transpose(1, 2)), "unit channel stride"), (lambda: scan(f(2, 3, 12, dtype=torch.float64)), "expected float32"),
        (lambda: scan(h0=f(1, 4)), "h0 must be"), (lambda: scan(h0=f(2, 4, dtype=torch.float16)), "h0 must be"),
        (lambda: scan(h0=f(2, 8)[:, :4]), "h0 must be contiguous"), (lambda: scan(h0=torch.zeros(2, 4)), "HIP device"),
        (lambda: scan(lengths=f(3, dtype=torch.int32)), "lengths must hold 2"), (lambda: scan(lengths=f(2, dtype=torch.int64)), "int32"),
        (lambda: scan(lengths=torch.zeros(2, dtype=torch.int32)), "HIP device"),
        (lambda: step(h=f(2, 3)), "h must be"), (lambda: step(h_out=f(4, 2).t()), "h_out must be"), (lambda: step(h=torch.zeros(2, 4)), "HIP device"),
        (lambda: step(alive=f(2)), "alive must be"), (lambda: step(alive=f(1, dtype=torch.bool)), "alive must hold"),
        (lambda: ops.linear8(f(3, 5), f(2, 4), None), "do not fit"), (lambda: ops.linear8(f(3, 5), f(2, 5), f(3)), "bias must hold"),
        (lambda: ops.linear8(f(3, 5), torch.zeros(2, 5), None), "HIP device"),
        (lambda: ops.checkpoint8(f(2, 3, dtype=torch.int32)), "expected float32"),
    ):
        with pytest.raises(RuntimeError, match=message):
            call()


def _f32(bits):
    import struct
    return struct.unpack("f", struct.pack("I", bits))[0]


@pytest.mark.parametrize("M,N,K", [(40, 21, 50), (700, 130, 33), (4100, 40, 40)])
@pytest.mark.parametrize("value", [0x7f800000, 0xff800000, 0x7f7fffff, 0xff7fffff, 0x7f7f8000, 0x7f7f7fff, 0x7f800001, 0x7fc00000],
                         ids=["inf", "-inf", "max", "-max", "rounds up in bf16", "rounds down in bf16", "NaN in the low half", "NaN"])
def test_weight_grad_of_float32_at_the_end_of_the_range(M, N, K, value):
    """dY as float32 enters in parts: an infinity stays one, a largest finite entry stays finite, and other rows of dW keep their
    bits.  Tolerance: three exact products of M terms each, added in float32: 3 M 2^-24 sum|terms|."""
    import numpy as np
    torch, Fn = _t()
    torch.manual_seed(M)
    x = torch.randn(M, K, device="cuda") * 2.0 ** -12
    x[M // 2, 3] = 0.0
    dy = torch.randn(M, N, device="cuda")
    ck = Fn.checkpoint8(x)
    dw, db = Fn.weight_grad8(dy, ck, bias=True)
    big = dy.clone()
    big[:, 5] = 0.0
    big.view(torch.int32)[M // 2, 5] = value - (1 << 32 if value >> 31 else 0)
    gw, gb = Fn.weight_grad8(big, ck, bias=True)
    v = _f32(value)
    xv = ck.restore().double().cpu().numpy()
    with np.errstate(all="ignore"):
        want = np.float64(v) * xv[M // 2] + (0.0 * xv).sum(0)
        got = gw[5].double().cpu().numpy()
        if np.isfinite(v):
            assert (np.abs(got - want) <= 3 * M * 2.0 ** -24 * np.abs(want)).all()
        else:
            assert np.array_equal(got, want, equal_nan=True)
    assert np.array_equal(gb[5].double().cpu().numpy(), np.float64(v), equal_nan=True)
    rest = [n for n in range(N) if n != 5]
    assert torch.equal(gw[rest], dw[rest]) and torch.equal(gb[rest], db[rest])


def test_more_than_2_31_threads():
    """A batch whose launch has more than 2^31 threads: forward and backward of its ends equal those of the ends alone."""
    torch, Fn = _t()
    B = 2 ** 25 + 100
    g = torch.Generator(device="cuda").manual_seed(1)
    z = torch.empty(B, 1, 6, dtype=torch.float16, device="cuda").normal_(generator=g).requires_grad_(True)
    dy = torch.empty(B, 1, 2, dtype=torch.float16, device="cuda").normal_(generator=g)
    y, last = Fn.gated_scan(z)
    dz, = torch.autograd.grad([y, last], z, [dy, torch.ones_like(last)])
    for rows in (slice(0, 64), slice(B // 2, B // 2 + 64), slice(B - 64, B)):
        zz = z.detach()[rows].clone().requires_grad_(True)
        yy, ll = Fn.gated_scan(zz)
        assert torch.equal(y[rows], yy) and torch.equal(last[rows], ll)
        assert torch.equal(dz[rows], torch.autograd.grad([yy, ll], zz, [dy[rows], torch.ones_like(ll)])[0])


@pytest.mark.parametrize("save", ["input", "int8"])
def test_gradient_of_time_major_rows_of_a_wider_matrix(save):
    """y and dz come back in z's axis order, also where z's rows have gaps."""
    torch, Fn = _t()
    torch.manual_seed(12)
    T, B, D = 21, 5, 12
    wide = torch.randn(T, B, 3 * D + 7, device="cuda")
    got = []
    for z in (wide[..., 2:2 + 3 * D].transpose(0, 1), wide[..., 2:2 + 3 * D].transpose(0, 1).contiguous()):
        z = z.detach().requires_grad_(True)
        y, last = Fn.gated_scan(z, save=save)
        grads = []
        z.register_hook(lambda g: grads.append(g))
        (y.square().sum() + last.sum()).backward()
        got.append((y, grads[0]))
    for a, b in zip(*got):
        assert torch.equal(a, b) and a.transpose(0, 1).is_contiguous() and b.is_contiguous()


@pytest.mark.parametrize("save", ["input", "int8"])
def test_training_past_32_bits(save):
    """Tensors of more than 2^32 bytes, forward and backward: the last sentences equal the same sentences alone (both calls are
    uncut, so bit for bit)."""
    torch, Fn = _t()
    B, T, D, n = 1100, 650, 2048, 64
    z = torch.zeros(B, T, 2 * D, dtype=torch.bfloat16, device="cuda")          # 5.9 GB
    z[-n:].normal_()
    z.requires_grad_(True)
    dy = torch.empty(B, T, D, dtype=torch.bfloat16, device="cuda").normal_()
    lengths = torch.full((B,), T, dtype=torch.int32, device="cuda")
    lengths[-3:] = torch.tensor([0, 17, 600])
    y, last = Fn.gated_scan(z, lengths=lengths, gated_output=False, save=save)
    dz, = torch.autograd.grad([y, last], z, [dy, torch.ones_like(last)])
    part = z.detach()[-n:].clone().requires_grad_(True)
    yp, lp = Fn.gated_scan(part, lengths=lengths[-n:], gated_output=False, save=save)
    dp, = torch.autograd.grad([yp, lp], part, [dy[-n:], torch.ones_like(lp)])
    assert torch.equal(y[-n:], yp) and torch.equal(last[-n:], lp) and torch.equal(dz[-n:], dp)


@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
def test_weight_grad_past_32_bits(dtype):
    """dy of more than 2^32 bytes, small whole numbers: every sum is exact, so the rows of both ends alone give the same bits."""
    torch, Fn = _t()
    dt = getattr(torch, dtype)
    M, N, K, n = 1_500_001, 1531, 40, 1000
    g = torch.Generator(device="cuda").manual_seed(3)
    x = torch.randint(-63, 64, (M, K), device="cuda", generator=g).to(dt)
    dy = torch.zeros(M, N, dtype=dt, device="cuda")
    ends = [slice(0, n), slice(M - n, M)]
    for e in ends:
        dy[e] = torch.randint(-8, 9, (n, N), device="cuda", generator=g).to(dt)
    dw, db = Fn.weight_grad8(dy, Fn.checkpoint8(x), bias=True)
    xe, de = torch.cat([x[e] for e in ends]), torch.cat([dy[e] for e in ends])
    ew, eb = Fn.weight_grad8(de, Fn.checkpoint8(xe), bias=True)
    assert torch.equal(dw, ew) and torch.equal(db, eb)
    assert torch.equal(ew.double(), de.double().t() @ xe.double()) and torch.equal(eb.double(), de.double().sum(0))


def test_step_operator_refuses_overlapping_states():
    """The operator itself, past functional's checks: a shifted state would be read by some lanes after others wrote it."""
    torch, Fn = _t()
    from sad_amd import lib
    step = lambda z, h, h_out: lib.load_ops().gated_scan_step(z, h, None, True, h_out)
    z, buf = torch.zeros(2, 12, device="cuda"), torch.zeros(3, 4, device="cuda")
    flat = torch.zeros(24, device="cuda")
    for args, message in (((z, buf[:2], buf[1:]), "must not overlap it"), ((z, buf[1:], buf[:2]), "must not overlap it"),
                          ((z, buf[:2], torch.zeros(1, 4, device="cuda").expand(2, 4)), "rows of h_out overlap"),
                          ((flat.view(2, 12), buf[:2], flat[16:].view(2, 4)), "must not overlap z")):
        with pytest.raises(RuntimeError, match=message):
            step(*args)
    step(z, buf[:2], buf[:2])
    step(z, torch.zeros(1, 4, device="cuda").expand(2, 4), buf[:2])
    step(z[:1], buf[:1], buf[1:2])
