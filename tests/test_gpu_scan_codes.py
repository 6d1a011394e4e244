"""GPU: the 8-bit codes that the scan keeps of its pre-activations, read back through the C entry, against the format's definition:
every 16-bit pattern, float32 over its whole range, rows of very different size, lost entries, odd channel counts."""
import ctypes

import numpy as np
import pytest

from oracle import scan_oracle as O

pytestmark = pytest.mark.gpu


def _codes(z, reverse, gated):
    """Values the codes stand for, [B,T,parts * D], NaN for lost entries; written from the layout in include/sad.h's terms:
    codes [B][blocks][parts][D][16], exponents [B][blocks][parts][ceil(D / 32)][16], a flag per 128 channels."""
    import torch
    from sad_amd import lib
    l = lib.load()
    B, T, W = z.shape
    parts = 3 if gated else 2
    D, nblk = W // parts, -(-T // 16)
    nb, ncg = -(-D // 32), -(-D // 128)
    kind = {torch.float32: lib.SRC_F32, torch.bfloat16: lib.SRC_BF16, torch.float16: lib.SRC_F16}[z.dtype]
    y, last = torch.empty(B, T, D, dtype=z.dtype, device="cuda"), torch.empty(B, D, device="cuda")
    kept = torch.empty(l.sad_gated_scan_kept_bytes(B, T, D), dtype=torch.uint8, device="cuda")
    codes = torch.full((l.sad_gated_scan_codes_bytes(B, T, D, int(gated)),), 77, dtype=torch.uint8, device="cuda")
    ws = torch.empty(l.sad_gated_scan_workspace_bytes(B, T, D), dtype=torch.uint8, device="cuda")
    a = lib.SadScanArgs()
    a.B, a.T, a.D, a.kind, a.gated, a.reverse = B, T, D, kind, int(gated), int(reverse)
    a.z, a.z_stride_b, a.z_stride_t = z.data_ptr(), z.stride(0), z.stride(1)
    a.y, a.y_stride_b, a.y_stride_t = y.data_ptr(), y.stride(0), y.stride(1)
    a.h_last, a.kept, a.codes = last.data_ptr(), kept.data_ptr(), codes.data_ptr()
    assert l.sad_gated_scan_fwd(ctypes.byref(a), ctypes.c_void_p(ws.data_ptr()), ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)) == 0
    raw = codes.cpu().numpy()
    n, m = B * nblk * parts * D * 16, B * nblk * parts * nb * 16
    code = raw[:n].view(np.int8).reshape(B, nblk, parts, D, 16).astype(np.float64)
    step = 2.0 ** (raw[n:n + m].reshape(B, nblk, parts, nb, 16).astype(np.float64) - 127)
    flag = raw[n + m:].view(np.uint32).reshape(B, nblk, ncg)
    v = np.where(code == -128, np.nan, code * np.repeat(step, 32, 3)[:, :, :, :D])
    assert set(np.unique(flag)) <= {0, 1}
    lost = np.isnan(v).any((2, 4))
    lost = np.pad(lost, ((0, 0), (0, 0), (0, ncg * 128 - D))).reshape(B, nblk, ncg, 128).any(3)
    assert (lost <= (flag == 1)).all()                            # a lost entry is always announced
    if reverse:
        v = v[..., ::-1]
    return v.transpose(0, 1, 4, 2, 3).reshape(B, nblk * 16, W)[:, :T]


@pytest.mark.parametrize("reverse", [False, True], ids=["fwd", "rev"])
@pytest.mark.parametrize("dtype", ["bfloat16", "float16"])
def test_every_16_bit_pattern(dtype, reverse):
    """Each pattern beside others of its size (a block of 32 neighbouring patterns), and in shuffled company."""
    import torch
    bits = np.arange(65536, dtype=np.uint16)
    mixed = np.random.default_rng(1).permutation(bits)
    for order in (bits, mixed):
        z = torch.from_numpy(order.reshape(1, -1, 256).view(np.int16)).view(getattr(torch, dtype)).cuda()      # [1,256,2 * 128]
        zz = z.double().cpu().numpy()
        assert np.array_equal(_codes(z, reverse, False), O.part_values(zz, False, dtype == "float16"), equal_nan=True)


@pytest.mark.parametrize("gated", [True, False])
@pytest.mark.parametrize("shape", [(2, 19, 33), (1, 16, 128), (3, 5, 161), (1, 33, 2), (2, 70, 258)], ids=str)
@pytest.mark.parametrize("dtype", ["float32", "bfloat16", "float16"])
def test_sizes_ranges_and_lost_entries(dtype, shape, gated):
    import torch
    B, T, D = shape
    r = np.random.default_rng(D)
    W = (3 if gated else 2) * D
    top = {"float32": 127, "bfloat16": 127, "float16": 15}[dtype]
    with np.errstate(over="ignore"):
        z = r.normal(size=(B, T, W)) * 2.0 ** r.integers(-top - 20, top, size=(B, T, 1))
    z = torch.from_numpy(z).to(getattr(torch, dtype)).cuda()
    for reverse in (False, True):
        zz = z.double().cpu().numpy()
        assert np.array_equal(_codes(z, reverse, gated), O.part_values(zz, gated, dtype == "float16"), equal_nan=True)
        bad = torch.from_numpy(r.random((B, T, W)) < 0.02).cuda()
        z = torch.where(bad, torch.full_like(z, float("nan") if reverse else float("inf")), z)
