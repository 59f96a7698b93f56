"""The block norm's paths for wide rows and many of them, on the GPU: rings of one and two stages that are refilled, one to four
chunks per thread, a row per warp with 6 to 16 warps and up to 32 loop steps.

Codes and scales are equal bit for bit to those of calls of few rows, which take another kernel (or another number of chunks), and on
sampled rows to the float64 oracle.  resid_out and out: within the tolerances of test_block_norm_gpu.py on the sampled rows."""
import pytest
import torch

import mx_oracle as mx
from gpu_util import poisoned, require_gpu
from test_block_norm_gpu import B, F, _make, _n, _near, _want

pytestmark = pytest.mark.gpu


def _rows_of(kw, rows):
    return {k: v[rows] if torch.is_tensor(v) and v.dim() == 2 and v.shape[0] > 1 else v for k, v in kw.items()}


def _logical(scales, T, H):
    """Scale bytes [T, H/32] of a tile-layout buffer, and whether its padding is zero."""
    r, c = -(-T // 128), -(-H // 128)
    s = scales.view(r, c, 32, 4, 4).permute(0, 3, 2, 1, 4).reshape(r * 128, c * 4)
    return s[:T, :H // 32], not (s[T:].any() or s[:, H // 32:].any())


def _check(p, T, H, kw, mx_too, out_too, few=96):
    dtype = (kw["resid"] if kw.get("resid") is not None else kw["y"]).dtype
    resid = torch.full((T, H), float("nan"), dtype=dtype, device="cuda")
    out = torch.full((T, H), float("nan"), dtype=B, device="cuda") if out_too else None
    amax = torch.full((1,), -1.0, device="cuda") if out_too else None
    codes = poisoned(T * H // 2).view(T, H // 2) if mx_too else None
    scales = poisoned(mx.scale_buffer_bytes(T, H)) if mx_too else None
    p.block_norm(**kw, resid_out=resid, out=out, amax=amax, codes=codes, scales=scales)
    torch.cuda.synchronize()
    assert p.read_device_error() == 0
    rows = torch.unique(torch.cat([torch.arange(3), torch.randint(0, T, (40,), generator=torch.Generator().manual_seed(T)),
                                   torch.arange(T - 3, T)]))
    part = _rows_of(kw, rows.cuda())
    r, z, dr, dz = _want(part)
    _near(resid[rows], r, dr, dtype)
    if out_too:
        _near(out[rows], z, dz, B)
        assert amax.item() == out.float().abs().max().item() and torch.isfinite(out.float()).all()
    if not mx_too:
        return
    byte, clean = _logical(scales, T, H)
    ref = mx.quantize(z)
    assert clean and (byte[rows].cpu().numpy() == ref[1]).all() and (codes[rows].cpu().numpy() == ref[0]).all()
    for i in range(0, T, few):
        n = min(few, T - i)
        got = p.block_norm(**_rows_of(kw, slice(i, i + n)), mx=True)
        assert torch.equal(got.codes, codes[i:i + n]) and torch.equal(_logical(got.scales, n, H)[0], byte[i:i + n])


# y and resid, rows, width, scale: a CTA per row where the scale is not positive or a row fills shared memory
@pytest.mark.parametrize("T,H,resid,y,scale", [
    (1500, 8192, B, B, 0.8),        # four chunks, two stages refilled
    (1600, 2816, F, F, -0.7), (1600, 2816, B, B, -1.0),
    (700, 16384, B, B, 1.0),        # two stages of 64 KB
    (700, 16384, F, F, 1.0),        # one stage of 128 KB, refilled
    (700, 16384, B, F, -1.0), (700, 14560, F, B, 1.0), (900, 12320, None, F, 0.5), (1000, 16384, F, None, 1.0)])
def test_cta_per_row(T, H, resid, y, scale):
    p = require_gpu()
    kw = {**_make(T, H, T + H, resid, y, gate="row" if y else ""), "scale": scale}
    _check(p, T, H, kw, True, False)
    _check(p, T, H, kw, True, True)
    _check(p, T, H, kw, False, True)


@pytest.mark.parametrize("T,H,resid,y", [
    (800, 4096, F, F),              # six warps
    (800, 4096, B, F), (1100, 5600, B, B), (800, 4064, None, B),
    (7200, 8192, B, None),          # twelve warps, 32 loop steps
    (7800, 4096, F, None), (4900, 6016, F, None)])
def test_warp_per_row_to_codes(T, H, resid, y):
    p = require_gpu()
    kw = {**_make(T, H, T + H, resid, y, gate="feature" if y else ""), "scale": 0.9}
    _check(p, T, H, kw, True, False)
    _check(p, T, H, kw, True, True)


@pytest.mark.parametrize("T,H,resid,y", [(4800, 6144, B, None), (9600, 4096, B, B), (5000, 4096, F, B), (4900, 8192, F, None), (7800, 4096, F, None),
                                         (1000, 2504, B, B)])
def test_warp_per_row_to_bf16(T, H, resid, y):
    p = require_gpu()
    _check(p, T, H, {**_make(T, H, T + H, resid, y, gate="row" if y else ""), "scale": -0.9}, False, True)
