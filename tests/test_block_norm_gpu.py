"""The block norm on the GPU against its float64 definition.

MXFP4 codes and scales are equal bit for bit.  bf16 outputs: half a step (2^-8) plus the fp32 error of the value, fp32
outputs: that error alone.  With u = 2^-24 the error of r is at most 20 u a, a = |scale| (|resid| + |gate n|) (a mean of
squares and its root, three products, a sum and a product), that of z at most |z| (16 + 20 k) u + 20 u a |f w| with
k = sqrt(sum a^2 / sum r^2) per row; both are taken twice here."""
import itertools

import numpy as np
import pytest
import torch

import mx_oracle as mx
from gpu_util import poisoned, require_gpu

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


def _n(t):
    return None if t is None else t.double().cpu().numpy()


def _want(kw):
    """Float64 r and z, and their tolerances."""
    names = ("resid", "norm_weight", "y", "post_weight", "gate")
    v = {k: _n(kw.get(k)) for k in names}
    eps, scale = float(np.float32(kw.get("eps", 1e-6))), float(np.float32(kw.get("scale", 1.0)))
    post = kw.get("post_norm")
    with np.errstate(over="ignore", invalid="ignore", divide="ignore"):
        r, z = mx.block_norm(eps=eps, post_norm=post, scale=scale, **v)
        n, _ = mx.block_norm(None, None, eps, v["y"], v["post_weight"], post, v["gate"]) if v["y"] is not None else (0, 0)
        a = abs(scale) * (np.abs(n) + (np.abs(v["resid"]) if v["resid"] is not None else 0))
        f = 1 / np.sqrt((r * r).mean(1, keepdims=True) + eps)
        k = np.sqrt((a * a).sum(1, keepdims=True) / np.maximum((r * r).sum(1, keepdims=True), 1e-300))
        w = 1.0 if v["norm_weight"] is None else np.abs(v["norm_weight"])
        return r, z, 40 * U * a, 2 * U * (np.abs(z) * (16 + 20 * k) + 20 * a * f * w)


def _near(got, ref, tol, dtype):
    got = _n(got)
    tol = tol + np.abs(ref) * (2.0 ** -8 if dtype == torch.bfloat16 else U) + 2.0 ** -133
    ok = (np.abs(got - ref) <= tol) | (np.isnan(got) & np.isnan(ref))
    assert ok.all(), (np.argwhere(~ok)[:4].tolist(), got[~ok][:4], ref[~ok][:4])


def _check(p, T, H, want_mx, want_out, resid_out=None, **kw):
    r, z, dr, dz = _want(kw)
    out = torch.full((T, H), float("nan"), dtype=torch.bfloat16, device="cuda") if want_out else None
    amax = torch.full((1,), -1.0, device="cuda") if want_out else None
    codes = poisoned(T * H // 2).view(T, H // 2) if want_mx else None
    scales = poisoned(mx.scale_buffer_bytes(T, H)) if want_mx else None
    if resid_out is None:
        resid_out = torch.full((T, H), float("nan"), dtype=torch.float32, device="cuda")
    got = p.block_norm(resid_out=resid_out, out=out, amax=amax, codes=codes, scales=scales, **kw)
    torch.cuda.synchronize()
    _near(got.resid, r, dr, resid_out.dtype)
    if want_out:
        _near(out, z, dz, torch.bfloat16)
        assert amax.item() == out.float().abs().max().item()
    if want_mx:
        byte, clean = mx.untile_scales(scales.cpu().numpy(), T, H)
        ref = mx.quantize(z)
        assert np.array_equal(byte, ref[1]) and clean
        assert np.array_equal(codes.cpu().numpy(), ref[0])
    return got


def _make(T, H, seed, resid, y, post=True, gate="", std=3.0):
    g = torch.Generator("cuda").manual_seed(seed)
    rn = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    kw = {"norm_weight": (1 + 0.1 * rn(H)).bfloat16()}
    if resid:
        kw["resid"] = rn(T, H).to(resid)
    if y:
        kw["y"] = (std * rn(T, H)).to(y)
        if post:
            kw["post_weight"] = (1 + 0.1 * rn(H)).bfloat16()
        shape = {"": None, "feature": (H,), "row": (T, 1), "full": (T, H)}[gate]
        if shape:
            kw["gate"] = torch.sigmoid(rn(*shape))
    return kw


B, F = torch.bfloat16, torch.float32


@pytest.mark.parametrize("T,H", [(1, 32), (1, 2816), (3, 96), (130, 160), (129, 2816), (64, 4096), (9, 4128), (5, 8224),
                                 (2, 16384), (300, 2112), (1190, 160), (1203, 2112), (1185, 544), (1, 12288)])
@pytest.mark.parametrize("resid,y", [(B, None), (F, None), (B, B), (F, F), (B, F), (None, B)])
def test_norm_to_mxfp4_and_bf16(T, H, resid, y):
    p = require_gpu()
    kw = _make(T, H, T + H, resid, y)
    _check(p, T, H, True, False, **kw)
    _check(p, T, H, True, True, scale=0.6, **kw)
    _check(p, T, H, False, True, scale=-1.7, eps=1e-5, **kw)


@pytest.mark.parametrize("T,H", [(1, 8), (5, 24), (33, 1000), (2, 5000), (1300, 8), (1200, 1000)])
def test_widths_of_a_multiple_of_eight(T, H):
    p = require_gpu()
    _check(p, T, H, False, True, **_make(T, H, H, F, B, gate="row"))


@pytest.mark.parametrize("gate,dtype", list(itertools.product(["feature", "row", "full"], [B, F])))
@pytest.mark.parametrize("T", [70, 1200])
def test_gates(T, gate, dtype):
    p = require_gpu()
    kw = _make(T, 704, 5, B, B, gate=gate)
    kw["gate"] = kw["gate"].to(dtype)
    _check(p, T, 704, True, True, scale=0.5, **kw)
    n = kw["gate"].shape[-1]
    kw["gate"] = torch.cat([kw["gate"], kw["gate"]], -1)[..., :n]                             # strided rows
    _check(p, T, 704, True, True, scale=0.5, **kw)
    kw["gate"] = torch.cat([kw["gate"][..., :1], kw["gate"]], -1)[..., 1:]                    # no wide loads
    _check(p, T, 704, True, True, scale=0.5, **kw)


@pytest.mark.parametrize("post_norm", [True, False])
def test_post_norm_and_weights_apart(post_norm):
    p = require_gpu()
    kw = _make(40, 512, 6, F, F, post=False)
    _check(p, 40, 512, True, True, post_norm=post_norm, **kw)
    kw["post_weight"] = kw["norm_weight"]
    kw["norm_weight"] = None
    _check(p, 40, 512, True, True, post_norm=post_norm, **kw)


def test_many_rows_equal_codes():
    """Enough elements that fp32 alone would put some on the wrong side of a rounding border."""
    p = require_gpu()
    for resid, y, gate in [(B, None, ""), (F, B, "row")]:
        _check(p, 2000, 2816, True, False, **_make(2000, 2816, 11, resid, y, gate=gate))


@pytest.mark.parametrize("T", [12, 1300])
@pytest.mark.parametrize("dtype", [B, F])
def test_rows_that_cancel_vanish_or_overflow(T, dtype):
    """resid = -n up to rounding, zero rows, subnormal and huge rows, NaN and infinities: the float64 codes all the same."""
    p = require_gpu()
    H = 160
    kw = _make(T, H, 8, dtype, dtype)
    r, _ = mx.block_norm(None, None, float(np.float32(1e-6)), _n(kw["y"]), _n(kw["post_weight"]))
    kw["resid"][:4] = torch.from_numpy(-r[:4]).to(dtype).cuda()
    kw["resid"][4], kw["y"][4] = 0, 0
    kw["resid"][5] *= 1e-40
    kw["y"][5] *= 1e-42
    kw["resid"][6] *= 1e30
    kw["y"][7] *= 1e25
    kw["resid"][8, 3], kw["y"][9, 5], kw["resid"][10, 0] = float("nan"), float("inf"), float("-inf")
    kw["y"][11] = 0
    r, z, dr, dz = _want(kw)
    codes, scales = poisoned(T * H // 2).view(T, H // 2), poisoned(mx.scale_buffer_bytes(T, H))
    out = torch.empty(T, H, dtype=B, device="cuda")
    p.block_norm(codes=codes, scales=scales, out=out, resid_out=kw["resid"], **kw)            # in place
    ref = mx.quantize(z)
    byte, clean = mx.untile_scales(scales.cpu().numpy(), T, H)
    assert np.array_equal(byte, ref[1]) and clean and np.array_equal(codes.cpu().numpy(), ref[0])
    assert np.array_equal(np.isnan(_n(out)), np.isnan(z))
    whole = np.isfinite(r).all(1)                              # the other rows: infinities, and x / inf = 0, or NaN
    _near(out[torch.from_numpy(whole)], z[whole], dz[whole], B)
    _near(kw["resid"][torch.from_numpy(whole)], r[whole], dr[whole], dtype)
    assert np.array_equal(_n(out)[~whole], z[~whole], equal_nan=True)


@pytest.mark.parametrize("T", [6, 1300])
@pytest.mark.parametrize("scale", [1.0, 0.7, -1.3, 0.0, -0.0])
@pytest.mark.parametrize("resid,y", [(B, None), (F, None), (B, B), (F, F), (None, B)])
def test_signs_of_zeros(T, scale, resid, y):
    """Codes keep the sign of a zero: resid + y that cancels exactly, zeros of either sign, a scale that is not positive."""
    p = require_gpu()
    kw = _make(T, 160, 30, resid, y, post=False)
    for k in ("resid", "y"):
        if kw.get(k) is not None:
            kw[k][0], kw[k][1], kw[k][2, 3], kw[k][3, :40] = 0.0, -0.0, -0.0, -0.0
            kw[k][4, ::3] = -0.0 if k == "y" else 0.0
            kw[k][5, 32:96] = 0.0 if k == "y" else -0.0
    if resid and y:
        kw["y"][2, 8:48] = -kw["resid"][2, 8:48]
        kw["resid"][3, 64] = 2.0 ** -3
        kw["y"][3, 64] = -(2.0 ** -3)
    codes, scales = poisoned(T * 80).view(T, 80), poisoned(mx.scale_buffer_bytes(T, 160))
    p.block_norm(codes=codes, scales=scales, scale=scale, **kw)
    ref = mx.quantize(_want({**kw, "scale": scale})[1])
    byte, _ = mx.untile_scales(scales.cpu().numpy(), T, 160)
    assert np.array_equal(byte, ref[1])
    bad = np.argwhere(codes.cpu().numpy() != ref[0])
    assert len(bad) == 0, bad[:6].tolist()


@pytest.mark.parametrize("T", [12, 1300])
def test_weights_that_are_not_finite(T):
    """A NaN or infinite weight of the second norm spoils exactly its block of every row."""
    p = require_gpu()
    for kind in (None, B):
        kw = _make(T, 160, 13, B, kind)
        clean = p.block_norm(mx=True, **kw)
        for bad in (float("nan"), float("inf")):
            kw["norm_weight"][70] = bad
            got = p.block_norm(mx=True, **kw)
            byte, _ = mx.untile_scales(got.scales.cpu().numpy(), T, 160)
            want, _ = mx.untile_scales(clean.scales.cpu().numpy(), T, 160)
            want[:, 2] = 255
            assert np.array_equal(byte, want)
            keep = [i for i in range(80) if not 32 <= i < 48]
            assert torch.equal(got.codes[:, keep], clean.codes[:, keep]) and not got.codes[:, 32:48].any()
            kw["norm_weight"][70] = 1.0
            clean = p.block_norm(mx=True, **kw)


def test_zero_eps_and_zero_rows():
    p = require_gpu()
    x = torch.zeros(3, 64, dtype=B, device="cuda")
    x[1] = 2.0 ** -100
    got = p.block_norm(x, eps=0.0, mx=True)
    v = _n(p.mx_dequantize(got.codes, got.scales))
    assert np.isnan(v[[0, 2]]).all() and (v[1] == 1.0).all()


def test_in_place_strided_and_defaults():
    p = require_gpu()
    base = _make(50, 512, 9, B, B)
    r, z, dr, dz = _want(base)
    wide = torch.full((50, 1024), 3.0, dtype=B, device="cuda")
    wide[:, :512], wide[:, 512:] = base["resid"], base["y"]
    kw = {**base, "resid": wide[:, :512], "y": wide[:, 512:]}
    got = p.block_norm(resid_out=kw["resid"], out=kw["y"], **kw)                              # r on resid, z on y
    _near(got.resid, r, dr, B)
    _near(got.out, z, dz, B)
    only_r = p.block_norm(base["resid"], y=base["y"], post_weight=base["post_weight"])
    assert only_r.out is None and torch.equal(only_r.resid, got.resid)
    only_z = p.block_norm(**base)
    assert only_z.resid is None and torch.equal(only_z.out, got.out)


@pytest.mark.parametrize("T", [50, 1300])
@pytest.mark.parametrize("dtype", [B, F])
def test_in_place_equals_apart(T, dtype):
    """Outputs on the inputs, and beside them in one buffer, give the bits that separate ones do."""
    p = require_gpu()
    base = _make(T, 512, 12, dtype, B, gate="row")
    new = lambda t: torch.empty_like(t)  # noqa: E731
    for mx_too in (False, True):
        want = p.block_norm(**base, resid_out=new(base["resid"]), out=new(base["y"]), mx=mx_too)
        kw = {**base, "resid": base["resid"].clone(), "y": base["y"].clone()}
        got = p.block_norm(**kw, resid_out=kw["resid"], out=kw["y"], mx=mx_too)
        assert torch.equal(got.resid, want.resid) and torch.equal(got.out, want.out)
        if mx_too:
            assert torch.equal(got.codes, want.codes) and torch.equal(got.scales, want.scales)
    wide = torch.empty(T, 1024, dtype=dtype, device="cuda")
    wide[:, 512:] = base["resid"]
    got = p.block_norm(**{**base, "resid": wide[:, 512:]}, resid_out=wide[:, :512], mx=True)
    assert torch.equal(got.resid, want.resid) and torch.equal(got.codes, want.codes)
    assert torch.equal(wide[:, 512:], base["resid"])
    with pytest.raises(p.NvFp4Error, match="ARG"):
        p.block_norm(wide[1:, :512], base["norm_weight"], resid_out=wide[:-1, :512])


def test_two_streams_at_once():
    p = require_gpu()
    for T in (3, 1300):
        kw = [_make(T, 2816, 20 + i, F, B, gate="row") for i in range(2)]
        want = [p.block_norm(mx=True, **k) for k in kw]
        torch.cuda.synchronize()
        streams = [torch.cuda.Stream() for _ in kw]
        got = [[p.block_norm(mx=True, stream=s, **k) for _ in range(8)] for k, s in zip(kw, streams)]
        torch.cuda.synchronize()
        for gs, w in zip(got, want):
            assert all(torch.equal(g.codes, w.codes) and torch.equal(g.scales, w.scales) for g in gs)


def test_amax_feeds_the_nvfp4_quantiser():
    p = require_gpu()
    kw = _make(200, 704, 10, F, F)
    out, amax = torch.empty(200, 704, dtype=B, device="cuda"), torch.empty(1, device="cuda")
    p.block_norm(out=out, amax=amax, **kw)
    assert torch.equal(amax, p.amax(out))
    a, b = p.quantize(out, amax_dev=amax), p.quantize(out, amax_dev=p.amax(out))
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


def test_captured_block():
    """Two layers of a dense MXFP4 feed-forward as they are used -- norm, product, gate, product, norm -- captured into one
    graph, replayed on new rows, against float64 with the device's codes taken as the operands."""
    p = require_gpu()
    T, H, I = 48, 704, 2112
    g = torch.Generator("cuda").manual_seed(3)
    rn = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    x, w = rn(T, H), [(1 + 0.1 * rn(H)).bfloat16() for _ in range(3)]
    gu, dn = p.mx_quantize(0.04 * rn(2 * I, H)), p.mx_quantize(0.03 * rn(H, I))

    def step():
        first = p.block_norm(x, w[0], mx=True)
        up = p.mx_gemm(first.codes, first.scales, *gu)
        h = p.mx_geglu_quantize(up)
        y = p.mx_gemm(*h, *dn)
        return first, up, h, y, p.block_norm(x, w[2], y=y, post_weight=w[1], scale=0.9,
                                             resid_out=torch.empty_like(x), mx=True)

    step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        first, up, h, y, last = step()
    for seed in range(2):
        x.copy_(rn(T, H))
        graph.replay()
        torch.cuda.synchronize()
        v = lambda c: _n(p.mx_dequantize(*c, dtype=torch.float32))  # noqa: E731
        _, z = mx.block_norm(_n(x), _n(w[0]), float(np.float32(1e-6)))
        assert np.array_equal(v(first[3:]), mx.dequantize(*mx.quantize(z)))
        for got, a, b in ((up, first[3:], gu), (y, h, dn)):
            a, b = v(a), v(b)
            s = np.abs(a) @ np.abs(b).T
            assert (np.abs(_n(got) - a @ b.T) <= 2.0 ** -8 * np.abs(a @ b.T) + 2.0 ** -17 * s).all()
        assert np.array_equal(v(h), mx.dequantize(*mx.quantize(mx.geglu(_n(up)[:, :I], _n(up)[:, I:]))))
        r, z = mx.block_norm(_n(x), _n(w[2]), float(np.float32(1e-6)), _n(y), _n(w[1]), scale=float(np.float32(0.9)))
        assert np.array_equal(v(last[3:]), mx.dequantize(*mx.quantize(z)))
        assert np.abs(_n(last.resid) - r).max() <= 1e-5


def test_refusals():
    p = require_gpu()
    x = torch.zeros(4, 64, device="cuda")
    w = torch.ones(64, dtype=B, device="cuda")
    for match, kw in [("resid or y", {}), ("need y", dict(resid=x, post_weight=w)), ("need y", dict(resid=x, gate=w)),
                      ("dtype", dict(resid=x.half(), norm_weight=w)), ("norm_weight", dict(resid=x, norm_weight=w.float())),
                      ("norm_weight", dict(resid=x, norm_weight=w[:32])), ("shape", dict(resid=x, y=x[:2])),
                      ("gate", dict(resid=x, y=x, gate=torch.ones(4, device="cuda"))),
                      ("contiguous", dict(resid=x, y=x, gate=torch.ones(128, device="cuda")[::2])),
                      ("amax", dict(resid=x, mx=True, amax=torch.empty(1, device="cuda"))),
                      ("type or pitch", dict(resid=x, y=x, resid_out=x.view(B)[:, :64])),
                      ("multiple of 32", dict(resid=x[:, :40].contiguous(), mx=True)),
                      ("cuda", dict(resid=x, norm_weight=w.cpu()))]:
        with pytest.raises(ValueError, match=match):
            p.block_norm(**kw)
    with pytest.raises(p.NvFp4Error, match="NULL"):
        p.block_norm(x)
    with pytest.raises(p.NvFp4Error, match="SHAPE"):
        p.block_norm(torch.zeros(1, 16392, device="cuda"), resid_out=torch.zeros(1, 16392, device="cuda"))
    with pytest.raises(p.NvFp4Error, match="ALIGN"):
        p.block_norm(torch.zeros(4, 66, device="cuda")[:, :64], w)
    with pytest.raises(p.NvFp4Error, match="ARG"):
        p.block_norm(x, w, eps=-1.0)


@pytest.mark.parametrize("T", [12, 1300])
@pytest.mark.parametrize("resid,y", [(B, None), (F, None), (B, B), (F, F), (None, B)])
def test_weight_times_reciprocal_rms_beyond_fp32(T, resid, y):
    """Small rows under large weights: w / rms leaves fp32, w (x / rms) does not -- codes, out and resid_out."""
    p = require_gpu()
    H = 160
    kw = _make(T, H, 21, resid, y)
    for k in ("resid", "y"):
        if kw.get(k) is not None:
            kw[k] *= 2.0 ** -14
            kw[k][:, 5:40:3], kw[k][2], kw[k][:, 64:96] = 0.0, 0.0, 0.0
    kw["norm_weight"][::2] = 2.0 ** 121                       # 1 / rms is up to 2^10 (eps), z below 2^127
    _check(p, T, H, True, True, **kw)
    _check(p, T, H, True, False, **kw)
    _check(p, T, H, False, True, **kw)
    if y:
        kw["post_weight"] = kw["norm_weight"]
        kw["norm_weight"] = None
        r, _, dr, _ = _want(kw)
        out = torch.empty(T, H, dtype=F, device="cuda")
        p.block_norm(**kw, resid_out=out)
        _near(out, r, dr, F)
        _check(p, T, H, True, True, **kw)


def _borders(shape, size, seed):
    """fp32 values within three steps of the rounding borders of an MXFP4 block whose largest is 4.5 (each block has one),
    times `size`, a power of two; either sign."""
    rng = np.random.default_rng(seed)
    x = rng.choice(np.array([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0], np.float32), shape)
    x = (x.view(np.int32) + rng.integers(-3, 4, shape, dtype=np.int32)).view(np.float32)
    x.reshape(-1, 32)[:, 9] = 4.5
    return torch.from_numpy(x * rng.choice(np.array([-1, 1], np.float32), shape) * np.float32(size)).cuda()


@pytest.mark.parametrize("T", [12, 739, 800])
@pytest.mark.parametrize("eps", [2.0 ** -20, 2.0 ** -60])
@pytest.mark.parametrize("e", [-60, -70, -74, -78, -85, -100, -110, -125])
def test_rows_whose_squares_underflow(T, eps, e):
    """Rows so far below eps that the norms only multiply by 1 / sqrt(eps), near the rounding borders of their codes."""
    p = require_gpu()
    H = 160
    r, one = _borders((T, H), 2.0 ** e, T - e), torch.ones(H, dtype=B, device="cuda")
    for scale in (1.0, 0.7, 2.0 ** 30):
        x = r * (1 / scale)                                   # 0.7: near the borders, seldom on one
        for kw in (dict(resid=x), dict(y=x), dict(y=x, post_weight=one), dict(resid=x, y=x), dict(resid=0.25 * x, y=0.5 * x),
                   dict(resid=-x, y=2.0 * x), dict(resid=x, y=x, gate=torch.full((T, 1), 0.5, device="cuda"))):
            _check(p, T, H, True, False, eps=eps, scale=scale, **kw)


@pytest.mark.parametrize("T", [12, 1300])
@pytest.mark.parametrize("y_exp,w_exp", [(-30, -108), (-30, -112), (-60, -84), (0, -126), (20, -126), (-10, -133)])
def test_products_of_input_and_weight_that_underflow(T, y_exp, w_exp):
    """A block whose y post_weight needs bits below the smallest fp32, brought back by the second weights."""
    p = require_gpu()
    for resid in (None, B, F):
        kw = _make(T, 256, 24, resid, B)
        kw["y"][:, 224:] *= 2.0 ** y_exp
        kw["post_weight"][224:] *= 2.0 ** w_exp
        kw["norm_weight"][224:] *= 2.0 ** 45
        if resid:
            kw["resid"][:, 224:] = 0
        _check(p, T, 256, True, False, **kw)
        _check(p, T, 256, True, False, eps=1e-30, gate=torch.rand(T, 1, device="cuda"), **kw)
        _check(p, T, 256, True, False, gate=torch.rand(256, device="cuda"), **kw)


@pytest.mark.parametrize("T", [12, 1300])
def test_products_that_underflow(T):
    """Blocks whose second weights, gates or inputs lie many powers of two below the row's."""
    p = require_gpu()
    H = 256
    for resid, y, gate in [(F, None, ""), (B, None, ""), (F, F, "feature"), (B, B, "row"), (None, F, "feature")]:
        kw = _make(T, H, 23, resid, y, gate=gate)
        kw["norm_weight"][32:64] *= 2.0 ** -70
        kw["norm_weight"][64:96] *= 2.0 ** -120
        for k in ("resid", "y"):
            if kw.get(k) is not None:
                kw[k][:, 96:128] *= 2.0 ** -80
                kw[k][:, 128:160] *= 2.0 ** -126
                kw[k][3] *= 2.0 ** 45
                kw[k][5] *= 2.0 ** 60
        if gate == "feature":
            kw["gate"][160:192] *= 2.0 ** -100
            kw["gate"][192:224] *= 2.0 ** -140
        if gate == "row":
            kw["gate"][6], kw["gate"][7] = 2.0 ** -100, 2.0 ** -130
        if y:
            kw["post_weight"][224:240] *= 2.0 ** -110
        _check(p, T, H, True, False, **kw)
        _check(p, T, H, True, False, eps=0.0, **kw)


@pytest.mark.parametrize("T", [20, 1300])
@pytest.mark.parametrize("H", [64, 256, 1024, 4096])
@pytest.mark.parametrize("dtype", [B, F])
def test_rows_of_one_element(T, H, dtype):
    """A lone element has z = sqrt(H) w, a power of two that the scale byte turns on, whatever its size and the roundings."""
    p = require_gpu()
    rng = np.random.default_rng(H)
    x = torch.zeros(T, H, dtype=dtype, device="cuda")
    at = torch.from_numpy(rng.integers(0, H, T)).cuda()
    x[torch.arange(T), at] = torch.from_numpy(rng.normal(0, 1, T) * 2.0 ** rng.integers(-40, 40, T)).to(dtype).cuda()
    w = torch.full((H,), 1.0, dtype=B, device="cuda")
    for kw in (dict(resid=x), dict(y=x, post_norm=False), dict(y=x, post_norm=True), dict(y=x, post_weight=w, norm_weight=w),
               dict(resid=x, y=x, post_norm=False), dict(resid=x, y=x, post_norm=True)):
        got = p.block_norm(**kw, eps=0.0, mx=True)
        z = torch.where(x != 0, torch.sign(x.double()) * H ** 0.5, 0.0)
        ref = mx.quantize(_n(z))
        byte, _ = mx.untile_scales(got.scales.cpu().numpy(), T, H)
        assert np.array_equal(byte, ref[1]) and np.array_equal(got.codes.cpu().numpy(), ref[0])


@pytest.mark.parametrize("T", [12, 1300])
@pytest.mark.parametrize("resid", [None, F])
@pytest.mark.parametrize("dtype", [B, F])
def test_gate_over_rms_that_underflows(T, resid, dtype):
    """gate / rms(y) below fp32 while gate * n is not."""
    p = require_gpu()
    for g_exp, scale in [(-110, 1.0), (-85, 1.0), (-85, 2.0 ** -30), (-60, 2.0 ** -60)]:
        kw = _make(T, 256, 25, resid, dtype, gate="row")
        kw["y"] *= 2.0 ** 45
        kw["gate"] *= 2.0 ** g_exp
        if resid:
            kw["resid"][:, 32:96], kw["resid"][::2] = 0.0, 0.0
        for mx_too, out_too in [(True, False), (True, True), (False, True)]:
            _check(p, T, 256, mx_too, out_too, scale=scale, **kw)


@pytest.mark.parametrize("T", [12, 1300])
@pytest.mark.parametrize("resid", [None, F])
def test_inputs_that_underflow_before_the_weight(T, resid):
    """y / rms(y) below fp32 where the post weight or a gate brings it back: the codes."""
    p = require_gpu()
    H = 256
    for gate, w_exp, g_exp in [("", 40, 0), ("row", 40, 0), ("feature", 20, 20), ("full", 20, 20), ("feature", 0, 40)]:
        kw = _make(T, H, 26, resid, B, gate=gate)
        kw["y"] *= 2.0 ** 30
        kw["y"][:, 32:64] *= 2.0 ** -100
        kw["y"][:, 32:64] *= 2.0 ** -55                            # 2^-125, and 2^-155 after the norm
        kw["post_weight"][32:64] *= 2.0 ** w_exp
        if g_exp:
            kw["gate"][..., 32:64] *= 2.0 ** g_exp
        if resid:
            kw["resid"][:, 32:64] = 0.0
        codes, scales = poisoned(T * H // 2).view(T, H // 2), poisoned(mx.scale_buffer_bytes(T, H))
        p.block_norm(codes=codes, scales=scales, **kw)
        ref = mx.quantize(_want(kw)[1])
        byte, clean = mx.untile_scales(scales.cpu().numpy(), T, H)
        assert np.array_equal(byte, ref[1]) and clean and np.array_equal(codes.cpu().numpy(), ref[0])
