"""MXFP4 quantisers and the dequantiser on the GPU against the float64 oracle: codes, scale bytes and values are equal
bit for bit, padding included."""
import numpy as np
import pytest
import torch

import mx_oracle as mx
import nvfp4_oracle as orc
from gpu_util import bf16_to_dev, poisoned, require_gpu

pytestmark = pytest.mark.gpu

SHAPES = [(1, 32), (1, 2816), (3, 96), (33, 160), (127, 2848), (128, 128), (129, 4096), (200, 2112), (300, 704),
          (5, 16384)]


def _check(codes, scales, want, rows, k):
    byte, clean = mx.untile_scales(scales.cpu().numpy(), rows, k)
    assert np.array_equal(byte, want[1])
    assert clean, "padding bytes must be written as zero"
    assert np.array_equal(codes.cpu().numpy(), want[0])


def _run(fn, x, rows, k):
    codes, scales = poisoned(rows * k // 2).view(rows, k // 2), poisoned(mx.scale_buffer_bytes(rows, k))
    got = fn(x, codes=codes, scales=scales)
    assert got[0] is codes and got[1] is scales
    return codes, scales


@pytest.mark.parametrize("rows,k", SHAPES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_quantize_bit_exact(rows, k, dtype):
    p = require_gpu()
    bits = orc.synth_bf16((rows, k), 1.0, seed=rows + k, outlier_frac=0.002)
    x = bf16_to_dev(bits).to(dtype)
    if dtype == torch.float32:
        x = x * 1.2345678
    _check(*_run(p.mx_quantize, x, rows, k), mx.quantize(x.double().cpu().numpy()), rows, k)


def _edge_rows():
    """Blocks on and next to every rounding border under many exponents, subnormals, zeros, signed zeros, NaN, infinities."""
    rng = np.random.default_rng(5)
    rows = []
    mids = np.array([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0, 7.5], np.float32)
    for e in list(range(-126, 126, 9)) + [125]:
        s = np.float32(2.0) ** np.float32(e)
        t = (mids * s).astype(np.float32)
        b = np.concatenate([t, np.nextafter(t, np.float32(0)), np.nextafter(t, np.float32(3e38))])[:31]
        b = np.concatenate([np.minimum(b, np.float32(7.75) * s), [np.float32(4.5) * s] * 5])[:32]
        rows.append(b.astype(np.float32) * rng.choice([-1, 1], 32))
    tiny = np.float32(1e-45)
    rows += [np.zeros(32), np.full(32, -0.0), np.full(32, tiny), np.arange(32) * tiny, np.full(32, 2.0 ** -127),
             np.full(32, 3.3e38), np.where(np.arange(32) == 7, np.nan, 1.0), np.where(np.arange(32) == 31, np.inf, 1.0),
             np.where(np.arange(32) == 0, -np.inf, 0.0), np.where(np.arange(32) < 31, -1e-30, 1.0)]
    return np.array(rows, np.float32)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_quantize_borders_and_special_values(dtype):
    p = require_gpu()
    x = torch.from_numpy(_edge_rows()).to(dtype)
    rows = x.shape[0]
    want = mx.quantize(x.double().numpy())
    assert 255 in want[1] and 0 in want[1]
    codes, scales = _run(p.mx_quantize, x.cuda(), rows, 32)
    _check(codes, scales, want, rows, 32)
    for dt in (torch.bfloat16, torch.float32):
        got = p.mx_dequantize(codes, scales, dtype=dt).double().cpu().numpy()
        assert np.array_equal(got, mx.dequantize(*want), equal_nan=True)


@pytest.mark.parametrize("rows,k", [(1, 32), (129, 160), (40, 2816)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_dequantize_every_code_and_scale(rows, k, dtype):
    p = require_gpu()
    rng = np.random.default_rng(rows)
    codes = rng.integers(0, 256, (rows, k // 2), dtype=np.uint8)
    byte = rng.integers(0, 253, (rows, k // 32), dtype=np.uint8)
    byte.reshape(-1)[:1] = 255
    wide = torch.full((rows, k + 16), 7.0, dtype=dtype, device="cuda")        # strided output: the rest stays
    got = p.mx_dequantize(torch.from_numpy(codes).cuda(), torch.from_numpy(mx.tile_scales(byte, k)).cuda(),
                          out=wide[:, :k])
    assert np.array_equal(got.double().cpu().numpy(), mx.dequantize(codes, byte), equal_nan=True)
    assert (wide[:, k:] == 7.0).all()


def test_swizzle_matches_oracle():
    p = require_gpu()
    rng = np.random.default_rng(2)
    for rows, k in [(1, 32), (130, 416), (2816, 2112)]:
        byte = rng.integers(0, 256, (rows, k // 32), dtype=np.uint8)
        got = p.mx_swizzle_scales(torch.from_numpy(byte).cuda(), rows, k)
        assert np.array_equal(got.cpu().numpy(), mx.tile_scales(byte, k))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_quantize_strided_rows(dtype):
    p = require_gpu()
    base = torch.randn(70, 512, generator=torch.Generator().manual_seed(1)).to(dtype).cuda()
    x = base[:, 64:64 + 224]
    _check(*_run(p.mx_quantize, x, 70, 224), mx.quantize(x.double().cpu().numpy()), 70, 224)


@pytest.mark.parametrize("rows,i", [(1, 2112), (1, 32), (130, 96), (257, 704), (64, 2848)])
@pytest.mark.parametrize("std", [0.3, 1.5, 6.0])
def test_geglu_codes_of_the_float64_value(rows, i, std):
    p = require_gpu()
    g = orc.synth_bf16((rows, i), std, seed=rows + i)
    u = orc.synth_bf16((rows, i), 1.0, seed=rows + i + 1, outlier_frac=0.01)
    x = torch.cat([bf16_to_dev(g), bf16_to_dev(u)], 1)
    want = mx.quantize(mx.geglu(orc.bf16_bits_to_f32(g), orc.bf16_bits_to_f32(u)))
    _check(*_run(p.mx_geglu_quantize, x, rows, i), want, rows, i)


def test_geglu_extreme_values():
    """Zero blocks, gates deep in the negative tail, products near both ends of the range, NaN and infinities."""
    p = require_gpu()
    n = np.arange(32)
    rows = [(0 * n, n), (n, 0 * n), (-6.0 - 0.1 * n, 1.0 + 0 * n), (-12.0 - n, 1e30 + 0 * n), (-9.0 - 0.25 * n, n - 16),
            (1e30 + 0 * n, 1e30 + 0 * n), (1e19 + 0 * n, 1e19 * (n + 1)), (1e-38 * n, 1e-3 * n), (-1e30 + 0 * n, n),
            (np.where(n == 3, -20.0, 1.0), np.where(n == 3, 1e38, 1.0)),
            (np.where(n == 3, np.nan, 1.0), n), (np.where(n == 3, -np.inf, 1.0), n), (np.where(n == 9, np.inf, 1.0), n),
            (n - 16.0, np.where(n == 30, -np.inf, 1.0)), (-0.0 * n, -n), (-2.0 ** -100 * n, 2.0 ** -20 + 0 * n),
            (-30.0 + 0 * n, 1.0 + n), (-1.0 * n, 2.0 ** -120 * n)]
    x = torch.tensor(np.array([np.concatenate([g, u]) for g, u in rows]), dtype=torch.float64).to(torch.bfloat16)
    v = x.double().numpy()
    want = mx.quantize(mx.geglu(v[:, :32], v[:, 32:]))
    _check(*_run(p.mx_geglu_quantize, x.cuda(), len(rows), 32), want, len(rows), 32)


def test_graph_replay_and_side_stream():
    """Captured on a side stream and replayed on new contents; outputs allocated by the call on that stream."""
    p = require_gpu()
    x = torch.randn(96, 704, device="cuda").bfloat16()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    codes, scales = p.mx_quantize(x, stream=s)
    s.synchronize()
    _check(codes, scales, mx.quantize(x.double().cpu().numpy()), 96, 704)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        c2, s2 = p.mx_quantize(x, codes=codes, scales=scales)
        v = p.mx_dequantize(c2, s2, dtype=torch.float32)
    for _ in range(2):
        x.copy_(torch.randn(96, 704, device="cuda").bfloat16())
        graph.replay()
        torch.cuda.synchronize()
        want = mx.quantize(x.double().cpu().numpy())
        _check(codes, scales, want, 96, 704)
        assert np.array_equal(v.double().cpu().numpy(), mx.dequantize(*want))


@pytest.mark.parametrize("gate", [-3e12, -1.5e13, -2e13, -1e19, -1e20, -1e38, -3.3895313892515355e38, 1e19, 1e38])
def test_geglu_gates_beyond_the_fp32_cube(gate):
    """Gates whose cube leaves fp32, among ordinary ones: h is a signed zero (or g u), whatever the up value beside it."""
    p = require_gpu()
    rng = np.random.default_rng(1)
    rows = []
    for u in (1.0, -1.0, 0.0, -0.0, 1e-20, -1e30, 3e38):
        for at in ([3], [0, 31], list(range(16)), list(range(16, 32)), list(range(0, 32, 2))):
            for g0, u0 in ((np.ones(32), np.arange(32.0)), (rng.normal(0, 1.5, 32), rng.normal(0, 1, 32)),
                           (np.full(32, -9.0), np.ones(32)), (np.full(32, 1e-30), np.ones(32)), (np.zeros(32), np.ones(32))):
                g1, u1 = g0.copy(), u0.copy()
                g1[at], u1[at] = gate, u
                rows.append((g1, u1))
    n = len(rows)                                              # one block each, all of them in the rows of one call
    g, u = (torch.tensor(np.array([r[i] for r in rows])).to(torch.bfloat16) for i in range(2))
    want = mx.quantize(mx.geglu(g.double().numpy(), u.double().numpy()))
    _check(*_run(p.mx_geglu_quantize, torch.cat([g, u], 1).cuda(), n, 32), want, n, 32)
    wide = [t.view(5, -1) for t in (g, u)]                     # and side by side: the other threads of the warp
    k = wide[0].shape[1]
    want = mx.quantize(mx.geglu(wide[0].double().numpy(), wide[1].double().numpy()))
    _check(*_run(p.mx_geglu_quantize, torch.cat(wide, 1).cuda(), 5, k), want, 5, k)


def test_geglu_masked_gates():
    """A padded batch: gates of the type's lowest value wherever a token or a feature is masked."""
    p = require_gpu()
    g = torch.Generator().manual_seed(4)
    gate, up = (torch.randn(150, 704, generator=g).bfloat16() for _ in range(2))
    gate[100:] = torch.finfo(torch.bfloat16).min
    gate[:, 650:] = torch.finfo(torch.bfloat16).min
    gate[::7, ::5] = torch.finfo(torch.bfloat16).min
    want = mx.quantize(mx.geglu(gate.double().numpy(), up.double().numpy()))
    _check(*_run(p.mx_geglu_quantize, torch.cat([gate, up], 1).cuda(), 150, 704), want, 150, 704)


def test_geglu_signed_zeros():
    """Zeros of either sign among ordinary values, in gate, up or both, and whole rows of them: the sign of h on a code of zero."""
    p = require_gpu()
    g = torch.Generator().manual_seed(6)
    gate, up = ((1.5 * torch.randn(200, 704, generator=g)).bfloat16() for _ in range(2))
    for t, s in ((gate, 0), (up, 1)):
        r = torch.rand(200, 704, generator=g)
        t[r < 0.05], t[(r > 0.05) & (r < 0.1)] = 0.0, -0.0
        t[190 + s], t[193 + s], t[196:, s::2] = 0.0, -0.0, 0.0
    gate[180:184], up[180:184] = 0.0, 0.0
    want = mx.quantize(mx.geglu(gate.double().numpy(), up.double().numpy()))
    _check(*_run(p.mx_geglu_quantize, torch.cat([gate, up], 1).cuda(), 200, 704), want, 200, 704)
