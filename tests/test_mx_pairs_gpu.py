"""The CTA-pair tiles of the MXFP4 GEMM against the float64 product of the operands' values.

Which kernel a call takes goes by its rounds of tiles; the rule is restated here and every size is asserted to take pairs, so that
a change of it cannot leave these tests to the narrow tiles.  Tolerance as in test_mx_gemm_gpu.py."""
import pytest
import torch

import mx_oracle as mx
from gpu_util import require_gpu
from test_mx_gemm_gpu import KINDS, _dev, _operand

pytestmark = pytest.mark.gpu

# one and several tiles per pair, one 256-row tile only either way, last tiles of one row or column, K in odd halves of a step
SIZES = [(1281, 2001, 160), (1000, 5000, 2848), (2048, 2048, 704), (129, 18817, 544), (18817, 129, 544), (4200, 7001, 800)]


def _assert_pairs(m, n, k):
    sms, kt = torch.cuda.get_device_properties(0).multi_processor_count, -(-k // 256)
    narrow = -(-(-(-m // 128) * -(-n // 128)) // sms)
    pairs = -(-(-(-m // 256) * -(-n // 256)) // (sms // 2))
    assert m > 128 and n > 128 and narrow * (2 + 2 * kt if kt > 2 else 6) > pairs * (9 + 2 * kt), "this size takes narrow tiles"


def _product(a, b, k, alpha):
    """alpha A B^T in float64 and the bound on fp32 accumulation."""
    v = [torch.from_numpy(mx.dequantize(*x)).cuda() for x in (a, b)]
    return alpha * v[0] @ v[1].T, 2.0 * (-(-k // 64) + 9) * 2.0 ** -23 * abs(alpha) * (v[0].abs() @ v[1].abs().T)


def _buffer(kind, m, n, pad):
    r, c = (n, m) if kind == "f32_col" else (m, n)
    wide = torch.full((r, c + pad), 5.0, dtype=torch.bfloat16 if kind == "bf16" else torch.float32, device="cuda")
    return wide, wide[:, :c]


@pytest.mark.parametrize("m,n,k", SIZES)
def test_products_alpha_and_pitch(m, n, k):
    p = require_gpu()
    _assert_pairs(m, n, k)
    a, b = _operand(m, k, m + k), _operand(n, k, n + k + 1)
    A, B = _dev(*a, k), _dev(*b, k)
    for alpha, pad in [(1.0, 0), (-0.375, 1), (3.0, 8)]:
        ref, tol = _product(a, b, k, alpha)
        for kind in KINDS:
            wide, out = _buffer(kind, m, n, pad)
            assert p.mx_gemm(*A, *B, out=out, out_kind=KINDS.index(kind), alpha=alpha) is out
            got = out.double().T if kind == "f32_col" else out.double()
            half = 2.0 ** -8 if kind == "bf16" else 2.0 ** -24
            bad = ~((got - ref).abs() <= half * ref.abs() + tol)
            assert not bad.any(), (kind, alpha, pad, int(bad.sum()), bad.nonzero()[:4].tolist())
            assert (wide[:, out.shape[1]:] == 5.0).all()
    assert p.read_device_error() == 0


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("m,n,k", [(1281, 2001, 160), (2048, 2048, 704), (1000, 5000, 2848)])
def test_same_bits_every_time(m, n, k, kind):
    """Calls and graph replays on one stream and two streams at once give the same bits."""
    p = require_gpu()
    _assert_pairs(m, n, k)
    A, B = _dev(*_operand(m, k, 7), k), _dev(*_operand(n, k, 8), k)
    call = lambda out=None, stream=None: p.mx_gemm(*A, *B, out=out, out_kind=KINDS.index(kind), stream=stream)  # noqa: E731
    one = call()
    assert all(torch.equal(one, call()) for _ in range(3))
    graph, out = torch.cuda.CUDAGraph(), torch.empty_like(one)
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        call(out)
    for _ in range(2):
        out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, one)
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [call(stream=s) for _ in range(4) for s in streams]
    torch.cuda.synchronize()
    assert all(torch.equal(g, one) for g in got)
    assert p.read_device_error() == 0


@pytest.mark.parametrize("m,n,k", [(2048, 2048, 704), (129, 18817, 544)])
def test_nan_scale_stays_in_its_row_and_column(m, n, k):
    p = require_gpu()
    _assert_pairs(m, n, k)
    a, b = _operand(m, k, 5), _operand(n, k, 6)
    got = p.mx_gemm(*_dev(*a, k), *_dev(*b, k), out_kind=p.OUT_F32_ROWMAJOR)
    a[1][m - 1, -1], b[1][n // 2, 0] = 255, 255
    nan = p.mx_gemm(*_dev(*a, k), *_dev(*b, k), out_kind=p.OUT_F32_ROWMAJOR)
    hit = torch.zeros(m, n, dtype=torch.bool, device="cuda")
    hit[m - 1], hit[:, n // 2] = True, True
    assert torch.isnan(nan[hit]).all() and torch.equal(nan[~hit], got[~hit])
