"""CPU checks of the MXFP4 operators: the oracle against the format's definition, and every refusal that is made before
the device is touched."""
import numpy as np
import pytest
import torch

import mx_oracle as mx
from __graft_entry__ import load_package


def test_oracle_rounds_to_nearest_even_codes():
    # e = 0 throughout: the block maximum is 4
    x = np.zeros((1, 32))
    x[0, :12] = [4.0, 0.25, 0.75, 1.25, 1.75, 2.5, 3.5, -0.25, -0.2500001, 0.7499999, -3.5000001, -0.0]
    codes, byte = mx.quantize(x)
    assert byte.tolist() == [[127]]
    assert mx.dequantize(codes, byte)[0, :12].tolist() == [4, 0, 1, 1, 2, 2, 4, 0, -0.5, 0.5, -4, 0]
    nib = np.stack([codes & 15, codes >> 4], -1).reshape(1, 32)
    assert nib[0, 7] == 8 and nib[0, 11] == 8                 # the sign is kept on zeros


def test_oracle_scale_bytes():
    x = np.zeros((6, 32))
    x[0, 3] = 7.999
    x[1, 3] = 2.0 ** -140
    x[2, 3] = 2.0 ** 127
    x[3, 3] = 2.0 ** 128
    x[4, 3] = np.nan
    _, byte = mx.quantize(x)
    assert byte[:, 0].tolist() == [127, 0, 252, 255, 255, 0]
    codes, byte = mx.quantize(x[:1])
    assert mx.dequantize(codes, byte)[0, 3] == 6.0            # saturated


def test_oracle_error_of_a_block_is_bounded():
    x = np.random.default_rng(0).standard_normal((64, 256))
    v = mx.dequantize(*mx.quantize(x))
    amax = np.abs(x.reshape(64, -1, 32)).max(2).repeat(32, 1)
    # half the widest step of the grid is 1, and saturation loses less than 2, of a block maximum of at least 4
    assert (np.abs(v - x) <= amax / 2).all()


def test_scale_buffer_bytes():
    p = load_package()
    for rows, k in [(1, 32), (128, 128), (129, 160), (8192, 2816), (0, 32), (4, 0)]:
        want = mx.scale_buffer_bytes(rows, k) if rows and k else 0
        assert p.mx_scale_buffer_bytes(rows, k) == want == p._mx_sigs().nvfp4b_mx_scale_buffer_bytes(rows, k)


def test_c_refusals():
    L = load_package()._mx_sigs()
    q, g, dq, mm = (L.nvfp4b_mx_quantize_bf16, L.nvfp4b_mx_geglu_quantize, L.nvfp4b_mx_dequantize, L.nvfp4b_mx_gemm)
    assert q(None, 64, 4, 64, 16, 16, None) == -3
    assert q(16, 64, 0, 64, 16, 16, None) == -1               # no rows
    assert q(16, 48, 4, 48, 16, 16, None) == -1               # K % 32
    assert q(16, 32, 4, 64, 16, 16, None) == -1               # pitch below the width
    assert q(8, 64, 4, 64, 16, 16, None) == -2
    assert q(16, 68, 4, 64, 16, 16, None) == -2               # pitch not a multiple of 16 bytes
    assert L.nvfp4b_mx_quantize_f32(16, 66, 4, 64, 16, 16, None) == -2
    assert g(16, 64, 4, 64, 16, 16, None) == -1               # pitch below 2 I
    assert g(16, 128, 4, 0, 16, 16, None) == -1
    assert g(16, 128, 4, 64, 16, None, None) == -3
    assert dq(16, 16, 4, 64, 16, 2, 64, None) == -7
    assert dq(16, 16, 4, 64, 8, 0, 64, None) == -2
    assert dq(16, 16, 4, 64, 16, 1, 62, None) == -1
    assert mm(16, 16, 16, 16, 1.0, 4, 4, 48, 16, 0, 4, None) == -1
    assert mm(16, 16, 16, 16, 1.0, 0, 4, 64, 16, 0, 4, None) == -1
    assert mm(16, 16, 16, None, 1.0, 4, 4, 64, 16, 0, 4, None) == -3
    assert mm(16, 16, 16, 16, 1.0, 4, 4, 64, 16, 5, 4, None) == -7
    assert mm(16, 16, 16, 16, 1.0, 4, 4, 64, 16, 1, 3, None) == -1   # column-major pitch below M
    assert mm(16, 16, 16, 16, 1.0, 4, 4, 64, 8, 0, 4, None) == -2
    assert L.nvfp4b_mx_swizzle_scales(16, 16, 4, 48, None) == -1


def test_python_refusals():
    p = load_package()
    with pytest.raises(ValueError, match="CUDA"):
        p.mx_quantize(torch.zeros(4, 64, dtype=torch.bfloat16))
    with pytest.raises(ValueError, match="dtype"):
        p.mx_quantize(torch.zeros(4, 64, dtype=torch.float16))
    with pytest.raises(ValueError, match="shape"):
        p.mx_quantize(torch.zeros(64))
    with pytest.raises(ValueError, match="CUDA"):
        p.mx_gemm(*[torch.zeros(4, 32, dtype=torch.uint8)] * 4)


def test_block_norm_c_refusals():
    p = load_package()
    L, A = p._mx_sigs(), p._BlockNormArgs

    def call(**kw):
        base = dict(T=4, H=64, resid=16, ld_resid=64, resid_out=16, ld_resid_out=64, eps=1e-6, scale=1.0)
        return L.nvfp4b_block_norm(A(**{**base, **kw}), None)

    assert L.nvfp4b_block_norm(None, None) == -3
    assert call(T=0) == -1 and call(H=60) == -1 and call(H=16392) == -1 and call(ld_resid=32) == -1
    assert call(H=40, ld_resid=40, ld_resid_out=40, codes=16, scales=16) == -1        # H % 32 with codes
    assert call(resid=None) == -3 and call(resid_out=None) == -3 and call(codes=16) == -3 and call(amax=16) == -3
    assert call(resid_f32=2) == -7 and call(eps=-1.0) == -7 and call(eps=float("nan")) == -7
    assert call(gate=16) == -7 and call(post_weight=16) == -7 and call(post_norm=1) == -7   # without y
    assert call(y=16, ld_y=64, gate=16, gate_col_stride=2) == -7
    assert call(y=16, ld_y=64, gate=16, gate_row_stride=-1) == -1
    assert call(resid=8) == -2 and call(ld_resid=68) == -2 and call(norm_weight=8, out=16, ld_out=64) == -2
    assert call(y=16, ld_y=64, gate=18, gate_f32=1) == -2
    assert call(out=16, ld_out=64, amax=18) == -2


def test_block_norm_refuses_rows_that_share_memory():
    """Rows of 64 bf16 (128 bytes) at made-up addresses; what is allowed launches, and is tested on the GPU."""
    p = load_package()
    L, A = p._mx_sigs(), p._BlockNormArgs
    base = 1 << 20

    def call(**kw):
        kw = {**dict(T=4, H=64, resid=base, ld_resid=64, eps=1e-6, scale=1.0), **kw}
        return L.nvfp4b_block_norm(A(**kw), None)

    far = base + (1 << 16)
    assert call(resid_out=base + 128, ld_resid_out=64) == -7                          # a row further on
    assert call(resid_out=base, ld_resid_out=72) == -7                                # another pitch
    assert call(resid_out=base, ld_resid_out=64, resid_out_f32=1) == -7               # another type
    assert call(resid_out=base - 512 + 16, ld_resid_out=64) == -7                     # the last row reaches in
    assert call(ld_resid=128, resid_out=base + 64, ld_resid_out=128) == -7            # half a row aside
    assert call(ld_resid=128, resid_out=base + 192, ld_resid_out=128) == -7           # wraps into the next row
    assert call(y=far, ld_y=64, out=far + 128, ld_out=64) == -7
    assert call(y=far, ld_y=64, y_f32=1, out=far, ld_out=64) == -7
    assert call(resid_out=far, ld_resid_out=64, out=far, ld_out=64) == -7             # two outputs
    assert call(codes=base + 256, scales=far) == -7
    assert call(y=far, ld_y=64, gate=far + 4096, gate_row_stride=64, gate_col_stride=1, out=far + 4096, ld_out=64) == -7
