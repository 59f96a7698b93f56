"""numpy float64 oracle of the MXFP4 operators (TEST INFRASTRUCTURE ONLY): OCP microscaling quantisation (e2m1 codes, one
e8m0 byte per 32 elements), its tile layout, the GELU gate and the block norm.

The scale layout and the activation follow the reference's NVFP4 ones (kernels/fp4_gemm.cu:14-33 with 32-element
blocks, kernels/elementwise.cu:10-22 and :44-47)."""
from __future__ import annotations

import numpy as np

GRID = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])


def quantize(x: np.ndarray) -> tuple[np.ndarray, np.ndarray]:
    """[rows, K] -> (codes [rows, K/2] uint8, logical scale bytes [rows, K/32] uint8), float64 arithmetic."""
    x = np.asarray(x, np.float64)
    b = x.reshape(x.shape[0], -1, 32)
    with np.errstate(invalid="ignore"):
        amax = np.abs(b).max(2)
        bad = ~(amax < 2.0 ** 128)
    e = np.frexp(np.where(bad | (amax == 0), 1.0, amax))[1] - 3          # floor(log2 amax) - 2
    e = np.where(amax == 0, -127, np.maximum(e, -127))
    byte = np.where(bad, 255, e + 127).astype(np.uint8)
    with np.errstate(invalid="ignore"):
        y = np.minimum(np.abs(np.ldexp(b, -e[..., None])), 6.0)
        d = np.abs(y[..., None] - GRID)
        code = np.argmin(d, axis=-1)                                      # the lower one of two equally near
        up = np.minimum(code + 1, 7)
        tie = np.take_along_axis(d, code[..., None], -1) == np.take_along_axis(d, up[..., None], -1)
        code = np.where(tie[..., 0] & (code & 1 == 1), up, code)          # ties to the even code
    code = np.where(bad[..., None], 0, code | (np.signbit(b) << 3)).astype(np.uint8).reshape(x.shape)
    return code[:, 0::2] | (code[:, 1::2] << 4), byte


def dequantize(codes: np.ndarray, byte: np.ndarray) -> np.ndarray:
    n = np.empty((codes.shape[0], 2 * codes.shape[1]), np.uint8)
    n[:, 0::2], n[:, 1::2] = codes & 15, codes >> 4
    v = GRID[n & 7] * np.where(n & 8, -1.0, 1.0)
    s = np.where(byte == 255, np.nan, np.ldexp(1.0, byte.astype(np.int64) - 127))
    return (v.reshape(codes.shape[0], -1, 32) * s[..., None]).reshape(n.shape)


def scale_buffer_bytes(rows: int, k: int) -> int:
    return -(-rows // 128) * -(-k // 128) * 512


def _offsets(rows: int, k: int) -> np.ndarray:
    m, b = np.meshgrid(np.arange(rows), np.arange(k // 32), indexing="ij")
    return ((m // 128) * -(-k // 128) + b // 4) * 512 + (m % 32) * 16 + (m % 128) // 32 * 4 + b % 4


def tile_scales(byte: np.ndarray, k: int) -> np.ndarray:
    out = np.zeros(scale_buffer_bytes(byte.shape[0], k), np.uint8)
    out[_offsets(byte.shape[0], k)] = byte
    return out


def untile_scales(buf: np.ndarray, rows: int, k: int) -> tuple[np.ndarray, bool]:
    """(logical bytes [rows, K/32], whether every padding byte is zero)."""
    off = _offsets(rows, k)
    rest = np.ones(buf.size, bool)
    rest[off] = False
    return buf[off], not buf[rest].any()


def geglu(g: np.ndarray, u: np.ndarray) -> np.ndarray:
    """gelu_tanh(g) u, with 0.5 (1 + tanh t) written as 1 / (1 + exp(-2 t)) (no cancellation)."""
    g, u = np.asarray(g, np.float64), np.asarray(u, np.float64)
    with np.errstate(over="ignore", invalid="ignore"):
        return g / (1.0 + np.exp(-np.sqrt(8.0 / np.pi) * (g + 0.044715 * g ** 3))) * u


def rms(x: np.ndarray, eps: float) -> np.ndarray:
    return x / np.sqrt((x * x).mean(1, keepdims=True) + eps)


def block_norm(resid=None, norm_weight=None, eps=1e-6, y=None, post_weight=None, post_norm=None, gate=None, scale=1.0):
    """(r, z): r = scale (resid + gate * [rms](y) post_weight), z = rms(r) norm_weight; all float64.  Without y r = scale
    resid; a resid of None is 0, so a zero that y alone gives is +0 before the scale."""
    r = resid
    if y is not None:
        n = np.asarray(y, np.float64)
        if post_norm if post_norm is not None else post_weight is not None:
            n = rms(n, eps)
        if post_weight is not None:
            n = n * post_weight
        r = (n if gate is None else n * gate) + (0.0 if resid is None else resid)
    r = np.asarray(r, np.float64) * scale
    z = rms(r, eps)
    return r, z if norm_weight is None else z * norm_weight
