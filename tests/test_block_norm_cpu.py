"""CPU checks of which buffers a block norm may share: refusals that are made before the device is touched."""
import pytest
import torch

from __graft_entry__ import load_package

pytestmark = pytest.mark.skipif(torch.cuda.is_available(), reason="made-up addresses: only where nothing can be launched")
BASE, T, H = 1 << 20, 4, 64                    # rows of 64 bf16 (128 bytes) at made-up addresses
OUT = {"resid_out": dict(resid_out=BASE, ld_resid_out=H), "out": dict(out=BASE, ld_out=H),
       "codes": dict(codes=BASE, scales=BASE + (1 << 20)), "scales": dict(codes=BASE + (1 << 20), scales=BASE),
       "amax": dict(amax=BASE, out=BASE + (1 << 20), ld_out=H)}
SIZE = {"resid_out": T * 128, "out": T * 128, "codes": T * 32, "scales": 512, "amax": 4}      # bytes


def _call(**kw):
    p = load_package()
    far = BASE + (1 << 24)
    args = {**dict(T=T, H=H, resid=far, ld_resid=H, eps=1e-6, scale=1.0), **kw}
    return p._mx_sigs().nvfp4b_block_norm(p._BlockNormArgs(**args), None)


def _inputs(at):
    far = BASE + (2 << 24)
    y = dict(y=far, ld_y=H)
    return {"post_weight": dict(y, post_weight=at), "norm_weight": dict(norm_weight=at),
            "gate per feature": dict(y, gate=at, gate_col_stride=1),
            "gate per token": dict(y, gate=at, gate_row_stride=1, gate_f32=1),
            "gate of a wide row": dict(y, gate=at, gate_row_stride=H),
            "gate per element": dict(y, gate=at, gate_row_stride=H, gate_col_stride=1),
            "resid": dict(resid=at, ld_resid=H), "y": dict(y=at, ld_y=H)}


BYTES = {"post_weight": 128, "norm_weight": 128, "gate per feature": 128, "gate per token": 16, "gate of a wide row": 386,
         "gate per element": T * 128, "resid": T * 128, "y": T * 128}


@pytest.mark.parametrize("out", OUT)
@pytest.mark.parametrize("name", BYTES)
def test_outputs_on_inputs_are_refused(out, name):
    last = (SIZE[out] - 1) // 16 * 16                          # the input starts in the output's last 16 bytes
    assert _call(**OUT[out], **_inputs(BASE + last)[name]) == -7
    first = (BYTES[name] - 1) // 16 * 16                       # and ends in its first 16
    assert _call(**OUT[out], **_inputs(BASE - first)[name]) == -7


@pytest.mark.parametrize("a", OUT)
@pytest.mark.parametrize("b", OUT)
def test_outputs_on_outputs_are_refused(a, b):
    names = [k for k in OUT[a] if not k.startswith("ld_") and OUT[a][k] == BASE]
    other = {k: v + (1 << 21) if not k.startswith("ld_") and v != BASE else v for k, v in OUT[b].items()}
    if a == b or "amax" in (a, b) and "out" in (a, b):
        return
    both = {**other, **{k: v for k, v in OUT[a].items() if k in names or k not in other}}
    assert _call(**both) == -7


def test_amax_in_out_is_refused():
    assert _call(out=BASE, ld_out=H, amax=BASE + T * 128 - 4) == -7
    assert _call(out=BASE, ld_out=2 * H, amax=BASE + 3 * 256 + 124) == -7


def test_neighbours_are_not_refused():
    """What touches only in a gap between rows, or at an end, passes the checks (and then finds no device here)."""
    for name, size in BYTES.items():
        for out, kw in OUT.items():
            for at in (BASE + -(-SIZE[out] // 16) * 16, BASE - -(-size // 16) * 16):
                assert _call(**kw, **_inputs(at)[name]) == -4, (name, out)
    gap = BASE + 128                                           # rows of 128 bytes, 256 apart
    for kw in (dict(norm_weight=gap), dict(y=gap, ld_y=2 * H), dict(y=BASE + (3 << 24), ld_y=H, gate=gap, gate_row_stride=2 * H),
               dict(y=BASE + (3 << 24), ld_y=H, gate=gap, gate_row_stride=H, gate_f32=1),
               dict(y=BASE + (3 << 24), ld_y=H, gate=gap, gate_row_stride=2 * H, gate_col_stride=1)):
        assert _call(resid_out=BASE, ld_resid_out=2 * H, **kw) == -4, kw
    assert _call(resid_out=BASE, ld_resid_out=2 * H, out=BASE + (1 << 20), ld_out=H, amax=gap + 64) == -4
