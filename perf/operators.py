"""MXFP4 operators and the block norm: cases, plain forms and 64-bit values.

MXFP4 (OCP microscaling): 32 consecutive elements share a power of two 2^e (one e8m0 byte, e + 127) and each is an e2m1
code of x / 2^e, two codes per byte, the even-index element in the low nibble.  With `own` false `run` computes the
operators from elementary torch operations; with `own` true it calls the package.  Quantised results are returned as the
values that their codes and scales stand for."""
import math

import torch

own = False

BF16, F32, F32_COL = "bf16", "f32", "f32_col"
DTYPE = {"bf16": torch.bfloat16, "f32": torch.float32, "f32_col": torch.float32}


def listed():
    return [
        # a verify step's rows through an odd width, fp32 as the dense Linear's activations are
        {"name": "quantize_16x2848_f32", "op": "quantize", "T": 16, "K": 2848, "x": F32},
        # the quantiser benchmark's largest batch
        {"name": "quantize_8192x2816_bf16", "op": "quantize", "T": 8192, "K": 2816, "x": BF16},
        # the dense feed-forward's gated activation: one token, and a prefill
        {"name": "geglu_1x2112", "op": "geglu", "T": 1, "I": 2112},
        {"name": "geglu_4096x2112", "op": "geglu", "T": 4096, "I": 2112},
        # one token through the dense gate and up projections
        {"name": "gemm_1x4224x2816", "op": "gemm", "M": 1, "N": 4224, "K": 2816, "out": BF16},
        # sixteen draft tokens through the vocabulary projection, fp32 logits
        {"name": "gemm_16x262144x2816", "op": "gemm", "M": 16, "N": 262144, "K": 2816, "out": F32},
        # ragged in every size, K a multiple of 32 only, the column-major output
        {"name": "gemm_333x2001x1056", "op": "gemm", "M": 333, "N": 2001, "K": 1056, "out": F32_COL},
        # 32 sequences x 16 draft tokens through the dense down projection
        {"name": "gemm_512x2816x2112", "op": "gemm", "M": 512, "N": 2816, "K": 2112, "out": BF16},
        # the GEMM benchmark's largest prefill
        {"name": "gemm_8192x14336x4096", "op": "gemm", "M": 8192, "N": 14336, "K": 4096, "out": BF16},
        # one token: the input norm, straight to MXFP4
        {"name": "norm_mx_1x2816", "op": "norm", "T": 1, "H": 2816, "y": "", "resid": BF16, "gate": "", "to": "mx"},
        # after the experts: post-norm, fp32 residual stream, the next norm in bf16 with its amax
        {"name": "norm_chain_512x2816", "op": "norm", "T": 512, "H": 2816, "y": F32, "resid": F32, "gate": "",
         "to": "bf16"},
        # a prefill's rows: post-norm with a gate per token, bf16 residual, the next norm straight to MXFP4
        {"name": "norm_gate_mx_8192x2816", "op": "norm", "T": 8192, "H": 2816, "y": BF16, "resid": BF16,
         "gate": "row", "to": "mx"},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["quantize", "geglu", "gemm", "gemm", "norm", "norm"])
    if op == "quantize":
        return {"op": op, "T": _log(rng, 1, 8192), "K": 32 * _log(rng, 1, 128), "x": rng.choice([BF16, F32])}
    if op == "geglu":
        return {"op": op, "T": _log(rng, 1, 8192), "I": 32 * _log(rng, 1, 128)}
    if op == "gemm":
        return {"op": op, "M": _log(rng, 1, 8192), "N": _log(rng, 16, 14336), "K": 32 * _log(rng, 1, 128),
                "out": rng.choice([BF16, F32, F32_COL])}
    to = rng.choice(["mx", "bf16"])
    return {"op": op, "T": _log(rng, 1, 8192), "H": 32 * _log(rng, 2, 88) if to == "mx" else 8 * _log(rng, 4, 352),
            "y": rng.choice(["", BF16, F32]), "resid": rng.choice([BF16, F32]),
            "gate": rng.choice(["", "row", "feature"]), "to": to}


# ---- inputs -----------------------------------------------------------------------------------------------------

def _scale_bytes(rows, K):
    return -(-rows // 128) * -(-K // 128) * 512


def _tiles(logical, K):
    """Logical scale bytes [rows, K/32] in the 128x4-tile layout that the tensor cores read, padding zero."""
    rows, kb = logical.shape
    r, c = -(-rows // 128), -(-kb // 4)
    p = torch.zeros(r * 128, c * 4, dtype=torch.uint8, device=logical.device)
    p[:rows, :kb] = logical
    return p.view(r, 4, 32, c, 4).permute(0, 3, 2, 1, 4).reshape(-1).contiguous()


def _mx(x):
    """(codes [rows, K/2], logical scale bytes [rows, K/32]) of x; x in 32 or 64 bits."""
    b = x.reshape(x.shape[0], -1, 32)
    if x.dtype == torch.float32:
        byte = ((b.abs().amax(-1).view(torch.int32) >> 23) - 2).clamp_(min=0)
    else:
        byte = (torch.frexp(b.abs().amax(-1))[1] + 124).clamp_(min=0)
    a = b * ((1150 - byte.long()) << 52).view(torch.float64).to(x.dtype)[..., None]
    m = a.abs()
    code = sum(t.to(torch.uint8) for t in (m > 0.25, m >= 0.75, m > 1.25, m >= 1.75, m > 2.5, m >= 3.5, m > 5.0))
    code += torch.signbit(a).to(torch.uint8) * 8
    code = code.reshape(x.shape[0], -1)
    return code[:, 0::2] | (code[:, 1::2] << 4), byte.to(torch.uint8)


_E2M1 = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0, -0.0, -0.5, -1.0, -1.5, -2.0, -3.0, -4.0, -6.0]


def _values(codes, byte, dtype=torch.float32):
    """The values of codes and logical scale bytes."""
    pair = torch.tensor([[_E2M1[i & 15], _E2M1[i >> 4]] for i in range(256)], dtype=dtype, device=codes.device)
    v = pair[codes.int()].view(codes.shape[0], -1, 32)
    v *= ((byte.long() + 896) << 52).view(torch.float64).to(dtype)[..., None]
    return v.view(codes.shape[0], -1)


def _normal(shape, g, std=1.0):
    return torch.randn(shape, generator=g, device="cuda") * std


def _outliers(shape, g):
    """N(0, 1) with one element in a thousand scaled by 50, as activations have."""
    x = _normal(shape, g)
    return torch.where(torch.rand(shape, generator=g, device="cuda") < 1e-3, 50.0 * x, x)


def _quantised(rows, K, g, std):
    codes = torch.empty(rows, K // 2, dtype=torch.uint8, device="cuda")
    byte = torch.empty(rows, K // 32, dtype=torch.uint8, device="cuda")
    step = max(1, (1 << 25) // K)
    for i in range(0, rows, step):
        n = min(step, rows - i)
        codes[i:i + n], byte[i:i + n] = _mx(_normal((n, K), g, std))
    return codes, byte


def prepare(case, seed):
    g = torch.Generator("cuda").manual_seed(seed)
    op, s = case["op"], {"case": case}
    if op in ("quantize", "geglu"):
        T = case["T"]
        K = case["K"] if op == "quantize" else case["I"]
        if op == "quantize":
            s["x"] = _outliers((T, K), g).to(DTYPE[case["x"]])
        else:
            s["x"] = torch.cat([_normal((T, K), g, 1.5), _normal((T, K), g)], 1).bfloat16()
        s["codes"] = torch.empty(T, K // 2, dtype=torch.uint8, device="cuda")
        s["scales"] = torch.empty(_scale_bytes(T, K), dtype=torch.uint8, device="cuda")
        s["values"] = torch.empty(T, K, dtype=DTYPE[case.get("x", BF16)], device="cuda")
    elif op == "gemm":
        M, N, K = case["M"], case["N"], case["K"]
        s["a"], s["a_byte"] = _quantised(M, K, g, 1.0)
        s["b"], s["b_byte"] = _quantised(N, K, g, 0.02)
        s["a_scales"], s["b_scales"] = _tiles(s["a_byte"], K), _tiles(s["b_byte"], K)
        s["out"] = torch.empty((N, M) if case["out"] == F32_COL else (M, N), dtype=DTYPE[case["out"]], device="cuda")
    else:
        T, H = case["T"], case["H"]
        s["resid"] = _outliers((T, H), g).to(DTYPE[case["resid"]])
        s["pre_w"] = (1.0 + _normal((H,), g, 0.1)).bfloat16()
        s["y"] = s["post_w"] = s["gate"] = None
        if case["y"]:
            s["y"] = _normal((T, H), g, 3.0).to(DTYPE[case["y"]])
            s["post_w"] = (1.0 + _normal((H,), g, 0.1)).bfloat16()
            if case["gate"]:
                s["gate"] = torch.sigmoid(_normal((T, 1) if case["gate"] == "row" else (H,), g))
        s["resid_out"] = torch.empty_like(s["resid"])
        if case["to"] == "mx":
            s["codes"] = torch.empty(T, H // 2, dtype=torch.uint8, device="cuda")
            s["scales"] = torch.empty(_scale_bytes(T, H), dtype=torch.uint8, device="cuda")
            s["values"] = torch.empty(T, H, dtype=torch.bfloat16, device="cuda")
        else:
            s["z"] = torch.empty(T, H, dtype=torch.bfloat16, device="cuda")
            s["amax"] = torch.empty(1, device="cuda")
    return s


SCALE, EPS = 0.75, 1e-6     # a layer's residual scale; the norms' epsilon


# ---- one pass ---------------------------------------------------------------------------------------------------

def run(s):
    return _run_own(s) if own else _run_plain(s)


def _run_own(s):
    from __graft_entry__ import load_package
    p = load_package()
    case, op = s["case"], s["case"]["op"]
    if op == "gemm":
        kind = {BF16: p.OUT_BF16_ROWMAJOR, F32: p.OUT_F32_ROWMAJOR, F32_COL: p.OUT_F32_COLMAJOR}[case["out"]]
        return p.mx_gemm(s["a"], s["a_scales"], s["b"], s["b_scales"], out=s["out"], out_kind=kind)
    if op == "norm":
        p.block_norm(s["resid"], s["pre_w"], eps=EPS, y=s["y"], post_weight=s["post_w"], gate=s["gate"],
                     scale=SCALE if s["y"] is not None else 1.0, resid_out=s["resid_out"] if case["y"] else None,
                     out=s.get("z"), amax=s.get("amax"), codes=s.get("codes"), scales=s.get("scales"))
        got = {"resid": s["resid_out"]} if case["y"] else {}
        if case["to"] == "mx":
            return {**got, "z": p.mx_dequantize(s["codes"], s["scales"], out=s["values"])}
        return {**got, "z": s["z"], "amax": s["amax"]}
    quantize = p.mx_quantize if op == "quantize" else p.mx_geglu_quantize
    quantize(s["x"], codes=s["codes"], scales=s["scales"])
    return p.mx_dequantize(s["codes"], s["scales"], out=s["values"])


def _run_plain(s):
    case, op = s["case"], s["case"]["op"]
    if op == "gemm":
        d = _values(s["a"], s["a_byte"]) @ _values(s["b"], s["b_byte"]).t()
        return d.t().contiguous() if case["out"] == F32_COL else d.to(DTYPE[case["out"]])
    if op == "quantize":
        return _values(*_mx(s["x"].float())).to(s["x"].dtype)
    if op == "geglu":
        # 64 bits: a product next to a rounding border of the 4-bit codes must fall on its own side
        g, u = s["x"].double().chunk(2, 1)
        h = 0.5 * g * (1.0 + torch.tanh(math.sqrt(2.0 / math.pi) * (g + 0.044715 * g * g * g))) * u
        return _values(*_mx(h)).bfloat16()
    wide = torch.float64 if case["to"] == "mx" else torch.float32      # 64 bits for 4-bit codes, as above
    r, got = s["resid"].to(wide), {}
    if case["y"]:
        y = s["y"].to(wide)
        n = y * torch.rsqrt((y * y).mean(1, keepdim=True) + EPS) * s["post_w"].to(wide)
        r = SCALE * (r + (n if s["gate"] is None else s["gate"].to(wide) * n))
        got["resid"] = r.to(s["resid"].dtype)
    z = r * torch.rsqrt((r * r).mean(1, keepdim=True) + EPS) * s["pre_w"].to(wide)
    if case["to"] == "mx":
        return {**got, "z": _values(*_mx(z)).bfloat16()}
    z = z.bfloat16()
    return {**got, "z": z, "amax": z.float().abs().max().view(1)}


def work(case):
    op = case["op"]
    if op == "gemm":
        M, N, K = case["M"], case["N"], case["K"]
        return {"bytes": (M + N) * K * 17 / 32 + M * N * (2 if case["out"] == BF16 else 4), "flops": 2 * M * N * K}
    if op == "norm":
        n, size = case["T"] * case["H"], {"": 0, BF16: 2, F32: 4}
        b = size[case["resid"]] + (size[case["resid"]] + size[case["y"]] if case["y"] else 0)
        b += 17 / 32 + 2 if case["to"] == "mx" else 2
        return {"bytes": n * b, "flops": n * (12 if case["y"] else 6)}
    n = case["T"] * (case["K"] if op == "quantize" else case["I"])
    x = 4 if op == "geglu" or case["x"] == F32 else 2          # read per element: gate and up in bf16, or x
    v = 4 if case.get("x") == F32 else 2                       # the values written
    return {"bytes": n * (x + 17 / 32 + v), "flops": n * (20 if op == "geglu" else 4)}


# ---- the definitions in 64 bits -----------------------------------------------------------------------------------

def _nearest(x):
    """Values of the MXFP4 quantisation of x (64 bits): half-even rounding on the e2m1 grid of each block."""
    b = x.reshape(x.shape[0], -1, 32)
    top = b.abs().amax(2, keepdim=True)
    e = torch.where(top > 0, torch.frexp(top)[1].double() - 3, torch.full_like(top, -127.0)).clamp(min=-127)
    v = (b / torch.exp2(e)).clamp(-6, 6)
    step = torch.where(v.abs() < 2, 0.5, torch.where(v.abs() < 4, 1.0, 2.0))
    return (torch.round(v / step) * step * torch.exp2(e)).reshape(x.shape)


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "gemm":
        grid = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6], dtype=torch.float64, device="cuda")

        def decode(codes, byte):
            v = torch.empty(codes.shape[0], 2 * codes.shape[1], dtype=torch.float64, device="cuda")
            for i, c in enumerate((codes & 15, codes >> 4)):
                v[:, i::2] = grid[(c & 7).int()] * (1.0 - 2.0 * (c >> 3).double())
            return v * torch.exp2(byte.double() - 127.0).repeat_interleave(32, 1)

        a, parts = decode(s["a"], s["a_byte"]), []
        for i in range(0, case["N"], 16384):
            parts.append(a @ decode(s["b"][i:i + 16384], s["b_byte"][i:i + 16384]).mT)
        d = torch.cat(parts, 1)
        return d.mT.contiguous() if case["out"] == F32_COL else d
    if op == "quantize":
        return _nearest(s["x"].double())
    if op == "geglu":
        g, u = s["x"][:, :case["I"]].double(), s["x"][:, case["I"]:].double()
        # 0.5 (1 + tanh t) = 1 / (1 + exp(-2 t))
        return _nearest(g / (1.0 + torch.exp(-math.sqrt(8.0 / math.pi) * (g + 0.044715 * g ** 3))) * u)
    r, got = s["resid"].double(), {}

    def norm(v, w):
        return v / torch.sqrt(v.square().sum(1, keepdim=True) / v.shape[1] + EPS) * w.double()

    if case["y"]:
        n = norm(s["y"].double(), s["post_w"])
        r = (r + (1.0 if s["gate"] is None else s["gate"].double()) * n) * SCALE
        got["resid"] = r
    z = norm(r, s["pre_w"])
    if case["to"] == "mx":
        return {**got, "z": _nearest(z)}
    return {**got, "z": z, "amax": None}
