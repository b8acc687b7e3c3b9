"""Operators of the library between its products, as cases that can be timed and compared: the norm in front of a group of
projections with an output in 8 or 4 bits, 4-bit microscaled floating point (quantization and product), and projections over
activations that a norm left quantized.

  norm         h = x + residual, rounded to their type (h = x without a residual); r = 1 / sqrt(mean(h^2) + eps), the sum and the root in 64
               bits, r rounded to f32; y = (h r) w, two products rounded to f32 each.  y in the input's type, or quantized:
                 q8_k   256 values: s = 127 / amax, q = the integer nearest to s y, scale 1 / s (all f32)
                 fp8    128 values (the last block may be shorter): E4M3 under the least power of two that brings amax to 448 or
                        less (not below 2^-100)
                 mxfp4  32 values: E2M1 under 2^(floor(log2(amax)) - 2), magnitudes above 6 become 6
               halves go to the even neighbour.
  quantize     a matrix of floats as MXFP4 blocks (a byte of scale, 32 codes of 4 bits), and the values that these stand for.
  product      y = x W^T in MXFP4: W's rows hold MXFP4 blocks, x's are quantized to them within the call.  f32 in, f32 out.
  projections  norm, then several matrices over its one quantized output: FP8 (E4M3 codes, a scale for every 128 x 128) or MXFP4.

A case is a dict of plain values; `prepare` makes what a program holds before the call, `run` is one pass.
"""
import math

import torch

own = False

DEVICE = "cuda:0"
EPS = 1e-5
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def listed():
    return [
        # one token in front of Llama-3-8B's attention: residual added, 8-bit output; the smallest call, latency counts
        {"name": "norm_decode", "family": "norm", "batch": 1, "cols": 4096, "type": "f32", "residual": True, "form": "fp8"},
        # an odd number of sequences of gpt-oss-20b's width (22 blocks and a half), hidden states in bf16
        {"name": "norm_batch_61_ragged", "family": "norm", "batch": 61, "cols": 2880, "type": "bf16", "residual": True, "form": "fp8"},
        # a 512-token chunk in front of K-quant projections
        {"name": "norm_prefill_q8_k", "family": "norm", "batch": 512, "cols": 4096, "type": "f32", "residual": True, "form": "q8_k"},
        # a batch of long prompts, the last norm's plain output among them: the largest
        {"name": "norm_long", "family": "norm", "batch": 16384, "cols": 4096, "type": "f32", "residual": True, "form": "none"},
        # a projection of a checkpoint in bf16 to 4 bits
        {"name": "quantize_matrix", "family": "quantize", "rows": 14336, "cols": 4096, "type": "bf16"},
        # a few hidden states
        {"name": "quantize_rows", "family": "quantize", "rows": 61, "cols": 2880, "type": "f32"},
        # one token through a gate projection: the weights' bytes count
        {"name": "product_decode", "family": "product", "batch": 1, "rows": 14336, "cols": 4096},
        # an odd number of sequences decoding together, gpt-oss-20b's width
        {"name": "product_batch_61_ragged", "family": "product", "batch": 61, "rows": 2880, "cols": 2880},
        # a 512-token chunk, gate or up
        {"name": "product_prefill", "family": "product", "batch": 512, "rows": 14336, "cols": 4096},
        # a long prompt's down projection
        {"name": "product_prefill_long", "family": "product", "batch": 4096, "rows": 4096, "cols": 14336},
        # one token: the norm and q, k, v of Llama-3-8B in 8 bits
        {"name": "projections_decode", "family": "projections", "batch": 1, "cols": 4096, "rows": "4096,1024,1024", "kind": "fp8"},
        # a 512-token chunk: the norm, gate and up in 4 bits
        {"name": "projections_prefill", "family": "projections", "batch": 512, "cols": 4096, "rows": "14336,14336", "kind": "mxfp4"},
    ]


def _log_int(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    family = rng.choice(("norm", "quantize", "product", "projections"))
    if family == "norm":
        form = rng.choice(("none", "fp8", "q8_k", "mxfp4"))
        unit = {"q8_k": 256, "mxfp4": 32}.get(form, rng.choice((1, 4, 128)))
        cols = max(unit, _log_int(rng, 96, 16384) // unit * unit)
        return {"family": family, "batch": _log_int(rng, 1, min(16384, 16384 * 4096 // cols)), "cols": cols, "type": rng.choice(("f32", "f32", "bf16", "f16")),
                "residual": rng.random() < 0.7, "form": form}
    if family == "quantize":
        cols = 32 * _log_int(rng, 2, 448)
        return {"family": family, "rows": _log_int(rng, 1, min(32768, 14336 * 4096 // cols)), "cols": cols, "type": rng.choice(("f32", "bf16", "f16"))}
    if family == "product":
        rows, cols = _log_int(rng, 96, 14336), 32 * _log_int(rng, 3, 448)
        return {"family": family, "batch": _log_int(rng, 1, min(4096, 4096 * 4096 * 14336 // (rows * cols))), "rows": rows, "cols": cols}
    kind = rng.choice(("fp8", "mxfp4"))
    cols = _log_int(rng, 96, 8192) // 4 * 4 if kind == "fp8" else 32 * _log_int(rng, 3, 256)
    rows = [_log_int(rng, 96, 8192) for _ in range(rng.choice((2, 3)))]
    return {"family": family, "batch": _log_int(rng, 1, min(2048, 512 * 4096 * 28672 // (sum(rows) * cols))), "cols": cols, "rows": ",".join(map(str, rows)),
            "kind": kind}


# ---- inputs ----

def _states(gen, rows, cols, type_, spread=1.0):
    """Hidden states: a spread of their own for every row, a few channels eight times as large."""
    x = torch.randn((rows, cols), generator=gen, device=DEVICE)
    x *= spread * (0.5 + torch.rand((rows, 1), generator=gen, device=DEVICE))
    x[:, torch.randint(0, cols, (max(1, cols // 512),), generator=gen, device=DEVICE)] *= 8.0
    return x.to(TYPES[type_])


def _weights(gen, rows, cols):
    """N(0, 0.02) weights whose spread differs from row to row."""
    return torch.randn((rows, cols), generator=gen, device=DEVICE) * (torch.rand((rows, 1), generator=gen, device=DEVICE) * 0.03 + 0.005)


def _fp8_matrix(gen, rows, cols):
    """E4M3 codes and an f32 scale for every 128 x 128 that takes a block's largest magnitude to about 448."""
    w = _weights(gen, rows, cols)
    scales = (torch.rand((-(-rows // 128), -(-cols // 128)), generator=gen, device=DEVICE) + 1.0) * (0.07 / 448)
    return {"w": (w / _expand(scales, rows, cols)).clamp_(-448, 448).to(torch.float8_e4m3fn), "scales": scales}


def _mxfp4_matrix(gen, rows, cols):
    """Codes, two a byte as GGUF has them (element i in the low half of byte i, element i + 16 in the high one), and a scale byte a block."""
    scale, z = _mxfp4_parts(_weights(gen, rows, cols))
    code = torch.bucketize(z.abs(), torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0], device=DEVICE)) + 8 * (z < 0)
    return {"codes": (code[..., :16] + 16 * code[..., 16:]).to(torch.uint8), "bytes": scale.to(torch.uint8)}


def _matrix(gen, kind, rows, cols):
    m = _fp8_matrix(gen, rows, cols) if kind == "fp8" else _mxfp4_matrix(gen, rows, cols)
    m |= {"kind": kind, "rows": rows, "cols": cols}
    if own:  # the resident copy that a program makes of its weights when it loads them
        import frink_amd as fa
        if kind == "fp8":
            m["resident"] = fa.Weights.from_device_fp8(m["w"], m["scales"], rows, cols)
        else:
            m["resident"] = fa.Weights.from_device(fa.MXFP4, torch.cat((m["bytes"], m["codes"]), 2).flatten(), rows, cols)
    return m


def prepare(case, seed):
    gen = torch.Generator(DEVICE)
    gen.manual_seed(seed)
    family, cols = case["family"], case["cols"]
    s = {"family": family, "case": case}
    if family == "quantize":
        s["x"] = _weights(gen, case["rows"], cols).to(TYPES[case["type"]])
        return s
    s["x"] = _states(gen, case["batch"], cols, case.get("type", "f32"))
    if family == "product":
        s["matrix"] = _matrix(gen, "mxfp4", case["rows"], cols)
        return s
    s["weight"] = 1.0 + 0.2 * torch.randn(cols, generator=gen, device=DEVICE)
    form = case["form"] if family == "norm" else case["kind"]
    s["residual"] = _states(gen, case["batch"], cols, case.get("type", "f32"), 3.0) if case.get("residual", True) else None
    if family == "projections":
        s["matrices"] = [_matrix(gen, case["kind"], int(r), cols) for r in case["rows"].split(",")]
    if own and form != "none":  # room for the quantized batch, as a program keeps it
        import frink_amd as fa
        s["acts"] = fa.BatchActs(case["batch"], cols, form)
    return s


# ---- the plain forms ----

def _expand(scales, rows, cols):
    return scales.repeat_interleave(128, 0)[:rows].repeat_interleave(128, 1)[:, :cols]


def _power(e):
    """2^e in f32, -126 <= e <= 127."""
    return ((e + 127).to(torch.int32) << 23).view(torch.float32)


def _blocks(v, n):
    return torch.nn.functional.pad(v, (0, -v.shape[-1] % n)).view(v.shape[0], -1, n)


def _q8_k(v):
    b = _blocks(v, 256)
    top = b.abs().amax(-1, keepdim=True)
    s = torch.full_like(top, 127.0) / top  # (a number divided by a tensor would be two roundings)
    return (torch.round(s * b).clamp(-127, 127) * (1.0 / s)).view(v.shape)


def _fp8(v):
    b = _blocks(v, 128)
    mantissa, exponent = torch.frexp(b.abs().amax(-1, keepdim=True))  # amax = mantissa 2^exponent; 448 = 0.875 x 2^9
    e = torch.where(mantissa <= 0.875, exponent - 9, exponent - 8).clamp(min=-100)
    return ((b * _power(-e)).to(torch.float8_e4m3fn).to(torch.float32) * _power(e)).view(v.shape[0], -1)[:, :v.shape[1]]


def _mxfp4_parts(v):
    """The scale bytes [rows][blocks][1] and the blocks' values under their scales."""
    b = _blocks(v, 32)
    exponent = torch.frexp(b.abs().amax(-1, keepdim=True)).exponent  # floor(log2(amax)) + 1
    e = (exponent - 3).clamp(min=-126)
    return e + 127, b * _power(-e)


def _mxfp4(v):
    byte, z = _mxfp4_parts(v)
    size = z.abs()
    step = torch.where(size < 2.0, 0.5, torch.where(size < 4.0, 1.0, 2.0))
    return ((torch.round(z / step) * step).clamp(-6.0, 6.0) * _power(byte - 127)).view(v.shape)


FORMS = {"q8_k": _q8_k, "fp8": _fp8, "mxfp4": _mxfp4}


def _norm(x, residual, weight):
    """(h, y in f32)"""
    h = x if residual is None else (x.float() + residual.float()).to(x.dtype)
    v = h.float()
    wide = v.double()
    r = (1.0 / torch.sqrt((wide * wide).mean(-1, keepdim=True) + EPS)).float()
    return h, v * r * weight


def _values(m):
    """A matrix in f32."""
    if m["kind"] == "fp8":
        return m["w"].to(torch.float32) * _expand(m["scales"], m["rows"], m["cols"])
    table = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0, -0.0, -0.5, -1.0, -1.5, -2.0, -3.0, -4.0, -6.0], device=DEVICE)
    codes = m["codes"].int()
    return (torch.cat((table[codes & 15], table[codes >> 4]), -1) * _power(m["bytes"].int() - 127)).view(m["rows"], m["cols"])


def run(s):
    family, case = s["family"], s["case"]
    if own:
        import frink_amd as fa
        if family == "quantize":
            return fa.dequantize_mxfp4(fa.quantize_mxfp4(s["x"]), case["cols"])
        if family == "product":
            return s["matrix"]["resident"].gemm_mxfp4(s["x"])
        y, h = fa.rms_norm(s["x"], s["weight"], EPS, residual=s["residual"], acts=s.get("acts"))
        if family == "projections":
            return [h] + [m["resident"].gemm_acts(y) for m in s["matrices"]]
        return [y if case["form"] == "none" else y.values(), h]
    if family == "quantize":
        return _mxfp4(s["x"].float())
    if family == "product":
        return _mxfp4(s["x"]) @ _values(s["matrix"]).T
    h, y = _norm(s["x"], s["residual"], s["weight"])
    if family == "projections":
        y = FORMS[case["kind"]](y)
        return [h] + [y @ _values(m).T for m in s["matrices"]]
    return [y.to(s["x"].dtype) if case["form"] == "none" else FORMS[case["form"]](y), h]


# ---- what a pass cannot do without ----

def _matrix_bytes(kind, rows, cols):
    return rows * cols + 4 * -(-rows // 128) * -(-cols // 128) if kind == "fp8" else rows * cols // 32 * 17


def work(case):
    family, cols = case["family"], case["cols"]
    size = 4 if case.get("type", "f32") == "f32" else 2
    if family == "quantize":  # the blocks written, the values written
        n = case["rows"] * cols
        return {"bytes": n * size + n // 32 * 17 + 4 * n, "flops": 4 * n}
    n = case["batch"] * cols
    if family == "product":
        return {"bytes": _matrix_bytes("mxfp4", case["rows"], cols) + 4 * (n + case["batch"] * case["rows"]), "flops": 2 * n * case["rows"]}
    norm = n * size * (3 if case.get("residual", True) else 1) + 4 * cols
    if family == "norm":
        return {"bytes": norm + int(n * {"none": size, "q8_k": 1 + 1 / 64, "fp8": 1 + 1 / 32, "mxfp4": 17 / 32}[case["form"]]), "flops": 6 * n}
    rows = [int(r) for r in case["rows"].split(",")]
    return {"bytes": norm + sum(_matrix_bytes(case["kind"], r, cols) + 4 * case["batch"] * r for r in rows), "flops": 2 * n * sum(rows) + 6 * n}


# ---- the definition in 64 bits ----

def _exact_norm(s):
    x = s["x"].double()
    h = x if s["residual"] is None else (x + s["residual"].double()).to(s["x"].dtype).double()
    r = (h.square().sum(1, keepdim=True) / h.shape[1] + EPS).pow(-0.5)
    return h, r, s["weight"].double()


def _two(e):
    """2^e in 64 bits, exactly (pow's last place can be off, and would decide which of two values is the nearer one)."""
    return ((e.long() + 1023) << 52).view(torch.float64)


def _floor_log2(v):
    """Of positive normal numbers, exactly."""
    return ((v.view(torch.int64) >> 52) - 1023).double()


def _nearest(z, bits, least, most):
    """z rounded to `bits` bits behind the leading one, exponents of `least` and more, magnitudes up to `most`."""
    step = _two(_floor_log2(z.abs().clamp(min=2.0 ** least)) - bits)
    return (torch.round(z / step) * step).clamp(-most, most)


def _exact_form(y, form):
    """y (f32 numbers in 64 bits) quantized."""
    n = {"q8_k": 256, "fp8": 128, "mxfp4": 32}[form]
    out = torch.empty_like(y)
    for k in range(0, y.shape[1], n):
        v = y[:, k:k + n]
        top = v.abs().max(1, keepdim=True).values
        if form == "q8_k":
            s = torch.div(torch.full_like(top, 127.0), top).float().double()
            q = torch.round((s * v).float().double()).clamp(-127.0, 127.0)
            out[:, k:k + n] = q * (1.0 / s).float().double()
            continue
        if form == "fp8":
            e = _floor_log2(top) - 8
            e = torch.where(top > 448.0 * _two(e), e + 1, e).clamp(min=-100.0)
            out[:, k:k + n] = _nearest(v / _two(e), 3, -6, 448.0) * _two(e)
        else:
            e = _floor_log2(top) - 2
            out[:, k:k + n] = _nearest(v / _two(e), 1, 0, 6.0) * _two(e)
    return out


def _exact_matrix(m):
    if m["kind"] == "fp8":
        w = m["w"].double()
        for r in range(0, m["rows"], 128):
            for k in range(0, m["cols"], 128):
                w[r:r + 128, k:k + 128] *= m["scales"][r // 128, k // 128].double()
        return w
    codes = torch.cat((m["codes"] & 15, m["codes"] >> 4), -1).double()
    sign, size = torch.where(codes >= 8, -1.0, 1.0), codes % 8
    # 0, 1/2, then (2 + mantissa) 2^(exponent - 2)
    value = torch.where(size < 2, size / 2, (2 + size % 2) * _two(torch.floor(size / 2) - 2))
    return (sign * value * _two(m["bytes"].double() - 127)).view(m["rows"], m["cols"])


def exact(case, seed):
    s = prepare(case, seed)
    family = case["family"]
    if family == "quantize":
        return _exact_form(s["x"].double(), "mxfp4")
    if family == "product":
        return _exact_form(s["x"].double(), "mxfp4") @ _exact_matrix(s["matrix"]).T
    h, r, w = _exact_norm(s)
    form = case["form"] if family == "norm" else case["kind"]
    if form == "none":
        return [h * r * w, h]
    # what is quantized are f32 numbers: r, h r and its product with w are rounded
    y = ((h * r.float().double()).float().double() * w).float().double()
    y = _exact_form(y, form)
    return [h] + [y @ _exact_matrix(m).T for m in s["matrices"]] if family == "projections" else [y, h]
