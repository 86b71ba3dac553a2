"""Cases that the microscaled (MX) rows, the norm that writes them, their product and the token sampler are timed on.

``run`` computes each operator in its plain form out of elementary torch operations, or, where ``own`` is true, through
the calls a user makes of ``nesgpu_amd.extensions.booleanOperations``.  The path these stand for is a network's
real-valued end: a layer's int32 sums (or floating activations) and a residual stream are normalised into 8-bit rows, multiplied by a readout's
4-bit weights, and a token (class) is drawn from the logits.
"""
import math

import torch

own = False

BLOCK = 32          # elements that share a scale
STEP = 128          # rows are padded to whole multiples of this many elements
TYPES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16, "int32": torch.int32}
# element formats: exponent of the largest value, mantissa bits, smallest normal exponent, largest value
FORMATS = {"fp4": (2, 1, 0, 6.0), "fp8": (8, 3, -6, 448.0)}


def listed():
    return [
        # a readout's weights or a batch of activations with rows that are no multiple of a block, converted once
        {"name": "quantise odd rows", "op": "quantise", "rows": 777, "K": 1000, "type": "fp32", "format": "fp8"},
        # all of a large layer's weights to 4 bits
        {"name": "quantise a large layer", "op": "quantise", "rows": 8192, "K": 16384, "type": "bf16", "format": "fp4"},
        # one request's row between two layers: latency
        {"name": "norm of one row", "op": "norm", "rows": 1, "K": 4096, "type": "bf16", "residual": "bf16",
         "format": "fp8"},
        # the int32 sums of a population's wide binary layer (8192 -> 1024, population 4096) joining a half stream
        {"name": "norm of a population's sums", "op": "norm", "rows": 4096, "K": 1024, "type": "int32",
         "residual": "fp16", "format": "fp8"},
        # a long prompt's or large batch's rows
        {"name": "norm of many rows", "op": "norm", "rows": 8192, "K": 8192, "type": "bf16", "residual": "bf16",
         "format": "fp8"},
        # one row against a vocabulary: the weights are streamed once
        {"name": "product, one row", "op": "product", "M": 1, "N": 32768, "K": 8192, "a": "fp8", "out": "fp32"},
        # a readout of ten classes over 16384 features, an odd part of a population
        {"name": "product, ten classes", "op": "product", "M": 1001, "N": 10, "K": 16384, "a": "fp8", "out": "fp32"},
        # one weight matrix for a whole population, the wide layer's shape
        {"name": "product, population", "op": "product", "M": 4096, "N": 1024, "K": 8192, "a": "fp4", "out": "bf16"},
        # a large batch against a vocabulary's part
        {"name": "product, large", "op": "product", "M": 4096, "N": 16384, "K": 8192, "a": "fp8", "out": "bf16"},
        # every member of a population answers one of ten classes from its last layer's int32 sums
        {"name": "sample ten classes", "op": "sample", "rows": 4096, "V": 10, "type": "int32", "temperature": 12.0,
         "top_k": 0, "top_p": 1.0, "min_p": 0.0, "per_row": False},
        # a few requests, each with settings of its own, an odd vocabulary with some tokens masked
        {"name": "sample a few rows", "op": "sample", "rows": 5, "V": 50001, "type": "fp16", "temperature": 0.8,
         "top_k": 60, "top_p": 0.95, "min_p": 0.02, "per_row": True},
        # a full batch over a large vocabulary, the nucleus only
        {"name": "sample a batch", "op": "sample", "rows": 256, "V": 131072, "type": "bf16", "temperature": 1.0,
         "top_k": 0, "top_p": 0.9, "min_p": 0.0, "per_row": False},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["quantise", "norm", "product", "sample"])
    if op == "quantise":
        K = _log(rng, 1, 32768)
        return {"op": op, "rows": _log(rng, 1, max(1, min(65536, (1 << 27) // K))), "K": K,
                "type": rng.choice(["fp32", "fp16", "bf16"]), "format": rng.choice(["fp4", "fp8"])}
    if op == "norm":
        K = _log(rng, 16, 20000)
        kind = rng.choice(["fp32", "fp16", "bf16", "int32"])
        residual = rng.choice(["none", rng.choice(["fp32", "fp16", "bf16"]) if kind == "int32" else kind])
        return {"op": op, "rows": _log(rng, 1, max(1, min(32768, (1 << 26) // K))), "K": K, "type": kind,
                "residual": residual, "format": rng.choice(["fp4", "fp8"])}
    if op == "product":
        M, N, K = _log(rng, 1, 8192), _log(rng, 1, 32768), _log(rng, 64, 16384)
        if M * N * K > 1 << 39:
            M = max(1, (1 << 39) // (N * K))
        return {"op": op, "M": M, "N": N, "K": K, "a": rng.choice(["fp4", "fp8"]), "out": rng.choice(["fp32", "bf16"])}
    V = _log(rng, 2, 200000)
    return {"op": op, "rows": _log(rng, 1, max(1, min(8192, (1 << 25) // V))), "V": V,
            "type": rng.choice(["fp32", "fp16", "bf16", "int32"]), "temperature": round(rng.uniform(0.3, 2.0), 3),
            "top_k": rng.choice([0, rng.randint(1, 100)]), "top_p": rng.choice([1.0, round(rng.uniform(0.2, 0.99), 3)]),
            "min_p": rng.choice([0.0, round(rng.uniform(0.01, 0.2), 3)]), "per_row": rng.random() < 0.5}


def _power(e):
    """2 ** e in 64 bits, exactly (the library's power function is off by a unit in the last place on some devices,
    which breaks the ties of a rounding)."""
    return ((e.long() + 1023) << 52).view(torch.float64)


# ---- the plain forms ------------------------------------------------------------------------------------------------
def _exponents(amax, emax):
    """floor(log2 amax) - emax of every block as it fits a scale byte; a block of zeros takes the smallest."""
    return torch.where(amax > 0, torch.frexp(amax)[1] - 1 - emax, -127).clamp(-127, 127)


def _blocks(x):
    """fp32 [rows, K] -> [rows, blocks, 32], the last block filled up with zeros."""
    rows, K = x.shape
    return torch.nn.functional.pad(x, (0, -K % BLOCK)).view(rows, -1, BLOCK)


def _mx_values(x, format):
    """The values that fp32 rows stand for after their conversion to MX rows (fp32, every one exact in bf16), and the
    blocks' scale bytes.  Blocks of finite values only."""
    emax, mbits, emin, top = FORMATS[format]
    b = _blocks(x)
    e = _exponents(b.abs().amax(dim=2, keepdim=True), emax)
    v = b.double() * _power(-e)
    grid = torch.frexp(v)[1].sub_(1).clamp_(min=emin) - mbits          # exponent of the step between neighbours
    v = (torch.round(v * _power(-grid)) * _power(grid)).clamp_(-top, top)           # ties to even
    v = (v * _power(e)).float()
    return v.view(x.size(0), -1)[:, :x.size(1)], e.squeeze(2) + 127


def _table(format, device):
    """What each code byte (E4M3) or nibble (E2M1) stands for, fp32."""
    n = torch.arange(16 if format == "fp4" else 256, device=device)
    mbits, ebits, bias = (1, 2, 1) if format == "fp4" else (3, 4, 7)
    m, e, s = n & ((1 << mbits) - 1), (n >> mbits) & ((1 << ebits) - 1), n >> (mbits + ebits)
    mant = m.float() / (1 << mbits)
    v = torch.where(e > 0, (1 + mant) * _power(e - bias), mant * 2.0 ** (1 - bias)).float()
    return torch.where(s > 0, -v, v)


def _decode(codes, scales, format):
    """MX rows (codes, scale bytes) -> fp32 [rows, padded K]."""
    table = _table(format, codes.device)
    if format == "fp4":
        v = table[torch.stack([codes & 15, codes >> 4], dim=2).view(codes.size(0), -1).int()]
    else:
        v = table[codes.int()]
    scale = _power(scales.long() - 127).float()
    return (v.view(codes.size(0), -1, BLOCK) * scale.unsqueeze(2)).view(codes.size(0), -1)


def _plain_quantise(s):
    return _mx_values(s["x"].float(), s["format"])[0].bfloat16()


def _plain_norm(s):
    x, residual = s["x"], s["residual"]
    h = x.float()
    if residual is not None:
        residual = (h + residual.float()).to(residual.dtype)
        h = residual.float()
    h = h.double()              # the 8-bit codes have borders: everything up to the one rounding in 64 bits
    r = torch.rsqrt(h.square().mean(dim=1, keepdim=True) + s["eps"])
    y = (h * r * s["weight"].double()).float()
    values = _mx_values(y, s["format"])[0].bfloat16()
    return {"values": values} if residual is None else {"values": values, "residual": residual}


def _plain_product(s):
    a = _decode(s["a_codes"], s["a_scales"], s["a"])
    b = _decode(s["b_codes"], s["b_scales"], "fp4")
    return (a @ b.t()).to(s["out"])


def _column(v, like):
    """A setting for all rows or one per row, as a 64-bit column."""
    return (v if torch.is_tensor(v) else torch.full((), v, device=like.device)).double().reshape(-1, 1)


def _plain_sample(s):
    x = s["logits"].double()                                           # sums have borders: 64 bits
    R, V = x.shape
    x = torch.where(torch.isnan(x), -math.inf, x)
    temperature, top_k = _column(s["temperature"], x), _column(s["top_k"], x)
    top_p, min_p = _column(s["top_p"], x), _column(s["min_p"], x)
    x, order = torch.sort(x, dim=1, descending=True, stable=True)      # ties: the lowest index first
    d = torch.where(x == x[:, :1], 0.0, (x - x[:, :1]) / temperature)
    rank = torch.arange(V, device=x.device)
    w = torch.where((x > -math.inf) & ((top_k <= 0) | (rank < top_k)), torch.exp(d), 0.0)
    before = torch.cumsum(w, dim=1) - w
    keep = ((top_p >= 1) | (before < top_p * w.sum(dim=1, keepdim=True))) & (w >= min_p.clamp(max=1.0)) & (w > 0)
    keep = keep | ((rank == 0) & (w > 0))
    w = torch.zeros_like(w).scatter_(1, order, torch.where(keep, w, 0.0))
    total = torch.cumsum(w, dim=1)
    u = (s["words"].long() & 0xFFFFFFFF).double().unsqueeze(1) / 4294967296.0
    token = (total <= u * total[:, -1:]).sum(dim=1)
    return torch.where(total[:, -1] > 0, token, -1).int()


# ---- the framework's calls ------------------------------------------------------------------------------------------
def _own(s):
    from nesgpu_amd.extensions import booleanOperations as ops
    if s["op"] == "quantise":
        return ops.mx_dequantize(ops.mx_quantize(s["x"], s["format"]))
    if s["op"] == "norm":
        rows, residual = ops.rms_norm_mx(s["x"], s["weight"], s["residual"], s["eps"], s["format"])
        values = ops.mx_dequantize(rows)
        return {"values": values} if residual is None else {"values": values, "residual": residual}
    if s["op"] == "product":
        a = ops.MXRows(s["a_codes"], s["a_scales"], s["K"], s["a"])
        b = ops.MXRows(s["b_codes"], s["b_scales"], s["K"], "fp4")
        return ops.mx_mm_nt(a, b, s["out"])
    return ops.sample_tokens_from_words(s["logits"], s["words"], s["temperature"], s["top_k"], s["top_p"], s["min_p"])


def run(state):
    if own:
        return _own(state)
    return {"quantise": _plain_quantise, "norm": _plain_norm, "product": _plain_product,
            "sample": _plain_sample}[state["op"]](state)


# ---- inputs ---------------------------------------------------------------------------------------------------------
def _activations(g, rows, K, device):
    """Rows as layers see them: normal values, a few columns that are larger throughout, rows of different size."""
    x = torch.randn((rows, K), generator=g, device=device)
    x *= torch.where(torch.rand((K,), generator=g, device=device) < 0.01, 20.0, 1.0)
    return x * torch.exp(0.5 * torch.randn((rows, 1), generator=g, device=device))


def _codes(x, format):
    """fp32 rows -> the code and scale bytes of MX rows, padded to whole steps, through the values they stand for."""
    rows, K = x.shape
    emax, mbits, emin, _ = FORMATS[format]
    x = torch.nn.functional.pad(x, (0, -K % STEP))
    v, scales = _mx_values(x, format)
    v = (v.view(rows, -1, BLOCK) * _power(127 - scales.unsqueeze(2))).view(rows, -1)
    e = torch.frexp(v.abs())[1] - 1
    normal = v.abs() >= 2.0 ** emin
    m = (v.abs() * _power(mbits - e.clamp(min=emin))).int()           # mantissa with its leading one where normal
    code = torch.where(normal, ((e - emin + 1) << mbits) + (m - (1 << mbits)), m)
    code = (code + (torch.signbit(v).int() << (3 if format == "fp4" else 7))).to(torch.uint8)
    if format == "fp4":
        code = code[:, 0::2] | (code[:, 1::2] << 4)
    return code.contiguous(), scales.to(torch.uint8).contiguous()


def prepare(case, seed):
    device = "cuda" if torch.cuda.is_available() else "cpu"
    g = torch.Generator(device=device)
    g.manual_seed(seed)
    s = {"op": case["op"]}
    if case["op"] == "quantise":
        s.update(x=_activations(g, case["rows"], case["K"], device).to(TYPES[case["type"]]), format=case["format"])
    elif case["op"] == "norm":
        rows, K = case["rows"], case["K"]
        x = _activations(g, rows, K, device)
        # a binary layer's sums: integers of about the square root of their number of terms
        x = torch.round(30.0 * x).int() if case["type"] == "int32" else x.to(TYPES[case["type"]])
        residual = None
        if case["residual"] != "none":
            size = 20.0 if case["type"] == "int32" else 3.0
            residual = (size * torch.randn((rows, K), generator=g, device=device)).to(TYPES[case["residual"]])
        weight = 1.0 + 0.2 * torch.randn((K,), generator=g, device=device)
        s.update(x=x, residual=residual, weight=weight.to(torch.float32 if residual is None else residual.dtype),
                 eps=1e-5, format=case["format"])
    elif case["op"] == "product":
        M, N, K = case["M"], case["N"], case["K"]
        s["a_codes"], s["a_scales"] = _codes(_activations(g, M, K, device), case["a"])
        s["b_codes"], s["b_scales"] = _codes(torch.randn((N, K), generator=g, device=device) / math.sqrt(K), "fp4")
        s.update(a=case["a"], out=TYPES[case["out"]], K=K)
    else:
        R, V = case["rows"], case["V"]
        x = 2.5 * torch.randn((R, V), generator=g, device=device)
        if V > 64:
            x[:, torch.randint(V, (V // 50,), generator=g, device=device)] = -math.inf      # tokens ruled out
        if case["type"] == "int32":
            x = torch.round(16.0 * x.clamp(min=-100.0)).int()
        elif R > 2:
            x[R // 2] = -math.inf                                      # a row that is left with nothing
        s["logits"] = x.to(TYPES[case["type"]])
        s["words"] = torch.randint(-2 ** 31, 2 ** 31, (R,), generator=g, device=device).int()
        for k in ("temperature", "top_k", "top_p", "min_p"):
            s[k] = case[k]
        if case["per_row"]:
            u = torch.rand((4, R), generator=g, device=device)
            s["temperature"] = case["temperature"] * (0.5 + u[0])
            s["top_k"] = (case["top_k"] * (0.5 + u[1])).int()
            s["top_p"] = torch.where(u[2] < 0.3, 1.0, case["top_p"] * (0.5 + 0.5 * u[2]))
            s["min_p"] = case["min_p"] * u[3]
    return s


_SIZE = {"fp32": 4, "fp16": 2, "bf16": 2, "int32": 4, "none": 0, "fp4": 0.5, "fp8": 1}


def _row_bytes(K, format):
    return math.ceil(K / STEP) * STEP * (_SIZE[format] + 1 / BLOCK)


def work(case):
    if case["op"] == "quantise":
        rows, K = case["rows"], case["K"]
        return {"bytes": rows * (K * (_SIZE[case["type"]] + 2) + 2 * _row_bytes(K, case["format"])), "flops": 4 * rows * K}
    if case["op"] == "norm":
        rows, K = case["rows"], case["K"]
        size = _SIZE[case["type"]] + 2 * _SIZE[case["residual"]] + 2
        return {"bytes": rows * (K * size + 2 * _row_bytes(K, case["format"])) + 4 * K, "flops": 9 * rows * K}
    if case["op"] == "product":
        M, N, K = case["M"], case["N"], case["K"]
        return {"bytes": M * _row_bytes(K, case["a"]) + N * _row_bytes(K, "fp4") + M * N * _SIZE[case["out"]],
                "flops": 2 * M * N * K}
    R, V = case["rows"], case["V"]
    return {"bytes": R * (V * _SIZE[case["type"]] + 8), "flops": 20 * R * V}


# ---- the definitions in 64 bits ---------------------------------------------------------------------------------------
def _exact_values(x, format):
    """float64 rows -> the float64 values of their MX form, from the definition: the nearest of the format's numbers."""
    rows, K = x.shape
    table = torch.tensor({"fp4": [0, .5, 1, 1.5, 2, 3, 4, 6],
                          "fp8": [m / 512 for m in range(8)] + [2.0 ** (e - 7) * (1 + m / 8) for e in range(1, 16)
                                                                for m in range(8) if (e, m) != (15, 7)]}[format],
                         dtype=torch.float64, device=x.device)
    b = torch.cat([x, x.new_zeros((rows, -K % BLOCK))], dim=1).reshape(rows, -1, BLOCK)
    amax = b.abs().max(dim=2, keepdim=True).values
    power = _power(torch.round(torch.log2(amax)).clamp(-1000, 1000))    # the power of two next to it, then the one below
    power = torch.where(power > amax, power / 2, power).clamp(min=2.0 ** (FORMATS[format][0] - 127))
    scale = power / 2.0 ** FORMATS[format][0]
    v = b / scale
    a = v.abs().contiguous()
    hi = torch.searchsorted(table, a).clamp(max=table.numel() - 1)      # first number not below
    lo = (hi - 1).clamp(min=0)
    up, down = table[hi] - a, a - table[lo]
    pick = torch.where((up < down) | ((up == down) & (hi % 2 == 0)), hi, lo)      # ties: the even code
    return (torch.sign(v) * table[pick] * scale).reshape(rows, -1)[:, :K]


def exact(case, seed):
    s = prepare(case, seed)
    if s["op"] == "quantise":
        return _exact_values(s["x"].double(), s["format"])
    if s["op"] == "norm":
        h, residual = s["x"].double(), s["residual"]
        if residual is not None:
            total = h + residual.double()
            h = total.to(residual.dtype).double()                       # the norm is of the stream as it is stored
        y = h * s["weight"].double() / torch.sqrt((h * h).sum(dim=1, keepdim=True) / h.size(1) + s["eps"])
        values = _exact_values(y.float().double(), s["format"])
        return {"values": values} if residual is None else {"values": values, "residual": total}
    if s["op"] == "product":
        b = _decode(s["b_codes"], s["b_scales"], "fp4").double()
        a = _decode(s["a_codes"], s["a_scales"], s["a"]).double()
        return a @ b.t()
    return None                                                         # token numbers: whole, compared for equality
