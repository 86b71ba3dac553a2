"""Plain numpy restatement, in 64 bits, of the microscaled rows, the norm that writes them, their product and the token
sampler (include/nesbin.h), for the tests.  Written from the definitions: nearest code by search over the format's
values, sums by ``math.fsum`` or exact fractions."""
import math
from fractions import Fraction

import numpy as np

FORMATS = ("fp4", "fp8")
EMAX = {"fp4": 2, "fp8": 8}


def table(format):
    """Magnitudes of the codes in their order."""
    if format == "fp4":
        return np.array([0, 0.5, 1, 1.5, 2, 3, 4, 6])
    sub = [m * 2.0 ** -9 for m in range(8)]
    normal = [2.0 ** (e - 7) * (1 + m / 8) for e in range(1, 16) for m in range(8)]
    return np.array(sub + normal[:-1])                        # the last code is NaN


def padded(K):
    return -(-K // 128) * 128


def _floor_log2(v):
    return math.frexp(v)[1] - 1


def quantize(x, format):
    """x float64 [rows, K] -> (codes uint8, scales uint8) with padded rows."""
    rows, K = x.shape
    Kp = padded(K)
    t = table(format)
    buf = np.zeros((rows, Kp))
    buf[:, :K] = x
    codes = np.zeros((rows, Kp), dtype=np.uint8)
    scales = np.zeros((rows, Kp // 32), dtype=np.uint8)
    for r in range(rows):
        for b in range(Kp // 32):
            v = buf[r, 32 * b:32 * b + 32]
            if not np.all(np.isfinite(v)):
                scales[r, b] = 255
                continue
            amax = np.abs(v).max()
            s = 0 if amax == 0 else max(_floor_log2(amax) - EMAX[format] + 127, 0)
            scales[r, b] = s
            q = np.ldexp(np.abs(v), 127 - s)                  # exact in 64 bits
            d = np.abs(q[:, None] - t[None, :])
            best = d.min(axis=1)
            for i in range(32):
                ties = np.nonzero(d[i] == best[i])[0]
                c = next((k for k in ties if k % 2 == 0), ties[0])      # halfway: the even code
                sign = 1 if math.copysign(1.0, v[i]) < 0 else 0
                codes[r, 32 * b + i] = c + sign * (8 if format == "fp4" else 128)
    if format == "fp4":
        codes = codes[:, 0::2] | (codes[:, 1::2] << 4)
    return codes, scales


def decode(codes, scales, K, format):
    """-> float64 [rows, K]"""
    t = table(format)
    if format == "fp4":
        c = np.stack([codes & 15, codes >> 4], axis=2).reshape(codes.shape[0], -1).astype(int)
        v = np.where(c & 8, -1.0, 1.0) * t[c & 7]
    else:
        c = codes.astype(int)
        full = np.append(t, np.nan)
        v = np.where(c & 128, -1.0, 1.0) * full[c & 127]
    s = np.repeat(scales.astype(int), 32, axis=1)
    v = np.ldexp(v, s - 127)
    v[s == 255] = np.nan
    return v[:, :K]


def rms_norm(x, weight, residual, eps, round_to):
    """x, residual as float64 arrays of exactly representable values -> (y as float32, new residual float64 or None).
    ``round_to`` rounds float32 to the residual's type."""
    new = None
    h = x.astype(np.float32)
    if residual is not None:
        new = round_to(h + residual.astype(np.float32)).astype(np.float64)
        h = new
    h = h.astype(np.float64)
    y = np.empty(h.shape, dtype=np.float32)
    for i in range(h.shape[0]):
        r = 1.0 / math.sqrt(math.fsum(float(v) * float(v) for v in h[i]) / h.shape[1] + eps)
        y[i] = ((h[i] * r) * weight).astype(np.float32)
    return y, new


def mm_nt(a, b):
    """float64 product and the sum of the products' magnitudes."""
    return a @ b.T, np.abs(a) @ np.abs(b).T


def sample(logits, word, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """One row (float64 logits) -> token.  Weights are whole multiples of 2^-f, as the format of the operator says: f =
    min(51, 61 - ceil(log2 V)) fraction bits; those below half a unit are 0.  (All of a row's zeros together stand for less
    than V 2^-(f+1) of the largest weight: 2^-28 at V = 131072 and at V <= 2^14 less than 2^-32, which only a word of 0 could
    ask for.)  Settings are float32, as a tensor of them is."""
    temperature, top_p, min_p = (float(np.float32(v)) for v in (temperature, top_p, min_p))
    x = [float(v) for v in logits]
    live = [i for i, v in enumerate(x) if v == v and v != -math.inf]
    if not live:
        return -1
    order = sorted(live, key=lambda i: (-x[i], i))
    top = x[order[0]]
    if not temperature > 0:
        return order[0]

    unit = 2 ** min(51, 61 - math.ceil(math.log2(len(x))))

    def weight(i):
        if x[i] == top:
            return Fraction(1)
        return Fraction(round(math.exp((x[i] - top) / temperature) * unit), unit)

    w = {i: weight(i) for i in order}
    keep = order[:top_k] if top_k > 0 else order
    if top_p < 1:
        target = Fraction(top_p) * sum(w[i] for i in keep)
        total, n = Fraction(0), 0
        while n == 0 or total < target:
            total += w[keep[n]]
            n += 1
        keep = keep[:n]
    keep = [i for i in keep if w[i] >= min(Fraction(min_p), Fraction(1))]
    total = sum(w[i] for i in keep)
    bar = Fraction(int(word), 2 ** 32) * total
    acc = Fraction(0)
    for i in sorted(keep):
        acc += w[i]
        if acc > bar:
            return i
    raise AssertionError("unreachable: the word is below 2**32")


def token_within(logits, word, token, slack, temperature=1.0):
    """Whether a row's token, nothing cut off, is the drawn one with real weights and borders moved by up to ``slack`` of the
    largest weight."""
    x = np.asarray(logits, dtype=np.float64)
    temperature = float(np.float32(temperature))
    w = np.where(x == x.max(), 1.0, np.exp((x - x.max()) / temperature))
    before, after, total = math.fsum(w[:token]), math.fsum(w[:token + 1]), math.fsum(w)
    return w[token] > 0 and before - slack <= int(word) / 2 ** 32 * total <= after + slack
