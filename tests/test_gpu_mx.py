"""Microscaled rows, the norm that writes them, their product and the token sampler on the GPU, against the 64-bit
restatement in oracle/mx.py."""
import numpy as np
import pytest
import torch

from oracle import mx as O

pytestmark = pytest.mark.gpu
DTYPES = [torch.float32, torch.float16, torch.bfloat16]
IDS = ["f32", "f16", "bf16"]


@pytest.fixture(scope="module")
def ops():
    assert torch.cuda.is_available()
    from nesgpu_amd.extensions import booleanOperations
    return booleanOperations


def host(t):
    return t.double().cpu().numpy()


def rows_of(shape, seed, dtype, spread=3.0):
    """Values of very different size per block, blocks of zeros, exact halfway points, signed zeros."""
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(shape, generator=g)
    x *= torch.exp2((torch.randn(shape[0], -(-shape[1] // 32), generator=g) * spread).round()).repeat_interleave(32, 1)[:, :shape[1]]
    x[:, 5::7] = torch.round(x[:, 5::7] * 4) / 4
    if shape[1] > 70:
        x[0, 32:64] = 0.0
        x[0, 40] = -0.0
    return x.to(dtype)


def as_mx(ops, codes, scales, K, format):
    return ops.MXRows(torch.from_numpy(codes).cuda(), torch.from_numpy(scales).cuda(), K, format)


# ---- conversion -------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("format", O.FORMATS)
@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("shape", [(1, 1), (3, 31), (2, 32), (5, 33), (4, 128), (3, 136), (3, 129), (7, 1000), (33, 256)])
def test_quantize(ops, shape, dtype, format):
    x = rows_of(shape, 11 * shape[1] + shape[0], dtype)
    want_c, want_s = O.quantize(host(x), format)
    got = ops.mx_quantize(x.cuda(), format)
    assert np.array_equal(got.scales.cpu().numpy(), want_s)
    assert np.array_equal(got.codes.cpu().numpy(), want_c)
    assert got.shape == shape
    back = ops.mx_dequantize(got, torch.float32)
    assert np.array_equal(host(back), O.decode(want_c, want_s, shape[1], format))


@pytest.mark.parametrize("format", O.FORMATS)
def test_quantize_extremes(ops, format):
    """Blocks at both ends of float32, subnormal ones, and blocks with an infinity or NaN."""
    x = torch.randn(8, 128, generator=torch.Generator().manual_seed(3))
    x[0] *= 1e-38
    x[1] *= 1e-42
    x[2] = 2.0 ** -149
    x[3, :64] = torch.finfo(torch.float32).max
    x[3, 64:] *= 2.0 ** 125
    x[4, 3] = float("inf")
    x[5, 40] = float("nan")
    x[6, 127] = -float("inf")
    x[7, :32] = 0
    want_c, want_s = O.quantize(x.double().numpy(), format)
    got = ops.mx_quantize(x.cuda(), format)
    assert np.array_equal(got.scales.cpu().numpy(), want_s)
    assert np.array_equal(got.codes.cpu().numpy(), want_c)
    back = host(ops.mx_dequantize(got, torch.float32))
    assert np.array_equal(back, O.decode(want_c, want_s, 128, format), equal_nan=True)
    assert np.isnan(back[4, :32]).all() and np.isfinite(back[4, 32:]).all()


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("format", O.FORMATS)
def test_dequantize_every_code_and_scale(ops, format, dtype):
    n = 256 if format == "fp8" else 128
    codes = np.tile(np.arange(n, dtype=np.uint8) if format == "fp8" else np.arange(64, dtype=np.uint8), (256, 1))
    if format == "fp4":
        codes = np.concatenate([codes, codes + 64, codes + 128, codes + 192], axis=1)
    K = codes.shape[1] * (2 if format == "fp4" else 1)
    scales = np.repeat(np.arange(256, dtype=np.uint8)[:, None], K // 32, axis=1)
    want = torch.from_numpy(O.decode(codes, scales, K, format).astype(np.float32)).to(dtype)
    got = ops.mx_dequantize(as_mx(ops, codes, scales, K, format), dtype).cpu()
    assert torch.equal(torch.nan_to_num(got, nan=12345.0), torch.nan_to_num(want, nan=12345.0))
    assert torch.equal(torch.isnan(got), torch.isnan(want))


def test_quantize_from_unaligned_storage_and_many_rows(ops):
    flat = torch.randn(1 + 300 * 64, generator=torch.Generator().manual_seed(9)).bfloat16().cuda()
    x = flat[1:].view(300, 64)                              # contiguous, two bytes off
    want_c, want_s = O.quantize(host(x), "fp4")
    got = ops.mx_quantize(x, "fp4")
    assert np.array_equal(got.codes.cpu().numpy(), want_c) and np.array_equal(got.scales.cpu().numpy(), want_s)


# ---- norm -------------------------------------------------------------------------------------------------------------
def _rounder(dtype):
    return lambda a: torch.from_numpy(np.ascontiguousarray(a)).to(dtype).float().numpy()


NORM_TYPES = [(torch.float32, None), (torch.float16, None), (torch.bfloat16, None), (torch.int32, None),
              (torch.float32, torch.float32), (torch.float16, torch.float16), (torch.bfloat16, torch.bfloat16),
              (torch.int32, torch.float32), (torch.int32, torch.float16), (torch.int32, torch.bfloat16)]


def norm_inputs(shape, x_type, r_type, seed):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(shape, generator=g) * torch.exp(torch.randn(shape[0], 1, generator=g))
    x = (x * 50).round().int() if x_type == torch.int32 else x.to(x_type)
    r = None if r_type is None else (torch.randn(shape, generator=g) * (40 if x_type == torch.int32 else 1)).to(r_type)
    w = 1 + 0.3 * torch.randn(shape[1], generator=g)
    return x, r, w.to(r_type or (torch.float32 if x_type == torch.int32 else x_type))


@pytest.mark.parametrize("types", NORM_TYPES, ids=lambda t: "-".join(str(d).replace("torch.", "") for d in t))
@pytest.mark.parametrize("shape", [(1, 1), (5, 24), (3, 77), (9, 512), (2, 520), (4, 2048), (3, 3000), (2, 5000), (1, 8192),
                                   (2, 9001), (2, 20000), (1, 40000)])
def test_norm(ops, shape, types):
    x, r, w = norm_inputs(shape, *types, seed=shape[1])
    eps = 1e-5
    y, new = O.rms_norm(host(x), host(w), None if r is None else host(r), eps, _rounder(types[1]) if r is not None else None)
    for format in O.FORMATS:
        if shape[0] * shape[1] > 20000 and format == "fp4":
            continue
        rows, got_r = ops.rms_norm_mx(x.cuda(), w.cuda(), None if r is None else r.cuda(), eps, format)
        if r is None:
            assert got_r is None
        else:
            assert got_r.dtype == r.dtype and np.array_equal(host(got_r), new)
        # every step before the codes is in 64 bits with one rounding to fp32: the codes themselves are equal
        want_c, want_s = O.quantize(y.astype(np.float64), format)
        assert np.array_equal(rows.scales.cpu().numpy(), want_s)
        assert np.array_equal(rows.codes.cpu().numpy(), want_c)


def test_norm_rows_of_zeros_nan_and_infinity(ops):
    x = torch.randn(4, 256, generator=torch.Generator().manual_seed(4))
    x[1] = 0
    x[2, 7] = float("nan")
    x[3, 9] = float("inf")
    w = torch.ones(256)
    rows, _ = ops.rms_norm_mx(x.cuda(), w.cuda())
    v = host(ops.mx_dequantize(rows, torch.float32))
    assert np.isfinite(v[0]).all() and np.array_equal(v[1], np.zeros(256)) and np.isnan(v[2]).all()
    assert np.isnan(v[3, :32]).all() and np.array_equal(v[3, 32:], np.zeros(224))       # inf * 0 and finite * 0


def test_norm_weight_of_another_type(ops):
    x, r, _ = norm_inputs((3, 300), torch.bfloat16, torch.bfloat16, 5)
    w = torch.rand(300, generator=torch.Generator().manual_seed(1))
    for dt in DTYPES:
        wt = w.to(dt)
        y, _ = O.rms_norm(host(x), host(wt), host(r), 1e-6, _rounder(torch.bfloat16))
        rows, _ = ops.rms_norm_mx(x.cuda(), wt.cuda(), r.cuda())
        assert np.array_equal(rows.codes.cpu().numpy(), O.quantize(y.astype(np.float64), "fp8")[0])


# ---- product ----------------------------------------------------------------------------------------------------------
def product_case(M, N, K, a_format, seed):
    g = np.random.default_rng(seed)
    a = g.standard_normal((M, K)) * np.exp2(g.integers(-6, 7, (M, 1))) * np.where(g.random(K) < 0.05, 20, 1)
    b = g.standard_normal((N, K)) / 8
    qa = ref_rows(a, a_format)
    qb = ref_rows(b, "fp4")
    return qa, qb


def ref_rows(x, format):
    """MX rows of float64 values, through torch for speed (the conversion itself is tested above)."""
    t = O.table(format)
    rows, K = x.shape
    Kp = O.padded(K)
    v = np.zeros((rows, Kp // 32, 32))
    v.reshape(rows, Kp)[:, :K] = x
    amax = np.abs(v).max(axis=2)
    e = np.where(amax > 0, np.frexp(np.where(amax > 0, amax, 1))[1] - 1 - O.EMAX[format], -127).clip(-127, 127)
    q = np.ldexp(np.abs(v), -e[:, :, None]).reshape(rows, Kp)
    hi = np.searchsorted(t, q).clip(1, len(t) - 1)
    c = np.where(t[hi] - q < q - t[hi - 1], hi, hi - 1)
    c = (c + np.signbit(v.reshape(rows, Kp)) * (8 if format == "fp4" else 128)).astype(np.uint8)
    if format == "fp4":
        c = c[:, 0::2] | (c[:, 1::2] << 4)
    return np.ascontiguousarray(c), (e + 127).astype(np.uint8)


SHAPES = [(1, 1, 1), (1, 32, 128), (3, 5, 33), (16, 16, 256), (17, 33, 640), (1, 1000, 4096), (2, 640, 1111), (100, 10, 2048),
          (64, 64, 512), (65, 130, 1000), (128, 256, 384), (200, 300, 129), (257, 513, 1280), (600, 520, 2304), (1, 7, 16384),
          (5, 4099, 512), (300, 10, 8192), (1030, 70, 130)]


@pytest.mark.parametrize("a_format", O.FORMATS)
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "x".join(map(str, s)))
def test_product(ops, shape, a_format):
    M, N, K = shape
    (ac, as_), (bc, bs) = product_case(M, N, K, a_format, M + 3 * N + K)
    want, size = O.mm_nt(O.decode(ac, as_, K, a_format), O.decode(bc, bs, K, "fp4"))
    A, B = as_mx(ops, ac, as_, K, a_format), as_mx(ops, bc, bs, K, "fp4")
    # products are exact and every partial sum is at most `size`: one rounding (allowed to be a truncation, 2^-23) per
    # addition into an accumulator; a step of 128 positions adds its groups of 8, and partial sums are joined at the end
    adds = 2 * 17 * (O.padded(K) // 128) + 64
    for dtype in DTYPES:
        got = host(ops.mx_mm_nt(A, B, dtype))
        half = 0.0 if dtype == torch.float32 else torch.finfo(dtype).eps / 2
        bound = adds * 2.0 ** -23 * size + half * np.abs(want) + (2.0 ** -25 if dtype == torch.float16 else 0)
        if dtype == torch.float16:
            ok = np.abs(want) < 65000
            assert np.all(np.abs(got - want)[ok] <= bound[ok] * (1 + half))
        else:
            assert np.all(np.abs(got - want) <= bound * (1 + half))


# larger sizes (which tile a size takes goes by the format too: see TILES for a list that has every tile of both), K of one step, of
# whole groups of four steps and of odd ones
LARGE = [(8100, 8191, 1100), (8192, 8192, 128), (8000, 8300, 512), (3000, 3000, 700), (2048, 2100, 1536), (2049, 2100, 200),
         (2000, 1100, 900), (1030, 1025, 2048), (1000, 1000, 1000), (20, 33000, 640), (7, 40000, 1150), (40, 8000, 3000),
         (1, 3000, 6000), (2000, 20, 2100), (3, 129, 33000)]


@pytest.mark.parametrize("a_format", O.FORMATS)
@pytest.mark.parametrize("shape", LARGE, ids=lambda s: "x".join(map(str, s)))
def test_product_of_large_sizes(ops, shape, a_format):
    M, N, K = shape
    g = torch.Generator(device="cuda").manual_seed(M + N + K)
    a = torch.randn(M, K, generator=g, device="cuda") * torch.exp2(torch.randint(-6, 7, (M, 1), generator=g, device="cuda"))
    a[:, ::19] *= 20
    A = ops.mx_quantize(a, a_format)
    B = ops.mx_quantize(torch.randn(N, K, generator=g, device="cuda") / 8, "fp4")
    a, b = ops.mx_dequantize(A, torch.float32).double(), ops.mx_dequantize(B, torch.float32).double()
    want, size = a @ b.t(), a.abs() @ b.abs().t()
    adds = 2 * 17 * (O.padded(K) // 128) + 64                # as in test_product
    for dtype in (torch.float32, torch.bfloat16):
        got = ops.mx_mm_nt(A, B, dtype).double()
        half = 0.0 if dtype == torch.float32 else torch.finfo(dtype).eps / 2
        err = (got - want).abs() - (adds * 2.0 ** -23 * size + half * want.abs()) * (1 + half)
        assert float(err.max()) <= 0


@pytest.mark.parametrize("a_format", O.FORMATS)
@pytest.mark.parametrize("shape", [(1, 64, 512), (70, 90, 256), (300, 300, 512)], ids=lambda s: "x".join(map(str, s)))
def test_product_of_small_whole_numbers_is_exact(ops, shape, a_format):
    M, N, K = shape
    g = np.random.default_rng(7)
    a, b = g.integers(-3, 4, (M, K)).astype(float), g.integers(-2, 3, (N, K)).astype(float)
    A, B = as_mx(ops, *ref_rows(a, a_format), K, a_format), as_mx(ops, *ref_rows(b, "fp4"), K, "fp4")
    assert np.array_equal(host(ops.mx_mm_nt(A, B)), a @ b.T)


@pytest.mark.parametrize("shape", [(1, 32, 512), (40, 40, 256), (260, 300, 512)], ids=lambda s: "x".join(map(str, s)))
def test_product_keeps_small_values_beside_large_ones(ops, shape):
    """E4M3 neighbours 17 binades apart whose large products cancel: what is left is the small ones' exact sum."""
    M, N, K = shape
    a = np.zeros((M, K))
    a[:, 0::8], a[:, 1::8] = 256.0, -256.0
    g = np.random.default_rng(2)
    a[:, 2::8] = g.integers(1, 8, (M, K // 8)) * 2.0 ** -9
    a[:, 5::8] = g.integers(8, 16, (M, K // 8)) * 2.0 ** -9
    b = np.ones((N, K))
    b[:, 2::8] = g.choice([0.5, 1.5, -3.0], (N, K // 8))
    ac, as_ = ref_rows(a, "fp8")
    assert np.all(as_ == 127)
    B = as_mx(ops, *ref_rows(b, "fp4"), K, "fp4")
    got = host(ops.mx_mm_nt(as_mx(ops, ac, as_, K, "fp8"), B))
    # the running sum passes through 256: multiples of 2^-10 below 2^9 are 19 bits, exact in fp32
    assert np.array_equal(got, a @ b.T)


def test_product_of_nan_blocks_and_extreme_scales(ops):
    K = 256
    (ac, as_), (bc, bs) = product_case(20, 24, K, "fp8", 1)
    as_[3, 2] = 255
    bs[5, 7] = 255
    ac[9, 100] = 0x7F
    got = host(ops.mx_mm_nt(as_mx(ops, ac, as_, K, "fp8"), as_mx(ops, bc, bs, K, "fp4")))
    nan = np.zeros((20, 24), dtype=bool)
    nan[3] = nan[9] = True
    nan[:, 5] = True
    assert np.array_equal(np.isnan(got), nan)
    # scales that leave float32's range by themselves and meet inside it
    a, b = np.ones((4, 128)), np.ones((4, 128))
    for fmt in O.FORMATS:
        (ac, as_), (bc, bs) = ref_rows(a, fmt), ref_rows(b, "fp4")
        as_[:] = 250
        bs[:] = 4
        want = O.decode(ac, as_, 128, fmt) @ O.decode(bc, bs, 128, "fp4").T
        assert np.array_equal(host(ops.mx_mm_nt(as_mx(ops, ac, as_, 128, fmt), as_mx(ops, bc, bs, 128, "fp4"))), want)


# ---- tokens -----------------------------------------------------------------------------------------------------------
def check_tokens(ops, x, words, **kw):
    R = x.shape[0]
    args = {k: (torch.tensor(v, dtype=torch.int32 if k == "top_k" else torch.float32).cuda() if isinstance(v, list) else v)
            for k, v in kw.items()}
    got = ops.sample_tokens_from_words(x.cuda(), words.cuda(), **args).cpu().tolist()
    xs = host(x)
    w = (words.long() & 0xFFFFFFFF).tolist()
    f32 = {k: ([float(np.float32(e)) if k != "top_k" else e for e in v] if isinstance(v, list) else v) for k, v in kw.items()}
    want = [O.sample(xs[r], w[r], **{k: (v[r] if isinstance(v, list) else v) for k, v in f32.items()}) for r in range(R)]
    assert got == want


def words_of(R, seed):
    w = torch.randint(-2 ** 31, 2 ** 31, (R,), generator=torch.Generator().manual_seed(seed)).int()
    if R > 3:
        w[0], w[1] = 0, -1                                  # the smallest and the largest word
    return w


SETTINGS = [dict(), dict(temperature=0.7), dict(top_k=1), dict(top_k=7), dict(top_p=0.8), dict(top_p=0.3, temperature=1.5),
            dict(min_p=0.1), dict(top_k=20, top_p=0.9, min_p=0.02, temperature=0.9), dict(temperature=0.0), dict(top_p=0.0),
            dict(min_p=1.0), dict(min_p=5.0), dict(top_k=10 ** 9, top_p=2.0), dict(temperature=100.0, top_p=0.999)]


@pytest.mark.parametrize("dtype", DTYPES + [torch.int32], ids=IDS + ["i32"])
@pytest.mark.parametrize("V", [1, 2, 10, 63, 64, 65, 500, 513, 2048, 2049, 5000])
def test_tokens(ops, V, dtype):
    g = torch.Generator().manual_seed(V)
    R = 12 if V < 1000 else 5
    x = torch.randn(R, V, generator=g) * 2.5
    x = (x * 3).round().int() if dtype == torch.int32 else x.to(dtype)
    if dtype != torch.int32 and V > 4:
        x[:, ::5] = -float("inf")
        x[2, 1::3] = float("nan")
        x[3] = -float("inf")
    for n, kw in enumerate(SETTINGS):
        check_tokens(ops, x, words_of(R, n), **kw)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.int32], ids=["bf16", "i32"])
def test_tokens_of_long_rows(ops, dtype):
    g = torch.Generator().manual_seed(77)
    for V in (16384, 16385, 40001, 131072):
        x = torch.randn(2, V, generator=g) * 2.5
        x = (x * 20).round().int() if dtype == torch.int32 else x.to(dtype)
        for n, kw in enumerate([dict(temperature=10.0 if dtype == torch.int32 else 1.0, top_p=0.9), dict(top_k=50),
                                dict(top_k=5000, top_p=0.95, min_p=1e-4, temperature=1.3), dict()]):
            check_tokens(ops, x, words_of(2, n), **kw)


def test_tokens_with_settings_per_row(ops):
    g = torch.Generator().manual_seed(5)
    R, V = 40, 700
    x = torch.randn(R, V, generator=g) * 3
    kw = dict(temperature=(torch.rand(R, generator=g) * 2).tolist(), top_k=torch.randint(-1, 60, (R,), generator=g).tolist(),
              top_p=(torch.rand(R, generator=g) * 1.2).tolist(), min_p=(torch.rand(R, generator=g) * 0.2).tolist())
    kw["temperature"][4] = 0.0
    kw["temperature"][5] = -1.0
    check_tokens(ops, x, words_of(R, 8), **kw)


@pytest.mark.parametrize("V", [40, 3000, 40000])
def test_tokens_of_equal_entries(ops, V):
    """Every border falls among equal entries: ties are kept by index, sums of equal weights are exact."""
    for dtype in (torch.float32, torch.float16, torch.int32):
        x = torch.zeros(6, V)
        x[2, : V // 2] = -1.0
        x[3, V // 2] = -0.0
        x = x.to(dtype)
        for kw in (dict(top_k=3), dict(top_p=0.5), dict(top_k=V // 2, top_p=0.5), dict(), dict(temperature=0.0)):
            check_tokens(ops, x, words_of(6, 1), **kw)


def test_tokens_with_infinities_and_extremes(ops):
    inf = float("inf")
    x = torch.tensor([[0.0, inf, 1.0, inf], [-inf, -inf, -inf, -inf], [-inf, 3e38, -3e38, 3e38], [float("nan"), -inf, -5.0, inf],
                      [float("nan")] * 4, [1e-45, 0.0, -0.0, -1e-45]])
    for kw in (dict(), dict(top_k=1), dict(top_p=0.4), dict(temperature=0.0), dict(temperature=float("inf")),
               dict(temperature=1e-30), dict(min_p=0.5), dict(temperature=1e30, top_k=2)):
        if kw.get("temperature") == inf:
            got = ops.sample_tokens_from_words(x.cuda(), words_of(6, 2).cuda(), **kw).cpu()
            assert got[1] == -1 and got[4] == -1 and (got[[0, 2, 3, 5]] >= 0).all()
            continue
        check_tokens(ops, x, words_of(6, 2), **kw)
    big = torch.tensor([[-2 ** 31, 2 ** 31 - 1, 0, 2 ** 31 - 1], [-2 ** 31] * 4, [-2 ** 31, -2 ** 31 + 1, 7, 8]], dtype=torch.int32)
    for kw in (dict(), dict(top_k=3), dict(top_p=0.9, temperature=1e9), dict(temperature=0.0)):
        check_tokens(ops, big, words_of(3, 3), **kw)


def test_tokens_follow_their_weights(ops):
    """Over evenly spread words every token comes as often as its weight says, to one word."""
    p = np.array([0.4, 0.3, 0.2, 0.05, 0.05])
    n = 4096
    x = torch.tensor(np.log(p), dtype=torch.float32).repeat(n, 1)
    words = ((torch.arange(n, dtype=torch.int64) << 20) + (1 << 19)).to(torch.uint32)
    got = ops.sample_tokens_from_words(x.cuda(), words.cuda()).cpu()
    assert np.all(np.abs(np.bincount(got.numpy(), minlength=5) - p * n) <= 1.01)


# ---- refusals and the run of them together ------------------------------------------------------------------------------
def test_refusals(ops):
    x = torch.zeros(4, 64, device="cuda")
    w = torch.zeros(4, dtype=torch.int32, device="cuda")
    with pytest.raises(RuntimeError, match="contiguous"):
        ops.mx_quantize(x[:, ::2])
    with pytest.raises(TypeError):
        ops.mx_quantize(x.double())
    with pytest.raises(ValueError):
        ops.mx_quantize(x, "fp6")
    with pytest.raises(AssertionError):
        ops.rms_norm_mx(x, torch.ones(63, device="cuda"))
    with pytest.raises(TypeError):
        ops.rms_norm_mx(x, torch.ones(64, device="cuda"), x.half())
    with pytest.raises(ValueError):
        ops.rms_norm_mx(x, torch.ones(64, device="cuda"), eps=-1.0)
    q4, q8 = ops.mx_quantize(x), ops.mx_quantize(x, "fp8")
    with pytest.raises(NotImplementedError):
        ops.mx_mm_nt(q4, q8)
    with pytest.raises(AssertionError):
        ops.mx_mm_nt(q4, ops.mx_quantize(x[:, :32].contiguous()))
    with pytest.raises(TypeError):
        ops.mx_mm_nt(q4, q4, torch.float64)
    with pytest.raises(AssertionError):
        ops.MXRows(q4.codes, q4.scales, 200)
    with pytest.raises(AssertionError):
        ops.sample_tokens_from_words(x, w[:3])
    with pytest.raises(TypeError):
        ops.sample_tokens_from_words(x, w.long())
    with pytest.raises(TypeError):
        ops.sample_tokens_from_words(x, w, temperature=torch.ones(4, device="cuda", dtype=torch.float64))
    with pytest.raises(ValueError):
        ops.sample_tokens_from_words(x, w, top_p=float("nan"))
    with pytest.raises(RuntimeError, match="at most"):
        ops.sample_tokens_from_words(torch.zeros(1, (1 << 20) + 1, device="cuda"), w[:1].clone())


def test_empty_inputs(ops):
    e = torch.zeros(0, 64, device="cuda")
    q = ops.mx_quantize(e)
    assert q.shape == (0, 64) and ops.mx_dequantize(q).shape == (0, 64)
    assert ops.mx_mm_nt(q, ops.mx_quantize(torch.ones(3, 64, device="cuda"))).shape == (0, 3)
    z = ops.mx_quantize(torch.zeros(3, 0, device="cuda"))
    assert torch.equal(ops.mx_mm_nt(z, z), torch.zeros(3, 3, device="cuda"))
    assert ops.rms_norm_mx(e, torch.ones(64, device="cuda"), e)[1].shape == (0, 64)
    assert ops.sample_tokens_from_words(e, torch.zeros(0, dtype=torch.int32, device="cuda")).shape == (0,)


def head(ops, act, stream, gain, weights, words, **kw):
    rows, stream = ops.rms_norm_mx(act, gain, stream, eps=1e-5)
    logits = ops.mx_mm_nt(rows, weights, torch.float32)
    return ops.sample_tokens_from_words(logits, words, **kw), stream, logits


def test_from_binary_layer_to_token(ops):
    """A binary layer's int32 activations and a residual stream -> norm -> readout -> a class per member, each step against
    the oracle on the step's own input."""
    from nesgpu_amd.modules import binary
    D, K, N = 96, 512, 37
    torch.manual_seed(3)
    layer = binary.BinarizedLinear(256, K, D, threshold=False)
    with torch.no_grad():
        layer.weight.copy_(torch.randn(K, 256))
    model = binary.PerturbedModel(layer, D)
    model.set_seed(5)
    model.set_noise(1.0)
    bits = torch.rand(D, 256, device="cuda") < 0.5
    act = model.forward(bits)
    assert act.dtype == torch.int32 and tuple(act.shape) == (D, K)
    stream = (torch.randn(D, K, device="cuda") * 10).half()
    gain = 1 + 0.1 * torch.randn(K, device="cuda")
    weights = ops.mx_quantize(torch.randn(N, K, device="cuda"), "fp4")
    words = ops.philox_words(D, 11)
    kw = dict(temperature=8.0, top_k=20, top_p=0.9)
    token, new, logits = head(ops, act, stream, gain, weights, words, **kw)
    y, want_new = O.rms_norm(host(act), host(gain), host(stream), 1e-5, _rounder(torch.float16))
    assert np.array_equal(host(new), want_new)
    qc, qs = O.quantize(y.astype(np.float64), "fp8")
    a = O.decode(qc, qs, K, "fp8")
    b = O.decode(weights.codes.cpu().numpy(), weights.scales.cpu().numpy(), K, "fp4")
    want, size = O.mm_nt(a, b)
    assert np.all(np.abs(host(logits) - want) <= (2 * 17 * 4 + 64) * 2.0 ** -23 * size)
    w = (words.cpu().to(torch.int64) & 0xFFFFFFFF).tolist()
    assert token.cpu().tolist() == [O.sample(host(logits)[d], w[d], **kw) for d in range(D)]


def test_captured_and_on_another_stream(ops):
    """The run of them in a graph, replayed on new inputs with eager work between, equals the eager run; so does a run on a
    side stream."""
    D, K, N = 40, 300, 5000
    g = torch.Generator(device="cuda").manual_seed(1)
    gain = torch.ones(K, device="cuda")
    weights = ops.mx_quantize(torch.randn(N, K, generator=g, device="cuda"), "fp4")
    kw = dict(temperature=2.0, top_p=0.9)

    def inputs():
        return (torch.randint(-200, 200, (D, K), generator=g, device="cuda").int(),
                torch.randn(D, K, generator=g, device="cuda").bfloat16(),
                torch.randint(-2 ** 31, 2 ** 31, (D,), generator=g, device="cuda").int())

    act, stream, words = inputs()
    head(ops, act, stream, gain, weights, words, **kw)
    torch.cuda.synchronize()
    graphs = []
    for _ in range(2):                                       # two graphs, replayed in turn
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = head(ops, act, stream, gain, weights, words, **kw)
        graphs.append((graph, out))
    for k in range(4):
        new = inputs()
        for t, n in zip((act, stream, words), new):
            t.copy_(n)
        want = head(ops, *new[:2], gain, weights, new[2], **kw)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            other = head(ops, *new[:2], gain, weights, new[2], **kw)
        torch.cuda.current_stream().wait_stream(side)
        graph, out = graphs[k % 2]
        graph.replay()
        torch.cuda.synchronize()
        for a, b, c in zip(want, out, other):
            assert torch.equal(a, b) and torch.equal(a, c)


# products whose tiles are made of fewer rows so that every CU has one, whole chunks and odd steps, a row to every side
FEW = [(1001, 10, 16000), (16, 1000, 2100), (15, 1001, 16384), (1, 1024, 512), (64, 500, 640), (1000, 1, 900), (5, 7, 50000),
       (250, 13, 700), (120, 33, 1300), (600, 3, 128), (3, 2000, 129), (63, 65, 4096)]


@pytest.mark.parametrize("a_format", O.FORMATS)
@pytest.mark.parametrize("shape", FEW, ids=lambda s: "x".join(map(str, s)))
def test_product_of_few_rows(ops, shape, a_format):
    M, N, K = shape
    g = torch.Generator(device="cuda").manual_seed(M + N + K)
    a = torch.randn(M, K, generator=g, device="cuda") * torch.exp2(torch.randint(-6, 7, (M, 1), generator=g, device="cuda"))
    b = torch.randn(N, K, generator=g, device="cuda") / 8
    a[M // 2, K // 2] = float("nan")                         # one row of NaN, its neighbours none
    A, B = ops.mx_quantize(a, a_format), ops.mx_quantize(b, "fp4")
    a, b = ops.mx_dequantize(A, torch.float32).double(), ops.mx_dequantize(B, torch.float32).double()
    got = ops.mx_mm_nt(A, B).double()
    assert bool(got[M // 2].isnan().all())
    rest = torch.arange(M, device="cuda") != M // 2
    got, a = got[rest], a[rest]
    want, size = a @ b.t(), a.abs() @ b.abs().t()
    adds = 2 * 17 * (O.padded(K) // 128) + 64                # as in test_product
    assert got.numel() == 0 or float(((got - want).abs() - adds * 2.0 ** -23 * size).max()) <= 0


def test_tokens_number_and_tensor_settings_are_one(ops):
    # 10 equal entries, top_p the decimal 0.3: as float32 it is above 3/10, so a fourth entry is kept, and likewise 0.7 is below
    R = 64
    x = torch.zeros(R, 10, device="cuda")
    words = words_of(R, 11).cuda()
    for value, kept in ((0.3, 4), (0.7, 7), (0.1, 2), (0.9, 9)):
        a = ops.sample_tokens_from_words(x, words, top_p=value)
        b = ops.sample_tokens_from_words(x, words, top_p=torch.full((R,), value, device="cuda"))
        assert torch.equal(a, b) and int(a.max()) == kept - 1


# ---- rows, starts and sizes that the tests above leave out ---------------------------------------------------------------
HARD = [dict(), dict(top_p=0.9), dict(top_k=2500), dict(min_p=0.02), dict(top_k=100, top_p=0.5, min_p=0.3),
        dict(temperature=1e-4, top_p=0.7), dict(temperature=1e4, top_p=0.7, min_p=0.99), dict(temperature=1e-12, top_p=0.9, top_k=3)]


def hard_rows(V, dtype):
    g = torch.Generator().manual_seed(V)
    whole = dtype == torch.int32
    lowest = -2.0 ** 31 if whole else float(torch.finfo(dtype).min)
    x = torch.zeros(8, V, dtype=torch.float64)
    x[0] = lowest if whole else -float("inf")
    x[0, [0, 5, V // 2, V - 9, V - 1]] = torch.tensor([1.0, -2.0, 0.5, 3.0, 2.0], dtype=torch.float64)
    x[1, V // 3] = 30.0
    x[2] = torch.randn(V, generator=g) * (1 if whole else 1e-4)
    x[3] = torch.rand(V, generator=g) * (3 if whole else 0.05)               # thousands of entries in one bin
    x[4] = torch.randn(V, generator=g) * (1e8 if whole else 1e4)
    x[5] = torch.where(torch.rand(V, generator=g) < 0.9, lowest, torch.randn(V, generator=g).double() * 2)
    x[6] = -7.0
    x[7] = torch.linspace(-20, 0, V)
    return (x.round() if whole else x).to(dtype)


@pytest.mark.parametrize("dtype", DTYPES + [torch.int32], ids=IDS + ["i32"])
@pytest.mark.parametrize("V", [777, 9001, 20011])
def test_tokens_of_hard_rows(ops, V, dtype):
    x = hard_rows(V, dtype)
    for n, kw in enumerate(HARD):
        words = words_of(8, n + 40)
        if V < 16384 or n:
            check_tokens(ops, x, words, **kw)
            continue
        # Rows in pieces take a piece's weights as multiples of 2^-f of the piece's largest, so some are finer than the oracle's
        # multiples of 2^-f of the row's.  Either is off by at most 2^-(f + 1) of the row's largest: a running sum by
        # V 2^-(f + 1), and the total times the word's fraction by as much again (f = 61 - 15 = 46 here).
        got = ops.sample_tokens_from_words(x.cuda(), words.cuda(), **kw).cpu().tolist()
        for r in range(8):
            word = int(words[r]) & 0xFFFFFFFF
            assert got[r] == O.sample(host(x)[r], word, **kw) or \
                O.token_within(host(x)[r], word, got[r], 2 * V * 2.0 ** -47, **kw)


@pytest.mark.parametrize("dtype", DTYPES + [torch.int32], ids=IDS + ["i32"])
def test_tokens_from_any_start(ops, dtype):
    """Rows that begin and end inside the 16 bytes of a load, with entries around them that would win."""
    g = torch.Generator().manual_seed(9)
    for V in (10, 501, 4999, 20003):
        for start in (1, 3):
            flat = torch.full((3 * V + 16,), 60000.0).to(dtype)
            x = (torch.randn(3, V, generator=g) * (40 if dtype == torch.int32 else 2)).to(dtype)
            flat[start:start + 3 * V] = x.view(-1)
            there = flat.cuda()[start:start + 3 * V].view(3, V)
            for n, kw in enumerate((dict(top_p=0.9, temperature=2.0), dict(temperature=0.0))):
                w = words_of(3, n)
                got = ops.sample_tokens_from_words(there, w.cuda(), **kw).cpu().tolist()
                assert got == [O.sample(host(x)[r], int(w[r]) & 0xFFFFFFFF, **kw) for r in range(3)]


@pytest.mark.parametrize("K", [65, 1500, 3001, 6007, 20001])
@pytest.mark.parametrize("dtype", DTYPES + [torch.int32], ids=IDS + ["i32"])
def test_rows_from_any_start(ops, dtype, K):
    """The conversions and the norm on tensors one element off a 16-byte border equal those on aligned copies."""
    g = torch.Generator().manual_seed(K)
    off = lambda t: torch.cat([t.new_full((1,), 50.0), t.reshape(-1)])[1:].view(t.shape)
    x = (torch.randn(7, K, generator=g) * (30 if dtype == torch.int32 else 1)).to(dtype).cuda()
    rdt = torch.float16 if dtype == torch.int32 else dtype
    r, w = (torch.randn(n, generator=g).to(rdt).cuda() for n in ((7, K), (K,)))
    assert off(x).data_ptr() % 16 and off(x).is_contiguous()
    for format in O.FORMATS:
        for res in (None, r):
            a, ra = ops.rms_norm_mx(x, w, res, 1e-5, format)
            b, rb = ops.rms_norm_mx(off(x), off(w), None if res is None else off(res), 1e-5, format)
            assert torch.equal(a.codes, b.codes) and torch.equal(a.scales, b.scales)
            assert res is None or torch.equal(ra, rb)
            y, want = O.rms_norm(host(x), host(w), None if res is None else host(res), 1e-5,
                                 (lambda v: v) if res is None else _rounder(rdt))
            codes, scales = O.quantize(y.astype(np.float64), format)
            assert np.array_equal(a.codes.cpu().numpy(), codes) and np.array_equal(a.scales.cpu().numpy(), scales)
        if dtype != torch.int32:
            a, b = ops.mx_quantize(x, format), ops.mx_quantize(off(x), format)
            assert torch.equal(a.codes, b.codes) and torch.equal(a.scales, b.scales)


@pytest.mark.parametrize("K", [500, 3000, 8000, 20000])
def test_norm_with_the_residual_in_place(ops, K):
    from nesgpu_amd import _lib
    g = torch.Generator(device="cuda").manual_seed(K)
    x, r = (torch.randn(9, K, generator=g, device="cuda").bfloat16() for _ in range(2))
    w = torch.ones(K, device="cuda")
    want, new = ops.rms_norm_mx(x, w, r, 1e-5, "fp8")
    codes, scales = torch.empty_like(want.codes), torch.empty_like(want.scales)
    _lib.call("nb_rms_norm_mx", codes.data_ptr(), scales.data_ptr(), r.data_ptr(), x.data_ptr(), 2, r.data_ptr(), 2,
              w.data_ptr(), 0, 1e-5, 1, 9, K, torch.cuda.current_stream().cuda_stream)
    assert torch.equal(r, new) and torch.equal(codes, want.codes) and torch.equal(scales, want.scales)


@pytest.mark.parametrize("a_format", O.FORMATS)
@pytest.mark.parametrize("shape", [(3, 70, 1024), (300, 200, 1024), (1, 2000, 4096), (600, 700, 640)],
                         ids=lambda s: "x".join(map(str, s)))
def test_product_with_scales_on_four_bytes(ops, shape, a_format):
    M, N, K = shape
    g = torch.Generator(device="cuda").manual_seed(K)
    A = ops.mx_quantize(torch.randn(M, K, generator=g, device="cuda"), a_format)
    B = ops.mx_quantize(torch.randn(N, K, generator=g, device="cuda"), "fp4")

    def moved(q, format):
        flat = torch.zeros(q.scales.numel() + 16, dtype=torch.uint8, device="cuda")
        flat[4:4 + q.scales.numel()] = q.scales.view(-1)
        return ops.MXRows(q.codes, flat[4:4 + q.scales.numel()].view(q.scales.shape), K, format)

    want = ops.mx_mm_nt(A, B)
    for a, b in ((moved(A, a_format), B), (A, moved(B, "fp4")), (moved(A, a_format), moved(B, "fp4"))):
        assert torch.equal(ops.mx_mm_nt(a, b), want)


def test_rows_are_copied_and_pickled(ops):
    import copy
    import pickle
    x = torch.randn(5, 200, device="cuda")
    for q in (ops.mx_quantize(x), ops.mx_quantize(x, "fp8")):
        want = ops.mx_dequantize(q)
        for other in (copy.copy(q), copy.deepcopy(q), pickle.loads(pickle.dumps(q))):
            assert torch.equal(ops.mx_dequantize(other), want)
            q.codes, other.scales                                # parts made in one and not in the other
            assert torch.equal(ops.mx_dequantize(other), want) and torch.equal(other.codes, q.codes)


def test_offsets_past_32_bits(ops):
    """The last rows of tensors of more than 2^31 elements (and bytes of codes) equal those rows alone."""
    g = torch.Generator(device="cuda").manual_seed(4)
    rows, K = 70001, 32768
    tail = torch.randn(3, K, generator=g, device="cuda").bfloat16()
    x = torch.zeros(rows, K, dtype=torch.bfloat16, device="cuda")
    x[-3:] = tail
    one = ops.mx_quantize(tail, "fp8")
    q = ops.mx_quantize(x, "fp8")
    assert torch.equal(q.codes[-3:], one.codes) and torch.equal(q.scales[-3:], one.scales)
    assert not bool(q.codes[:-3].any())
    assert torch.equal(ops.mx_dequantize(q)[-3:], ops.mx_dequantize(one))
    w = torch.ones(K, device="cuda")
    n, new = ops.rms_norm_mx(x, w, x)
    n1, new1 = ops.rms_norm_mx(tail, w, tail)
    assert torch.equal(n.codes[-3:], n1.codes) and torch.equal(n.scales[-3:], n1.scales) and torch.equal(new[-3:], new1)
    for N in (8, 300):
        B = ops.mx_quantize(torch.randn(N, K, generator=g, device="cuda"), "fp4")
        c, c1 = ops.mx_mm_nt(q, B)[-3:].double(), ops.mx_mm_nt(one, B).double()
        size = ops.mx_dequantize(one, torch.float32).double().abs() @ ops.mx_dequantize(B, torch.float32).double().abs().t()
        adds = 2 * 17 * (K // 128) + 64                      # as in test_product, for each of the two
        assert float(((c - c1).abs() - 2 * adds * 2.0 ** -23 * size).max()) <= 0
    del n, new, q
    words = torch.randint(-2 ** 31, 2 ** 31, (rows,), generator=g, device="cuda").int()
    for kw in (dict(top_p=0.9), dict(temperature=0.0)):
        assert torch.equal(ops.sample_tokens_from_words(x, words, **kw)[-3:],
                           ops.sample_tokens_from_words(tail, words[-3:].contiguous(), **kw))


@pytest.mark.parametrize("a_format", O.FORMATS)
@pytest.mark.parametrize("K", [65535 * 128, 65536 * 128, 65537 * 128])
def test_product_of_the_longest_rows(ops, K, a_format):
    """Ones: every sum is K, a whole number below 2^24 that fp32 holds at each step."""
    one = {"fp4": 0x22, "fp8": 0x38}

    def rows(n, format):
        return ops.MXRows(torch.full((n, K // (2 if format == "fp4" else 1)), one[format], dtype=torch.uint8, device="cuda"),
                          torch.full((n, K // 32), 127, dtype=torch.uint8, device="cuda"), K, format)

    for M, N in ((300, 70), (2, 5)):
        got = ops.mx_mm_nt(rows(M, a_format), rows(N, "fp4"))
        assert bool((got == K).all())


@pytest.mark.parametrize("a_format", O.FORMATS)
def test_product_of_very_many_rows(ops, a_format):
    """More tiles of one operand than fit 16 + 5 bits."""
    M, N, K = 200_000_003, 3, 1
    A = ops.MXRows(torch.zeros(M, 64 if a_format == "fp4" else 128, dtype=torch.uint8, device="cuda"),
                   torch.full((M, 4), 127, dtype=torch.uint8, device="cuda"), K, a_format)
    A.codes[-2:, 0] = 0x02 if a_format == "fp4" else 0x38
    B = ops.mx_quantize(torch.tensor([[1.0], [-2.0], [3.0]], device="cuda"), "fp4")
    got = ops.mx_mm_nt(A, B, torch.bfloat16)
    assert not bool(got[:-2].any())
    assert got[-2:].tolist() == [[1.0, -2.0, 3.0]] * 2


@pytest.mark.parametrize("R, V", [(1200, 1500), (700, 3000), (600, 6001), (300, 12001)], ids=str)
def test_tokens_of_many_rows(ops, R, V):
    """Rows that outnumber what the card holds at once: a few distinct ones repeated, drawn as the few are."""
    g = torch.Generator().manual_seed(R)
    few = torch.cat([hard_rows(V, torch.float32), torch.randn(8, V, generator=g) * 2.5])
    at = torch.randint(0, 16, (R,), generator=g)
    words = words_of(R, 3)
    x = few[at].cuda()
    for kw in HARD:
        got = ops.sample_tokens_from_words(x, words.cuda(), **kw).cpu()
        for lo in range(0, R, 100):                          # in pieces small enough for the other form
            part = ops.sample_tokens_from_words(x[lo:lo + 100], words[lo:lo + 100].cuda(), **kw).cpu()
            assert torch.equal(got[lo:lo + 100], part)


@pytest.mark.parametrize("V", [20, 300, 5000, 20003])
def test_tokens_with_extreme_settings_per_row(ops, V):
    nan, inf = float("nan"), float("inf")
    x = torch.randn(4, V, generator=torch.Generator().manual_seed(V)).cuda() * 2
    words = words_of(4, 1).cuda()
    t = lambda *v: torch.tensor(v, device="cuda")
    top = x.argmax(1).int()
    plain = ops.sample_tokens_from_words(x, words)
    assert torch.equal(ops.sample_tokens_from_words(x, words, top_p=t(nan, inf, 1.0, 2.0), min_p=t(nan, -1.0, -inf, 0.0)), plain)
    assert torch.equal(ops.sample_tokens_from_words(x, words, temperature=t(nan, 0.0, -inf, -1.0)), top)
    assert torch.equal(ops.sample_tokens_from_words(x, words, top_p=t(-1.0, -inf, 0.0, 1e-30)), top)
    assert torch.equal(ops.sample_tokens_from_words(x, words, min_p=t(1.0, inf, 2.0, 1.0)), top)
    k = torch.tensor([1, 0, -(2 ** 31), 2 ** 31 - 1], dtype=torch.int32, device="cuda")
    got = ops.sample_tokens_from_words(x, words, top_k=k)
    assert got[0] == top[0] and torch.equal(got[1:], plain[1:])


# rows of more than one launch: 2^24 of at most 64 entries, 2^21 of up to 16376, 2^21 / 3 of 16385 (more than 2^34 entries)
@pytest.mark.parametrize("R, V, dtype", [((1 << 24) + 5, 10, torch.int32), ((1 << 21) + 3, 70, torch.float16),
                                         (1_050_000, 16385, torch.bfloat16)], ids=str)
def test_tokens_of_rows_beyond_one_launch(ops, R, V, dtype):
    """Every row is one of 32 under one of 32 words and one of 32 settings: all equal the table of those, and the table the oracle."""
    g = torch.Generator(device="cuda").manual_seed(V)
    few = torch.randn(32, V, generator=g, device="cuda") * 2.5
    few = (few * 3).round().int() if dtype == torch.int32 else few.to(dtype)
    words = torch.randint(-2 ** 31, 2 ** 31, (32,), generator=g, device="cuda").int()
    settings = dict(temperature=0.5 + torch.rand(32, generator=g, device="cuda"), top_p=torch.rand(32, generator=g, device="cuda"),
                    min_p=0.1 * torch.rand(32, generator=g, device="cuda"),
                    top_k=torch.randint(0, 40, (32,), generator=g, device="cuda").int())
    a, b, c = (i.reshape(-1) for i in torch.meshgrid(*[torch.arange(32, device="cuda")] * 3, indexing="ij"))
    table = ops.sample_tokens_from_words(few[a], words[b], **{k: v[c] for k, v in settings.items()})
    for i in torch.randint(0, 32 ** 3, (40,), generator=g, device="cuda").tolist():
        want = O.sample(host(few[a[i]]), int(words[b[i]]) & 0xFFFFFFFF, **{k: v[c[i]].item() for k, v in settings.items()})
        assert int(table[i]) == want
    a, b, c = (torch.randint(0, 32, (R,), generator=g, device="cuda") for _ in range(3))
    got = ops.sample_tokens_from_words(few[a], words[b], **{k: v[c] for k, v in settings.items()})
    assert torch.equal(got, table[(a * 32 + b) * 32 + c])


@pytest.mark.parametrize("N", [1, 3])
def test_product_of_more_rows_than_a_launch_of_square_tiles_holds(ops, N):
    """More than 2^23 tiles of 64 x 64."""
    M, K = (1 << 29) + 70, 1
    A = ops.MXRows(torch.zeros(M, 64, dtype=torch.uint8, device="cuda"),
                   torch.full((M, 4), 127, dtype=torch.uint8, device="cuda"), K, "fp4")
    A.codes[-2:, 0] = 0x02
    A.codes[1 << 28, 0] = 0x02
    B = ops.mx_quantize(torch.tensor([[1.0], [-2.0], [3.0]], device="cuda")[:N].contiguous(), "fp4")
    got = ops.mx_mm_nt(A, B, torch.bfloat16)
    for at in (M - 2, M - 1, 1 << 28):
        assert got[at].tolist() == [1.0, -2.0, 3.0][:N]
        got[at] = 0
    assert not bool(got.any())


# ---- every kernel of the product and of the sampler ----------------------------------------------------------------------
# sizes by the tile that they take; the test asks the library whether they still do
TILES = {
    "fp8": {(256, 256): [(4001, 8190)], (128, 128): [(2047, 4095), (2000, 4000)], (64, 128): [(3000, 3000), (4137, 745)],
            (64, 64): [(2049, 2100), (1596, 436)], (16, 64): [(939, 164), (64, 7132)], (16, 32): [(645, 179), (300, 1100)],
            (16, 16): [(2489, 35), (1, 3786)], (8, 16): [(101, 163), (27, 983)], (16, 4): [(1, 671)], (4, 4): [(39, 36)]},
    "fp4": {(256, 256): [(4001, 8190)], (128, 128): [(3001, 2501), (2047, 4095)], (64, 128): [(273, 3825), (1023, 1025)],
            (64, 64): [(588, 1432), (300, 1100)], (16, 64): [(70, 2000), (344, 407)], (16, 32): [(794, 97), (33, 1900)],
            (16, 16): [(127, 275)], (8, 8): [(276, 35)], (16, 8): [(27, 983)], (4, 4): [(30, 18)]},
}


@pytest.mark.parametrize("K, moved", [(512, False), (1024, True), (1104, False)], ids=["512", "1024-scales-on-4-bytes", "1104"])
@pytest.mark.parametrize("a_format, tile, shape", [(f, t, s) for f, v in TILES.items() for t, shapes in v.items() for s in shapes],
                         ids=lambda v: "x".join(map(str, v)) if isinstance(v, tuple) else v)
def test_every_tile_makes_exact_sums(ops, a_format, tile, shape, K, moved):
    """E4M3: of every eight neighbours two large values that cancel and two that are 17 binades smaller; E2M1: small whole numbers.
    Blocks and rows have scales of their own.  With blocks 2^0 to 2^4 apart the running sum is a multiple of 2^-10 below 2^13, 23 bits
    times the two rows' scales: exact in fp32, and what is stored is that sum rounded once.  The fp16 product is first called inside a
    captured graph, and replayed with the signs of A's codes turned."""
    from nesgpu_amd import _lib
    M, N = shape
    taken = _lib.load().nb_mx_mm_tile(M, N, K, O.FORMATS.index(a_format))
    assert (taken >> 16, taken & 0xFFFF) == tile
    g = torch.Generator(device="cuda").manual_seed(M + N + K)
    power = lambda lo, hi, *size: torch.exp2(torch.randint(lo, hi + 1, size, generator=g, device="cuda").float())
    whole = lambda lo, hi, *size: torch.randint(lo, hi + 1, size, generator=g, device="cuda").float()
    if a_format == "fp8":
        a, b = torch.zeros(M, K, device="cuda"), torch.ones(N, K, device="cuda")
        a[:, 0::8], a[:, 1::8] = 256.0, -256.0
        a[:, 2::8], a[:, 5::8] = whole(1, 7, M, K // 8) / 512, whole(8, 15, M, K // 8) / 512
        b[:, 2::8] = torch.tensor([0.5, 1.5, -3.0], device="cuda")[whole(0, 2, N, K // 8).long()]
    else:
        a, b = whole(-3, 3, M, K), whole(-2, 2, N, K)
    blocks = -(-K // 32)
    a *= power(0, 3, M, blocks).repeat_interleave(32, 1)[:, :K] * power(-6, 6, M, 1)
    b *= power(0, 1, N, blocks).repeat_interleave(32, 1)[:, :K] * power(-3, 3, N, 1)
    A, B = ops.mx_quantize(a, a_format), ops.mx_quantize(b, "fp4")
    assert torch.equal(ops.mx_dequantize(A, torch.float32), a) and torch.equal(ops.mx_dequantize(B, torch.float32), b)
    if moved:
        flat = torch.zeros(A.scales.numel() + 16, dtype=torch.uint8, device="cuda")
        flat[4:4 + A.scales.numel()] = A.scales.view(-1)
        A = ops.MXRows(A.codes, flat[4:4 + A.scales.numel()].view(A.scales.shape), K, a_format)
    want = (a.double() @ b.double().t()).float()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = ops.mx_mm_nt(A, B, torch.float16)
    for sign in (1, -1, 1):
        graph.replay()
        assert torch.equal(out, (sign * want).half())
        A.codes.bitwise_xor_(0x80 if a_format == "fp8" else 0x88)
    A.codes.bitwise_xor_(0x80 if a_format == "fp8" else 0x88)
    assert torch.equal(ops.mx_mm_nt(A, B), want)
    assert torch.equal(ops.mx_mm_nt(A, B, torch.bfloat16), want.bfloat16())


# rows that outnumber what the card holds at once, by the four forms that such rows take; the last entries of each form too
@pytest.mark.parametrize("dtype", DTYPES + [torch.int32], ids=IDS + ["i32"])
@pytest.mark.parametrize("R, V", [(1100, 1017), (1100, 2040), (600, 2041), (600, 4088), (600, 4089), (600, 8184), (300, 8185),
                                  (300, 16376)], ids=str)
def test_tokens_of_many_rows_of_every_type(ops, R, V, dtype):
    """Twelve rows under four words, each as often as it comes: alike wherever they stand, in storage that starts inside a load, and
    those looked at equal to the oracle."""
    g = torch.Generator().manual_seed(R + V)
    few = torch.randn(4, V, generator=g) * 2.5
    few = torch.cat([hard_rows(V, dtype), ((few * 3).round().int() if dtype == torch.int32 else few.to(dtype))])
    few[1, -1] = few[1, 0] = few[1].max()                    # the largest entry at both ends
    four = torch.tensor([0, -1, 123456789, -1234567890], dtype=torch.int32)
    row, word = torch.randint(0, 12, (R,), generator=g), torch.randint(0, 4, (R,), generator=g)
    flat = torch.empty(R * V + 1, dtype=dtype, device="cuda")
    x = flat[1:].view(R, V)
    x.copy_(few.cuda()[row.cuda()])
    words = four[word].cuda()
    pair = row * 4 + word
    first = torch.full((48,), -1)
    for i in range(R - 1, -1, -1):
        first[pair[i]] = i
    assert int(first.min()) >= 0
    for n, kw in enumerate(HARD + [dict(temperature=0.0)]):
        got = ops.sample_tokens_from_words(x, words, **kw).cpu()
        assert torch.equal(got, got[first[pair]])
        for p in ((5 * n + 7 * k) % 48 for k in range(3 if V > 5000 else 8)):
            want = O.sample(host(few[p // 4]), int(four[p % 4]) & 0xFFFFFFFF, **kw)
            assert int(got[first[p]]) == want, (n, p)
