"""Microscaled rows, norm, product and token sampler without a GPU: the oracle's own pins, and what is refused before
anything is launched."""
import copy
import ctypes
import math
import os
import pickle
import sys
import threading

import numpy as np
import pytest
import torch

from oracle import mx as O

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture(scope="module")
def lib():
    from nesgpu_amd import _lib
    if not os.path.exists(_lib.LIB_PATH):
        import __graft_entry__ as g
        g.build()
    return _lib.load()


# ---- oracle pins ----------------------------------------------------------------------------------------------------
def test_tables():
    assert O.table("fp4").max() == 6 and O.table("fp8").max() == 448 and len(O.table("fp8")) == 127
    f8 = torch.arange(127, dtype=torch.uint8).view(torch.float8_e4m3fn).double().numpy()
    assert np.array_equal(O.table("fp8"), f8)


@pytest.mark.parametrize("format", O.FORMATS)
def test_values_of_the_format_are_kept(format):
    t = O.table(format)
    x = np.zeros((1, 256))
    x[0, :len(t)] = t
    x[0, 128:128 + len(t)] = -t
    x[0, 0::32] = t[-1]                                    # every block reaches the largest value: scale 1
    c, s = O.quantize(x, format)
    assert np.all(s == 127)
    assert np.array_equal(O.decode(c, s, 256, format), x)


@pytest.mark.parametrize("format", O.FORMATS)
def test_error_is_at_most_half_a_step(format):
    g = np.random.default_rng(1)
    x = g.standard_normal((4, 320)) * np.exp(g.standard_normal((4, 1)) * 5)
    c, s = O.quantize(x, format)
    v = O.decode(c, s, 320, format)
    half = {"fp4": 2.0 ** -2, "fp8": 2.0 ** -4}[format]    # of the value's own binade ...
    scale = np.ldexp(1.0, np.repeat(s.astype(int), 32, axis=1)[:, :320] - 127)
    smallest = {"fp4": 0.25, "fp8": 2.0 ** -10}[format]    # ... or half the smallest code
    top = O.table(format)[-1] * scale
    inside = np.abs(x) <= top
    assert np.all(np.abs(v - x)[inside] <= np.maximum(half * np.abs(x), smallest * scale)[inside])
    assert np.array_equal(np.abs(v)[~inside], top[~inside])              # saturated


def test_sampler_keeps_the_shortest_prefix():
    x = np.log([0.5, 0.25, 0.125, 0.125])
    # words spread over the unit interval: the shares of what is kept
    def shares(**kw):
        got = [O.sample(x, int(u * 2 ** 32), **kw) for u in (np.arange(64) + 0.5) / 64]
        return [got.count(i) for i in range(4)]
    assert shares() == [32, 16, 8, 8]
    assert shares(top_k=1) == [64, 0, 0, 0] and shares(top_k=3)[3] == 0
    assert shares(top_p=0.74)[2:] == [0, 0]
    assert shares(min_p=0.3)[2:] == [0, 0]
    assert shares(temperature=0.0) == [64, 0, 0, 0]
    assert O.sample(np.full(5, -np.inf), 7) == -1
    assert O.sample(np.array([np.nan, 1.0, -np.inf]), 2 ** 32 - 1) == 1
    assert [O.sample(np.zeros(4), w, top_p=0.5) for w in (0, 2 ** 31 - 1, 2 ** 31, 2 ** 32 - 1)] == [0, 0, 1, 1]


# ---- refusals ---------------------------------------------------------------------------------------------------------
def test_c_abi_refuses_before_launching(lib):
    one, odd = ctypes.c_void_p(256), ctypes.c_void_p(257)
    err = lib.nb_last_error_string
    assert lib.nb_mx_quantize(one, one, one, 0, 0, -1, 32, None) == 2
    assert lib.nb_mx_quantize(one, one, one, 3, 0, 1, 32, None) == 2 and b"type" in err()
    assert lib.nb_mx_quantize(one, one, one, 0, 2, 1, 32, None) == 2 and b"format" in err()
    assert lib.nb_mx_quantize(None, one, one, 0, 0, 1, 32, None) == 1
    assert lib.nb_mx_quantize(odd, one, one, 0, 0, 1, 32, None) == 3
    assert lib.nb_mx_quantize(one, one, odd, 1, 0, 1, 32, None) == 3
    assert lib.nb_mx_quantize(one, one, one, 0, 0, 1 << 39, 1 << 39, None) == 2
    assert lib.nb_mx_quantize(None, None, None, 0, 0, 0, 32, None) == 0              # nothing to do
    assert lib.nb_mx_dequantize(one, 3, one, one, 0, 1, 32, None) == 2
    assert lib.nb_mx_dequantize(one, 0, one, None, 0, 1, 32, None) == 1
    # norm: a residual of another floating type, half a pair, a negative eps
    assert lib.nb_rms_norm_mx(one, one, one, one, 2, one, 0, one, 0, 1e-6, 1, 1, 32, None) == 2 and b"residual" in err()
    assert lib.nb_rms_norm_mx(one, one, None, one, 2, one, 2, one, 0, 1e-6, 1, 1, 32, None) == 1
    assert lib.nb_rms_norm_mx(one, one, None, one, 2, None, 0, one, 0, -1.0, 1, 1, 32, None) == 2
    assert lib.nb_rms_norm_mx(one, one, None, one, 2, None, 0, one, 0, float("nan"), 1, 1, 32, None) == 2
    assert lib.nb_rms_norm_mx(one, one, None, one, 2, None, 0, one, 3, 1e-6, 1, 1, 32, None) == 2
    # product: no inner length, an output type, formats
    assert lib.nb_mx_mm_nt(one, 0, one, one, 0, one, one, 1, 1, 0, None) == 2
    assert lib.nb_mx_mm_nt(one, 3, one, one, 0, one, one, 1, 1, 32, None) == 2
    assert lib.nb_mx_mm_nt(one, 0, one, one, 5, one, one, 1, 1, 32, None) == 2
    assert lib.nb_mx_mm_nt(one, 0, one, odd, 0, one, one, 1, 1, 32, None) == 3
    assert lib.nb_mx_mm_nt(None, 0, None, None, 0, None, None, 0, 5, 32, None) == 0
    # tokens
    args = (None, 1.0, None, 0, None, 1.0, None, 0.0)
    assert lib.nb_sample_tokens(one, one, 0, one, *args, 1, 0, None, 0, None) == 2
    assert lib.nb_sample_tokens(one, one, 0, one, *args, 1, (1 << 20) + 1, None, 0, None) == 2
    assert lib.nb_sample_tokens(one, one, 4, one, *args, 1, 8, None, 0, None) == 2
    assert lib.nb_sample_tokens(one, None, 0, one, *args, 1, 8, None, 0, None) == 1
    assert lib.nb_sample_tokens(one, odd, 0, one, *args, 1, 8, None, 0, None) == 3
    assert lib.nb_sample_tokens(one, one, 0, one, None, math.nan, *args[2:], 1, 8, None, 0, None) == 2
    assert lib.nb_sample_tokens(None, None, 0, None, *args, 0, 8, None, 0, None) == 0


def test_python_refuses_host_tensors():
    from nesgpu_amd.extensions import booleanOperations as ops
    x = torch.zeros(2, 64)
    with pytest.raises(RuntimeError, match="CUDA"):
        ops.mx_quantize(x)
    with pytest.raises(RuntimeError, match="CUDA"):
        ops.rms_norm_mx(x, torch.ones(64))
    with pytest.raises(RuntimeError, match="CUDA"):
        ops.sample_tokens_from_words(x, torch.zeros(2, dtype=torch.int32))
    with pytest.raises(RuntimeError, match="CUDA"):
        ops.MXRows(torch.zeros(2, 64, dtype=torch.uint8), torch.zeros(2, 4, dtype=torch.uint8), 64)
    with pytest.raises(ValueError, match="format"):
        ops.MXRows(x, x, 64, "fp6")


# ---- rows that a kernel wrote, taken apart while another thread uses them ----------------------------------------------
def _before_line(n, call, other):
    """Runs ``call``, and ``other`` before the n-th line that it runs in the rows' own code, as a thread that takes its turn there
    would.  -> (what call gave, what other gave in a list, empty where there are fewer lines)"""
    from nesgpu_amd.extensions import booleanOperations as ops
    left, got = [n], []

    def trace(frame, event, arg):
        if frame.f_code.co_filename != ops.__file__:
            return None
        if event == "line":
            left[0] -= 1
            if left[0] == -1:
                got.append(other())                          # not traced: the tracer is off inside itself
        return trace

    before = sys.gettrace()
    sys.settrace(trace)
    try:
        return call(), got
    finally:
        sys.settrace(before)


@pytest.mark.parametrize("format", O.FORMATS)
@pytest.mark.parametrize("call", ["pointers", "codes", "scales"])
@pytest.mark.parametrize("other", ["pointers", "codes", "scales"])
def test_rows_are_taken_apart_between_any_two_lines_of_their_use(format, call, other):
    from nesgpu_amd.extensions import booleanOperations as ops
    rows, K = 5, 200
    n = 256 if format == "fp8" else 128
    for line in range(100):
        q = ops.MXRows._empty(rows, K, format, "cpu")
        use = {"pointers": q._pointers, "codes": lambda: q.codes, "scales": lambda: q.scales}
        codes = q._pointers()[0]
        scales = codes + rows * n

        def right(which, got):
            if which == "pointers":
                return tuple(got) == (codes, scales)
            if which == "codes":
                return (got.data_ptr(), tuple(got.shape), got.stride()) == (codes, (rows, n), (n, 1))
            return (got.data_ptr(), tuple(got.shape), got.stride()) == (scales, (rows, 8), (8, 1))

        mine, theirs = _before_line(line, use[call], use[other])
        assert right(call, mine) and all(right(other, t) for t in theirs), line
        assert all(right(which, use[which]()) for which in use), line
        if not theirs:
            break
    assert line > 2 and not theirs


def test_rows_are_used_by_two_threads():
    from nesgpu_amd.extensions import booleanOperations as ops
    rows, K = 3, 130
    before, turns, wrong = sys.getswitchinterval(), 2000, []
    sys.setswitchinterval(1e-6)
    try:
        for _ in range(turns):
            q = ops.MXRows._empty(rows, K, "fp8", "cpu")
            start = q._pointers()[0]
            other = threading.Thread(target=lambda: (q.scales, q.codes))
            other.start()
            for _ in range(20):
                if q._pointers() != (start, start + rows * 256) or q.scales.data_ptr() != start + rows * 256:
                    wrong.append(q)
            other.join()
    finally:
        sys.setswitchinterval(before)
    assert not wrong


def test_copies_of_rows_keep_their_parts_in_one_place():
    """What is written through a copy's codes is what the kernels read there, whether the parts were made before or not."""
    from nesgpu_amd.extensions import booleanOperations as ops
    for made in (False, True):
        q = ops.MXRows._empty(4, 40, "fp4", torch.device("cpu"))
        q._joint.copy_(torch.arange(q._joint.numel()) % 251)
        if made:
            q.codes
        for other in (copy.copy(q), copy.deepcopy(q), pickle.loads(pickle.dumps(q))):
            assert other._pointers() == (other.codes.data_ptr(), other.scales.data_ptr())
            assert torch.equal(other.codes, q.codes) and torch.equal(other.scales, q.scales)
            assert (other.rows, other.K, other.format, other.device) == (q.rows, q.K, q.format, q.device)
        assert copy.copy(q)._pointers() == q._pointers()


# ---- rows of logits beyond one launch -----------------------------------------------------------------------------------
@pytest.mark.parametrize("R, V", [(1 << 22, 10), (4096 * 1024, 10), ((1 << 22) + 3, 1000), (1 << 30, 64), (1 << 20, 1 << 14),
                                  (1 << 22, 20000), (1 << 20, 1 << 20)])
def test_any_number_of_rows_of_logits_is_taken(lib, R, V):
    """The rows' number is looked at before the pointers: what stops these calls is the missing logits (status 1), not a
    shape (2)."""
    one = ctypes.c_void_p(256)
    args = (None, 1.0, None, 0, None, 1.0, None, 0.0)
    assert lib.nb_sample_tokens(one, None, 0, one, *args, R, V, None, 0, None) == 1
    work = lib.nb_sample_tokens_workspace_bytes(R, V)
    assert (work > 0) == (V > 16376) and work < 13 << 29          # 6.5 GiB
    if work:                                                      # and a short one is refused
        assert lib.nb_sample_tokens(one, one, 0, one, *args, R, V, one, work - 1, None) == 2
    assert lib.nb_sample_tokens(one, None, 0, one, *args, (1 << 40) + 1, V, None, 0, None) == 2


# ---- the product's tiles --------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("format", [0, 1])
def test_every_size_has_a_tile_that_one_launch_holds(lib, format):
    """All sizes up to 2^30 whose output of two bytes each fits 288 GB; a launch has threads for 2^22 tiles of 256 x 256 or 2^23 of others, and
    2^23 - 1 or 2^24 - 1 of the narrow ones."""
    most = {(256, 256): 1 << 22, (128, 128): 1 << 23, (64, 128): 1 << 23, (64, 64): 1 << 23, (16, 64): (1 << 24) - 1,
            (16, 32): (1 << 24) - 1}
    sizes = sorted({min(int(2 ** (e / 2)) + d, 1 << 30) for e in range(61) for d in (0, 1)})
    for M in sizes:
        for N in sizes:
            if M * N > 1 << 37:
                continue
            for K in (1, 700, 65535 * 128, 65536 * 128):
                if K > 700 and M + N > 1 << 17:
                    continue
                t = lib.nb_mx_mm_tile(M, N, K, format)
                rows, columns = t >> 16, t & 0xFFFF
                assert rows and columns, (M, N, K)
                tiles = -(-M // rows) * -(-N // columns)
                assert tiles <= most.get((rows, columns), (1 << 23) - 1), (M, N, K, rows, columns)
    for bad in ((0, 1, 1), (1, 1, 0), (1, -1, 1), ((1 << 30) + 1, 1, 1), (1, 1, (1 << 30) + 1)):
        assert lib.nb_mx_mm_tile(*bad, format) == 0
    assert lib.nb_mx_mm_tile(1, 1, 1, 2) == 0
