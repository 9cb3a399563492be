"""The 8-bit serving operators (RowCache, Linear8) against their definition in
64 bits (oracle/quant_oracle.py).

Codes and scales are equal. Values read back are the FP32 product of code and
scale (one rounding, 2^-24) rounded to the output type (2^-11 for FP16).
Products: the sum of codes is exact in int32; a term is rounded when it is
converted, when it meets the token's scale, the channel's, and the bias, once
per segment as the segments are added, each by 2^-24 of the terms' magnitudes:
(segments + 4) 2^-24, and the rounding to the output type.
"""
import ctypes
import importlib

import numpy as np
import pytest
import torch

from oracle import quant_oracle as qo

gpu = pytest.mark.gpu


@pytest.fixture(scope="module")
def Q(pkg):
    return importlib.import_module(pkg.__name__ + ".quant")


def rows_of(rng, rows, cols, dtype=np.float16):
    x = rng.standard_normal((rows, cols)) * np.exp(rng.standard_normal((rows, 1)))
    return x.astype(dtype)


def dev(x):
    return torch.from_numpy(np.ascontiguousarray(x)).cuda()


def store_of(pkg, tmp_path, params):
    synth = importlib.import_module(pkg.__name__ + ".synth")
    return pkg.Weights(synth.write_manifest(str(tmp_path), params, {"type": "nafnet_residual", "base_channels": 32,
                                                                   "num_levels": 1, "in_channels": 1}))


def host(t):
    torch.cuda.synchronize()
    return t.cpu().numpy()


def bytes_of(cols, bits):
    return (cols * bits + 7) // 8


def assert_held(cache, at, q, s, bits):
    codes, scales = host(cache.codes), host(cache.scales)
    np.testing.assert_array_equal(codes[at][:, :bytes_of(q.shape[1], bits)], qo.pack(q, bits))
    np.testing.assert_array_equal(scales[at], s)


def assert_read(got, q, s):
    want = qo.values(q, s)
    tol = qo.output_bound(want, np.abs(want) * 2.0 ** -24, got.dtype)
    np.testing.assert_array_equal(np.isnan(got), np.isnan(want))
    # The scale of the largest FP32 values, fl32(max fl32(1 / qmax)), may be rounded up so that qmax times it lies 2^103
    # or more (half a step) above the largest FP32 number: rounding to nearest makes that an infinity. Of FP16 the
    # border is 65520.
    border = 65520.0 if got.dtype == np.float16 else (2.0 - 2.0 ** -24) * 2.0 ** 127
    over = np.abs(want) >= border
    np.testing.assert_array_equal(got[over], np.sign(want[over]) * np.inf)
    fine = np.isfinite(want) & ~over
    assert (np.abs(got.astype(np.float64) - want)[fine] <= tol[fine]).all()


def assert_product(got, y, e):
    tol = qo.output_bound(y, e, got.dtype)
    np.testing.assert_array_equal(np.isnan(got), np.isnan(y))
    fine = np.isfinite(y)
    off = np.abs(got.astype(np.float64) - y)[fine]
    assert (off <= tol[fine]).all(), f"{(off > tol[fine]).sum()} of {off.size} off, worst {np.max(off / tol[fine])} bounds"


# ---------------------------------------------------------------------------------------------------------------------
# Refusals that need no GPU: the checks come before any CUDA call
# ---------------------------------------------------------------------------------------------------------------------

FAKE = 1 << 20  # never dereferenced


def write_args(**k):
    a = dict(x=FAKE, dtype=1, ldx=32, rows=4, cols=32, slots=None, row0=0, codes=FAKE, ld=32, scales=FAKE, capacity=8,
             bits=8, group=0, err=None, stream=None)
    a.update(k)
    return tuple(a.values())


def read_args(**k):
    a = dict(codes=FAKE, ld=32, scales=FAKE, capacity=8, cols=32, bits=8, group=0, page_rows=2, table=FAKE, table_ld=4,
             table_cols=4, lengths=None, batch=1, max_rows=8, out=FAKE, dtype=1, out_batch=256, ldo=32, err=None,
             stream=None)
    a.update(k)
    return tuple(a.values())


@pytest.mark.parametrize("bad", [dict(dtype=2), dict(bits=6), dict(cols=0), dict(cols=-1), dict(group=5),
                                 dict(group=4), dict(group=-32), dict(ld=31), dict(capacity=-1), dict(capacity=1 << 31),
                                 dict(rows=-1), dict(rows=1 << 31), dict(row0=5), dict(row0=-1), dict(rows=9),
                                 dict(codes=None), dict(scales=None), dict(scales=FAKE + 2), dict(x=None),
                                 dict(x=FAKE + 1), dict(ldx=31), dict(row0=(1 << 63) - 1)])
def test_cache_write_refuses(pkg, bad):
    rc = pkg.lib().dn_launch_cache_write(*write_args(**bad))
    assert rc == (pkg.DN_ERR_DTYPE if "dtype" in bad else pkg.DN_ERR_INVALID_ARG)
    assert pkg.lib().dn_last_error()


@pytest.mark.parametrize("bad", [dict(dtype=-1), dict(bits=16), dict(group=12), dict(ld=15, bits=4), dict(page_rows=0),
                                 dict(page_rows=1 << 31), dict(batch=-1), dict(batch=65536), dict(table=None),
                                 dict(table_cols=-1), dict(batch=2, table_ld=3), dict(out=None), dict(out=FAKE + 1),
                                 dict(ldo=31), dict(max_rows=-1), dict(batch=2, out_batch=255), dict(codes=None)])
def test_cache_read_refuses(pkg, bad):
    rc = pkg.lib().dn_launch_cache_read_pages(*read_args(**bad))
    assert rc == (pkg.DN_ERR_DTYPE if "dtype" in bad else pkg.DN_ERR_INVALID_ARG)


def test_row_numbers_and_tables_that_are_not_aligned_to_their_type_are_refused(pkg):
    """A kernel's load of such a word would be a fault. (No rows: what passes the check launches nothing.)"""
    lib, bad = pkg.lib(), pkg.DN_ERR_INVALID_ARG
    for off in (1, 2, 4):
        assert lib.dn_launch_cache_write(*write_args(slots=FAKE + off, rows=0)) == bad
        assert lib.dn_launch_cache_read_rows(FAKE, 32, FAKE, 8, 32, 8, 0, FAKE + off, 0, 0, FAKE, 1, 32, None, None) == bad
    for off in (1, 2):
        for k in (dict(table=FAKE + off), dict(lengths=FAKE + off), dict(err=FAKE + off)):
            assert lib.dn_launch_cache_read_pages(*read_args(max_rows=0, **k)) == bad
        assert lib.dn_launch_cache_write(*write_args(err=FAKE + off, rows=0)) == bad
        assert lib.dn_launch_cache_read_rows(FAKE, 32, FAKE, 8, 32, 8, 0, None, 0, 0, FAKE, 1, 32, FAKE + off, None) == bad
    assert lib.dn_launch_cache_write(*write_args(slots=FAKE + 8, err=FAKE + 4, rows=0)) == pkg.DN_OK
    assert lib.dn_launch_cache_read_pages(*read_args(table=FAKE + 4, lengths=FAKE + 4, err=FAKE + 4, max_rows=0)) == pkg.DN_OK


def test_nothing_to_do_needs_no_gpu(pkg):
    assert pkg.lib().dn_launch_cache_write(*write_args(rows=0, x=None)) == pkg.DN_OK
    for k in (dict(max_rows=0, out=None), dict(table_cols=0), dict(batch=0)):
        assert pkg.lib().dn_launch_cache_read_pages(*read_args(**k)) == pkg.DN_OK


def test_classes_refuse(pkg, Q):
    for k in (dict(bits=5), dict(group=7), dict(cols=0), dict(page_rows=0), dict(pages=-1), dict(group=12, cols=24),
              dict(pages=1 << 20, page_rows=1 << 11)):
        with pytest.raises(pkg.InvalidArgumentError):
            Q.RowCache(**{**dict(pages=2, page_rows=4, cols=32), **k})
    with pytest.raises(pkg.InvalidArgumentError):
        Q.Linear8.from_tensors(torch.zeros(4, 4))


def test_a_copied_or_loaded_cache_uses_its_own_tensors(Q, monkeypatch):
    """Not the addresses of the cache that it was made from. (Tensors of the CPU stand in.)"""
    import contextlib
    import copy
    import pickle

    monkeypatch.setattr(torch.cuda, "device", lambda d: contextlib.nullcontext())
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
    zeros = torch.zeros
    monkeypatch.setattr(torch, "zeros", lambda *a, device=None, **k: zeros(*a, **k))
    cache = Q.RowCache(2, 3, 20, bits=4)
    cache.codes.fill_(3)
    for other in (copy.deepcopy(cache), pickle.loads(pickle.dumps(cache))):
        assert other._held == (other.codes.data_ptr(), 16, other.scales.data_ptr(), 6)
        assert other._err_ptr == other._err.data_ptr() != cache._err_ptr and other._held[0] != cache._held[0]
        assert (other.pages, other.page_rows, other.cols, other.bits, other.group) == (2, 3, 20, 4, 20)
        assert torch.equal(other.codes, cache.codes)
    for name in ("codes", "scales"):
        with pytest.raises(AttributeError):
            setattr(cache, name, torch.ones(1))


def test_a_layer_is_not_copied(Q):
    import copy
    import pickle

    layer = Q.Linear8.__new__(Q.Linear8)
    layer._h = None
    for f in (copy.copy, copy.deepcopy, pickle.dumps):
        with pytest.raises(TypeError):
            f(layer)


def test_row_numbers_that_no_64_bit_word_holds_are_refused(pkg, Q, monkeypatch):
    """ctypes would cut them to a row or page that is there."""
    import contextlib

    monkeypatch.setattr(torch.cuda, "device", lambda d: contextlib.nullcontext())
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
    monkeypatch.setattr(torch.cuda, "current_device", lambda: -1)
    monkeypatch.setattr(Q, "_stream", lambda d: 0)
    zeros, empty = torch.zeros, torch.empty
    monkeypatch.setattr(torch, "zeros", lambda *a, device=None, **k: zeros(*a, **k))
    monkeypatch.setattr(torch, "empty", lambda *a, device=None, **k: empty(*a, **k))
    calls = []

    class Lib:
        def __getattr__(self, name):
            return lambda *args: calls.append(args) or 0

    monkeypatch.setattr(Q, "lib", Lib)
    cache = Q.RowCache(4, 2, 16)
    layer = Q.Linear8.__new__(Q.Linear8)
    layer._h, layer.device, layer.segments, layer.in_channels, layer.out_channels = None, -1, 1, 16, 4
    x = zeros(2, 16, dtype=torch.float16)
    for far in (1 << 64, (1 << 64) + 1, -(1 << 64)):
        for bad in (lambda: cache.write(x, row0=far), lambda: cache.read_rows(row0=far, rows=2),
                    lambda: layer.forward_cached(cache, [far])):
            with pytest.raises(pkg.InvalidArgumentError):
                bad()
    assert not calls
    cache.write(x, row0=6), cache.read_rows(row0=6, rows=2), layer.forward_cached(cache, [3])
    assert len(calls) == 3


def test_layer_create_refuses(pkg):
    lib, h = pkg.lib(), ctypes.c_void_p()
    for args in [(FAKE, 1, 8, None, 0, 8, 0, 1), (FAKE, 1, 8, None, 3, 8, 1, 1), (FAKE, 1, 8, None, 4, 8, 0, 3),
                 (FAKE, 1, 8, None, 4, 8, 0, 0), (None, 1, 8, None, 4, 8, 0, 1), (FAKE, 1, 7, None, 4, 8, 0, 1),
                 (FAKE + 1, 1, 8, None, 4, 8, 0, 1), (FAKE, 1, 8, FAKE + 1, 4, 8, 0, 1)]:
        assert lib.dn_linear8_create_device(*args, 0, None, ctypes.byref(h)) == pkg.DN_ERR_INVALID_ARG
    assert lib.dn_linear8_create_device(FAKE, 1, 1 << 18, None, 4, 1 << 18, 0, 1, 0, None,
                                        ctypes.byref(h)) == pkg.DN_ERR_UNSUPPORTED
    assert lib.dn_linear8_create_device(FAKE, 1, 34, None, 4, 34, 0, 17, 0, None,
                                        ctypes.byref(h)) == pkg.DN_ERR_UNSUPPORTED
    assert lib.dn_linear8_create_device(FAKE, 3, 8, None, 4, 8, 0, 1, 0, None, ctypes.byref(h)) == pkg.DN_ERR_DTYPE
    assert h.value is None


def test_layer_create_from_a_store_refuses(pkg, tmp_path):
    store = store_of(pkg, tmp_path, {"a.weight": np.zeros((4, 3, 3, 3), np.float16),
                                     "b.weight": np.zeros((4, 6), np.float16), "b.bias": np.zeros(5, np.float16)})
    h, lib = ctypes.c_void_p(), pkg.lib()

    def create(w, b, gate=0, segments=1):
        return lib.dn_linear8_create(store._h, w, b, gate, segments, 0, ctypes.byref(h))

    assert create(b"none", None) == pkg.DN_ERR_NOT_FOUND
    assert create(b"b.weight", b"none") == pkg.DN_ERR_NOT_FOUND
    assert create(b"a.weight", None) == pkg.DN_ERR_FORMAT
    assert create(b"b.weight", b"b.bias") == pkg.DN_ERR_FORMAT
    assert create(b"b.weight", None, segments=4) == pkg.DN_ERR_INVALID_ARG


# ---------------------------------------------------------------------------------------------------------------------
# The cache
# ---------------------------------------------------------------------------------------------------------------------

@gpu
@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("dtype", [np.float16, np.float32])
@pytest.mark.parametrize("rows,cols,group", [(1, 1, 0), (1, 8, 0), (3, 7, 0), (5, 24, 0), (70, 32, 0), (33, 32, 8),
                                             (9, 64, 16), (6, 96, 0), (13, 192, 64), (7, 520, 0), (40, 512, 32),
                                             (5, 1000, 0), (4, 2048, 0), (3, 2064, 0), (2, 5001, 0), (2, 4608, 2304),
                                             (2, 4096, 0), (3, 9000, 0), (2, 20008, 0)])
def test_codes_and_scales(Q, bits, dtype, rows, cols, group):
    rng = np.random.default_rng(rows * 1000 + cols + bits)
    x = rows_of(rng, rows, cols, dtype)
    cache = Q.RowCache(1, rows + 2, cols, bits=bits, group=group)
    cache.write(dev(x), row0=1)
    q, s = qo.quantise(x, bits, group)
    assert_held(cache, slice(1, rows + 1), q, s, bits)
    for at in (0, rows + 1):
        assert not host(cache.codes)[at].any() and not host(cache.scales)[at].any()
    for out in (torch.float16, torch.float32):
        assert_read(host(cache.read_rows(row0=1, rows=rows, dtype=out)), q, s)
    cache.sync()


@gpu
@pytest.mark.parametrize("bits", [8, 4])
def test_every_pair_of_fp16_significands(Q, bits):
    """Every quotient of two FP16 significands, over the powers of two that
    reach a code: each one falls on its side of a border."""
    sig = np.arange(1024, 2048, dtype=np.float64)
    for j in range(10):
        x = np.concatenate([sig[:, None], np.where(sig[None] / 2 ** j <= sig[:, None], sig[None] / 2 ** j, 0.0)], 1)
        x = np.pad(x, ((0, 0), (0, 7))).astype(np.float16)
        x[:, 1::2] *= -1
        cache = Q.RowCache(1, 1024, x.shape[1], bits=bits)
        cache.write(dev(x))
        assert_held(cache, slice(None), *qo.quantise(x, bits), bits)


@gpu
@pytest.mark.parametrize("bits", [8, 4])
def test_fp32_next_to_a_border(Q, bits):
    """FP32 values at, one step below and one above the middle of two codes."""
    qmax = 127 if bits == 8 else 7
    rng = np.random.default_rng(5)
    a = np.concatenate([rng.uniform(1e-3, 1e3, 60), np.float64(qmax) * np.array([1, 3, 2.0 ** -20, 7])]).astype(np.float32)
    s = a * (np.float32(1) / np.float32(qmax))
    mid = ((np.arange(qmax) + 0.5)[None] * s[:, None].astype(np.float64)).astype(np.float32)
    x = np.concatenate([a[:, None], mid, np.nextafter(mid, np.float32(0)), np.nextafter(mid, np.float32(np.inf))], 1)
    x = np.concatenate([x, -x], 1)
    x = np.where(np.abs(x) <= a[:, None], x, 0).astype(np.float32)
    cache = Q.RowCache(1, len(a), x.shape[1], bits=bits)
    cache.write(dev(x))
    assert_held(cache, slice(None), *qo.quantise(x, bits), bits)


@gpu
@pytest.mark.parametrize("dtype", [np.float16, np.float32])
@pytest.mark.parametrize("cols", [32, 33])
def test_rows_of_zeros_extremes_and_values_that_are_not_finite(Q, dtype, cols):
    top = np.finfo(dtype).max
    least = np.finfo(dtype).smallest_subnormal
    x = np.zeros((10, cols), dtype)
    x[1, 3] = top
    x[2] = -top
    x[3, 0] = least
    x[4] = np.linspace(-1, 1, cols).astype(dtype) * dtype(8) * least
    x[5], x[5, 1] = 1, np.nan
    x[6], x[6, 2] = 1, np.inf
    x[7], x[7, cols - 1] = 1, -np.inf
    x[8] = np.nan
    x[9] = np.linspace(-top, top, cols, dtype=np.float64).astype(dtype)
    for bits in (8, 4):
        cache = Q.RowCache(1, 10, cols, bits=bits)
        cache.write(dev(x))
        q, s = qo.quantise(x, bits)
        assert_held(cache, slice(None), q, s, bits)
        assert_read(host(cache.read_rows(rows=10, dtype=torch.float32)), q, s)


@gpu
@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("dtype", [np.float16, np.float32])
@pytest.mark.parametrize("rows,cols,gap", [(1, 1, 0), (5, 2, 0), (40, 7, 0), (33, 9, 1), (50, 17, 0), (20, 25, 3),
                                           (300, 25, 0), (9, 63, 0), (9, 65, 7), (7, 250, 0), (5, 255, 1), (5, 257, 0),
                                           (4, 333, 2), (3, 505, 0), (3, 1001, 0), (2, 2034, 1), (2, 2035, 0),
                                           (2, 2041, 0), (2, 2047, 0), (20000, 11, 0), (12000, 40, 1)])
def test_rows_that_begin_anywhere(Q, bits, dtype, rows, cols, gap):
    """Rows at every place within 16 bytes: nothing of their neighbours (NaN) is
    taken in, and no byte beside a row's own is written, in the cache or in out."""
    rng = np.random.default_rng(rows + cols)
    x = rows_of(rng, rows, cols, dtype)
    q, s = qo.quantise(x, bits)
    ld, pad = cols + gap, 16
    t = torch.float16 if dtype == np.float16 else torch.float32
    for first in (range(8) if rows < 100 else (0, 3)):
        flat = torch.full((pad + rows * ld + 2 * pad,), float("nan"), dtype=t, device="cuda")
        v = flat[pad + first:].as_strided((rows, cols), (ld, 1))
        v.copy_(dev(x))
        cache = Q.RowCache(1, rows + 2, cols, bits=bits)
        cache.codes.fill_(0xa5)
        cache.scales.fill_(-3.0)
        cache.write(v, row0=1)
        assert_held(cache, slice(1, rows + 1), q, s, bits)
        codes = host(cache.codes)
        assert (codes[:, bytes_of(cols, bits):] == 0xa5).all() and (codes[[0, -1]] == 0xa5).all()
        flat.fill_(7.0)
        cache.read_rows(row0=1, rows=rows, out=v)
        assert_read(host(v.contiguous()), q, s)
        v.fill_(7.0)
        assert (host(flat) == 7.0).all()
        cache.sync()


@gpu
@pytest.mark.parametrize("dtype", [np.float16, np.float32])
@pytest.mark.parametrize("cols,group", [(64, 8), (96, 32), (512, 256), (3 * 2040, 2040)])
def test_groups_of_rows_that_begin_anywhere(Q, dtype, cols, group):
    rng = np.random.default_rng(cols)
    x = rows_of(rng, 21, cols, dtype)
    t = torch.float16 if dtype == np.float16 else torch.float32
    for bits in (8, 4):
        q, s = qo.quantise(x, bits, group)
        for first, ld in ((1, cols), (3, cols + 5), (6, cols + 2)):
            v = torch.full((21 * ld + 16,), float("nan"), dtype=t, device="cuda")[first:].as_strided((21, cols), (ld, 1))
            v.copy_(dev(x))
            cache = Q.RowCache(21, 1, cols, bits=bits, group=group)
            cache.write(v)
            assert_held(cache, slice(None), q, s, bits)
            v.fill_(7.0)
            cache.read_rows(rows=21, out=v)
            assert_read(host(v.contiguous()), q, s)


@gpu
def test_strides_and_alignment(Q):
    rng = np.random.default_rng(3)
    x = rows_of(rng, 9, 64)
    q, s = qo.quantise(x)
    wide = torch.zeros(9, 200, dtype=torch.float16, device="cuda")
    for first in (0, 8, 1):  # the last is no multiple of a vector
        v = wide[:, first:first + 64]
        v.copy_(dev(x))
        cache = Q.RowCache(1, 9, 64)
        cache.write(v)
        assert_held(cache, slice(None), q, s, 8)
        out = torch.full((9, 200), 7.0, dtype=torch.float16, device="cuda")
        cache.read_rows(rows=9, out=out[:, first:first + 64])
        got = host(out)
        assert_read(got[:, first:first + 64], q, s)
        assert (np.delete(got, np.s_[first:first + 64], axis=1) == 7).all()
    one = dev(x)[4:5].expand(9, 64)  # one row over and over: stride 0 is no row stride
    with pytest.raises(ValueError):
        cache.write(one)
    with pytest.raises(ValueError):
        cache.write(dev(x).t())


@gpu
@pytest.mark.parametrize("cols,group", [(1, 0), (24, 0), (33, 0), (40, 8), (48, 16), (64, 0), (64, 32), (200, 0), (250, 0),
                                        (256, 0), (300, 0), (512, 64), (1000, 0), (2049, 0), (2304, 0), (4608, 2304)])
@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("dtype", [np.float16, np.float32])
def test_caches_of_any_alignment(pkg, cols, group, bits, dtype):
    """The C entry points over codes that begin anywhere, with any stride that
    holds a row: written (consecutive and scattered rows) and read back by row and
    by page, and no byte beside a row's own is touched."""
    rng = np.random.default_rng(cols + bits)
    lib, stream = pkg.lib(), torch.cuda.current_stream().cuda_stream
    code, t = (1, torch.float16) if dtype == np.float16 else (0, torch.float32)
    rows, cap, page_rows, n = 13, 24, 5, bytes_of(cols, bits)
    groups = cols // (group or cols)
    x, x2 = rows_of(rng, rows, cols, dtype), rows_of(rng, rows, cols, dtype)
    slots = rng.integers(-1, cap, rows)
    slots[4], slots[9] = slots[1], slots[0]  # the later row counts
    want = np.zeros((cap, cols), dtype)
    want[3:3 + rows] = x
    for r, at in enumerate(slots):
        if at >= 0:
            want[at] = x2[r]
    q, s = qo.quantise(want, bits, group)
    written = np.zeros(cap, bool)
    written[3:3 + rows] = True
    written[slots[slots >= 0]] = True
    table = np.array([[4, 0, 2], [1, 1, 3]], np.int32)
    for first, gap in ((0, 0), (1, 0), (2, 3), (4, 4), (8, 8), (3, 1), (16, (-n) % 16), (8, (-n) % 8), (4, (-n) % 4)):
        ld = n + gap
        flat = torch.full((16 + first + cap * ld + 16,), 0xa5, dtype=torch.uint8, device="cuda")
        scales = torch.full((cap + 2, groups), -3.0, device="cuda")
        err = torch.zeros(1, dtype=torch.int32, device="cuda")
        p, ps = flat.data_ptr() + 16 + first, scales[1:].data_ptr()
        dx, dx2, dslots = dev(x), dev(x2), dev(slots)
        pkg.check(lib.dn_launch_cache_write(dx.data_ptr(), code, cols, rows, cols, None, 3, p, ld, ps, cap, bits, group,
                                            err.data_ptr(), stream))
        pkg.check(lib.dn_launch_cache_write(dx2.data_ptr(), code, cols, rows, cols, dslots.data_ptr(), 0, p, ld, ps, cap,
                                            bits, group, err.data_ptr(), stream))
        held = host(flat)
        body = held[16 + first:16 + first + cap * ld].reshape(cap, ld)
        np.testing.assert_array_equal(body[written][:, :n], qo.pack(q, bits)[written])
        np.testing.assert_array_equal(host(scales)[1:-1][written], s[written])
        assert (body[:, n:] == 0xa5).all() and (body[~written] == 0xa5).all() and (host(scales)[[0, -1]] == -3).all()
        assert (held[:16 + first] == 0xa5).all() and (held[16 + first + cap * ld:] == 0xa5).all()
        out = torch.full((rows, cols), 7.0, dtype=t, device="cuda")
        pkg.check(lib.dn_launch_cache_read_rows(p, ld, ps, cap, cols, bits, group, dslots.data_ptr(), 0, rows, out.data_ptr(),
                                                code, cols, err.data_ptr(), stream))
        got = host(out)
        assert (got[slots < 0] == 7).all()
        assert_read(got[slots >= 0], q[slots[slots >= 0]], s[slots[slots >= 0]])
        pkg.check(lib.dn_launch_cache_read_rows(p, ld, ps, cap, cols, bits, group, None, 3, rows, out.data_ptr(), code, cols,
                                                err.data_ptr(), stream))
        assert_read(host(out), q[3:3 + rows], s[3:3 + rows])
        seqs = torch.full((2, 13, cols), 7.0, dtype=t, device="cuda")
        dt, lengths = dev(table), dev(np.array([12, 7], np.int32))
        pkg.check(lib.dn_launch_cache_read_pages(p, ld, ps, cap, cols, bits, group, page_rows, dt.data_ptr(), 3, 3,
                                                 lengths.data_ptr(), 2, 13, seqs.data_ptr(), code, 13 * cols, cols,
                                                 err.data_ptr(), stream))
        got = host(seqs)
        for b, length in enumerate((12, 7)):
            at = (table[b][:, None] * page_rows + np.arange(page_rows)).ravel()[:length]
            fine = (at < cap) & written[np.minimum(at, cap - 1)]  # the last page ends behind the cache
            assert_read(got[b, :length][fine], q[at[fine]], s[at[fine]])
            assert (got[b, :length][at >= cap] == 7).all() and (got[b, length:] == 7).all()
        assert (host(flat) == held).all()
        assert bool(err.item()) == bool((table * page_rows + page_rows > cap).any())


@gpu
@pytest.mark.parametrize("rows,cols,group", [(1, 32, 0), (40, 32, 0), (256, 24, 0), (300, 32, 0), (2000, 64, 16),
                                             (300, 33, 0), (90, 512, 32), (260, 2304, 0), (30, 2304, 0),
                                             (90, 333, 0), (400, 1001, 0), (2, 5, 0)])
@pytest.mark.parametrize("bits", [8, 4])
def test_scattered_rows_the_last_of_a_slot_counts(Q, rows, cols, group, bits):
    rng = np.random.default_rng(rows + cols)
    x = rows_of(rng, rows, cols)
    capacity = rows + 7
    slots = rng.integers(-2, max(2, rows // 3), rows)  # negative ones, and the same ones over and over
    before = rows_of(rng, capacity, cols)
    cache = Q.RowCache(capacity, 1, cols, bits=bits, group=group)
    cache.write(dev(before))
    cache.write(dev(x), slots=dev(slots))
    want = before.copy()
    for r, at in enumerate(slots):
        if at >= 0:
            want[at] = x[r]
    q, s = qo.quantise(want, bits, group)
    assert_held(cache, slice(None), q, s, bits)
    out = torch.full((rows, cols), 3.0, dtype=torch.float32, device="cuda")
    got = host(cache.read_rows(dev(slots), out=out))
    assert (got[slots < 0] == 3).all()
    assert_read(got[slots >= 0], q[slots[slots >= 0]], s[slots[slots >= 0]])
    cache.sync()


@gpu
@pytest.mark.parametrize("rows", [6, 400])
def test_a_slot_behind_the_cache_is_skipped_and_reported(pkg, Q, rows):
    cache = Q.RowCache(rows, 1, 32)
    x = torch.ones(rows, 32, dtype=torch.float16, device="cuda")
    slots = torch.arange(rows, device="cuda")
    slots[2], slots[3] = rows, 1 << 40
    cache.write(x, slots=slots)
    with pytest.raises(pkg.DenoiserError) as e:
        cache.sync()
    assert e.value.code == pkg.DN_ERR_DEVICE
    cache.sync()  # reported once
    want = np.ones(rows, bool)
    want[2:4] = False
    np.testing.assert_array_equal(host(cache.scales)[:, 0] != 0, want)
    out = cache.read_rows(slots, out=torch.full_like(x, 5.0))
    with pytest.raises(pkg.DenoiserError):
        cache.sync()
    assert (host(out)[2:4] == 5).all() and (host(out)[:2] == 1).all()
    table = torch.tensor([[0, rows, -1]], dtype=torch.int32, device="cuda")
    out = cache.read(table, out=torch.full((1, 3, 32), 5.0, dtype=torch.float16, device="cuda"))
    with pytest.raises(pkg.DenoiserError):
        cache.sync()
    assert (host(out)[0, 0] == 1).all() and (host(out)[0, 1:] == 5).all()


@gpu
@pytest.mark.parametrize("bits,cols,group", [(8, 64, 0), (8, 40, 8), (4, 96, 32), (4, 64, 0), (8, 33, 0), (4, 35, 0),
                                             (8, 640, 0)])
@pytest.mark.parametrize("page_rows", [1, 5, 16])
@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
def test_pages(Q, bits, cols, group, page_rows, dtype):
    """Ragged sequences: nothing, one row, pages that end inside, more than the
    table holds; a page twice; a page that is not there; rows behind stay."""
    rng = np.random.default_rng(cols + page_rows)
    pages, n = 11, 4
    x = rows_of(rng, pages * page_rows, cols)
    cache = Q.RowCache(pages, page_rows, cols, bits=bits, group=group)
    cache.write(dev(x))
    q, s = qo.quantise(x, bits, group)
    most = n * page_rows
    lengths = np.array([0, 1, most, most - 1, most + 100, page_rows + 1, -3], np.int32)
    table = rng.integers(0, pages, (len(lengths), n)).astype(np.int32)
    table[2] = table[2, 0]
    table[4, 1] = -1
    out = torch.full((len(lengths), most + 2, cols), 9.0, dtype=dtype, device="cuda")
    wide = np.concatenate([table, np.full_like(table, 1 << 20)], 1)  # columns that are not of the view
    got = host(cache.read(dev(wide)[:, :n], dev(lengths), out=out))
    for b, length in enumerate(lengths):
        for i in range(most + 2):
            page = table[b, i // page_rows] if i < most else -1
            if i < length and page >= 0:
                r = page * page_rows + i % page_rows
                assert_read(got[b, i:i + 1], q[r:r + 1], s[r:r + 1])
            else:
                assert (got[b, i] == 9).all()
    cache.sync()
    short = host(cache.read(dev(table), dev(lengths), out=torch.zeros(len(lengths), 3, cols, dtype=dtype, device="cuda")))
    np.testing.assert_array_equal(short[2:4, :min(3, most - 1)], got[2:4, :min(3, most - 1)])
    full = host(cache.read(dev(table[:1]), dtype=dtype))
    r = (table[0][:, None] * page_rows + np.arange(page_rows)).ravel()
    assert_read(full[0], q[r], s[r])


@gpu
def test_a_copied_cache(pkg, Q):
    import copy

    rng = np.random.default_rng(12)
    x, x2 = rows_of(rng, 9, 48), rows_of(rng, 9, 48)
    cache = Q.RowCache(3, 3, 48)
    cache.write(dev(x))
    other = copy.deepcopy(cache)
    other.write(dev(x2))
    assert_held(cache, slice(None), *qo.quantise(x), 8)
    assert_held(other, slice(None), *qo.quantise(x2), 8)
    del cache
    torch.cuda.empty_cache()
    q, s = qo.quantise(x2)
    assert_read(host(other.read_rows(rows=9)), q, s)
    other.write(dev(x), slots=torch.full((9,), 9, device="cuda"))
    with pytest.raises(pkg.DenoiserError):
        other.sync()


@gpu
def test_rows_behind_4_gigabytes(Q):
    """Byte offsets past 2^32: 70 million rows of 64 columns."""
    rng = np.random.default_rng(1)
    cache = Q.RowCache(70_000, 1000, 64)
    x = rows_of(rng, 300, 64)
    slots = np.sort(rng.choice(70_000_000, 300, replace=False))
    slots[-1] = 70_000_000 - 1
    assert (slots[-1] + 1) * 64 > 1 << 32
    cache.write(dev(x), slots=dev(slots))
    q, s = qo.quantise(x)
    np.testing.assert_array_equal(host(cache.codes[dev(slots)]), q.view(np.uint8))
    assert_read(host(cache.read_rows(dev(slots), dtype=torch.float32)), q, s)
    last = torch.tensor([[69_999]], dtype=torch.int32, device="cuda")
    got = host(cache.read(last, dtype=torch.float32))[0]
    assert_read(got[-1:], q[-1:], s[-1:])
    w = rows_of(rng, 24, 64)
    layer = Q.Linear8.from_tensors(dev(w))
    y, e = qo.product(q[-1:], s[-1:], *qo.quantise(w))
    assert_product(host(layer.forward_cached(cache, [69_999], out_dtype=torch.float32))[-1:], y, e)
    layer.sync()


# ---------------------------------------------------------------------------------------------------------------------
# Linear8
# ---------------------------------------------------------------------------------------------------------------------

def make(Q, rng, k, n, gate, bias, segments=1, dtype=np.float16):
    w = (rng.standard_normal((n, k)) / np.sqrt(k)).astype(dtype)
    b = (0.3 * rng.standard_normal(n)).astype(dtype) if bias else None
    layer = Q.Linear8.from_tensors(dev(w), None if b is None else dev(b), gate=gate, segments=segments)
    return layer, (*qo.quantise(w), b)


@gpu
@pytest.mark.parametrize("rows,k,n", [
    (1, 1, 1), (1, 512, 1024), (1, 4096, 40), (2, 16, 2), (3, 100, 6), (5, 1000, 520), (8, 64, 64), (16, 48, 130),
    (17, 31, 34), (32, 2048, 66), (33, 128, 256), (64, 4100, 12), (100, 256, 256), (127, 64, 128), (128, 256, 512),
    (129, 257, 514), (130, 32, 8), (200, 96, 200), (300, 64, 258), (257, 1024, 96), (384, 512, 300), (1000, 17, 18),
    (4096, 64, 64), (2500, 640, 160), (700, 33, 1030), (1300, 384, 384), (3, 2047, 70), (4, 4096, 66),
    (8, 2048, 300), (6, 1025, 34), (10, 3, 6), (9, 1024, 520), (13, 1000, 520), (12, 1001, 2368), (16, 777, 130),
    (16, 1024, 2370), (13, 2150, 18), (12, 300, 2400)])
@pytest.mark.parametrize("gate", [False, True])
@pytest.mark.parametrize("x_type,y_type", [(np.float16, torch.float16), (np.float32, torch.float16),
                                           (np.float16, torch.float32)])
def test_token_rows(Q, rows, k, n, gate, x_type, y_type):
    if gate and n % 2:
        n += 1
    rng = np.random.default_rng(rows + k + n)
    layer, (qw, sw, b) = make(Q, rng, k, n, gate, bias=rows % 2 == 0)
    x = rows_of(rng, rows, k, x_type)
    got = host(layer(dev(x), out_dtype=y_type))
    layer.sync()
    assert_product(got, *qo.product(*qo.quantise(x), qw, sw, b, gate))


@gpu
@pytest.mark.parametrize("rows,k,n", [(19000, 300, 256), (5000, 272, 1030), (4999, 520, 1024), (9473, 261, 512)])
@pytest.mark.parametrize("gate", [False, True])
@pytest.mark.parametrize("y_type", [torch.float16, torch.float32])
def test_many_tiles(Q, rows, k, n, gate, y_type):
    """More tiles than SMs, in the widest form."""
    rng = np.random.default_rng(rows)
    layer, (qw, sw, b) = make(Q, rng, k, n, gate, bias=True)
    x = rows_of(rng, rows, k)
    got = host(layer(dev(x), out_dtype=y_type))
    layer.sync()
    assert_product(got, *qo.product(*qo.quantise(x), qw, sw, b, gate))


@gpu
@pytest.mark.parametrize("n_img,k,h,w,n", [(1, 3, 1, 1, 5), (1, 32, 33, 47, 64), (2, 64, 16, 20, 128), (3, 17, 9, 7, 34),
                                           (1, 256, 24, 32, 256), (2, 300, 13, 11, 520), (1, 128, 64, 64, 32),
                                           (2, 16, 1, 129, 8), (1, 512, 8, 16, 64), (5, 48, 3, 5, 96),
                                           (3, 17, 8, 9, 34), (2, 3, 2, 4, 7), (1, 100, 24, 40, 250), (4, 65, 1, 136, 130),
                                           (1, 32, 40, 200, 64), (2, 128, 30, 44, 256), (1, 96, 16, 21, 20), (700, 8, 1, 8, 12),
                                           (1, 700, 20, 30, 300), (3, 260, 8, 12, 290), (2, 1300, 4, 24, 40), (2, 264, 3, 24, 520),
                                           (1, 2000, 1, 77, 33), (1, 130, 48, 100, 258), (2, 4200, 2, 16, 12),
                                           (700, 8, 1, 40, 12), (300, 40, 4, 8, 70)])
@pytest.mark.parametrize("gate", [False, True])
def test_planes(Q, n_img, k, h, w, n, gate):
    if gate and n % 2:
        n += 1
    rng = np.random.default_rng(k + n)
    layer, (qw, sw, b) = make(Q, rng, k, n, gate, bias=True)
    rows = rows_of(rng, n_img * h * w, k)
    x = np.ascontiguousarray(rows.reshape(n_img, h, w, k).transpose(0, 3, 1, 2))
    got = host(layer.forward_nchw(dev(x)))
    layer.sync()
    y, e = qo.product(*qo.quantise(rows), qw, sw, b, gate)
    assert_product(got.transpose(0, 2, 3, 1).reshape(y.shape), y, e)


@gpu
@pytest.mark.parametrize("frames,rows,cols,n", [(1, 1, 16, 2), (1, 200, 64, 64), (2, 129, 20, 6), (3, 1003, 96, 100),
                                                (5, 640, 64, 64), (5, 300, 32, 32), (7, 128, 33, 130), (8, 70, 48, 34),
                                                (4, 257, 200, 300), (2, 500, 512, 512), (8, 390, 128, 256),
                                                (1, 333, 260, 260), (3, 64, 8, 16)])
@pytest.mark.parametrize("gate", [False, True])
@pytest.mark.parametrize("y_type", [torch.float16, torch.float32])
def test_cached_rows(Q, frames, rows, cols, n, gate, y_type):
    rng = np.random.default_rng(frames + rows + cols)
    layer, (qw, sw, b) = make(Q, rng, frames * cols, n, gate, bias=frames % 2 == 1, segments=frames)
    x = rows_of(rng, (frames + 2) * rows, cols)
    x[rows // 2] = 0
    cache = Q.RowCache(frames + 2, rows, cols)
    cache.write(dev(x))
    pages = [int(p) for p in rng.integers(0, frames + 2, frames)]
    q, s = qo.quantise(x)
    q, s = q.reshape(-1, rows, cols)[pages], s.reshape(-1, rows, 1)[pages]
    q, s = np.concatenate(list(q), 1), np.concatenate(list(s), 1)
    y, e = qo.product(q, s, qw, sw, b, gate, frames)
    assert_product(host(layer.forward_cached(cache, pages, out_dtype=y_type)), y, e)
    part = rows // 2 + 1
    out = torch.full((part + 3, y.shape[1] + 5), 4.0, dtype=y_type, device="cuda")
    layer.forward_cached(cache, pages, rows=part, out=out[:part, 2:2 + y.shape[1]])
    layer.sync()
    got = host(out)
    assert_product(got[:part, 2:2 + y.shape[1]], y[:part], e[:part])
    assert (got[part:] == 4).all() and (got[:, :2] == 4).all() and (got[:, 2 + y.shape[1]:] == 4).all()


@gpu
@pytest.mark.parametrize("rows,k,n", [(4, 64, 32), (150, 64, 96), (300, 700, 80)])
def test_strided_rows_and_what_lies_around_the_output(Q, rows, k, n):
    rng = np.random.default_rng(rows)
    layer, (qw, sw, b) = make(Q, rng, k, n, False, True)
    x = rows_of(rng, rows, k)
    y, e = qo.product(*qo.quantise(x), qw, sw, b)
    for first, off in ((0, 0), (8, 16), (3, 1)):
        wide = torch.zeros(rows, k + 24, dtype=torch.float16, device="cuda")
        wide[:, first:first + k] = dev(x)
        out = torch.full((rows + 2, n + 40), 4.0, dtype=torch.float16, device="cuda")
        layer(wide[:, first:first + k], out=out[1:rows + 1, off:off + n])
        got = host(out)
        assert_product(got[1:rows + 1, off:off + n], y, e)
        assert (got[0] == 4).all() and (got[-1] == 4).all()
        assert (np.delete(got, np.s_[off:off + n], axis=1) == 4).all()


@gpu
@pytest.mark.parametrize("rows,k", [(5, 64), (200, 64), (200, 600)])
def test_rows_that_are_not_finite_stay_by_themselves(Q, rows, k):
    rng = np.random.default_rng(k)
    layer, (qw, sw, b) = make(Q, rng, k, 48, True, True)
    x = rows_of(rng, rows, k)
    x[1, 3], x[2] = np.inf, np.nan
    x[3] = 0
    got = host(layer(dev(x)))
    assert np.isnan(got[1:3]).all() and np.isfinite(np.delete(got, [1, 2], axis=0)).all()
    assert_product(got, *qo.product(*qo.quantise(x), qw, sw, b, True))
    pix = host(layer.forward_nchw(dev(x.T.reshape(1, k, 1, rows))))
    np.testing.assert_array_equal(pix[0, :, 0].T, got)


def far_rows(rng, rows, k):
    """FP32 tokens from 2^-100 to the largest numbers, far ones beside ordinary ones."""
    x = rng.standard_normal((rows, k)) * 2.0 ** np.resize([0, 125, -100, 96, 103, 124, 20], rows)[:, None]
    return np.clip(x, -np.finfo(np.float32).max, np.finfo(np.float32).max).astype(np.float32)


@gpu
@pytest.mark.parametrize("rows,k,n", [(1, 512, 40), (2, 64, 8), (3, 300, 66), (7, 512, 1024), (13, 1000, 34),
                                      (150, 512, 96), (260, 100, 200), (700, 1030, 520), (129, 64, 30)])
@pytest.mark.parametrize("gate", [False, True])
@pytest.mark.parametrize("y_type", [torch.float16, torch.float32])
def test_tokens_far_from_one(Q, rows, k, n, gate, y_type):
    """The output is finite although the sum of codes times the token's scale is
    not (and the sum times the channel's scale alone is far below one)."""
    rng = np.random.default_rng(rows + n)
    x = far_rows(rng, rows + 1, k)[1:]  # the single token is a far one
    w = (rng.standard_normal((n, k)) * 2.0 ** -120 / np.sqrt(k)).astype(np.float32)
    b = rng.standard_normal(n).astype(np.float32)
    layer = Q.Linear8.from_tensors(dev(w), dev(b), gate=gate)
    q, s = qo.quantise(x)
    y, e = qo.product(q, s, *qo.quantise(w), b, gate)
    sums = q.astype(np.float64) @ qo.quantise(w)[0].astype(np.float64).T
    assert np.abs(sums * s).max() > 2.0 ** 128 and np.abs(y).max() < 60000
    got = host(layer(dev(x), out_dtype=y_type))
    layer.sync()
    assert np.isfinite(got).all()
    assert_product(got, y, e)


@gpu
@pytest.mark.parametrize("frames,rows,cols,n", [(1, 300, 64, 64), (2, 130, 20, 6), (3, 203, 96, 100), (5, 170, 64, 64),
                                                (8, 390, 128, 256)])
@pytest.mark.parametrize("gate", [False, True])
@pytest.mark.parametrize("y_type", [torch.float16, torch.float32])
def test_cached_rows_far_from_one(Q, frames, rows, cols, n, gate, y_type):
    rng = np.random.default_rng(frames + rows)
    x = far_rows(rng, frames * rows, cols)
    w = (rng.standard_normal((n, frames * cols)) * 2.0 ** -120 / np.sqrt(cols)).astype(np.float32)
    b = rng.standard_normal(n).astype(np.float32)
    layer = Q.Linear8.from_tensors(dev(w), dev(b), gate=gate, segments=frames)
    cache = Q.RowCache(frames, rows, cols)
    cache.write(dev(x))
    q, s = (np.concatenate(list(a.reshape(frames, rows, -1)), 1) for a in qo.quantise(x))
    y, e = qo.product(q, s, *qo.quantise(w), b, gate, frames)
    assert np.abs(y).max() < 60000
    got = host(layer.forward_cached(cache, list(range(frames)), out_dtype=y_type))
    layer.sync()
    assert np.isfinite(got).all()
    assert_product(got, y, e)


@gpu
@pytest.mark.parametrize("n", [1, 2, 5, 9, 12, 20, 33, 100, 259, 854])
@pytest.mark.parametrize("k", [40, 300])
@pytest.mark.parametrize("y_type", [torch.float16, torch.float32])
def test_rows_with_something_beside_them(Q, n, k, y_type):
    """Output rows of any length with an aligned stride: what lies between them,
    in front of the first and behind the last one stays as it was."""
    rng = np.random.default_rng(n + k)
    ld = (n + 7) // 8 * 8 + 8
    cached = Q.RowCache(2, 150, k)
    for rows in (5, 74, 150):
        for gate in (False, True):
            layer, (qw, sw, b) = make(Q, rng, k, 2 * n if gate else n, gate, True)
            x = rows_of(rng, rows, k)
            y, e = qo.product(*qo.quantise(x), qw, sw, b, gate)
            cached.write(dev(x))
            for off in (0, 8, 4):
                def calls():
                    yield lambda o: layer(dev(x), out=o)
                    yield lambda o: layer(dev(x.astype(np.float32)), out=o)
                    yield lambda o: layer.forward_cached(cached, [0], rows=rows, out=o)
                for call in calls():
                    flat = torch.full((16 + (rows + 1) * ld,), 9.0, dtype=y_type, device="cuda")
                    out = flat[16 + off:].as_strided((rows, n), (ld, 1))
                    call(out)
                    assert_product(host(out.contiguous()), y, e)
                    out.fill_(9.0)
                    assert (host(flat) == 9).all()
            layer.sync()
        pair, (qp, sp, bp) = make(Q, rng, 2 * k, n, False, True, segments=2)
        flat = torch.full(((rows + 1) * ld,), 9.0, dtype=y_type, device="cuda")
        out = flat.as_strided((rows, n), (ld, 1))
        pair.forward_cached(cached, [0, 0], rows=rows, out=out)
        q, s = qo.quantise(x)
        assert_product(host(out.contiguous()), *qo.product(np.concatenate([q, q], 1), np.concatenate([s, s], 1), qp, sp, bp,
                                                           False, 2))
        out.fill_(9.0)
        assert (host(flat) == 9).all()


@gpu
def test_in_place_calls_are_refused_and_columns_side_by_side_are_not(pkg, Q):
    rng = np.random.default_rng(5)
    layer, (qw, sw, b) = make(Q, rng, 32, 32, False, True)
    one = Q.Linear8.from_tensors(torch.ones(8, 32, dtype=torch.float16, device="cuda"))
    for rows in (1, 3, 40, 300):
        flat = torch.zeros(rows * 64 + 200, dtype=torch.float16, device="cuda")
        x = flat[:rows * 32].view(rows, 32)
        shifted = flat[16:16 + rows * 32].view(rows, 32)
        wide = flat[:rows * 64].view(rows, 64)
        floats = flat[:rows * 64].view(torch.float32).view(rows, 32)
        for bad in (lambda: layer(x, out=x), lambda: layer(x, out=shifted), lambda: layer(shifted, out=x),
                    lambda: layer(wide[:, :32], out=wide[:, 16:48]), lambda: layer(wide[:, 24:56], out=wide[:, :32]),
                    lambda: layer(floats, out=wide[:, :32]), lambda: one(x, out=x[:, 24:]),
                    lambda: layer.forward_nchw(x.view(1, 32, rows, 1), out=shifted.view(1, 32, rows, 1))):
            with pytest.raises(pkg.InvalidArgumentError):
                bad()
        assert not bool(flat.any())
        x0 = rows_of(rng, rows, 32)
        y, e = qo.product(*qo.quantise(x0), qw, sw, b)
        for i, o in ((slice(0, 32), slice(32, 64)), (slice(32, 64), slice(0, 32))):  # one buffer, side by side
            wide[:, i] = dev(x0)
            layer(wide[:, i], out=wide[:, o])
            assert_product(host(wide[:, o]), y, e)
            np.testing.assert_array_equal(host(wide[:, i]), x0)
        x.copy_(dev(x0))  # one behind the other
        assert_product(host(layer(x, out=flat[rows * 32:rows * 64].view(rows, 32))), y, e)


@gpu
def test_the_longest_sum(Q):
    """131072 channels, every product of codes 127 * 127: the int32 sum's limit."""
    k = 131072
    x = torch.ones(20, k, dtype=torch.float16, device="cuda")
    x[1::2] = -1
    layer = Q.Linear8.from_tensors(torch.full((40, k), 0.5, dtype=torch.float16, device="cuda"))
    for rows in (1, 20):
        y, e = qo.product(*qo.quantise(host(x[:rows])), *qo.quantise(np.full((40, k), 0.5, np.float16)))
        assert_product(host(layer(x[:rows], out_dtype=torch.float32)), y, e)
    layer.sync()


@gpu
def test_behind_a_long_kernel(Q):
    """The product's weight loads run ahead of the earlier work on the stream;
    its bounded waits do not begin before that is done."""
    rng = np.random.default_rng(9)
    layer, (qw, sw, b) = make(Q, rng, 2048, 600, False, True)
    x = rows_of(rng, 200, 2048)
    dx = dev(x)
    torch.cuda._sleep(int(2.6 * 1.965e9))
    got = layer(dx)
    layer.sync()
    assert_product(host(got), *qo.product(*qo.quantise(x), qw, sw, b))


@gpu
def test_no_rows_is_no_work(Q):
    layer = Q.Linear8.from_tensors(torch.ones(6, 32, dtype=torch.float16, device="cuda"))
    assert layer(torch.zeros(0, 32, dtype=torch.float16, device="cuda")).shape == (0, 6)
    assert layer.forward_nchw(torch.zeros(2, 32, 0, 4, dtype=torch.float16, device="cuda")).shape == (2, 6, 0, 4)
    cache = Q.RowCache(0, 4, 32)
    cache.write(torch.zeros(0, 32, dtype=torch.float16, device="cuda"))
    assert cache.read_rows(rows=0).shape == (0, 32)
    assert cache.read(torch.zeros(2, 0, dtype=torch.int32, device="cuda")).shape == (2, 0, 32)
    cache = Q.RowCache(2, 4, 32)
    assert layer.forward_cached(cache, [1], rows=0).shape == (0, 6)


@gpu
def test_layers_from_a_store_and_from_tensors_are_the_same(pkg, Q, tmp_path):
    rng = np.random.default_rng(2)
    w, b = (rng.standard_normal((34, 20)) / 4).astype(np.float16), rng.standard_normal(34).astype(np.float16)
    store = store_of(pkg, tmp_path, {"c.weight": w.reshape(34, 20, 1, 1), "c.bias": b, "d.weight": w})
    x = dev(rows_of(rng, 50, 20))
    want = host(Q.Linear8.from_tensors(dev(w), dev(b), gate=True)(x))
    layer = Q.Linear8(store, "c.weight", "c.bias", gate=True)
    assert (layer.in_channels, layer.out_channels, layer.gate, layer.segments) == (20, 17, True, 1)
    np.testing.assert_array_equal(host(layer(x)), want)
    np.testing.assert_array_equal(host(Q.Linear8(store, "d.weight")(x)), host(Q.Linear8.from_tensors(dev(w))(x)))


@gpu
def test_a_layer_that_finds_no_memory_does_not_fail_the_next_one(pkg, Q, tmp_path):
    """The failed allocation is reported once, by the call that made it."""
    big, small = np.zeros((4096, 4096), np.float16), np.ones((8, 16), np.float16)
    store = store_of(pkg, tmp_path, {"big.weight": big, "small.weight": small})
    Q.Linear8(store, "small.weight")(torch.ones(2, 16, dtype=torch.float16, device="cuda"))
    torch.cuda.synchronize()
    torch.cuda.empty_cache()
    taken = []
    while torch.cuda.mem_get_info()[0] > 60 << 20:  # the layer's weight passes through 64 MB
        taken.append(torch.empty(torch.cuda.mem_get_info()[0] - (40 << 20), dtype=torch.uint8, device="cuda"))
    with pytest.raises(pkg.DenoiserError) as e:
        Q.Linear8(store, "big.weight")
    assert e.value.code == pkg.DN_ERR_CUDA
    del taken
    torch.cuda.empty_cache()
    layer = Q.Linear8(store, "small.weight")
    x = torch.ones(2, 16, dtype=torch.float16, device="cuda")
    assert bool((layer(x) == 16).all())
    Q.Linear8(store, "big.weight")


@gpu
def test_layers_of_a_device_that_is_not_there_are_refused(pkg, tmp_path):
    store = store_of(pkg, tmp_path, {"b.weight": np.ones((4, 16), np.float16)})
    w, lib, h = torch.ones(4, 16, dtype=torch.float16, device="cuda"), pkg.lib(), ctypes.c_void_p()
    for device in (-1, torch.cuda.device_count()):
        assert lib.dn_linear8_create(store._h, b"b.weight", None, 0, 1, device, ctypes.byref(h)) == pkg.DN_ERR_INVALID_ARG
        assert lib.dn_linear8_create_device(w.data_ptr(), 1, 16, None, 4, 16, 0, 1, device, None,
                                            ctypes.byref(h)) == pkg.DN_ERR_INVALID_ARG
    assert h.value is None and torch.cuda.current_device() == 0


@gpu
def test_calls_refuse(pkg, Q):
    h = torch.float16
    layer = Q.Linear8.from_tensors(torch.ones(6, 32, dtype=h, device="cuda"))
    two = Q.Linear8.from_tensors(torch.ones(6, 32, dtype=h, device="cuda"), segments=2)
    x = torch.ones(4, 32, dtype=h, device="cuda")
    cache, c4 = Q.RowCache(3, 4, 32), Q.RowCache(3, 4, 32, bits=4)
    c16 = Q.RowCache(3, 4, 16)
    bad = [lambda: layer(x[:, :31]), lambda: layer(x.cpu()), lambda: layer(x.t().contiguous().t()),
           lambda: layer(x, out=torch.empty(4, 5, dtype=h, device="cuda")), lambda: two(x),
           lambda: two.forward_nchw(x.reshape(1, 32, 2, 2)), lambda: layer.forward_nchw(x),
           lambda: layer.forward_cached(c4, [0]), lambda: layer.forward_cached(c16, [0]),
           lambda: layer.forward_cached(cache, [3]), lambda: layer.forward_cached(cache, [-1]),
           lambda: layer.forward_cached(cache, [0, 1]), lambda: two.forward_cached(c16, [0]),
           lambda: layer.forward_cached(cache, [0], rows=5), lambda: layer.forward_cached(cache, [0], rows=-1),
           lambda: cache.write(x, row0=9), lambda: cache.write(x, slots=torch.arange(3, device="cuda")),
           lambda: cache.write(x, slots=torch.arange(4, device="cuda", dtype=torch.int32)),
           lambda: cache.read_rows(), lambda: cache.read_rows(row0=10, rows=3),
           lambda: cache.read(torch.zeros(1, 2, device="cuda")),
           lambda: cache.read(torch.zeros(1, 2, dtype=torch.int32, device="cuda"), torch.zeros(2, dtype=torch.int32, device="cuda"))]
    for i, f in enumerate(bad):
        with pytest.raises(pkg.InvalidArgumentError):
            f()
            raise AssertionError(f"call {i} was not refused")
    for f in (lambda: layer(x.double()), lambda: cache.write(x.to(torch.bfloat16)),
              lambda: layer(x, out_dtype=torch.bfloat16), lambda: layer.forward_nchw(x.float().reshape(1, 32, 2, 2))):
        with pytest.raises(pkg.DenoiserError) as e:
            f()
        assert e.value.code == pkg.DN_ERR_DTYPE
    lib, n = pkg.lib(), ctypes.c_int64()
    big = torch.ones(600, 32, device="cuda")
    out = torch.empty(600, 6, dtype=h, device="cuda")
    for rows in (1, 600):
        pkg.check(lib.dn_linear8_workspace(layer._h, rows, 0, 0, ctypes.byref(n)))
        if n.value:
            ws = torch.empty(n.value + 16, dtype=torch.uint8, device="cuda")
            for p, size in ((None, n.value), (ws.data_ptr(), n.value - 1), (ws.data_ptr() + 4, n.value)):
                assert lib.dn_linear8_forward(layer._h, big.data_ptr(), 0, 32, rows, out.data_ptr(), 1, 6, p, size,
                                              None) == pkg.DN_ERR_INVALID_ARG


# ---------------------------------------------------------------------------------------------------------------------
# Frames of a temporal model in the cache
# ---------------------------------------------------------------------------------------------------------------------

class FakeModel:
    """encode: 10 times the frame, in the slot; decode: the window's slots."""

    def __init__(self, T):
        self.slots, self.encoded, self.num_frames = [None] * T, 0, T

    def encode_frame(self, x, slot, stream=None):
        self.slots[slot] = float(x.ravel()[0]) * 10
        self.encoded += 1

    def decode_window(self, slots, beauty, stream=None):
        return [(tuple(self.slots[s] for s in slots), float(beauty.ravel()[0]))]


class FakeStore:
    """Adds a quarter to what it holds, so that a frame past it shows."""

    def __init__(self, model, h=2, w=2):
        self.model, self.held, self.h, self.w = model, {}, h, w

    def park(self, slot, entry, stream=None):
        self.held[entry] = self.model.slots[slot] + 0.25

    def restore(self, entry, slot, stream=None):
        self.model.slots[slot] = self.held[entry]


@pytest.mark.parametrize("T", [3, 5])
def test_streams_served_in_turn(pkg, T):
    """Every frame is encoded once, and every window is its clip's, each frame
    as it comes out of the store."""
    S = importlib.import_module(pkg.__name__ + ".sharding")
    lengths = [6, 1, 4]
    clips = [(lambda f, k=k: torch.full((3, 2, 2), 100.0 * k + f), n) for k, n in enumerate(lengths)]
    m = FakeModel(T)
    got = S.denoise_streams(m, clips, T, store=FakeStore(m))
    assert [(k, i) for k, i, _ in got] == [(k, i) for i in range(6) for k in range(3) if i < lengths[k]]
    for k, i, y in got:
        want = tuple((100.0 * k + f) * 10 + 0.25 for f in S.window(i, T, lengths[k]))
        assert y == (want, 100.0 * k + i)
    assert m.encoded == sum(lengths)
    with pytest.raises(ValueError):
        S.denoise_streams(m, clips, 4)
    assert S.denoise_streams(m, [], T) == []
    for store in (FakeStore(m, 2, 4), FakeStore(FakeModel(T))):
        with pytest.raises(ValueError):
            S.denoise_streams(m, clips, T, store=store)
    with pytest.raises(ValueError):
        S.denoise_streams(m, clips + [(lambda f: torch.zeros(3, 2, 4), 2)], T, store=FakeStore(m))


def small_temporal(pkg, tmp_path, kind, T):
    synth = importlib.import_module(pkg.__name__ + ".synth")
    cfg = synth.NAFConfig(base_channels=8, enc_blocks=(1, 1), middle_blocks=1, dec_blocks=(1, 1))
    return pkg.Model(synth.make_model_dir(str(tmp_path), cfg, 4, kind, T, True)[0])


@gpu
@pytest.mark.parametrize("kind,T", [("legacy", 3), ("py", 5)])
@pytest.mark.parametrize("bits", [8, 4])
def test_streams_through_the_frame_store(pkg, Q, tmp_path, kind, T, bits):
    """A parked frame is its features' codes; outputs of clips in turn are those
    of a decode whose slots hold the values that the codes stand for, and do not
    depend on the other clips."""
    S = importlib.import_module(pkg.__name__ + ".sharding")
    m = small_temporal(pkg, tmp_path, kind, T)
    H, W = 30, 42
    rng = np.random.default_rng(6)
    clips = [[dev(rng.uniform(0, 1, (3, H, W)).astype(np.float16)) for _ in range(n)] for n in (5, 3)]
    store = Q.FrameStore(m, H, W, 2, bits=bits)
    m.encode_frame(clips[0][1].unsqueeze(0), 1)
    raw = [host(m.frame_features(H, W, 1, l)).copy() for l in range(m.num_levels + 1)]
    assert [r.shape[1] for r in raw] == m.enc_channels + [2 * m.enc_channels[-1]]
    store.park(1, 1)
    store.restore(1, 0)
    for l, (r, c) in enumerate(zip(raw, store.caches)):
        q, s = qo.quantise(r, bits)
        assert_held(c, slice(c.page_rows, 2 * c.page_rows), q, s, bits)
        assert_read(host(m.frame_features(H, W, 0, l)), q, s)
        np.testing.assert_array_equal(host(m.frame_features(H, W, 1, l)), r)
        c.sync()
    take = [(lambda f, c=c: c[f], len(c)) for c in clips]
    both = {(k, i): y.clone() for k, i, y in S.denoise_streams(m, take, T, bits=bits)}
    m.sync()
    assert sorted(both) == [(k, i) for k, c in enumerate(clips) for i in range(len(c))]
    for k, c in enumerate(clips):
        alone = {i: y.clone() for _, i, y in S.denoise_streams(m, [take[k]], T, bits=bits)}
        for i in range(len(c)):
            assert torch.equal(alone[i], both[k, i]), (k, i)
    for i in (0, 3):
        win = S.window(i, T, 5)
        for f in dict.fromkeys(win):
            m.encode_frame(clips[0][f].unsqueeze(0), f % T)
            for l in range(m.num_levels + 1):
                v = m.frame_features(H, W, f % T, l)
                q, s = qo.quantise(host(v), bits)
                # the FP32 product of code and scale, rounded to FP16, as the cache reads it
                v.copy_(dev((q.astype(np.float32) * s).astype(np.float16)))
        want = m.decode_window([f % T for f in win], clips[0][i].unsqueeze(0))[0]
        assert torch.equal(both[0, i], want), i
    for bad in (lambda: store.park(1, 2), lambda: store.restore(-1, 0), lambda: store.park(T, 0),
                lambda: m.frame_features(H, W, 0, m.num_levels + 1), lambda: m.frame_features(H, W, 0, -1)):
        with pytest.raises(pkg.InvalidArgumentError):
            bad()
    assert store.bytes < sum(r.nbytes for r in raw) * 2


@gpu
def test_a_slot_without_a_frame_of_the_size_is_not_parked(pkg, Q, tmp_path):
    """Nothing is held that was not encoded: another frame size drops the slots,
    a store that is made or that refuses drops none."""
    m = small_temporal(pkg, tmp_path, "py", 3)
    rng = np.random.default_rng(3)
    small = dev(rng.uniform(0, 1, (1, 3, 30, 42)).astype(np.float16))
    large = dev(rng.uniform(0, 1, (1, 3, 46, 42)).astype(np.float16))
    store = Q.FrameStore(m, 30, 42, 2)
    assert m.slot_frame(1) == (0, 0)
    with pytest.raises(pkg.InvalidArgumentError):
        store.park(1, 0)  # nothing was ever encoded
    m.encode_frame(small, 1)
    assert [m.slot_frame(s) for s in range(3)] == [(0, 0), (30, 42), (0, 0)]
    want = [host(m.frame_features(30, 42, 1, l)).copy() for l in range(m.num_levels + 1)]
    store.park(1, 0)
    held = [host(c.codes).copy() for c in store.caches]
    other = Q.FrameStore(m, 46, 42, 1)  # made for another size: the slots stay
    assert m.slot_frame(1) == (30, 42)
    for bad in (lambda: other.park(1, 0), lambda: store.park(0, 1), lambda: store.park(3, 1), lambda: m.slot_frame(-1),
                lambda: m.feature_shape(30, 42, -1), lambda: m.feature_shape(0, 42, 0)):
        with pytest.raises(pkg.InvalidArgumentError):
            bad()
    for l, f in enumerate(want):
        assert m.feature_shape(30, 42, l) == f.shape
        np.testing.assert_array_equal(host(m.frame_features(30, 42, 1, l)), f)
    assert not any(host(c.codes).any() for c in other.caches)
    m.encode_frame(large, 1)
    assert m.slot_frame(1) == (46, 42)
    with pytest.raises(pkg.InvalidArgumentError):
        store.park(1, 0)  # the slot holds a frame of the other size
    other.park(1, 0)
    m.encode_frame(small, 0)  # drops slot 1 once more
    with pytest.raises(pkg.InvalidArgumentError):
        store.park(1, 0)
    for c, codes in zip(store.caches, held):
        np.testing.assert_array_equal(host(c.codes), codes)
    store.restore(0, 2)
    assert [m.slot_frame(s) for s in range(3)] == [(30, 42), (0, 0), (30, 42)]
    for l, f in enumerate(want):
        assert_read(host(m.frame_features(30, 42, 2, l)), *qo.quantise(f))
    store.park(2, 1)
    m(torch.cat([large] * 3).unsqueeze(0))  # a whole clip fills all slots
    assert [m.slot_frame(s) for s in range(3)] == [(46, 42)] * 3
    other.restore(0, 0)
    m.sync()


@gpu
def test_streams_on_a_stream_of_their_own(pkg, Q, tmp_path):
    """The store is made on the stream it is used on: what the current stream
    does later does not reach it."""
    S = importlib.import_module(pkg.__name__ + ".sharding")
    m = small_temporal(pkg, tmp_path, "py", 3)
    rng = np.random.default_rng(7)
    clips = [[dev(rng.uniform(0, 1, (3, 30, 42)).astype(np.float16)) for _ in range(4)] for _ in range(2)]
    take = [(lambda f, c=c: c[f], 4) for c in clips]
    want = [y.clone() for _, _, y in S.denoise_streams(m, take, 3)]
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    torch.cuda._sleep(20_000_000)
    got = S.denoise_streams(m, take, 3, stream=side)
    torch.cuda.synchronize()
    for (k, i, y), w in zip(got, want):
        assert torch.equal(y, w), (k, i)


# ---------------------------------------------------------------------------------------------------------------------
# Together
# ---------------------------------------------------------------------------------------------------------------------

@gpu
def test_a_run_of_all_of_them(Q):
    """Frames come one by one: an 8-bit layer makes their features, the cache
    holds the last five (frame f in page f % 5), the fusion layer reads the
    window from it, and a window is read back."""
    rng = np.random.default_rng(8)
    rows, c, T = 210, 32, 5
    make_f, (qf, sf, bf) = make(Q, rng, 12, 2 * c, True, True)
    fuse, (qg, sg, bg) = make(Q, rng, T * c, 24, False, True, segments=T)
    cache = Q.RowCache(T, rows, c)
    feats = []
    for f in range(8):
        x = rows_of(rng, rows, 12)
        y = make_f(dev(x))
        assert_product(host(y), *qo.product(*qo.quantise(x), qf, sf, bf, True))
        feats.append(host(y))
        cache.write(y, row0=(f % T) * rows)
        if f < 2:
            continue
        window = [min(max(f - T + 1 + t, 0), f) for t in range(T)]  # the first one over and over at the start
        held = [qo.quantise(feats[i]) for i in window]
        q, s = np.concatenate([a for a, _ in held], 1), np.concatenate([b for _, b in held], 1)
        got = fuse.forward_cached(cache, [i % T for i in window])
        assert_product(host(got), *qo.product(q, s, qg, sg, bg, False, T))
        table = torch.tensor([[i % T for i in window]], dtype=torch.int32, device="cuda")
        back = host(cache.read(table))[0].reshape(T, rows, c)
        for t in range(T):
            assert_read(back[t], *held[t])
    cache.sync()
    make_f.sync()
    fuse.sync()


@gpu
@pytest.mark.parametrize("rows,k", [(3, 256), (500, 64), (500, 600)])
def test_streams_and_two_calls_at_once(Q, rows, k):
    rng = np.random.default_rng(rows)
    layer, (qw, sw, b) = make(Q, rng, k, 64, False, True)
    xs = [rows_of(rng, rows, k) for _ in range(6)]
    want = [host(layer(dev(x))) for x in xs]
    dxs = [dev(x) for x in xs]
    streams = [torch.cuda.Stream() for _ in range(3)]
    torch.cuda.synchronize()
    for _ in range(5):
        got = [layer(x, stream=streams[i % 3]) for i, x in enumerate(dxs)]
        for g, w in zip(got, want):
            np.testing.assert_array_equal(host(g), w)


@gpu
@pytest.mark.parametrize("rows", [2, 400])
def test_captured_and_replayed(Q, rows):
    """Write, fusion and read-back in one graph, replayed on new inputs and
    slots; two graphs of one layer replayed at the same time."""
    rng = np.random.default_rng(rows)
    layer, (qw, sw, b) = make(Q, rng, 64, 48, False, True)
    pair, (qp, sp, bp) = make(Q, rng, 128, 32, False, False, segments=2)
    cache = Q.RowCache(2, rows, 48)
    cache2 = Q.RowCache(2, rows, 64)
    x = torch.zeros(rows, 64, dtype=torch.float16, device="cuda")
    slots = torch.zeros(rows, dtype=torch.int64, device="cuda")

    def step():
        y = layer(x)
        cache.write(y, slots=slots)
        cache2.write(x, row0=rows)
        return y, cache.read_rows(slots), pair.forward_cached(cache2, [1, 1])

    graphs = []
    for _ in range(2):
        s = torch.cuda.Stream()
        with torch.cuda.stream(s):
            step()
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs = step()
        graphs.append((g, outs))
    for i in range(4):
        xs = rows_of(rng, rows, 64)
        at = rng.permutation(2 * rows)[:rows]
        x.copy_(dev(xs))
        slots.copy_(dev(at))
        for g, _ in graphs:
            g.replay()
        q, s = qo.quantise(xs)
        y, e = qo.product(q, s, qw, sw, b)
        yp, ep = qo.product(np.concatenate([q, q], 1), np.concatenate([s, s], 1), qp, sp, None, False, 2)
        for _, (ya, back, fused) in graphs:
            assert_product(host(ya), y, e)
            assert_read(host(back), *qo.quantise(host(ya)))
            assert_product(host(fused), yp, ep)
    streams = [torch.cuda.Stream() for _ in graphs]
    torch.cuda.synchronize()
    layers = []
    for s in streams:  # two graphs of the one layer, each with its own workspace
        xin = dev(rows_of(rng, rows, 64))
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            out = layer(xin)
        layers.append((g, xin, out))
    want = [host(layer(xin)) for _, xin, _ in layers]
    for _ in range(10):
        for (g, _, _), s in zip(layers, streams):
            with torch.cuda.stream(s):
                g.replay()
    for (_, _, out), w in zip(layers, want):
        np.testing.assert_array_equal(host(out), w)


@gpu
def test_the_same_call_gives_the_same_bits(Q):
    rng = np.random.default_rng(4)
    for rows, k, n in ((7, 900, 66), (900, 64, 96), (900, 900, 300)):
        layer, _ = make(Q, rng, k, n, True, True)
        x = dev(rows_of(rng, rows, k))
        first = host(layer(x))
        for _ in range(3):
            np.testing.assert_array_equal(host(layer(x)), first)
