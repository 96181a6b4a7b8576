"""MXFP4 rows (nemo_mxfp4_quantize, nemo_mxfp4_dequantize) and their product (nemo_gemm_mxfp4)
against plain 64-bit forms."""
import ctypes as C

import numpy as np
import pytest
import torch

import nemoasr_b200 as nb
import operators_ref as R

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _no_device_errors():
    yield
    torch.cuda.synchronize()
    assert nb.api().nemo_gpu_check_device_errors() == 0, nb.api().nemo_gpu_last_error().decode()


def rows_of(rng, r, k, elt):
    x = rng.standard_normal((r, k)) * np.exp(rng.standard_normal((r, 1)) * 2)
    return R.to_dev(x.astype(np.float32), elt)


# ---- quantisation --------------------------------------------------------------------------

@pytest.mark.parametrize("elt", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("r,k", [(1, 32), (3, 64), (7, 1024), (31, 96), (128, 128), (129, 160), (257, 4096)])
def test_quantise(r, k, elt):
    x = rows_of(np.random.default_rng(r * k), r, k, elt)
    q, s = R.gpu_quantise(x, elt)
    code, byte = R.unpack(q, s, k)
    want_code, want_byte = R.quantise(R.f64(x))
    assert np.array_equal(byte, want_byte)
    assert np.array_equal(code, want_code)
    # bytes of a row's columns past the last block are 0; those of rows past the last are left alone
    sb = s.cpu().numpy()
    at = R.scale_index(-(-r // 128) * 128, -(-k // 128) * 4)
    assert (sb[at[:r, k // 32:]] == 0).all()
    assert (sb[at[r:]] == 0xEE).all()
    y = torch.empty_like(x)
    nb.check(nb.api().nemo_mxfp4_dequantize(q.data_ptr(), k // 2, s.data_ptr(), r, k, y.data_ptr(), R.ELT[elt][1], k, R.stream_ptr()), "dequantize")
    v = R.values(want_code, want_byte)
    assert np.array_equal(R.f64(y), R.f64(torch.from_numpy(v).to(R.ELT[elt][0])))


def test_quantise_borders():
    """Ties, saturation, signs, zeros, the smallest and largest magnitudes, infinities and NaN."""
    base = np.array([0, 0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5, 6, 7, 7.99, 0.2499999, 0.2500001, 0.7499999, 1.2500001, 4.999999])
    row = np.concatenate((base, -base)).astype(np.float32)
    rows = []
    for e in (0, 1, -3, 40, -60, 124, -125, -126):
        rows.append(np.ldexp(row, e).astype(np.float32))
    rows.append(np.zeros(32, np.float32))
    rows.append(np.full(32, -0.0, np.float32))
    rows.append(np.full(32, np.float32(1e-45)))          # the smallest subnormal
    rows.append(np.where(np.arange(32) == 5, np.finfo(np.float32).max, np.float32(1e-45)).astype(np.float32))
    rows.append(np.where(np.arange(32) == 31, np.float32(2.0 ** -127), 0).astype(np.float32))
    for bad in (np.inf, -np.inf, np.nan):
        v = row.copy()
        v[17] = bad
        rows.append(v)
    x = np.stack(rows)
    x = np.concatenate((x, np.broadcast_to(row, x.shape)), 1)  # the second block of each row is ordinary
    q, s = R.gpu_quantise(R.to_dev(x), "f32")
    code, byte = R.unpack(q, s, 64)
    want_code, want_byte = R.quantise(x.astype(np.float64))
    assert np.array_equal(byte, want_byte), (byte, want_byte)
    assert np.array_equal(code, want_code)
    y = torch.empty(x.shape, device="cuda")
    nb.check(nb.api().nemo_mxfp4_dequantize(q.data_ptr(), 32, s.data_ptr(), len(x), 64, y.data_ptr(), 0, 64, R.stream_ptr()), "dequantize")
    assert np.array_equal(R.f64(y), R.values(want_code, want_byte), equal_nan=True)


@pytest.mark.parametrize("elt", ["f32", "bf16"])
def test_quantise_pitches(elt):
    """Rows and codes with pitches and bases that forbid 16-byte access; what lies between is left."""
    rng = np.random.default_rng(5)
    r, k = 37, 96
    wide = rows_of(rng, r, k + 5, elt)
    x = wide[:, 3:3 + k]
    buf = torch.full((r, k // 2 + 3), 0xEE, dtype=torch.uint8, device="cuda")
    q = buf[:, 1:1 + k // 2]
    s = torch.full((nb.api().nemo_mxfp4_scale_bytes(r, k),), 0xEE, dtype=torch.uint8, device="cuda")
    nb.check(nb.api().nemo_mxfp4_quantize(x.data_ptr(), R.ELT[elt][1], x.stride(0), r, k, q.data_ptr(), q.stride(0), s.data_ptr(), R.stream_ptr()), "quantize")
    code, byte = R.unpack(q, s, k)
    want = R.quantise(R.f64(x))
    assert np.array_equal(code, want[0]) and np.array_equal(byte, want[1])
    assert (buf[:, 0] == 0xEE).all() and (buf[:, k // 2 + 1:] == 0xEE).all()
    out = torch.full((r, k + 7), 9.0, device="cuda").to(R.ELT[elt][0])
    y = out[:, 1:1 + k]
    nb.check(nb.api().nemo_mxfp4_dequantize(q.data_ptr(), q.stride(0), s.data_ptr(), r, k, y.data_ptr(), R.ELT[elt][1], y.stride(0), R.stream_ptr()), "dequantize")
    assert np.array_equal(R.f64(y), R.f64(torch.from_numpy(R.values(*want)).to(R.ELT[elt][0])))
    assert (out[:, 0] == 9).all() and (out[:, k + 1:] == 9).all()


# ---- product -------------------------------------------------------------------------------

ACTS = {"none": 0, "silu": 1, "relu": 2, "glu": 3}


def product(a, w, m, n, k, act="none", bias=None, alpha=1.0, out="f32", C0=None, ldc=None, stream=None):
    nout = n // 2 if act == "glu" else n
    ldc = ldc or nout
    c = C0 if C0 is not None else torch.full((m, ldc), -77.0, dtype=R.ELT[out][0], device="cuda")
    g = nb.GemmMxfp4Args(A=a[0].data_ptr(), lda=a[0].stride(0), a_scales=a[1].data_ptr(), W=w[0].data_ptr(), ldw=w[0].stride(0), w_scales=w[1].data_ptr(),
                         bias=None if bias is None else bias.data_ptr(), C=c.data_ptr(), ldc=ldc, c_elt=R.ELT[out][1], M=m, N=n, K=k, act=ACTS[act],
                         accumulate=int(C0 is not None), alpha=alpha)
    nb.check(nb.api().nemo_gemm_mxfp4(C.byref(g), R.stream_ptr() if stream is None else stream), "gemm")
    return c


def coded(rng, r, k, lo, hi, fill=0):
    code = rng.integers(0, 16, (r, k))
    byte = rng.integers(lo, hi + 1, (r, k // 32))
    return R.pack(code, byte, fill), R.values(code, byte)


SHAPES = [(1, 128, 32), (1, 1024, 4096), (2, 8, 64), (7, 256, 1024), (15, 136, 96), (16, 128, 256), (17, 200, 288), (33, 1000, 512), (64, 384, 160), (65, 128, 2048),
          (100, 130, 352), (128, 256, 256), (129, 256, 1056), (200, 72, 4096), (300, 1024, 736), (1000, 640, 1024), (190, 4096, 256), (321, 1000, 96), (600, 2048, 32), (1200, 2048, 288)]


@pytest.mark.parametrize("m,n,k", SHAPES)
def test_product_exact(m, n, k):
    """Scales of 1/2 and 1: every product and every partial sum is a multiple of 1/16 below 2^18
    (36 K / 4096 of them fit 2^18), so the fp32 sums are exact and the result has to be equal. The
    scale bytes of rows past the last one are NaN bytes: nothing may read them into the result."""
    rng = np.random.default_rng(m * 7 + n * 3 + k)
    a, av = coded(rng, m, k, 126, 127, fill=255)
    w, wv = coded(rng, n, k, 126, 127, fill=255)
    got = R.f64(product(a, w, m, n, k))
    assert np.array_equal(got, av @ wv.T)


@pytest.mark.parametrize("act", ["none", "silu", "relu", "glu"])
@pytest.mark.parametrize("out", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("m,n,k", [(1, 512, 1024), (7, 2048, 1024), (20, 256, 96), (150, 512, 544), (260, 768, 256), (5, 512, 4096), (40, 256, 8192), (190, 256, 8192), (700, 4096, 128)])
def test_product(m, n, k, out, act):
    rng = np.random.default_rng(m + n + k)
    a, av = coded(rng, m, k, 118, 124)
    w, wv = coded(rng, n, k, 116, 122)
    bias = rng.standard_normal(n).astype(np.float32)
    got = R.f64(product(a, w, m, n, k, act, torch.from_numpy(bias).cuda(), 0.5, out))
    v, mag = av @ wv.T + bias, np.abs(av) @ np.abs(wv).T + np.abs(bias)
    # K products are exact; each addition loses at most a step (it may truncate) of a sum below mag
    e = k * 2 * R.U * mag
    want = R.activate(v, act) * 0.5
    if act == "glu":
        h = n // 2
        sig = 1 / (1 + np.exp(-v[:, h:]))
        bound = 0.5 * (e[:, :h] * sig + np.abs(v[:, :h]) * e[:, h:] / 4 + np.abs(v[:, :h]) * sig * (10 + 2 * np.abs(v[:, h:])) * R.U)
    elif act == "silu":
        bound = 0.5 * 1.1 * e + np.abs(want) * (10 + 2 * np.abs(v)) * R.U
    else:
        bound = 0.5 * e
    R.check(got, want, bound, out, f"{m}x{n}x{k} {act}")


def test_product_accumulates_and_leaves_the_rest():
    rng = np.random.default_rng(3)
    m, n, k = 70, 200, 320
    a, av = coded(rng, m, k, 126, 127)
    w, wv = coded(rng, n, k, 126, 127)
    c0 = torch.from_numpy(rng.integers(-50, 50, (m + 1, 256)).astype(np.float32)).cuda()
    c = product(a, w, m, n, k, C0=c0.clone(), ldc=256, alpha=0.5)
    assert np.array_equal(R.f64(c)[:m, :n], R.f64(c0)[:m, :n] + 0.5 * (av @ wv.T))
    assert torch.equal(c[:, n:], c0[:, n:]) and torch.equal(c[m:], c0[m:])


@pytest.mark.parametrize("m", [3, 140])
def test_product_nan_scales(m):
    """A NaN block makes its row (or column) of the result NaN and no other."""
    rng = np.random.default_rng(m)
    n, k = 136, 416
    code, byte = rng.integers(0, 16, (m, k)), rng.integers(126, 128, (m, k // 32))
    byte[1, 12] = 255
    a, av = R.pack(code, byte), R.values(code, byte)
    wc, wb = rng.integers(0, 16, (n, k)), rng.integers(126, 128, (n, k // 32))
    wb[130, 0] = 255
    got = R.f64(product(a, R.pack(wc, wb), m, n, k))
    assert np.array_equal(got, av @ R.values(wc, wb).T, equal_nan=True)
    assert np.isnan(got[1]).all() and np.isnan(got[:, 130]).all() and np.isnan(got).sum() == n + m - 1


def test_product_scale_range():
    """Scales far from 1 meet in the product: 2^-100 times 2^100, and sums far below 1."""
    rng = np.random.default_rng(8)
    m, n, k = 5, 128, 128
    for lo, hi in ((27, 227), (127, 20), (2, 250)):
        a, av = coded(rng, m, k, lo, lo)
        w, wv = coded(rng, n, k, hi, hi)
        with np.errstate(over="ignore"):
            want = (av @ wv.T).astype(np.float32)
        assert np.array_equal(R.f64(product(a, w, m, n, k)), want.astype(np.float64))


def test_product_pitched_codes_and_repeats():
    """Codes inside wider rows; the same call twice gives the same bits, split over k or not."""
    rng = np.random.default_rng(9)
    for m, n, k in ((6, 256, 2048), (133, 256, 288)):
        (aq, as_), av = coded(rng, m, k, 120, 125)
        (wq, ws), wv = coded(rng, n, k, 120, 125)
        aw = torch.full((m, k // 2 + 48), 0x77, dtype=torch.uint8, device="cuda")
        aw[:, 16:16 + k // 2] = aq
        first = product((aw[:, 16:], as_), (wq, ws), m, n, k)
        again = product((aq, as_), (wq, ws), m, n, k)
        assert torch.equal(first, again)
        R.check(R.f64(first), av @ wv.T, k * 2 * R.U * (np.abs(av) @ np.abs(wv).T), "f32")


@pytest.mark.parametrize("out", ["bf16", "f16"])
@pytest.mark.parametrize("m,n,k,ldc", [(3, 130, 64, 130), (70, 1001, 96, 1001), (129, 136, 256, 137), (200, 264, 512, 272), (300, 40, 32, 48)])
def test_product_narrow_types_and_odd_pitches(m, n, k, ldc, out):
    """16-bit outputs whose rows allow 16-byte stores and whose do not; what lies behind the columns stays."""
    rng = np.random.default_rng(m + n)
    a, av = coded(rng, m, k, 122, 123)
    w, wv = coded(rng, n, k, 122, 123)
    c = product(a, w, m, n, k, out=out, ldc=ldc)
    want = torch.from_numpy(av @ wv.T).to(R.ELT[out][0])  # the sums are exact in fp32: one rounding
    assert torch.equal(c[:, :n].cpu(), want)
    assert (c[:, n:] == -77).all()


def test_product_split_accumulates():
    """A few rows over a long k (split over a cluster) into what is there."""
    rng = np.random.default_rng(12)
    m, n, k = 9, 384, 8192
    a, av = coded(rng, m, k, 126, 126)
    w, wv = coded(rng, n, k, 126, 126)
    c0 = torch.from_numpy(rng.integers(-50, 50, (m, n)).astype(np.float32)).cuda()
    c = product(a, w, m, n, k, C0=c0.clone(), alpha=0.5)
    assert np.array_equal(R.f64(c), R.f64(c0) + 0.5 * (av @ wv.T))
