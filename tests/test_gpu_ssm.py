"""Causal convolution (nemo_causal_conv) and selective scan (nemo_selective_scan) with carried
state against plain 64-bit forms."""
import ctypes as C

import numpy as np
import pytest
import torch

import nemoasr_b200 as nb
import operators_ref as R

pytestmark = pytest.mark.gpu


def dev32(a):
    return None if a is None else torch.from_numpy(np.ascontiguousarray(a, np.float32)).cuda()


def ptr(t):
    return None if t is None else t.data_ptr()


def some_lens(rng, S, c):
    n = rng.integers(0, c + 1, S).astype(np.int32)
    n[0] = c
    if S > 1:
        n[1] = 0
    return n


# ---- convolution ---------------------------------------------------------------------------

def conv(x, w, bias, hist, elt, act, lens=None, hist_out="new", y=None, taps=None):
    S, c, D = x.shape
    y = torch.full((S, c, D), 55.0, dtype=x.dtype, device="cuda") if y is None else y
    taps = taps or w.shape[1]
    ho = hist if hist_out == "same" else torch.full((S, taps - 1, D), 44.0, dtype=x.dtype, device="cuda") if hist_out == "new" else None
    a = nb.CausalConvArgs(x=x.data_ptr(), x_ld=x.stride(1), x_sstride=x.stride(0), w=w.data_ptr(), bias=ptr(bias), hist_in=ptr(hist), hist_out=ptr(ho),
                          y=y.data_ptr(), y_ld=y.stride(1), y_sstride=y.stride(0), lens=ptr(lens), streams=S, c=c, D=D, taps=taps, elt=R.ELT[elt][1],
                          act={"none": 0, "silu": 1}[act])
    nb.check(nb.api().nemo_causal_conv(C.byref(a), R.stream_ptr()), "conv")
    return y, ho


@pytest.mark.parametrize("elt", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("taps", [1, 2, 3, 4, 5, 8])
@pytest.mark.parametrize("S,c,D", [(1, 1, 8), (3, 1, 200), (5, 7, 64), (2, 9, 33), (1, 300, 72), (4, 65, 256)])
def test_conv(S, c, D, taps, elt):
    rng = np.random.default_rng(S * c * D + taps)
    x, hist = R.to_dev(rng.standard_normal((S, c, D)), elt), R.to_dev(rng.standard_normal((S, taps - 1, D)), elt)
    w, bias = rng.standard_normal((D, taps)).astype(np.float32), rng.standard_normal(D).astype(np.float32)
    for act, ragged in (("silu", False), ("none", True)):
        lens = some_lens(rng, S, c) if ragged else None
        y, h = conv(x, dev32(w), dev32(bias), hist, elt, act, None if lens is None else torch.from_numpy(lens).cuda())
        n = lens if ragged else np.full(S, c)
        want, wh, bound = R.conv(R.f64(x), w.astype(np.float64), bias.astype(np.float64), R.f64(hist), n, act)
        R.check(R.f64(y), want, bound, elt)
        assert np.array_equal(R.f64(h), wh)
        assert (R.f64(y)[np.isnan(want)] == 55).all()  # rows behind the last one


@pytest.mark.parametrize("elt", ["f32", "bf16"])
def test_conv_in_pieces(elt):
    """A recording in pieces of any length, the history carried in place, gives the recording's bits."""
    rng = np.random.default_rng(1)
    S, c, D, taps = 3, 61, 40, 4
    x = R.to_dev(rng.standard_normal((S, c, D)), elt)
    w, bias = dev32(rng.standard_normal((D, taps))), dev32(rng.standard_normal(D))
    whole, last = conv(x, w, bias, None, elt, "silu")
    hist = torch.zeros(S, taps - 1, D, dtype=x.dtype, device="cuda")
    y, t = torch.empty_like(whole), 0
    for n in (1, 1, 2, 1, 7, 30, 3, 16):
        part, _ = conv(x[:, t:t + n], w, bias, hist, elt, "silu", hist_out="same", y=y[:, t:t + n])
        t += n
    assert t == c and torch.equal(y, whole) and torch.equal(hist, last)


def test_conv_strides_without_bias_or_history():
    rng = np.random.default_rng(2)
    S, c, D, taps = 2, 21, 24, 3
    buf = R.to_dev(rng.standard_normal((S, c + 2, D + 11)), "f32")
    x = buf[:, 1:1 + c, 5:5 + D]
    out = torch.full((S, c, D + 3), 7.0, device="cuda")
    w = rng.standard_normal((D, taps)).astype(np.float32)
    y, _ = conv(x, dev32(w), None, None, "f32", "silu", hist_out=None, y=out[:, :, 2:2 + D])
    want, _, bound = R.conv(R.f64(x), w.astype(np.float64), None, np.zeros((S, taps - 1, D)), np.full(S, c), "silu")
    R.check(R.f64(y), want, bound, "f32")
    assert (out[:, :, :2] == 7).all() and (out[:, :, 2 + D:] == 7).all()


def test_conv_lens_out_of_range_and_no_rows():
    rng = np.random.default_rng(3)
    S, c, D, taps = 3, 5, 16, 4
    x, hist = R.to_dev(rng.standard_normal((S, c, D))), R.to_dev(rng.standard_normal((S, taps - 1, D)))
    w = dev32(rng.standard_normal((D, taps)))
    odd = torch.tensor([-4, 2, 900], dtype=torch.int32, device="cuda")
    fit = torch.tensor([0, 2, 5], dtype=torch.int32, device="cuda")
    a, b = conv(x, w, None, hist, "f32", "none", odd), conv(x, w, None, hist, "f32", "none", fit)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    # no rows at all: the history moves to its new place
    y, h = conv(x[:, :0], w, None, hist, "f32", "none")
    torch.cuda.synchronize()
    assert torch.equal(h, hist)


# ---- scan ----------------------------------------------------------------------------------

def inputs(rng, S, c, D, N, G, elt, with_z=True, with_skip=True, with_bias=True, state=True):
    f = dict(x=rng.standard_normal((S, c, D)), dt=rng.standard_normal((S, c, D)) * 0.5, B=rng.standard_normal((S, c, G, N)), C=rng.standard_normal((S, c, G, N)),
             z=rng.standard_normal((S, c, D)) if with_z else None)
    g = {k: None if v is None else R.to_dev(v, elt) for k, v in f.items()}
    g["A"] = dev32(-np.exp(rng.standard_normal((D, N))))
    g["skip"] = dev32(rng.standard_normal(D)) if with_skip else None
    g["dt_bias"] = dev32(rng.uniform(-6, 0.5, D)) if with_bias else None
    g["state"] = dev32(rng.standard_normal((S, D, N))) if state else None
    return g


def scan(g, elt, lens=None, softplus=True, y=None, state_out="new"):
    S, c, D = g["x"].shape
    N, G = g["A"].shape[1], g["B"].shape[2]
    y = torch.full((S, c, D), 55.0, dtype=g["x"].dtype, device="cuda") if y is None else y
    so = g["state"] if state_out == "same" else torch.full((S, D, N), 44.0, device="cuda") if state_out == "new" else None
    z = g["z"]
    a = nb.SelectiveScanArgs(x=ptr(g["x"]), x_ld=g["x"].stride(1), x_sstride=g["x"].stride(0), dt=ptr(g["dt"]), dt_ld=g["dt"].stride(1), dt_sstride=g["dt"].stride(0),
                             z=ptr(z), z_ld=z.stride(1) if z is not None else 0, z_sstride=z.stride(0) if z is not None else 0, B=ptr(g["B"]), C=ptr(g["C"]),
                             bc_ld=g["B"].stride(1), bc_sstride=g["B"].stride(0), A=ptr(g["A"]), skip=ptr(g["skip"]), dt_bias=ptr(g["dt_bias"]), dt_softplus=int(softplus),
                             state_in=ptr(g["state"]), state_out=ptr(so), y=y.data_ptr(), y_ld=y.stride(1), y_sstride=y.stride(0), lens=ptr(lens), streams=S, c=c,
                             D=D, N=N, groups=G, elt=R.ELT[elt][1])
    nb.check(nb.api().nemo_selective_scan(C.byref(a), R.stream_ptr()), "scan")
    return y, so


def want_of(g, lens=None, softplus=True):
    h = {k: None if v is None else R.f64(v) for k, v in g.items()}
    return R.scan(h["x"], h["dt"], h["A"], h["B"], h["C"], h["skip"], h["z"], h["dt_bias"], softplus, h["state"], lens)


@pytest.mark.parametrize("elt", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("S,c,D,N,G", [(1, 1, 8, 16, 1), (4, 1, 96, 16, 1), (3, 7, 64, 16, 2), (2, 33, 40, 1, 1), (1, 40, 24, 3, 3), (2, 17, 48, 8, 1), (1, 50, 36, 24, 1),
                                       (2, 20, 16, 64, 2), (1, 9, 12, 128, 1), (1, 70, 130, 16, 1), (1, 257, 64, 16, 1), (2, 21, 20, 100, 1), (1, 1100, 64, 16, 4)])
def test_scan(S, c, D, N, G, elt):
    rng = np.random.default_rng(S * c * D + N)
    g = inputs(rng, S, c, D, N, G, elt)
    for ragged in (False, True):
        lens = some_lens(rng, S, c) if ragged else None
        y, h = scan(g, elt, None if lens is None else torch.from_numpy(lens).cuda())
        wy, wh, ey, eh = want_of(g, lens)
        R.check(R.f64(y), wy, ey, elt, "y")
        R.check(R.f64(h), wh, eh, "f32", "state")
        assert (R.f64(y)[np.isnan(wy)] == 55).all()


@pytest.mark.parametrize("c", [1, 6, 90])
def test_scan_without_options(c):
    """No gate, skip, step bias, softplus, state: each left out."""
    rng = np.random.default_rng(c)
    g = inputs(rng, 2, c, 48, 16, 1, "f32", with_z=False, with_skip=False, with_bias=False, state=False)
    g["dt"] = R.to_dev(np.abs(rng.standard_normal((2, c, 48))) * 0.1)
    y, h = scan(g, "f32", softplus=False)
    wy, wh, ey, eh = want_of(g, softplus=False)
    R.check(R.f64(y), wy, ey, "f32", "y")
    R.check(R.f64(h), wh, eh, "f32", "state")
    y2, _ = scan(g, "f32", softplus=False, state_out=None)
    assert torch.equal(y, y2)


@pytest.mark.parametrize("elt", ["f32", "bf16"])
def test_scan_in_pieces(elt):
    """A recording in pieces with the state carried in place: y and the state of the recording."""
    rng = np.random.default_rng(4)
    S, c, D, N = 2, 150, 64, 16
    g = inputs(rng, S, c, D, N, 1, elt, state=False)
    wy, wh, ey, eh = want_of(g)
    part = dict(g, state=torch.zeros(S, D, N, device="cuda"))
    y, t = torch.empty_like(g["x"]), 0
    for n in (1, 1, 5, 1, 14, 64, 1, 63):
        for k in ("x", "dt", "z", "B", "C"):
            part[k] = g[k][:, t:t + n]
        scan(part, elt, state_out="same", y=y[:, t:t + n])
        t += n
    assert t == c
    R.check(R.f64(y), wy, ey, elt, "y")
    R.check(R.f64(part["state"]), wh, eh, "f32", "state")


def test_scan_strides():
    """Rows inside wider rows (one projection's output holds x and z, another dt, B and C)."""
    rng = np.random.default_rng(6)
    S, c, D, N = 3, 19, 40, 16
    g = inputs(rng, S, c, D, N, 1, "bf16")
    xz = torch.zeros(S, c, 2 * D + 3, dtype=torch.bfloat16, device="cuda")
    xz[..., 1:1 + D], xz[..., 1 + D:1 + 2 * D] = g["x"], g["z"]
    bc = torch.zeros(S, c, 2 * N + 1, dtype=torch.bfloat16, device="cuda")
    bc[..., :N], bc[..., N + 1:] = g["B"][:, :, 0], g["C"][:, :, 0]
    wy, wh, ey, eh = want_of(g)
    out = torch.full((S, c + 1, D + 2), 3.0, dtype=torch.bfloat16, device="cuda")
    v = dict(g, x=xz[..., 1:1 + D], z=xz[..., 1 + D:1 + 2 * D], B=bc[..., :N].unsqueeze(2), C=bc[..., N + 1:].unsqueeze(2))
    y, h = scan(v, "bf16", y=out[:, :c, 1:1 + D])
    R.check(R.f64(y), wy, ey, "bf16", "y")
    R.check(R.f64(h), wh, eh, "f32", "state")
    assert (out[:, c:] == 3).all() and (out[..., 0] == 3).all() and (out[..., D + 1:] == 3).all()


def test_scan_extremes():
    """Decays of exactly 0 and 1, growth, steps far beyond softplus's knee, infinities and NaN stay
    in their channel."""
    rng = np.random.default_rng(7)
    S, c, D, N = 1, 80, 64, 16
    g = inputs(rng, S, c, D, N, 1, "f32")
    A = R.f64(g["A"])
    A[0], A[1], A[2], A[3] = 0.0, -1e6, 0.05, -200.0
    g["A"] = dev32(A)
    dt = R.f64(g["dt"])
    dt[:, :, 5] = 60.0    # softplus(60) = 60
    dt[:, :, 6] = -60.0   # softplus(-60) = 8.7e-27
    g["dt"] = R.to_dev(dt)
    clean, hc = scan(g, "f32")
    wy, wh, ey, eh = want_of(g)
    R.check(R.f64(clean), wy, ey, "f32", "y")
    R.check(R.f64(hc), wh, eh, "f32", "state")
    x = g["x"].clone()
    x[0, 10, 20], x[0, 11, 21] = float("nan"), float("inf")
    y, h = scan(dict(g, x=x), "f32")
    keep = [d for d in range(D) if d not in (20, 21)]
    assert torch.equal(y[:, :, keep], clean[:, :, keep]) and torch.equal(h[:, keep], hc[:, keep])
    assert torch.equal(y[:, :10, 20], clean[:, :10, 20]) and torch.isnan(y[0, 10:, 20]).all() and torch.isnan(h[0, 20]).all()
    assert not torch.isfinite(y[0, 11:, 21]).any() and not torch.isfinite(h[0, 21]).any()


def test_scan_no_rows():
    rng = np.random.default_rng(8)
    g = inputs(rng, 2, 3, 16, 16, 1, "f32")
    for k in ("x", "dt", "z", "B", "C"):
        g[k] = g[k][:, :0]
    _, h = scan(g, "f32")
    assert torch.equal(h, g["state"])


@pytest.mark.parametrize("c,D", [(70, 64), (300, 64), (300, 2048), (3000, 32)])
def test_scan_state_replaced_in_place(c, D):
    """State out over state in, streams of all lengths (none among them), time cut or not: the bits of
    a call with a state of its own, every time."""
    rng = np.random.default_rng(c + D)
    S = 6
    g = inputs(rng, S, c, D, 16, 1, "bf16")
    lens = torch.tensor([0, 1, 3, c // 2, c - 1, c], dtype=torch.int32, device="cuda")
    y, h = scan(g, "bf16", lens)
    assert torch.equal(h[0], g["state"][0])
    for _ in range(20):
        own = dict(g, state=g["state"].clone())
        y2, _ = scan(own, "bf16", lens, state_out="same")
        assert torch.equal(y, y2) and torch.equal(own["state"], h)


def test_scan_growth_past_the_range_of_a_chunk():
    """A channel that grows by e^3 a row, without input until its last rows: its growth over a chunk of
    time overflows, its state does not. And states of 1e-30 that grow back to about 1."""
    S, c, D, N = 1, 1100, 32, 16
    rng = np.random.default_rng(11)
    g = inputs(rng, S, c, D, N, 1, "f32", with_bias=False, state=False)
    x = R.f64(g["x"])
    x[:, :c - 9] = 0
    g["x"], g["dt"] = R.to_dev(x), R.to_dev(np.ones((S, c, D)))
    A = R.f64(g["A"])
    A[3] = 3.0
    A[4] = np.log(1e30) / c
    g["A"] = dev32(A)
    g["state"] = torch.zeros(S, D, N, device="cuda")
    g["state"][:, 4] = 1e-30
    y, h = scan(g, "f32", softplus=False)
    wy, wh, ey, eh = want_of(g, softplus=False)
    assert np.isfinite(wh).all()
    R.check(R.f64(y), wy, ey, "f32", "y")
    R.check(R.f64(h), wh, eh, "f32", "state")


@pytest.mark.parametrize("elt", ["f32", "bf16"])
@pytest.mark.parametrize("S,c,D,N,G", [(1, 5, 1, 1, 1), (2, 9, 3, 5, 3), (1, 100, 1, 16, 1), (3, 1, 2, 3, 2), (2, 5, 40, 16, 5), (1, 130, 264, 32, 3)])
def test_scan_narrow(S, c, D, N, G, elt):
    """A channel or two, groups smaller than a warp's channels."""
    rng = np.random.default_rng(S + c + D)
    g = inputs(rng, S, c, D, N, G, elt)
    y, h = scan(g, elt)
    wy, wh, ey, eh = want_of(g)
    R.check(R.f64(y), wy, ey, elt, "y")
    R.check(R.f64(h), wh, eh, "f32", "state")


@pytest.mark.parametrize("c", [1, 6, 50, 900])
def test_scan_steps_of_zero_keep_the_state(c):
    """A step of exactly 0 decays by exactly 1: the state's bits stay, whatever A is."""
    rng = np.random.default_rng(c)
    g = inputs(rng, 2, c, 48, 16, 1, "f32", with_bias=False)
    g["dt"] = torch.zeros_like(g["dt"])
    _, h = scan(g, "f32", softplus=False)
    assert torch.equal(h, g["state"])
