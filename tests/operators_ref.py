"""Plain 64-bit forms of the 4-bit rows, the causal convolution and the selective scan, with error
bounds that follow the fp32 arithmetic of the kernels step by step."""
import numpy as np
import torch

import nemoasr_b200 as nb

ELT = {"f32": (torch.float32, 0), "bf16": (torch.bfloat16, 1), "f16": (torch.float16, 2)}
U = 2.0 ** -24  # half a step of fp32, relative


def half_step(elt, v):
    """Half a step of the type around |v| (its subnormal step included)."""
    fi = torch.finfo(ELT[elt][0])
    return np.maximum(np.abs(v) * (fi.eps / 2), fi.tiny * fi.eps / 2)


def rounding(elt, v):
    """What storing v in the type may add: nothing for fp32, whose arithmetic the bounds count."""
    return np.zeros_like(v) if elt == "f32" else half_step(elt, v)


def to_dev(a, elt="f32"):
    return torch.from_numpy(np.ascontiguousarray(a)).to(ELT[elt][0]).cuda()


def f64(t):
    return t.detach().double().cpu().numpy()


def stream_ptr():
    return torch.cuda.current_stream().cuda_stream


# ---- 4-bit rows ----------------------------------------------------------------------------

GRID = np.array([0, 0.5, 1, 1.5, 2, 3, 4, 6.0])


def quantise(x):
    """x [R][K] (64 bits) -> codes (0..15) [R][K] and scale bytes [R][K / 32]."""
    r, k = x.shape
    b = x.reshape(r, k // 32, 32)
    bad = ~np.isfinite(b).all(-1)
    top = np.abs(np.where(np.isfinite(b), b, 0)).max(-1)
    _, e = np.frexp(top)  # top in [2^(e-1), 2^e)
    byte = np.where(top > 0, np.clip(e - 3, -127, 125) + 127, 0)
    with np.errstate(invalid="ignore"):
        v = np.abs(b) / np.ldexp(1.0, byte - 127)[..., None]
        dist = np.abs(v[..., None] - GRID)
        dist = np.where(np.isnan(dist), 0, dist)
    # nearest; ties to the even code (the even indices of the grid)
    code = np.zeros(v.shape, np.int64)
    best = dist[..., 0].copy()
    for i in range(1, 8):
        closer = (dist[..., i] < best) | ((dist[..., i] == best) & (i % 2 == 0))
        code = np.where(closer, i, code)
        best = np.where(closer, dist[..., i], best)
    code = np.where(np.signbit(b), code + 8, code)
    code = np.where(bad[..., None], 0, code)
    return code.reshape(r, k), np.where(bad, 255, byte)


def values(code, byte):
    r, k = code.shape
    mag = GRID[code & 7]
    v = np.where(code >= 8, -mag, mag).reshape(r, k // 32, 32)
    s = np.where(byte == 255, np.nan, np.ldexp(1.0, byte - 127))
    return (v * s[..., None]).reshape(r, k)


def scale_index(rows, blocks):
    """Byte of row r and block b in the tiled scale buffer."""
    r, b = np.arange(rows)[:, None], np.arange(blocks)[None, :]
    kt = (blocks + 3) // 4
    return ((r // 128) * kt + b // 4) * 512 + (r % 32) * 16 + (r % 128) // 32 * 4 + b % 4


def pack(code, byte, fill=0):
    """Device tensors of the packed codes and the tiled scale bytes; bytes of no row are `fill`,
    those of a row's columns past the last block 0."""
    r, nb_ = byte.shape
    n = ((r + 127) // 128) * ((nb_ + 3) // 4) * 512
    s = np.full(n, fill, np.uint8)
    full = np.zeros((r, (nb_ + 3) // 4 * 4), np.uint8)
    full[:, :nb_] = byte
    s[scale_index(r, full.shape[1])] = full
    q = (code[:, 0::2] | code[:, 1::2] << 4).astype(np.uint8)
    return torch.from_numpy(q).cuda(), torch.from_numpy(s).cuda()


def unpack(q, s, k):
    q = q.cpu().numpy().astype(np.int64)
    code = np.stack((q & 15, q >> 4), -1).reshape(q.shape[0], -1)[:, :k]
    return code, s.cpu().numpy().astype(np.int64)[scale_index(q.shape[0], k // 32)]


def gpu_quantise(x, elt, K=None):
    """Codes and scale bytes of a device tensor [R][ld] through the library (scales start as 0xee)."""
    R, K = x.shape[0], K or x.shape[1]
    q = torch.full((R, K // 2), 0xEE, dtype=torch.uint8, device="cuda")
    s = torch.full((nb.api().nemo_mxfp4_scale_bytes(R, K),), 0xEE, dtype=torch.uint8, device="cuda")
    nb.check(nb.api().nemo_mxfp4_quantize(x.data_ptr(), ELT[elt][1], x.stride(0), R, K, q.data_ptr(), q.stride(0), s.data_ptr(), stream_ptr()), "quantize")
    return q, s


def activate(v, act):
    sig = lambda t: 1.0 / (1.0 + np.exp(-t))  # noqa: E731
    if act == "silu":
        return v * sig(v)
    if act == "relu":
        return np.where(v < 0, 0, v)
    if act == "glu":
        h = v.shape[-1] // 2
        return v[..., :h] * sig(v[..., h:])
    return v


# ---- convolution ---------------------------------------------------------------------------

def conv(x, w, bias, hist, lens, act):
    """x [S][c][D], w [D][taps], hist [S][taps-1][D] -> y (rows behind the last one NaN), history, bound."""
    S, c, D = x.shape
    taps = w.shape[1]
    u = np.concatenate((hist, x), 1)
    v = np.zeros((S, c, D)) + (0 if bias is None else bias)
    mag = np.abs(v)
    for j in range(taps):
        v = v + u[:, j:j + c] * w[:, j]
        mag = mag + np.abs(u[:, j:j + c] * w[:, j])
    bound = (taps + 1) * U * mag  # one rounding per term, of a sum no larger than mag
    if act == "silu":
        y = activate(v, "silu")
        # silu's slope is below 1.1; exponential, sum and quotient: 2 |v| u in the exponent, 8 u else
        bound = 1.1 * bound + np.abs(y) * (8 + 2 * np.abs(v)) * U
    else:
        y = v
    h = np.stack([u[s, lens[s]:lens[s] + taps - 1] for s in range(S)]) if taps > 1 else np.zeros((S, 0, D))
    for s in range(S):
        y[s, lens[s]:] = np.nan
    return y, h, bound


# ---- scan ----------------------------------------------------------------------------------

def scan(x, dt, A, B, C, skip=None, z=None, dt_bias=None, softplus=True, state=None, lens=None):
    """x, dt, z [S][c][D]; A [D][N]; B, C [S][c][G][N]; state [S][D][N]. -> y (rows behind the last
    one NaN), state, bound of y, bound of the state."""
    S, c, D = x.shape
    N, G = A.shape[1], B.shape[2]
    h = np.zeros((S, D, N)) if state is None else state.copy()
    eh = np.zeros_like(h)
    y, ey = np.full((S, c, D), np.nan), np.full((S, c, D), np.nan)
    lens = np.full(S, c) if lens is None else lens
    for t in range(c):
        on = lens > t
        raw = dt[:, t] + (0 if dt_bias is None else dt_bias)
        step = np.logaddexp(0, raw) if softplus else raw
        # the sum is rounded once: u |raw| before softplus (slope below 1). softplus is max(v, 0) +
        # log1p(e^-|v|): exponential 4 u (2^-22), quotient 4 u, series and sum 4 u
        es = U * np.abs(raw) + (12 * U * np.abs(step) if softplus else 0)
        wide = lambda v: np.repeat(v[:, t], D // G, 1)  # noqa: E731
        b, g = wide(B), wide(C)
        arg = step[..., None] * A
        a = np.exp(arg)
        # the exponent carries A's conversion to base 2, the product and the step; exp2 is 2 ulp. Where time
        # is cut (64 rows and more, into two chunks at least) a chunk's decay is exp of A times the sum of its
        # steps: at most c / 2 additions, each off by u of a sum no larger than the whole
        ea = a * (es[..., None] * np.abs(A) + np.abs(arg) * (3 + (c / 2 if c >= 64 else 0)) * U + 4 * U)
        in_ = (step * x[:, t])[..., None] * b
        ein = (es * np.abs(x[:, t]))[..., None] * np.abs(b) + np.abs(in_) * 3 * U
        hn = a * h + in_
        en = a * eh + ea * np.abs(h) + ein + U * (np.abs(a * h) + np.abs(in_)) * 2
        h = np.where(on[:, None, None], hn, h)
        eh = np.where(on[:, None, None], en, eh)
        v = (h * g).sum(-1)
        ev = (eh * np.abs(g)).sum(-1) + (N + 2) * U * (np.abs(h * g).sum(-1))
        if skip is not None:
            v = v + skip * x[:, t]
            ev = ev + 2 * U * (np.abs(skip * x[:, t]) + np.abs(v))
        if z is not None:
            s = activate(z[:, t], "silu")
            ev = ev * np.abs(s) + np.abs(v * s) * (10 + 2 * np.abs(z[:, t])) * U
            v = v * s
        y[:, t] = np.where(on[:, None], v, np.nan)
        ey[:, t] = ev
    return y, h, ey, eh


def check(got, want, bound, elt, what=""):
    """|got - want| <= bound + what storing it adds, where want is a number."""
    on = ~np.isnan(want)
    err = np.abs(got - want)
    lim = bound + rounding(elt, np.abs(np.where(on, want, 0)) + np.where(on, bound, 0)) + np.finfo(np.float32).tiny
    worst = np.max(np.where(on, err / lim, 0)) if on.any() else 0.0
    assert not np.isnan(got[on]).any(), what
    assert worst <= 1.0, f"{what}: error is {worst:.3g} of the bound"
