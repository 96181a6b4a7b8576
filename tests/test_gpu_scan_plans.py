"""nemo_selective_scan under every plan of cutting time (whole, in a block, across a cluster; one to eight
lanes a channel), with error bounds that follow the plan step by step."""
import numpy as np
import pytest
import torch

import operators_ref as R
from test_gpu_ssm import inputs, scan, want_of

pytestmark = pytest.mark.gpu
U = R.U


def plan(S, c, D, N, G, elt):
    """Chunks of time, and rows of a tile, as the entry point takes them for contiguous inputs."""
    lanes = 1 if N <= 16 else 2 if N <= 32 else 4 if N <= 64 else 8
    items = S * G * -(-(D // G) // (32 // lanes))
    chunks = 1
    while items < 148 * 5 and chunks < 64 and items * chunks < 148 * 32 and chunks * 64 <= c:
        chunks *= 2
    e = 4 if elt == "f32" else 8
    tile = max(4, lanes)
    if lanes == 1 and c >= 32 and (D // G) % e == 0 and N % e == 0:
        tile = 8
    return chunks, tile


def bounds(g, lens, chunks, tile):
    """Error bounds of y [S][c][D] and of the state [S][D][N] of the 64-bit form.

    A row: its step is off by es (one rounding before softplus, 12 u in it); the decay exp(step A) by es |A|
    plus, relative to it, 3 u |step A| (conversion to base 2, product, step) and 4 u (the exponential, 2 ulp); the input
    by es |x B| + 3 u; their sum by 2 u of both. A chunk's first state is folded from the ends of those before it:
    h <- decay h + end, the end with the error of its rows started from zero, the decay (two halves) with 8 u for its
    exponentials and (rows + 12) u |A sum| for a sum of so many steps (12: product, halves, joining a block's warps), besides
    what the steps are off by; 4 u of each term for the roundings. The output: N + 2 roundings of the sum, skip
    and gate as the stage tests count them."""
    f = {k: None if v is None else R.f64(v) for k, v in g.items()}
    S, c, D = f["x"].shape
    A, N, G = f["A"], f["A"].shape[1], f["B"].shape[2]
    raw = f["dt"] + (0 if f["dt_bias"] is None else f["dt_bias"])
    step = np.logaddexp(0, raw)
    es = U * np.abs(raw) + 12 * U * step

    def rows(s, t0, t1, h, eh, out=None):
        for t in range(t0, t1):
            b, cc = (np.repeat(f[k][s, t], D // G, 0) for k in ("B", "C"))
            arg = step[s, t][:, None] * A
            a = np.exp(arg)
            ea = a * (es[s, t][:, None] * np.abs(A) + 3 * U * np.abs(arg) + 4 * U)
            x = f["x"][s, t]
            in_ = (step[s, t] * x)[:, None] * b
            ein = (es[s, t] * np.abs(x))[:, None] * np.abs(b) + 3 * U * np.abs(in_)
            eh = a * eh + ea * np.abs(h) + ein + 2 * U * (np.abs(a * h) + np.abs(in_))
            h = a * h + in_
            if out is not None:
                v = (h * cc).sum(-1)
                ev = (eh * np.abs(cc)).sum(-1) + (N + 2) * U * np.abs(h * cc).sum(-1)
                if f["skip"] is not None:
                    v = v + f["skip"] * x
                    ev = ev + 2 * U * (np.abs(f["skip"] * x) + np.abs(v))
                if f["z"] is not None:
                    z = f["z"][s, t]
                    gate = R.activate(z, "silu")
                    ev = ev * np.abs(gate) + np.abs(v * gate) * (10 + 2 * np.abs(z)) * U
                out[s, t] = ev
        return h, eh

    ey, eh_last = np.zeros((S, c, D)), np.zeros((S, D, N))
    for s in range(S):
        n = int(lens[s])
        per = -(-n // (chunks * tile)) * tile
        h = np.zeros((D, N)) if f["state"] is None else f["state"][s]
        eh, zero = np.zeros((D, N)), np.zeros((D, N))
        for k in range(chunks):
            t0, t1 = min(n, k * per), min(n, (k + 1) * per)
            h1, e1 = rows(s, t0, t1, h, eh, ey)  # as the chunk writes it
            if k == chunks - 1:
                eh_last[s] = e1
                break
            end, e0 = rows(s, t0, t1, h if k == 0 else zero, zero)
            if k:
                arg = step[s, t0:t1].sum(0)[:, None] * A
                a = np.exp(arg)
                ea = a * (es[s, t0:t1].sum(0)[:, None] * np.abs(A) + (per + 12) * U * np.abs(arg) + 8 * U)
                e0 = a * eh + ea * np.abs(h) + e0 + 4 * U * (np.abs(a * h) + np.abs(end))
            h, eh = h1, e0
    return ey, eh_last


def run(S, c, D, N, G, elt, chunks, ragged, in_place=False):
    rng = np.random.default_rng(S * c + D + N)
    g = inputs(rng, S, c, D, N, G, elt)
    assert plan(S, c, D, N, G, elt)[0] == chunks
    lens = np.full(S, c, np.int32)
    if ragged:  # ends inside the first chunk, inside each block's, and none at all
        lens[1:] = [c * i // S + 1 for i in range(1, S)]
        lens[S - 1] = 0
        lens[S // 2] = 3
    wy, wh, _, _ = want_of(g, lens)
    ey, eh = bounds(g, lens, *plan(S, c, D, N, G, elt))
    state = g["state"].clone()
    y, h = scan(g, elt, torch.from_numpy(lens).cuda() if ragged else None)
    R.check(R.f64(y), wy, ey, elt, "y")
    R.check(R.f64(h), wh, eh, "f32", "state")
    assert (R.f64(y)[np.isnan(wy)] == 55).all() and torch.equal(g["state"], state)
    y2, _ = scan(g, elt, torch.from_numpy(lens).cuda() if ragged else None, state_out="same")
    assert torch.equal(y, y2) and torch.equal(g["state"], h)


@pytest.mark.parametrize("S,c,D,N,G,chunks", [(1, 2100, 32, 16, 1, 64), (10, 2100, 16, 16, 1, 64), (3, 600, 32, 16, 1, 16), (2, 257, 64, 16, 1, 8), (2, 100, 64, 8, 2, 2), (2, 1100, 32, 4, 1, 32)])
@pytest.mark.parametrize("elt", ["f32", "bf16"])
def test_time_cut(S, c, D, N, G, chunks, elt):
    run(S, c, D, N, G, elt, chunks, ragged=S > 2)


@pytest.mark.parametrize("S,c,D,N,G,chunks", [(2, 64, 24, 64, 1, 2), (4, 300, 24, 64, 1, 8), (3, 1100, 16, 128, 2, 32), (4, 520, 20, 100, 1, 16), (2, 200, 24, 33, 1, 4), (4, 700, 24, 24, 1, 16),
                                              (1, 2100, 8, 40, 1, 64), (3, 130, 12, 65, 3, 4)])
@pytest.mark.parametrize("elt", ["f32", "f16"])
def test_time_cut_many_states(S, c, D, N, G, chunks, elt):
    """Two to eight lanes a channel, states padded or not, across warps and clusters."""
    run(S, c, D, N, G, elt, chunks, ragged=S > 2)


@pytest.mark.parametrize("N,c", [(16, 70), (3, 66)])
def test_time_whole(N, c):
    """Enough channels: 64 rows and more in one chunk."""
    run(24, c, 992, N, 1, "f32", 1, ragged=True)
