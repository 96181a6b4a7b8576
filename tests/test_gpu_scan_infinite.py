"""Infinite inputs, steps and states in nemo_selective_scan: the definition's infinities, whatever the
number of states is padded to and wherever time is cut."""
import numpy as np
import pytest
import torch

import operators_ref as R
from test_gpu_ssm import dev32, inputs, scan, want_of

pytestmark = pytest.mark.gpu


def compare(got, want, bound, elt, what):
    """The same infinities and NaN; finite values within the bound."""
    fin = np.isfinite(want)
    assert np.array_equal(got[~fin], want[~fin], equal_nan=True), what
    assert np.isfinite(got[fin]).all(), what
    R.check(got, np.where(fin, want, np.nan), np.where(fin, bound, 0), elt, what)


def positive(rng, S, c, D, N, elt):
    """B, C and skip above 0 and modest decays: an infinite state keeps its sign, and its outputs have it too."""
    g = inputs(rng, S, c, D, N, 1, elt)
    for k in ("B", "C"):
        g[k] = R.to_dev(np.abs(rng.standard_normal((S, c, 1, N))) + 0.1, elt)
    g["skip"] = dev32(np.abs(rng.standard_normal(D)) + 0.1)
    g["A"] = dev32(-np.exp(rng.uniform(-2, 1.5, (D, N))))
    return g


@pytest.mark.filterwarnings("ignore:.*invalid value")
@pytest.mark.parametrize("elt", ["f32", "bf16"])
@pytest.mark.parametrize("c", [1, 9, 29])
@pytest.mark.parametrize("N", [1, 3, 5, 12, 20, 24, 30, 36, 100, 128])
def test_infinite_inputs_of_padded_states(N, c, elt):
    """An infinite input or step makes its channel's states and outputs infinite from its row on: states
    that only fill up a lane take no part."""
    rng = np.random.default_rng(100 * N + c)
    S, D = 2, 40
    g = positive(rng, S, c, D, N, elt)
    t = min(c - 1, 3)
    g["x"][0, t, 5], g["x"][1, t, 6] = float("inf"), -float("inf")
    g["dt"][0, t, 7], g["x"][0, t, 7] = float("inf"), 1.0
    y, h = scan(g, elt)
    wy, wh, ey, eh = want_of(g)
    assert np.isinf(wy[0, t:, 5]).all() and np.isinf(wy[1, t:, 6]).all() and np.isinf(wy[0, t:, 7]).all()
    compare(R.f64(y), wy, ey, elt, "y")
    compare(R.f64(h), wh, eh, "f32", "state")


@pytest.mark.filterwarnings("ignore:.*invalid value")
@pytest.mark.parametrize("c,N,D", [(150, 12, 40), (150, 3, 40), (700, 24, 40), (700, 1, 24), (200, 100, 24), (2100, 12, 32)])
def test_infinite_inputs_of_padded_states_where_time_is_cut(c, N, D):
    """The same where chunks of time meet, with streams of all lengths; other channels keep their bits."""
    rng = np.random.default_rng(c + N)
    S = 4
    g = positive(rng, S, c, D, N, "f32")
    lens = np.array([c, c // 2, 3, 0], np.int32)
    clean, hc = scan(g, "f32", torch.from_numpy(lens).cuda())
    x = g["x"].clone()
    for s, t, d in ((0, 5, 3), (0, c - 2, 4), (1, c // 3, 5), (2, 2, 6), (3, 0, 7)):  # (the last stream has no rows)
        x[s, t, d] = float("inf")
    x[1, c // 2, 8] = float("inf")  # behind the last row
    g = dict(g, x=x)
    wy, wh, ey, eh = want_of(g, lens)
    y, h = scan(g, "f32", torch.from_numpy(lens).cuda())
    live = ~np.isnan(wy)
    assert np.isinf(wy[0, 5:, 3]).all() and np.isinf(wh[2, 6]).all() and np.isfinite(wh[3]).all()
    compare(np.where(live, R.f64(y), np.nan), wy, ey, "f32", "y")
    compare(R.f64(h), wh, eh, "f32", "state")
    assert (R.f64(y)[~live] == 55).all()
    for s, odd in ((0, (3, 4)), (1, (5,)), (2, (6,)), (3, ())):
        keep = [d for d in range(D) if d not in odd]
        assert torch.equal(y[s][:, keep], clean[s][:, keep]) and torch.equal(h[s][keep], hc[s][keep])


@pytest.mark.filterwarnings("ignore:.*invalid value")
@pytest.mark.parametrize("c,N,D", [(70, 16, 40), (300, 16, 40), (300, 12, 40), (300, 24, 40), (200, 100, 24), (1100, 16, 32), (2500, 8, 40), (700, 64, 24)])
@pytest.mark.parametrize("in_place", [False, True])
def test_infinite_states_where_time_is_cut(c, N, D, in_place):
    """Infinite states stay so through any number of decays that are not 0, wherever the rows are cut into
    chunks; so do those that an infinite input, or an infinite step, makes on the way. Other channels keep their bits."""
    rng = np.random.default_rng(c + N)
    S = 2
    g = positive(rng, S, c, D, N, "f32")
    clean, hc = scan(g, "f32")
    g["state"] = g["state"].clone()
    g["state"][0, 3, 0], g["state"][1, 4, N - 1] = float("inf"), -float("inf")
    x, dt = g["x"].clone(), g["dt"].clone()
    x[0, c // 3, 11], x[1, 2, 12] = float("inf"), -float("inf")
    dt[0, c // 2, 13], x[0, c // 2, 13] = float("inf"), 1.0
    g = dict(g, x=x, dt=dt)
    wy, wh, ey, eh = want_of(g)
    y, h = scan(g, "f32", state_out="same" if in_place else "new")
    assert np.isinf(wy[0, :, 3]).all() and np.isinf(wy[1, :, 4]).all() and np.isinf(wh[0, 13]).all()
    compare(R.f64(y), wy, ey, "f32", "y")
    compare(R.f64(h), wh, eh, "f32", "state")
    for s, odd in ((0, (3, 11, 13)), (1, (4, 12))):
        keep = [d for d in range(D) if d not in odd]
        assert torch.equal(y[s][:, keep], clean[s][:, keep]) and torch.equal(h[s][keep], hc[s][keep])
