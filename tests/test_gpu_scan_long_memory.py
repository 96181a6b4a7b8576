"""Long memories of nemo_selective_scan: what its decays are off by on average, which adds up over the rows."""
import numpy as np
import pytest
import torch

from test_gpu_ssm import scan

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("lo,hi,limit", [(1e-5, 3e-3, 5e-9), (3e-3, 3e-2, 1.7e-8), (3e-2, 0.2, 8e-9)])
@pytest.mark.parametrize("S,c,D", [(12, 256, 2048), (1, 256, 2048), (12, 1, 2048)])
def test_mean_error_of_decays(S, c, D, lo, hi, limit):
    """States of 1 that only decay, by exponents spread evenly over their logarithm: after T rows the state is
    exp of the sum of A times the steps, and its relative error the sum of T errors. A decay is off by
    5e-8 (root of the mean square) at most and the product by half a step, so the mean of T x 16 x D errors a
    stream, over half a million of them, lies within 5e-10 of what decays are off by on average: by at most 5.3e-9 up
    to 3e-3 (3.6e-9 over that range), 1.5e-8 up to 0.03, 6.3e-9 up to 0.3 in magnitude, as counted over a
    million values each. Where time is cut (one stream: into 8 chunks) a chunk adds the error of two exponentials,
    3e-8 each, and of a sum of 32 steps to its 32 rows: 2e-9 a row."""
    N, T, calls = 16, 256, 256 // c
    g = torch.Generator("cuda").manual_seed(S + c)
    A = -torch.exp(torch.rand(D, N, generator=g, device="cuda") * 0.5)
    span = np.log(hi / lo) - 0.5
    steps = torch.exp(torch.rand(S, T, D, generator=g, device="cuda") * span + np.log(lo))
    zero, one = torch.zeros(S, c, D, device="cuda"), torch.ones(S, c, 1, N, device="cuda")
    state = torch.ones(S, D, N, device="cuda")
    for k in range(calls):
        args = dict(x=zero, dt=steps[:, k * c:(k + 1) * c], z=None, B=one, C=one, A=A, skip=None, dt_bias=None, state=state)
        scan(args, "f32", softplus=False, state_out="same")
    want = torch.exp(steps.double().sum(1)[..., None] * A.double())
    mean = float(((state.double() - want) / want).mean()) / T
    assert abs(mean) <= limit + (2e-9 if S == 1 else 0), mean
