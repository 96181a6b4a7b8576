"""The convolution and the scan over rows laid out time by time (all streams of a row side by side), in
reverse and with gaps: the bits of the streams one after the other."""
import numpy as np
import pytest
import torch

import operators_ref as R
from test_gpu_ssm import conv, dev32, inputs, scan

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("S,c,D", [(3, 1, 64), (5, 9, 64), (2, 70, 40)])
@pytest.mark.parametrize("ragged", [False, True])
def test_time_by_time(S, c, D, ragged):
    rng = np.random.default_rng(S + c)
    g = inputs(rng, S, c, D, 16, 1, "bf16")
    w, bias = dev32(rng.standard_normal((D, 4))), dev32(rng.standard_normal(D))
    lens = torch.tensor([c, 0, c // 2, 1, c][:S], dtype=torch.int32, device="cuda") if ragged else None
    want = conv(g["x"], w, bias, None, "bf16", "silu", lens) + scan(g, "bf16", lens)
    turn = lambda v: v.transpose(0, 1).contiguous().transpose(0, 1)  # noqa: E731
    t = {k: turn(v) if v is not None and k in ("x", "dt", "z", "B", "C") else v for k, v in g.items()}
    fill = lambda: turn(torch.full((S, c, D), 55.0, dtype=torch.bfloat16, device="cuda"))  # noqa: E731
    got = conv(t["x"], w, bias, None, "bf16", "silu", lens, y=fill()) + scan(t, "bf16", lens, y=fill())
    for a, b in zip(got, want):
        assert torch.equal(a, b)
    # the streams backwards in memory, with a gap between them
    buf = torch.full((S, c * D + 24), 55.0, dtype=torch.bfloat16, device="cuda")

    class Back:  # y as the entry points take it: the last stream's memory first
        def __init__(self):
            self.at = buf[S - 1:]

        def data_ptr(self):
            return self.at.data_ptr()

        def stride(self, d):
            return (-buf.stride(0), D, 1)[d]
    for call, ref in ((lambda y: conv(g["x"], w, bias, None, "bf16", "silu", lens, y=y), want[0]), (lambda y: scan(g, "bf16", lens, y=y), want[2])):
        buf.fill_(55.0)
        call(Back())
        torch.cuda.synchronize()
        assert torch.equal(buf.flip(0)[:, :c * D].view(S, c, D), ref) and (buf[:, c * D:] == 55).all()
