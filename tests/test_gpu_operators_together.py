"""The 4-bit and state-space operators as they are used together: the mixer of a streaming
state-space layer (4-bit projections, causal convolution, selective scan), eager, on another
stream, captured and replayed, and next to itself; and far offsets."""
import ctypes as C
import os
import subprocess
import sys

import numpy as np
import pytest
import torch

import nemoasr_b200 as nb
import operators_ref as R

pytestmark = pytest.mark.gpu
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture(autouse=True)
def _no_device_errors():
    yield
    torch.cuda.synchronize()
    assert nb.api().nemo_gpu_check_device_errors() == 0, nb.api().nemo_gpu_last_error().decode()


class Mixer:
    """rows [S][c][d] -> out [S][c][d]: x, z = in_proj(rows); u = conv(x); dt, B, C = x_proj(u);
    y = scan(u, dt, B, C, z); out += 0.5 out_proj(y). Weights, states and every intermediate are its own."""

    def __init__(self, seed, S, c, d=128, inner=256, N=16, taps=4):
        g = np.random.default_rng(seed)
        f = lambda *s: (g.standard_normal(s)).astype(np.float32)  # noqa: E731
        dev = lambda a: torch.from_numpy(np.ascontiguousarray(a, np.float32)).cuda()  # noqa: E731
        self.S, self.c, self.d, self.inner, self.N, self.taps = S, c, d, inner, N, taps
        self.w = {k: dev(f(n, kk) / np.sqrt(kk)) for k, n, kk in (("in", 2 * inner, d), ("x", inner + 2 * N, inner), ("out", d, inner))}
        self.wq = {k: R.gpu_quantise(v, "f32") for k, v in self.w.items()}
        self.conv_w, self.conv_b = dev(f(inner, taps) / 2), dev(f(inner) * 0.1)
        self.A, self.skip, self.dt_bias = dev(-np.exp(f(inner, N) * 0.5)), dev(f(inner)), dev(g.uniform(-5, -1, inner))
        self.rows, self.lens = dev(f(S, c, d)), torch.full((S,), c, dtype=torch.int32, device="cuda")
        self.hist, self.state = torch.zeros(S, taps - 1, inner, device="cuda"), torch.zeros(S, inner, N, device="cuda")
        e = lambda *s: torch.zeros(*s, device="cuda")  # noqa: E731
        self.xz, self.u, self.dbc, self.y, self.out = e(S, c, 2 * inner), e(S, c, inner), e(S, c, inner + 2 * N), e(S, c, inner), e(S, c, d)
        self.q = {k: (torch.zeros(S * c, kk // 2, dtype=torch.uint8, device="cuda"),
                      torch.zeros(nb.api().nemo_mxfp4_scale_bytes(S * c, kk), dtype=torch.uint8, device="cuda")) for k, kk in (("in", d), ("x", inner), ("out", inner))}

    def project(self, name, src, dst, stream, acc=False, alpha=1.0):
        n, k = self.w[name].shape
        m = self.S * self.c
        q, s = self.q[name]
        nb.check(nb.api().nemo_mxfp4_quantize(src.data_ptr(), 0, k, m, k, q.data_ptr(), k // 2, s.data_ptr(), stream), "quantise")
        a = nb.GemmMxfp4Args(A=q.data_ptr(), lda=k // 2, a_scales=s.data_ptr(), W=self.wq[name][0].data_ptr(), ldw=k // 2, w_scales=self.wq[name][1].data_ptr(),
                             C=dst.data_ptr(), ldc=n, c_elt=0, M=m, N=n, K=k, act=0, accumulate=int(acc), alpha=alpha)
        nb.check(nb.api().nemo_gemm_mxfp4(C.byref(a), stream), "product")

    def step(self):
        st, S, c, D, N = R.stream_ptr(), self.S, self.c, self.inner, self.N
        self.project("in", self.rows, self.xz, st)
        a = nb.CausalConvArgs(x=self.xz.data_ptr(), x_ld=2 * D, x_sstride=2 * D * c, w=self.conv_w.data_ptr(), bias=self.conv_b.data_ptr(), hist_in=self.hist.data_ptr(),
                              hist_out=self.hist.data_ptr(), y=self.u.data_ptr(), y_ld=D, y_sstride=D * c, lens=self.lens.data_ptr(), streams=S, c=c, D=D,
                              taps=self.taps, elt=0, act=1)
        nb.check(nb.api().nemo_causal_conv(C.byref(a), st), "conv")
        self.project("x", self.u, self.dbc, st)
        w = D + 2 * N
        p = self.dbc.data_ptr()
        a = nb.SelectiveScanArgs(x=self.u.data_ptr(), x_ld=D, x_sstride=D * c, dt=p, dt_ld=w, dt_sstride=w * c, z=self.xz.data_ptr() + 4 * D, z_ld=2 * D,
                                 z_sstride=2 * D * c, B=p + 4 * D, C=p + 4 * (D + N), bc_ld=w, bc_sstride=w * c, A=self.A.data_ptr(), skip=self.skip.data_ptr(),
                                 dt_bias=self.dt_bias.data_ptr(), dt_softplus=1, state_in=self.state.data_ptr(), state_out=self.state.data_ptr(), y=self.y.data_ptr(),
                                 y_ld=D, y_sstride=D * c, lens=self.lens.data_ptr(), streams=S, c=c, D=D, N=N, groups=1, elt=0)
        nb.check(nb.api().nemo_selective_scan(C.byref(a), st), "scan")
        self.project("out", self.y, self.out, st, acc=True, alpha=0.5)

    def outputs(self):
        torch.cuda.synchronize()
        return [t.clone() for t in (self.xz, self.u, self.dbc, self.y, self.out, self.hist, self.state)]


def projected(src, w, bound_of=None):
    """64-bit product of quantised rows and weights, and its bound."""
    a, b = R.values(*R.quantise(src)), R.values(*R.quantise(w))
    return a @ b.T, src.shape[1] * 2 * R.U * (np.abs(a) @ np.abs(b).T)


@pytest.mark.parametrize("S,c", [(1, 1), (3, 1), (5, 7), (1, 40), (2, 150)])
def test_each_stage(S, c):
    """Each stage against its 64-bit form on what the stage before it wrote, with ragged rows."""
    m = Mixer(S * 100 + c, S, c)
    g = np.random.default_rng(c)
    lens = g.integers(0, c + 1, S)
    lens[0] = c
    m.lens.copy_(torch.from_numpy(lens.astype(np.int32)))
    m.hist.normal_(generator=torch.Generator("cuda").manual_seed(1))
    m.state.normal_(generator=torch.Generator("cuda").manual_seed(2))
    hist, state, out = R.f64(m.hist), R.f64(m.state), R.f64(m.out)
    m.step()
    flat = lambda t: R.f64(t).reshape(S * c, -1)  # noqa: E731
    D, N = m.inner, m.N
    want, bound = projected(flat(m.rows), R.f64(m.w["in"]))
    R.check(flat(m.xz), want, bound, "f32", "in")
    want, wh, bound = R.conv(R.f64(m.xz)[..., :D], R.f64(m.conv_w), R.f64(m.conv_b), hist, lens, "silu")
    R.check(R.f64(m.u), want, bound, "f32", "conv")
    assert np.array_equal(R.f64(m.hist), wh)
    want, bound = projected(flat(m.u), R.f64(m.w["x"]))
    R.check(flat(m.dbc), want, bound, "f32", "x")
    dbc = R.f64(m.dbc)
    wy, wh, ey, eh = R.scan(R.f64(m.u), dbc[..., :D], R.f64(m.A), dbc[..., None, D:D + N], dbc[..., None, D + N:], R.f64(m.skip), R.f64(m.xz)[..., D:],
                            R.f64(m.dt_bias), True, state, lens)
    R.check(R.f64(m.y), wy, ey, "f32", "scan")
    R.check(R.f64(m.state), wh, eh, "f32", "state")
    want, bound = projected(flat(m.y), R.f64(m.w["out"]))
    R.check(flat(m.out), out.reshape(S * c, -1) + 0.5 * want, bound + 2 * R.U * np.abs(want), "f32", "out")


@pytest.mark.parametrize("S,c", [(2, 1), (3, 7), (1, 260)])
def test_graph_and_stream_repeat_the_eager_bits(S, c):
    """Three steps, the states carried: eager, on another stream, and replayed from one graph."""
    eager, side, graph = Mixer(5, S, c), Mixer(5, S, c), Mixer(5, S, c)
    for _ in range(3):
        eager.step()
    want = eager.outputs()
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        for _ in range(3):
            side.step()
    for a, b in zip(side.outputs(), want):
        assert torch.equal(a, b)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        graph.step()
    for _ in range(3):
        g.replay()
    for a, b in zip(graph.outputs(), want):
        assert torch.equal(a, b)
    # new rows in the same buffers: a replay computes them, not what it computed before
    graph.rows.mul_(1.5)
    eager.rows.mul_(1.5)
    g.replay()
    eager.step()
    for a, b in zip(graph.outputs(), eager.outputs()):
        assert torch.equal(a, b)


@pytest.mark.parametrize("S,c", [(4, 1), (1, 700)])
def test_calls_at_once(S, c):
    """Two mixers on two streams at the same time, and two captured graphs replayed at the same time,
    share nothing: their bits are those of each alone."""
    alone = [Mixer(k, S, c) for k in (1, 2)]
    for m in alone:
        for _ in range(4):
            m.step()
    want = [m.outputs() for m in alone]
    for captured in (False, True):
        pair, streams, graphs = [Mixer(k, S, c) for k in (1, 2)], [torch.cuda.Stream() for _ in range(2)], []
        torch.cuda.synchronize()
        if captured:
            for m in pair:
                graphs.append(torch.cuda.CUDAGraph())
                with torch.cuda.graph(graphs[-1]):
                    m.step()
        for _ in range(4):
            for i in range(2):
                with torch.cuda.stream(streams[i]):
                    graphs[i].replay() if captured else pair[i].step()
        for m, w in zip(pair, want):
            for a, b in zip(m.outputs(), w):
                assert torch.equal(a, b)


def test_first_call_inside_a_capture():
    """A process whose very first calls are captured: nothing of them needs an eager call before."""
    code = f"""
import sys; sys.path[:0] = [{os.path.join(ROOT, 'nemo-c_b200')!r}, {os.path.join(ROOT, 'tests')!r}]
import torch, ctypes as C, nemoasr_b200 as nb
L = nb.api()
x = torch.randn(20, 256, device='cuda'); q = torch.zeros(20, 128, dtype=torch.uint8, device='cuda')
s = torch.zeros(L.nemo_mxfp4_scale_bytes(20, 256), dtype=torch.uint8, device='cuda'); c = torch.zeros(20, 20, device='cuda'); y = torch.zeros_like(x)
torch.cuda.synchronize()
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g):
    st = torch.cuda.current_stream().cuda_stream
    nb.check(L.nemo_mxfp4_quantize(x.data_ptr(), 0, 256, 20, 256, q.data_ptr(), 128, s.data_ptr(), st))
    a = nb.GemmMxfp4Args(A=q.data_ptr(), lda=128, a_scales=s.data_ptr(), W=q.data_ptr(), ldw=128, w_scales=s.data_ptr(), C=c.data_ptr(), ldc=20, M=20, N=20, K=256, alpha=1.0)
    nb.check(L.nemo_gemm_mxfp4(C.byref(a), st))
    nb.check(L.nemo_mxfp4_dequantize(q.data_ptr(), 128, s.data_ptr(), 20, 256, y.data_ptr(), 0, 256, st))
g.replay(); torch.cuda.synchronize()
assert torch.allclose(c, y @ y.T, rtol=1e-4, atol=1e-4) and float(c.abs().sum()) > 0
assert L.nemo_gpu_check_device_errors() == 0
print('captured')
"""
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "captured" in r.stdout, r.stderr[-2000:]


# ---- offsets past 32 bits ------------------------------------------------------------------

def test_far_streams_and_rows():
    """Streams 2^31 elements and more apart, rows 2^30 apart: offsets that do not fit 32 bits."""
    g = np.random.default_rng(0)
    S, c, D, taps, N = 2, 3, 32, 4, 16
    far = (1 << 31) + 64
    buf = torch.empty(far + c * D, dtype=torch.bfloat16, device="cuda")
    x = torch.as_strided(buf, (S, c, D), (far, D, 1))
    x.copy_(R.to_dev(g.standard_normal((S, c, D)), "bf16"))
    near = x.clone()
    w = torch.from_numpy(g.standard_normal((D, taps)).astype(np.float32)).cuda()
    ys = []
    for v in (x, near):
        y = torch.zeros(S, c, D, dtype=torch.bfloat16, device="cuda")
        a = nb.CausalConvArgs(x=v.data_ptr(), x_ld=D, x_sstride=v.stride(0), w=w.data_ptr(), y=y.data_ptr(), y_ld=D, y_sstride=c * D, streams=S, c=c, D=D, taps=taps,
                              elt=1, act=1)
        nb.check(nb.api().nemo_causal_conv(C.byref(a), R.stream_ptr()))
        ys.append(y)
    assert torch.equal(*ys) and ys[0].abs().sum() > 0
    dt, bc = R.to_dev(g.standard_normal((S, c, D)), "bf16"), R.to_dev(g.standard_normal((S, c, N)), "bf16")
    A = -torch.rand(D, N, device="cuda")
    outs = []
    for v, yl in ((x, far // 2), (near, D)):
        state = torch.zeros(S, D, N, device="cuda")
        y = torch.as_strided(torch.empty(c * yl * 2, dtype=torch.bfloat16, device="cuda"), (S, c, D), (c * yl if yl == D else D, yl, 1))
        a = nb.SelectiveScanArgs(x=v.data_ptr(), x_ld=D, x_sstride=v.stride(0), dt=dt.data_ptr(), dt_ld=D, dt_sstride=c * D, B=bc.data_ptr(), C=bc.data_ptr(), bc_ld=N,
                                 bc_sstride=c * N, A=A.data_ptr(), dt_softplus=1, state_out=state.data_ptr(), y=y.data_ptr(), y_ld=yl, y_sstride=y.stride(0), streams=S,
                                 c=c, D=D, N=N, groups=1, elt=1)
        nb.check(nb.api().nemo_selective_scan(C.byref(a), R.stream_ptr()))
        outs.append((y.clone(), state))
    assert torch.equal(outs[0][0], outs[1][0]) and torch.equal(outs[0][1], outs[1][1])


def test_far_rows_of_the_product():
    """Output rows 2^30 elements apart, code rows 2^31 bytes apart, values 2^31 elements apart."""
    g = np.random.default_rng(1)
    m, n, k = 3, 40, 64
    src = torch.empty((m - 1) * ((1 << 31) + 8) + k, dtype=torch.bfloat16, device="cuda")
    x = torch.as_strided(src, (m, k), ((1 << 31) + 8, 1))
    x.copy_(R.to_dev(g.standard_normal((m, k)), "bf16"))
    qbuf = torch.empty((m - 1) * (1 << 31) + k // 2, dtype=torch.uint8, device="cuda")
    q = torch.as_strided(qbuf, (m, k // 2), (1 << 31, 1))
    s = torch.zeros(512, dtype=torch.uint8, device="cuda")
    nb.check(nb.api().nemo_mxfp4_quantize(x.data_ptr(), 1, x.stride(0), m, k, q.data_ptr(), q.stride(0), s.data_ptr(), R.stream_ptr()))
    w = R.gpu_quantise(R.to_dev(g.standard_normal((n, k))), "f32")
    c = torch.empty((m - 1) * (1 << 30) + n, device="cuda")
    a = nb.GemmMxfp4Args(A=q.data_ptr(), lda=1 << 31, a_scales=s.data_ptr(), W=w[0].data_ptr(), ldw=k // 2, w_scales=w[1].data_ptr(), C=c.data_ptr(), ldc=1 << 30, M=m,
                         N=n, K=k, alpha=1.0)
    nb.check(nb.api().nemo_gemm_mxfp4(C.byref(a), R.stream_ptr()))
    want = R.values(*R.quantise(R.f64(x))) @ R.values(*R.unpack(*w, k)).T
    bound = k * 2 * R.U * (np.abs(R.values(*R.quantise(R.f64(x)))) @ np.abs(R.values(*R.unpack(*w, k))).T)
    R.check(R.f64(torch.as_strided(c, (m, n), (1 << 30, 1))), want, bound, "f32")
