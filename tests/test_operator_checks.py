"""Arguments of the 4-bit and state-space operators that are refused on the host, before any launch
(no pointer here is ever read), and calls that have nothing to do."""
import ctypes as C

import pytest

import nemoasr_b200 as nb

P = 0x10000  # aligned, never dereferenced


def refused(rc, word):
    assert rc == -1 and word.encode() in nb.api().nemo_gpu_last_error(), nb.api().nemo_gpu_last_error()


def test_scale_bytes():
    f = nb.api().nemo_mxfp4_scale_bytes
    assert f(1, 32) == 512 and f(128, 128) == 512 and f(129, 128) == 1024 and f(128, 160) == 1024 and f(300, 4096) == 3 * 32 * 512
    assert f(0, 128) == 0 and f(5, 0) == 0 and f(-3, 128) == 0
    assert f(1 << 33, 1 << 20) == (1 << 26) * (1 << 13) * 512  # past 32 bits


@pytest.mark.parametrize("which", ["nemo_mxfp4_quantize", "nemo_mxfp4_dequantize"])
def test_mxfp4_rows_refused(which):
    def call(x=P, elt=0, ldx=64, rows=4, K=64, q=P, ldq=32, s=P):
        f = getattr(nb.api(), which)
        return f(x, elt, ldx, rows, K, q, ldq, s, None) if which.endswith("quantize") and "de" not in which else f(q, ldq, s, rows, K, x, elt, ldx, None)
    refused(call(K=48), "multiple of 32")
    refused(call(K=-32), "bad shape")
    refused(call(rows=-1), "bad shape")
    refused(call(elt=3), "element type")
    refused(call(elt=-1), "element type")
    refused(call(x=None), "null")
    refused(call(q=None), "null")
    refused(call(s=None), "null")
    refused(call(ldx=63), "pitches")
    refused(call(ldq=31), "pitches")
    refused(call(x=P + 2), "aligned")
    refused(call(x=P + 1, elt=1), "aligned")
    assert call(rows=0, x=None) == 0 and call(K=0) == 0


def test_gemm_mxfp4_refused():
    def call(**kw):
        d = dict(A=P, lda=512, a_scales=P, W=P, ldw=512, w_scales=P, bias=P, C=P, ldc=256, c_elt=0, M=4, N=256, K=1024, act=0, accumulate=0, alpha=1.0)
        d.update(kw)
        return nb.api().nemo_gemm_mxfp4(C.byref(nb.GemmMxfp4Args(**d)), None)
    assert nb.api().nemo_gemm_mxfp4(None, None) == -1
    for name in ("A", "W", "C", "a_scales", "w_scales"):
        refused(call(**{name: None}), "null")
    refused(call(M=-1), "bad shape")
    refused(call(M=(1 << 30) + 1), "bad shape")
    refused(call(N=(1 << 31) - 1), "bad shape")
    refused(call(K=1000), "multiple of 32")
    refused(call(K=0), "multiple of 32")
    refused(call(N=128, act=3), "256")
    refused(call(act=4), "activation")
    refused(call(c_elt=7), "element type")
    refused(call(c_elt=1, accumulate=1), "fp32")
    refused(call(A=P + 8), "16-byte")
    refused(call(w_scales=P + 4), "16-byte")
    refused(call(lda=520), "16-byte")
    refused(call(lda=496), "below")
    refused(call(ldc=255), "ldc")
    refused(call(C=P + 2), "aligned")
    refused(call(bias=P + 2), "aligned")
    assert call(M=0, A=None) == 0 and call(N=0) == 0


def test_causal_conv_refused():
    def call(**kw):
        d = dict(x=P, x_ld=64, x_sstride=640, w=P, bias=P, hist_in=P, hist_out=P, y=P, y_ld=64, y_sstride=640, lens=None, streams=2, c=10, D=64, taps=4, elt=1, act=1)
        d.update(kw)
        return nb.api().nemo_causal_conv(C.byref(nb.CausalConvArgs(**d)), None)
    assert nb.api().nemo_causal_conv(None, None) == -1
    refused(call(taps=0), "taps")
    refused(call(taps=9), "taps")
    refused(call(streams=-1), "bad shape")
    refused(call(c=(1 << 30) + 1), "bad shape")
    refused(call(elt=5), "element type")
    refused(call(act=2), "activation")
    refused(call(act=3), "activation")
    for name in ("x", "y", "w"):
        refused(call(**{name: None}), "null")
    refused(call(x_ld=63), "pitches")
    refused(call(y_ld=1), "pitches")
    refused(call(hist_in=P + 1), "aligned")
    refused(call(bias=P + 2), "aligned")
    assert call(streams=0) == 0 and call(D=0) == 0 and call(c=0, hist_out=None) == 0


def test_selective_scan_refused():
    def call(**kw):
        d = dict(x=P, x_ld=64, x_sstride=640, dt=P, dt_ld=64, dt_sstride=640, z=P, z_ld=64, z_sstride=640, B=P, C=P, bc_ld=32, bc_sstride=320, A=P, skip=P, dt_bias=P,
                 dt_softplus=1, state_in=P, state_out=P, y=P, y_ld=64, y_sstride=640, lens=None, streams=2, c=10, D=64, N=16, groups=2, elt=1)
        d.update(kw)
        return nb.api().nemo_selective_scan(C.byref(nb.SelectiveScanArgs(**d)), None)
    assert nb.api().nemo_selective_scan(None, None) == -1
    refused(call(N=0), "N=0")
    refused(call(N=129), "N=129")
    refused(call(groups=0), "groups")
    refused(call(groups=3), "groups")
    refused(call(c=-1), "bad shape")
    refused(call(c=(1 << 31) - 1), "bad shape")
    refused(call(D=1 << 25, groups=1), "bad shape")
    refused(call(elt=4), "element type")
    for name in ("x", "dt", "B", "C", "A", "y"):
        refused(call(**{name: None}), "null")
    for name, v in (("x_ld", 63), ("dt_ld", 63), ("z_ld", 63), ("y_ld", 63), ("bc_ld", 31)):
        refused(call(**{name: v}), "pitches")
    refused(call(dt=P + 1), "aligned")
    refused(call(state_in=P + 2), "aligned")
    assert call(streams=0) == 0 and call(D=0, groups=1) == 0 and call(c=0, state_out=None) == 0
