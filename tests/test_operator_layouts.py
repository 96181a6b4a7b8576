"""Row layouts of the convolution's and the scan's outputs: streams that would write over each other are
refused on the host, before any launch (no pointer here is ever read)."""
import ctypes as C
import itertools

import pytest

import nemoasr_b200 as nb

P = 0x10000  # aligned, never dereferenced


def test_rows_overlap():
    """Every small layout against the elements themselves."""
    f = nb.api().nb_rows_overlap
    f.argtypes = [C.c_int64] * 5
    seen = {0: 0, 1: 0}
    for streams, rows, width, ss, ld in itertools.product((1, 2, 3, 5), (1, 2, 3, 4), (1, 2, 4), range(-14, 27), range(1, 17)):
        if rows > 1 and ld < width:
            continue
        at = [s * ss + t * ld + e for s in range(streams) for t in range(rows) for e in range(width)]
        want = int(len(set(at)) < len(at))
        assert f(streams, ss, rows, ld, width) == want, (streams, ss, rows, ld, width)
        seen[want] += 1
    assert min(seen.values()) > 2000
    big = 1 << 62
    assert f(1 << 30, big, 1 << 30, 64, 64) == 0 and f(2, -big, 1 << 30, big, 64) == 1 and f(1 << 30, 64, 1 << 30, 64 << 30, 64) == 0


def conv(**kw):
    d = dict(x=P, x_ld=64, x_sstride=640, w=P, y=P, y_ld=64, y_sstride=640, streams=2, c=10, D=64, taps=4, elt=1, act=1)
    d.update(kw)
    return nb.api().nemo_causal_conv(C.byref(nb.CausalConvArgs(**d)), None)


def scan(**kw):
    d = dict(x=P, x_ld=64, x_sstride=640, dt=P, dt_ld=64, dt_sstride=640, B=P, C=P, bc_ld=16, bc_sstride=160, A=P, state_out=P, y=P, y_ld=64, y_sstride=640, streams=2,
             c=10, D=64, N=16, groups=1, elt=1)
    d.update(kw)
    return nb.api().nemo_selective_scan(C.byref(nb.SelectiveScanArgs(**d)), None)


@pytest.mark.parametrize("call", [conv, scan])
@pytest.mark.parametrize("bad", [dict(y_sstride=0), dict(y_sstride=63), dict(y_sstride=-63), dict(y_sstride=64), dict(y_sstride=639), dict(y_sstride=0, c=1), dict(y_sstride=32, c=1),
                                 dict(y_sstride=0, lens=P), dict(y_sstride=0, lens=P, c=1), dict(y_sstride=64, y_ld=64 * 3, streams=4), dict(y_sstride=100, y_ld=150)])
def test_overlapping_outputs_refused(call, bad):
    assert call(**bad) == -1 and b"overlap" in nb.api().nemo_gpu_last_error(), nb.api().nemo_gpu_last_error()
