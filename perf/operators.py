"""Cases for the serving operators of a streaming state-space layer: microscaled 4-bit floating
point (quantisation, product), the short causal convolution and the selective scan.

`run` computes a case in its plain form (elementary torch operations in 32 bits) or, where `own`
is true, through the library's entry points (include/nemo_gpu.h). Shapes: one encoder chunk is
1..14 rows of 1024 columns a stream, batches are 256 and 1024 streams, feed-forward layers are
4096 wide; the state-space layers are 2048 wide (twice the model) with 16 states a channel.
"""
import ctypes
import math
import os
import sys

import torch

own = False

ELT = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
ELT_ID = {"f32": 0, "bf16": 1, "f16": 2}
ACT_ID = {"none": 0, "silu": 1, "relu": 2, "glu": 3}


def listed():
    return [
        # one stream's chunk of activations, before a projection
        dict(name="quantise one chunk", op="quantise", rows=7, K=1024, elt="f32"),
        # a checkpoint's feed-forward weights of four layers, quantised at load
        dict(name="quantise weights", op="quantise", rows=16384, K=4096, elt="bf16"),
        # feed-forward output projection, one stream at the lowest latency
        dict(name="product one row", op="product", M=1, N=1024, K=4096, elt="f32", out="f32", act="none", bias=True, alpha=0.5),
        # gated projection, one stream's chunk of 560 ms
        dict(name="product chunk glu", op="product", M=7, N=2048, K=1024, elt="f32", out="f32", act="glu", bias=True, alpha=1.0),
        # feed-forward input projection of 256 streams
        dict(name="product 256 streams", op="product", M=1792, N=4096, K=1024, elt="bf16", out="bf16", act="silu", bias=True, alpha=1.0),
        # feed-forward output projection of 1024 streams with chunks of 14 rows, one stream short
        dict(name="product 1023 streams", op="product", M=14322, N=1024, K=4096, elt="bf16", out="f32", act="none", bias=True, alpha=0.5),
        # one new row for each of 256 streams
        dict(name="conv single rows", op="conv", S=256, c=1, D=2048, taps=4, elt="bf16", ragged=False),
        # a whole recording of odd length
        dict(name="conv recording", op="conv", S=1, c=32767, D=2048, taps=4, elt="bf16", ragged=False),
        # one new row for each of 256 streams
        dict(name="scan single rows", op="scan", S=256, c=1, D=2048, N=16, G=1, elt="f32", ragged=False),
        # chunks of up to 7 rows for 256 streams, each with its own number of rows
        dict(name="scan chunks", op="scan", S=256, c=7, D=2048, N=16, G=1, elt="f32", ragged=True),
        # a whole recording
        dict(name="scan recording", op="scan", S=1, c=16384, D=2048, N=16, G=1, elt="bf16", ragged=False),
        # prompts of different lengths in one batch
        dict(name="scan prompts", op="scan", S=8, c=2500, D=2048, N=16, G=1, elt="bf16", ragged=True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _one(rng):
    op = rng.choice(["quantise", "product", "product", "conv", "scan", "scan"])
    elt = rng.choice(["f32", "bf16", "f16"])
    if op == "quantise":
        return dict(op=op, rows=_log(rng, 1, 20000), K=32 * _log(rng, 1, 256), elt=elt)
    if op == "product":
        act = rng.choice(["none", "silu", "relu", "glu"])
        n = 256 * _log(rng, 1, 32) if act == "glu" else 8 * _log(rng, 4, 1024)
        return dict(op=op, M=_log(rng, 1, 16000), N=n, K=32 * _log(rng, 1, 256), elt=elt, out=rng.choice(["f32", "bf16", "f16"]), act=act,
                    bias=rng.random() < 0.7, alpha=rng.choice([0.5, 1.0]))
    streams = _log(rng, 1, 1024)
    c, d = _log(rng, 1, max(2, 33000 // streams)), 8 * _log(rng, 8, 512)
    if op == "conv":
        return dict(op=op, S=streams, c=c, D=d, taps=rng.choice([2, 3, 4, 4, 5, 8]), elt=elt, ragged=rng.random() < 0.5)
    g = rng.choice([1, 1, 2, 4])
    return dict(op=op, S=streams, c=c, D=d, N=rng.choice([1, 4, 8, 16, 16, 24, 32, 64]), G=g, elt=elt, ragged=rng.random() < 0.5)


def draw(rng):
    every = [(c["op"], work(c)) for c in listed()]
    while True:
        k = _one(rng)
        w = work(k)
        # no more bytes and no more operations than the listed cases of its operator have
        if all(w[m] <= max(v[m] for op, v in every if op == k["op"]) for m in ("bytes", "flops")):
            return k


def _rows(case):
    """Rows of each stream: all of them, or anything from none to all (a stream without any among them)."""
    s, c = case["S"], case["c"]
    if not case["ragged"]:
        return torch.full((s,), c, dtype=torch.int32)
    g = torch.Generator().manual_seed(1000003 * s + c)
    n = torch.randint(0, c + 1, (s,), generator=g, dtype=torch.int32)
    n[0] = c
    return n


def work(case):
    size = {"f32": 4, "bf16": 2, "f16": 2}
    e, op = size[case["elt"]], case["op"]
    if op == "quantise":  # the input, the codes and scales, and the values they stand for
        n = case["rows"] * case["K"]
        return {"bytes": n * (2 * e + 17 / 32), "flops": 4 * n}
    if op == "product":
        m, n, k = case["M"], case["N"], case["K"]
        out = n // 2 if case["act"] == "glu" else n
        return {"bytes": m * k * e + n * k * 17 / 32 + m * out * size[case["out"]] + 4 * n, "flops": 2 * m * n * k}
    rows, s, d = int(_rows(case).sum()), case["S"], case["D"]
    if op == "conv":
        return {"bytes": 2 * rows * d * e + 2 * s * (case["taps"] - 1) * d * e + 4 * d * (case["taps"] + 1), "flops": 2 * rows * d * (case["taps"] + 4)}
    n = case["N"]
    return {"bytes": rows * (4 * d + 2 * case["G"] * n) * e + 8 * s * d * n + 4 * d * (n + 2), "flops": rows * d * (7 * n + 10)}


def _activations(g, rows, k, elt):
    """Rows of different loudness with a few large columns, as after a normalisation's gain."""
    x = torch.randn(rows, k, generator=g, device="cuda")
    x *= torch.exp(torch.randn(rows, 1, generator=g, device="cuda") * 0.5)
    x *= torch.exp(torch.randn(1, k, generator=g, device="cuda") * 0.7)
    return x.to(ELT[elt])


def _scale_tiles(rows, k):
    return (rows + 127) // 128, (k + 127) // 128


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    op, elt = case["op"], ELT[case["elt"]]
    st = dict(case=dict(case))

    def randn(*shape):
        return torch.randn(*shape, generator=g, device="cuda")

    def scratch(rows, k):
        a, b = _scale_tiles(rows, k)
        return torch.empty(rows, k // 2, dtype=torch.uint8, device="cuda"), torch.empty(a * b * 512, dtype=torch.uint8, device="cuda")

    if op == "quantise":
        st["x"] = _activations(g, case["rows"], case["K"], case["elt"])
        st["codes"], st["scales"] = scratch(case["rows"], case["K"])
        st["values"] = torch.empty_like(st["x"])
        return st
    if op == "product":
        m, n, k = case["M"], case["N"], case["K"]
        st["x"] = _activations(g, m, k, case["elt"])
        st["w_codes"], st["w_scales"] = _pack(*_encode(randn(n, k) * (1.0 / math.sqrt(k))))
        st["bias"] = randn(n) * 0.1 if case["bias"] else None
        st["codes"], st["scales"] = scratch(m, k)
        st["y"] = torch.empty(m, n // 2 if case["act"] == "glu" else n, dtype=ELT[case["out"]], device="cuda")
        return st
    s, c, d = case["S"], case["c"], case["D"]
    st["lens"] = _rows(case).cuda() if case["ragged"] else None
    st["x"] = randn(s, c, d).to(elt)
    st["y"] = torch.zeros(s, c, d, dtype=elt, device="cuda")  # rows behind a stream's last one stay as they are
    if op == "conv":
        st["w"] = randn(d, case["taps"]) * (1.0 / math.sqrt(case["taps"]))
        st["bias"] = randn(d) * 0.1
        st["hist"] = randn(s, case["taps"] - 1, d).to(elt)
        st["hist_out"] = torch.empty_like(st["hist"])
        return st
    n, groups = case["N"], case["G"]
    st["dt"] = (randn(s, c, d) * 0.5).to(elt)
    st["z"] = randn(s, c, d).to(elt)
    st["B"] = randn(s, c, groups, n).to(elt)
    st["C"] = randn(s, c, groups, n).to(elt)
    st["A"] = -torch.arange(1, n + 1, device="cuda", dtype=torch.float32) * torch.exp(randn(d, n) * 0.1)
    st["skip"] = 1.0 + randn(d) * 0.1
    # steps between 0.001 and 0.1 at a zero input, spread evenly over their logarithm
    step = torch.exp(torch.rand(d, generator=g, device="cuda") * (math.log(0.1) - math.log(0.001)) + math.log(0.001))
    st["dt_bias"] = torch.log(torch.expm1(step))
    st["state"] = randn(s, d, n) * 0.5
    st["state_out"] = torch.empty_like(st["state"])
    return st


# ---- plain forms ---------------------------------------------------------------------------

def _encode(x):
    """Codes (0..15) and scale bytes of rows of blocks of 32: the scale is the power of two two
    below the block's largest magnitude's, codes round to nearest, ties to the even code."""
    r, k = x.shape
    b = x.float().reshape(r, k // 32, 32)
    top = b.abs().amax(-1)
    byte = ((top.view(torch.int32) >> 23) - 2).clamp(min=0)  # the exponent field: floor(log2) + 127
    inv = torch.exp2((127 - byte).float())
    v = b * inv[..., None]
    a = v.abs()
    code = (a > 0.25).int() + (a >= 0.75).int() + (a > 1.25).int() + (a >= 1.75).int() + (a > 2.5).int() + (a >= 3.5).int() + (a > 5.0).int()
    code = code + 8 * torch.signbit(v).int()
    return code.reshape(r, k).to(torch.uint8), byte.to(torch.uint8)


def _pack(codes, byte):
    """Two codes a byte, the even one low; scale bytes in tiles of 128 rows by 4 blocks."""
    r, nb = byte.shape
    a, b = (r + 127) // 128, (nb + 3) // 4
    full = torch.zeros(a * 128, b * 4, dtype=torch.uint8, device=byte.device)
    full[:r, :nb] = byte
    tiles = full.reshape(a, 4, 32, b, 4).permute(0, 3, 2, 1, 4).contiguous().reshape(-1)
    return codes[:, 0::2] | (codes[:, 1::2] << 4), tiles


def _values(codes, byte):
    """What codes and scale bytes stand for, in 32 bits."""
    table = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0, -0.0, -0.5, -1.0, -1.5, -2.0, -3.0, -4.0, -6.0], device=codes.device)
    r, k = codes.shape
    return (table[codes.int()].reshape(r, k // 32, 32) * torch.exp2(byte.float() - 127.0)[..., None]).reshape(r, k)


def _unpack(packed, tiles, k):
    r = packed.shape[0]
    a, b = _scale_tiles(r, k)
    codes = torch.stack((packed & 15, packed >> 4), -1).reshape(r, k)
    return codes, tiles.reshape(a, b, 32, 4, 4).permute(0, 3, 2, 1, 4).reshape(a * 128, b * 4)[:r, : k // 32]


def _sigmoid(v):
    return 1.0 / (1.0 + torch.exp(-v))


def _activate(v, act):
    if act == "silu":
        return v * _sigmoid(v)
    if act == "relu":
        return v.clamp(min=0)
    if act == "glu":
        h = v.shape[1] // 2
        return v[:, :h] * _sigmoid(v[:, h:])
    return v


def _plain_product(st, case):
    a = _values(*_encode(st["x"]))
    w = _values(*_unpack(st["w_codes"], st["w_scales"], case["K"]))
    v = a @ w.T
    if st["bias"] is not None:
        v = v + st["bias"]
    return (_activate(v, case["act"]) * case["alpha"]).to(ELT[case["out"]])


def _alive(st, c):
    """[S][c]: whether a row is one of its stream's."""
    if st["lens"] is None:
        return None
    return torch.arange(c, device="cuda")[None, :] < st["lens"][:, None]


def _plain_conv(st, case):
    taps, c = case["taps"], case["c"]
    u = torch.cat((st["hist"], st["x"]), 1)
    v = (u.float().unfold(1, taps, 1) * st["w"]).sum(-1) + st["bias"]
    y = (v * _sigmoid(v)).to(st["x"].dtype)
    alive = _alive(st, c)
    if alive is None:
        return y, u[:, c:].clone()
    at = st["lens"].long()[:, None] + torch.arange(taps - 1, device="cuda")[None, :]
    return torch.where(alive[..., None], y, torch.zeros_like(y)), torch.gather(u, 1, at[..., None].expand(-1, -1, u.shape[2]))


def _recurrence(a, b):
    """h[t] = a[t] h[t-1] + b[t] along axis 1 with h[-1] = 0: neighbours are joined, the half as
    long recurrence of the pairs is solved, and the steps between follow from it."""
    n = a.shape[1]
    if n == 1:
        return b
    m = n // 2
    odd_a, odd_b = a[:, 1 : 2 * m : 2], b[:, 1 : 2 * m : 2]
    half = _recurrence(odd_a * a[:, 0 : 2 * m : 2], odd_a * b[:, 0 : 2 * m : 2] + odd_b)
    h = torch.empty_like(b)
    h[:, 1 : 2 * m : 2] = half
    h[:, 0] = b[:, 0]
    rest = (n - 1) // 2  # the even steps behind the first one
    if rest:
        h[:, 2::2] = a[:, 2::2] * half[:, :rest] + b[:, 2::2]
    return h


def _plain_scan(st, case):
    s, c, d, n, groups = (case[k] for k in ("S", "c", "D", "N", "G"))
    dt = st["dt"].float() + st["dt_bias"]
    dt = torch.where(dt > 20, dt, torch.log1p(torch.exp(dt.clamp(max=20))))
    alive = _alive(st, c)
    if alive is not None:
        dt = dt * alive[..., None]  # a step of zero keeps the state
    x = st["x"].float()
    a = torch.exp(dt[..., None] * st["A"])
    wide = lambda v: v.float().repeat_interleave(d // groups, 2) if groups > 1 else v.float()  # noqa: E731
    b = (dt * x)[..., None] * wide(st["B"])
    b[:, 0] += a[:, 0] * st["state"]
    h = _recurrence(a, b)
    y = (h * wide(st["C"])).sum(-1) + st["skip"] * x
    z = st["z"].float()
    y = (y * (z * _sigmoid(z))).to(st["x"].dtype)
    return (y if alive is None else torch.where(alive[..., None], y, torch.zeros_like(y))), h[:, -1].clone()


# ---- the library's entry points ------------------------------------------------------------

def _library():
    sys.path.insert(0, os.path.join(os.getcwd(), "nemo-c_b200"))
    import nemoasr_b200
    return nemoasr_b200


def _ptr(t):
    return None if t is None else t.data_ptr()


def _own(st, case):
    nb = sys.modules.get("nemoasr_b200") or _library()
    lib, op, stream = nb.api(), case["op"], torch.cuda.current_stream().cuda_stream
    if op in ("quantise", "product"):
        x, k = st["x"], case["K"]
        nb.check(lib.nemo_mxfp4_quantize(x.data_ptr(), ELT_ID[case["elt"]], k, x.shape[0], k, st["codes"].data_ptr(), k // 2, st["scales"].data_ptr(), stream),
                 "nemo_mxfp4_quantize")
        if op == "quantise":
            nb.check(lib.nemo_mxfp4_dequantize(st["codes"].data_ptr(), k // 2, st["scales"].data_ptr(), x.shape[0], k, st["values"].data_ptr(),
                                               ELT_ID[case["elt"]], k, stream), "nemo_mxfp4_dequantize")
            return st["values"]
        y = st["y"]
        a = nb.GemmMxfp4Args(A=st["codes"].data_ptr(), lda=k // 2, a_scales=st["scales"].data_ptr(), W=st["w_codes"].data_ptr(), ldw=k // 2,
                             w_scales=st["w_scales"].data_ptr(), bias=_ptr(st["bias"]), C=y.data_ptr(), ldc=y.shape[1], c_elt=ELT_ID[case["out"]],
                             M=case["M"], N=case["N"], K=k, act=ACT_ID[case["act"]], accumulate=0, alpha=case["alpha"])
        nb.check(lib.nemo_gemm_mxfp4(ctypes.byref(a), stream), "nemo_gemm_mxfp4")
        return y
    s, c, d, e = case["S"], case["c"], case["D"], ELT_ID[case["elt"]]
    x, y = st["x"], st["y"]
    if op == "conv":
        a = nb.CausalConvArgs(x=x.data_ptr(), x_ld=d, x_sstride=c * d, w=st["w"].data_ptr(), bias=st["bias"].data_ptr(), hist_in=st["hist"].data_ptr(),
                              hist_out=st["hist_out"].data_ptr(), y=y.data_ptr(), y_ld=d, y_sstride=c * d, lens=_ptr(st["lens"]), streams=s, c=c, D=d,
                              taps=case["taps"], elt=e, act=ACT_ID["silu"])
        nb.check(lib.nemo_causal_conv(ctypes.byref(a), stream), "nemo_causal_conv")
        return y, st["hist_out"]
    n, gn = case["N"], case["G"] * case["N"]
    a = nb.SelectiveScanArgs(x=x.data_ptr(), x_ld=d, x_sstride=c * d, dt=st["dt"].data_ptr(), dt_ld=d, dt_sstride=c * d, z=st["z"].data_ptr(), z_ld=d,
                             z_sstride=c * d, B=st["B"].data_ptr(), C=st["C"].data_ptr(), bc_ld=gn, bc_sstride=c * gn, A=st["A"].data_ptr(),
                             skip=st["skip"].data_ptr(), dt_bias=st["dt_bias"].data_ptr(), dt_softplus=1, state_in=st["state"].data_ptr(),
                             state_out=st["state_out"].data_ptr(), y=y.data_ptr(), y_ld=d, y_sstride=c * d, lens=_ptr(st["lens"]), streams=s, c=c, D=d,
                             N=n, groups=case["G"], elt=e)
    nb.check(lib.nemo_selective_scan(ctypes.byref(a), stream), "nemo_selective_scan")
    return y, st["state_out"]


def run(st):
    case = st["case"]
    if own:
        return _own(st, case)
    if case["op"] == "quantise":
        return _values(*_encode(st["x"])).to(st["x"].dtype)
    if case["op"] == "product":
        return _plain_product(st, case)
    if case["op"] == "conv":
        return _plain_conv(st, case)
    return _plain_scan(st, case)


# ---- the definitions in 64 bits ------------------------------------------------------------

def _nearest(x):
    """Rows in 64 bits, each block of 32 rounded to the grid 0, 0.5 .. 2, 3, 4, 6 times its power of two."""
    r, k = x.shape
    v = x.double().reshape(r, k // 32, 32)
    _, e = torch.frexp(v.abs().amax(-1, keepdim=True))  # |top| in [2^(e-1), 2^e)
    scale = torch.ldexp(torch.ones_like(v[..., :1]), (e - 3).clamp(min=-127))
    q = v / scale
    _, f = torch.frexp(q.abs())
    grid = torch.ldexp(torch.ones_like(q), (f - 2).clamp(min=-1))  # half of the value's power of two: one bit behind the first
    return ((torch.round(q / grid) * grid).clamp(-6, 6) * scale).reshape(r, k)


def exact(case, seed):
    st, op = prepare(case, seed), case["op"]
    if op == "quantise":
        return _nearest(st["x"])
    if op == "product":
        k, n = case["K"], case["N"]
        low = torch.arange(n, device="cuda")
        kb = torch.arange(k // 32, device="cuda")
        tile = (low // 128)[:, None] * ((k + 127) // 128) + (kb // 4)[None, :]
        byte = st["w_scales"][tile * 512 + ((low % 32) * 16 + (low % 128) // 32 * 4)[:, None] + (kb % 4)[None, :]].double()
        nib = torch.empty(n, k, dtype=torch.int64, device="cuda")
        nib[:, 0::2], nib[:, 1::2] = (st["w_codes"] & 15).long(), (st["w_codes"] >> 4).long()
        e, m = (nib & 7) >> 1, (nib & 1).double()
        mag = torch.where(e == 0, m * 0.5, (1 + m * 0.5) * torch.pow(2.0, (e - 1).double()))
        w = torch.where(nib >= 8, -mag, mag) * torch.pow(2.0, byte - 127).repeat_interleave(32, 1)
        v = _nearest(st["x"]) @ w.T
        if st["bias"] is not None:
            v = v + st["bias"].double()
        if case["act"] == "glu":
            v = v[:, : n // 2] * torch.sigmoid(v[:, n // 2 :])
        elif case["act"] == "silu":
            v = v * torch.sigmoid(v)
        elif case["act"] == "relu":
            v = torch.relu(v)
        return v * case["alpha"]
    s, c, d = case["S"], case["c"], case["D"]
    rows = _rows(case).cuda()
    x = st["x"].double()
    y = torch.zeros(s, c, d, dtype=torch.float64, device="cuda")
    if op == "conv":
        taps = case["taps"]
        u = torch.cat((st["hist"].double(), x), 1)
        for j in range(taps):
            y += u[:, j : j + c] * st["w"][:, j].double()
        y += st["bias"].double()
        y *= torch.sigmoid(y)
        y[torch.arange(c, device="cuda")[None, :] >= rows[:, None]] = 0
        return y, torch.stack([u[i, int(rows[i]) : int(rows[i]) + taps - 1] for i in range(s)])
    n, groups = case["N"], case["G"]
    h, A = st["state"].double(), st["A"].double()
    for t in range(c):
        on = (rows > t)[:, None, None]
        dt = torch.nn.functional.softplus(st["dt"][:, t].double() + st["dt_bias"].double(), threshold=1000)[..., None]
        b, g = (v[:, t].double()[:, :, None, :].expand(s, groups, d // groups, n).reshape(s, d, n) for v in (st["B"], st["C"]))
        h = torch.where(on, torch.exp(dt * A) * h + dt * x[:, t, :, None] * b, h)
        z = st["z"][:, t].double()
        y[:, t] = torch.where(on[..., 0], ((h * g).sum(-1) + st["skip"].double() * x[:, t]) * z * torch.sigmoid(z), y[:, t])
    return y, h
