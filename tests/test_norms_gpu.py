"""norms.BlockNorm against its formula in 64 bits, over widths that vector loads fit and do not, types, gates, strides
and aliased outputs.

Tolerance. The kernel computes in fp32 and rounds each output once to its type. A row's sums pass at most 64 sequential
additions a thread and 10 levels of a tree, every value about 20 more operations: E = 128 x 2^-24 of the terms'
magnitudes bounds the fp32 error. With M = |a r| + |b g| (|post value| + |post bias|) the magnitude of r's terms, r is
off by at most E M before its rounding, and h by E (M + mean M) |w| / s for its root s, plus twice E' |h| for the error
of s itself, E' = E rms(M) / s. Rounding is monotone, so an output lies between the rounded ends of that interval.
"""
from __future__ import annotations

import os
import subprocess
import sys
from concurrent.futures import ThreadPoolExecutor
from pathlib import Path

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

from vllm_espalier_b200 import EspError, norms
from vllm_espalier_b200 import _lib

E = 128 * 2.0 ** -24
EPS = 1e-6


def center(v, kind):
    return v - v.mean(1, keepdim=True) if kind == "layer" else v


def root(v, kind):
    return (center(v, kind).pow(2).mean(1, keepdim=True) + EPS).sqrt()


def reference(kind, act, a, b, offset, x, residual, x2, gate, post, post_bias, pre, pre_bias, use_post):
    """(r, its tolerance before rounding, h or None, its tolerance before rounding), fp64."""
    d = lambda t: None if t is None else t.double()  # noqa: E731
    x, residual, x2, gate, post, post_bias, pre, pre_bias = map(d, (x, residual, x2, gate, post, post_bias, pre,
                                                                    pre_bias))
    v = x if x2 is None else x + x2
    mag = x.abs() + (0 if x2 is None else x2.abs())
    if use_post:
        s, w = root(v, kind), (1.0 if post is None else offset + post)
        rel = mag.pow(2).mean(1, keepdim=True).sqrt() / s
        mag = (mag + mag.mean(1, keepdim=True)) / s * torch.as_tensor(w).abs()
        v = center(v, kind) / s * w
        mag = mag + 2 * rel * v.abs()
        if post_bias is not None:
            v, mag = v + post_bias, mag + post_bias.abs()
    g = 1.0
    if gate is not None:
        g = {"none": lambda t: t, "sigmoid": torch.sigmoid, "tanh": torch.tanh}[act](gate)
    v, mag = v * g * b, mag * abs(b) * torch.as_tensor(g).abs()
    if residual is not None:
        v, mag = v + a * residual, mag + (a * residual).abs()
    h = h_tol = None
    if pre is not None or pre_bias is not None:
        s = root(v, kind)
        w = offset + pre
        h = center(v, kind) / s * w
        rel = mag.pow(2).mean(1, keepdim=True).sqrt() / s
        h_tol = E * ((mag + mag.mean(1, keepdim=True)) / s * w.abs() + 2 * rel * h.abs() + h.abs())
        if pre_bias is not None:
            h, h_tol = h + pre_bias, h_tol + E * pre_bias.abs()
    return v, E * mag, h, h_tol


def check(got, want, tol):
    low, high = (want - tol).to(got.dtype), (want + tol).to(got.dtype)
    out = ~((low <= got) & (got <= high))
    assert not out.any(), f"{int(out.sum())} outside, first {got[out][:4]} for {want[out][:4]} +- {tol[out][:4]}"


def inputs(dev, rows, d, dtype, r_dtype, two, gate, layer, seed, scale=1.0):
    g = torch.Generator(device=dev).manual_seed(seed)
    n = lambda *s, std=1.0, mean=0.0, t=dtype: (torch.randn(*s, device=dev, generator=g) * std + mean).to(t)  # noqa: E731
    shape = {"none": None, "channel": (d,), "row": (rows, 1), "element": (rows, d)}[gate]
    return {"x": n(rows, d, std=scale), "residual": n(rows, d, std=3 * scale, t=r_dtype),
            "x2": n(rows, d, std=0.5 * scale) if two else None, "gate": n(*shape, mean=0.3) if shape else None,
            "post": n(d, std=0.1, mean=1.0), "post_bias": n(d, std=0.1) if layer else None,
            "pre": n(d, std=0.1, mean=1.0), "pre_bias": n(d, std=0.1) if layer else None}


def run_and_check(dev, rows, d, dtype, r_dtype, kind="rms", two=False, gate="none", act="none", use_post=True, seed=0,
                  scale=1.0, a=0.9, b=1.25, offset=0.0):
    t = inputs(dev, rows, d, dtype, r_dtype, two, gate, kind == "layer", seed, scale)
    if not use_post:
        t["post"] = t["post_bias"] = None
    op = norms.BlockNorm(d, pre=t["pre"], pre_bias=t["pre_bias"], post=t["post"], post_bias=t["post_bias"], kind=kind,
                         eps=EPS, weight_offset=offset, gate_act=act, residual_scale=a, block_scale=b)
    r, h = op(t["x"], t["residual"], x2=t["x2"], gate=t["gate"])
    assert r.dtype == r_dtype and h.dtype == dtype
    want = reference(kind, act, a, b, offset, use_post=use_post, **t)
    check(r, want[0], want[1])
    check(h, want[2], want[3])
    return op, t, r, h


DT = [(torch.bfloat16, torch.bfloat16), (torch.float16, torch.float32), (torch.float32, torch.float32),
      (torch.bfloat16, torch.float32)]


@pytest.mark.gpu
@pytest.mark.parametrize("d", [1, 2, 7, 8, 33, 128, 1000, 2047, 2048, 2056, 4096, 8191, 8192, 16384, 16392, 49152])
@pytest.mark.parametrize("rows", [1, 5])
@pytest.mark.parametrize("kind", ["rms", "layer"])
def test_widths(dev, d, rows, kind):
    dtype, r_dtype = DT[(d + rows) % 4]
    run_and_check(dev, rows, d, dtype, r_dtype, kind, two=d % 2 == 0, gate="channel", act="sigmoid", seed=d)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,r_dtype", DT)
@pytest.mark.parametrize("gate", ["none", "channel", "row", "element"])
@pytest.mark.parametrize("act", ["none", "sigmoid", "tanh"])
@pytest.mark.parametrize("d,use_post", [(2048, True), (2048, False), (515, True), (1408, True)])
def test_gates(dev, dtype, r_dtype, gate, act, d, use_post):
    run_and_check(dev, 37, d, dtype, r_dtype, "rms", two=True, gate=gate, act=act, use_post=use_post, seed=3)


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [2, 147, 149, 700, 5003])
def test_many_rows(dev, rows):
    run_and_check(dev, rows, 2048, torch.bfloat16, torch.bfloat16, two=True, gate="row", seed=rows)


@pytest.mark.gpu
@pytest.mark.parametrize("d,rows", [(8, 5000), (256, 2500), (1000, 1300), (1408, 1500), (4096, 500), (8192, 400)])
@pytest.mark.parametrize("kind,gate,act", [("rms", "element", "sigmoid"), ("layer", "channel", "tanh")])
def test_many_rows_of_other_widths(dev, d, rows, kind, gate, act):
    """More rows than the GPU takes at once, and a row alone: the same bits."""
    dtype, r_dtype = DT[d // 8 % 4]
    op, t, r, h = run_and_check(dev, rows, d, dtype, r_dtype, kind, two=d != 1000, gate=gate, act=act, seed=d)
    for i in (0, rows // 2, rows - 1):
        one = slice(i, i + 1)
        r1, h1 = op(t["x"][one], t["residual"][one], x2=None if t["x2"] is None else t["x2"][one],
                    gate=t["gate"] if gate == "channel" else t["gate"][one])
        assert torch.equal(r1, r[one]) and torch.equal(h1, h[one])


@pytest.mark.gpu
def test_weight_offset(dev):
    run_and_check(dev, 9, 2048, torch.bfloat16, torch.bfloat16, offset=1.0)


@pytest.mark.gpu
@pytest.mark.parametrize("d", [2048, 777])
def test_parts_left_out(dev, d):
    """No residual, no pre norm, norms without a weight, and the plain norm before a first block."""
    t = inputs(dev, 6, d, torch.bfloat16, torch.bfloat16, False, "none", False, 5)
    r, h = norms.BlockNorm(d, pre=t["pre"])(t["x"])
    want = reference("rms", "none", 1.0, 1.0, 0.0, t["x"], None, None, None, None, None, t["pre"], None, False)
    assert torch.equal(r, t["x"])
    check(h, want[2], want[3])
    r, h = norms.BlockNorm(d, post=t["post"], residual_scale=0.5)(t["x"], t["residual"])
    want = reference("rms", "none", 0.5, 1.0, 0.0, t["x"], t["residual"], None, None, t["post"], None, None, None, True)
    assert h is None
    check(r, want[0], want[1])
    r, h = norms.BlockNorm(d, pre=True, post=True)(t["x"], t["residual"])
    ones = torch.ones(d, device=dev)
    want = reference("rms", "none", 1.0, 1.0, 0.0, t["x"], t["residual"], None, None, None, None, ones, None, True)
    check(r, want[0], want[1])
    check(h, want[2], want[3])


@pytest.mark.gpu
@pytest.mark.parametrize("d,pad", [(2048, 0), (2048, 8), (2048, 3), (2050, 1)])
def test_strided_rows_and_outputs_in_place(dev, d, pad):
    """Rows inside a wider buffer, at an offset no vector load fits; outputs over the residual and over x."""
    dtype = torch.bfloat16
    t = inputs(dev, 21, d, dtype, dtype, True, "element", False, 7)

    def inside(v, off):
        wide = torch.full((v.shape[0], d + pad + off), float("nan"), dtype=v.dtype, device=dev)
        wide[:, off:off + d] = v
        return wide[:, off:off + d]
    op = norms.BlockNorm(d, pre=t["pre"], post=t["post"], gate_act="tanh", residual_scale=0.9)
    r0, h0 = op(t["x"], t["residual"], x2=t["x2"], gate=t["gate"])
    x, residual, gate = inside(t["x"], pad), inside(t["residual"], 0), inside(t["gate"], pad)
    r, h = op(x, residual, x2=inside(t["x2"], pad), gate=gate)
    want = reference("rms", "tanh", 0.9, 1.0, 0.0, t["x"], t["residual"], t["x2"], t["gate"], t["post"], None,
                     t["pre"], None, True)
    for q in ((r0, h0), (r, h)):
        check(q[0], want[0], want[1])
        check(q[1], want[2], want[3])
    r2, h2 = op(x, residual, x2=inside(t["x2"], pad), gate=gate, out=residual, normed=x)
    assert r2.data_ptr() == residual.data_ptr() and h2.data_ptr() == x.data_ptr()
    assert torch.equal(r2, r) and torch.equal(h2, h)
    columns = t["x"].t().contiguous().t()       # rows that are not contiguous at all
    r3, h3 = op(columns, t["residual"], x2=t["x2"], gate=t["gate"])
    assert torch.equal(r3, r0) and torch.equal(h3, h0)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("d", [1, 2, 3, 7, 8, 9, 15, 17, 31, 250, 257, 263, 1016, 1023, 1025, 2047, 2049, 4095, 8191])
@pytest.mark.parametrize("off,pad", [(0, 1), (1, 0), (3, 2), (5, 5), (6, 1), (7, 0)])
def test_any_alignment(dev, dtype, d, off, pad):
    """16-bit rows that start on any 2-byte boundary, outputs into buffers whose other values stay, and in place."""
    rows = 4
    t = inputs(dev, rows, d, dtype, dtype, True, "element", True, 11)

    def inside(v, o, fill=float("nan")):
        wide = torch.full((rows, d + off + pad + 8), fill, dtype=dtype, device=dev)
        if v is not None:
            wide[:, o:o + d] = v
        return wide, wide[:, o:o + d]
    op = norms.BlockNorm(d, pre=t["pre"], pre_bias=t["pre_bias"], post=t["post"], post_bias=t["post_bias"],
                         kind="layer", eps=EPS, gate_act="sigmoid", residual_scale=0.9, block_scale=1.25)
    x, residual = inside(t["x"], off)[1], inside(t["residual"], pad)[1]
    x2, gate = inside(t["x2"], off + 1)[1], inside(t["gate"], pad + 2)[1]
    (wide_r, r), (wide_h, h) = inside(None, off + 2, 7.0), inside(None, pad + 1, 7.0)
    op(x, residual, x2=x2, gate=gate, out=r, normed=h)
    want = reference("layer", "sigmoid", 0.9, 1.25, 0.0, use_post=True, **t)
    check(r, want[0], want[1])
    check(h, want[2], want[3])
    for wide, o in ((wide_r, off + 2), (wide_h, pad + 1)):
        assert (wide[:, :o] == 7).all() and (wide[:, o + d:] == 7).all()
    r0, h0 = r.clone(), h.clone()
    op(x, residual, x2=x2, gate=gate, out=residual, normed=x)
    assert torch.equal(residual, r0) and torch.equal(x, h0)


@pytest.mark.gpu
@pytest.mark.parametrize("d", [2048, 1023])
def test_rows_do_not_touch_each_other(dev, d):
    """A row's bits do not depend on the others, be they NaN, and not on how many there are."""
    t = inputs(dev, 300, d, torch.bfloat16, torch.bfloat16, True, "row", False, 9)
    op = norms.BlockNorm(d, pre=t["pre"], post=t["post"])
    r, h = op(t["x"], t["residual"], x2=t["x2"], gate=t["gate"])
    r1, h1 = op(t["x"][17:18], t["residual"][17:18], x2=t["x2"][17:18], gate=t["gate"][17:18])
    assert torch.equal(r[17:18], r1) and torch.equal(h[17:18], h1)
    x = t["x"].clone()
    x[::2] = float("nan")
    r2, h2 = op(x, t["residual"], x2=t["x2"], gate=t["gate"])
    assert torch.equal(r2[1::2], r[1::2]) and torch.equal(h2[1::2], h[1::2]) and r2[::2].isnan().all()


@pytest.mark.gpu
@pytest.mark.parametrize("d", [2048, 99])
def test_extreme_values(dev, d):
    """All-zero rows, values near the types' limits, constant rows of a layer norm."""
    op = norms.BlockNorm(d, pre=True, kind="rms")
    r, h = op(torch.zeros(3, d, device=dev, dtype=torch.float16), torch.zeros(3, d, device=dev))
    assert (r == 0).all() and (h == 0).all()
    x = torch.full((2, d), 60000.0, device=dev, dtype=torch.float16)
    _, h = op(x)
    assert (h == 1).all()
    x = torch.full((2, d), 1e15, device=dev)
    _, h = op(x)
    assert torch.allclose(h, torch.ones_like(h), rtol=E)
    r, h = norms.BlockNorm(d, pre=True, kind="layer")(torch.full((2, d), 8.0, device=dev, dtype=torch.bfloat16))
    assert (h == 0).all() and (r == 8).all()


@pytest.mark.gpu
def test_no_rows_and_other_streams(dev):
    op = norms.BlockNorm(64, pre=True)
    x = torch.randn(0, 64, device=dev)
    assert [t.shape for t in op(x, x)] == [x.shape, x.shape]
    t = inputs(dev, 64, 2048, torch.bfloat16, torch.bfloat16, False, "none", False, 1)
    op = norms.BlockNorm(2048, pre=t["pre"])
    r, h = op(t["x"], t["residual"])
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        r1, h1 = op(t["x"], t["residual"])
    graph, out, normed = torch.cuda.CUDAGraph(), torch.empty_like(r), torch.empty_like(h)
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        op(t["x"], t["residual"], out=out, normed=normed)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(r, r1) and torch.equal(h, h1) and torch.equal(r, out) and torch.equal(h, normed)


@pytest.mark.gpu
def test_refusals(dev):
    x = torch.zeros(4, 64, device=dev, dtype=torch.bfloat16)
    op = norms.BlockNorm(64, pre=True)
    bad = [dict(x=x[0]), dict(x=x[:, :32]), dict(x=x.cpu()), dict(x=x.long()), dict(x=x, residual=x[:2]),
           dict(x=x, x2=x.float()), dict(x=x, residual=x.long()), dict(x=x, gate=x[:2]), dict(x=x, gate=x[0].cpu()),
           dict(x=x, out=x.float()), dict(x=x, normed=x[:1])]
    for kw in bad:
        with pytest.raises(ValueError):
            op.forward(**kw)
    with pytest.raises(ValueError):
        norms.BlockNorm(64, post=True)(x, normed=x)
    for kw in (dict(d=0), dict(d=49153), dict(d=64, kind="batch"), dict(d=64, gate_act="relu"),
               dict(d=64, pre_bias=x[0]), dict(d=64, pre=x[0].cpu()), dict(d=64, pre=x[0, :8]),
               dict(d=64, pre=x[0], post=x[0].float())):
        with pytest.raises(ValueError):
            norms.BlockNorm(**kw)


def test_library_refusals():
    """The C entry point's own checks (no GPU needed: they precede any CUDA call)."""
    lib = _lib.lib()
    op = _lib.esp_block_norm_op_t(64, 0, 1, 0, 1e-6, 0.0, 1.0, 1.0, 2, None, None, None, None)

    def call(x=16, gate=None, gate_kind=0, r=16, h=16, rows=1, x_dtype=1, r_dtype=1, gate_dtype=1, op=op):
        return lib.esp_block_norm(op and _lib.C.addressof(op), x, 64, None, 0, x_dtype, None, 0, r_dtype, gate,
                                  gate_kind, gate_dtype, 0, r, 64, h, 64, rows, None)
    for kw in (dict(x=None), dict(gate_kind=1), dict(gate=16), dict(gate=16, gate_kind=4), dict(h=None), dict(rows=-1),
               dict(x_dtype=3), dict(r_dtype=-1), dict(gate=16, gate_kind=1, gate_dtype=9), dict(op=None)):
        assert call(**kw) == _lib.ESP_ERR_INVALID, kw
        assert lib.esp_last_error()
    assert call(rows=0) == _lib.ESP_OK
    for name, value in (("d", 0), ("d", 49153), ("post", 3), ("gate_act", 7), ("w_dtype", 4)):
        other = _lib.esp_block_norm_op_t.from_buffer_copy(op)
        setattr(other, name, value)
        assert call(op=other) == _lib.ESP_ERR_INVALID, name
    with pytest.raises(EspError):
        _lib.check(call(rows=-1))


@pytest.mark.gpu
def test_widths_around_the_default_shared_memory():
    """Rows of about 48 KB of fp32 in a process of its own: a wider row before them would have raised the kernel's limit."""
    code = ("import torch, test_norms_gpu as t\n"
            "for d in (12288, 12257, 12256, 8193, 12289):\n"
            "    t.run_and_check(torch.device('cuda:0'), 3, d, torch.bfloat16, torch.float32, 'layer', two=True, "
            "gate='channel', act='tanh', seed=d)\n")
    here = Path(__file__).resolve().parent
    env = dict(os.environ, PYTHONPATH=os.pathsep.join([str(here.parent), str(here), os.environ.get("PYTHONPATH", "")]))
    done = subprocess.run([sys.executable, "-c", code], env=env, capture_output=True, text=True, timeout=600)
    assert done.returncode == 0, done.stderr[-2000:]


@pytest.mark.gpu
def test_threads_of_different_widths(dev):
    """Host threads on streams of their own launch one kernel with different amounts of shared memory: the wide rows' kernel
    at two widths, the rows' ring with and without a second input."""
    g = torch.Generator(device=dev).manual_seed(1)
    wide, ring = [norms.BlockNorm(d, pre=True) for d in (13000, 40000)], norms.BlockNorm(4096, pre=True)
    w = [torch.randn(1, op.d, device=dev, generator=g) for op in wide]
    x = torch.randn(400, 4096, device=dev, generator=g).to(torch.bfloat16)
    calls = [(op, t, None) for op, t in zip(wide, w)] + [(ring, x, None), (ring, x, x)]
    want = [op(t, x2=x2)[1] for op, t, x2 in calls]

    def work(call):
        (op, t, x2), stream = call, torch.cuda.Stream()
        r, h = torch.empty_like(t), torch.empty_like(t)
        code = 2 if t.dtype == torch.float32 else 1
        at = (op._ref, t.data_ptr(), op.d, x2.data_ptr() if x2 is not None else None, op.d, code, None, 0, code, None, 0, 0, 0,
              r.data_ptr(), op.d, h.data_ptr(), op.d, t.shape[0], stream.cuda_stream)
        refused = 0
        for i in range(3000):
            refused += _lib.lib().esp_block_norm(*at) != _lib.ESP_OK
            if i % 100 == 99:
                stream.synchronize()
        return refused, h
    torch.cuda.synchronize()
    with ThreadPoolExecutor(4) as pool:
        for (refused, h), expected in zip(pool.map(work, calls), want):
            assert refused == 0 and torch.equal(h, expected)


def test_weights_on_another_device_are_refused(monkeypatch):
    """No GPU needed: tensors without storage, refused before anything reads them."""
    monkeypatch.setattr(torch.cuda, "is_available", lambda: False)      # (a GPU's would be looked for)
    with FakeTensorMode():
        w = [torch.empty(64, device=f"cuda:{i}") for i in (0, 1)]
        for kw in (dict(pre=w[0], post=w[1]), dict(pre=w[0], pre_bias=w[1])):
            with pytest.raises(ValueError, match="device"):
                norms.BlockNorm(64, **kw)
        for kw in (dict(pre=w[1]), dict(post=w[1], pre=True), dict(pre=w[1], pre_bias=w[1])):
            with pytest.raises(ValueError, match="device|cuda:1"):
                norms.BlockNorm(64, **kw)(torch.empty(2, 64, device="cuda:0"))


@pytest.mark.gpu
def test_rows_up_to_the_most_there_may_be(dev):
    """2^31 - 1 rows of eight values, the same input in each: every one of them is written (34 GB), none past the last."""
    rows, x = 2 ** 31 - 1, torch.arange(8, dtype=torch.bfloat16, device=dev)[None]
    if torch.cuda.mem_get_info(dev)[0] < 40 << 30:
        pytest.skip("less than 40 GB free")
    buffer = torch.full((rows + 1, 8), -1.0, dtype=torch.bfloat16, device=dev)
    norms.BlockNorm(8, block_scale=2.0)(x.expand(rows, 8), out=buffer[:rows])
    words, want = buffer.view(torch.int64).view(-1, 2), (2 * x).view(torch.int64)
    for at in range(0, rows, 1 << 28):
        assert (words[at:min(at + (1 << 28), rows)] == want).all()
    assert (buffer[rows] == -1).all()
    with pytest.raises(EspError):
        norms.BlockNorm(8)(x.expand(rows + 1, 8), out=x.expand(rows + 1, 8))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,gate_dtype,d", [(torch.float32, torch.float32, 2048), (torch.float32, torch.float32, 515),
                                                (torch.bfloat16, torch.bfloat16, 2048), (torch.float16, torch.float16, 515),
                                                (torch.bfloat16, torch.float32, 64), (torch.float32, torch.float32, 8200)])
@pytest.mark.parametrize("gate", ["channel", "row", "element"])
@pytest.mark.parametrize("rows", [3, 3001])
def test_sigmoid_of_an_fp32_stream(dev, dtype, gate_dtype, d, gate, rows):
    """r = 1 sigmoid(g) in fp32: the exponential is within 2 units, 1 + e and 1 / (1 + e) round once each: 3 units, of 2^-23
    of the value at most (and their products, far below a hundredth of one)."""
    if gate != "row" and gate_dtype != dtype:
        pytest.skip("rows of another type than x: one kernel for all gates")
    shape = {"channel": (d,), "row": (rows, 1), "element": (rows, d)}[gate]
    g = (torch.rand(*shape, device=dev, generator=torch.Generator(device=dev).manual_seed(d)) * 107 - 87).to(gate_dtype)
    one = torch.ones(rows, d, device=dev, dtype=dtype)
    r, _ = norms.BlockNorm(d, gate_act="sigmoid")(one, torch.zeros(rows, d, device=dev), gate=g)
    want = torch.sigmoid(g.double()).expand(rows, d)
    assert r.dtype == torch.float32
    worst = ((r.double() - want).abs() / want).max().item()
    assert worst <= 3.03 * 2.0 ** -23, worst * 2 ** 23


def test_weights_that_are_no_tensors_are_refused():
    """A list or an array is no norm without a weight."""
    for kw in (dict(pre=[1.0] * 8), dict(post=torch.ones(8).numpy()), dict(pre=2.0), dict(pre=True, pre_bias=[0.0] * 8),
               dict(post=True, post_bias=True)):
        with pytest.raises(ValueError, match="tensor"):
            norms.BlockNorm(8, **kw)
    assert norms.BlockNorm(8, pre=True, post=False).has_pre and not norms.BlockNorm(8, pre=False).has_pre
