"""adapters.Adapters against the formula in 64 bits, over batch sizes and mixes, ranks, widths, types and strides; what
lies past a slot's rank or in another slot is never read.

Tolerance. u = x A^T is a sum of K exact products in fp32: a matrix instruction may truncate each of its additions (2^-23
of the magnitudes), in chains of at most K / 16 + 16 of them, and u may be carried as two 16-bit halves (2^-16 of it): e_u
= (K / 16 + 16) 2^-23 |x| |A|^T + 2^-16 |u|. The second product adds (rank / 8 + 16) 2^-23 |u| |B|^T, the sum with y one
fp32 rounding. Rounding to the output's type is monotone, so an output lies between the rounded ends of that interval.
"""
from __future__ import annotations

from concurrent.futures import ThreadPoolExecutor

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

from vllm_espalier_b200 import _lib, adapters


def make(dev, dtype, k, widths, slots, rank, seed, ranks=None, poison=True):
    """Random adapters; past each slot's rank rounded up to 8 NaN (poison), zeros between."""
    g = torch.Generator(device=dev).manual_seed(seed)
    a = (torch.randn(slots, len(widths), rank, k, device=dev, generator=g) * k ** -0.5).to(dtype)
    b = (torch.randn(slots, sum(widths), rank, device=dev, generator=g) * rank ** -0.5).to(dtype)
    if ranks is None:
        ranks = [max(1, rank - 3 * (s % 4)) if s % 5 != 4 else 0 for s in range(slots)]
    for s, q in enumerate(ranks):
        up = -(-q // 8) * 8
        a[s, :, q:up], b[s, :, q:up] = 0, 0
        if poison:
            a[s, :, up:], b[s, :, up:] = float("nan"), float("nan")
    scales = torch.rand(slots, device=dev, generator=g) + 0.5
    return adapters.Adapters(a, b, widths, torch.tensor(ranks, dtype=torch.int32, device=dev), scales)


def rows(dev, ad, T, seed, ids="mixed"):
    g = torch.Generator(device=dev).manual_seed(seed + 1000)
    x = torch.randn(T, ad.k, device=dev, generator=g).to(ad.dtype)
    y = torch.randn(T, ad.n, device=dev, generator=g).to(ad.dtype)
    if ids == "mixed":
        i = torch.randint(-1, ad.slots, (T,), device=dev, generator=g)
    elif ids == "runs":
        i = (torch.arange(T, device=dev) * 3 // max(1, T)) % ad.slots
    else:
        i = torch.full((T,), ids, device=dev)
    return x, y, i.to(torch.int32)


def reference(ad, x, y, ids):
    """(out, tolerance before the output's rounding) in fp64."""
    out, tol = y.double(), 2.0 ** -24 * y.double().abs()
    K = ad.k
    for s in sorted(set(ids.tolist())):
        if not 0 <= s < ad.slots:
            continue
        q = ad.rank if ad.ranks is None else int(ad.ranks[s])
        at, scale, col = (ids == s).nonzero()[:, 0], 1.0 if ad.scales is None else float(ad.scales[s]), 0
        if q == 0:
            continue
        xs = x[at].double()
        for m, w in enumerate(ad.widths):
            a, b = ad.a[s, m, :q].double(), ad.b[s, col:col + w, :q].double()
            u, mag = xs @ a.T, xs.abs() @ a.abs().T
            e_u = (K / 16 + 16) * 2.0 ** -23 * mag + 2.0 ** -16 * u.abs()
            out[at, col:col + w] += scale * (u @ b.T)
            tol[at, col:col + w] += scale * (e_u @ b.abs().T + (q / 8 + 16) * 2.0 ** -23 * (u.abs() @ b.abs().T))
            col += w
    return out, tol + 2.0 ** -24 * out.abs()


def check(got, ad, x, y, ids):
    want, tol = reference(ad, x, y, ids)
    low, high = (want - tol).to(got.dtype), (want + tol).to(got.dtype)
    bad = ~((low <= got) & (got <= high))
    assert not bad.any(), f"{int(bad.sum())} outside, first {got[bad][:4]} for {want[bad][:4]} +- {tol[bad][:4]}"
    plain = (ids < 0) | (ids >= ad.slots)
    assert torch.equal(got[plain], y[plain])


@pytest.mark.gpu
@pytest.mark.parametrize("T", [1, 2, 3, 15, 16, 17, 31, 48, 63, 64, 65, 100, 128, 129, 257, 1000, 2500])
@pytest.mark.parametrize("ids", ["mixed", "runs", 2])
def test_batches(dev, T, ids):
    ad = make(dev, torch.bfloat16, 2048, [512, 128, 128], 6, 16, T)
    x, y, i = rows(dev, ad, T, T, ids)
    check(ad(x, y, i), ad, x, y, i)


@pytest.mark.gpu
@pytest.mark.parametrize("rank", [8, 16, 24, 32, 40, 48, 56, 64, 72, 96, 120, 128])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("T", [5, 200])
def test_ranks(dev, rank, dtype, T):
    ad = make(dev, dtype, 512, [256, 72], 7, rank, rank)
    x, y, i = rows(dev, ad, T, rank)
    check(ad(x, y, i), ad, x, y, i)


@pytest.mark.gpu
@pytest.mark.parametrize("k", [8, 16, 24, 40, 256, 264, 1032, 2048, 4096, 6000])
@pytest.mark.parametrize("widths", [[8], [32], [40], [136, 8, 24], [256, 256, 64, 32], [1400, 136, 136]])
@pytest.mark.parametrize("T", [4, 90])
def test_shapes(dev, k, widths, T):
    dtype = torch.float16 if k % 16 else torch.bfloat16
    ad = make(dev, dtype, k, widths, 3, 16, k)
    x, y, i = rows(dev, ad, T, k)
    check(ad(x, y, i), ad, x, y, i)


@pytest.mark.gpu
@pytest.mark.parametrize("T,rank", [(1, 128), (77, 128), (700, 128), (700, 64)])
def test_four_wide_matrices(dev, T, rank):
    ad = make(dev, torch.bfloat16, 384, [256, 128, 128, 256], 3, rank, T)
    x, y, i = rows(dev, ad, T, 4)
    check(ad(x, y, i), ad, x, y, i)


@pytest.mark.gpu
@pytest.mark.parametrize("slots", [1, 33, 1000, 4096])
@pytest.mark.parametrize("T", [40, 600])
def test_many_slots(dev, slots, T):
    ad = make(dev, torch.float16, 64, [64], slots, 8, slots)
    x, y, i = rows(dev, ad, T, slots)
    check(ad(x, y, i), ad, x, y, i)


@pytest.mark.gpu
@pytest.mark.parametrize("T", [7, 300])
def test_no_ranks_no_scales(dev, T):
    full = make(dev, torch.bfloat16, 256, [128, 64], 4, 24, 1, ranks=[24] * 4)
    ad = adapters.Adapters(full.a, full.b, full.widths)
    x, y, i = rows(dev, ad, T, 3)
    check(ad(x, y, i), ad, x, y, i)


@pytest.mark.gpu
@pytest.mark.parametrize("T", [9, 33, 64, 65, 500])
def test_rows_without_an_adapter_keep_y(dev, T):
    """Ids -1, past the slots and at the type's ends, and a slot of rank 0: y's bits, NaN in x or not."""
    ad = make(dev, torch.bfloat16, 256, [128], 5, 16, 1)
    x, y, i = rows(dev, ad, T, 0, 0)
    i[1::2] = torch.tensor([-1, 5, 2 ** 31 - 1, -2 ** 31, 4], dtype=torch.int32, device=dev)[
        torch.arange(T // 2, device=dev) % 5]
    x[1::2] = float("nan")
    got = ad(x, y, i)
    assert torch.equal(got[1::2], y[1::2])
    check(got[::2], ad, x[::2], y[::2], i[::2])
    i.fill_(-1)
    assert torch.equal(ad(x, y, i), y)
    z = y.clone()
    assert ad(x, z, i, out=z) is z and torch.equal(z, y)


@pytest.mark.gpu
@pytest.mark.parametrize("T", [5, 50, 400])
def test_strides_and_in_place(dev, T):
    ad = make(dev, torch.bfloat16, 256, [128, 64], 4, 16, 2)
    x, y, i = rows(dev, ad, T, 6)
    want = ad(x, y, i)
    wide_x = torch.full((T, 256 + 24), float("nan"), dtype=x.dtype, device=dev)
    wide_x[:, 8:264] = x
    wide_y = torch.full((T, 192 + 16), float("nan"), dtype=y.dtype, device=dev)
    wide_y[:, 16:] = y
    out = torch.full((T, 200), 7.0, dtype=y.dtype, device=dev)
    ad(wide_x[:, 8:264], wide_y[:, 16:], i, out=out[:, :192])
    assert torch.equal(out[:, :192], want) and (out[:, 192:] == 7).all()
    ad(x, wide_y[:, 16:], i, out=wide_y[:, 16:])
    assert torch.equal(wide_y[:, 16:], want) and wide_y[:, :16].isnan().all()
    odd = torch.empty(T, 257, dtype=x.dtype, device=dev)       # rows on no 16-byte boundary, and columns first
    odd[:, 1:] = x
    assert torch.equal(ad(odd[:, 1:], y, i), want)
    assert torch.equal(ad(x.t().contiguous().t(), y.t().contiguous().t(), i), want)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_a_rows_bits_are_its_own(dev, dtype):
    """The same row gives the same bits alone, in a decode batch, in a prefill of one adapter and in a shuffled one,
    whatever (NaN included) stands in the other rows."""
    ad = make(dev, dtype, 2048, [4096, 512, 512], 8, 64, 3)
    x, y, i = rows(dev, ad, 3000, 1)
    want = ad(x, y, i)
    for lo, hi in ((0, 1), (5, 6), (0, 40), (100, 164), (100, 165), (7, 900)):
        assert torch.equal(ad(x[lo:hi], y[lo:hi], i[lo:hi].contiguous()), want[lo:hi])
    order = torch.randperm(3000, device=dev)
    assert torch.equal(ad(x[order], y[order], i[order]), want[order])
    same = torch.full_like(i, int(i[3]))
    if int(i[3]) >= 0:
        assert torch.equal(ad(x, y, same)[3], want[3])
    x2 = x.clone()
    x2[1::2] = float("nan")
    assert torch.equal(ad(x2, y, i)[::2], want[::2])


@pytest.mark.gpu
def test_large_inner_products_in_fp16(dev):
    """u past fp16's range (its own 65504): the sum is held in more."""
    ad = make(dev, torch.float16, 512, [64], 2, 16, 5, ranks=[16, 16])
    ad.a.fill_(8.0)
    ad.b.copy_((torch.randn(ad.b.shape, device=dev, generator=torch.Generator(device=dev).manual_seed(1)) * 2 ** -10))
    x, y, i = rows(dev, ad, 40, 2, 1)
    x.abs_().mul_(60.0)
    check(ad(x, y, i), ad, x, y, i)


@pytest.mark.gpu
@pytest.mark.parametrize("T", [20, 300])
def test_streams_and_graphs(dev, T):
    ad = make(dev, torch.bfloat16, 512, [256], 4, 16, 2)
    x, y, i = rows(dev, ad, T, 6)
    want = ad(x, y, i)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        other = ad(x, y, i)
    out, graph = torch.empty_like(y), torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        ad(x, y, i, out=out)
    i2 = i.flip(0).contiguous()
    want2 = ad(x, y, i2)
    i.copy_(i2)                    # a replay takes the ids of its time
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(want, other) and torch.equal(out, want2)


@pytest.mark.gpu
def test_load_and_clear(dev):
    ad = adapters.Adapters.empty(128, [64, 32], 3, 16, torch.float16, dev)
    x, y, i = rows(dev, ad, 12, 1)
    assert torch.equal(ad(x, y, i), y)
    g = torch.Generator().manual_seed(4)
    a = [torch.randn(5, 128, generator=g) * 0.1, torch.randn(5, 128, generator=g) * 0.1]
    b = [torch.randn(64, 5, generator=g), torch.randn(32, 5, generator=g)]
    ad.a[1].fill_(float("nan"))      # what an earlier adapter left
    ad.load(1, a, b, scale=0.25)
    check(ad(x, y, i), ad, x, y, i)
    ad.load(2, [a[0], None], [b[0], None])
    got = ad(x, y, i)
    check(got, ad, x, y, i)
    assert torch.equal(got[i == 2][:, 64:], y[i == 2][:, 64:])
    ad.clear(1)
    ad.clear(2)
    assert torch.equal(ad(x, y, i), y)
    for args in ((3, a, b), (-1, a, b), (0, a[:1], b), (0, [None, None], [None, None]), (0, [a[0], None], b),
                 (0, [a[0][:, :8], None], [b[0], None]), (0, [torch.zeros(17, 128), None], [torch.zeros(64, 17), None])):
        with pytest.raises(ValueError):
            ad.load(*args)
    with pytest.raises(ValueError):
        ad.clear(3)


@pytest.mark.gpu
def test_refusals(dev):
    ad = make(dev, torch.bfloat16, 64, [32, 16], 3, 8, 1)
    x, y, i = rows(dev, ad, 4, 1)
    assert ad(x[:0], y[:0], i[:0]).shape == (0, 48)
    bad = [(x.half(), y, i), (x[:, :32], y, i), (x, y[:, :40], i), (x, y[:3], i), (x, y, i[:3]), (x, y, i.long()),
           (x.cpu(), y, i), (x, y, i.cpu()), (x[0], y, i), (x, y, i.repeat(2)[::2])]
    for args in bad:
        with pytest.raises(ValueError):
            ad(*args)
    for out in (y[:3], y.float(), torch.empty(4, 49, dtype=y.dtype, device=dev)[:, 1:]):
        with pytest.raises(ValueError):
            ad(x, y, i, out=out)
    a, b = ad.a, ad.b
    for args in ((a[0], b, [32, 16]), (a, b, [48]), (a, b, [32, 24]), (a.float(), b.float(), [32, 16]),
                 (a, b.half(), [32, 16]), (a.cpu(), b.cpu(), [32, 16]), (a, b, [32, 16], ad.ranks.long()),
                 (a, b, [32, 16], ad.ranks[:2]), (a, b, [32, 16], None, ad.scales.half()),
                 (a[:, :, :, ::2], b, [32, 16]), (a[:, :, :4], b[:, :, :4], [32, 16])):
        with pytest.raises(ValueError):
            adapters.Adapters(*args)


def test_library_refusals():
    lib = _lib.lib()

    def call(x=16, ids=16, out=16, t=4, xs=64, ws=None, ws_bytes=0, **kw):
        ad = _lib.esp_adapters_t(16, 16, None, None, 1, 2, 8, 64, 1, (_lib.I * 4)(32))
        for name, v in kw.items():
            if name == "width":
                ad.widths[0] = v
            else:
                setattr(ad, name, v)
        return lib.esp_adapt(_lib.C.addressof(ad), x, xs, 16, 32, ids, t, out, 32, ws, ws_bytes, None)
    for kw in (dict(x=None), dict(ids=None), dict(out=None), dict(t=-1), dict(x=24), dict(xs=60), dict(dtype=2),
               dict(slots=0), dict(slots=4097), dict(rank=4), dict(rank=136), dict(rank=12), dict(k=60), dict(k=0),
               dict(n_mats=0), dict(n_mats=5), dict(width=20), dict(width=0), dict(a=None), dict(b=24)):
        assert call(**kw) == _lib.ESP_ERR_INVALID, kw
        assert lib.esp_last_error()
    assert call(t=0) == _lib.ESP_OK
    assert lib.esp_adapt(None, 16, 64, 16, 32, 16, 1, 16, 32, None, 0, None) == _lib.ESP_ERR_INVALID
    if lib.esp_adapt_ws_bytes(1000, 2):
        assert call(t=1000) == _lib.ESP_ERR_SCRATCH
        assert call(t=1000, ws=16, ws_bytes=lib.esp_adapt_ws_bytes(1000, 2) - 1) == _lib.ESP_ERR_SCRATCH
        assert call(t=1000, ws=20, ws_bytes=1 << 20) == _lib.ESP_ERR_SCRATCH


# Tiles of 64 rows (more than 1024 rows on 148 SMs, 24 or 40 an adapter): the same properties there.
@pytest.mark.gpu
@pytest.mark.parametrize("rank", [8, 16, 24, 32, 40, 56, 64, 72, 128])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("widths", [[264], [256, 72], [256, 72, 40]])
def test_prefill_ranks(dev, rank, dtype, widths):
    ad = make(dev, dtype, 528, widths, 7, rank, rank)
    x, y, i = rows(dev, ad, 1100, rank, "runs" if rank % 16 else "mixed")
    check(ad(x, y, i), ad, x, y, i)


@pytest.mark.gpu
@pytest.mark.parametrize("k", [8, 24, 40, 256, 1032, 6000])
@pytest.mark.parametrize("widths", [[8], [40], [136, 8, 24], [256, 256, 64, 32], [1400, 136, 136]])
@pytest.mark.parametrize("rank", [16, 32])
def test_prefill_shapes(dev, k, widths, rank):
    ad = make(dev, torch.float16 if k % 16 else torch.bfloat16, k, widths, 3, rank, k)
    x, y, i = rows(dev, ad, 1090, k)
    check(ad(x, y, i), ad, x, y, i)


@pytest.mark.gpu
@pytest.mark.parametrize("T", [1024, 1025, 1039, 1087, 1088, 1089, 4100])
@pytest.mark.parametrize("slots,ids", [(5, "runs"), (5, "mixed"), (42, "runs"), (46, "mixed")])
def test_prefill_batches(dev, T, slots, ids):
    ad = make(dev, torch.bfloat16, 256, [128, 40, 40], slots, 32, T)
    x, y, i = rows(dev, ad, T, T, ids)
    check(ad(x, y, i), ad, x, y, i)


@pytest.mark.gpu
def test_prefill_rows_streams_and_strides(dev):
    test_no_ranks_no_scales(dev, 1200)
    test_rows_without_an_adapter_keep_y(dev, 1201)
    test_strides_and_in_place(dev, 1202)
    test_streams_and_graphs(dev, 1203)


@pytest.mark.gpu
def test_a_rows_bits_are_its_own_at_rank_32(dev):
    """Rank 32 of three matrices takes shorter rings in a prefill: the same bits as in a decode batch and alone."""
    ad = make(dev, torch.bfloat16, 2048, [1024, 256, 256], 4, 32, 3)
    x, y, i = rows(dev, ad, 2000, 1)
    want = ad(x, y, i)
    for lo, hi in ((0, 1), (5, 45), (100, 300), (0, 1024), (0, 1025)):
        assert torch.equal(ad(x[lo:hi], y[lo:hi], i[lo:hi].contiguous()), want[lo:hi])


@pytest.mark.gpu
def test_threads_of_different_adapters(dev):
    """Host threads on streams of their own use adapters of one rank and of one matrix or three: one kernel, two amounts of
    shared memory."""
    calls = []
    for widths in ([128], [128, 64, 64]):
        ad = make(dev, torch.bfloat16, 256, widths, 3, 64, 7)
        calls += [(ad, rows(dev, ad, 1100, 5))] * 2
    want = [ad(*r) for ad, r in calls]

    def work(call):
        (ad, (x, y, ids)), stream = call, torch.cuda.Stream()
        out, need = torch.empty_like(y), _lib.lib().esp_adapt_ws_bytes(1100, 3)
        ws = torch.empty(need, dtype=torch.uint8, device=dev)
        at = (ad._ref, x.data_ptr(), ad.k, y.data_ptr(), ad.n, ids.data_ptr(), 1100, out.data_ptr(), ad.n, ws.data_ptr(), need,
              stream.cuda_stream)
        refused = 0
        for i in range(2000):
            refused += _lib.lib().esp_adapt(*at) != _lib.ESP_OK
            if i % 50 == 49:
                stream.synchronize()
        stream.synchronize()
        return refused, out
    torch.cuda.synchronize()
    with ThreadPoolExecutor(4) as pool:
        for (refused, out), expected in zip(pool.map(work, calls), want):
            assert refused == 0 and torch.equal(out, expected)


def test_sizes_past_the_calls_integers_are_refused(monkeypatch):
    """No GPU and no memory needed: shapes without storage."""
    monkeypatch.setattr(torch.cuda, "is_available", lambda: False)
    with FakeTensorMode():
        e = lambda *s, t=torch.float16: torch.empty(*s, dtype=t, device="cuda:0")  # noqa: E731
        ad = adapters.Adapters(e(1, 1, 8, 8), e(1, 8, 8), [8])
        for rows in (2 ** 26 + 1, 2 ** 32 + 4):
            with pytest.raises(ValueError, match="rows"):
                ad(e(rows, 8), e(rows, 8), e(rows, t=torch.int32))
        for k, n in ((2 ** 32 + 8, 8), (8, 2 ** 32 + 8), (2 ** 30 + 8, 8)):
            with pytest.raises(ValueError, match="at most"):
                adapters.Adapters(e(1, 1, 8, k), e(1, n, 8), [n])
    ad = _lib.esp_adapters_t(16, 16, None, None, 1, 2, 8, 64, 1, (_lib.I * 4)(32))
    for name, value in (("k", 2 ** 31 - 8), ("width", 2 ** 31 - 136)):
        other = _lib.esp_adapters_t.from_buffer_copy(ad)
        if name == "width":
            other.widths[0] = value
        else:
            other.k = value
        assert _lib.lib().esp_adapt(_lib.C.addressof(other), 16, 64, 16, 32, 16, 1, 16, 32, None, 0,
                                    None) == _lib.ESP_ERR_INVALID, name


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("rank", [16, 32, 64, 128])
@pytest.mark.parametrize("T", [1, 50, 1100])
def test_inner_products_are_held_in_fp32(dev, dtype, rank, T):
    """Two inner products whose leading 20 bits cancel in the output: every product and sum is exact in fp32, so 2^-20
    comes out, and nothing where the inner products are held in fewer than 21 bits."""
    ad = adapters.Adapters(torch.zeros(1, 1, rank, 256, dtype=dtype, device=dev),
                           torch.zeros(1, 64, rank, dtype=dtype, device=dev), [64])
    x = torch.zeros(T, 256, dtype=dtype, device=dev)
    x[:, [3, 100, 200]] = 1
    for r, values in ((1, (1, 2.0 ** -9, 2.0 ** -20)), (6, (-1, -2.0 ** -9, 0))):
        ad.a[0, 0, r, [3, 100, 200]] = torch.tensor(values, device=dev).to(dtype)
        ad.b[0, :, r] = 1
    got = ad(x, torch.zeros(T, 64, dtype=dtype, device=dev), torch.zeros(T, dtype=torch.int32, device=dev))
    assert (got == 2.0 ** -20).all(), got.unique()


@pytest.mark.gpu
@pytest.mark.parametrize("widths", [[64, 40], [32, 40, 64], [32, 32, 32, 64]])
@pytest.mark.parametrize("rank", [8, 16, 32, 64, 128])
@pytest.mark.parametrize("T", [3, 1100])
def test_a_large_matrix_leaves_the_others_their_digits_in_fp16(dev, widths, rank, T):
    """Inner products of the first matrix 2^30 times those of the others: each keeps 2^-16 of itself."""
    ad = make(dev, torch.float16, 256, widths, 2, rank, 5, ranks=[rank, rank])
    ad.a[:, 0].mul_(2.0 ** 14)
    ad.a[:, 1:].mul_(2.0 ** -16)
    ad.b[:, :widths[0]].mul_(2.0 ** -8)
    ad.b[:, widths[0]:].mul_(2.0 ** 11)
    x, y, i = rows(dev, ad, T, 4)
    check(ad(x, y.zero_(), i), ad, x, y, i)
