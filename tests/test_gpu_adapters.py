"""Low-rank adapters (`mgb_adapters_add`, `mgb_qmatmul_adapters`) against the
formula in 64 bits.

Tolerance.  An output is base + s * sum_r b_r h_r with h_r = sum_j a_j x_j.  The
kernels accumulate in f32 from operands of at least 22 bits, so every product
is off by at most 2^-21 of itself and every addition by 2^-24 of the running
sum.  With the magnitudes M = s * sum_r |b_r| sum_j |a_j x_j| an output is off
by at most (2^-21 + (k + rank) 2^-24) M + 2 * 2^-24 (|base| + |y|) (each term
rounded at every later addition); over a whole array the roundings are
independent, so the 2-norm of the difference stays below 2^-19 of the result's.
"""

from __future__ import annotations

import numpy as np
import pytest

import magnetar_b200 as mgb
import synthetic

pytestmark = pytest.mark.gpu

INF = float("inf")
DTYPES = {"f32": mgb.F32, "f16": mgb.F16, "bf16": mgb.BF16}


@pytest.fixture(scope="module")
def torch_cuda(cuda_device):
    import torch

    torch.cuda.set_device(cuda_device)
    return torch


def _torch_dtype(torch, dtype):
    return {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}[dtype]


def _inputs(torch, m, k, n, rank, count, dtype, seed=1):
    g = torch.Generator().manual_seed(seed)
    dt = _torch_dtype(torch, dtype)
    a = (torch.randn(count, rank, k, generator=g) / k ** 0.5).to(dt)
    b = (torch.randn(count, n, rank, generator=g) / rank ** 0.5).to(dt)
    scales = 0.5 + torch.rand(count, generator=g)
    return (a, b, scales, torch.randn(m, k, generator=g), torch.randn(m, n, generator=g))


def _call(torch, a, b, scales, dtype, ids, x, base, y=None, bad=None, stream=0, ws=None):
    count, rank, k = a.shape
    n, m = b.shape[1], x.shape[0]
    ad = mgb.adapters(a.data_ptr(), b.data_ptr(), count, rank, k, n, DTYPES[dtype],
                      scales.data_ptr() if scales is not None else 0)
    size = mgb.adapters_workspace_bytes(ad, m)
    if ws is None:
        ws = torch.full((max(1, size),), 0xFF, dtype=torch.uint8, device="cuda")
    y = torch.full((m, n), float("nan"), device="cuda") if y is None else y
    mgb.adapters_add(ad, ids.data_ptr(), x.data_ptr(), m, y.data_ptr(),
                     base_ptr=base.data_ptr() if base is not None else 0,
                     bad_ptr=bad.data_ptr() if bad is not None else 0,
                     workspace_ptr=ws.data_ptr(), workspace_bytes=size,
                     stream=stream or torch.cuda.current_stream().cuda_stream)
    return y


def _expected(a, b, scales, ids, x, base):
    """(y, magnitudes) in 64 bits."""
    y, mag = base.double().clone(), base.double().abs() * 0
    for row, i in enumerate(ids.tolist()):
        if i < 0:
            continue
        aa, bb = a[int(i)].double(), b[int(i)].double()
        s = float(scales[int(i)])
        y[row] += s * (bb @ (aa @ x[row].double()))
        mag[row] = abs(s) * (bb.abs() @ (aa.abs() @ x[row].double().abs()))
    return y, mag


def _check(got, want, mag, base, k, rank):
    got = got.double().cpu()
    e = 2.0 ** -24
    bound = (8 + k + rank) * e * mag + 2 * e * (base.double().abs() + want.abs())
    worst = ((got - want).abs() / bound.clamp_min(1e-300)).max()
    assert bool(((got - want).abs() <= bound).all()), float(worst)
    assert float((got - want).norm() / want.norm().clamp_min(1e-30)) < 2.0 ** -19


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("m,k,n,rank,count", [
    (1, 1, 1, 1, 1), (1, 64, 64, 8, 2), (1, 4096, 1024, 16, 8), (3, 33, 7, 3, 2),
    (7, 95, 130, 11, 5), (16, 256, 512, 16, 4), (17, 1000, 264, 24, 3), (40, 512, 96, 64, 40),
    (65, 136, 1001, 5, 7), (130, 320, 200, 128, 2), (200, 64, 72, 256, 3)])
def test_matches_the_formula(torch_cuda, dtype, m, k, n, rank, count):
    torch = torch_cuda
    a, b, scales, x, base = _inputs(torch, m, k, n, rank, count, dtype)
    g = torch.Generator().manual_seed(m + k)
    ids = torch.randint(-1, count, (m,), generator=g).float()
    want, mag = _expected(a, b, scales, ids, x, base)
    dev = [t.cuda() for t in (a, b, scales, ids, x, base)]
    y = _call(torch, *dev[:3], dtype, *dev[3:])
    _check(y, want, mag, base, k, rank)
    none = (ids < 0).nonzero()[:, 0]
    assert torch.equal(y.cpu()[none], base[none])  # bit for bit
    # the same call twice: the same bits
    assert torch.equal(_call(torch, *dev[:3], dtype, *dev[3:]), y)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("m", [70, 300, 1500])
@pytest.mark.parametrize("order", ["prompts", "alternating", "one", "none"])
def test_many_rows(torch_cuda, dtype, m, order):
    """Prompts of consecutive rows, rows that take turns, one adapter, none."""
    torch = torch_cuda
    k, n, rank, count = 264, 328, 16, 6
    a, b, scales, x, base = _inputs(torch, m, k, n, rank, count, dtype)
    at = torch.arange(m)
    ids = {"prompts": torch.bucketize(at, torch.tensor([5, 33, m // 2, m - 1])) - 1,
           "alternating": at % (count + 1) - 1, "one": at * 0 + 3, "none": at * 0 - 1}[order].float()
    want, mag = _expected(a, b, scales, ids, x, base)
    dev = [t.cuda() for t in (a, b, scales, ids, x, base)]
    y = _call(torch, *dev[:3], dtype, *dev[3:])
    _check(y, want, mag, base, k, rank)
    # in place: base is y
    z = dev[5].clone()
    assert torch.equal(_call(torch, *dev[:3], dtype, *dev[3:5], z, y=z), y)


def test_no_base_and_no_scales(torch_cuda):
    torch = torch_cuda
    a, b, _, x, base = _inputs(torch, 9, 128, 64, 8, 3, "bf16")
    ids = torch.tensor([0, 1, 2, -1, 2, 2, 0, -7.5, 1.0])  # any negative id: no adapter
    one = torch.ones(3)
    want, mag = _expected(a, b, one, ids, x, base * 0)
    y = _call(torch, a.cuda(), b.cuda(), None, "bf16", ids.cuda(), x.cuda(), None)
    _check(y, want, mag, base * 0, 128, 8)
    assert bool((y[3] == 0).all()) and bool((y[7] == 0).all())


@pytest.mark.parametrize("m", [9, 150])
def test_invalid_ids_are_reported_and_skipped(torch_cuda, m):
    torch = torch_cuda
    a, b, scales, x, base = _inputs(torch, m, 96, 64, 8, 4, "f32")
    dev = [t.cuda() for t in (a, b, scales)]
    xd, based = x.cuda(), base.cuda()
    bad = torch.zeros(1, dtype=torch.int32, device="cuda")
    for wrong in (4.0, 1e9, 0.5, float("nan"), float("inf")):
        ids = torch.arange(m).float() % 4
        ids[7], ids[5] = wrong, wrong
        y = _call(torch, *dev, "f32", ids.cuda(), xd, based, bad=bad)
        assert int(bad) == 5
        want, mag = _expected(a, b, scales, torch.where(ids == torch.arange(m) % 4, ids, -1.0), x, base)
        _check(y, want, mag, base, 96, 8)
        assert torch.equal(y[5].cpu(), base[5]) and torch.equal(y[7].cpu(), base[7])
    ids = (torch.arange(m).float() % 5 - 1)
    _call(torch, *dev, "f32", ids.cuda(), xd, based, bad=bad)
    assert int(bad) == -1  # 0xFFFFFFFF


def test_nan_stays_in_its_row(torch_cuda):
    """A row's NaN or infinity reaches that row alone, and an unused adapter's none."""
    torch = torch_cuda
    for m in (6, 96):
        a, b, scales, x, base = _inputs(torch, m, 128, 64, 16, 3, "bf16")
        a[2], b[2] = float("nan"), float("inf")
        x[1, 3] = float("nan")
        ids = torch.zeros(m)
        ids[2::2] = 1
        y = _call(torch, *[t.cuda() for t in (a, b, scales)], "bf16", ids.cuda(), x.cuda(), base.cuda()).cpu()
        assert bool(y[1].isnan().all())
        rest = torch.arange(m) != 1
        assert bool(y[rest].isfinite().all())


@pytest.mark.parametrize("offset", [1, 2, 3])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_unaligned_buffers(torch_cuda, dtype, offset):
    """Every buffer starts `offset` elements past an aligned address."""
    torch = torch_cuda
    for m in (5, 90):
        k, n, rank, count = 128, 96, 16, 3
        parts = _inputs(torch, m, k, n, rank, count, dtype)
        ids = torch.arange(m).float() % (count + 1) - 1
        want, mag = _expected(*parts[:3], ids, *parts[3:])

        def off(t):
            buf = torch.empty(t.numel() + offset, dtype=t.dtype, device="cuda")
            buf[offset:] = t.flatten().cuda()
            return buf[offset:].view(t.shape)

        y = off(torch.zeros(m, n))
        _call(torch, *[off(t) for t in parts[:3]], dtype, off(ids), off(parts[3]), off(parts[4]), y=y)
        _check(y, want, mag, parts[4], k, rank)


def test_rows_behind_the_last_are_left(torch_cuda):
    torch = torch_cuda
    for m in (5, 90):
        a, b, scales, x, base = _inputs(torch, m + 3, 128, 72, 8, 3, "f16")
        ids = torch.zeros(m + 3)
        y = torch.full((m + 3, 72), 7.0, device="cuda")
        _call(torch, *[t.cuda() for t in (a, b, scales)], "f16", ids.cuda(), x[:m].cuda(), base.cuda(), y=y)
        assert bool((y[m:] == 7.0).all())


@pytest.mark.parametrize("m", [4, 120])
def test_large_and_small_activations(torch_cuda, m):
    """Rows of very different magnitude (f32's range is kept)."""
    torch = torch_cuda
    a, b, scales, x, base = _inputs(torch, m, 256, 64, 16, 3, "bf16")
    x *= 10.0 ** torch.linspace(-20, 20, m)[:, None]
    ids = torch.arange(m).float() % 3
    want, mag = _expected(a, b, scales, ids, x, base * 0)
    y = _call(torch, *[t.cuda() for t in (a, b, scales)], "bf16", ids.cuda(), x.cuda(), None)
    got = y.double().cpu()
    assert bool(((got - want).abs() <= (8 + 256 + 16) * 2.0 ** -24 * mag + 2.0 ** -23 * want.abs()).all())
    rows = (got - want).norm(dim=1) / want.norm(dim=1)
    assert float(rows.max()) < 2.0 ** -19


@pytest.mark.parametrize("fmt,m,n,k", [(mgb.Q4_K, 1, 96, 512), (mgb.Q4_K, 2, 300, 1024),
                                       (mgb.Q8_0, 5, 64, 96), (mgb.Q6_K, 33, 520, 512),
                                       (mgb.IQ4_NL, 140, 256, 256)])
def test_beside_a_packed_projection(torch_cuda, fmt, m, n, k):
    """The projection's y plus the adapters', bit for bit the two calls; rows
    without an adapter are the projection's."""
    torch = torch_cuda
    stream = torch.cuda.current_stream().cuda_stream
    src = torch.from_numpy(synthetic.packed_weights(fmt, n, k, seed=5)).cuda()
    w = torch.empty(mgb.packed_bytes(fmt, n, k), dtype=torch.uint8, device="cuda")
    mgb.repack(fmt, src.data_ptr(), n, k, w.data_ptr(), stream)
    a, b, scales, x, _ = (t.cuda() for t in _inputs(torch, m, k, n, 16, 4, "bf16"))
    bias = torch.randn(n, device="cuda")
    ids = (torch.arange(m, device="cuda") % 5 - 1).float()
    ad = mgb.adapters(a.data_ptr(), b.data_ptr(), 4, 16, k, n, mgb.BF16, scales.data_ptr())
    size = mgb.qmatmul_adapters_workspace_bytes(fmt, m, n, k, ad)
    ws = torch.empty(max(1, size), dtype=torch.uint8, device="cuda")
    y = torch.full((m, n), float("nan"), device="cuda")
    mgb.qmatmul_adapters(fmt, w.data_ptr(), n, k, x.data_ptr(), m, y.data_ptr(), ad, ids.data_ptr(),
                         addend_ptr=bias.data_ptr(), addend_len=n, workspace_ptr=ws.data_ptr(),
                         workspace_bytes=size, stream=stream)
    plain = torch.full((m, n), float("nan"), device="cuda")
    mgb.qmatmul(fmt, w.data_ptr(), n, k, x.data_ptr(), m, plain.data_ptr(), bias.data_ptr(), n,
                ws.data_ptr(), size, stream)
    torch.cuda.synchronize()
    assert torch.equal(y[ids < 0], plain[ids < 0])
    both = _call(torch, a, b, scales, "bf16", ids, x, plain)
    assert torch.equal(y, both)
    assert m < 2 or not torch.equal(y, plain)
    assert mgb.take_device_error(0) == 0


def test_other_stream_and_graph(torch_cuda):
    """On a side stream, and captured and replayed with new inputs; two graphs
    with a workspace each do not disturb one another."""
    torch = torch_cuda
    for m in (3, 100):
        a, b, scales, x, base = (t.cuda() for t in _inputs(torch, m, 128, 96, 16, 4, "f16"))
        ids = (torch.arange(m, device="cuda") % 5 - 1).float()
        want = _call(torch, a, b, scales, "f16", ids, x, base)
        torch.cuda.synchronize()
        side = torch.cuda.Stream()
        y = torch.empty_like(base)
        with torch.cuda.stream(side):
            _call(torch, a, b, scales, "f16", ids, x, base, y=y, ws=torch.empty(1 << 20, dtype=torch.uint8, device="cuda"))
        side.synchronize()
        assert torch.equal(y, want)
        graphs = []
        for _ in range(2):
            gx, gy = x.clone(), torch.empty_like(base)
            ws = torch.empty(1 << 20, dtype=torch.uint8, device="cuda")
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                _call(torch, a, b, scales, "f16", ids, gx, base, y=gy, ws=ws)
            graphs.append((graph, gx, gy, ws))
        graphs[0][1].mul_(2)
        for graph, *_ in graphs * 3:
            graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(graphs[1][2], want)
        assert torch.equal(graphs[0][2], _call(torch, a, b, scales, "f16", ids, x * 2, base))


@pytest.mark.parametrize("count,m", [(5000, 40), (5000, 600), (3, 5000), (4095, 4500), (9000, 4500),
                                     (5000, 24576), (5000, 24577), (2, 25001)])
def test_more_adapters_and_rows_than_the_sort_holds(torch_cuda, count, m):
    """Adapters whose ids share a bucket of the sort, and more rows than it keeps."""
    torch = torch_cuda
    k, n, rank = 40, 36, 4
    a, b, scales, x, base = _inputs(torch, m, k, n, rank, count, "f16")
    g = torch.Generator().manual_seed(4)
    ids = torch.randint(-1, count, (m,), generator=g)
    ids[::7] = 1  # one bucket for 1, 4096 and 8191 where there are that many
    ids[1::7] = min(4096, count - 1)
    ids[2::7] = min(8191, count - 1)
    want, mag = _expected(a, b, scales, ids.float(), x, base)
    dev = [t.cuda() for t in (a, b, scales, ids.float(), x, base)]
    y = _call(torch, *dev[:3], "f16", *dev[3:])
    _check(y, want, mag, base, k, rank)
    assert torch.equal(_call(torch, *dev[:3], "f16", *dev[3:]), y)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("m", [1, 4, 5, 40, 200])
@pytest.mark.parametrize("rank", [64, 65, 130, 256])
def test_large_ranks_in_place(torch_cuda, dtype, m, rank):
    """Ranks of one pass and of several, which add up in y, where base is y."""
    torch = torch_cuda
    k, n, count = 136, 72, 2
    a, b, scales, x, base = _inputs(torch, m, k, n, rank, count, dtype)
    ids = (torch.arange(m) % 3 - 1).float() if m > 1 else torch.ones(1)
    want, mag = _expected(a, b, scales, ids, x, base)
    dev = [t.cuda() for t in (a, b, scales, ids, x, base)]
    y = _call(torch, *dev[:3], dtype, *dev[3:5], dev[5], y=dev[5])
    _check(y, want, mag, base, k, rank)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("rank", [1, 3, 8, 16, 24, 40, 64])
@pytest.mark.parametrize("k,n", [(1, 1), (3, 31), (4, 33), (1032, 100), (2200, 72)])
def test_tiles_on_both_sides_of_a_few_rows(torch_cuda, dtype, rank, k, n):
    """One to six rows of an adapter in one call; lengths of one and odd ones."""
    torch = torch_cuda
    count = 6
    ids = torch.tensor([a for a in range(count) for _ in range(a + 1)] + [-1]).float()
    ids = ids[torch.randperm(len(ids), generator=torch.Generator().manual_seed(rank))]
    m = len(ids)
    a, b, scales, x, base = _inputs(torch, m, k, n, rank, count, dtype)
    want, mag = _expected(a, b, scales, ids, x, base)
    dev = [t.cuda() for t in (a, b, scales, ids, x, base)]
    _check(_call(torch, *dev[:3], dtype, *dev[3:]), want, mag, base, k, rank)
    # infinities of a row's own adapter reach that row alone
    x[2, 0] = float("inf")
    got = _call(torch, *dev[:3], dtype, dev[3], x.cuda(), dev[5]).cpu()
    rest = torch.arange(m) != 2
    _check(got[rest].cuda(), want[rest], mag[rest], base[rest], k, rank)
    assert ids[2] < 0 or not bool(got[2].isfinite().any())


@pytest.mark.parametrize("count,rank", [(64, 64), (8, 16), (5000, 16)])
def test_smaller_batches_take_the_largest_ones_workspace(torch_cuda, count, rank):
    """A workspace sized once for the most rows serves every smaller call."""
    torch = torch_cuda
    k, n, most = 4096, 32, 704
    fmt = mgb.Q4_K
    stream = torch.cuda.current_stream().cuda_stream
    g = torch.Generator(device="cuda").manual_seed(count)
    a = torch.randn(count, rank, k, generator=g, device="cuda").to(torch.float16) / 64
    b = torch.randn(count, n, rank, generator=g, device="cuda").to(torch.float16)
    x = torch.randn(most, k, generator=g, device="cuda")
    base = torch.randn(most, n, generator=g, device="cuda")
    ids = (torch.arange(most, device="cuda") % min(count, 7) - 1).float()
    ad = mgb.adapters(a.data_ptr(), b.data_ptr(), count, rank, k, n, mgb.F16)
    src = torch.from_numpy(synthetic.packed_weights(fmt, n, k, seed=5)).cuda()
    w = torch.empty(mgb.packed_bytes(fmt, n, k), dtype=torch.uint8, device="cuda")
    mgb.repack(fmt, src.data_ptr(), n, k, w.data_ptr(), stream)
    for call, need in ((mgb.adapters_add, mgb.adapters_workspace_bytes(ad, most)),
                       (mgb.qmatmul_adapters, mgb.qmatmul_adapters_workspace_bytes(fmt, most, n, k, ad))):
        ws = torch.empty(need, dtype=torch.uint8, device="cuda")
        for m in (0, 1, 128, 129, 147, 148, 300, 575, 576, 703, most):
            y = torch.full((most, n), 7.0, device="cuda")
            if call is mgb.adapters_add:
                call(ad, ids.data_ptr(), x.data_ptr(), m, y.data_ptr(), base_ptr=base.data_ptr(),
                     workspace_ptr=ws.data_ptr(), workspace_bytes=need, stream=stream)
                own = _call(torch, a, b, None, "f16", ids[:m], x[:m], base[:m]) if m else y[:0]
                assert torch.equal(y[:m], own)
            else:
                call(fmt, w.data_ptr(), n, k, x.data_ptr(), m, y.data_ptr(), ad, ids.data_ptr(),
                     workspace_ptr=ws.data_ptr(), workspace_bytes=need, stream=stream)
                torch.cuda.synchronize()
                assert bool(y[:m].isfinite().all())
            assert bool((y[m:] == 7.0).all())


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("count,per", [(4, 1), (2, 4), (2, 5), (3, 40), (8, 20)])
@pytest.mark.parametrize("rank", [3, 16, 24, 72])
@pytest.mark.parametrize("k", [37, 40])
def test_infinite_and_largest_activations(torch_cuda, dtype, count, per, rank, k):
    """Infinities stay what f32 arithmetic makes of them, and the largest finite values
    stay finite, however many rows share the adapter.  A's first column passes x on to the
    first rank alone, everything else is positive: an infinite x among values of its sign
    makes every output infinite."""
    torch = torch_cuda
    n, m = 70, count * per
    g = torch.Generator().manual_seed(rank + k)
    dt = _torch_dtype(torch, dtype)
    a = (0.5 + 0.5 * torch.rand(count, rank, k, generator=g)).to(dt)
    a[:, :, 0] = 0
    a[:, 0, 0] = 1
    b = (0.0625 + 0.0625 * torch.rand(count, n, rank, generator=g)).to(dt)
    one = torch.ones(count)
    x = 0.1 + torch.rand(m, k, generator=g)
    base = torch.randn(m, n, generator=g)
    ids = (torch.arange(m) // per).float()
    x[0, 5] = INF
    x[1] *= -1
    x[1, k - 1] = -INF
    big = float(torch.finfo(torch.float32).max)
    x[2], x[3] = 0, 0
    x[2, 0], x[3, 0] = big, -big
    dev = [t.cuda() for t in (a, b, one, ids, x, base)]
    y = _call(torch, *dev[:3], dtype, *dev[3:])
    assert bool((y[0] == INF).all()) and bool((y[1] == -INF).all())
    x[:2] = 0
    want, mag = _expected(a, b, one, ids, x, base)
    _check(y[2:], want[2:], mag[2:], base[2:], k, rank)


@pytest.mark.parametrize("per", [1, 4, 5, 40])
def test_largest_f32_factors(torch_cuda, per):
    """f32 factors next to the type's largest value."""
    torch = torch_cuda
    big = float(torch.finfo(torch.float32).max)
    count, rank, k, n = 4, 8, 40, 36
    m = count * per
    a, b = torch.zeros(count, rank, k), torch.zeros(count, n, rank)
    a[:, 0, 0], a[:, 1, 1] = big, 1.0   # h[0] = big x[0], h[1] = x[1]
    b[:, ::2, 0], b[:, 1::2, 1] = 0.5, -big
    x = torch.zeros(m, k)
    x[:, :2] = 0.25
    ids = (torch.arange(m) % count).float()
    base, one = torch.zeros(m, n), torch.ones(count)
    want, mag = _expected(a, b, one, ids, x, base)
    dev = [t.cuda() for t in (a, b, one, ids, x)]
    _check(_call(torch, *dev[:3], "f32", *dev[3:], None), want, mag, base, k, rank)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("m,k,rank,count", [(64, 4096, 16, 1), (128, 8192, 64, 1), (1000, 8192, 128, 3),
                                            (20000, 4096, 16, 1), (20000, 8192, 64, 4)])
def test_sums_over_long_rows(torch_cuda, dtype, m, k, rank, count):
    """The 2-norm's error of long sums, whose lengths a thread depend on the batch.

    A thread adds at most k / 64 sums of 32 products, each addition off by up to 2^-24 of
    the running sum; those are independent, and running sums grow with the root of their
    number: 0.3 2^-24 (k / 128)^(1/2), 2.4 2^-24 for k = 8,192.  A tensor core's sum is cut at
    each of up to 12 steps, by half of 2^-23 of what it holds: 6 2^-24 within a group of 32
    products, and for h, rank / 8 times 3 of them (in passes of 64: 24), 12 2^-24 in y, two
    thirds of each on average over the growing sum.  In all below 16 2^-24 = 2^-20."""
    torch = torch_cuda
    n = 96
    g = torch.Generator(device="cuda").manual_seed(m + k)
    dt = _torch_dtype(torch, dtype)
    randn = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    a, b = (randn(count, rank, k) / k ** 0.5).to(dt), (randn(count, n, rank) / rank ** 0.5).to(dt)
    x, ids = randn(m, k), (torch.arange(m, device="cuda") % count).float()
    y = _call(torch, a, b, None, dtype, ids, x, None)
    want = torch.empty(m, n, dtype=torch.float64, device="cuda")
    for i in range(count):
        want[ids == i] = (x[ids == i].double() @ a[i].double().T) @ b[i].double().T
    assert float((y - want).norm() / want.norm()) < 2.0 ** -20


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("m", [4, 40, 200])
def test_activations_next_to_the_smallest_values(torch_cuda, dtype, m):
    """Rows of 1e-30 down to subnormal ones.  A term of an operand is a multiple of 2^-136
    (tf32) or 2^-133 (bf16), so x and h are within 2^-133 besides their 22 bits, and every
    sum within f32's own smallest step, 2^-149."""
    torch = torch_cuda
    k, n, rank = 256, 64, 16
    a, b, one, x, _ = _inputs(torch, m, k, n, rank, 1, dtype)
    one[:] = 1
    x *= 10.0 ** torch.linspace(-30, -43, m).double()[:, None]
    x = x.float()
    ids = torch.zeros(m)
    want, mag = _expected(a, b, one, ids, x, torch.zeros(m, n))
    y = _call(torch, *[t.cuda() for t in (a, b, one)], dtype, ids.cuda(), x.cuda(), None)
    step = 2.0 ** -133 * (a[0].double().abs().sum(1) + 1) + k * 2.0 ** -149
    small = b[0].double().abs() @ step + rank * 2.0 ** -149
    assert bool(((y.double().cpu() - want).abs() <= (8 + k + rank) * 2.0 ** -24 * mag + 2.0 ** -23 * want.abs() + small).all())


@pytest.mark.parametrize("m", [1, 5, 150])
@pytest.mark.parametrize("k,n,rank", [(1, 1, 1), (8, 36, 16), (33, 40, 70)])
def test_f32_factors_low_terms_multiply(torch_cuda, m, k, n, rank):
    """v = 1 + 2^-11 - 2^-22 is two terms exactly, and v v ends in the product of the lower
    ones, 2^-22: left out, four times the 2^-24 that a rounded result is off by.  What is
    left here is one cut of a sum just above 1, below 2^-23, and y's rounding."""
    torch = torch_cuda
    v = 1 + 2.0 ** -11 - 2.0 ** -22
    x, ids, one = torch.zeros(m, k), torch.zeros(m), torch.ones(1)
    x[:, 0] = v
    for first, second in ((v, 1.0), (1.0, v)):
        a, b = torch.zeros(1, rank, k), torch.zeros(1, n, rank)
        a[0, 0, 0], b[0, :, 0] = first, second
        y = _call(torch, *[t.cuda() for t in (a, b, one)], "f32", ids.cuda(), x.cuda(), None)
        assert float((y.double() - v * v).abs().max()) <= 3 * 2.0 ** -24
