"""Sampling (`mgb_sample`) against its definition in 64 bits.

Tokens, and how many are kept, are whole numbers and must be equal.  A border
can be missed only where two 64-bit sums are closer than the weights'
resolution (2^-31 relative); the seeded inputs here have no such case (checked
where the margin is computed).  A log-probability is the logarithm of a quotient
of weights that are off by 2^-31, rounded to f32: off by at most 2^-24 of itself
plus 2^-29.
"""

from __future__ import annotations

import math

import numpy as np
import pytest

import magnetar_b200 as mgb

pytestmark = pytest.mark.gpu

INF = float("inf")


@pytest.fixture(scope="module")
def torch_cuda(cuda_device):
    import torch

    torch.cuda.set_device(cuda_device)
    return torch


def _call(torch, logits, temperature=None, top_k=None, top_p=None, min_p=None, uniform=None,
          vocab=None, ws=None, out=None):
    rows, ld = logits.shape
    vocab = vocab or ld
    dev = lambda v: None if v is None else torch.as_tensor(v, dtype=torch.float32).cuda()  # noqa: E731
    p = [dev(v) for v in (temperature, top_k, top_p, min_p, uniform)]
    logits = logits.cuda()
    ids, logprob, kept = out or (torch.full((rows,), 9e9, device="cuda"),
                                 torch.full((rows,), 9e9, device="cuda"),
                                 torch.full((rows,), 99, dtype=torch.int32, device="cuda"))
    size = mgb.sample_workspace_bytes(rows, vocab)
    ws = torch.full((max(1, size),), 0xFF, dtype=torch.uint8, device="cuda") if ws is None else ws
    ptr = lambda t: 0 if t is None else t.data_ptr()  # noqa: E731
    mgb.sample(logits.data_ptr(), rows, vocab, ids.data_ptr(), ld, ptr(p[0]), ptr(p[1]), ptr(p[2]),
               ptr(p[3]), ptr(p[4]), logprob.data_ptr(), kept.data_ptr(), ws.data_ptr(), size,
               torch.cuda.current_stream().cuda_stream)
    torch.cuda.synchronize()
    return ids.cpu().numpy(), logprob.cpu().numpy(), kept.cpu().numpy()


def _one(z, temperature=1.0, top_k=0.0, top_p=1.0, min_p=0.0, u=None):
    """(token, logprob, kept, margin of the draw) of one row, from the definition."""
    z = np.asarray(z, dtype=np.float32).astype(np.float64)
    z = np.where(np.isnan(z), -INF, z)
    order = np.argsort(-z, kind="stable")
    order = order[z[order] > -INF]
    if not len(order):
        return -1, -INF, 0, 1.0
    if u is None or not temperature > 0:
        return int(order[0]), 0.0, 1, 1.0
    top = z[order[0]]
    with np.errstate(all="ignore"):
        w = np.where(z == top, 1.0, np.exp((z - top) / np.float64(np.float32(temperature))))
    w = np.where(z == -INF, 0.0, w)
    if top_k >= 1:
        order = order[: int(min(top_k, 2.0 ** 40))]
    if top_p < 1:
        before = np.cumsum(w[order]) - w[order]
        order = order[: max(1, int((before < np.float64(np.float32(top_p)) * w[order].sum()).sum()))]
    if min_p > 0:
        keep = w[order] >= np.float64(np.float32(min_p))
        keep |= z[order] == top
        order = order[keep]
    kept = np.sort(order)
    c = np.cumsum(w[kept])
    at = int((c <= np.float64(np.float32(u)) * c[-1]).sum())
    margin = np.abs(c / c[-1] - np.float64(np.float32(u))).min()
    return int(kept[at]), math.log(w[kept[at]] / c[-1]), len(kept), margin


def _check(torch, logits, temperature=None, top_k=None, top_p=None, min_p=None, uniform=None,
           vocab=None):
    ids, logprob, kept = _call(torch, logits, temperature, top_k, top_p, min_p, uniform, vocab)
    at = lambda v, r, d: d if v is None else float(v[r])  # noqa: E731
    for r in range(logits.shape[0]):
        token, lp, n, margin = _one(logits[r, :vocab].numpy() if vocab else logits[r].numpy(),
                                    at(temperature, r, 1.0), at(top_k, r, 0.0), at(top_p, r, 1.0),
                                    at(min_p, r, 0.0), at(uniform, r, None))
        assert kept[r] == n, (r, kept[r], n)
        if margin > 2.0 ** -31:
            assert ids[r] == token, (r, ids[r], token)
            # The difference of a Python float and a numpy float32 is rounded to 32 bits: a
            # correct half step of the answer (2.385e-7 at 5.03, where steps are 4.77e-7 and
            # 3.02e-7 is allowed) reads as a whole one.  So in 64 bits, the bound as it was.
            got = float(logprob[r])
            assert lp == got or abs(lp - got) <= 2.0 ** -24 * abs(lp) + 2.0 ** -29
        else:
            assert abs(ids[r] - token) <= logits.shape[1]
    return ids


def _rows(torch, rows, vocab, seed=0, spread=3.0):
    g = torch.Generator().manual_seed(seed + rows + vocab)
    return torch.randn(rows, vocab, generator=g) * spread, torch.rand(rows, generator=g)


VOCABS = [1, 2, 3, 31, 33, 255, 1000, 1025, 4099, 32000, 50257, 128256]


@pytest.mark.parametrize("vocab", VOCABS)
@pytest.mark.parametrize("rows", [1, 5])
def test_greedy(torch_cuda, vocab, rows):
    torch = torch_cuda
    z, u = _rows(torch, rows, vocab)
    assert (_check(torch, z) == z.argmax(1).numpy()).all()
    _check(torch, z, temperature=torch.zeros(rows), uniform=u)
    _check(torch, z.round(), temperature=-torch.ones(rows), uniform=u)  # ties: the lowest index
    _check(torch, z, temperature=torch.full((rows,), float("nan")), uniform=u)


@pytest.mark.parametrize("vocab", VOCABS)
@pytest.mark.parametrize("settings", [
    {}, dict(temperature=0.7), dict(top_k=1), dict(top_k=2), dict(top_k=50, top_p=0.9),
    dict(top_k=1000), dict(top_p=0.5), dict(top_p=0.999), dict(min_p=0.05),
    dict(temperature=1.3, top_k=400, top_p=0.8, min_p=0.02), dict(temperature=5.0)])
def test_settings(torch_cuda, vocab, settings):
    torch = torch_cuda
    rows = 4
    z, u = _rows(torch, rows, vocab)
    kw = {k: torch.full((rows,), float(v)) for k, v in settings.items()}
    _check(torch, z, uniform=u, **kw)


@pytest.mark.parametrize("vocab", [40, 3001, 40000])
@pytest.mark.parametrize("grid", [0.25, 1.0, 8.0])
def test_ties_at_the_borders(torch_cuda, vocab, grid):
    """Logits on a coarse grid: hundreds of equal values at every border."""
    torch = torch_cuda
    rows = 6
    z, u = _rows(torch, rows, vocab, seed=3)
    z = (z / grid).round() * grid
    for kw in (dict(top_k=7), dict(top_k=vocab // 3), dict(top_p=0.3), dict(top_p=0.97),
               dict(top_k=vocab // 2, top_p=0.6), dict(min_p=0.2)):
        _check(torch, z, uniform=u, **{k: torch.full((rows,), float(v)) for k, v in kw.items()})


def test_all_equal(torch_cuda):
    """Every logit the same (0, and the type's lowest value): uniform over what is kept."""
    torch = torch_cuda
    lowest = float(torch.finfo(torch.float32).min)
    for vocab in (1, 10, 5000, 70000):
        for value in (0.0, -0.0, 1e30, lowest):
            z = torch.full((3, vocab), value)
            u = torch.tensor([0.0, 0.37, 0.99999994])
            _check(torch, z, uniform=u)
            _check(torch, z, uniform=u, top_k=torch.full((3,), 3.0))
            _check(torch, z, uniform=u, top_p=torch.full((3,), 0.5))


def test_signed_zeros_are_one_value(torch_cuda):
    torch = torch_cuda
    z = torch.tensor([[-0.0, 0.0, -0.0, 0.0, -1.0]])
    assert _check(torch, z)[0] == 0
    _check(torch, z, top_k=torch.tensor([2.0]), uniform=torch.tensor([0.9]))


@pytest.mark.parametrize("vocab", [64, 50257])
def test_masks(torch_cuda, vocab):
    """-inf, NaN and the type's lowest value among the logits; rows with one
    token left and with none."""
    torch = torch_cuda
    z, u = _rows(torch, 8, vocab, seed=5)
    g = torch.Generator().manual_seed(4)
    z[1] = torch.where(torch.rand(vocab, generator=g) < 0.9, -INF, z[1])
    z[2] = torch.where(torch.rand(vocab, generator=g) < 0.5, float("nan"), z[2])
    z[3] = -INF
    z[4] = float("nan")
    z[5] = -INF
    z[5, vocab - 1] = -100.0
    z[6] = torch.finfo(torch.float32).min
    z[6, 5] = 1.0
    z[7, : vocab // 2] = torch.finfo(torch.float32).min
    for kw in ({}, dict(top_k=40), dict(top_p=0.9), dict(top_k=vocab), dict(min_p=0.1),
               dict(top_k=3, top_p=0.5, min_p=0.01)):
        kw = {k: torch.full((8,), float(v)) for k, v in kw.items()}
        ids = _check(torch, z, uniform=u, **kw)
        assert ids[3] == -1 and ids[4] == -1 and ids[5] == vocab - 1 and ids[6] == 5
    assert _check(torch, z)[3] == -1


def test_infinite_logits_share_everything(torch_cuda):
    torch = torch_cuda
    z, _ = _rows(torch, 3, 100)
    z[:, 17] = z[:, 60] = INF
    u = torch.tensor([0.0, 0.49, 0.51])
    ids, logprob, kept = _call(torch, z, uniform=u, min_p=torch.full((3,), 0.1))
    assert ids.tolist() == [17, 17, 60] and kept.tolist() == [2, 2, 2]
    assert np.allclose(logprob, math.log(0.5), atol=1e-6)
    ids, _, kept = _call(torch, z, uniform=u, top_k=torch.ones(3))
    assert ids.tolist() == [17] * 3 and kept.tolist() == [1] * 3


def test_extreme_parameters(torch_cuda):
    """Every value of every parameter has a meaning; none faults."""
    torch = torch_cuda
    z, u = _rows(torch, 1, 300)
    nan = float("nan")
    for t in (1e-30, 1e-10, 1e-3, 1e3, 1e30):
        _check(torch, z, temperature=[t], uniform=u)
    ids, _, kept = _call(torch, z, temperature=[INF], uniform=[0.5])
    assert kept[0] == 300 and ids[0] == 150  # uniform over the vocabulary
    base = _one(z[0].numpy(), u=float(u[0]))
    for kw in (dict(top_k=[nan]), dict(top_k=[-3.0]), dict(top_k=[0.5]), dict(top_k=[1e30]),
               dict(top_k=[INF]), dict(top_p=[nan]), dict(top_p=[1.0]), dict(top_p=[7.0]),
               dict(min_p=[nan]), dict(min_p=[-1.0])):
        ids, _, kept = _call(torch, z, uniform=u, **kw)
        assert (ids[0], kept[0]) == (base[0], base[2]), kw
    for kw in (dict(top_p=[0.0]), dict(top_p=[-2.0]), dict(top_p=[1e-30]), dict(min_p=[1.0]),
               dict(min_p=[9.0]), dict(top_k=[1.9])):
        ids, logprob, kept = _call(torch, z, uniform=u, **kw)
        assert kept[0] == 1 and ids[0] == int(z.argmax()) and logprob[0] == 0.0, kw
    first = _one(z[0].numpy(), u=0.0)[0]
    for v in (0.0, -1.0, nan, -INF):
        assert _call(torch, z, uniform=[v])[0][0] == first
    last = _call(torch, z, uniform=[np.float32(1 - 2 ** -24)])[0][0]
    for v in (1.0, 2.0, INF):
        assert _call(torch, z, uniform=[v])[0][0] == last


def test_row_stride_and_absent_outputs(torch_cuda):
    """Rows inside a wider buffer (padding of +inf and NaN is never read), odd
    alignment, and any output left out."""
    torch = torch_cuda
    z, u = _rows(torch, 5, 1003)
    wide = torch.full((5, 1011), INF)
    wide[:, 1003:1006] = float("nan")
    wide[:, :1003] = z
    assert (_check(torch, wide, uniform=u, vocab=1003) == _call(torch, z, uniform=u)[0]).all()
    dev, ud = torch.cat((torch.zeros(1), z.flatten())).cuda(), u.cuda()
    ids, kept = torch.zeros(7, device="cuda"), torch.zeros(5, dtype=torch.int32, device="cuda")
    ws = torch.empty(max(1, mgb.sample_workspace_bytes(5, 1003)), dtype=torch.uint8, device="cuda")
    mgb.sample(dev.data_ptr() + 4, 5, 1003, ids.data_ptr() + 4, uniform_ptr=ud.data_ptr(),
               workspace_ptr=ws.data_ptr(), workspace_bytes=ws.numel(),
               stream=torch.cuda.current_stream().cuda_stream)
    mgb.sample(dev.data_ptr() + 4, 5, 1003, 0, uniform_ptr=ud.data_ptr(), kept_ptr=kept.data_ptr(),
               workspace_ptr=ws.data_ptr(), workspace_bytes=ws.numel(),
               stream=torch.cuda.current_stream().cuda_stream)
    torch.cuda.synchronize()
    assert (ids.cpu().numpy()[1:6] == _call(torch, z, uniform=u)[0]).all()
    assert float(ids[0]) == 0 and float(ids[6]) == 0  # neighbours are left
    assert (kept.cpu() == 1003).all()


@pytest.mark.parametrize("rows", [2, 40, 200, 700])
def test_many_rows_with_settings_of_their_own(torch_cuda, rows):
    torch = torch_cuda
    vocab = 9001
    z, u = _rows(torch, rows, vocab, seed=8)
    g = torch.Generator().manual_seed(rows)
    pick = torch.randint(0, 5, (rows,), generator=g)
    _check(torch, z, temperature=torch.where(pick == 0, 0.0, 0.5 + torch.rand(rows, generator=g)),
           top_k=torch.where(pick == 1, 40.0, 0.0) + torch.where(pick == 4, 3000.0, 0.0),
           top_p=torch.where(pick >= 3, 0.9, 1.0), min_p=torch.where(pick == 2, 0.03, 0.0), uniform=u)


def test_the_largest_vocabulary(torch_cuda):
    torch = torch_cuda
    z, u = _rows(torch, 2, 1 << 20, seed=2)
    _check(torch, z, uniform=u)
    _check(torch, z, uniform=u, top_p=torch.full((2,), 0.9))
    _check(torch, z, uniform=u, top_k=torch.full((2,), 100.0))


def test_frequencies(torch_cuda):
    """20,000 draws of one distribution with equally spaced random numbers: each
    token's count is its probability times 20,000 to within two (every token
    owns one interval of the line, whose ends each add at most one)."""
    torch = torch_cuda
    rows = 20000
    z = torch.randn(1, 50, generator=torch.Generator().manual_seed(1)) * 2
    u = (torch.arange(rows) + 0.5) / rows
    ids = _call(torch, z.expand(rows, 50).contiguous(), temperature=torch.full((rows,), 0.8), uniform=u)[0]
    p = torch.softmax(z[0].double() / 0.800000011920929, 0).numpy()
    count = np.bincount(ids.astype(int), minlength=50)
    assert np.abs(count - p * rows).max() <= 2


def test_streams_and_graph(torch_cuda):
    torch = torch_cuda
    z, u = _rows(torch, 6, 20000)
    want = _call(torch, z, top_p=torch.full((6,), 0.9), uniform=u)
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        got = _call(torch, z, top_p=torch.full((6,), 0.9), uniform=u)
    assert all((a == b).all() for a, b in zip(got, want))
    dz, du, dp = z.cuda(), u.cuda(), torch.full((6,), 0.9).cuda()
    ids = torch.zeros(6, device="cuda")
    ws = torch.empty(max(1, mgb.sample_workspace_bytes(6, 20000)), dtype=torch.uint8, device="cuda")
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        mgb.sample(dz.data_ptr(), 6, 20000, ids.data_ptr(), top_p_ptr=dp.data_ptr(),
                   uniform_ptr=du.data_ptr(), workspace_ptr=ws.data_ptr(), workspace_bytes=ws.numel(),
                   stream=torch.cuda.current_stream().cuda_stream)
    for _ in range(3):
        graph.replay()
    torch.cuda.synchronize()
    assert (ids.cpu().numpy() == want[0]).all()
    du.copy_(1 - u)
    graph.replay()
    torch.cuda.synchronize()
    assert (ids.cpu().numpy() == _call(torch, z, top_p=torch.full((6,), 0.9), uniform=1 - u)[0]).all()


@pytest.mark.parametrize("vocab", [4096, 4099, 70001, 131001])
def test_batches_that_fill_the_device(torch_cuda, vocab):
    """More rows than half the SMs: masks, ties, infinities and settings of all kinds
    in one call, on rows that are not 16-byte aligned too."""
    torch = torch_cuda
    rows = 160
    ld = vocab + 1 if vocab % 2 else vocab + 4
    z, u = _rows(torch, rows, ld, seed=8)
    at = torch.arange(rows)
    z[at % 5 == 1] = (z[at % 5 == 1] * 2).round() / 2
    z[at % 10 == 2, vocab // 3:] = -INF
    z[at % 10 == 7] = torch.finfo(torch.float32).min
    z[7, 3] = 1.0
    z[12] = -INF
    z[17, ::3] = INF
    z[22] = 0.25
    z[27, 1::2] = float("nan")
    z[32, 5:] = -INF
    pick = lambda *v: torch.tensor(v, dtype=torch.float32)[at % len(v)]  # noqa: E731
    _check(torch, z, temperature=pick(1.0, 0.7, 0.0, 2.5, 1.0, 1.0, 0.05),
           top_k=pick(0, 50, 0, 1, 700, 0, 200, 256, 257, 0, 1500), top_p=pick(1.0, 0.95, 0.5),
           min_p=pick(0.0, 0.0, 0.0, 0.1), uniform=u, vocab=vocab)


def test_broad_rows(torch_cuda):
    """High temperatures: every token within a few histogram bins; and the nucleus of
    nearly equal logits."""
    torch = torch_cuda
    for rows, vocab in ((3, 20000), (80, 20000)):
        z, u = _rows(torch, rows, vocab, seed=6)
        for t, p in ((50.0, 0.4), (3e4, 0.9), (1e9, 0.7)):
            _check(torch, z, temperature=torch.full((rows,), t), top_p=torch.full((rows,), p), uniform=u)
        _check(torch, 1.0 + z * 2.0 ** -20, top_p=torch.full((rows,), 0.3), uniform=u)
        _check(torch, z * 1e30, top_p=torch.full((rows,), 0.3), top_k=torch.full((rows,), 900.0), uniform=u)


@pytest.mark.parametrize("rows,vocab", [(2, 393216), (1, 393217), (3, (1 << 20) - 3), (76, 300001)])
def test_vocabularies_past_the_shared_memory(torch_cuda, rows, vocab):
    """The largest rows that are staged, and those that are read again; parts of a row
    above 65,000 tokens."""
    torch = torch_cuda
    z, u = _rows(torch, rows, vocab, seed=3)
    at = torch.arange(rows)
    _check(torch, z, uniform=u, top_p=torch.tensor([0.9, 1.0, 0.3])[at % 3],
           top_k=torch.tensor([0.0, 60.0, 5000.0, 0.0])[at % 4])


@pytest.mark.parametrize("rows,vocab", [(2, 12), (3, 5000), (100, 5000)])
@pytest.mark.parametrize("top_k", [0, 5])
@pytest.mark.parametrize("temperature", [1.0, 0.7])
def test_the_log_probability_of_an_unlikely_token(torch_cuda, rows, vocab, top_k, temperature):
    """A uniform of 0 draws the first token, 25 to 28 nats below the largest: its weight is
    a few units of 2^-43, its log-probability that of its logit.  The kept total is off by
    at most 2^-44 a token and 2^-31 of itself, the answer besides by its own rounding."""
    torch = torch_cuda
    z = torch.full((rows, vocab), -INF if top_k else -60.0 * temperature)
    nats = torch.linspace(25, 28, rows)
    z[:, 0] = -nats * temperature
    z[:, 7] = 0.0
    z[:, 9] = -1.25
    z[:, 3] = -40.0 * temperature
    t = torch.full((rows,), temperature)
    ids, logprob, _ = _call(torch, z, temperature=t, uniform=torch.zeros(rows),
                            top_k=torch.full((rows,), float(top_k)))
    assert (ids == 0).all()
    zd = z.double() / t.double()[:, None]
    want = (zd[:, 0] - torch.logsumexp(zd, 1)).numpy()
    bound = 2.0 ** -24 * np.abs(want) + 2.0 ** -29
    assert (np.abs(logprob.astype(np.float64) - want) <= bound).all()


@pytest.mark.parametrize("rows,vocab", [(1, 12), (3, 5000), (100, 5000)])
@pytest.mark.parametrize("top_k", [0, 9])
def test_small_min_p(torch_cuda, rows, vocab, top_k):
    """Borders below and between the units of 2^-43 in which masses are summed, and next to
    the largest: what is kept is what the definition keeps."""
    torch = torch_cuda
    base = torch.full((rows, vocab), -INF)
    near = float(np.nextafter(np.float32(2.0 ** -10), np.float32(0)))
    for values, min_p, kept in (([-33.0, 0.0, -31.0, -1.0], 1e-14, 3),    # e^-31 = 3.4e-14
                                ([0.0, -28.8, -2.0], 3.2e-13, 2),          # e^-28.8 = 3.11e-13
                                ([0.0, -28.7, -2.0], 3.4e-13, 3),          # e^-28.7 = 3.43e-13
                                ([-80.0, -87.0, 0.0, -90.0], 1e-38, 3),    # e^-87 = 1.6e-38
                                ([2.0 ** -10, near, 0.0], 1.0, 1)):        # 1 - 5.8e-11
        z = base.clone()
        z[:, 2:2 + len(values)] = torch.tensor(values)
        _check(torch, z, uniform=torch.full((rows,), 0.3), min_p=torch.full((rows,), min_p),
               top_k=torch.full((rows,), float(top_k)))
        n = _call(torch, z, uniform=torch.full((rows,), 0.3), min_p=torch.full((rows,), min_p),
                  top_k=torch.full((rows,), float(top_k)))[2]
        assert (n == kept).all(), (values, n)


def test_the_smallest_temperatures(torch_cuda):
    """Temperatures down to the smallest normal number divide logits that are as close."""
    torch = torch_cuda
    for t in (1e-29, 1e-31, 1e-33, 1.2e-38):
        z = torch.tensor([[0.0, -t, -2 * t, -300 * t if t > 1e-36 else -1.0]])
        for kw in ({}, dict(top_p=[0.7]), dict(top_k=[2.0]), dict(top_k=[3.0], top_p=[0.7]), dict(min_p=[0.2])):
            for u in (0.1, 0.8):
                _check(torch, z, temperature=[t], uniform=[u], **kw)
