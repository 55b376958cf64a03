"""The packed mixture-of-experts layer (`mgb_moe_route`, `mgb_moe_experts`,
`mgb_moe_layer`) against its formula in 64 bits over the oracle's dequantised
weights.

Tolerance.  h = silu(g) u with g, u sums over `hidden` products and y a sum over
`ffn` (times top_k) products, every operand of at least 22 bits, accumulated in
f32.  Dequantised weights are exact in f32 up to the reference's own two
roundings (scale and min: 2^-23 relative to their larger term), which the
64-bit reference shares because it starts from the oracle's f32 values; the
kernels' integer codes times f32 factors are off by 2^-22 of the term's
magnitude.  silu's slope is at most 1.1, expf adds 2^-22 relative.  All
roundings are independent, so the 2-norm over a row of outputs is off by less
than 2^-18 of the row magnitude, computed as the same formula over absolute
values divided by the square root of the number of terms (random signs).
"""

from __future__ import annotations

import numpy as np
import pytest

import magnetar_b200 as mgb
import synthetic

pytestmark = pytest.mark.gpu

FORMATS = [mgb.Q4_K, mgb.Q5_K, mgb.Q6_K, mgb.Q8_0, mgb.IQ4_NL, mgb.Q4_0]


@pytest.fixture(scope="module")
def torch_cuda(cuda_device):
    import torch

    torch.cuda.set_device(cuda_device)
    return torch


class Layer:
    """Experts of random codes, centred and scaled so that outputs are of order one."""

    def __init__(self, torch, oracle, gate_up, down, experts, hidden, ffn, seed=3):
        self.torch, self.E, self.K, self.F = torch, experts, hidden, ffn
        self.host, dev = [], []
        for i, (fmt, rows, cols) in enumerate(((gate_up, experts * ffn, hidden),
                                               (gate_up, experts * ffn, hidden),
                                               (down, experts * hidden, ffn))):
            data = synthetic.packed_weights(fmt, rows, cols, seed=seed + i)
            block = data.reshape(-1, synthetic.BLOCK[fmt][1])
            unit = {mgb.Q8_0: 73.9, mgb.IQ4_NL: 69.0, mgb.Q4_0: 4.6, mgb.Q4_K: 250.0,
                    mgb.Q5_K: 490.0, mgb.Q6_K: 1366.0}[fmt]
            rng = np.random.default_rng(seed + 10 + i)
            d = rng.uniform(0.5, 1.5, len(block)) / (unit * cols ** 0.5)
            field = lambda v: v.astype(np.float16).view(np.uint8).reshape(-1, 2)  # noqa: E731
            if fmt == mgb.Q6_K:
                block[:, 208:210] = field(d)
            else:
                block[:, 0:2] = field(d)
            if fmt in (mgb.Q4_K, mgb.Q5_K):
                block[:, 2:4] = field(d * (7.5 if fmt == mgb.Q4_K else 15.5))
            self.host.append(torch.from_numpy(np.array(oracle.dequantize(fmt, data, rows, cols))).double())
            src = torch.from_numpy(data).cuda()
            out = torch.empty(mgb.packed_bytes(fmt, rows, cols), dtype=torch.uint8, device="cuda")
            mgb.repack(fmt, src.data_ptr(), rows, cols, out.data_ptr(),
                       torch.cuda.current_stream().cuda_stream)
            torch.cuda.synchronize()
            dev.append(out)
        self.dev = dev
        self.ex = mgb.experts(gate_up, dev[0].data_ptr(), dev[1].data_ptr(), down,
                              dev[2].data_ptr(), experts, hidden, ffn)

    def run(self, x, ids, weights, addend=None, y=None, bad=None, ws=None):
        torch, m, top_k = self.torch, x.shape[0], ids.shape[1]
        size = mgb.moe_workspace_bytes(self.ex, m, top_k)
        if ws is None:
            ws = torch.full((max(1, size),), 0xFF, dtype=torch.uint8, device="cuda")
        y = torch.full((m, self.K), float("nan"), device="cuda") if y is None else y
        mgb.moe_experts(self.ex, x.data_ptr(), m, ids.data_ptr(), weights.data_ptr(), top_k,
                        y.data_ptr(), addend_ptr=addend.data_ptr() if addend is not None else 0,
                        bad_ptr=bad.data_ptr() if bad is not None else 0,
                        workspace_ptr=ws.data_ptr(), workspace_bytes=size,
                        stream=torch.cuda.current_stream().cuda_stream)
        return y

    def expected(self, x, ids, weights, addend=None):
        """(y, row magnitudes) in 64 bits."""
        torch = self.torch
        x, weights = x.double().cpu(), weights.double().cpu()
        gate, up = (t.view(self.E, self.F, self.K) for t in self.host[:2])
        down = self.host[2].view(self.E, self.K, self.F)
        y = torch.zeros(x.shape[0], self.K, dtype=torch.float64)
        mag = torch.zeros(x.shape[0], dtype=torch.float64)
        for t in range(x.shape[0]):
            for j, e in enumerate(ids[t].tolist()):
                if not (0 <= e < self.E and e == int(e)):
                    continue
                e = int(e)
                g, u = gate[e] @ x[t], up[e] @ x[t]
                y[t] += weights[t, j] * (down[e] @ (g * torch.sigmoid(g) * u))
                # spread of the products that make g, u and y
                gs = ((gate[e] * x[t]) ** 2).sum(1).sqrt()
                us = ((up[e] * x[t]) ** 2).sum(1).sqrt()
                hs = gs * us + g.abs() * us + gs * u.abs() + (g * u).abs()
                mag[t] += abs(weights[t, j]) * ((down[e] * hs) ** 2).sum().sqrt()
        if addend is not None:
            y += addend.double().cpu()
            mag += addend.double().cpu().norm(dim=1)
        return y, mag

    def check(self, got, want, mag):
        off = (got.double().cpu() - want).norm(dim=1)
        assert bool(got.isfinite().all())
        assert bool((off <= 2.0 ** -18 * mag + 1e-30).all()), float((off / mag).max())


def _choices(torch, m, experts, top_k, seed=0):
    g = torch.Generator().manual_seed(seed + m)
    ids = torch.stack([torch.randperm(experts, generator=g)[:top_k] for _ in range(m)]).float()
    return ids, 0.1 + torch.rand(m, top_k, generator=g)


def _x(torch, m, k, seed=9):
    return torch.randn(m, k, generator=torch.Generator().manual_seed(seed)).cuda()


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("m", [1, 2, 7, 9, 40])
def test_every_format(torch_cuda, oracle, fmt, m):
    torch = torch_cuda
    layer = Layer(torch, oracle, fmt, fmt, 4, 512, 256)
    ids, weights = _choices(torch, m, 4, 2)
    x = _x(torch, m, 512)
    y = layer.run(x, ids.cuda(), weights.cuda())
    layer.check(y, *layer.expected(x, ids, weights))
    assert torch.equal(layer.run(x, ids.cuda(), weights.cuda()), y)  # deterministic
    assert mgb.take_device_error(0) == 0


@pytest.mark.parametrize("gate_up,down,experts,hidden,ffn,top_k", [
    (mgb.Q4_K, mgb.Q6_K, 8, 1024, 768, 2), (mgb.Q8_0, mgb.IQ4_NL, 5, 96, 32, 3),
    (mgb.IQ4_NL, mgb.Q8_0, 6, 1440, 992, 3), (mgb.Q4_0, mgb.Q4_K, 3, 32, 256, 3),
    (mgb.Q5_K, mgb.Q4_0, 2, 256, 2080, 1), (mgb.Q6_K, mgb.Q8_0, 64, 256, 64, 8),
    (mgb.Q4_K, mgb.Q5_K, 2, 2304, 4352, 2), (mgb.Q8_0, mgb.Q8_0, 1, 32, 32, 1)])
@pytest.mark.parametrize("m", [1, 5, 33])
def test_shapes(torch_cuda, oracle, gate_up, down, experts, hidden, ffn, top_k, m):
    torch = torch_cuda
    layer = Layer(torch, oracle, gate_up, down, experts, hidden, ffn)
    ids, weights = _choices(torch, m, experts, top_k)
    x = _x(torch, m, hidden)
    layer.check(layer.run(x, ids.cuda(), weights.cuda()), *layer.expected(x, ids, weights))


@pytest.mark.parametrize("m", [1, 64, 129, 256])
def test_all_tokens_on_one_expert(torch_cuda, oracle, m):
    torch = torch_cuda
    layer = Layer(torch, oracle, mgb.Q4_K, mgb.Q4_K, 3, 256, 256)
    ids, weights = torch.ones(m, 1), torch.rand(m, 1) + 0.1
    x = _x(torch, m, 256)
    layer.check(layer.run(x, ids.cuda(), weights.cuda()), *layer.expected(x, ids, weights))


def test_unused_repeated_and_invalid_slots(torch_cuda, oracle):
    torch = torch_cuda
    layer = Layer(torch, oracle, mgb.Q8_0, mgb.Q8_0, 4, 64, 96)
    ids = torch.tensor([[0, 0, 0], [-1, 2, -1], [-1, -1, -1], [3, 1, 3], [2, -5, 2.0]])
    weights = torch.rand(5, 3) + 0.1
    weights[1, 0] = weights[2, 1] = float("nan")  # weights of unused slots are not read into y
    x = _x(torch, 5, 64)
    x[2] = float("nan")  # a token that no expert takes
    addend = torch.randn(5, 64).cuda()
    bad = torch.zeros(1, dtype=torch.int32, device="cuda")
    y = layer.run(x, ids.cuda(), weights.cuda(), addend=addend, bad=bad)
    assert int(bad) == -1
    clean = torch.where(ids < 0, 0.0, weights)
    layer.check(y, *layer.expected(x, ids, clean, addend))
    assert torch.equal(y[2], addend[2])
    z = addend.clone()  # the addend may be y
    assert torch.equal(layer.run(x, ids.cuda(), weights.cuda(), addend=z, y=z), y)
    for wrong in (4.0, 1.5, float("nan"), 1e30):
        ids[3, 2] = ids[4, 0] = wrong
        y = layer.run(x, ids.cuda(), weights.cuda(), addend=addend, bad=bad)
        assert int(bad) == 11
        layer.check(y, *layer.expected(x, torch.where(ids == wrong, -1.0, ids) if wrong == wrong
                                       else ids.nan_to_num(-1.0), clean, addend))


def test_nan_stays_in_its_token(torch_cuda, oracle):
    torch = torch_cuda
    layer = Layer(torch, oracle, mgb.Q4_K, mgb.Q4_K, 2, 256, 256)
    x = _x(torch, 6, 256)
    x[4, 7] = float("nan")
    ids, weights = _choices(torch, 6, 2, 2)
    y = layer.run(x, ids.cuda(), weights.cuda())
    assert bool(y[4].isnan().all())
    rest = [0, 1, 2, 3, 5]
    want, mag = layer.expected(torch.where(x.isnan(), 0.0, x), ids, weights)
    layer.check(y[rest], want[rest], mag[rest])


def test_activations_of_any_magnitude(torch_cuda, oracle):
    """Tokens from 1e-6 to 1e6, and values that differ by 2^20 within a token."""
    torch = torch_cuda
    layer = Layer(torch, oracle, mgb.Q4_K, mgb.Q8_0, 2, 256, 256)
    x = _x(torch, 9, 256).cpu() * 10.0 ** torch.linspace(-6, 6, 9)[:, None]
    x[:, ::5] *= 2.0 ** -20
    ids, weights = torch.arange(9)[:, None].float() % 2, torch.rand(9, 1) + 0.5
    y = layer.run(x.cuda(), ids.cuda(), weights.cuda())
    want, mag = layer.expected(x, ids, weights)
    # silu(g) u is about g u / 2 for small g: relative to its own size
    off = (y.double().cpu() - want).norm(dim=1)
    g = layer.host[0].view(2, 256, 256)
    u = layer.host[1].view(2, 256, 256)
    for t in range(9):
        e = int(ids[t, 0])
        gs, us = (((w[e] * x[t].double()) ** 2).sum(1).sqrt() for w in (g, u))
        size = float(weights[t, 0]) * ((layer.host[2].view(2, 256, 256)[e] * gs * us) ** 2).sum().sqrt()
        assert float(off[t]) <= 2.0 ** -18 * float(max(size, want[t].norm())), t


def _route(torch, router, x, top_k, normalize, scale=1.0):
    m, (experts, hidden) = x.shape[0], router.shape
    ids = torch.full((m, top_k), float("nan"), device="cuda")
    weights = torch.full((m, top_k), float("nan"), device="cuda")
    size = mgb.moe_route_workspace_bytes(experts, hidden, m)
    ws = torch.full((max(1, size),), 0xFF, dtype=torch.uint8, device="cuda")
    mgb.moe_route(router.data_ptr(), experts, hidden, x.data_ptr(), m, top_k, normalize,
                  ids.data_ptr(), weights.data_ptr(), scale, ws.data_ptr(), size,
                  torch.cuda.current_stream().cuda_stream)
    return ids.cpu(), weights.cpu()


@pytest.mark.parametrize("experts,hidden,top_k", [(1, 1, 1), (8, 64, 2), (20, 1441, 3),
                                                  (128, 2048, 8), (1024, 96, 32), (60, 4096, 4)])
@pytest.mark.parametrize("m", [1, 6, 64, 256])
@pytest.mark.parametrize("normalize", [False, True])
def test_routing(torch_cuda, experts, hidden, top_k, m, normalize):
    """The 64-bit choice and weights.  A weight is a quotient of exponentials of
    logits that are off by 2^-24 of the sum of their terms' magnitudes, so by
    less than 2^-20 for logits of order one, and is rounded to f32."""
    torch = torch_cuda
    g = torch.Generator().manual_seed(experts + m)
    router = torch.randn(experts, hidden, generator=g) / hidden ** 0.5
    x = torch.randn(m, hidden, generator=g)
    ids, weights = _route(torch, router.cuda(), x.cuda(), top_k, normalize, 1.5)
    z = x.double() @ router.double().t()
    order = torch.sort(z, dim=1, descending=True, stable=True)
    # no choice of these inputs is closer than the logits' error
    gap = order.values[:, :-1] - order.values[:, 1:]
    sure = (gap[:, :top_k] > 1e-6).all(1) if experts > 1 else torch.ones(m, dtype=torch.bool)
    assert float(sure.double().mean()) > 0.9
    assert torch.equal(ids[sure].long(), order.indices[sure, :top_k])
    p = torch.softmax(z, 1).gather(1, ids.long())
    want = 1.5 * (p / p.sum(1, keepdim=True) if normalize else p)
    assert float(((weights.double() - want) / want).abs().max()) < 2.0 ** -18


def test_routing_ties_and_nan(torch_cuda):
    """Equal logits: the lower id first.  A NaN logit sorts last."""
    torch = torch_cuda
    x = torch.ones(3, 4).cuda()
    router = torch.zeros(70, 4)
    router[5], router[66], router[40] = 1.0, 1.0, 2.0
    router[3] = float("nan")
    ids, weights = _route(torch, router.cuda(), x, 5, True)
    assert ids.tolist() == [[40, 5, 66, 0, 1]] * 3
    want = torch.softmax(torch.tensor([8.0, 4, 4, 0, 0]).double(), 0)
    assert float((weights.double() - want).abs().max()) < 2.0 ** -22
    ids, _ = _route(torch, router.cuda(), x * float("nan"), 3, True)
    assert ids.tolist() == [[0, 1, 2]] * 3


@pytest.mark.parametrize("m,top_k,normalize", [(1, 1, True), (1, 4, False), (3, 2, True), (64, 4, True)])
def test_layer_is_its_two_calls(torch_cuda, oracle, m, top_k, normalize):
    torch = torch_cuda
    layer = Layer(torch, oracle, mgb.Q4_K, mgb.Q6_K, 16, 512, 256)
    x = _x(torch, m, 512)
    router = (torch.randn(16, 512) / 512 ** 0.5).cuda()
    addend = torch.randn(m, 512).cuda()
    ids, weights = _route(torch, router, x, top_k, normalize, 2.0)
    two = layer.run(x, ids.cuda(), weights.cuda(), addend=addend)
    size = mgb.moe_workspace_bytes(layer.ex, m, top_k)
    for keep in (False, True):
        ws = torch.full((size,), 0xFF, dtype=torch.uint8, device="cuda")
        y = torch.full((m, 512), float("nan"), device="cuda")
        gi, gw = torch.empty(m, top_k, device="cuda"), torch.empty(m, top_k, device="cuda")
        mgb.moe_layer(layer.ex, router.data_ptr(), x.data_ptr(), m, top_k, normalize, y.data_ptr(),
                      2.0, addend.data_ptr(), gi.data_ptr() if keep else 0,
                      gw.data_ptr() if keep else 0, ws.data_ptr(), size,
                      torch.cuda.current_stream().cuda_stream)
        assert torch.equal(y, two)
        if keep:
            assert torch.equal(gi.cpu(), ids) and torch.equal(gw.cpu(), weights)


def test_rows_behind_the_last_and_streams(torch_cuda, oracle):
    """Rows past m are left; a side stream and a replayed graph give the same bits."""
    torch = torch_cuda
    layer = Layer(torch, oracle, mgb.Q4_K, mgb.Q4_K, 4, 256, 512)
    x = _x(torch, 5, 256)
    ids, weights = (t.cuda() for t in _choices(torch, 5, 4, 2))
    want = layer.run(x, ids, weights)
    y = torch.full((8, 256), 7.0, device="cuda")
    layer.run(x, ids, weights, y=y)
    assert torch.equal(y[:5], want) and bool((y[5:] == 7.0).all())
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        y = layer.run(x, ids, weights)
    side.synchronize()
    assert torch.equal(y, want)
    gx, gy = x.clone(), torch.empty(5, 256, device="cuda")
    gi = ids.clone()
    ws = torch.empty(mgb.moe_workspace_bytes(layer.ex, 5, 2), dtype=torch.uint8, device="cuda")
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        layer.run(gx, gi, weights, y=gy, ws=ws)
    for _ in range(3):
        graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(gy, want)
    gx.mul_(0.5)
    gi.copy_(ids.flip(0))  # other experts on replay
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(gy, layer.run(x * 0.5, ids.flip(0).contiguous(), weights))


def test_the_largest_plan(torch_cuda, oracle):
    """256 tokens, 32 slots each, 1,024 experts."""
    torch = torch_cuda
    layer = Layer(torch, oracle, mgb.Q8_0, mgb.Q4_0, 1024, 64, 32)
    m, top_k = 256, 32
    ids, weights = _choices(torch, m, 1024, top_k)
    x = _x(torch, m, 64)
    y = layer.run(x, ids.cuda(), weights.cuda())
    some = torch.arange(0, m, 37)
    layer.check(y[some.cuda()], *layer.expected(x[some.cuda()], ids[some], weights[some]))
    # all of them on one expert
    ids = torch.full((m, top_k), 1023.0)
    y = layer.run(x, ids.cuda(), weights.cuda())
    layer.check(y[some.cuda()], *layer.expected(x[some.cuda()], ids[some], weights[some]))
    assert mgb.take_device_error(0) == 0


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("m,experts,top_k", [(9, 8, 2), (20, 5, 1), (33, 16, 2), (40, 2, 2), (24, 24, 4)])
def test_passes_of_8_and_of_16(torch_cuda, oracle, fmt, m, experts, top_k):
    """Few and many tokens an expert, on both sides of the passes' sizes."""
    torch = torch_cuda
    layer = Layer(torch, oracle, fmt, fmt, experts, 256, 512)
    ids, weights = _choices(torch, m, experts, top_k)
    ids[: m // 2, 0] = 1  # one expert has more than most
    x = _x(torch, m, 256)
    layer.check(layer.run(x, ids.cuda(), weights.cuda()), *layer.expected(x, ids, weights))
    assert mgb.take_device_error(0) == 0


@pytest.mark.parametrize("experts", [1, 2, 7, 8, 9, 31, 32, 33, 64])
@pytest.mark.parametrize("hidden", [1024, 1056, 4096])
def test_routing_by_several_warps(torch_cuda, experts, hidden):
    """Few experts, whose logits several warps share."""
    torch = torch_cuda
    m, top_k = 3, min(2, experts)
    g = torch.Generator().manual_seed(experts)
    router = torch.randn(experts, hidden, generator=g)
    x = torch.randn(m, hidden, generator=g)
    z = x.double() @ router.double().T
    ids, weights = torch.empty(m, top_k, device="cuda"), torch.empty(m, top_k, device="cuda")
    r, xd = router.cuda(), x.cuda()  # (kept until the call is done)
    mgb.moe_route(r.data_ptr(), experts, hidden, xd.data_ptr(), m, top_k, False,
                  ids.data_ptr(), weights.data_ptr(), stream=torch.cuda.current_stream().cuda_stream)
    torch.cuda.synchronize()
    best = torch.topk(z, top_k)
    assert torch.equal(ids.cpu().long(), best.indices)
    # a logit's f32 chains: at most 2^-20 of the root of the sum of its squares
    off = 2.0 ** -20 * (x.norm(dim=1) * router.norm(dim=1).max()).max().double()
    want = torch.softmax(z, 1).gather(1, best.indices)
    assert bool(((weights.cpu().double() - want).abs() <= 2 * off * want + 1e-7).all())


@pytest.mark.parametrize("experts", [2, 8, 16, 32])
@pytest.mark.parametrize("hidden", [1025, 1281, 2051, 4100, 4103])
@pytest.mark.parametrize("offset", [0, 1])
def test_routing_reads_the_last_columns(torch_cuda, experts, hidden, offset):
    """Widths that several warps cannot share evenly: the choice hangs on the last
    column alone, whose terms lie 16 / experts apart while all others add up to less
    than 0.1.  The router starts `offset` elements past an aligned address.

    A logit is off by at most (hidden / 128 + 8) 2^-24 of the sum of its terms'
    magnitudes, a weight by twice that and its own rounding."""
    torch = torch_cuda
    m, top_k = 3, 2
    g = torch.Generator().manual_seed(experts + hidden)
    router = (torch.rand(experts, hidden, generator=g) - 0.5) * (0.1 / hidden)
    router[:, -1] = torch.randperm(experts, generator=g).float() * (4.0 / experts)
    x = torch.rand(m, hidden, generator=g)
    x[:, -1] = torch.tensor([4.0, -4.0, 2.0])
    z = x.double() @ router.double().T
    terms = (x.double().abs() @ router.double().abs().T).max()
    buf = torch.zeros(router.numel() + offset, device="cuda")
    buf[offset:] = router.flatten().cuda()
    ids, weights = _route(torch, buf[offset:].view(router.shape), x.cuda(), top_k, False)
    best = torch.topk(z, top_k)
    assert torch.equal(ids.long(), best.indices)
    want = torch.softmax(z, 1).gather(1, best.indices)
    off = 2 * (hidden / 128 + 8) * 2.0 ** -24 * float(terms) + 2.0 ** -23
    assert bool(((weights.double() - want).abs() <= off * want).all())


def test_routing_sums_long_rows(torch_cuda):
    """The widest rows: logits of about 2^18 that differ by 4.  Expert 9's terms 1 + 2^-14
    are sums of up to 2^10 that f32 holds exactly; past that every other step of a longer
    f32 chain loses the 2^-14.  Chains of 16 terms stay exact here, and so do their
    64-bit sums: only the weights' own roundings are left."""
    torch = torch_cuda
    experts, hidden = 64, 1 << 18
    router = torch.zeros(experts, hidden)
    router[9] = 1 + 2.0 ** -14  # in all 2^18 + 16
    router[4] = 1.0
    router[4, 77] = 13.0        # 2^18 + 12
    for offset in (0, 1):
        buf = torch.zeros(router.numel() + offset, device="cuda")
        buf[offset:] = router.flatten().cuda()
        ids, weights = _route(torch, buf[offset:].view(router.shape),
                              torch.ones(2, hidden, device="cuda"), 2, True)
        assert ids.tolist() == [[9.0, 4.0]] * 2
        want = torch.softmax(torch.tensor([4.0, 0.0]).double(), 0)
        assert float((weights.double() - want).abs().max()) <= 2.0 ** -24


def test_routing_of_wide_rows_against_64_bits(torch_cuda):
    """2^18 columns: a logit's chains of 16 terms are off by at most 16 2^-24 of their
    terms' magnitudes, and by about 2^-24 of each partial sum (independent roundings): far
    below the margin of 1e-3 that the choices of these inputs have."""
    torch = torch_cuda
    experts, hidden, m, top_k = 40, 1 << 18, 2, 4
    g = torch.Generator().manual_seed(6)
    router = torch.randn(experts, hidden, generator=g) / 256
    x = torch.randn(m, hidden, generator=g)
    z = x.double() @ router.double().T
    order = torch.sort(z, dim=1, descending=True)
    assert float((order.values[:, :top_k] - order.values[:, 1:top_k + 1]).min()) > 1e-3
    ids, weights = _route(torch, router.cuda(), x.cuda(), top_k, False)
    assert torch.equal(ids.long(), order.indices[:, :top_k])
    # 2^18 roundings of partial sums of up to 4 / 256 * 3, each at most 2^-24 of them: their
    # root-sum-square is below 512 * 0.047 * 2^-24 = 1.5e-6; a logit is off by less than six
    # times that, a weight by twice a logit and its own rounding
    want = torch.softmax(z, 1).gather(1, ids.long())
    assert bool(((weights.double() - want).abs() <= (2 * 9e-6 + 2.0 ** -23) * want).all())


@pytest.mark.parametrize("fmt", FORMATS)
def test_infinities_stay_in_their_token(torch_cuda, oracle, fmt):
    """Infinite activations, and finite ones whose h overflows: NaN for that token, and the
    others' results as without it, in passes of 8 and of 16 tokens."""
    torch = torch_cuda
    layer = Layer(torch, oracle, fmt, fmt, 2, 256, 256)
    for m in (6, 40):
        x = _x(torch, m, 256)
        ids, weights = _choices(torch, m, 2, 2)
        clean = layer.run(x, ids.cuda(), weights.cuda())
        x[1, 7], x[3, 200] = float("inf"), float("-inf")
        x[5] *= 1e30
        y = layer.run(x, ids.cuda(), weights.cuda())
        assert bool(y[[1, 3, 5]].isnan().all())
        rest = [t for t in range(m) if t not in (1, 3, 5)]
        assert torch.equal(y[rest], clean[rest])
