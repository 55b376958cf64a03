"""The row-choice operators as a served decode step uses them: embedding, a packed
projection with each request's adapter, a mixture-of-experts layer, the packed
vocabulary projection, a sampled token of every row, and that token's embedding in
the next step.

The experts' and the sampler's results are held against their definitions (with the
tolerances of their own tests) at the values that reach them; the chain run eagerly,
captured and replayed, and as two graphs on two streams gives the same bits.
"""

from __future__ import annotations

import pytest

import magnetar_b200 as mgb
import synthetic
from test_gpu_experts import Layer
from test_gpu_sample import _one

pytestmark = pytest.mark.gpu

HIDDEN, FFN, EXPERTS, TOP_K, VOCAB, RANK, ADAPTERS = 512, 256, 8, 2, 4160, 8, 5


@pytest.fixture(scope="module")
def torch_cuda(cuda_device):
    import torch

    torch.cuda.set_device(cuda_device)
    return torch


class Model:
    def __init__(self, torch, oracle):
        self.torch = torch
        g = torch.Generator().manual_seed(21)
        stream = torch.cuda.current_stream().cuda_stream

        def packed(fmt, rows, cols, seed):
            src = torch.from_numpy(synthetic.packed_weights(fmt, rows, cols, seed=seed)).cuda()
            out = torch.empty(mgb.packed_bytes(fmt, rows, cols), dtype=torch.uint8, device="cuda")
            mgb.repack(fmt, src.data_ptr(), rows, cols, out.data_ptr(), stream)
            torch.cuda.synchronize()
            return out

        self.embed = packed(mgb.Q8_0, VOCAB, HIDDEN, 1)
        self.proj = packed(mgb.Q4_K, HIDDEN, HIDDEN, 2)
        self.head = packed(mgb.Q8_0, VOCAB, HIDDEN, 3)
        self.a = (torch.randn(ADAPTERS, RANK, HIDDEN, generator=g) / HIDDEN ** 0.5).bfloat16().cuda()
        self.b = torch.randn(ADAPTERS, HIDDEN, RANK, generator=g).bfloat16().cuda()
        self.adapters = mgb.adapters(self.a.data_ptr(), self.b.data_ptr(), ADAPTERS, RANK, HIDDEN,
                                     HIDDEN, mgb.BF16)
        self.layer = Layer(torch, oracle, mgb.Q4_K, mgb.Q6_K, EXPERTS, HIDDEN, FFN)
        self.router = (torch.randn(EXPERTS, HIDDEN, generator=g) / HIDDEN ** 0.5).cuda()


class State:
    """The buffers of one batch of m requests: tokens in, tokens out, in place."""

    def __init__(self, model, m):
        torch = model.torch
        self.model, self.m = model, m
        g = torch.Generator().manual_seed(m)
        dev = lambda t: t.float().cuda()  # noqa: E731
        self.tokens = dev(torch.randint(0, VOCAB, (m,), generator=g))
        self.start = self.tokens.clone()
        self.which = dev(torch.randint(-1, ADAPTERS, (m,), generator=g))
        at = torch.arange(m)
        self.temperature, self.top_k = dev(0.25 * (at % 4)), dev(torch.tensor([0, 40, 300])[at % 3])
        self.top_p, self.min_p = dev(torch.tensor([1.0, 0.9])[at % 2]), dev(torch.tensor([0, 0.02])[at // 2 % 2])
        self.uniform = torch.rand(m, generator=g).cuda()
        new = lambda *s: torch.full(s, float("nan"), device="cuda")  # noqa: E731
        self.x, self.p, self.y = new(m, HIDDEN), new(m, HIDDEN), new(m, HIDDEN)
        self.logits, self.logprob = new(m, VOCAB), new(m)
        self.ids, self.weights = new(m, TOP_K), new(m, TOP_K)
        self.kept = torch.zeros(m, dtype=torch.int32, device="cuda")
        sizes = (mgb.qmatmul_adapters_workspace_bytes(mgb.Q4_K, m, HIDDEN, HIDDEN, model.adapters),
                 mgb.moe_workspace_bytes(model.layer.ex, m, TOP_K),
                 mgb.qmatmul_workspace_bytes(mgb.Q8_0, m, VOCAB, HIDDEN),
                 mgb.sample_workspace_bytes(m, VOCAB), 1)
        self.ws = torch.full((max(sizes),), 0xFF, dtype=torch.uint8, device="cuda")  # one for all calls

    def step(self):
        M, m, s = self.model, self.m, self.model.torch.cuda.current_stream().cuda_stream
        ws = dict(workspace_ptr=self.ws.data_ptr(), workspace_bytes=self.ws.numel(), stream=s)
        mgb.embedding(mgb.Q8_0, M.embed.data_ptr(), VOCAB, HIDDEN, False, self.tokens.data_ptr(), m,
                      self.x.data_ptr(), scale=0.01, stream=s)
        mgb.qmatmul_adapters(mgb.Q4_K, M.proj.data_ptr(), HIDDEN, HIDDEN, self.x.data_ptr(), m,
                             self.p.data_ptr(), M.adapters, self.which.data_ptr(), **ws)
        mgb.moe_layer(M.layer.ex, M.router.data_ptr(), self.p.data_ptr(), m, TOP_K, True,
                      self.y.data_ptr(), addend_ptr=self.x.data_ptr(), ids_ptr=self.ids.data_ptr(),
                      weights_ptr=self.weights.data_ptr(), **ws)
        mgb.qmatmul(mgb.Q8_0, M.head.data_ptr(), VOCAB, HIDDEN, self.y.data_ptr(), m,
                    self.logits.data_ptr(), **ws)
        mgb.sample(self.logits.data_ptr(), m, VOCAB, self.tokens.data_ptr(),
                   temperature_ptr=self.temperature.data_ptr(), top_k_ptr=self.top_k.data_ptr(),
                   top_p_ptr=self.top_p.data_ptr(), min_p_ptr=self.min_p.data_ptr(),
                   uniform_ptr=self.uniform.data_ptr(), logprob_ptr=self.logprob.data_ptr(),
                   kept_ptr=self.kept.data_ptr(), **ws)

    def results(self):
        return [t.clone() for t in (self.x, self.p, self.y, self.logits, self.tokens, self.logprob, self.kept)]


@pytest.mark.parametrize("m", [1, 7, 33, 100])
def test_decode_steps(torch_cuda, oracle, m):
    torch = torch_cuda
    model = Model(torch, oracle)
    eager = State(model, m)
    trail = []
    for _ in range(3):
        eager.step()
        torch.cuda.synchronize()
        trail.append(eager.results())
        layer = model.layer
        layer.check(eager.y, *layer.expected(eager.p, eager.ids, eager.weights, eager.x))
        z = eager.logits.cpu().numpy()
        for r in range(m):
            token, _, kept, margin = _one(z[r], float(eager.temperature[r]), float(eager.top_k[r]),
                                          float(eager.top_p[r]), float(eager.min_p[r]),
                                          float(eager.uniform[r]))
            assert int(eager.kept[r]) == kept
            assert margin <= 2.0 ** -31 or int(eager.tokens[r]) == token
    assert bool(eager.logits.isfinite().all())
    assert m == 1 or len(set(eager.tokens.tolist())) > 1

    # rows without an adapter are the plain projection's, bit for bit
    plain = torch.empty_like(eager.p)
    mgb.qmatmul(mgb.Q4_K, model.proj.data_ptr(), HIDDEN, HIDDEN, eager.x.data_ptr(), m, plain.data_ptr(),
                workspace_ptr=eager.ws.data_ptr(), workspace_bytes=eager.ws.numel(),
                stream=torch.cuda.current_stream().cuda_stream)
    torch.cuda.synchronize()
    none = eager.which < 0
    assert torch.equal(plain[none], eager.p[none])
    assert bool((plain[~none] != eager.p[~none]).any(dim=1).all())

    # captured once and replayed: the tokens feed the next replay; two at once
    pairs = []
    for _ in range(2):
        state, graph, side = State(model, m), torch.cuda.CUDAGraph(), torch.cuda.Stream()
        state.step()  # (kernels are loaded before the capture)
        torch.cuda.synchronize()
        with torch.cuda.graph(graph):
            state.step()
        state.tokens.copy_(state.start)
        pairs.append((state, graph, side))
    torch.cuda.synchronize()
    for want in trail:
        for state, graph, side in pairs:
            with torch.cuda.stream(side):
                graph.replay()
        torch.cuda.synchronize()
        for state, *_ in pairs:
            for got, w in zip(state.results(), want):
                assert torch.equal(got, w)
    assert mgb.take_device_error(0) == 0


def test_two_host_threads(torch_cuda, oracle):
    """Two threads drive a batch each on streams of their own."""
    torch = torch_cuda
    import threading

    model = Model(torch, oracle)
    want, sizes = [], (5, 40)
    for m in sizes:
        state = State(model, m)
        for _ in range(12):
            state.step()
        torch.cuda.synchronize()
        want.append(state.results())
    states, errors = [State(model, m) for m in sizes], []
    torch.cuda.synchronize()
    start = threading.Barrier(len(states), timeout=60)

    def drive(state):
        try:
            side = torch.cuda.Stream()
            start.wait()
            with torch.cuda.stream(side):
                for _ in range(12):
                    state.step()
            side.synchronize()
        except Exception as e:  # noqa: BLE001
            errors.append(e)

    threads = [threading.Thread(target=drive, args=(s,)) for s in states]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors
    for state, results in zip(states, want):
        for got, w in zip(state.results(), results):
            assert torch.equal(got, w)
    assert mgb.take_device_error(0) == 0
