"""Workloads of the row-choice operators: the low-rank adapters, the packed
experts and the sampled token of every row of a served batch.

`listed()` names fixed cases, `draw(rng)` gives more of the same ranges,
`prepare` makes a case's inputs on the GPU, `run` makes one pass (`own` False:
elementary torch operations; True: this repository's kernels), `work` counts
what a pass cannot do without and `exact` gives its results in 64 bits.

Packed weights are made in the device layout of include/magnetar_b200.h, the
form in which a program holds them between calls.
"""

from __future__ import annotations

import math
import pathlib
import sys

import torch

own = False

Q8_0, Q4_K, Q6_K, IQ4_NL, Q5_K, Q4_0 = 0, 1, 2, 5, 12, 13
FORMAT = {"q8_0": Q8_0, "q4_k": Q4_K, "q6_k": Q6_K, "iq4_nl": IQ4_NL, "q5_k": Q5_K, "q4_0": Q4_0}
# values per block and device-layout bytes of a block's quants and of its scale header
BLOCK = {Q8_0: (32, 32, 2), Q4_K: (256, 128, 16), Q6_K: (256, 192, 32), IQ4_NL: (32, 16, 2),
         Q5_K: (256, 128, 48), Q4_0: (32, 16, 2)}
CODEBOOK = [-127, -104, -83, -65, -49, -35, -22, -10, 1, 13, 25, 38, 53, 69, 89, 113]
DTYPE = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


# ---- cases ----------------------------------------------------------------------------


def listed():
    return [
        # one request decoding one token through its adapter on a square projection
        dict(name="adapters one token", op="adapters", m=1, k=4096, n=4096, rank=16, count=8,
             dtype="bf16", none=0.0, prompts=0),
        # a decode batch in which nearly every request brings its own adapter
        dict(name="adapters decode 64", op="adapters", m=64, k=4096, n=14336, rank=16, count=64,
             dtype="f16", none=0.1, prompts=0),
        # ragged sizes throughout, f32 factors, half of the rows without an adapter
        dict(name="adapters ragged f32", op="adapters", m=37, k=1345, n=1003, rank=11, count=5,
             dtype="f32", none=0.5, prompts=0),
        # prefill of six prompts of unequal length, each under one adapter
        dict(name="adapters prefill 2048", op="adapters", m=2048, k=4096, n=14336, rank=64, count=8,
             dtype="bf16", none=0.1, prompts=6),
        # one token through many small experts
        dict(name="experts one token small", op="experts", m=1, hidden=2048, ffn=768, experts=64,
             top_k=8, gate_up_format="q4_k", down_format="q4_k", normalize=True),
        # one token through two of eight wide experts, the down projection in a wider format
        dict(name="experts one token wide", op="experts", m=1, hidden=4096, ffn=14336, experts=8,
             top_k=2, gate_up_format="q4_k", down_format="q6_k", normalize=True),
        # a handful of tokens, sizes that are whole 32-value blocks but not whole 256s
        dict(name="experts ragged", op="experts", m=5, hidden=1440, ffn=992, experts=20, top_k=3,
             gate_up_format="iq4_nl", down_format="q8_0", normalize=False),
        # a small decode batch over many experts: most of them are chosen by a token or two
        dict(name="experts decode 16", op="experts", m=16, hidden=4096, ffn=1536, experts=64,
             top_k=8, gate_up_format="q8_0", down_format="q8_0", normalize=False),
        # a decode batch over eight wide experts: each serves about sixteen tokens
        dict(name="experts decode 64", op="experts", m=64, hidden=4096, ffn=14336, experts=8,
             top_k=2, gate_up_format="q4_k", down_format="q5_k", normalize=True),
        # one request, the usual settings
        dict(name="sample one row", op="sample", rows=1, vocab=32000, kind="usual"),
        # odd vocabulary, part of it masked, ties at the borders, min-p instead of top-p
        dict(name="sample ragged masked", op="sample", rows=7, vocab=50257, kind="masked"),
        # a decode batch in which every row has settings of its own
        dict(name="sample batch mixed", op="sample", rows=256, vocab=128256, kind="mixed"),
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["adapters", "experts", "sample"])
    if op == "adapters":
        step = rng.choice([1, 8, 64])  # odd sizes, whole 16-byte runs, whole tiles
        k = max(step, _log(rng, 64, 8192) // step * step)
        n = max(step, _log(rng, 64, 14336) // step * step)
        rank = _log(rng, 1, 128) if step == 1 else rng.choice([4, 8, 16, 24, 32, 64, 128])
        count = _log(rng, 1, 64)
        m = _log(rng, 1, 2048)
        # no dearer than the largest listed case, in its plain form either
        m = max(1, min(m, 2048 * 18432 // (k + n), 2048 * 512 * 18432 // (count * rank * (k + n))))
        return dict(op=op, m=m, k=k, n=n, rank=rank, count=count,
                    dtype=rng.choice(["f32", "f16", "bf16"]), none=rng.choice([0.0, 0.1, 0.5]),
                    prompts=rng.choice([0, 0, 3]) if m >= 8 else 0)
    if op == "experts":
        gate_up = rng.choice(["q4_k", "q4_k", "q5_k", "q6_k", "q8_0", "iq4_nl", "q4_0"])
        down = rng.choice([gate_up, "q4_k", "q6_k", "q8_0"])
        hidden = max(1, _log(rng, 512, 4096) // BLOCK[FORMAT[gate_up]][0]) * BLOCK[FORMAT[gate_up]][0]
        ffn = max(1, _log(rng, 256, 14336) // BLOCK[FORMAT[down]][0]) * BLOCK[FORMAT[down]][0]
        most = min(128, 64 * 4096 * 1536 // (hidden * ffn))  # as many weights as a listed case
        experts = _log(rng, min(4, most), most)
        return dict(op=op, m=_log(rng, 1, 64), hidden=hidden, ffn=ffn, experts=experts,
                    top_k=rng.randint(1, min(8, experts)), gate_up_format=gate_up, down_format=down,
                    normalize=rng.random() < 0.5)
    vocab = _log(rng, 1000, 152000)
    rows = max(1, min(_log(rng, 1, 256), 256 * 128256 // vocab))
    return dict(op=op, rows=rows, vocab=vocab, kind=rng.choice(["usual", "masked", "mixed"]))


# ---- inputs ---------------------------------------------------------------------------


def _plane_rows(fmt, rows, cols):
    """(bytes of a row's quants, bytes of a row's scale header)."""
    elems, qs, sc = BLOCK[fmt]
    return cols // elems * qs, cols // elems * sc


def _packed(fmt, rows, cols, g):
    """A packed matrix in the device layout: uniform codes, zero-mean values of
    about 0.02 (1 / sqrt of a few thousand columns)."""
    dev = "cuda"
    elems, qs, sc = BLOCK[fmt]
    qrow, srow = _plane_rows(fmt, rows, cols)
    buf = torch.randint(0, 256, (rows * (qrow + srow),), dtype=torch.uint8, device=dev, generator=g)
    head = buf[rows * qrow:].view(-1, sc)
    # the standard deviation of (scale x code) at d = 1
    unit = {Q8_0: 73.9, IQ4_NL: 69.0, Q4_0: 4.6, Q4_K: 250.0, Q5_K: 490.0, Q6_K: 1366.0}[fmt]
    d = (torch.rand(head.shape[0], device=dev, generator=g) + 0.5) * (0.02 / unit)
    if fmt == Q6_K:
        head[:, 16:18] = d.half().view(torch.uint8).view(-1, 2)
        head[:, 18:] = 0
    elif fmt in (Q4_K, Q5_K):
        # dmin at the middle of the codes, so that values are centred on zero
        head[:, 0:2] = d.half().view(torch.uint8).view(-1, 2)
        head[:, 2:4] = (d * (7.5 if fmt == Q4_K else 15.5)).half().view(torch.uint8).view(-1, 2)
    else:
        head[:, 0:2] = d.half().view(torch.uint8).view(-1, 2)
    return buf


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed))
    s = dict(case)
    randn = lambda *shape: torch.randn(*shape, device="cuda", generator=g)  # noqa: E731
    rand = lambda *shape: torch.rand(*shape, device="cuda", generator=g)  # noqa: E731
    if case["op"] == "adapters":
        m, k, n, rank, count = (case[v] for v in ("m", "k", "n", "rank", "count"))
        dt = DTYPE[case["dtype"]]
        s["x"] = randn(m, k)
        s["base"] = randn(m, n)
        s["a"] = (randn(count, rank, k) / math.sqrt(k)).to(dt)
        s["b"] = (randn(count, n, rank) / math.sqrt(rank)).to(dt)
        s["scales"] = 0.5 + rand(count)
        if case["prompts"]:  # consecutive rows of one prompt share its adapter
            cut = torch.sort(torch.randint(0, m, (case["prompts"] - 1,), device="cuda", generator=g)).values
            prompt = torch.bucketize(torch.arange(m, device="cuda"), cut, right=True)
            chosen = torch.randint(0, count, (case["prompts"],), device="cuda", generator=g)
            chosen = torch.where(rand(case["prompts"]) < case["none"], -1, chosen)
            ids = chosen[prompt]
        else:
            ids = torch.randint(0, count, (m,), device="cuda", generator=g)
            ids = torch.where(rand(m) < case["none"], -1, ids)
        s["ids"] = ids.float()
        s["y"] = torch.empty(m, n, device="cuda")
    elif case["op"] == "experts":
        m, hidden, ffn, experts, top_k = (case[v] for v in ("m", "hidden", "ffn", "experts", "top_k"))
        s["x"] = randn(m, hidden)
        s["router"] = randn(experts, hidden) / math.sqrt(hidden)
        s["gate"] = _packed(FORMAT[case["gate_up_format"]], experts * ffn, hidden, g)
        s["up"] = _packed(FORMAT[case["gate_up_format"]], experts * ffn, hidden, g)
        s["down"] = _packed(FORMAT[case["down_format"]], experts * hidden, ffn, g)
        s["y"] = torch.empty(m, hidden, device="cuda")
        s["ids"] = torch.empty(m, top_k, device="cuda")
        s["weights"] = torch.empty(m, top_k, device="cuda")
    else:
        rows, vocab, kind = case["rows"], case["vocab"], case["kind"]
        # a peaked head over a broad body, spread differently in every row
        logits = randn(rows, vocab) * (1.0 + 2.0 * rand(rows, 1))
        logits += 6.0 * (rand(rows, vocab) < 20.0 / vocab)
        off = torch.zeros(rows, device="cuda")
        s["temperature"] = 0.6 + 0.6 * rand(rows)
        s["top_k"], s["top_p"], s["min_p"] = off + 50, off + 0.95, off.clone()
        if kind == "masked":  # a grammar's mask, logits on a coarse grid (ties), min-p
            logits = (logits * 8).round() / 8
            logits = torch.where(rand(rows, vocab) < 0.4, -math.inf, logits)
            s["top_k"], s["top_p"], s["min_p"] = off.clone(), off + 1.0, 0.02 + 0.1 * rand(rows)
        elif kind == "mixed":
            pick = torch.randint(0, 6, (rows,), device="cuda", generator=g)
            # 0: greedy; 1: usual; 2: nothing cut off; 3: top-p alone; 4: top-k alone, large;
            # 5: all three
            s["temperature"] = torch.where(pick == 0, off, s["temperature"])
            s["top_k"] = torch.where((pick == 2) | (pick == 3), off,
                                     torch.where(pick == 4, off + 1000, s["top_k"]))
            s["top_p"] = torch.where((pick == 2) | (pick == 4), off + 1.0, s["top_p"])
            s["min_p"] = torch.where(pick == 5, off + 0.05, off)
            logits = torch.where((pick >= 4)[:, None], logits.bfloat16().float(), logits)
        s["logits"] = logits
        s["uniform"] = rand(rows)
        s["ids"] = torch.empty(rows, device="cuda")
        s["logprob"] = torch.empty(rows, device="cuda")
        s["kept"] = torch.empty(rows, dtype=torch.int32, device="cuda")
    return s


# ---- one pass -------------------------------------------------------------------------


def run(s):
    if own:
        return {"adapters": _own_adapters, "experts": _own_experts, "sample": _own_sample}[s["op"]](s)
    return {"adapters": _adapters, "experts": _experts, "sample": _sample}[s["op"]](s)


def _adapters(s):
    """Every row against every adapter, the other adapters' products dropped."""
    m, rank, count = s["m"], s["rank"], s["count"]
    h = (s["x"] @ s["a"].float().view(count * rank, -1).t()).view(m, count, rank)
    chosen = s["ids"].long()[:, None] == torch.arange(count, device="cuda")
    h = torch.where(chosen[:, :, None], h * s["scales"][:, None], 0.0)
    b = s["b"].float().permute(0, 2, 1).reshape(count * rank, -1)
    return s["base"] + h.view(m, count * rank) @ b


def _values(fmt, buf, rows, cols):
    """The f32 values of a packed matrix in the device layout."""
    elems, qs, sc = BLOCK[fmt]
    qrow, srow = _plane_rows(fmt, rows, cols)
    quants, head = buf[:rows * qrow], buf[rows * qrow:].view(-1, sc)
    f16 = lambda b: b.contiguous().view(torch.float16).float()  # noqa: E731
    if fmt == Q8_0:
        return (quants.view(torch.int8).view(-1, 32).float() * f16(head)).view(rows, cols)
    if fmt == Q6_K:
        pair = quants.view(-1, 48)  # two runs: 16 nibble bytes each, then 8 bytes of high bits each
        low = torch.stack((pair[:, :32] & 15, pair[:, :32] >> 4), -1).view(-1, 2, 2, 2, 4, 2)
        high = pair[:, 32:].reshape(-1, 2, 2, 1, 4, 1)  # run, half, -, byte
        shift = torch.tensor([[[0, 2]], [[4, 6]]], dtype=torch.uint8, device="cuda")
        code = low + (((high >> shift) & 3) << 4)
        q = code.view(-1, 8, 2, 16).float() - 32.0
        scale = head[:, :16].contiguous().view(torch.int8).float().view(-1, 8, 2, 1)
        return ((f16(head[:, 16:18]).view(-1, 1, 1, 1) * scale) * q).view(rows, cols)
    code = torch.stack((quants & 15, quants >> 4), -1).view(-1, 32)
    if fmt == Q4_0:
        return ((code.float() - 8.0) * f16(head)).view(rows, cols)
    if fmt == IQ4_NL:
        table = torch.tensor(CODEBOOK, dtype=torch.float32, device="cuda")
        return (table[code.int()] * f16(head)).view(rows, cols)
    if fmt == Q5_K:
        # byte j of a run's word: bits 2 w and 2 w + 1 are the fifth bits of values 8 w + 2 j, + 1
        word = head[:, 16:].reshape(-1, 1, 4, 1)
        bit = torch.arange(8, dtype=torch.uint8, device="cuda").view(4, 1, 2)
        code = code + (((word >> bit) & 1) << 4).view(-1, 32)
    # sixteen 6-bit fields: the eight scales, then the eight mins
    three = head[:, 4:16].reshape(-1, 4, 3).int()
    word = three[:, :, 0] | (three[:, :, 1] << 8) | (three[:, :, 2] << 16)
    field = (word[:, :, None] >> torch.tensor([0, 6, 12, 18], device="cuda")) & 63
    field = field.view(-1, 2, 8).float()
    scale = f16(head[:, 0:2]) * field[:, 0]
    least = f16(head[:, 2:4]) * field[:, 1]
    return (code.view(-1, 8, 32).float() * scale[:, :, None] - least[:, :, None]).view(rows, cols)


def _experts(s):
    """Every token through every expert, weighted by its routing (zero where not chosen)."""
    m, hidden, ffn, experts, top_k = (s[v] for v in ("m", "hidden", "ffn", "experts", "top_k"))
    z = s["x"].double() @ s["router"].double().t()
    z, ids = torch.sort(z, dim=1, descending=True, stable=True)
    p = torch.exp(z - z[:, :1])
    total = p[:, :top_k] if s["normalize"] else p
    ids, weights = ids[:, :top_k], (p[:, :top_k] / total.sum(1, keepdim=True)).float()
    share = torch.zeros(m, experts, device="cuda").scatter(1, ids, weights)
    gate = s["x"] @ _values(FORMAT[s["gate_up_format"]], s["gate"], experts * ffn, hidden).t()
    up = s["x"] @ _values(FORMAT[s["gate_up_format"]], s["up"], experts * ffn, hidden).t()
    h = gate / (1 + torch.exp(-gate)) * up
    h = h.view(m, experts, ffn).permute(1, 0, 2)
    down = _values(FORMAT[s["down_format"]], s["down"], experts * hidden, ffn).view(experts, hidden, ffn)
    y = (h @ down.transpose(1, 2)) * share.t()[:, :, None]
    return {"y": y.sum(0), "ids": ids.float(), "weights": weights}


def _sample(s):
    """Sorted probabilities in 64 bits; the draw in token order."""
    logits, vocab = s["logits"].double(), s["vocab"]
    greedy = s["temperature"] <= 0
    t = torch.where(greedy, 1.0, s["temperature"].double())[:, None]
    order = torch.sort(logits, dim=1, descending=True, stable=True)
    z = order.values
    w = torch.exp((z - z[:, :1]) / t)  # relative to the largest
    place = torch.arange(vocab, device="cuda")
    top_k = torch.where(s["top_k"] < 1, float(vocab), s["top_k"].double())
    top_k = torch.where(greedy, 1.0, top_k)[:, None]
    keep = (place < top_k) & (z > -math.inf)
    mass = torch.where(keep, w, 0.0)
    before = torch.cumsum(mass, 1) - mass
    cut = (s["top_p"].double() < 1)[:, None]
    keep &= ~cut | (before < s["top_p"].double()[:, None] * mass.sum(1, keepdim=True))
    keep &= (w >= s["min_p"].double()[:, None]) | (place == 0)
    back = torch.zeros_like(w).scatter(1, order.indices, torch.where(keep, w, 0.0))
    inclusive = torch.cumsum(back, 1)
    total = inclusive[:, -1:]
    token = (inclusive <= s["uniform"].double()[:, None] * total).sum(1)
    logprob = torch.log(back.gather(1, token[:, None]) / total)[:, 0]
    return {"ids": token.float(), "logprob": logprob.float(), "kept": keep.sum(1, dtype=torch.int32)}


def _package():
    here = str(pathlib.Path(__file__).resolve().parents[1] / "magnetar-provider-cpu_b200")
    if here not in sys.path:
        sys.path.insert(0, here)
    import magnetar_b200

    return magnetar_b200


def _own_adapters(s):
    mgb = _package()
    if "handle" not in s:  # described once, as a program does that keeps its adapters resident
        s["handle"] = mgb.adapters(s["a"].data_ptr(), s["b"].data_ptr(), s["count"], s["rank"],
                                   s["k"], s["n"], {"f32": mgb.F32, "f16": mgb.F16, "bf16": mgb.BF16}[s["dtype"]],
                                   s["scales"].data_ptr())
        size = mgb.adapters_workspace_bytes(s["handle"], s["m"])
        s["workspace"] = torch.empty(max(1, size), dtype=torch.uint8, device="cuda")
    mgb.adapters_add(s["handle"], s["ids"].data_ptr(), s["x"].data_ptr(), s["m"], s["y"].data_ptr(),
                     base_ptr=s["base"].data_ptr(), workspace_ptr=s["workspace"].data_ptr(),
                     workspace_bytes=s["workspace"].numel(),
                     stream=torch.cuda.current_stream().cuda_stream)
    return s["y"]


def _own_experts(s):
    mgb = _package()
    if "handle" not in s:
        s["handle"] = mgb.experts(FORMAT[s["gate_up_format"]], s["gate"].data_ptr(), s["up"].data_ptr(),
                                  FORMAT[s["down_format"]], s["down"].data_ptr(), s["experts"],
                                  s["hidden"], s["ffn"])
        size = mgb.moe_workspace_bytes(s["handle"], s["m"], s["top_k"])
        s["workspace"] = torch.empty(size, dtype=torch.uint8, device="cuda")
    mgb.moe_layer(s["handle"], s["router"].data_ptr(), s["x"].data_ptr(), s["m"], s["top_k"],
                  s["normalize"], s["y"].data_ptr(), ids_ptr=s["ids"].data_ptr(),
                  weights_ptr=s["weights"].data_ptr(), workspace_ptr=s["workspace"].data_ptr(),
                  workspace_bytes=s["workspace"].numel(),
                  stream=torch.cuda.current_stream().cuda_stream)
    return {"y": s["y"], "ids": s["ids"], "weights": s["weights"]}


def _own_sample(s):
    mgb = _package()
    if "workspace" not in s:
        size = mgb.sample_workspace_bytes(s["rows"], s["vocab"])
        s["workspace"] = torch.empty(max(1, size), dtype=torch.uint8, device="cuda")
    mgb.sample(s["logits"].data_ptr(), s["rows"], s["vocab"], s["ids"].data_ptr(),
               temperature_ptr=s["temperature"].data_ptr(), top_k_ptr=s["top_k"].data_ptr(),
               top_p_ptr=s["top_p"].data_ptr(), min_p_ptr=s["min_p"].data_ptr(),
               uniform_ptr=s["uniform"].data_ptr(), logprob_ptr=s["logprob"].data_ptr(),
               kept_ptr=s["kept"].data_ptr(), workspace_ptr=s["workspace"].data_ptr(),
               workspace_bytes=s["workspace"].numel(),
               stream=torch.cuda.current_stream().cuda_stream)
    return {"ids": s["ids"], "logprob": s["logprob"], "kept": s["kept"]}


# ---- what a pass cannot do without --------------------------------------------------------


def _expected_distinct(choices, of):
    """The expected number of different values among `choices` uniform draws."""
    return of * (1.0 - (1.0 - 1.0 / of) ** choices)


def work(case):
    if case["op"] == "adapters":
        m, k, n, rank, count = (case[v] for v in ("m", "k", "n", "rank", "count"))
        size = 4 if case["dtype"] == "f32" else 2
        rows = m * (1 - case["none"])
        used = _expected_distinct(max(1, (case["prompts"] or m) * (1 - case["none"])), count)
        return {"bytes": 4 * (rows * k + 2 * m * n) + used * rank * (k + n) * size + 4 * m,
                "flops": 2 * rows * rank * (k + n)}
    if case["op"] == "experts":
        m, hidden, ffn, experts, top_k = (case[v] for v in ("m", "hidden", "ffn", "experts", "top_k"))
        used = experts * (1.0 - (1.0 - top_k / experts) ** m)
        row = lambda fmt, cols: sum(_plane_rows(FORMAT[fmt], 1, cols))  # noqa: E731
        weights = used * (2 * ffn * row(case["gate_up_format"], hidden) + hidden * row(case["down_format"], ffn))
        return {"bytes": weights + 4 * (experts * hidden + 2 * m * hidden + 2 * m * top_k),
                "flops": 2 * m * (experts * hidden + 3 * top_k * hidden * ffn)}
    rows, vocab = case["rows"], case["vocab"]
    return {"bytes": 4 * rows * vocab + 32 * rows, "flops": 3 * rows * vocab}


# ---- the same in 64 bits, from the definitions ------------------------------------------------


def exact(case, seed):
    s = prepare(case, seed)
    return {"adapters": _exact_adapters, "experts": _exact_experts, "sample": _exact_sample}[case["op"]](s)


def _exact_adapters(s):
    y = s["base"].double()
    x = s["x"].double()
    for a in range(s["count"]):
        rows = (s["ids"] == a).nonzero()[:, 0]
        if rows.numel():
            delta = (x[rows] @ s["a"][a].double().t()) @ s["b"][a].double().t()
            y[rows] += delta * s["scales"][a].double()
    return y


def _exact_matrix(fmt, buf, rows, cols, first, count):
    """Stored rows first .. first + count in 64 bits, value by value index."""
    elems, qs, sc = BLOCK[fmt]
    qrow, srow = _plane_rows(fmt, rows, cols)
    q = buf[:rows * qrow].view(rows, qrow)[first:first + count].int()
    h = buf[rows * qrow:].view(rows, -1, sc)[first:first + count].int()
    at = torch.arange(cols, device="cuda")
    run, i = at // 32, at % 32
    half = lambda b: (b[..., 0] | (b[..., 1] << 8)).short().view(torch.float16).double()  # noqa: E731
    if fmt == Q8_0:
        code = q[:, at]
        return torch.where(code > 127, code - 256, code).double() * half(h)[:, run]
    if fmt == Q6_K:
        low = (q[:, run // 2 * 48 + run % 2 * 16 + i // 2] >> (4 * (i % 2))) & 15
        high = q[:, run // 2 * 48 + 32 + run % 2 * 8 + i // 16 * 4 + (i % 8) // 2]
        code = low + 16 * ((high >> (4 * ((i // 8) % 2) + 2 * (i % 2))) & 3)
        scale = h[:, at // 256, 2 * (run % 8) + i // 16]
        scale = torch.where(scale > 127, scale - 256, scale)
        return half(h[..., 16:18])[:, at // 256] * (scale * (code - 32)).double()
    code = (q[:, at // 2] >> (4 * (at % 2))) & 15
    if fmt == Q4_0:
        return (code - 8).double() * half(h)[:, run]
    if fmt == IQ4_NL:
        return torch.tensor(CODEBOOK, device="cuda").double()[code] * half(h)[:, run]
    if fmt == Q5_K:
        byte = h[:, at // 256, 16 + 4 * (run % 8) + (i % 8) // 2]
        code = code + 16 * ((byte >> (2 * (i // 8) + i % 2)) & 1)
    bits = h[:, :, 4:16].long()

    def field(j):  # the j-th 6-bit field of the 96 bits
        b = 6 * j
        two = bits[:, at // 256, b // 8] | (bits[:, at // 256, torch.clamp(b // 8 + 1, max=11)] << 8)
        return (two >> (b % 8)) & 63

    scale, least = field(run % 8), field(8 + run % 8)
    return half(h[..., 0:2])[:, at // 256] * (scale * code).double() - \
        half(h[..., 2:4])[:, at // 256] * least.double()


def _exact_experts(s):
    m, hidden, ffn, experts, top_k = (s[v] for v in ("m", "hidden", "ffn", "experts", "top_k"))
    x = s["x"].double()
    z = torch.einsum("mk,ek->me", x, s["router"].double())
    p = torch.softmax(z, 1)
    ids = torch.argsort(-z, dim=1, stable=True)[:, :top_k]
    weights = p.gather(1, ids)
    if s["normalize"]:
        weights = weights / weights.sum(1, keepdim=True)
    y = torch.zeros(m, hidden, dtype=torch.float64, device="cuda")
    gate_up, down = FORMAT[s["gate_up_format"]], FORMAT[s["down_format"]]
    part = 1024  # stored rows at a time
    for e in torch.unique(ids).tolist():
        token, slot = (ids == e).nonzero(as_tuple=True)
        h = []
        for f in range(0, ffn, part):
            c = min(part, ffn - f)
            gate = x[token] @ _exact_matrix(gate_up, s["gate"], experts * ffn, hidden, e * ffn + f, c).t()
            up = x[token] @ _exact_matrix(gate_up, s["up"], experts * ffn, hidden, e * ffn + f, c).t()
            h.append(gate * torch.sigmoid(gate) * up)
        h = torch.cat(h, 1)
        out = [h @ _exact_matrix(down, s["down"], experts * hidden, ffn, e * hidden + f,
                                 min(part, hidden - f)).t() for f in range(0, hidden, part)]
        y.index_add_(0, token, torch.cat(out, 1) * weights[token, slot][:, None])
    return {"y": y, "ids": ids.double(), "weights": weights}


def _exact_sample(s):
    """Row by row: the kept set by counting down the sorted tokens, the draw by index."""
    out = []
    for r in range(s["rows"]):
        z = s["logits"][r].double()
        if s["temperature"][r] <= 0:
            out.append((int(torch.argmax(z)), 0.0, 1))
            continue
        p = torch.softmax(z / s["temperature"][r].double(), 0)
        order = torch.argsort(-z, stable=True)
        order = order[: int((z > -math.inf).sum())]
        if s["top_k"][r] >= 1:
            order = order[: int(s["top_k"][r])]
        if s["top_p"][r] < 1:
            share = torch.cumsum(p[order], 0) / p[order].sum()
            order = order[: 1 + int((share < s["top_p"][r].double()).sum())]
        if s["min_p"][r] > 0:
            order = order[p[order] / p[order[0]] >= s["min_p"][r].double()]
        kept = torch.sort(order).values
        share = torch.cumsum(p[kept], 0)
        at = int((share <= s["uniform"][r].double() * share[-1]).sum())
        out.append((int(kept[at]), float(torch.log(p[kept[at]] / share[-1])), int(order.numel())))
    ids, logprob, kept = zip(*out)
    return {"ids": torch.tensor(ids, dtype=torch.float64),
            "logprob": torch.tensor(logprob, dtype=torch.float64),
            "kept": torch.tensor(kept, dtype=torch.int32)}
