"""Argument checks of the row-choice operators (adapters, experts, sampling):
every refusal comes before any device work, so it is the same without a GPU."""

from __future__ import annotations

import pytest

import magnetar_b200 as mgb

FAKE = 1 << 40  # never dereferenced: every case fails validation first
BIG = 1 << 40


def _status(fn, *args):
    s = fn(*args)
    assert s != mgb.OK
    return s, mgb.last_error()


def _adapters(**change):
    d = dict(a_ptr=FAKE, b_ptr=FAKE, count=4, rank=8, k=64, n=96, dtype=mgb.BF16, scales_ptr=0)
    d.update(change)
    return mgb.adapters(**d)


def _add(ad, ids=FAKE, x=FAKE, m=2, base=FAKE, y=FAKE, ws=FAKE, ws_bytes=BIG):
    return _status(mgb.lib().mgb_adapters_add, ad, ids, x, m, base, y, None, ws, ws_bytes, None)


@pytest.mark.parametrize("change,status,words", [
    (dict(dtype=3), mgb.DTYPE_UNSUPPORTED, "dtype 3"),
    (dict(rank=257), mgb.INVALID_ARGUMENT, "rank 257"),
    (dict(rank=0), mgb.INVALID_ARGUMENT, "at least 1"),
    (dict(count=0), mgb.INVALID_ARGUMENT, "at least 1"),
    (dict(k=0), mgb.INVALID_ARGUMENT, "at least 1"),
    (dict(n=0), mgb.INVALID_ARGUMENT, "at least 1"),
    (dict(count=(1 << 24) + 1), mgb.INVALID_ARGUMENT, "too large"),
    (dict(k=1 << 62), mgb.INVALID_ARGUMENT, "too large"),
    (dict(n=(1 << 64) - 1), mgb.INVALID_ARGUMENT, "too large"),
    (dict(a_ptr=0), mgb.INVALID_ARGUMENT, "null"),
    (dict(b_ptr=0), mgb.INVALID_ARGUMENT, "null"),
    (dict(a_ptr=FAKE + 1), mgb.INVALID_ARGUMENT, "aligned"),
    (dict(b_ptr=FAKE + 2, dtype=mgb.F32), mgb.INVALID_ARGUMENT, "aligned"),
    (dict(scales_ptr=FAKE + 2), mgb.INVALID_ARGUMENT, "aligned")])
def test_adapter_descriptors_are_checked(change, status, words):
    got, said = _add(_adapters(**change))
    assert got == status and words in said


def test_adapter_calls_are_checked():
    ad = _adapters()
    need = mgb.adapters_workspace_bytes(ad, 2)
    assert need > 0
    for kw in (dict(ids=None), dict(x=None), dict(y=None)):
        assert _add(ad, **kw)[0] == mgb.INVALID_ARGUMENT
    assert "needs" in _add(ad, ws_bytes=need - 1)[1]
    assert "needs" in _add(ad, ws=None)[1]
    assert "16-byte" in _add(ad, ws=FAKE + 8)[1]
    assert "aligned" in _add(ad, x=FAKE + 2)[1]
    assert "too large" in _add(ad, m=1 << 40)[1]
    assert mgb.lib().mgb_adapters_add(None, FAKE, FAKE, 1, None, FAKE, None, FAKE, BIG, None) == \
        mgb.INVALID_ARGUMENT
    # the size query answers 0 for what the call refuses
    assert mgb.adapters_workspace_bytes(_adapters(rank=300), 2) == 0
    assert mgb.lib().mgb_adapters_workspace_bytes(None, 2) == 0


def test_projection_with_adapters_is_checked():
    ad = _adapters(k=256, n=96)

    def call(fmt=mgb.Q4_K, n=96, k=256, addend=None, addend_len=0, ad=ad):
        return _status(mgb.lib().mgb_qmatmul_adapters, fmt, FAKE, n, k, FAKE, 2, FAKE, addend,
                       addend_len, ad, FAKE, None, FAKE, BIG, None)

    assert "256 inputs and 96 outputs beside" in call(n=128)[1]
    assert "beside a projection" in call(k=512)[1]
    assert call(fmt=3)[0] == mgb.UNSUPPORTED
    assert "addend has 5 values" in call(addend=FAKE, addend_len=5)[1]
    assert call(ad=None)[0] == mgb.INVALID_ARGUMENT
    both = mgb.qmatmul_adapters_workspace_bytes(mgb.Q4_K, 64, 4096, 4096,
                                                _adapters(k=4096, n=4096))
    assert both >= mgb.qmatmul_workspace_bytes(mgb.Q4_K, 64, 4096, 4096)
    assert both >= mgb.adapters_workspace_bytes(_adapters(k=4096, n=4096), 64)


def _experts(**change):
    d = dict(gate_up_fmt=mgb.Q4_K, gate_ptr=FAKE, up_ptr=FAKE, down_fmt=mgb.Q8_0, down_ptr=FAKE,
             count=8, hidden=512, ffn=96)
    d.update(change)
    return mgb.experts(**d)


def _moe(ex, x=FAKE, m=2, ids=FAKE, weights=FAKE, top_k=2, y=FAKE, ws=FAKE, ws_bytes=BIG):
    return _status(mgb.lib().mgb_moe_experts, ex, x, m, ids, weights, top_k, None, y, None, ws,
                   ws_bytes, None)


@pytest.mark.parametrize("change,status,words", [
    (dict(gate_up_fmt=3), mgb.UNSUPPORTED, "format 3"),
    (dict(down_fmt=7), mgb.UNSUPPORTED, "format 7"),
    (dict(hidden=480), mgb.INVALID_ARGUMENT, "480 are not a multiple"),
    (dict(ffn=80), mgb.INVALID_ARGUMENT, "80 are not a multiple"),
    (dict(hidden=0), mgb.INVALID_ARGUMENT, "not a multiple"),
    (dict(ffn=0), mgb.INVALID_ARGUMENT, "not a multiple"),
    (dict(count=0), mgb.INVALID_ARGUMENT, "experts"),
    (dict(count=1025), mgb.INVALID_ARGUMENT, "1025 experts"),
    (dict(hidden=1 << 40), mgb.INVALID_ARGUMENT, "too large"),
    (dict(gate_ptr=0), mgb.INVALID_ARGUMENT, "null"),
    (dict(down_ptr=FAKE + 8), mgb.INVALID_ARGUMENT, "16-byte")])
def test_expert_descriptors_are_checked(change, status, words):
    got, said = _moe(_experts(**change))
    assert got == status and words in said


def test_expert_calls_are_checked():
    ex = _experts()
    need = mgb.moe_workspace_bytes(ex, 2, 2)
    assert need > 0
    for kw in (dict(x=None), dict(ids=None), dict(weights=None), dict(y=None)):
        assert _moe(ex, **kw)[0] == mgb.INVALID_ARGUMENT
    assert "257 tokens" in _moe(ex, m=257)[1]
    assert "top_k 0" in _moe(ex, top_k=0)[1]
    assert "top_k 33" in _moe(ex, top_k=33)[1]
    assert "needs" in _moe(ex, ws_bytes=0)[1]
    assert "16-byte" in _moe(ex, x=FAKE + 4)[1]
    assert mgb.moe_workspace_bytes(ex, 257, 2) == 0
    assert mgb.moe_workspace_bytes(_experts(gate_up_fmt=3), 2, 2) == 0
    layer = mgb.lib().mgb_moe_layer
    assert layer(ex, None, FAKE, 2, 2, 1, 1.0, None, FAKE, None, None, FAKE, BIG, None) == \
        mgb.INVALID_ARGUMENT
    # a choice of more experts than there are
    assert layer(ex, FAKE, FAKE, 2, 9, 1, 1.0, None, FAKE, None, None, FAKE, BIG, None) == \
        mgb.INVALID_ARGUMENT
    assert "expected 1 to 8" in mgb.last_error()
    assert layer(ex, FAKE, FAKE, 2, 2, 1, 1.0, None, FAKE, None, None, FAKE, need - 1, None) == \
        mgb.INVALID_ARGUMENT


def test_routing_calls_are_checked():
    def call(router=FAKE, experts=8, hidden=100, x=FAKE, m=2, top_k=2, ids=FAKE, weights=FAKE):
        return _status(mgb.lib().mgb_moe_route, router, experts, hidden, x, m, top_k, 1, 1.0, ids,
                       weights, FAKE, BIG, None)[1]

    assert "null" in call(router=None) and "null" in call(x=None)
    assert "null" in call(ids=None) and "null" in call(weights=None)
    assert "1025 experts" in call(experts=1025)
    assert "hidden 0" in call(hidden=0)
    assert "257 tokens" in call(m=257)
    assert "top_k 9" in call(top_k=9)
    assert "aligned" in call(x=FAKE + 2)


def test_sampling_calls_are_checked():
    def call(logits=FAKE, rows=2, vocab=100, ld=100, temperature=None, ids=FAKE, ws_bytes=BIG):
        return _status(mgb.lib().mgb_sample, logits, rows, vocab, ld, temperature, None, None, None,
                       None, ids, None, None, FAKE, ws_bytes, None)[1]

    assert "vocabulary of 0" in call(vocab=0)
    assert "vocabulary of 1048577" in call(vocab=(1 << 20) + 1, ld=1 << 21)
    assert "row stride 99" in call(ld=99)
    assert "null" in call(logits=None)
    assert "too many rows" in call(rows=1 << 40)
    assert "too many rows" in call(rows=1 << 30, ld=1 << 60)
    assert "aligned" in call(logits=FAKE + 2)
    assert "aligned" in call(temperature=FAKE + 1)
    assert "aligned" in call(ids=FAKE + 1)
    assert mgb.sample_workspace_bytes(4, 0) == 0


def test_empty_calls_do_nothing():
    """No rows: no pointer is needed and nothing is launched (no GPU is asked for)."""
    lib = mgb.lib()
    assert lib.mgb_sample(None, 0, 100, 100, None, None, None, None, None, None, None, None, None,
                          0, None) == mgb.OK
    assert lib.mgb_adapters_add(_adapters(), None, None, 0, None, None, None, None, 0, None) == mgb.OK
    assert lib.mgb_moe_experts(_experts(), None, 0, None, None, 2, None, None, None, None, 0,
                               None) == mgb.OK
    assert lib.mgb_moe_route(None, 8, 64, None, 0, 2, 1, 1.0, FAKE, FAKE, None, 0, None) == mgb.OK


def test_a_misaligned_report_is_refused():
    ad, ex = _adapters(), _experts()
    assert mgb.lib().mgb_adapters_add(ad, FAKE, FAKE, 1, None, FAKE, FAKE + 2, FAKE, BIG, None) == \
        mgb.INVALID_ARGUMENT
    assert "aligned" in mgb.last_error()
    assert mgb.lib().mgb_moe_experts(ex, FAKE, 1, FAKE, FAKE, 2, None, FAKE, FAKE + 2, FAKE, BIG, None) == \
        mgb.INVALID_ARGUMENT
    assert "aligned" in mgb.last_error()


@pytest.mark.parametrize("count", [1, 8, 64, 4094, 5000])
@pytest.mark.parametrize("rank", [16, 64, 100, 256])
@pytest.mark.parametrize("k", [64, 4096])
def test_a_larger_batch_never_needs_a_smaller_workspace(count, rank, k):
    """A workspace sized once for the most rows serves every smaller call."""
    ad = _adapters(count=count, rank=rank, k=k, n=4096)
    most = 0
    for m in list(range(0, 3000)) + list(range(3000, 40000, 7)) + [1 << 20, 1 << 24]:
        need = mgb.adapters_workspace_bytes(ad, m)
        assert need >= most, m
        most = need


@pytest.mark.parametrize("gate_up,down,experts,hidden,ffn", [
    (mgb.Q4_K, mgb.Q6_K, 8, 4096, 14336), (mgb.Q8_0, mgb.Q8_0, 64, 4096, 1536),
    (mgb.IQ4_NL, mgb.Q8_0, 20, 1440, 992), (mgb.Q5_K, mgb.Q4_0, 1, 256, 256)])
def test_more_tokens_never_need_a_smaller_workspace(gate_up, down, experts, hidden, ffn):
    ex = _experts(gate_up_fmt=gate_up, down_fmt=down, count=experts, hidden=hidden, ffn=ffn)
    size = [[mgb.moe_workspace_bytes(ex, m, top_k) for top_k in range(1, 33)] for m in range(257)]
    assert all(a <= b for row in size for a, b in zip(row, row[1:]))
    assert all(a <= b for row, after in zip(size, size[1:]) for a, b in zip(row, after))
    # routing and sampling take none
    assert mgb.moe_route_workspace_bytes(experts, hidden, 256) == 0
    assert mgb.sample_workspace_bytes(256, 128256) == 0


def test_adapters_refuse_overlapping_buffers():
    ad = _adapters()  # k 64, n 96
    x, y = FAKE, FAKE + 2 * 96 * 4
    for bad in (dict(x=y, y=y), dict(x=y + 4 * 191, y=y), dict(x=y - 4 * 127, y=y),
                dict(x=x - 4096, y=y, base=y + 4), dict(x=x - 4096, y=y, base=y - 4 * 191)):
        assert "overlaps" in _add(ad, **bad)[1]
