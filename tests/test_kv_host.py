"""Host side of the quantised cache on the CPU: pending arrays that read what
an op is about to write."""

from __future__ import annotations

import gc

import pytest
import torch


@pytest.fixture()
def core(monkeypatch):
    """mx.core with a materialisation that only records its node."""
    from phew_b200.mx import core as c

    gc.collect()
    order = []

    def fake(node):
        order.append(node)
        object.__setattr__(node, "_mt", torch.zeros(node.shape, dtype=node.dtype.torch))
        object.__setattr__(node, "_op", None)

    monkeypatch.setattr(c, "_materialize", fake)
    c.order = order
    yield c
    del c.order


def _arr(core, shape, dtype=torch.bfloat16):
    return core.array._wrap(torch.ones(shape, dtype=dtype))


def test_pending_readers_are_settled_before_a_write(core):
    cache, other = _arr(core, (4, 8)), _arr(core, (4, 8))
    core.trace_enter()
    try:
        direct = cache * 2.0
        view = cache[1:3] + 1.0                       # the same storage
        reduced = core.sum(cache, axis=-1, keepdims=True)
        nested = direct + other                       # reads it through `direct` alone
        apart = other * 3.0
        core.settle_readers([cache._t])
        assert not direct.pending and not view.pending and not reduced.pending
        assert nested.pending and apart.pending
        assert core._fused_dag(nested)[2][0] is direct   # computed: an input from here on
        core.settle_readers([cache._t])                  # nothing left to do
        assert len(core.order) == 3
        core.settle_readers([other._t[3]])
        assert not nested.pending and not apart.pending
    finally:
        core.trace_exit()


def test_deferred_nodes_are_forgotten_when_they_die(core):
    x = _arr(core, (4, 8))
    core.trace_enter()
    try:
        y = (x * 2.0) + 1.0
        assert len(core._deferred) == 2
        del y
        assert not core._deferred
        core.settle_readers([x._t])
    finally:
        core.trace_exit()
    assert not core.order
