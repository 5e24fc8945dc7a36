"""Host side of the quantised cache on the CPU: pending arrays that read what
an op is about to write, the error flag that all of a device's caches share."""

from __future__ import annotations

import contextlib
import gc
import threading
import time
from types import SimpleNamespace

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


@pytest.fixture()
def flags(monkeypatch):
    """kv_cache with no flag made yet; tensors lie on the CPU and take a while."""
    from phew_b200 import kv_cache

    made, zeros = [], torch.zeros

    def slow_zeros(*a, device=None, **k):
        time.sleep(0.02)
        made.append(zeros(*a, **k))
        return made[-1]

    events = []
    stream = SimpleNamespace(synchronize=lambda: events.append("synchronised"))
    state = SimpleNamespace(made=made, events=events, capturing=False, get=kv_cache.cache_error_flag, module=kv_cache)
    monkeypatch.setattr(kv_cache, "_error_flags", {})
    monkeypatch.setattr(torch, "zeros", slow_zeros)
    monkeypatch.setattr(torch.cuda, "device", lambda d: contextlib.nullcontext())
    monkeypatch.setattr(torch.cuda, "current_stream", lambda d=None: stream)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: state.capturing)
    return state


def test_threads_share_one_error_flag(flags):
    """A second flag would be freed while a cache still hands its address to kernels."""
    device, got, start = torch.device("cuda", 0), [], threading.Barrier(8)

    def make():
        start.wait()
        got.append(flags.get(device))

    threads = [threading.Thread(target=make) for _ in range(8)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert len(got) == 8 and all(f is got[0] for f in got)
    assert len(flags.made) == 1 and flags.events == ["synchronised"]
    assert flags.module._error_flags == {0: got[0]}
    other = flags.get(torch.device("cuda", 1))
    assert other is not got[0] and flags.get(torch.device("cuda", 1)) is other


def test_no_error_flag_is_made_inside_a_capture(flags):
    flags.capturing = True
    with pytest.raises(RuntimeError, match="inside a capture"):
        flags.get(torch.device("cuda", 0))
    assert not flags.made and not flags.module._error_flags
    flags.capturing = False
    f = flags.get(torch.device("cuda", 0))
    flags.capturing = True
    assert flags.get(torch.device("cuda", 0)) is f
