"""Quantised key/value cache where it can go wrong beyond its sizes: calls
inside mx.compile, values of very different magnitude, bad pages, calls in
which nothing is asked."""

from __future__ import annotations

import pytest
import torch

from test_gpu_kv_cache import DTYPES, Plan, ints, rand

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _clean(mx):
    from phew_b200.ops import check_device_errors

    yield
    mx.synchronize()
    check_device_errors()


# --- inside mx.compile ---------------------------------------------------------------


def test_pending_readers_of_the_cache_see_it_before_the_update(mx):
    """Elementwise ops and row sums that were asked for before a write give what they give op by op."""
    x = rand((1, 2, 5, 128), "bfloat16", 1, 3.0)

    def step(cache, table):
        scales = cache.keys[1]
        before = scales * 2.0
        part = cache.values[2][1:] + 1.0
        total = mx.sum(scales * scales, axis=-1, keepdims=True)
        mx.fast.quantized_cache_update(cache, mx.array(x), mx.array(x), [3], block_table=table)
        return before, part, total * 0.5, scales * 2.0

    got = []
    for f in (step, mx.compile(step)):
        plan = Plan(mx, [40])
        got.append([a._t.clone() for a in f(plan.cache, mx.array(plan.table))])
    assert not torch.equal(got[0][0], got[0][3])  # the update changed what is read
    assert all(torch.equal(a, b) for a, b in zip(*got))
