"""Quantised key/value cache where it can go wrong beyond its sizes: calls
inside mx.compile and captures, errors by row and group, values of very
different magnitude, bad pages, what is no number, two calls at once."""

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


# --- attention, row by row and group by group -------------------------------------------


def bounds(plan, q, counts, scale, causal, tensor_core=False):
    """(output, bound of its error's norm, what a lost tile of 32 keys would change) in 64 bits, the last two
    per row and group of the head dimension.

    Errors are independent from key to key, so norms add in squares.  With w_j a row's softmax weights, s_j and
    n_j a value's scale and codes, v'_j = s_j (n_j - 8), or s_j n_j where bf16 sums hold bare codes, or the
    values themselves on the tcgen05 path (more than 64 rows):
      * the output rounded once: u |o|, and below 2^-14, where f16's steps stay 2^-24, half a step for each of a
        group's values: 2^-25 sqrt(group)
      * weights times scales rounded by at most h of them (2^-11 as one f16 term, 2^-22 as two): h N,
        N = sqrt(sum w_j^2 |v'_j|^2); 1.5 of it, the most that two keys can give.  On the tcgen05 path weights and
        values, sqrt(2) of it
      * scores off by e: e N.  Products of bare key codes are cut at 2^-14 of the largest query times a code's
        step: 6 sqrt(D / 3) 2^-14 max|q| max s scale at six sigma; of codes less 8, and in f32's sums and
        queries of 22 bits, 2^-19 |q| |k| scale by Cauchy and Schwarz.  On the tcgen05 path a key's values are
        rounded by 2^-11 each: 6 / sqrt(3) 2^-11 sqrt(sum q_d^2 k_d^2) scale at six sigma
      * weights in 32 bits: the largest is 2^-8 or more, and 2^(s - m) below fp32's 2^-126 is zero, so keys of less
        than 2^-118 of the largest weight may count as nothing: sum w_j |v_j| over those
      * f16's smallest steps: 2^-23 of the largest weight times scale, for each key: sqrt(keys) of that
      * 32-bit sums: 2^-21 of the sum of the magnitudes, 2^-19 where bare codes pile up over 32 additions."""
    u = 2.0 ** {"bfloat16": -8, "float16": -11, "float32": -24}[plan.dtype]
    B, H, L, D = q.shape
    G, per = plan.group, H // plan.kv_heads
    ng = D // G
    out = torch.zeros(q.shape, dtype=torch.float64, device="cuda")
    tol = torch.zeros((B, H, L, ng), dtype=torch.float64, device="cuda")
    tile = torch.zeros_like(tol)
    h = 2.0 ** -22 if plan.dtype == "float32" else 2.0 ** -11 * (2 ** 0.5 if tensor_core else 1.0)
    bare = plan.dtype == "bfloat16" and not tensor_core
    for b, n in enumerate(plan.lengths):
        c = L if counts is None else counts[b]
        if n == 0 or c == 0:
            continue
        K, V = plan.values(0, b), plan.values(1, b)
        cols = plan.table[b, : -(-n // plan.page)].long()
        pick = lambda t: t._t[cols].transpose(0, 1).flatten(1, 2)[:, :n].double()  # noqa: E731
        sk, sv, zv = pick(plan.parts(0)[1]).abs(), pick(plan.parts(1)[1]), pick(plan.parts(1)[2])
        for head in range(H):
            k, v, s_v, z_v = K[head // per], V[head // per], sv[head // per], zv[head // per]
            x = q[b, head, :c].double()
            s = (x @ k.T) * scale
            if causal:
                i = torch.arange(c, device="cuda")[:, None]
                s = s.masked_fill(torch.arange(n, device="cuda")[None] > n - c + i, -torch.inf)
            w = torch.where((s > -torch.inf).any(-1, keepdim=True), torch.softmax(s, -1), 0.0)
            o = w @ v
            vg = v.unflatten(-1, (ng, G))
            centre = z_v[..., None] if bare else z_v[..., None] + 8 * s_v[..., None]
            lone = (vg if tensor_core else vg - centre).norm(dim=-1)  # |v'_j| of a group
            N = (w.square() @ lone.square()).sqrt()
            seen = (w > 0).double()
            qk = x.norm(dim=-1, keepdim=True) * (seen * k.norm(dim=-1)).amax(-1, keepdim=True) * abs(scale)
            if plan.dtype == "float32":
                cut = 0.0
            elif tensor_core:
                cut = 2.0 ** -11 * 6 / 3 ** 0.5 * abs(scale) * (seen * (x.square() @ k.square().T)).amax(-1, keepdim=True).sqrt()
            else:
                cut = (6 * (D / 3) ** 0.5 * 2.0 ** -14 * abs(scale) * x.abs().amax(-1, keepdim=True)
                       * (seen * sk[head // per].amax(-1)).amax(-1, keepdim=True))
            e = qk * 2.0 ** -19 + cut
            step = s_v.abs()
            top = torch.stack([(w * step[:, g]).amax(-1) for g in range(ng)], -1)
            piles = w @ (8 * step + (vg.abs().amax(-1) if tensor_core else centre[..., 0].abs()))
            og = o.unflatten(-1, (ng, G)).norm(dim=-1)
            out[b, head, :c] = o
            none = w * (w < 2.0 ** -118 * w.amax(-1, keepdim=True))
            floor = none @ vg.norm(dim=-1) + (2.0 ** -25 * G ** 0.5 if plan.dtype == "float16" else 0.0)
            tol[b, head, :c] = (u * og + floor + (1.5 * h + e) * N + n ** 0.5 * 2.0 ** -23 * 8 * G ** 0.5 * top
                                + 2.0 ** (-19 if bare else -21) * G ** 0.5 * piles)
            lost = w.clone()
            lost[:, max(0, n // 2 - 16) : n // 2 + 16] = 0
            total = lost.sum(-1, keepdim=True)
            lost = lost / torch.where(total > 0, total, 1.0)
            tile[b, head, :c] = (o - lost @ v).unflatten(-1, (ng, G)).norm(dim=-1)
    return out, tol, tile


def groups_err(got, want, group):
    return (got.double() - want).unflatten(-1, (-1, group)).norm(dim=-1)


def attend_closely(mx, plan, q, counts=None, causal=False, scale=None, sharp=True, copies=1):
    """Attention within the bound above, and where `sharp`, that the bound would notice a lost tile or zeros.
    `copies` of the batch in one call: enough of them leave a warp whole sequences instead of a tile or two."""
    scale = plan.head_dim ** -0.5 if scale is None else scale
    rows = q.shape[2] * (q.shape[1] // plan.kv_heads)
    tensor_core = plan.dtype != "float32" and rows > 64 and scale > 0
    o = mx.fast.quantized_cache_attention(
        mx.array(q.repeat(copies, 1, 1, 1)), plan.cache, mx.array(ints(plan.lengths * copies)),
        block_table=mx.array(plan.table.repeat(copies, 1)),
        counts=None if counts is None else mx.array(ints(counts * copies)), scale=scale,
        mask="causal" if causal else None)._t.unflatten(0, (copies, -1))
    want, tol, tile = bounds(plan, q, counts, scale, causal, tensor_core)
    if sharp:
        n = torch.tensor(plan.lengths, device="cuda")[:, None, None, None].expand_as(tol)
        live = (tol > 0) & (n >= 64)
        assert live.any()
        assert float((want.unflatten(-1, (-1, plan.group)).norm(dim=-1) > 4 * tol)[live].double().mean()) > 0.99
        assert float((tile > 2 * tol)[live].double().mean()) > (0.4 if causal else 0.99)
    err = groups_err(o, want, plan.group)
    worst = float((err / tol.clamp_min(1e-300)).nan_to_num(torch.inf).masked_fill((tol == 0) & (err == 0), 0.0).max())
    assert worst <= 1.0, f"{worst:.3g} of the bound"
    return o[0]


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("head_dim,group,heads", [(64, 32, 4), (64, 64, 24), (128, 32, 8), (128, 64, 2), (128, 64, 24),
                                                  (128, 128, 10), (256, 32, 2), (256, 64, 16), (256, 128, 6)])
def test_tokens_closely(mx, dtype, head_dim, group, heads):
    plan = Plan(mx, [1, 2500, 130, 0, 700], kv_heads=2, head_dim=head_dim, group=group, dtype=dtype, seed=heads)
    attend_closely(mx, plan, rand((5, heads, 1, head_dim), dtype, 3))
    attend_closely(mx, plan, rand((5, heads, 3, head_dim), dtype, 4), [1, 3, 2, 3, 0], causal=True)


@pytest.mark.parametrize("dtype", list(DTYPES))
def test_long_histories_closely(mx, dtype):
    plan = Plan(mx, [9000, 1, 4096], kv_heads=1, page=64, dtype=dtype, seed=2)
    attend_closely(mx, plan, rand((3, 4, 1, 128), dtype, 5))


@pytest.mark.parametrize("dtype", ["bfloat16", "float16"])
@pytest.mark.parametrize("head_dim,group", [(64, 32), (64, 64), (128, 32), (128, 64), (128, 128), (256, 64)])
@pytest.mark.parametrize("tokens,heads", [(40, 4), (150, 4), (300, 8)])  # packed and split; packed; expanded
@pytest.mark.parametrize("causal", [False, True])
def test_chunks_closely(mx, dtype, head_dim, group, tokens, heads, causal):
    plan = Plan(mx, [1500, tokens, 0, 131], kv_heads=2, head_dim=head_dim, group=group, dtype=dtype, page=24, seed=tokens)
    attend_closely(mx, plan, rand((4, heads, tokens, head_dim), dtype, 7), [tokens, tokens, 3, 31], causal=causal)


@pytest.mark.parametrize("dtype", ["bfloat16", "float16"])
@pytest.mark.parametrize("head_dim,group", [(64, 32), (128, 64), (128, 128), (256, 64)])
@pytest.mark.parametrize("tokens", [60, 500])  # packed (heads of 256: expanded), expanded
def test_chunks_to_the_types_own_rounding(mx, dtype, head_dim, group, tokens):
    """The norm of the whole error of a chunk over normal keys and values.  Independent errors add in squares, each
    uniform up to its bound, so a third of that in square: the output's rounding, u at the start of a binade and
    less behind it; weights and values, 2^-11; keys, 2^-11 of sqrt(sum q_d^2 k_d^2) scale = 1 in a score.  5 % for
    what 10^5 values and more leave to chance."""
    u = 2.0 ** {"bfloat16": -8, "float16": -11}[dtype]
    plan = Plan(mx, [3000, 1100], kv_heads=2, head_dim=head_dim, group=group, dtype=dtype, page=64, seed=tokens)
    q = rand((2, 8, tokens, head_dim), dtype, 17)
    o = mx.fast.quantized_cache_attention(mx.array(q), plan.cache, mx.array(ints(plan.lengths)),
                                          block_table=mx.array(plan.table), scale=head_dim ** -0.5, mask="causal")._t
    want = bounds(plan, q, None, head_dim ** -0.5, True, True)[0]
    off = float((o.double() - want).norm() / want.norm())
    assert off <= 1.05 * ((u * u + 3 * 2.0 ** -22) / 3) ** 0.5, f"{off:.3g}"


# --- values of very different magnitude ---------------------------------------------------


def spread(dtype, bits):
    """Two factors 2^bits apart (24 at most in f16) whose values, and the steps between them, every type holds."""
    if dtype == "float16":
        bits = min(bits, 24)
        return 2.0 ** (bits // 2), 2.0 ** (bits // 2 - bits)
    return 2.0 ** bits, 1.0


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("bits", [10, 20, 36])
@pytest.mark.parametrize("head_dim,group,heads", [(64, 32, 2), (128, 64, 8), (128, 32, 20), (256, 32, 2)])
def test_groups_of_different_magnitude(mx, dtype, bits, head_dim, group, heads):
    """Small values beside large ones: each group to its own precision."""
    plan = Plan(mx, [1200, 90], kv_heads=2, head_dim=head_dim, group=group, dtype=dtype, seed=bits)
    large, small = spread(dtype, bits)
    factor = torch.full((head_dim // group,), large, device="cuda")
    factor[1::2] = small
    for part in plan.cache.values[1:]:
        part._t.copy_(part._t.float() * factor)
    attend_closely(mx, plan, rand((2, heads, 1, head_dim), dtype, 6))


@pytest.mark.parametrize("copies", [1, 1500])
@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("heads,tokens", [(2, 1), (8, 2), (16, 3), (30, 3)])
@pytest.mark.parametrize("at", [0, 5, 700])
def test_a_large_value_of_no_weight(mx, dtype, heads, tokens, at, copies):
    """A key that no query attends to may have values of any size, wherever a warp meets it."""
    plan = Plan(mx, [1200], kv_heads=2, dtype=dtype, page=1200, spare=0)
    large, small = spread(dtype, 36)
    k, v = plan.dense
    k[:, :, at] = -8.0
    v *= small
    v[:, :, at] *= large / small
    sides = [mx.quantize(mx.array(x), group_size=64, bits=4) for x in plan.dense]
    plan.cache = mx.fast.QuantizedKVCache(*sides, group_size=64, bits=4)
    attend_closely(mx, plan, rand((1, heads, tokens, 128), dtype, 8).abs(), scale=0.125, copies=copies)


@pytest.mark.parametrize("copies", [1, 1500])
@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("heads,kv_heads,tokens", [(2, 2, 3), (4, 2, 7), (2, 1, 30), (4, 2, 80)])
def test_a_large_value_that_later_tokens_alone_see(mx, dtype, heads, kv_heads, tokens, copies):
    plan = Plan(mx, [200], kv_heads=kv_heads, dtype=dtype, page=200, spare=0)
    large, small = spread(dtype, 60)
    v = plan.dense[1]
    v *= small
    v[:, :, 199] *= large / small
    sides = [mx.quantize(mx.array(x), group_size=64, bits=4) for x in plan.dense]
    plan.cache = mx.fast.QuantizedKVCache(*sides, group_size=64, bits=4)
    q = rand((1, heads, tokens, 128), dtype, 9)
    o = attend_closely(mx, plan, q, causal=True, sharp=False, copies=copies)
    plan.lengths = [199]  # without that key the other rows have a bound of their own
    want, tol, _ = bounds(plan, q[:, :, :-1], None, 128 ** -0.5, True, dtype != "float32" and tokens * heads // kv_heads > 64)
    assert bool((groups_err(o[:, :, :-1], want, 64) <= tol).all())


@pytest.mark.parametrize("copies", [1, 1500])
@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("heads,tokens", [(2, 1), (8, 2), (30, 3)])
def test_large_values_whose_weight_fades(mx, dtype, heads, tokens, copies):
    """Scores rise along the keys; the first keys, whose values are large, weigh nothing in the end."""
    plan = Plan(mx, [700], kv_heads=2, dtype=dtype, page=700, spare=0)
    large, small = spread(dtype, 36)
    k, v = plan.dense
    k.copy_(torch.linspace(-4, 4, 700, device="cuda")[:, None] + 0.02 * k)
    v *= small
    v[:, :, :64] *= large / small
    sides = [mx.quantize(mx.array(x), group_size=64, bits=4) for x in plan.dense]
    plan.cache = mx.fast.QuantizedKVCache(*sides, group_size=64, bits=4)
    q = torch.ones((1, heads, tokens, 128), device="cuda").to(DTYPES[dtype])
    attend_closely(mx, plan, q, scale=0.5, sharp=False, copies=copies)


@pytest.mark.parametrize("copies", [1, 1500])
@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
@pytest.mark.parametrize("heads,tokens", [(2, 1), (8, 2), (30, 3)])
@pytest.mark.parametrize("drop", [20.0, 100.0, 400.0])
def test_values_of_the_whole_range(mx, dtype, heads, tokens, drop, copies):
    """The first 64 keys' values are 2^140 of the others', with scores `drop` below theirs: by 2^29 of their weight,
    and they decide the output, by 2^144, and both count, by 2^577, and they are nothing."""
    plan = Plan(mx, [700], kv_heads=2, dtype=dtype, page=700, spare=0)
    k, v = plan.dense
    k *= 0.02
    k[:, :, :64] -= drop / 64
    v *= 2.0 ** -20
    v[:, :, :64] *= 2.0 ** 70
    v[:, :, :64] *= 2.0 ** 70
    sides = [mx.quantize(mx.array(x), group_size=64, bits=4) for x in plan.dense]
    plan.cache = mx.fast.QuantizedKVCache(*sides, group_size=64, bits=4)
    q = torch.ones((1, heads, tokens, 128), device="cuda").to(DTYPES[dtype])
    attend_closely(mx, plan, q, scale=0.5, sharp=False, copies=copies)


@pytest.mark.parametrize("dtype", ["bfloat16", "float16"])
@pytest.mark.parametrize("tokens", [40, 300])  # packed, expanded; both split along the keys
@pytest.mark.parametrize("what", ["value", "groups", "keys"])
@pytest.mark.parametrize("causal", [False, True])
def test_chunks_over_more_than_f16_holds(mx, dtype, tokens, what, causal):
    """A key of no weight with a large value, groups of different magnitude, keys next to nothing among others: what
    a tile of 128 keys cannot hold in f16 units of its own."""
    plan = Plan(mx, [900, 500], kv_heads=2, dtype=dtype, page=100)
    large, small = spread(dtype, 36)
    k, v = plan.dense
    q = rand((2, 8, tokens, 128), dtype, 16)
    if what == "value":
        q = q.abs()
        at = int(plan.table[0, 4])
        k[at, :, 50] = -8.0
        v *= small
        v[at, :, 50] *= large / small
    elif what == "groups":
        v[..., :64] *= large
        v[..., 64:] *= small
    else:
        k[int(plan.table[1, 2]), :, :50] *= 2.0 ** (-24 if dtype == "float16" else -36)
    sides = [mx.quantize(mx.array(x), group_size=64, bits=4) for x in plan.dense]
    plan.cache = mx.fast.QuantizedKVCache(*sides, group_size=64, bits=4)
    attend_closely(mx, plan, q, causal=causal, sharp=False)


@pytest.mark.parametrize("dtype", ["bfloat16", "float16"])
@pytest.mark.parametrize("tokens", [40, 300])
def test_chunks_over_zeros(mx, dtype, tokens):
    """Tokens of zeros, and heads of the head dimension that are next to nothing, among ordinary ones."""
    plan = Plan(mx, [900, 500], kv_heads=2, dtype=dtype, page=100)
    for x in plan.dense:
        x[:, :, 10:13] = 0.0
        x[:, 1, :, 64:] *= 2.0 ** -12
    sides = [mx.quantize(mx.array(x), group_size=64, bits=4) for x in plan.dense]
    plan.cache = mx.fast.QuantizedKVCache(*sides, group_size=64, bits=4)
    attend_closely(mx, plan, rand((2, 8, tokens, 128), dtype, 18), causal=True, sharp=False)


# --- pages that are none of the cache's ------------------------------------------------------


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("page,head_dim,group", [(16, 128, 64), (8, 64, 32), (40, 256, 32), (3, 128, 128)])
@pytest.mark.parametrize("tokens", [1, 40, 100, 300])
@pytest.mark.parametrize("entry", [-1, 1 << 30])
def test_keys_of_a_bad_page_count_as_zeros(mx, dtype, page, head_dim, group, tokens, entry):
    """Nothing of the cache's first page, or any other, reaches the output."""
    from phew_b200._native import PhewError
    from phew_b200.ops import check_device_errors

    plan = Plan(mx, [170], kv_heads=2, head_dim=head_dim, group=group, page=page, dtype=dtype, spare=1)
    free = (set(range(plan.cache.pages)) - set(plan.table[0].tolist())).pop()
    for part in (*plan.cache.keys, *plan.cache.values):
        part._t[free].zero_()
    q = rand((1, 4, tokens, head_dim), dtype, 10)
    run = lambda: mx.fast.quantized_cache_attention(  # noqa: E731
        mx.array(q), plan.cache, [170], block_table=mx.array(plan.table), scale=head_dim ** -0.5, mask="causal")._t
    plan.table[0, 1] = free
    want = run()
    plan.table[0, 1] = entry
    got = run()
    with pytest.raises(PhewError, match="outside a sequence's pages"):
        check_device_errors()
    assert torch.equal(got, want)


# --- writing what is no number ----------------------------------------------------------------


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("bits,head_dim,group", [(4, 128, 64), (8, 64, 32), (4, 256, 128), (8, 128, 128)])
def test_update_keeps_what_is_no_number(mx, dtype, bits, head_dim, group):
    """A group with a NaN reads back as NaN; its neighbours, and infinities, are mx.quantize's."""
    x = rand((1, 2, 9, head_dim), dtype, 11)
    nan = torch.zeros((1, 2, 9, head_dim // group), dtype=torch.bool, device="cuda")
    for head, row, col, bad in [(0, 0, 0, float("nan")), (0, 3, head_dim - 1, -float("nan")), (1, 4, group - 1, float("nan")),
                                (1, 1, 3, float("inf")), (1, 2, 17, -float("inf"))]:
        x[0, head, row, col] = bad
        nan[0, head, row, col // group] |= bad != bad
    x[0, 1, 8] = float("nan")
    nan[0, 1, 8] = True
    x[0, 0, 7] = float("inf")
    cache = mx.fast.QuantizedKVCache.zeros(1, 2, 9, head_dim, dtype, group_size=group, bits=bits)
    got = mx.fast.quantized_cache_update(cache, mx.array(x), mx.array(-x), [0], fetch=True)
    for y, side, dense in ((x, cache.keys, got[0]._t), (-x, cache.values, got[1]._t)):
        want = [a._t for a in mx.quantize(mx.array(y), group_size=group, bits=bits)]
        assert torch.isnan(side[1]._t[nan]).all() and torch.isnan(side[2]._t[nan]).all()
        for a, w in zip(side[1:], want[1:]):
            assert torch.equal(a._t[~nan].view(torch.uint8), w[~nan].view(torch.uint8))
        codes = lambda t: t.view(torch.int32).unflatten(-1, (head_dim // group, -1))  # noqa: E731
        assert torch.equal(codes(side[0]._t)[~nan], codes(want[0])[~nan])
        assert not codes(side[0]._t)[nan].any()
        plain = mx.dequantize(*(mx.array(a) for a in want), group_size=group, bits=bits)._t.unflatten(-1, (-1, group))
        read = mx.fast.quantized_cache_fetch(cache, [9])[0 if y is x else 1]._t
        for v in (dense, read):
            v = v.unflatten(-1, (-1, group))
            assert torch.isnan(v[nan]).all()
            assert torch.equal(v[~nan].nan_to_num(7.0), plain[~nan].nan_to_num(7.0))


# --- large queries and keys -------------------------------------------------------------------------------


@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
@pytest.mark.parametrize("tokens", [1, 3, 100])
def test_queries_whose_sum_passes_the_range(mx, dtype, tokens):
    """Finite scores of queries of up to 2^126: their sum over the head dimension alone is past 32 bits."""
    plan = Plan(mx, [300], dtype=dtype, kv_heads=1)
    for part in plan.cache.keys[1:]:
        part._t.mul_(2.0 ** -20)
    q = rand((1, 2, tokens, 128), dtype, 12).abs()
    for up in (1.0, 2.0 ** 124):
        attend_closely(mx, plan, q * up, scale=2.0 ** 17 / up)


@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
@pytest.mark.parametrize("tokens", [1, 3, 100])
@pytest.mark.parametrize("up", [2.0 ** 118, 2.0 ** -70])
def test_large_and_small_keys(mx, dtype, tokens, up):
    """Keys near the ends of the range, whose scores are finite."""
    plan = Plan(mx, [300], dtype=dtype, kv_heads=1)
    for part in plan.cache.keys[1:]:
        part._t.mul_(up)
    attend_closely(mx, plan, rand((1, 2, tokens, 128), dtype, 15), scale=0.1 / up)


# --- nothing asked ---------------------------------------------------------------------------


@pytest.mark.parametrize("captured", [False, True])
def test_no_queries_over_long_histories(mx, captured):
    """A chunk step in which no sequence has a token: zeros, and the scratch is free for what comes next."""
    B, tokens = 8, 300
    plan = Plan(mx, [20000] * B, kv_heads=2, page=256)
    q, table = mx.array(rand((B, 8, tokens, 128), "bfloat16", 13)), mx.array(plan.table)
    n, counts = mx.array(ints(plan.lengths)), mx.array(ints([0] * B))
    scratch = 2 * B * 2 * 20096 * 128  # 16-bit values of both sides

    def step():
        o = mx.fast.quantized_cache_attention(q, plan.cache, n, block_table=table, counts=counts, scale=0.1, mask="causal")._t
        return o, [torch.full((scratch // 2,), 3.0, dtype=torch.bfloat16, device="cuda") for _ in range(2)]

    step()
    torch.cuda.synchronize()
    replay = None
    if captured:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step()
        replay = graph.replay
    for _ in range(10):
        if replay:
            replay()
        else:
            out = step()
        o, after = out
        assert not o.any() and all(bool((a == 3.0).all()) for a in after)


# --- the first cache of a device -----------------------------------------------------------------


@pytest.mark.filterwarnings("ignore:The CUDA Graph is empty")
def test_first_cache_inside_a_capture_is_refused(mx, monkeypatch):
    """Its error flag would be the graph's memory, zeroed by every replay.  Later caches may be made there."""
    from phew_b200 import kv_cache

    plan = Plan(mx, [40], page=16)
    q, n, table = mx.array(rand((1, 4, 1, 128), "bfloat16", 14)), mx.array(ints([40])), mx.array(plan.table)

    def attend():
        cache = mx.fast.QuantizedKVCache(plan.cache.keys, plan.cache.values)
        return mx.fast.quantized_cache_attention(q, cache, n, block_table=table, scale=0.1)._t

    want = attend().clone()
    torch.cuda.synchronize()
    with monkeypatch.context() as m:
        m.setattr(kv_cache, "_error_flags", {})
        with pytest.raises(RuntimeError, match="inside a capture"):
            with torch.cuda.graph(torch.cuda.CUDAGraph()):
                attend()
        assert not kv_cache._error_flags
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        o = attend()
    graph.replay()
    assert torch.equal(o, want)


def test_caches_made_by_threads_report_to_one_flag(mx, monkeypatch):
    import threading

    from phew_b200 import kv_cache

    monkeypatch.setattr(kv_cache, "_error_flags", {})
    plan, caches, start = Plan(mx, [40]), [], threading.Barrier(8)
    kv_cache._error_flags.clear()

    def make():
        start.wait()
        caches.append(mx.fast.QuantizedKVCache(plan.cache.keys, plan.cache.values))

    threads = [threading.Thread(target=make) for _ in range(8)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    flag = kv_cache._error_flags[plan.cache.device.index]
    assert len(caches) == 8 and all(c._flag == flag.data_ptr() for c in caches) and not flag.any()


# --- two at once -----------------------------------------------------------------------------------


@pytest.mark.parametrize("tokens", [40, 300])  # packed, expanded; both split along the keys
@pytest.mark.parametrize("odd", [False, True])
def test_chunks_on_two_streams(mx, tokens, odd):
    """Each call has its scratch, and the launches behind it wait for their own; over a tile that f16 does not hold
    in one of the caches too."""
    plans = [Plan(mx, [1500, 700], kv_heads=2, page=64, seed=i) for i in range(2)]
    if odd:
        plans[1].cache.values[1]._t[int(plans[1].table[0, 3]), :, 5] = 2.0 ** 40
    qs = [mx.array(rand((2, 8, tokens, 128), "bfloat16", 20 + i)) for i in range(2)]
    n = [mx.array(ints(p.lengths)) for p in plans]
    tables = [mx.array(p.table) for p in plans]
    run = lambda i: mx.fast.quantized_cache_attention(  # noqa: E731
        qs[i], plans[i].cache, n[i], block_table=tables[i], scale=128 ** -0.5, mask="causal")._t
    want = [run(i).clone() for i in range(2)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    outs = [[], []]
    for _ in range(20):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                outs[i].append(run(i))
    torch.cuda.synchronize()
    for i in range(2):
        assert torch.isfinite(want[i]).all() and all(torch.equal(o, want[i]) for o in outs[i])


def test_chunk_replays_over_other_contents(mx):
    """A captured chunk whose cache comes to hold what f16 does not, and no longer does."""
    plan = Plan(mx, [700], kv_heads=2, page=64)
    q, table, n = mx.array(rand((1, 8, 300, 128), "bfloat16", 21)), mx.array(plan.table), mx.array(ints([700]))
    run = lambda: mx.fast.quantized_cache_attention(q, plan.cache, n, block_table=table, scale=0.1, mask="causal")._t  # noqa: E731
    run()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        o = run()
    scales = plan.cache.values[1]._t
    old = scales.clone()
    for factor in (1.0, 2.0 ** 40, 1.0, 2.0 ** 40):
        scales.copy_(old)
        scales[int(plan.table[0, 2]), :, 7] *= factor
        graph.replay()
        want, tol, _ = bounds(plan, q._t, None, 0.1, True, True)
        assert bool((groups_err(o, want, 64) <= tol).all())
