"""Quantised key/value cache: writes against mx.quantize, reads against
mx.dequantize (bit for bit both), attention against a 64-bit softmax over the
cache's values, at the lengths, pages and masks where it can go wrong."""

from __future__ import annotations

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

DTYPES = {"bfloat16": torch.bfloat16, "float16": torch.float16, "float32": torch.float32}
#: half a rounding step relative to the value
UNIT = {"bfloat16": 2.0 ** -8, "float16": 2.0 ** -11, "float32": 2.0 ** -24}


@pytest.fixture(autouse=True)
def _clean(mx):
    from phew_b200.ops import check_device_errors

    yield
    mx.synchronize()
    check_device_errors()


def rand(shape, dtype, seed, scale=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(shape, generator=g, device="cuda") * scale).to(DTYPES[dtype])


def ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


class Plan:
    """A cache with random contents and where each sequence's pages lie."""

    def __init__(self, mx, lengths, *, kv_heads=2, head_dim=128, group=64, bits=4, page=16, dtype="bfloat16",
                 spare=2, seed=0, scale=1.0):
        self.mx, self.bits, self.group, self.page = mx, bits, group, page
        self.lengths, self.dtype, self.kv_heads, self.head_dim = list(lengths), dtype, kv_heads, head_dim
        need = [-(-n // page) for n in lengths]
        columns = max(1, max(need))
        pages = sum(need) + spare
        rng = np.random.default_rng(seed)
        order = rng.permutation(pages)
        table = np.full((len(lengths), columns), -7, np.int32)  # entries behind a sequence are never read
        at = 0
        for b, n in enumerate(need):
            table[b, :n] = order[at:at + n]
            at += n
        self.table = ints(table.tolist())
        shape = (pages, kv_heads, page, head_dim)
        self.dense = [rand(shape, dtype, 10 * seed + i, scale) for i in range(2)]
        sides = [mx.quantize(mx.array(x), group_size=group, bits=bits) for x in self.dense]
        self.cache = mx.fast.QuantizedKVCache(*sides, group_size=group, bits=bits)

    def parts(self, side):
        return self.cache.keys if side == 0 else self.cache.values

    def values(self, side, b, length=None):
        """[kv_heads, length, head_dim] of sequence b in 64 bits: scale * code + bias, unrounded."""
        length = self.lengths[b] if length is None else length
        codes, scales, biases = (p._t for p in self.parts(side))
        cols = self.table[b, : -(-length // self.page)].long()
        pick = lambda t: t[cols].transpose(0, 1).flatten(1, 2)[:, :length]  # noqa: E731
        words = pick(codes.view(torch.int32)).to(torch.int64) & 0xFFFFFFFF
        shift = torch.arange(0, 32, self.bits, device="cuda")
        n = ((words[..., None] >> shift) & ((1 << self.bits) - 1)).flatten(-2).double()
        sc, bi = (pick(t).double().repeat_interleave(self.group, -1) for t in (scales, biases))
        return sc * n + bi


def attend64(plan, q, counts, scale, causal):
    """(output, bound) in 64 bits.  The bound is the arithmetic of one kernel pass: with S the sum of
    |q||k| behind a score and V the largest |value| a row can weigh (codes centred, so at most 8 steps
    and the centre),
      * output rounded once:                         u |o|
      * softmax weights rounded to the type's 16 bits before the product (bf16; the other types keep
        16 bits and more):                           u V
      * scores summed in fp32 over head_dim terms and the weights' exponentials: a relative error of
        2 (head_dim / 2 + 8) 2^-24 scale S + 2^-20 of each weight, on numerator and denominator
      * long queries read keys and values rounded to the type, as the dense attention does: u scale S on
        a score (2^-8 or 2^-11 of it, independent roundings: root of head_dim of them at most six sigma)
        and u V."""
    u = UNIT[plan.dtype]
    B, H, L, D = q.shape
    per = H // plan.kv_heads
    out = torch.zeros(q.shape, dtype=torch.float64, device="cuda")
    tol = torch.zeros_like(out)
    tensor_path = plan.dtype != "float32"
    for b, n in enumerate(plan.lengths):
        c = L if counts is None else counts[b]
        if n == 0 or c == 0:
            continue
        K, V = plan.values(0, b), plan.values(1, b)
        for h in range(H):
            k, v = K[h // per], V[h // per]
            x = q[b, h, :c].double()
            s = (x @ k.T) * scale
            if causal:
                i = torch.arange(c, device="cuda")[:, None]
                j = torch.arange(n, device="cuda")[None]
                s = s.masked_fill(j > n - c + i, -torch.inf)
            some = (s > -torch.inf).any(-1, keepdim=True)
            p = torch.where(some, torch.softmax(s, -1), 0.0)
            o = p @ v
            big = v.abs().max()
            ds = abs(scale) * (x.abs() @ k.abs().T).amax(-1, keepdim=True) * (D / 2 + 8) * 2.0 ** -24
            rel = 2 * ds + 2.0 ** -20
            t = u * o.abs() + rel * 2 * big
            if tensor_path:
                noise = abs(scale) * u * 6 * (x.square() @ k.square().T).amax(-1, keepdim=True).sqrt()
                t = t + 2 * u * big + 2 * noise * big * 0.5
            out[b, h, :c], tol[b, h, :c] = o, t + 1e-30
    return out, tol


def check(got, want, tol):
    err = (got.double() - want).abs()
    assert bool((err <= tol).all()), f"worst {float((err / tol.clamp_min(1e-30)).max()):.3g} of the bound"


# --- writing -------------------------------------------------------------------


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("bits,group,head_dim", [(4, 64, 128), (8, 32, 64), (4, 128, 256), (8, 128, 128),
                                                 (4, 32, 256), (4, 64, 64)])
def test_update_is_quantize_in_place(mx, dtype, bits, group, head_dim):
    before, new = [0, 5, 17, 40], [7, 1, 0, 4]
    plan = Plan(mx, [a + n for a, n in zip(before, new)], kv_heads=3, head_dim=head_dim, group=group, bits=bits,
                page=8, dtype=dtype, seed=bits + group)
    old = [[p._t.clone() for p in plan.parts(s)] for s in range(2)]
    x = [rand((4, 3, 7, head_dim), dtype, 70 + s, 3.0) for s in range(2)]
    x[0][0, 0, 0] = 1.25  # a constant row: the smallest scale
    x[1][0, 1, 1] = 0.0
    got = mx.fast.quantized_cache_update(plan.cache, mx.array(x[0]), mx.array(x[1]), mx.array(ints(before)),
                                         block_table=mx.array(plan.table), counts=mx.array(ints(new)), fetch=True)
    for s in range(2):
        want = [a._t for a in mx.quantize(mx.array(x[s]), group_size=group, bits=bits)]
        dense = mx.dequantize(*(mx.array(a) for a in want), group_size=group, bits=bits)._t
        for b in range(4):
            dense[b, :, new[b]:] = 0
            for i in range(new[b]):
                page, row = divmod(before[b] + i, 8)
                page = int(plan.table[b, page])
                for o, w in zip(old[s], want):
                    o.view(torch.uint8)[page, :, row] = w.contiguous().view(torch.uint8)[b, :, i]
        for o, p in zip(old[s], plan.parts(s)):
            assert torch.equal(o.view(torch.uint8), p._t.view(torch.uint8))  # written rows and all others
        assert torch.equal(got[s]._t.contiguous().view(torch.uint8), dense.contiguous().view(torch.uint8))


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("bits", [4, 8])
def test_update_codes_at_borders(mx, dtype, bits):
    """Values on and next to the borders between codes round as in mx.quantize."""
    top = (1 << bits) - 1
    base = torch.arange(64, device="cuda", dtype=torch.float32) % (top + 1)
    base[0], base[1] = 0, top
    rows = []
    for scale in (1.0, 0.1, 3.0e-3, 7.7, 1e-30 if dtype != "float16" else 1e-4, 1000.0):
        for off in (0.0, 0.5, 0.49999997, 0.25):
            rows.append(((base + off) * scale).clamp(0, top * scale))
    x = torch.stack(rows).to(DTYPES[dtype])[None, None]
    n = x.shape[2]
    cache = mx.fast.QuantizedKVCache.zeros(1, 1, n, 64, dtype, group_size=64, bits=bits)
    mx.fast.quantized_cache_update(cache, mx.array(x), mx.array(-x), [0])
    for s, side in ((1.0, cache.keys), (-1.0, cache.values)):
        for got, want in zip(side, mx.quantize(mx.array(x * s), group_size=64, bits=bits)):
            assert torch.equal(got._t.view(torch.uint8), want._t.view(torch.uint8))


def test_update_reads_strided_views(mx):
    """k and v sliced out of a fused [batch, tokens, 3, heads, head_dim] projection, and ones that need a copy."""
    plan = Plan(mx, [33, 12], kv_heads=4, page=24)
    qkv = rand((2, 12, 3, 4, 128), "bfloat16", 5)
    k, v = qkv[:, :, 1].transpose(1, 2), qkv[:, :, 2].transpose(1, 2)
    odd = rand((2, 4, 12, 131), "bfloat16", 6)[..., 1:129]  # rows off the 16-byte grid
    for kk, vv in ((k, v), (odd, v), (k, odd)):
        mx.fast.quantized_cache_update(plan.cache, mx.array(kk), mx.array(vv), [21, 0],
                                       block_table=mx.array(plan.table))
        got = mx.fast.quantized_cache_fetch(plan.cache, plan.lengths, block_table=mx.array(plan.table))
        for g, x in zip(got, (kk, vv)):
            want = mx.dequantize(*mx.quantize(mx.array(x)))._t
            assert torch.equal(g._t[0, :, 21:33], want[0])
            assert torch.equal(g._t[1, :, :12], want[1])


# --- reading -------------------------------------------------------------------


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("bits,group,head_dim,page", [(4, 64, 128, 16), (8, 32, 64, 7), (4, 128, 128, 1),
                                                      (8, 64, 256, 40), (4, 32, 64, 64)])
@pytest.mark.parametrize("max_length", [None, 50, 1])
def test_fetch_is_dequantize(mx, dtype, bits, group, head_dim, page, max_length):
    plan = Plan(mx, [50, 0, 1, 23], kv_heads=3, head_dim=head_dim, group=group, bits=bits, page=page, dtype=dtype)
    got = mx.fast.quantized_cache_fetch(plan.cache, mx.array(ints(plan.lengths)), block_table=mx.array(plan.table),
                                        max_length=max_length)
    out = plan.table.shape[1] * page if max_length is None else max_length
    for s in range(2):
        assert got[s].shape == (4, 3, out, head_dim)
        flat = mx.dequantize(*plan.parts(s), group_size=group, bits=bits)._t
        for b, n in enumerate(plan.lengths):
            m = min(n, out)
            rows = flat[plan.table[b, : -(-n // page)].long()].transpose(0, 1).flatten(1, 2)[:, :m]
            assert torch.equal(got[s]._t[b, :, :m].contiguous().view(torch.uint8), rows.contiguous().view(torch.uint8))
            assert not got[s]._t[b, :, m:].any()


def test_fetch_without_a_table(mx):
    plan = Plan(mx, [48], page=48, spare=3)
    k, v = mx.fast.quantized_cache_fetch(plan.cache, [48, 5, 0])
    flat = mx.dequantize(*plan.cache.keys)._t
    assert torch.equal(k._t[0], flat[0]) and torch.equal(k._t[1, :, :5], flat[1, :, :5])
    assert not k._t[1, :, 5:].any() and not k._t[2].any() and v.shape == (3, 2, 48, 128)


# --- attention -----------------------------------------------------------------


def attend(mx, plan, q, counts=None, scale=None, causal=False):
    scale = plan.head_dim ** -0.5 if scale is None else scale
    o = mx.fast.quantized_cache_attention(
        mx.array(q), plan.cache, mx.array(ints(plan.lengths)), block_table=mx.array(plan.table),
        counts=None if counts is None else mx.array(ints(counts)), scale=scale, mask="causal" if causal else None)
    assert o.shape == tuple(q.shape) and o.dtype.name == plan.dtype
    check(o._t, *attend64(plan, q, counts, scale, causal))
    return o._t


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("head_dim,group", [(64, 32), (64, 64), (128, 32), (128, 64), (128, 128), (256, 32),
                                            (256, 64), (256, 128)])
@pytest.mark.parametrize("per", [1, 5, 8])
def test_attention_single_tokens(mx, dtype, head_dim, group, per):
    plan = Plan(mx, [1, 130, 0, 31, 1000], kv_heads=2, head_dim=head_dim, group=group, dtype=dtype, seed=per)
    attend(mx, plan, rand((5, 2 * per, 1, head_dim), dtype, 3))


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("page", [1, 3, 16, 40, 256])
def test_attention_pages(mx, dtype, page):
    """Pages of one row, of an odd size, ending inside a tile, longer than a tile."""
    plan = Plan(mx, [257, 15, 16, 17, 128, 129], kv_heads=1, page=page, dtype=dtype)
    attend(mx, plan, rand((6, 4, 1, 128), dtype, 4))


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("tokens,heads,head_dim,group", [(2, 4, 128, 64), (5, 16, 64, 32), (7, 6, 256, 128),
                                                         (16, 8, 128, 128), (33, 2, 128, 64), (70, 8, 128, 32)])
@pytest.mark.parametrize("causal", [True, False])
def test_attention_several_tokens(mx, dtype, tokens, heads, head_dim, group, causal):
    """Drafted tokens and chunks in a padded batch; sequences shorter than their queries leave rows empty."""
    lengths = [tokens, 300, 3, 0, 129, 1]
    counts = [tokens, tokens, tokens, 1, max(1, tokens // 2), 0]
    plan = Plan(mx, lengths, kv_heads=2, head_dim=head_dim, group=group, dtype=dtype, seed=tokens)
    o = attend(mx, plan, rand((6, heads, tokens, head_dim), dtype, 5), counts, causal=causal)
    assert not o[3].any() and not o[5].any() and not o[4, :, counts[4]:].any()
    if causal and tokens > 3:
        assert not o[2, :, : tokens - 3].any()  # three keys: only the last three tokens see any


@pytest.mark.parametrize("dtype", ["bfloat16", "float16"])
@pytest.mark.parametrize("tokens,lengths,heads,kv_heads", [(128, [128, 500], 4, 4), (200, [200, 1000], 8, 2),
                                                           (256, [4096], 5, 1), (130, [131, 130], 6, 2)])
@pytest.mark.parametrize("causal", [True, False])
def test_attention_chunks(mx, dtype, tokens, lengths, heads, kv_heads, causal):
    plan = Plan(mx, lengths, kv_heads=kv_heads, dtype=dtype, seed=tokens)
    attend(mx, plan, rand((len(lengths), heads, tokens, 128), dtype, 6), causal=causal)


@pytest.mark.parametrize("dtype", ["bfloat16", "float16"])
@pytest.mark.parametrize("head_dim,group", [(64, 32), (64, 64), (128, 32), (128, 128), (256, 32), (256, 128)])
@pytest.mark.parametrize("tokens,heads", [(40, 4), (150, 4), (150, 12), (400, 8)])
def test_attention_chunks_of_every_head(mx, dtype, head_dim, group, tokens, heads):
    """Few row blocks (packed tiles) and many (the cache expanded first), padded batches, odd pages."""
    lengths, counts = [900, tokens, 0, 131], [tokens, tokens, 3, 100 if tokens > 100 else 7]
    plan = Plan(mx, lengths, kv_heads=2, head_dim=head_dim, group=group, dtype=dtype, page=24, seed=heads)
    attend(mx, plan, rand((4, heads, tokens, head_dim), dtype, 7), counts, causal=True)


def test_attention_chunk_with_a_wide_table(mx):
    """A table for far more tokens than the sequence has: too much to expand, and many empty splits."""
    plan = Plan(mx, [700], kv_heads=2, page=16)
    wide = torch.full((1, 1 << 17), -5, dtype=torch.int32, device="cuda")
    wide[:, : plan.table.shape[1]] = plan.table
    plan.table = wide
    attend(mx, plan, rand((1, 8, 300, 128), "bfloat16", 17), causal=True)
    attend(mx, plan, rand((1, 8, 1, 128), "bfloat16", 18))


@pytest.mark.parametrize("head_dim,tokens", [(128, 70), (128, 600), (256, 200)])
@pytest.mark.parametrize("stage", [0, 1])
def test_stalled_pipeline_is_reported(mx, head_dim, tokens, stage):
    """A value tile that is never announced: the waits run out, the call reports it and the next one works."""
    from phew_b200 import _native
    from phew_b200.ops import check_device_errors

    plan = Plan(mx, [700], kv_heads=2, head_dim=head_dim, dtype="bfloat16")
    q = rand((1, 4, tokens, head_dim), "bfloat16", 19)
    attend(mx, plan, q, causal=True)
    mx.synchronize()
    _native.call("phew_test_inject_stall", stage, 20_000_000)
    mx.fast.quantized_cache_attention(mx.array(q), plan.cache, [700], block_table=mx.array(plan.table), mask="causal")
    with pytest.raises(_native.PhewError, match="timed out"):
        check_device_errors()
    for _ in range(3):
        attend(mx, plan, q, causal=True)


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("tokens", [1, 40])
@pytest.mark.parametrize("scale", [-0.2, 0.0, 3.0])
def test_attention_any_scale(mx, dtype, tokens, scale):
    """Negative and zero scales, and one that makes nearly one-hot weights."""
    plan = Plan(mx, [200, 77], dtype=dtype)
    attend(mx, plan, rand((2, 4, tokens, 128), dtype, 8), scale=scale)


@pytest.mark.parametrize("dtype", list(DTYPES))
def test_attention_rising_scores(mx, dtype):
    """Scores that grow along the keys move the running maximum at every tile; falling ones never."""
    plan = Plan(mx, [700], kv_heads=2, dtype=dtype, page=700)
    ramp = torch.linspace(-4, 4, 700, device="cuda")
    k = torch.ones((1, 2, 700, 128), device="cuda") * ramp[:, None]
    k[:, 1] = -k[:, 1]
    k = (k + 0.05 * rand(k.shape, "float32", 1)).to(DTYPES[dtype])
    mx.fast.quantized_cache_update(plan.cache, mx.array(k), mx.array(rand(k.shape, dtype, 2)), [0],
                                   block_table=mx.array(plan.table))
    q = torch.ones((1, 4, 3, 128), device="cuda").to(DTYPES[dtype])
    attend(mx, plan, q, scale=0.5)


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("tokens", [3, 130])
def test_attention_ignores_what_it_may_not_see(mx, dtype, tokens):
    """Rows behind a sequence and pages of others may hold NaN and infinities; a causal key that only
    later queries see may be infinite without touching the earlier ones."""
    n = 150
    plan = Plan(mx, [n], kv_heads=1, dtype=dtype, page=64)
    q = rand((1, 2, tokens, 128), dtype, 9)
    want = attend(mx, plan, q, causal=True).clone()
    used = plan.table[0].tolist()
    for side in range(2):
        for part in plan.parts(side)[1:]:
            for page in range(part.shape[0]):
                if page not in used:
                    part._t[page] = float("nan")
            part._t[used[-1], :, n % 64:] = float("inf")
    assert torch.equal(attend(mx, plan, q, causal=True), want)
    for side in range(2):  # the last key: only the last query sees it
        plan.parts(side)[1]._t[used[-1], :, n % 64 - 1] = float("inf")
    o = mx.fast.quantized_cache_attention(mx.array(q), plan.cache, [n], block_table=mx.array(plan.table),
                                          scale=128 ** -0.5, mask="causal")._t
    assert torch.equal(o[:, :, :-1], want[:, :, :-1]) and not torch.isfinite(o[:, :, -1]).any()


def test_attention_many_short_and_one_long(mx):
    """Work split over a ragged batch: more sequences than blocks, and one much longer than the rest."""
    lengths = [1 + (37 * b) % 50 for b in range(700)]
    lengths[311] = 9000
    plan = Plan(mx, lengths, kv_heads=1, head_dim=64, group=32)
    attend(mx, plan, rand((700, 2, 1, 64), "bfloat16", 11))


def test_attention_one_long_sequence(mx):
    plan = Plan(mx, [70001], kv_heads=1, page=256, dtype="float16")
    attend(mx, plan, rand((1, 8, 1, 128), "float16", 12))


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("head_dim,group", [(128, 64), (64, 32), (256, 128)])
def test_attention_flat_sums(mx, dtype, head_dim, group):
    """Nearly equal weights over 40000 keys, where sums of codes are hundreds of times what is left of them.

    Norm of the error over the norm of the outputs, which are N keys' mean, sigma / sqrt(N) in size; every error
    below is independent of the values it meets and of its neighbours, so norms add in squares:
      * output rounded once, and 16-bit types' weights rounded before their product: a uniform error of at most
        u, root mean square u / sqrt(3) of a value at the start of its binade: at most sqrt(2 / 3) u together
      * weights' exponentials: below 2^-20 of each
      * 32-bit sums: 64 sequences of 2 heads over 1250 tiles of 32 keys leave a warp about 100 tiles, 200
        additions to an output, each off by at most 2^-24 of the running sum.  That sum holds what the centring
        leaves, half a code step (4 sigma / 15 / 2 = 0.13 sigma) times its 3200 keys at most, where the outputs
        hold sigma sqrt(3200): sqrt(200) 2^-24 0.13 sqrt(3200) = 2^-17.4, and the biases' sums the same again."""
    n, u = 40000, UNIT[dtype]
    plan = Plan(mx, [n], kv_heads=2, head_dim=head_dim, group=group, page=64, dtype=dtype, seed=3)
    B = 64
    q = rand((B, 2, 1, head_dim), dtype, 4, 0.05)
    scale = head_dim ** -0.5
    o = mx.fast.quantized_cache_attention(mx.array(q), plan.cache, mx.array(ints([n] * B)),
                                          block_table=mx.array(plan.table.expand(B, -1)), scale=scale)._t.double()
    for h in range(2):
        p = torch.softmax(q[:, h, 0].double() @ plan.values(0, 0)[h].T * scale, -1)
        want = p @ plan.values(1, 0)[h]
        worst = float(((o[:, h, 0] - want).norm(dim=-1) / want.norm(dim=-1)).max())
        assert worst <= u + 2.0 ** -20 + 2 * 2.0 ** -17.4, f"{worst:.3g}"


def test_attention_flat_sums_of_a_long_share(mx):
    """As above where a warp takes 1180 tiles of 32 keys (512 sequences of 131072 on the same pages), and bf16's
    sums hold the codes themselves: 16 tiles of them at a time, 32 steps that each lose at most 2^-24 of the sum so
    far on average, always downwards.  That is 7.5 steps times the keys, 1.63 sigma times them, where the outputs
    hold sigma sqrt(131072) = 362 sigma: 32 2^-24 1.63 362 = 2^-9.8."""
    n, B = 131072, 512
    plan = Plan(mx, [n], kv_heads=1, page=256, seed=5)
    q = rand((B, 1, 1, 128), "bfloat16", 6, 0.05)
    o = mx.fast.quantized_cache_attention(mx.array(q), plan.cache, mx.array(ints([n] * B)),
                                          block_table=mx.array(plan.table.expand(B, -1)), scale=128 ** -0.5)._t
    rows = slice(0, B, 64)
    p = torch.softmax(q[rows, 0, 0].double() @ plan.values(0, 0)[0].T * 128 ** -0.5, -1)
    want = p @ plan.values(1, 0)[0]
    worst = float(((o[rows, 0, 0].double() - want).norm(dim=-1) / want.norm(dim=-1)).max())
    assert worst <= UNIT["bfloat16"] + 2.0 ** -20 + 2.0 ** -9.8, f"{worst:.3g}"


def test_attention_reads_strided_queries(mx):
    plan = Plan(mx, [90, 14], kv_heads=2)
    x = rand((2, 5, 3, 4, 128), "bfloat16", 13)
    q = x[:, :, 0].transpose(1, 2)
    same = attend(mx, plan, q, causal=True)
    assert torch.equal(same, attend(mx, plan, q.contiguous(), causal=True))
    odd = torch.cat([q, q[..., :3]], -1)[..., : 128]
    assert torch.equal(same, attend(mx, plan, odd, causal=True))


@pytest.mark.parametrize("tokens", [100, 200])  # packed, expanded
def test_attention_chunk_reads_strided_queries(mx, tokens):
    plan = Plan(mx, [300, tokens], kv_heads=2)
    x = rand((2, tokens, 3, 8, 128), "bfloat16", 14)
    q = x[:, :, 1].transpose(1, 2)
    same = attend(mx, plan, q, causal=True)
    assert torch.equal(same, attend(mx, plan, q.contiguous(), causal=True))
    one = q[:1, :1].expand(2, 8, tokens, 128)  # broadcast over sequences and heads
    assert torch.equal(attend(mx, plan, one, causal=True), attend(mx, plan, one.contiguous(), causal=True))


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("tokens", [2, 100, 200])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
def test_attention_queries_that_are_no_numbers(mx, dtype, tokens, bad):
    """An odd query's row is no number; its neighbours do not notice."""
    plan = Plan(mx, [300, 40], kv_heads=2, dtype=dtype)
    q = rand((2, 8, tokens, 128), dtype, 15)
    want = attend(mx, plan, q)
    q[1, 2, 1, 77] = bad
    got = mx.fast.quantized_cache_attention(mx.array(q), plan.cache, mx.array(ints(plan.lengths)), block_table=mx.array(
        plan.table), scale=128 ** -0.5)._t
    assert not torch.isfinite(got[1, 2, 1]).any()
    got[1, 2, 1] = want[1, 2, 1]
    assert torch.equal(got, want)


@pytest.mark.parametrize("dtype", ["bfloat16", "float16"])
@pytest.mark.parametrize("tokens", [3, 100, 200])
def test_attention_values_at_the_end_of_the_range(mx, dtype, tokens):
    """Groups from -top to top: code 15 of such a scale rounds past the type's range in f16 (65536), and the rows
    that do not see that key must not meet an infinity.  (bf16's range is as large as that of 32-bit sums: a
    quarter of it.)"""
    plan = Plan(mx, [tokens + 60], kv_heads=1, dtype=dtype, spare=0)
    last = tokens + 59
    page, row = int(plan.table[0, last // plan.page]), last % plan.page
    top = torch.finfo(DTYPES[dtype]).max * (0.25 if dtype == "bfloat16" else 1.0)
    plan.dense[1][page, 0, row] = torch.tensor([-top, top], dtype=DTYPES[dtype], device="cuda").repeat(64)
    sides = [mx.quantize(mx.array(x), group_size=64, bits=4) for x in plan.dense]
    plan.cache = mx.fast.QuantizedKVCache(*sides, group_size=64, bits=4)
    v = plan.values(1, 0)[0, -1]
    assert float(v.max()) >= top  # (65536 > 65504 in f16)
    q = rand((1, 8, tokens, 128), dtype, 16)
    o = mx.fast.quantized_cache_attention(mx.array(q), plan.cache, mx.array(ints([tokens + 60])),
                                          block_table=mx.array(plan.table), scale=128 ** -0.5, mask="causal")._t
    want, tol = attend64(plan, q, None, 128 ** -0.5, True)
    check(o[:, :, -1], want[:, :, -1], tol[:, :, -1])
    plan.lengths = [tokens + 59]  # the bound of the other rows is that of the keys that they see
    check(o[:, :, :-1], *attend64(plan, q[:, :, :-1], None, 128 ** -0.5, True))


def test_attention_far_rows(mx):
    """A cache of more than 2^32 bytes of codes: rows near its end."""
    pages, page = 1100, 16384  # 18 M rows of 2 heads x 128 bytes: 4.6 GB a side
    cache = mx.fast.QuantizedKVCache.zeros(pages, 2, page, 256, "bfloat16", group_size=128)
    table = ints([[1099, 3]])
    k, v = (rand((1, 2, 300, 256), "bfloat16", 14 + i) for i in range(2))
    mx.fast.quantized_cache_update(cache, mx.array(k), mx.array(v), [16200], block_table=mx.array(table))
    q = rand((1, 4, 1, 256), "bfloat16", 16)
    o = mx.fast.quantized_cache_attention(mx.array(q), cache, [16500], block_table=mx.array(table), scale=4.0)._t
    kd, vd = (mx.dequantize(*mx.quantize(mx.array(x), group_size=128), group_size=128)._t.double() for x in (k, v))
    # the 16200 rows before hold zeros: score 0, value 0
    for h in range(4):
        s = torch.cat([torch.zeros(16200, device="cuda").double(), (kd[0, h // 2] @ q[0, h, 0].double()) * 4.0])
        want = torch.softmax(s, 0)[16200:] @ vd[0, h // 2]
        # keys and values here are rounded to bf16 (2^-8 of each): a score moves by at most
        # six sigma of 4 |q| |k| 2^-8 / sqrt(3), values by 2^-8
        noise = 4.0 * 2.0 ** -8 / 3 ** 0.5 * 6 * float((kd[0, h // 2].square() @ q[0, h, 0].double().square()).max()) ** 0.5
        assert float((o[0, h, 0].double() - want).abs().max()) <= (2 * 2.0 ** -8 + 2 * noise) * float(vd.abs().max())
    got = mx.fast.quantized_cache_fetch(cache, [16500], block_table=mx.array(table))[0]._t
    assert torch.equal(got[0, :, 16200:16500].double(), kd[0]) and not got[0, :, :16200].any()


# --- streams, graphs, errors, refusals --------------------------------------------


def test_step_in_a_graph_with_moving_lengths(mx):
    """A captured decode step (write, then attend) replays at other lengths, and two graphs of the
    same cache replayed in turn do not disturb one another."""
    plan = Plan(mx, [40, 200], kv_heads=2)
    table, lengths, offsets = mx.array(plan.table), ints([1, 1]), ints([0, 0])
    k, v = (rand((2, 2, 1, 128), "bfloat16", 20 + i) for i in range(2))
    q = rand((2, 8, 1, 128), "bfloat16", 22)

    def step():
        mx.fast.quantized_cache_update(plan.cache, mx.array(k), mx.array(v), mx.array(offsets), block_table=table)
        return mx.fast.quantized_cache_attention(mx.array(q), plan.cache, mx.array(lengths), block_table=table,
                                                 scale=0.1)._t

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            o = step()
        graphs.append((g, o))
    for n, (g, o) in zip([(40, 200), (7, 111), (33, 1), (1, 160)], graphs * 2):
        lengths.copy_(ints(list(n)))
        offsets.copy_(lengths - 1)
        k.copy_(rand(k.shape, "bfloat16", 30 + n[0]))
        g.replay()
        torch.cuda.synchronize()
        plan.lengths = list(n)
        check(o, *attend64(plan, q, None, 0.1, False))


@pytest.mark.parametrize("tokens", [100, 300])  # packed and split along the keys; expanded
def test_chunks_in_a_graph_with_moving_lengths(mx, tokens):
    """A captured chunk (write, attend, read back) replays with other lengths and counts, against the eager calls."""
    plan = Plan(mx, [900, 500], kv_heads=2)
    table, lengths, counts = mx.array(plan.table), ints([tokens, tokens]), ints([tokens, tokens])
    offsets = ints([0, 0])
    k, v = (rand((2, 2, tokens, 128), "bfloat16", 40 + i) for i in range(2))
    q = rand((2, 8, tokens, 128), "bfloat16", 42)

    def step():
        mx.fast.quantized_cache_update(plan.cache, mx.array(k), mx.array(v), mx.array(offsets), block_table=table,
                                       counts=mx.array(counts))
        o = mx.fast.quantized_cache_attention(mx.array(q), plan.cache, mx.array(lengths), block_table=table,
                                              counts=mx.array(counts), scale=0.1, mask="causal")
        kv = mx.fast.quantized_cache_fetch(plan.cache, mx.array(lengths), block_table=table, max_length=700)
        return o._t, kv[0]._t, kv[1]._t

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = step()
    for n, c in [((900, 500), (tokens, tokens)), ((tokens, 1), (tokens, 1)), ((77, 333), (5, 0)), ((640, 0), (90, 0))]:
        lengths.copy_(ints(list(n)))
        counts.copy_(ints(list(c)))
        offsets.copy_(lengths - counts)
        k.copy_(rand(k.shape, "bfloat16", 50 + n[0]))
        g.replay()
        plan.lengths = list(n)
        check(out[0], *attend64(plan, q, list(c), 0.1, True))
        assert all(torch.equal(a, b) for a, b in zip(out, step()))


def test_two_streams_at_once(mx):
    """Calls on two streams share nothing but the cache they read."""
    plan = Plan(mx, [3000] * 4, kv_heads=4, page=64)
    qs = [rand((4, 16, 1, 128), "bfloat16", 40 + i) for i in range(2)]
    want = [attend(mx, plan, q).clone() for q in qs]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    outs = [[], []]
    n, table = mx.array(ints(plan.lengths)), mx.array(plan.table)
    for _ in range(20):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                outs[i].append(mx.fast.quantized_cache_attention(mx.array(qs[i]), plan.cache, n, block_table=table,
                                                                 scale=128 ** -0.5)._t)
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(o, want[i]) for o in outs[i])


@pytest.mark.parametrize("entry", [-1, 9, 1 << 30])
def test_bad_pages_are_reported_and_not_touched(mx, entry):
    from phew_b200._native import PhewError
    from phew_b200.ops import check_device_errors

    plan = Plan(mx, [40], page=16, spare=6)  # 9 pages
    good = plan.table.clone()
    bad = good.clone()
    bad[0, 1] = entry
    before = [p._t.clone() for s in range(2) for p in plan.parts(s)]
    x = rand((1, 2, 20, 128), "bfloat16", 50)
    calls = [
        lambda: mx.fast.quantized_cache_update(plan.cache, mx.array(x), mx.array(x), [14], block_table=mx.array(bad)),
        lambda: mx.fast.quantized_cache_fetch(plan.cache, [40], block_table=mx.array(bad)),
        lambda: mx.fast.quantized_cache_attention(mx.array(x[:, :, :1].contiguous()), plan.cache, [40],
                                                  block_table=mx.array(bad)),
        lambda: mx.fast.quantized_cache_attention(mx.array(torch.cat([x] * 4, 2)), plan.cache, [40],
                                                  block_table=mx.array(bad)),
        # more tokens than the sequence's pages hold
        lambda: mx.fast.quantized_cache_attention(mx.array(x[:, :, :1].contiguous()), plan.cache, [49],
                                                  block_table=mx.array(good)),
        lambda: mx.fast.quantized_cache_attention(mx.array(torch.cat([x] * 4, 2)), plan.cache, [-3],
                                                  block_table=mx.array(good)),
        lambda: mx.fast.quantized_cache_fetch(plan.cache, [49], block_table=mx.array(good), max_length=60),
        lambda: mx.fast.quantized_cache_update(plan.cache, mx.array(x), mx.array(x), [-30], block_table=mx.array(good)),
    ]
    for call in calls:
        call()
        with pytest.raises(PhewError, match="outside a sequence's pages"):
            check_device_errors()
        check_device_errors()  # reported once
    # the update through the bad entry wrote positions 14, 15 and 32, 33 and nothing else
    rows = [(int(good[0, 0]), r) for r in (14, 15)] + [(int(good[0, 2]), r) for r in (0, 1)]
    for old, p in zip(before, [p for s in range(2) for p in plan.parts(s)]):
        for page, r in rows:
            old[page, :, r] = p._t[page, :, r]
        assert torch.equal(old, p._t)


def test_refusals(mx):
    f = mx.fast
    plan = Plan(mx, [40, 20])
    c, t = plan.cache, mx.array(plan.table)
    x = mx.array(rand((2, 2, 3, 128), "bfloat16", 60))
    with pytest.raises(ValueError, match="bits must be 4 or 8"):
        f.QuantizedKVCache(c.keys, c.values, bits=2)
    with pytest.raises(ValueError, match="group_size"):
        f.QuantizedKVCache(c.keys, c.values, group_size=16)
    with pytest.raises(ValueError, match="scales shape"):
        f.QuantizedKVCache(c.keys, c.values, group_size=128)
    with pytest.raises(ValueError, match="head_dim must be"):
        f.QuantizedKVCache.zeros(2, 2, 16, 96, group_size=32)
    with pytest.raises(TypeError, match="value codes must be uint32"):
        f.QuantizedKVCache(c.keys, (c.values[1], *c.values[1:]))
    with pytest.raises(TypeError, match="must be bfloat16"):
        f.QuantizedKVCache(c.keys, (c.values[0], c.values[1], c.values[2].astype(mx.float16)))
    with pytest.raises(ValueError, match="contiguous"):
        k0 = mx.array(torch.cat([c.keys[0]._t] * 2, -1)[..., :16])
        f.QuantizedKVCache((k0, *c.keys[1:]), c.values)
    with pytest.raises(TypeError, match="k must be bfloat16"):
        f.quantized_cache_update(c, x.astype(mx.float32), x, [0, 0], block_table=t)
    with pytest.raises(ValueError, match="v shape"):
        f.quantized_cache_update(c, x, mx.array(x._t[:, :, :2]), [0, 0], block_table=t)
    with pytest.raises(ValueError, match="k shape"):
        f.quantized_cache_update(c, mx.array(x._t[:, :1]), x, [0, 0], block_table=t)
    with pytest.raises(ValueError, match="offsets shape"):
        f.quantized_cache_update(c, x, x, [0], block_table=t)
    with pytest.raises(TypeError, match="offsets must be int32"):
        f.quantized_cache_update(c, x, x, mx.array(torch.zeros(2, dtype=torch.int64, device="cuda")), block_table=t)
    with pytest.raises(ValueError, match="block_table shape"):
        f.quantized_cache_fetch(c, [1, 2, 3], block_table=t)
    with pytest.raises(ValueError, match="a page for each"):
        f.quantized_cache_fetch(c, [1] * 50)
    with pytest.raises(ValueError, match="max_length"):
        f.quantized_cache_fetch(c, [1, 2], block_table=t, max_length=0)
    with pytest.raises(ValueError, match="mask must be"):
        f.quantized_cache_attention(x, c, [40, 20], block_table=t, mask=x)
    with pytest.raises(ValueError, match="query heads"):
        f.quantized_cache_attention(mx.array(rand((2, 3, 1, 128), "bfloat16", 1)), c, [40, 20], block_table=t)
    with pytest.raises(ValueError, match="q is empty"):
        f.quantized_cache_attention(mx.array(x._t[:, :, :0]), c, [40, 20], block_table=t)
    eight = Plan(mx, [40, 20], bits=8).cache
    with pytest.raises(ValueError, match="4-bit codes"):
        f.quantized_cache_attention(x, eight, [40, 20], block_table=t)


# --- together --------------------------------------------------------------------


@pytest.mark.parametrize("dtype", ["bfloat16", "float16"])
def test_prompt_then_decode(mx, dtype):
    """As a serving loop uses them: a prompt written (its values fed to the dense attention), then single
    tokens written and attended to, then a drafted block, on one paged cache."""
    B, H, KV, D, P = 2, 4, 4, 128, 128
    plan = Plan(mx, [P + 20] * B, kv_heads=KV, dtype=dtype, seed=9)
    table = mx.array(plan.table)
    q, k, v = (rand((B, n, P, D), dtype, 80 + i) for i, n in enumerate((H, KV, KV)))
    kh, vh = mx.fast.quantized_cache_update(plan.cache, mx.array(k), mx.array(v), [0] * B, block_table=table,
                                            fetch=True)
    dense = mx.fast.scaled_dot_product_attention(mx.array(q), kh, vh, scale=D ** -0.5, mask="causal")._t
    plan.lengths = [P] * B
    cached = attend(mx, plan, q, causal=True)
    big = float(vh._t.double().abs().max())
    # both round weights to 16 bits (u V each) and the output (u |o|), and differ in rounding k and v
    assert float((dense.double() - cached.double()).abs().max()) <= 16 * UNIT[dtype] * big
    for step in range(3):
        k1, v1 = (rand((B, KV, 1, D), dtype, 90 + 2 * step + i) for i in range(2))
        mx.fast.quantized_cache_update(plan.cache, mx.array(k1), mx.array(v1), ints(plan.lengths), block_table=table)
        plan.lengths = [n + 1 for n in plan.lengths]
        attend(mx, plan, rand((B, H, 1, D), dtype, 100 + step))
    counts = [5, 2]
    k5, v5 = (rand((B, KV, 5, D), dtype, 110 + i) for i in range(2))
    mx.fast.quantized_cache_update(plan.cache, mx.array(k5), mx.array(v5), ints(plan.lengths), block_table=table,
                                   counts=ints(counts))
    plan.lengths = [n + c for n, c in zip(plan.lengths, counts)]
    attend(mx, plan, rand((B, H, 5, D), dtype, 120), counts, causal=True)
