"""A quantised key/value cache: tokens written into pages, read back, attended to.

The k and v that ``mx.fast.quantized_scaled_dot_product_attention`` takes
(phew ``emit/codegen.py:428-449``), kept between calls: the affine group-wise
codes of ``mx.quantize``, in pages, written one step at a time and read in
place.  Lengths, offsets and block tables are int32 arrays on the device, so
a step captured into a CUDA graph replays with new ones.
"""

from __future__ import annotations

import ctypes
import functools
import threading

import torch

from . import _native
from . import dtypes as dt
from .mx import core

_error_flags: dict[int, torch.Tensor] = {}
_error_flags_lock = threading.Lock()
_Strides = ctypes.c_int64 * 3


def cache_error_flag(device: torch.device) -> torch.Tensor:
    """Two device ints (0 = clean): [0] set when a position or a page lies
    outside the cache, [1] when a bounded wait ran out.  One pair to a device,
    made once, and zero on every stream when it is returned."""
    f = _error_flags.get(device.index)
    if f is None:
        with _error_flags_lock:
            f = _error_flags.get(device.index)
            if f is None:
                with torch.cuda.device(device):
                    if torch.cuda.is_current_stream_capturing():
                        # (it would be the graph's memory, and zeroed by every replay)
                        raise RuntimeError("QuantizedKVCache: a device's first cache cannot be made inside a capture")
                    f = torch.zeros(2, dtype=torch.int32, device=device)
                    torch.cuda.current_stream().synchronize()
                _error_flags[device.index] = f
    return f


def check_cache_errors() -> None:
    """Raise if a kernel of the cache met a position outside a sequence's
    pages or a block table entry that is no page, or gave up a wait
    (synchronises)."""
    for f in list(_error_flags.values()):
        code, waited = f.tolist()
        if code or waited:
            f.zero_()
        if waited:
            raise _native.PhewError(waited, "quantised cache: a device-side wait timed out (pipeline stalled)")
        if code:
            raise _native.PhewError(
                code, "quantised cache: a length or offset outside a sequence's pages, or a block "
                      "table entry that is no page of the cache")


class QuantizedKVCache:
    """Keys and values in pages of token rows, ``(codes, scales, biases)`` each:

    * codes ``[pages, kv_heads, page_size, head_dim * bits / 32]`` uint32 (or
      int32), packed as by ``mx.quantize`` along the head dimension;
    * scales, biases ``[pages, kv_heads, page_size, head_dim / group_size]`` in
      the cache's dtype (float32, float16 or bfloat16).

    ``bits`` 4 or 8 (attention reads 4), ``head_dim`` 64, 128 or 256,
    ``group_size`` 32, 64 or 128.  The arrays are the caller's: ``update``
    writes into them.  A block table ``[batch, columns]`` names each sequence's
    pages in order; without one page b belongs to sequence b.  A device's first
    cache synchronises with it once, and cannot be made inside a graph capture.
    """

    __slots__ = ("keys", "values", "pages", "kv_heads", "page_size", "head_dim", "group_size", "bits",
                 "dtype", "device", "_torch_dtype", "_unit", "_struct", "_flag", "_flag_tensor", "_written")

    def __init__(self, keys, values, *, group_size: int = 64, bits: int = 4) -> None:
        if len(keys) != 3 or len(values) != 3:
            raise ValueError("QuantizedKVCache: keys and values are (codes, scales, biases) each")
        parts = [a if isinstance(a, core.array) else core.array(a) for a in (*keys, *values)]
        g, nb = int(group_size), int(bits)
        if nb not in (4, 8):
            raise ValueError(f"QuantizedKVCache: bits must be 4 or 8, got {bits}")
        if g not in (32, 64, 128):
            raise ValueError(f"QuantizedKVCache: group_size must be 32, 64 or 128, got {group_size}")
        codes, scales = parts[0], parts[1]
        if codes.ndim != 4:
            raise ValueError(f"QuantizedKVCache: codes must be [pages, kv_heads, page_size, words], got {codes.shape}")
        dim = codes.shape[-1] * 32 // nb
        if dim not in (64, 128, 256) or dim % g:
            raise ValueError(f"QuantizedKVCache: head_dim must be 64, 128 or 256 and a multiple of group_size, "
                             f"got {dim} at group_size {g}")
        if scales.dtype.code is None:
            raise TypeError(f"QuantizedKVCache: unsupported scale dtype {scales.dtype.name}")
        want = codes.shape[:-1] + (dim // g,)
        for i, a in enumerate(parts):
            name = ("key ", "value ")[i // 3] + ("codes", "scales", "biases")[i % 3]
            if i % 3 == 0:
                if a.dtype.name not in ("uint32", "int32"):
                    raise TypeError(f"QuantizedKVCache: {name} must be uint32, got {a.dtype.name}")
                if a.shape != codes.shape:
                    raise ValueError(f"QuantizedKVCache: {name} shape {a.shape} != {codes.shape}")
            else:
                if a.dtype is not scales.dtype:
                    raise TypeError(f"QuantizedKVCache: {name} must be {scales.dtype.name}, got {a.dtype.name}")
                if a.shape != want:
                    raise ValueError(f"QuantizedKVCache: {name} shape {a.shape} != {want}")
            if not a._t.is_contiguous() or a._t.data_ptr() % 16:
                raise ValueError(f"QuantizedKVCache: {name} must be contiguous and 16-byte aligned "
                                 "(the cache is written in place)")
            if a._t.device != codes._t.device:
                raise ValueError(f"QuantizedKVCache: {name} lies on another device")
        if codes.size == 0:
            raise ValueError("QuantizedKVCache: empty cache")
        self.keys, self.values = tuple(parts[:3]), tuple(parts[3:])
        self._written = tuple(a._t for a in parts)  # what an update writes into
        self.pages, self.kv_heads, self.page_size = codes.shape[:3]
        self.head_dim, self.group_size, self.bits, self.dtype = dim, g, nb, scales.dtype
        self.device = codes._t.device
        self._struct = _native.KVCache(*(ctypes.c_void_p(a._t.data_ptr()) for a in parts), self.pages,
                                       self.page_size, self.kv_heads, dim, g, nb, self.dtype.code)
        self._torch_dtype, self._unit = self.dtype.torch, 16 // self.dtype.size
        self._flag_tensor = cache_error_flag(self.device)  # (kernels get its address: it lives as long as the cache)
        self._flag = self._flag_tensor.data_ptr()

    @classmethod
    def zeros(cls, pages: int, kv_heads: int, page_size: int, head_dim: int, dtype="bfloat16", *,
              group_size: int = 64, bits: int = 4) -> "QuantizedKVCache":
        """A cache of its own arrays, all zero."""
        if int(bits) not in (4, 8) or int(group_size) not in (32, 64, 128):
            raise ValueError("QuantizedKVCache: bits must be 4 or 8, group_size 32, 64 or 128")
        d, rows = dt.from_any(dtype), (int(pages), int(kv_heads), int(page_size))

        def side():
            codes = torch.zeros(rows + (head_dim * int(bits) // 32,), dtype=torch.int32, device=core.device())
            sb = [torch.zeros(rows + (head_dim // int(group_size),), dtype=d.torch, device=core.device())
                  for _ in range(2)]
            return tuple(core.array(t) for t in (codes, *sb))

        return cls(side(), side(), group_size=group_size, bits=bits)


def _as_ints(x) -> torch.Tensor:
    """The tensor of an array, or of a host sequence copied in as int32."""
    if isinstance(x, core.array):
        return x._t
    return core.array(x, None if isinstance(x, torch.Tensor) else core.int32)._t


def _copied(t: torch.Tensor) -> torch.Tensor:
    """A contiguous copy, made on the tensor's device."""
    with torch.cuda.device(t.device):
        return core.contiguous_copy(core.array._wrap(t))._t


def _ints(x, batch: int, what: str, cache: QuantizedKVCache) -> torch.Tensor:
    """An int32 [batch] array on the cache's device."""
    t = _as_ints(x)
    if t.dtype != torch.int32:
        raise TypeError(f"{what} must be int32, got {dt.from_any(t.dtype).name}")
    if t.shape != (batch,):
        raise ValueError(f"{what} shape {tuple(t.shape)} != {(batch,)}")
    if t.device != cache.device:
        raise ValueError(f"{what} lies on another device than the cache")
    return t if t.is_contiguous() else _copied(t)


def _table(block_table, batch: int, what: str, cache: QuantizedKVCache):
    """(tensor that holds the table or None, pointer, row stride, columns)."""
    if block_table is None:
        if batch > cache.pages:
            raise ValueError(f"{what}: without a block_table the cache needs a page for each of the {batch} "
                             f"sequences, it has {cache.pages}")
        return None, None, 0, 1
    t = _as_ints(block_table)
    if t.dtype != torch.int32:
        raise TypeError(f"{what}: block_table must be int32, got {dt.from_any(t.dtype).name}")
    if t.dim() != 2 or t.shape[0] != batch or t.shape[1] == 0:
        raise ValueError(f"{what}: block_table shape {tuple(t.shape)} is not [{batch}, columns]")
    if t.device != cache.device:
        raise ValueError(f"{what}: block_table lies on another device than the cache")
    stride, unit = t.stride()
    if unit != 1 and t.shape[1] > 1:
        t = _copied(t)
        stride = t.shape[1]
    return t, t.data_ptr(), stride, t.shape[1]


@functools.lru_cache(maxsize=1024)
def _strides(token: int, head: int, batch: int):
    return _Strides(token, head, batch)


def _rows(x, what: str, cache: QuantizedKVCache):
    """(tensor, strides {token, head, batch}) of a [batch, heads, tokens, head_dim]
    view that the kernels read in place: unit stride along the head dimension
    and 16-byte aligned rows; anything else is copied first."""
    t = x._t if isinstance(x, core.array) else core.asarray_device(x, contiguous=False)._t
    if t.dtype != cache._torch_dtype:
        raise TypeError(f"{what} must be {cache.dtype.name} like the cache, got {dt.from_any(t.dtype).name}")
    if t.dim() != 4 or t.shape[3] != cache.head_dim:
        raise ValueError(f"{what} shape {tuple(t.shape)} is not [batch, heads, tokens, {cache.head_dim}]")
    if t.numel() == 0:
        raise ValueError(f"{what} is empty")
    if t.device != cache.device:
        raise ValueError(f"{what} lies on another device than the cache")
    b, h, n, unit = t.stride()
    if unit != 1 or (b | h | n) % cache._unit or t.data_ptr() % 16:
        t = _copied(t)
        b, h, n, unit = t.stride()
    return t, _strides(n, h, b)


def _empty_like(t: torch.Tensor) -> torch.Tensor:
    """A contiguous array like `t` (empty_like is the quickest way to one, but keeps a view's strides)."""
    return torch.empty_like(t) if t.is_contiguous() else t.new_empty(t.shape)


def _stream(cache: QuantizedKVCache) -> int:
    return torch.cuda.current_stream(cache.device).cuda_stream


_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)
if _raw_stream is not None:  # the same stream without a Stream object around it

    def _stream(cache: QuantizedKVCache) -> int:  # noqa: F811
        return _raw_stream(cache.device.index)


_functions: dict[str, object] = {}


def _call(name: str, cache: QuantizedKVCache, *args) -> None:
    """Calls an entry point on the cache's device and current stream there."""
    fn = _functions.get(name)
    if fn is None:
        fn = _functions[name] = getattr(_native.load(), name)
    if torch.cuda.current_device() == cache.device.index:
        status = fn(cache._struct, *args, cache._flag, _stream(cache))
    else:
        with torch.cuda.device(cache.device):  # kernels launch on the current device
            status = fn(cache._struct, *args, cache._flag, _stream(cache))
    if status:
        _native.check(status, name)


@functools.lru_cache(maxsize=1024)
def _workspace(device: int, page_size: int, kv_heads: int, head_dim: int, group_size: int, dtype: int, batch: int,
               heads: int, tokens: int, columns: int) -> int:
    """Scratch bytes of an attention call; they depend on its sizes and the device alone."""
    c = _native.KVCache(page_size=page_size, kv_heads=kv_heads, head_dim=head_dim, group_size=group_size, dtype=dtype)
    with torch.cuda.device(device):
        return int(_native.load().phew_kv_attention_workspace(c, batch, heads, tokens, columns))


def quantized_cache_update(cache: QuantizedKVCache, k, v, offsets, *, block_table=None, counts=None,
                           fetch: bool = False):
    """Quantises ``k``, ``v`` ``[batch, kv_heads, tokens, head_dim]`` (the cache's
    dtype) into the cache at positions ``offsets[b] + token``, in place.

    ``counts`` (int32 ``[batch]``, default all) limits a padded batch to its
    first tokens; every other row of the cache stays as it was.  A row's codes,
    scales and biases are those of ``mx.quantize`` on it, but a group that holds
    a NaN reads back as NaN (scale and bias NaN, codes 0).  With ``fetch`` the
    values that the new tokens now stand for are returned as ``(k, v)`` like
    the inputs (``mx.dequantize``'s, zero behind ``counts``), e.g. for a prompt's
    own attention.  Two tokens of one call must not land in the same row.
    A position or page outside the cache is left unwritten and reported by
    ``ops.check_device_errors``.  Inside ``mx.compile`` pending arrays that
    read the cache's arrays are computed before the write.
    """
    k, ks = _rows(k, "quantized_cache_update: k", cache)
    v, vs = _rows(v, "quantized_cache_update: v", cache)
    shape = k.shape
    batch, heads, tokens, _ = shape
    if heads != cache.kv_heads:
        raise ValueError(f"quantized_cache_update: k shape {tuple(shape)} does not have the cache's "
                         f"{cache.kv_heads} heads")
    if v.shape != shape:
        raise ValueError(f"quantized_cache_update: v shape {tuple(v.shape)} != k's {tuple(shape)}")
    off = _ints(offsets, batch, "quantized_cache_update: offsets", cache)
    cnt = None if counts is None else _ints(counts, batch, "quantized_cache_update: counts", cache)
    keep, table, stride, columns = _table(block_table, batch, "quantized_cache_update", cache)
    core.settle_readers(cache._written)
    out = None
    if fetch:
        out = (_empty_like(k), _empty_like(k))
    _call("phew_kv_update", cache, k.data_ptr(), v.data_ptr(), ks, vs, batch, tokens, off.data_ptr(),
          None if cnt is None else cnt.data_ptr(), table, stride, columns,
          out[0].data_ptr() if fetch else None, out[1].data_ptr() if fetch else None)
    del keep
    return (core.array._wrap(out[0]), core.array._wrap(out[1])) if fetch else None


def quantized_cache_fetch(cache: QuantizedKVCache, lengths, *, block_table=None, max_length: int | None = None):
    """The first ``lengths[b]`` tokens of every sequence as dense ``(k, v)``
    ``[batch, kv_heads, max_length, head_dim]`` in the cache's dtype
    (``mx.dequantize``'s values), zero behind a sequence.  ``max_length``
    defaults to what a sequence's pages hold; longer sequences are cut there.
    """
    n = _as_ints(lengths)
    if n.dim() != 1 or n.shape[0] == 0:
        raise ValueError(f"quantized_cache_fetch: lengths shape {tuple(n.shape)} is not [batch]")
    batch = n.shape[0]
    n = _ints(n, batch, "quantized_cache_fetch: lengths", cache)
    keep, table, stride, columns = _table(block_table, batch, "quantized_cache_fetch", cache)
    out_len = columns * cache.page_size if max_length is None else int(max_length)
    if out_len <= 0:
        raise ValueError(f"quantized_cache_fetch: max_length must be positive, got {max_length}")
    shape = (batch, cache.kv_heads, out_len, cache.head_dim)
    one = cache.keys[1]._t
    k = one.new_empty(shape)
    v = torch.empty_like(k)
    _call("phew_kv_fetch", cache, k.data_ptr(), v.data_ptr(), batch, out_len, n.data_ptr(), table, stride, columns)
    del keep
    return core.array._wrap(k), core.array._wrap(v)


def quantized_cache_attention(q, cache: QuantizedKVCache, lengths, *, block_table=None, counts=None,
                              scale: float = 1.0, mask=None):
    """``softmax(scale * q k^T) v`` over a 4-bit cache -> ``[batch, heads, tokens, head_dim]``.

    ``q`` ``[batch, heads, tokens, head_dim]`` in the cache's dtype, heads a
    multiple of the cache's (query head h reads cache head h // (heads /
    kv_heads)); ``lengths`` (int32 ``[batch]``) the keys of each sequence, new
    tokens included; ``counts`` (int32 ``[batch]``, default all) its query
    tokens in a padded batch.  ``mask`` None, or ``"causal"``: the last query
    token sits at the sequence's last key.  Rows that see no key, and rows
    behind ``counts``, are zero.  A block table entry that is no page of the
    cache stands for keys and values of zero, a length past a sequence's pages
    ends at them; both are reported by ``ops.check_device_errors``.

    Scores, softmax statistics and sums are 32-bit.  With up to 64 query rows
    (tokens x heads / kv_heads) to a cache head, and always in float32, the
    codes enter the products as they are and weights times value scales are
    rounded to 11 bits (22 in float32, queries too); with more, keys, values
    and weights are rounded to 11 bits each.  Errors of an output's norm are then
    1.7e-3 in bfloat16 (its own rounding); in float16 (2.1e-4) 3e-4, above 64
    rows 4e-4 to 5e-4.

    Above 64 rows the call takes scratch from torch's allocator, up to 1 GiB,
    and which kernels it runs goes by the tokens that the block table could
    hold, not by the lengths: a table as wide as the longest sequence needs is
    the fastest, and heads of 256 whose table passes the scratch (2 x batch x
    kv_heads x tokens x 512 bytes) are several times slower.
    """
    if mask is not None and not (isinstance(mask, str) and mask == "causal"):
        raise ValueError(f"quantized_cache_attention: mask must be None or 'causal', got {mask!r}")
    if cache.bits != 4:
        raise ValueError(f"quantized_cache_attention: the cache must hold 4-bit codes, it holds {cache.bits}-bit "
                         "ones (quantized_cache_fetch reads them back for the dense attention)")
    q, qs = _rows(q, "quantized_cache_attention: q", cache)
    shape = q.shape
    batch, heads, tokens, _ = shape
    if heads % cache.kv_heads:
        raise ValueError(f"quantized_cache_attention: {heads} query heads over {cache.kv_heads} cache heads")
    n = _ints(lengths, batch, "quantized_cache_attention: lengths", cache)
    cnt = None if counts is None else _ints(counts, batch, "quantized_cache_attention: counts", cache)
    keep, table, stride, columns = _table(block_table, batch, "quantized_cache_attention", cache)
    size = _workspace(cache.device.index, cache.page_size, cache.kv_heads, cache.head_dim, cache.group_size,
                      cache.dtype.code, batch, heads, tokens, columns)
    work = n.new_empty(size // 4)
    o = _empty_like(q)
    _call("phew_kv_attention", cache, q.data_ptr(), qs, o.data_ptr(), batch, heads, tokens, n.data_ptr(),
          None if cnt is None else cnt.data_ptr(), table, stride, columns, scale, 0 if mask is None else 1,
          work.data_ptr(), size)
    del keep, work
    return core.array._wrap(o)
