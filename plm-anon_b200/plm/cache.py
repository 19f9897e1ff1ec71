"""Paged caches of several sequences: rotating and appending keys and values, and attention over them.

``PagedCache`` holds the pages, in the model dtype or as e4m3 codes with a scale for each block of tokens and head;
``Sequences`` says which rows of a call belong to which sequence, how many tokens each has in the cache, and where its
pages are. ``append`` and ``attention`` enqueue ``plm_cache_append`` and ``plm_cache_attention`` (include/plm_native.h
has the definitions) on the current stream and never synchronise, so both can be captured into a CUDA graph; a replay
reads the lengths and block tables anew from the tensors of its ``Sequences``.

    cache = PagedCache.allocate(num_pages, kv_heads, 64, 128, dtype="e4m3", scale_block=32)
    seqs = Sequences(row_start, context, block_tables, max_rows=1, max_keys=8192)
    q = append(ctx, cache, seqs, k, v, q=q, cos_sin=decoder.cos_sin)
    out = attention(ctx, cache, seqs, q, window=4096, sinks=4)

What contradicts the host's bounds on the device (a row range, a page, a position) is skipped and recorded:
``Context.check`` raises for it.
"""

from __future__ import annotations

import ctypes
import struct

import torch

from . import native
from .native import NativeError

MAX_SCALE_BLOCK = 64

# A call's descriptor is packed from its own fields here and the finished bytes of its cache and sequences: a third of the
# time of filling ctypes structures, and the smallest calls last as long as their host side.
_APPEND = struct.Struct("@iiPPPqqqPqiiPP")    # plm_cache_append_desc up to the cache
_ATTENTION = struct.Struct("@iiPqPqifiiPPPq")  # plm_cache_attention_desc up to the cache
_entry_points: dict = {}


def _entry(name: str, argtypes: list):
    """A function of the library that takes its descriptor as bytes."""
    fn = _entry_points.get(name)
    if fn is None:
        fn = native.library()[name]  # an object of its own, with a signature of its own
        fn.argtypes, fn.restype = argtypes, ctypes.c_int32
        _entry_points[name] = fn
    return fn


def _raw_stream(index: int, stream) -> int:
    return torch._C._cuda_getCurrentRawStream(index) if stream is None else stream.cuda_stream
_MODEL_DTYPES = {torch.bfloat16: native.PLM_BF16, torch.float16: native.PLM_F16}


def _same_device(what: str, device: torch.device, **tensors) -> None:
    for name, t in tensors.items():
        if t is not None and t.device != device:
            raise NativeError(f"{what}: {name} is on {t.device}, not on {device}")


class PagedCache:
    """Pages of keys and values, [num_pages, kv_heads, page_size, head_dim] each: bfloat16 or float16, or
    float8_e4m3fn with ``k_scale`` and ``v_scale`` [num_pages, kv_heads, page_size / scale_block] float32."""

    def __init__(self, k: torch.Tensor, v: torch.Tensor, k_scale: torch.Tensor | None = None,
                 v_scale: torch.Tensor | None = None) -> None:
        if k.dim() != 4 or k.shape != v.shape or k.dtype != v.dtype:
            raise NativeError("PagedCache: k and v are [num_pages, kv_heads, page_size, head_dim] of one shape and dtype")
        if not (k.is_contiguous() and v.is_contiguous()):
            raise NativeError("PagedCache: k and v must be contiguous")
        if k.numel() == 0:
            raise NativeError(f"PagedCache: pages of {list(k.shape)}")
        pages, kv_heads, page, head_dim = k.shape
        e4m3 = k.dtype == torch.float8_e4m3fn
        if not e4m3 and k.dtype not in _MODEL_DTYPES:
            raise NativeError(f"PagedCache: pages of {k.dtype} (bfloat16, float16 or float8_e4m3fn)")
        if e4m3 != (k_scale is not None) or e4m3 != (v_scale is not None):
            raise NativeError("PagedCache: float8_e4m3fn pages have k_scale and v_scale, 16-bit pages have none")
        block = 0
        if e4m3:
            for name, s in (("k_scale", k_scale), ("v_scale", v_scale)):
                if s.dtype != torch.float32 or s.dim() != 3 or not s.is_contiguous() or s.shape != k_scale.shape or \
                        s.shape[:2] != k.shape[:2] or s.shape[2] < 1 or page % s.shape[2]:
                    raise NativeError(f"PagedCache: {name} is contiguous float32 [num_pages, kv_heads, page_size / "
                                      "scale_block]")
            block = page // k_scale.shape[2]
        _same_device("PagedCache", k.device, v=v, k_scale=k_scale, v_scale=v_scale)
        self.k, self.v, self.k_scale, self.v_scale = k, v, k_scale, v_scale
        self.num_pages, self.num_kv_heads, self.page_size, self.head_dim = pages, kv_heads, page, head_dim
        self.scale_block = block
        self.dtype, self.device = k.dtype, k.device
        self.desc = native.PagedCacheDesc(
            kind=native.CACHE_E4M3 if e4m3 else native.CACHE_MODEL, k=k.data_ptr(), v=v.data_ptr(),
            k_scale=native.ptr(k_scale), v_scale=native.ptr(v_scale), scale_block=block, num_pages=pages,
            page_size=page, num_kv_heads=kv_heads, head_dim=head_dim)
        self._bytes = bytes(self.desc)
        self._index = k.get_device()
        self._workspaces: dict = {}  # bytes that an attention call of some sizes needs

    @classmethod
    def allocate(cls, num_pages: int, num_kv_heads: int, page_size: int, head_dim: int, *,
                 dtype: torch.dtype | str = torch.bfloat16, scale_block: int = 16,
                 device: torch.device | str = "cuda") -> "PagedCache":
        """Zeroed pages. ``dtype`` is bfloat16, float16, or "e4m3" for codes with a scale per ``scale_block`` tokens
        (a power of two, at most the page size and 64)."""
        shape = (num_pages, num_kv_heads, page_size, head_dim)
        if dtype not in ("e4m3", torch.float8_e4m3fn):
            return cls(torch.zeros(shape, dtype=dtype, device=device), torch.zeros(shape, dtype=dtype, device=device))
        if scale_block < 1 or scale_block > min(page_size, MAX_SCALE_BLOCK) or page_size % scale_block:
            raise NativeError(f"PagedCache: {scale_block} tokens to a scale with pages of {page_size}")
        scales = (num_pages, num_kv_heads, page_size // scale_block)
        codes = [torch.zeros(shape, dtype=torch.uint8, device=device).view(torch.float8_e4m3fn) for _ in range(2)]
        return cls(*codes, torch.ones(scales, device=device), torch.ones(scales, device=device))


class Sequences:
    """The sequences of a call, on the device: ``row_start`` int32 [n + 1], the first row of each (and the end of the
    last); ``context`` int64 [n], the tokens each has in the cache before its rows; ``block_tables`` int32
    [n, max_pages], logical to physical page. ``max_rows`` bounds the rows of one sequence, ``max_keys`` its context and
    rows together (how attention divides long caches goes by it; the default is what a block table can hold)."""

    def __init__(self, row_start: torch.Tensor, context: torch.Tensor, block_tables: torch.Tensor, *, max_rows: int,
                 max_keys: int = 0) -> None:
        n = context.numel()
        if row_start.dtype != torch.int32 or row_start.dim() != 1 or row_start.numel() != n + 1 or \
                not row_start.is_contiguous():
            raise NativeError("Sequences: row_start is contiguous int32 [n + 1]")
        if context.dtype != torch.int64 or context.dim() != 1 or n < 1 or not context.is_contiguous():
            raise NativeError("Sequences: context is contiguous int64 [n]")
        if block_tables.dtype != torch.int32 or block_tables.dim() != 2 or block_tables.shape[0] != n or \
                block_tables.shape[1] < 1 or (block_tables.shape[1] > 1 and block_tables.stride(1) != 1):
            raise NativeError("Sequences: block_tables is int32 [n, max_pages] with contiguous rows")
        if not (1 <= max_rows < 1 << 31 and 0 <= max_keys < 1 << 63):
            raise NativeError(f"Sequences: at most {max_rows} rows and {max_keys} keys to a sequence")
        _same_device("Sequences", row_start.device, context=context, block_tables=block_tables)
        self.row_start, self.context, self.block_tables = row_start, context, block_tables
        self.count, self.max_rows, self.max_keys, self.device = n, max_rows, max_keys, row_start.device
        pages = block_tables.shape[1]
        self.desc = native.SequencesDesc(
            n_seqs=n, max_rows=max_rows, max_keys=max_keys, row_start=row_start.data_ptr(), context=context.data_ptr(),
            block_tables=block_tables.data_ptr(), table_stride=block_tables.stride(0) if n > 1 else pages,
            max_pages=pages)
        self._bytes = bytes(self.desc)
        self._index = row_start.get_device()


def _heads(what: str, name: str, t: torch.Tensor, rows: int, heads: int | None, head_dim: int, dtype) -> int:
    """Checks [rows, heads, head_dim] with heads side by side in a row; returns the row stride in elements."""
    shape = t.shape
    if len(shape) != 3 or shape[0] != rows or shape[2] != head_dim or (heads is not None and shape[1] != heads):
        raise NativeError(f"{what}: {name} is {list(shape)}, not [{rows}, {heads or 'heads'}, {head_dim}]")
    if shape[1] < 1:
        raise NativeError(f"{what}: {name} has no heads")
    if t.dtype != dtype:
        raise NativeError(f"{what}: {name} is {t.dtype}, not {dtype}")
    stride = t.stride()
    if stride[2] != 1 or (shape[1] > 1 and stride[1] != head_dim):
        raise NativeError(f"{what}: the heads of a row of {name} must be contiguous")
    return stride[0] if rows > 1 else shape[1] * head_dim


def _common(what: str, ctx, cache: PagedCache, seqs: Sequences, rows: int, dtype) -> int:
    code = _MODEL_DTYPES.get(dtype)
    if code is None:
        raise NativeError(f"{what}: rows of {dtype} (bfloat16 or float16)")
    if cache.desc.kind == native.CACHE_MODEL and cache.dtype != dtype:
        raise NativeError(f"{what}: rows of {dtype} and pages of {cache.dtype}")
    if rows < 1:
        raise NativeError(f"{what}: no rows")
    return code


def _devices(what: str, ctx, cache: PagedCache, seqs: Sequences, **tensors) -> None:
    """Raises for what is not on the context's device."""
    device = torch.device("cuda", ctx.device)
    _same_device(what, device, cache=cache, sequences=seqs, **tensors)


def _table(what: str, name: str, t: torch.Tensor | None, rows: int) -> int:
    if t is None:
        return 0
    if t.dtype != torch.int32 or t.dim() != 1 or t.shape[0] != rows or (rows > 1 and t.stride(0) != 1):
        raise NativeError(f"{what}: {name} is contiguous int32 [{rows}]")
    return t.data_ptr()


def _output(like: torch.Tensor, stream) -> torch.Tensor:
    """An output tensor owned by the stream that writes it."""
    if stream is None:
        return torch.empty(like.shape, dtype=like.dtype, device=like.device)
    with torch.cuda.stream(stream):
        return torch.empty(like.shape, dtype=like.dtype, device=like.device)


def _scratch(size: int, device: torch.device, stream) -> torch.Tensor:
    """Bytes for one call, from the allocator of the stream that it runs on (a captured call's from its graph's pool)."""
    if stream is None:
        return torch.empty(size, dtype=torch.uint8, device=device)
    with torch.cuda.stream(stream):
        return torch.empty(size, dtype=torch.uint8, device=device)


def append(ctx: native.Context, cache: PagedCache, seqs: Sequences, k: torch.Tensor, v: torch.Tensor, *,
           q: torch.Tensor | None = None, q_out: torch.Tensor | None = None, cos_sin: torch.Tensor | None = None,
           positions: torch.Tensor | None = None, stream=None) -> torch.Tensor | None:
    """Rotates the rows' ``q`` and ``k`` by ``cos_sin`` ([max_pos, head_dim]: cos | sin, as ``rope_cache`` makes it; None:
    no rotation) at ``positions`` (int32 [rows]; None: the logical indices) and writes ``k`` and ``v`` into the pages.

    ``q`` [rows, heads, head_dim], ``k`` and ``v`` [rows, kv_heads, head_dim] may be slices of one projection's rows.
    Returns the rotated queries: ``q_out`` (``q`` itself is allowed), or a new tensor. Rows that no sequence holds are not
    written, and a row whose position ``cos_sin`` does not have is recorded and left out, key and value too. e4m3 pages:
    the call sets the scales of the blocks it begins and raises those it continues, bringing the tokens before its own to
    the new scale; tokens behind the appended ones in a block are no longer valid."""
    what = "cache.append"
    rows, hd = k.shape[0], cache.head_dim
    dtype = k.dtype
    code = _common(what, ctx, cache, seqs, rows, dtype)
    k_stride = _heads(what, "k", k, rows, cache.num_kv_heads, hd, dtype)
    v_stride = _heads(what, "v", v, rows, cache.num_kv_heads, hd, dtype)
    heads = q_stride = q_out_stride = q_ptr = q_out_ptr = cos_ptr = max_pos = 0
    if q is not None:
        q_stride = _heads(what, "q", q, rows, None, hd, dtype)
        heads = q.shape[1]
        q_out_stride = heads * hd if q_out is None else _heads(what, "q_out", q_out, rows, heads, hd, dtype)
    elif q_out is not None:
        raise NativeError(f"{what}: q_out without q")
    if cos_sin is not None:
        if cos_sin.dtype != dtype or cos_sin.dim() != 2 or cos_sin.shape[1] != hd or not cos_sin.is_contiguous() or \
                cos_sin.shape[0] < 1:
            raise NativeError(f"{what}: cos_sin is contiguous {dtype} [max_pos, {hd}]")
        cos_ptr, max_pos = cos_sin.data_ptr(), cos_sin.shape[0]
    positions_ptr = _table(what, "positions", positions, rows)
    index = ctx.device
    for t in (cache, seqs, k, v, q, q_out, cos_sin, positions):
        if t is not None and (t._index if t is cache or t is seqs else t.get_device()) != index:
            _devices(what, ctx, cache, seqs, k=k, v=v, q=q, q_out=q_out, cos_sin=cos_sin, positions=positions)
    if q is not None:
        if q_out is None:
            q_out = _output(q, stream)
        q_ptr, q_out_ptr = q.data_ptr(), q_out.data_ptr()
    desc = _APPEND.pack(code, rows, q_ptr, k.data_ptr(), v.data_ptr(), q_stride, k_stride, v_stride, q_out_ptr,
                        q_out_stride, heads, max_pos, cos_ptr, positions_ptr) + cache._bytes + seqs._bytes
    status = _entry("plm_cache_append", [ctypes.c_void_p, ctypes.c_char_p, ctypes.c_void_p])(
        ctx.handle, desc, _raw_stream(index, stream))
    if status:
        native.check(status, "plm_cache_append")
    return q_out


def attention(ctx: native.Context, cache: PagedCache, seqs: Sequences, q: torch.Tensor, *,
              out: torch.Tensor | None = None, scale: float | None = None, window: int = 0, sinks: int = 0,
              depth: torch.Tensor | None = None, own_start: torch.Tensor | None = None, stream=None) -> torch.Tensor:
    """Attention of ``q`` [rows, heads, head_dim] over the sequences' cached keys, the rows' own among them (append
    first): causal, or under the round mask with ``depth`` and ``own_start`` (int32 [rows], as ``round_layout`` gives
    them). With ``window`` a row sees its own position and the ``window - 1`` before it, and the first ``sinks`` tokens.
    ``scale`` defaults to 1 / sqrt(head_dim). Returns ``out``, or a new tensor; rows that no sequence holds are not
    written, and a row that sees no key gets zeros."""
    what = "cache.attention"
    rows, hd = q.shape[0], cache.head_dim
    dtype = q.dtype
    code = _common(what, ctx, cache, seqs, rows, dtype)
    q_stride = _heads(what, "q", q, rows, None, hd, dtype)
    heads = q.shape[1]
    if heads % cache.num_kv_heads:
        raise NativeError(f"{what}: {heads} heads over {cache.num_kv_heads} kv heads")
    out_stride = _heads(what, "out", out, rows, heads, hd, dtype) if out is not None else heads * hd
    if scale is not None and not 2.0 ** -126 <= scale < 2.0 ** 128:  # an fp32 number; 0 asks for the default
        raise NativeError(f"{what}: scale {scale}")
    if (depth is None) != (own_start is None):
        raise NativeError(f"{what}: depth and own_start go together")
    if not (0 <= window < 1 << 31 and 0 <= sinks < 1 << 31):
        raise NativeError(f"{what}: window {window}, sinks {sinks}")
    depth_ptr, own_ptr = _table(what, "depth", depth, rows), _table(what, "own_start", own_start, rows)
    index = ctx.device
    for t in (cache, seqs, q, out, depth, own_start):
        if t is not None and (t._index if t is cache or t is seqs else t.get_device()) != index:
            _devices(what, ctx, cache, seqs, q=q, out=out, depth=depth, own_start=own_start)
    if out is None:
        out = _output(q, stream)
    fields = (code, rows, q.data_ptr(), q_stride, out.data_ptr(), out_stride, heads, scale or 0.0, window, sinks, depth_ptr,
              own_ptr)
    tail = cache._bytes + seqs._bytes
    sizes = (code, rows, heads, window, sinks, seqs.count, seqs.max_rows, seqs.max_keys, seqs.desc.max_pages)
    size = cache._workspaces.get(sizes)
    if size is None:
        size = _workspace_bytes(ctx, _ATTENTION.pack(*fields, 0, 0) + tail)
        if len(cache._workspaces) >= 256:  # sizes of calls long past
            cache._workspaces.clear()
        cache._workspaces[sizes] = size
    workspace = _scratch(size, q.device, stream) if size else None
    desc = _ATTENTION.pack(*fields, workspace.data_ptr() if size else 0, size) + tail
    status = _entry("plm_cache_attention", [ctypes.c_void_p, ctypes.c_char_p, ctypes.c_void_p])(
        ctx.handle, desc, _raw_stream(index, stream))
    if status:
        native.check(status, "plm_cache_attention")
    return out


def _workspace_bytes(ctx, desc: bytes) -> int:
    size = ctypes.c_int64(0)
    native.check(_entry("plm_cache_attention_workspace", [ctypes.c_void_p, ctypes.c_char_p, ctypes.c_void_p])(
        ctx.handle, desc, ctypes.addressof(size)), "plm_cache_attention_workspace")
    return size.value
