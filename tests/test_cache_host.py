"""The paged-cache operators without a GPU: struct layouts, and every refusal of plm.cache and of the C entry points
(whose checks come before anything of the context or the device is touched)."""

from __future__ import annotations

import ctypes
import subprocess
from pathlib import Path

import pytest
import torch

from plm import cache as api
from plm import native
from plm.native import NativeError

HEADER = Path(__file__).resolve().parent.parent / "include" / "plm_native.h"
MIRRORS = {"plm_paged_cache": native.PagedCacheDesc, "plm_sequences": native.SequencesDesc,
           "plm_cache_append_desc": native.CacheAppendDesc, "plm_cache_attention_desc": native.CacheAttentionDesc}


def test_structs_match_c_layout(tmp_path):
    lines = ["#include <stdio.h>", "#include <stddef.h>", f'#include "{HEADER}"', "int main(void) {"]
    for struct, mirror in MIRRORS.items():
        lines.append(f'  printf("{struct} %zu\\n", sizeof({struct}));')
        lines += [f'  printf("{struct}.{f} %zu\\n", offsetof({struct}, {f}));' for f, _ in mirror._fields_]
    (tmp_path / "layout.c").write_text("\n".join(lines + ["  return 0; }"]))
    subprocess.run(["gcc", "-o", str(tmp_path / "layout"), str(tmp_path / "layout.c")], check=True)
    text = subprocess.run([str(tmp_path / "layout")], capture_output=True, text=True, check=True).stdout
    sizes = dict(line.rsplit(" ", 1) for line in text.splitlines())
    for struct, mirror in MIRRORS.items():
        assert int(sizes[struct]) == ctypes.sizeof(mirror)
        for field, _ in mirror._fields_:
            assert int(sizes[f"{struct}.{field}"]) == getattr(mirror, field).offset, f"{struct}.{field}"


def test_packed_descriptors_match_ctypes():
    """plm.cache packs a call's own fields in front of the bytes of its cache and sequences."""
    for pack, desc in ((api._APPEND, native.CacheAppendDesc), (api._ATTENTION, native.CacheAttentionDesc)):
        own = [f for f, _ in desc._fields_ if f not in ("cache", "seqs")]
        assert pack.size == desc.cache.offset
        assert desc.seqs.offset == desc.cache.offset + ctypes.sizeof(native.PagedCacheDesc)
        assert ctypes.sizeof(desc) == desc.seqs.offset + ctypes.sizeof(native.SequencesDesc)
        values = list(range(1, len(own) + 1))
        filled = desc.from_buffer_copy(pack.pack(*values) + bytes(ctypes.sizeof(desc) - pack.size))
        assert [getattr(filled, f) for f in own] == values


def _cache(dtype=torch.bfloat16, **kw):
    return api.PagedCache.allocate(4, 2, kw.pop("page", 16), kw.pop("head_dim", 64), dtype=dtype, device="cpu", **kw)


def _seqs(n=1, pages=4, **kw):
    return api.Sequences(torch.zeros(n + 1, dtype=torch.int32), torch.zeros(n, dtype=torch.int64),
                         torch.zeros(n, pages, dtype=torch.int32), **{"max_rows": 1, **kw})


def test_cache_refusals():
    z = lambda *s, dtype=torch.bfloat16: torch.zeros(*s, dtype=dtype)  # noqa: E731
    scale = torch.ones(4, 2, 1)
    codes = torch.zeros(4, 2, 16, 64, dtype=torch.uint8).view(torch.float8_e4m3fn)
    for k, v, ks, vs in [
        (z(4, 2, 16), z(4, 2, 16), None, None), (z(4, 2, 16, 64), z(4, 2, 16, 128), None, None),
        (z(4, 2, 16, 64), z(4, 2, 16, 64, dtype=torch.float16), None, None),
        (z(4, 2, 16, 64, dtype=torch.float32),) * 2 + (None, None), (z(4, 2, 64, 16).transpose(2, 3),) * 2 + (None, None),
        (z(4, 2, 16, 64), z(4, 2, 16, 64), scale, scale), (codes, codes, None, None), (codes, codes, scale, None),
        (codes, codes, scale.double(), scale), (codes, codes, scale, torch.ones(4, 2, 2)),
        (codes, codes, torch.ones(4, 2, 3), torch.ones(4, 2, 3)), (codes, codes, torch.ones(4, 1, 1), torch.ones(4, 1, 1)),
    ]:
        with pytest.raises(NativeError):
            api.PagedCache(k, v, ks, vs)
    for block in (0, 3, 32, 128):
        with pytest.raises(NativeError):
            _cache("e4m3", scale_block=block)
    assert _cache("e4m3", scale_block=8).scale_block == 8


def test_sequences_refusals():
    i32, i64 = torch.int32, torch.int64
    good = dict(row_start=torch.zeros(3, dtype=i32), context=torch.zeros(2, dtype=i64),
                block_tables=torch.zeros(2, 4, dtype=i32))
    api.Sequences(**good, max_rows=1)
    for change in (dict(row_start=torch.zeros(2, dtype=i32)), dict(row_start=torch.zeros(3, dtype=i64)),
                   dict(context=torch.zeros(2, dtype=i32)), dict(block_tables=torch.zeros(2, 4, dtype=i64)),
                   dict(block_tables=torch.zeros(1, 4, dtype=i32)), dict(block_tables=torch.zeros(4, 2, dtype=i32).T),
                   dict(block_tables=torch.zeros(2, 0, dtype=i32)), dict(row_start=torch.zeros(6, dtype=i32)[::2])):
        with pytest.raises(NativeError):
            api.Sequences(**{**good, **change}, max_rows=1)
    with pytest.raises(NativeError):
        api.Sequences(**good, max_rows=0)
    with pytest.raises(NativeError):
        api.Sequences(**good, max_rows=1, max_keys=-1)


class _NoContext:
    device = 0
    handle = None


def test_append_refusals():
    ctx, cache, seqs = _NoContext(), _cache(), _seqs()
    z = lambda *s, dtype=torch.bfloat16: torch.zeros(*s, dtype=dtype)  # noqa: E731
    k = z(3, 2, 64)
    for kwargs in (dict(k=z(3, 2, 128), v=k), dict(k=k, v=z(2, 2, 64)), dict(k=z(3, 1, 64), v=k),
                   dict(k=k, v=z(3, 2, 64, dtype=torch.float16)), dict(k=z(3, 64, 2).transpose(1, 2), v=k),
                   dict(k=z(3, 2, 64, dtype=torch.float32), v=k), dict(k=z(3, 2, 64, dtype=torch.float16), v=k),
                   dict(k=z(0, 2, 64), v=z(0, 2, 64)), dict(k=k, v=k, q=z(2, 4, 64)), dict(k=k, v=k, q_out=z(3, 4, 64)),
                   dict(k=k, v=k, q=z(3, 4, 64), q_out=z(3, 2, 64)), dict(k=k, v=k, cos_sin=z(10, 128)),
                   dict(k=k, v=k, cos_sin=z(10, 64, dtype=torch.float32)),
                   dict(k=k, v=k, positions=torch.zeros(2, dtype=torch.int32)),
                   dict(k=k, v=k, positions=torch.zeros(3, dtype=torch.int64))):
        with pytest.raises(NativeError):
            api.append(ctx, cache, seqs, **kwargs)
    with pytest.raises(NativeError, match="is on cpu"):
        api.append(ctx, cache, seqs, k, k)


def test_attention_refusals():
    ctx, cache, seqs = _NoContext(), _cache(), _seqs()
    z = lambda *s, dtype=torch.bfloat16: torch.zeros(*s, dtype=dtype)  # noqa: E731
    q, t = z(3, 4, 64), torch.zeros(3, dtype=torch.int32)
    for kwargs in (dict(q=z(3, 3, 64)), dict(q=z(3, 4, 128)), dict(q=z(3, 4, 64, dtype=torch.float16)),
                   dict(q=z(3, 256)), dict(q=z(0, 4, 64)), dict(q=q, out=z(3, 2, 64)), dict(q=q, out=z(2, 4, 64)),
                   dict(q=q, scale=0.0), dict(q=q, scale=float("nan")), dict(q=q, scale=float("inf")),
                   dict(q=q, window=-1), dict(q=q, sinks=1 << 31), dict(q=q, depth=t), dict(q=q, own_start=t), dict(q=q, depth=t.long(), own_start=t),
                   dict(q=q, depth=t[:2], own_start=t[:2])):
        with pytest.raises(NativeError):
            api.attention(ctx, cache, seqs, **kwargs)
    with pytest.raises(NativeError, match="is on cpu"):
        api.attention(ctx, cache, seqs, q)


def test_what_would_pass_for_a_default_is_refused():
    """Numbers that become 0 in their C type, and empty tensors, whose address is null: neither stands for "none"."""
    ctx, cache, seqs = _NoContext(), _cache(), _seqs()
    z = lambda *s: torch.zeros(*s, dtype=torch.bfloat16)  # noqa: E731
    k = z(3, 2, 64)
    for scale in (1e-50, 1e39):
        with pytest.raises(NativeError, match="scale"):
            api.attention(ctx, cache, seqs, z(3, 4, 64), scale=scale)
    with pytest.raises(NativeError, match="cos_sin"):
        api.append(ctx, cache, seqs, k, k, cos_sin=z(0, 64))
    with pytest.raises(NativeError, match="no heads"):
        api.append(ctx, cache, seqs, k, k, q=z(3, 0, 64))
    with pytest.raises(NativeError, match="no heads"):
        api.attention(ctx, cache, seqs, z(3, 0, 64))
    with pytest.raises(NativeError, match="at most"):
        _seqs(max_rows=(1 << 32) + 1)
    with pytest.raises(NativeError, match="pages of"):
        api.PagedCache(z(4, 0, 16, 64), z(4, 0, 16, 64))


# ---- the C entry points: a zeroed block stands for the context, which no refusal reads
_BLOCK = ctypes.create_string_buffer(512)
A = 1 << 20  # some 16-byte aligned address


def _descs():
    cache = native.PagedCacheDesc(kind=native.CACHE_E4M3, k=A, v=A, k_scale=A, v_scale=A, scale_block=16, num_pages=4,
                                  page_size=16, num_kv_heads=2, head_dim=64)
    seqs = native.SequencesDesc(n_seqs=1, max_rows=1, max_keys=64, row_start=A, context=A, block_tables=A,
                                table_stride=4, max_pages=4)
    append = native.CacheAppendDesc(dtype=0, rows=1, q=A, k=A, v=A, q_stride=256, k_stride=128, v_stride=128, q_out=A,
                                    q_out_stride=256, num_heads=4, max_pos=8, cos_sin=A, cache=cache, seqs=seqs)
    attend = native.CacheAttentionDesc(dtype=0, rows=1, q=A, q_stride=256, out=A, out_stride=256, num_heads=4,
                                       cache=cache, seqs=seqs)
    return append, attend


SHARED = [("dtype", 2), ("rows", 0), ("rows", 1 << 25), ("cache.kind", 2), ("cache.k", None), ("cache.v", A + 8),
          ("cache.k_scale", None), ("cache.v_scale", None), ("cache.scale_block", 0), ("cache.scale_block", 12),
          ("cache.scale_block", 32), ("cache.num_pages", 0), ("cache.page_size", 24), ("cache.page_size", 8192),
          ("cache.page_size", 0), ("cache.num_kv_heads", 0), ("cache.head_dim", 96), ("seqs.n_seqs", 0),
          ("seqs.n_seqs", 65536), ("seqs.max_rows", 0), ("seqs.row_start", None), ("seqs.context", None),
          ("seqs.block_tables", None), ("seqs.max_pages", 0), ("seqs.table_stride", 3), ("seqs.max_pages", 1 << 27)]
APPEND = [("k", None), ("v", A + 4), ("k_stride", 64), ("v_stride", 132), ("q_stride", 128), ("q_out", None),
          ("q_out_stride", 250), ("num_heads", 0), ("cos_sin", A + 2), ("max_pos", 0), ("q", A + 2)]
ATTEND = [("q", None), ("out", None), ("q", A + 2), ("out_stride", 100), ("q_stride", 260), ("num_heads", 3),
          ("num_heads", 0), ("window", -1), ("sinks", -1), ("scale", -1.0), ("scale", float("nan")),
          ("scale", float("inf")), ("depth", A), ("own_start", A)]


@pytest.mark.parametrize("call,field,value", [("append", f, v) for f, v in SHARED + APPEND] +
                         [("attend", f, v) for f, v in SHARED + ATTEND])
def test_c_entry_points_refuse(call, field, value):
    append, attend = _descs()
    desc = append if call == "append" else attend
    at, name = desc, field
    if "." in field:
        part, name = field.split(".")
        at = getattr(desc, part)
    setattr(at, name, value)
    fn = native.library().plm_cache_append if call == "append" else native.library().plm_cache_attention
    assert fn(ctypes.addressof(_BLOCK), ctypes.byref(desc), None) in (-1, -4)
    assert native.last_error().startswith("plm_cache_")


def test_c_entry_points_refuse_null():
    append, attend = _descs()
    lib = native.library()
    assert lib.plm_cache_append(None, ctypes.byref(append), None) == -1
    assert lib.plm_cache_attention(None, ctypes.byref(attend), None) == -1
    assert lib.plm_cache_append(ctypes.addressof(_BLOCK), None, None) == -1
    assert lib.plm_cache_attention(ctypes.addressof(_BLOCK), None, None) == -1
    assert lib.plm_cache_attention_workspace(None, ctypes.byref(attend), ctypes.byref(ctypes.c_int64())) == -1
    assert lib.plm_cache_attention_workspace(ctypes.addressof(_BLOCK), ctypes.byref(attend), None) == -1


def test_c_attention_refuses_a_missing_workspace():
    """A call that has to share out its keys needs scratch of its own; a block of zeros has no SMs, and so one worker."""
    _, attend = _descs()
    lib, needed = native.library(), ctypes.c_int64(0)
    assert lib.plm_cache_attention_workspace(ctypes.addressof(_BLOCK), ctypes.byref(attend), ctypes.byref(needed)) == 0
    assert needed.value > 0
    for workspace, size in ((None, 1 << 30), (A, needed.value - 1), (A + 4, 1 << 30)):
        attend.workspace, attend.workspace_bytes = workspace, size
        assert lib.plm_cache_attention(ctypes.addressof(_BLOCK), ctypes.byref(attend), None) == -1
        assert "workspace" in native.last_error()
