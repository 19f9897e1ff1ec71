"""The paged-cache operators where the host's bounds and the device's lengths are far apart, where a mask leaves a row or a
sequence nothing, and at the ends of their number ranges; against the definitions in 64 bits (cache_reference.py)."""

from __future__ import annotations

import pytest
import torch

from tests.cache_reference import UNREACHABLE, within
from tests.test_cache_ops import PAGES, Setup, _assert_pages, _bits

pytestmark = pytest.mark.gpu


def _int32(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _loose(st, max_keys):
    """The sequences of ``st`` with block tables for ``max_keys`` tokens and that bound (or, given by the tables, none)."""
    from plm import cache as api

    narrow = st.seqs.block_tables
    wide = torch.full((narrow.shape[0], max_keys // st.cache.page_size), -1, dtype=torch.int32, device="cuda")
    wide[:, :narrow.shape[1]] = narrow
    return [api.Sequences(st.seqs.row_start, st.seqs.context, wide, max_rows=st.seqs.max_rows, max_keys=bound)
            for bound in (max_keys, 0)]


@pytest.fixture(params=[0xFF, 0x71], ids=["nan", "huge"])
def hostile(request, monkeypatch):
    """Every workspace of a call full of NaN, or of numbers near 1.2e30: what nobody has written shows."""
    from plm import cache as api

    plain = api._scratch

    def scratch(size, device, stream):
        return plain(size, device, stream).fill_(request.param)

    monkeypatch.setattr(api, "_scratch", scratch)


@pytest.mark.parametrize("dtype,e4m3", PAGES)
@pytest.mark.parametrize("rows,context,heads,kv_heads,max_keys,options", [
    ([1], [99], 16, 16, 8192, {}), ([1], [199], 32, 8, 32768, {}), ([1], [16], 1, 1, 8192, {}),
    ([1], [299], 2, 1, 32768, {}), ([1] * 4, [49] * 4, 8, 8, 32768, {}),
    ([1] * 8, [17, 300, 45, 0, 80, 16, 15, 130], 2, 2, 8192, {}),
    ([2] * 3, [250, 17, 60], 16, 2, 8192, {}),                             # 16 packed rows: the wider tile
    ([0] * 31 + [1] + [0] * 32, [511] * 64, 8, 8, 512, {}),                # slots of which one holds a row
    ([1] * 2, [120, 40], 8, 8, 32768, dict(window=4096, sinks=4)),         # contexts short of the window
])
def test_decode_of_keys_far_below_the_bound(ctx, hostile, dtype, e4m3, rows, context, heads, kv_heads, max_keys, options):
    """Fewer chunks of keys than the CTAs that the host's bound calls for: some have nothing to do."""
    from plm import cache as api

    st = Setup(rows=rows, context=context, kv_heads=kv_heads, head_dim=128, page=16, dtype=dtype, e4m3=e4m3,
               seed=len(rows) + heads)
    st.poison_behind()
    q = st.randn(st.total, heads, 128)
    want, bound = st.expected(q, **options)
    for seqs in _loose(st, max_keys):
        assert within(api.attention(ctx, st.cache, seqs, q, **options), want, bound)
    ctx.check()


@pytest.mark.parametrize("e4m3", [False, True])
@pytest.mark.parametrize("rows,heads", [([1], 8), ([1, 2], 4), ([40], 4)])
def test_one_graph_from_short_to_long_and_back(ctx, hostile, e4m3, rows, heads):
    """A graph captured under a large bound serves every length below it."""
    from plm import cache as api

    longest = 2000
    st = Setup(rows=rows, context=[longest] * len(rows), kv_heads=4, head_dim=128, page=16, dtype="bf16", e4m3=e4m3, seed=3)
    q = st.randn(st.total, heads, 128)
    seqs = _loose(st, 32768)[0]
    api.attention(ctx, st.cache, seqs, q)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = api.attention(ctx, st.cache, seqs, q)
    for context in (0, 30, 100, 333, longest, 64, 3):
        st.ctx_host = [max(0, context - 5 * s) for s in range(len(rows))]
        st.seqs.context.copy_(torch.tensor(st.ctx_host, device="cuda"))
        out.fill_(7.0)
        graph.replay()
        ctx.check()
        want, bound = st.expected(q)
        assert within(out, want, bound), context


def test_c_entry_points_with_a_workspace_of_the_callers(ctx):
    """plm.native's functions with descriptors of one's own: a workspace of NaN, and nothing written behind it."""
    from plm import cache as api
    from plm import native

    st = Setup(rows=[1, 1], context=[60, 199], kv_heads=8, head_dim=128, page=16, dtype="bf16", e4m3=True, seed=2)
    q, k, v = st.randn(2, 8, 128), st.randn(2, 8, 128), st.randn(2, 8, 128)
    seqs = _loose(st, 32768)[0]
    model = st.model()
    model.append(st.starts, st.ctx_host, st.tables, k.double().cpu(), v.double().cpu())
    row = 8 * 128
    native.cache_append(ctx, native.CacheAppendDesc(dtype=native.PLM_BF16, rows=2, k=k.data_ptr(), v=v.data_ptr(), k_stride=row,
                                                    v_stride=row, cache=st.cache.desc, seqs=seqs.desc))
    _assert_pages(st.cache, model)
    out = torch.zeros_like(q)
    desc = native.CacheAttentionDesc(dtype=native.PLM_BF16, rows=2, q=q.data_ptr(), q_stride=row, out=out.data_ptr(),
                                     out_stride=row, num_heads=8, cache=st.cache.desc, seqs=seqs.desc)
    size = native.cache_attention_workspace(ctx, desc)
    workspace = torch.full((size + 4096,), 0xFF, dtype=torch.uint8, device="cuda")
    desc.workspace, desc.workspace_bytes = workspace.data_ptr(), size
    native.cache_attention(ctx, desc)
    ctx.check()
    want, bound = st.expected(q)
    assert within(out, want, bound)
    assert (workspace[size:] == 0xFF).all()
    assert torch.equal(_bits(out), _bits(api.attention(ctx, st.cache, seqs, q)))


@pytest.mark.parametrize("e4m3", [False, True])
@pytest.mark.parametrize("rows,context,depth", [
    ([1], [15], 5), ([1], [63], 16), ([4], [12], 1 << 30), ([16], [0], 40), ([40], [8], 300), ([200], [56], 1 << 30),
    ([1, 1, 1], [31, 20, 47], 100), ([3, 2], [13, 62], 70),
    ([1] * 1100, [15] * 1100, 9),                      # more sequences than one even launch takes
])
def test_window_past_every_key_gives_zeros(ctx, e4m3, rows, context, depth):
    """A window that lies behind all keys of a sequence, and no sinks: zeros, also where keys end with a chunk or a tile."""
    from plm import cache as api

    st = Setup(rows=rows, context=context, kv_heads=2, head_dim=128, page=16, dtype="bf16", e4m3=e4m3, seed=rows[0],
               spare_rows=2)
    q = st.randn(st.held, 2, 128)
    out = torch.full_like(q, 7.0)
    api.attention(ctx, st.cache, st.seqs, q, out=out, window=2, depth=_int32([depth] * st.held),
                  own_start=_int32([UNREACHABLE] * st.held))
    ctx.check()
    assert (out[:st.total] == 0).all() and (out[st.total:] == 7.0).all()


@pytest.mark.parametrize("e4m3", [False, True])
def test_window_past_the_keys_of_one_sequence(ctx, e4m3):
    """Beside a sequence whose rows see nothing the others keep their results."""
    from plm import cache as api

    st = Setup(rows=[1, 1, 1], context=[300, 31, 100], kv_heads=2, head_dim=128, page=16, dtype="bf16", e4m3=e4m3, seed=1)
    q = st.randn(3, 2, 128)
    depth, own = _int32([0, 500, 0]), _int32([UNREACHABLE] * 3)
    out = torch.full_like(q, 7.0)
    api.attention(ctx, st.cache, st.seqs, q, out=out, window=64, depth=depth, own_start=own)
    ctx.check()
    want, bound = st.expected(q, window=64, depth=depth, own_start=own)
    assert within(out, want, bound) and (out[1] == 0).all()


@pytest.mark.parametrize("dtype,e4m3", PAGES)
@pytest.mark.parametrize("context,depth,own", [(0, -1, UNREACHABLE), (50, -1, UNREACHABLE), (50, -9, 0), (200, -40, -3),
                                               (15, -1, UNREACHABLE)])
@pytest.mark.parametrize("rows", [[1], [1, 1, 1], [1, 2]])
def test_a_single_row_may_hide_anything(ctx, dtype, e4m3, context, depth, own, rows):
    """One row, which does not see all keys up to its own: what the hidden ones hold stays out of it."""
    from plm import cache as api

    st = Setup(rows=rows, context=[context] * len(rows), kv_heads=2, head_dim=128, page=16, dtype=dtype, e4m3=e4m3, seed=4)
    first = context + depth + 1  # hidden, up to the own block or the row itself
    last = context + (own if own <= 0 else 1)
    for s in range(len(rows)):
        for kv in range(max(first, 0), last):
            p, slot = st.tables[s][kv // 16], kv % 16
            for t in (st.cache.k, st.cache.v):
                if e4m3:
                    t.view(torch.uint8)[p, :, slot] = 0x7F
                else:
                    t[p, :, slot] = float("nan") if kv % 2 else float("inf")
    q = st.randn(st.total, 4, 128)
    depths, owns = _int32([depth] * st.total), _int32([own] * st.total)
    out = api.attention(ctx, st.cache, st.seqs, q, depth=depths, own_start=owns)
    ctx.check()
    want, bound = st.expected(q, depth=depths, own_start=owns)
    assert within(out[0], want[0], bound[0])  # of a sequence's second row the hidden tokens are its first row's
    if context == 0:
        assert (out[0] == 0).all()
    if len(rows) == 3:
        assert within(out, want, bound)


@pytest.mark.parametrize("rows", [1, 30])
@pytest.mark.parametrize("context", [(1 << 63) - 1, (1 << 63) - 30, 1 << 62, (1 << 32) + 60, -(1 << 63)])
def test_context_past_every_number(ctx, rows, context):
    """A context whose sum with the rows passes 64 bits is one that the block table does not hold: skipped and recorded."""
    from plm import cache as api
    from plm.native import NativeError

    st = Setup(rows=[rows] * 3, context=[50, 60, 70], kv_heads=2, head_dim=64, page=16, dtype="bf16", e4m3=True, seed=9)
    q, k, v = st.randn(st.total, 2, 64), st.randn(st.total, 2, 64), st.randn(st.total, 2, 64)
    good = api.attention(ctx, st.cache, st.seqs, q)
    st.seqs.context[1] = context
    out = torch.full_like(q, 7.0)
    api.attention(ctx, st.cache, st.seqs, q, out=out)
    with pytest.raises(NativeError, match="out of range"):
        ctx.check()
    assert torch.equal(_bits(out[:rows]), _bits(good[:rows])) and torch.equal(_bits(out[2 * rows:]), _bits(good[2 * rows:]))
    assert (out[rows:2 * rows] == 7.0).all()
    before = st.cache.k.view(torch.uint8).clone()
    api.append(ctx, st.cache, st.seqs, k, v)
    with pytest.raises(NativeError, match="out of range"):
        ctx.check()
    changed = (st.cache.k.view(torch.uint8) != before).flatten(1).any(dim=1).nonzero().flatten().tolist()
    assert changed and set(changed) <= set(st.tables[0]) | set(st.tables[2])


@pytest.mark.parametrize("dtype,e4m3", PAGES)
@pytest.mark.parametrize("head_dim,block", [(64, 16), (128, 16), (64, 64), (128, 64)])
def test_append_skips_rows_without_a_position(ctx, dtype, e4m3, head_dim, block):
    """A row whose position lies outside the table is recorded and left out: query, key, value, and its say in a scale."""
    from plm import cache as api
    from plm.native import NativeError
    from plm.model import rope_cache

    st = Setup(rows=[30, 70], context=[40, 3], kv_heads=2, head_dim=head_dim, page=64, dtype=dtype, e4m3=e4m3, block=block,
               seed=4)
    cos_sin = rope_cache(head_dim, 50, 10000.0, st.dtype).cuda()
    q, k, v = st.randn(100, 4, head_dim), st.randn(100, 2, head_dim), st.randn(100, 2, head_dim)
    positions = torch.randint(0, 50, (100,), generator=st.g, device="cuda").to(torch.int32)
    bad = [0, 7, 29, 33, 99] + list(range(43, 63))  # the last ones all of a block of 16 tokens (logical 16 .. 31)
    for i, r in enumerate(bad):
        positions[r] = (-1, 50, 1 << 30, -(1 << 31))[i % 4]
        k[r] *= 100.0
        v[r] *= 100.0
    whole = [t.clone() for t in (st.cache.k.view(torch.uint8), st.cache.v.view(torch.uint8))]
    scales = None if not e4m3 else [st.cache.k_scale.clone(), st.cache.v_scale.clone()]
    q_out = torch.full_like(q, 7.0)
    api.append(ctx, st.cache, st.seqs, k, v, q=q, q_out=q_out, cos_sin=cos_sin, positions=positions)
    with pytest.raises(NativeError, match="out of range"):
        ctx.check()
    got = api.PagedCache(*(t.clone() for t in (st.cache.k, st.cache.v, st.cache.k_scale, st.cache.v_scale) if t is not None))
    assert (q_out[bad] == 7.0).all()
    rest = [r for r in range(100) if r not in bad]
    assert not (q_out[rest] == 7.0).all(dim=-1).any()
    places = {}
    for s in range(2):
        for r in range(st.starts[s], st.starts[s + 1]):
            logical = st.ctx_host[s] + r - st.starts[s]
            places[r] = (st.tables[s][logical // 64], logical % 64)
    for plane, was in ((got.k, whole[0]), (got.v, whole[1])):
        plane, was = plane.view(torch.uint8), was.view(torch.uint8)
        for r in bad:
            p, slot = places[r]
            assert torch.equal(plane[p, :, slot], was[p, :, slot])
    # the others as if the bad rows were as small as can be: zeros at a good position
    st.cache.k.view(torch.uint8).copy_(whole[0])
    st.cache.v.view(torch.uint8).copy_(whole[1])
    if e4m3:
        st.cache.k_scale.copy_(scales[0])
        st.cache.v_scale.copy_(scales[1])
    for r in bad:
        positions[r], k[r], v[r] = 0, 0.0, 0.0
    api.append(ctx, st.cache, st.seqs, k, v, q=q, q_out=q_out, cos_sin=cos_sin, positions=positions)
    ctx.check()
    for r in rest:
        p, slot = places[r]
        for a, b in ((got.k, st.cache.k), (got.v, st.cache.v)):
            assert torch.equal(a.view(torch.uint8)[p, :, slot], b.view(torch.uint8)[p, :, slot])
        if e4m3:
            for a, b in ((got.k_scale, st.cache.k_scale), (got.v_scale, st.cache.v_scale)):
                assert torch.equal(a[p, :, slot // block], b[p, :, slot // block])
    if e4m3 and block == 16:  # no row of it: the block is as it was
        p = st.tables[1][0]
        assert torch.equal(got.k_scale[p, :, 1], scales[0][p, :, 1]) and torch.equal(got.v_scale[p, :, 1], scales[1][p, :, 1])


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("rows", [40, 200])
def test_prefill_weights_far_below_the_largest(ctx, dtype, rows):
    """A largest score below 0 and many more than 2^20 below it: their share of the sum is not rounded away."""
    from plm import cache as api

    context = 1024 - rows
    st = Setup(rows=[rows], context=[context], kv_heads=1, head_dim=64, page=16, dtype=dtype, e4m3=False, seed=1)
    for kv in range(context + rows):
        p, slot = st.tables[0][kv // 16], kv % 16
        large = kv % 128 == 0
        st.cache.k[p, 0, slot] = 0.0
        st.cache.k[p, 0, slot, 0] = -2.75 if large else -17.0  # 2^-3.97 and 2^-24.5
        st.cache.v[p, 0, slot] = 0.0 if large else 512.0
    q = torch.zeros(rows, 1, 64, dtype=st.dtype, device="cuda")
    q[:, :, 0] = 1.0
    out = api.attention(ctx, st.cache, st.seqs, q, scale=1.0)
    ctx.check()
    want, bound = st.expected(q, scale=1.0)
    assert within(out, want, bound)


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("rows", [1, 2, 60, 200])
@pytest.mark.parametrize("exponent", [-10, 10, 30, 60, 90, 110])
@pytest.mark.parametrize("context,block,apart", [(300, 16, False), (300, 2, False), (3000, 16, True)],
                         ids=["blocks", "tokens", "halves"])
def test_blocks_of_zeros_beside_large_values(ctx, dtype, rows, exponent, context, block, apart):
    """Keys whose values are all zero, in blocks of the smallest scale, keep their share of the softmax's sum whatever the
    other blocks' scales are: mixed with them, or the older half of a long context (parts of their own)."""
    from plm import cache as api

    if dtype == "f16" and exponent > 6:
        exponent = 6  # the output has to hold the result
    st = Setup(rows=[rows], context=[context], kv_heads=2, head_dim=128, page=16, dtype=dtype, e4m3=True, block=block,
               seed=rows)
    st.cache.k_scale.fill_(2.0 ** -7)
    g = torch.Generator(device="cuda").manual_seed(2)
    zero = torch.rand(st.cache.v_scale.shape, generator=g, device="cuda") < 0.5
    if apart:
        zero[:] = False
        zero[st.tables[0][:context // 32]] = True
    st.cache.v_scale.copy_(torch.where(zero, 2.0 ** -100, 2.0 ** exponent))
    st.cache.v.view(torch.uint8).masked_fill_(zero.repeat_interleave(block, dim=2)[..., None], 0)
    q = st.randn(rows, 4, 128, scale=2.0)
    out = api.attention(ctx, st.cache, st.seqs, q)
    ctx.check()
    want, bound = st.expected(q)
    assert within(out, want, bound)


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("rows", [40, 200])
@pytest.mark.parametrize("ratio", [0, 3, 8, 11, 15])
def test_prefill_weights_beside_smaller_values(ctx, dtype, rows, ratio):
    """Few keys with the largest scores by far and values of a scale 2^-ratio: weights are rounded relative to the largest
    term, score and scale together, also where a tile's codes are brought to one scale."""
    from plm import cache as api

    context = 1024 - rows
    st = Setup(rows=[rows], context=[context], kv_heads=1, head_dim=64, page=16, dtype=dtype, e4m3=True, seed=1)
    st.cache.k_scale.fill_(0.125)
    st.cache.v_scale.fill_(1.0)
    for s in (st.cache.k, st.cache.v):
        s.view(torch.uint8).zero_()
    for kv in range(context + rows):
        p, slot = st.tables[0][kv // 16], kv % 16
        large = kv % 128 == 16
        if large:
            st.cache.v_scale[p] = 2.0 ** -ratio
        st.cache.v[p, 0, slot, :32] = torch.full((32,), 0.0 if large else 120.0, device="cuda").to(torch.float8_e4m3fn)
        if not large:
            st.cache.k[p, 0, slot, :1] = torch.full((1,), -144.0, device="cuda").to(torch.float8_e4m3fn)
    q = torch.zeros(rows, 1, 64, dtype=st.dtype, device="cuda")
    q[:, :, 0] = 1.0  # scores of 0 and of -18, 2^-26
    out = api.attention(ctx, st.cache, st.seqs, q, scale=1.0)
    ctx.check()
    want, bound = st.expected(q, scale=1.0)
    assert within(out, want, bound)
