"""plm_cache_append and plm_cache_attention on the GPU against their definitions in 64 bits (cache_reference.py).

Appending rounds every value once: rotated values are exact products rounded to fp32 and then to their storage type, so
16-bit pages agree bit for bit and e4m3 codes and scales too (a value whose 64-bit sum rounds differently through fp32
is rounded through fp32 by the reference as well). Attention is held to the bound that ``attend`` derives.
"""

from __future__ import annotations

import pytest
import torch

from tests.cache_reference import CacheModel, attend, visible, within

pytestmark = pytest.mark.gpu

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16}


class Setup:
    """Random pages, block tables and sequences. Pages of the pool that no sequence owns are filled with NaN."""

    def __init__(self, *, rows, context, kv_heads, head_dim, page, dtype, e4m3, block=16, seed=0, spare_rows=0,
                 spread=1.0):
        from plm import cache as api

        block = min(block, page)
        g = torch.Generator(device="cuda").manual_seed(seed)
        self.rows, self.ctx_host, self.dtype = rows, context, DTYPES[dtype]
        need = [max(1, -(-(n + c) // page)) for n, c in zip(rows, context)]
        pages = sum(need) + 3
        perm = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)
        tables = torch.full((len(rows), max(need)), -1, dtype=torch.int32, device="cuda")
        at = 0
        for s, n in enumerate(need):
            tables[s, :n] = perm[at:at + n]
            at += n
        spare = perm[at:].long()
        self.starts = [0]
        for n in rows:
            self.starts.append(self.starts[-1] + n)
        self.total = self.starts[-1]
        self.held = self.total + spare_rows
        shape = (pages, kv_heads, page, head_dim)
        x = [torch.randn(shape, generator=g, device="cuda") for _ in range(2)]
        if e4m3:
            scales = [torch.exp2(torch.randint(-9, -5, (pages, kv_heads, page // block), generator=g, device="cuda")
                                 .float() * spread) for _ in range(2)]
            pages_kv = [(t * 100).to(torch.float8_e4m3fn) for t in x]
            for t in pages_kv:
                t.view(torch.uint8)[spare] = 0x7F  # NaN
            self.cache = api.PagedCache(*pages_kv, *scales)
        else:
            pages_kv = [t.to(self.dtype) for t in x]
            for t in pages_kv:
                t[spare] = float("nan")
            self.cache = api.PagedCache(*pages_kv)
        self.seqs = api.Sequences(torch.tensor(self.starts, dtype=torch.int32, device="cuda"),
                                  torch.tensor(context, dtype=torch.int64, device="cuda"), tables,
                                  max_rows=max(max(rows), 1),
                                  max_keys=max(n + c for n, c in zip(rows, context)))
        self.tables = tables.tolist()
        self.g = g

    def model(self):
        c = self.cache
        return CacheModel(c.k, c.v, c.k_scale, c.v_scale)

    def randn(self, *shape, scale=1.0):
        return (torch.randn(*shape, generator=self.g, device="cuda") * scale).to(self.dtype)

    def poison_behind(self):
        """NaN in the slots behind every sequence's last key (stale or never written)."""
        page = self.cache.page_size
        for s, (n, c) in enumerate(zip(self.rows, self.ctx_host)):
            last = n + c
            if last % page:
                for t in (self.cache.k, self.cache.v):
                    p, slot = self.tables[s][last // page], last % page
                    if t.dtype == torch.float8_e4m3fn:
                        t.view(torch.uint8)[p, :, slot:] = 0x7F
                    else:
                        t[p, :, slot:] = float("nan")

    def expected(self, q, *, window=0, sinks=0, depth=None, own_start=None, scale=None):
        model = self.model()
        outs, bounds = [], []
        for s, (n, c) in enumerate(zip(self.rows, self.ctx_host)):
            if n == 0:
                continue
            lo, hi = self.starts[s], self.starts[s + 1]
            k, v, vs = model.dense(self.tables[s], n + c)
            mask = visible(n, c, window, sinks, None if depth is None else depth[lo:hi].tolist(),
                           None if own_start is None else own_start[lo:hi].tolist())
            out, bound = attend(q[lo:hi].double().cpu(), k, v, vs, mask, self.dtype, scale)
            outs.append(out)
            bounds.append(bound)
        return torch.cat(outs), torch.cat(bounds)


def _bits(x):
    return x.view(torch.int16)


def _check_attention(ctx, st, heads, **options):
    from plm import cache as api

    hd = st.cache.head_dim
    q = st.randn(st.held, heads, hd)
    out = torch.full((st.held, heads, hd), 7.0, dtype=st.dtype, device="cuda")
    got = api.attention(ctx, st.cache, st.seqs, q, out=out, **options)
    ctx.check()
    assert got is out
    assert (out[st.total:] == 7.0).all(), "rows behind the last sequence were written"
    want, bound = st.expected(q, **options)
    assert within(out[:st.total], want, bound)
    return q, out


PAGES = [pytest.param("bf16", False, id="bf16"), pytest.param("f16", False, id="f16"),
         pytest.param("bf16", True, id="e4m3-bf16"), pytest.param("f16", True, id="e4m3-f16")]


@pytest.mark.parametrize("dtype,e4m3", PAGES)
@pytest.mark.parametrize("rows,context,heads,kv_heads,head_dim,page", [
    ([1], [0], 16, 16, 128, 16),                      # the first token of a sequence
    ([1], [1], 8, 8, 64, 16),
    ([1], [1023], 16, 16, 128, 16),
    ([1], [2047], 8, 2, 128, 64),
    ([1, 1, 1, 1, 1], [0, 15, 16, 700, 63], 14, 2, 128, 16),   # a group of 7
    ([1] * 33, list(range(0, 330, 10)), 8, 8, 64, 16),
    ([2, 0, 5, 1], [30, 40, 3, 0], 4, 4, 128, 16),    # a sequence without rows
    ([17], [100], 4, 4, 128, 16),
    ([56], [333], 16, 16, 128, 16),
    ([127], [0], 4, 4, 128, 32),
    ([128], [128], 4, 2, 128, 64),
    ([129], [511], 6, 2, 64, 16),
    ([300], [77], 4, 1, 128, 16),
    ([513, 1, 40], [0, 600, 129], 4, 2, 64, 32),
    ([1, 2], [77, 30], 2, 1, 128, 1), ([40, 3], [20, 130], 2, 1, 64, 1), ([1], [300], 2, 2, 64, 8),
    ([140], [9], 2, 2, 128, 4), ([30, 1], [5000, 4100], 2, 1, 128, 4096),
    ([20] * 40, list(range(0, 400, 10)), 2, 2, 64, 16),        # more sequences than a warp has lanes
    ([300] * 3, [1500, 0, 700], 16, 2, 128, 64),               # many units of a group of 8
])
def test_attention_causal(ctx, dtype, e4m3, rows, context, heads, kv_heads, head_dim, page):
    st = Setup(rows=rows, context=context, kv_heads=kv_heads, head_dim=head_dim, page=page, dtype=dtype, e4m3=e4m3,
               seed=len(rows) + rows[0], spare_rows=3)
    st.poison_behind()
    _check_attention(ctx, st, heads)


@pytest.mark.parametrize("dtype,e4m3", PAGES)
@pytest.mark.parametrize("rows,context,window,sinks", [
    ([1], [0], 1, 0), ([1], [500], 1, 0), ([1], [500], 64, 4), ([1], [1000], 333, 130), ([1], [200], 1000, 4),
    ([1], [900], 100, 2000),                          # sinks past the context: everything is visible
    ([40], [0], 7, 3), ([200], [300], 64, 1), ([300], [0], 128, 0), ([260], [500], 130, 65),
    ([1, 33, 1, 2], [700, 10, 0, 129], 50, 5),
])
def test_attention_window(ctx, dtype, e4m3, rows, context, window, sinks):
    st = Setup(rows=rows, context=context, kv_heads=2, head_dim=128, page=16, dtype=dtype, e4m3=e4m3, seed=window)
    st.poison_behind()
    _check_attention(ctx, st, 4, window=window, sinks=sinks)


@pytest.mark.parametrize("dtype,e4m3", PAGES)
@pytest.mark.parametrize("k,context,heads,kv_heads,window,sinks", [
    (7, 1000, 16, 16, 0, 0), (4, 0, 8, 8, 0, 0), (6, 333, 8, 2, 0, 0), (8, 2050, 4, 4, 0, 0), (7, 700, 4, 4, 100, 4),
    (4, 5, 4, 2, 3, 1), (12, 250, 4, 4, 0, 0),
])
def test_attention_round_mask(ctx, dtype, e4m3, k, context, heads, kv_heads, window, sinks):
    from plm.mask import round_layout

    _, _, depth, own_start = round_layout([k] * k)
    st = Setup(rows=[len(depth)], context=[context], kv_heads=kv_heads, head_dim=128, page=16, dtype=dtype, e4m3=e4m3,
               seed=k)
    st.poison_behind()
    _check_attention(ctx, st, heads, window=window, sinks=sinks, depth=depth.to(torch.int32).cuda(),
                     own_start=own_start.to(torch.int32).cuda())


@pytest.mark.parametrize("dtype,e4m3", PAGES)
@pytest.mark.parametrize("rows", [3, 40, 200])
def test_attention_rows_that_see_nothing(ctx, dtype, e4m3, rows):
    """depth -1 and no own block on an empty context: zeros, whatever the pages hold."""
    st = Setup(rows=[rows], context=[0], kv_heads=2, head_dim=128, page=16, dtype=dtype, e4m3=e4m3, seed=rows)
    depth = torch.arange(rows, dtype=torch.int32, device="cuda")
    depth[::2] = -1
    own = torch.full((rows,), 1 << 30, dtype=torch.int32, device="cuda")
    _, out = _check_attention(ctx, st, 2, depth=depth, own_start=own)
    assert (out[:rows:2] == 0).all()


@pytest.mark.parametrize("dtype,e4m3", PAGES)
@pytest.mark.parametrize("rows,context", [([5], [90]), ([40], [20]), ([150], [100]), ([300], [10])])
def test_attention_masked_tokens_may_hold_anything(ctx, dtype, e4m3, rows, context):
    """NaN and infinities in tokens that some rows see and others do not: only the rows that see them take them over."""
    n, c = rows[0], context[0]
    st = Setup(rows=rows, context=context, kv_heads=2, head_dim=128, page=16, dtype=dtype, e4m3=e4m3, seed=n + 1)
    for back, bad in ((1, "nan"), (n // 3, "inf"), (n // 2, "-inf")):
        kv = c + n - back - 1
        p, slot = st.tables[0][kv // 16], kv % 16
        if e4m3:
            st.cache.v.view(torch.uint8)[p, :, slot, back % 100] = 0x7F
        else:
            st.cache.v[p, :, slot, back % 100] = float(bad)
    last = c + n - 1
    key = st.cache.k.view(torch.uint8) if e4m3 else st.cache.k
    key[st.tables[0][last // 16], 0, last % 16, 3] = 0x7F if e4m3 else float("nan")
    q, out = _check_attention(ctx, st, 2)
    assert torch.isfinite(out[:n // 3]).all()
    assert torch.isnan(out[n - 1, 0]).all()


@pytest.mark.parametrize("e4m3", [False, True])
def test_attention_many_sequences(ctx, e4m3):
    """More sequences than one even launch takes: every tile a CTA of its own."""
    from plm import cache as api

    n = 1100
    st = Setup(rows=[1, 0] * (n // 2), context=[(7 * i) % 90 for i in range(n)], kv_heads=1, head_dim=64, page=16,
               dtype="bf16", e4m3=e4m3, seed=n)
    q = st.randn(st.held, 2, 64)
    out = api.attention(ctx, st.cache, st.seqs, q)
    ctx.check()
    want, bound = st.expected(q)
    assert within(out, want, bound)


@pytest.mark.parametrize("rows", [3, 40, 200])
def test_attention_positions_far_ahead(ctx, rows):
    """A depth far past the keys moves the window behind all of them: the sinks alone stay visible."""
    st = Setup(rows=[rows], context=[50], kv_heads=2, head_dim=128, page=16, dtype="bf16", e4m3=False, seed=rows)
    depth = torch.full((rows,), 1 << 30, dtype=torch.int32, device="cuda")
    own = torch.full((rows,), 1 << 30, dtype=torch.int32, device="cuda")
    _check_attention(ctx, st, 2, window=10, sinks=(1 << 31) - 1, depth=depth, own_start=own)
    _check_attention(ctx, st, 2, window=10, sinks=3, depth=depth, own_start=own)


@pytest.mark.parametrize("rows", [1, 60, 200])
def test_attention_scales_far_apart(ctx, rows):
    """Scales of a sequence's blocks over 2^50: the weights' rounding stays relative to the largest term."""
    st = Setup(rows=[rows], context=[300], kv_heads=2, head_dim=128, page=16, dtype="bf16", e4m3=True, seed=3)
    st.cache.k_scale.fill_(2.0 ** -7)
    g = torch.Generator(device="cuda").manual_seed(5)
    st.cache.v_scale.copy_(torch.exp2(torch.randint(-60, -10, st.cache.v_scale.shape, generator=g, device="cuda").float()))
    _check_attention(ctx, st, 2)
    # and scales that are no powers of two
    st.cache.v_scale.uniform_(0.001, 1.0, generator=g)
    st.cache.k_scale.uniform_(0.001, 0.02, generator=g)
    _check_attention(ctx, st, 2)
    # keys' scales alone over 2^40, and both a little apart
    st.cache.v_scale.fill_(2.0 ** -6)
    st.cache.k_scale.copy_(torch.exp2(torch.randint(-48, -7, st.cache.k_scale.shape, generator=g, device="cuda").float()))
    _check_attention(ctx, st, 2)
    st.cache.v_scale.copy_(torch.exp2(torch.randint(-20, -8, st.cache.k_scale.shape, generator=g, device="cuda").float()))
    _check_attention(ctx, st, 2)


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("e4m3", [False, True])
@pytest.mark.parametrize("rows", [1, 40, 200])
def test_attention_large_and_small_queries(ctx, dtype, e4m3, rows):
    """Rows whose queries differ by 2^30 in size (as far as the type holds them), with a score scale to match."""
    from plm import cache as api

    st = Setup(rows=[rows], context=[100], kv_heads=1, head_dim=64, page=16, dtype=dtype, e4m3=e4m3, seed=rows)
    q = st.randn(rows, 2, 64)
    size = 2.0 ** 30 if dtype == "bf16" else 2.0 ** 8
    q[::2] = (q[::2].float() * size).to(st.dtype)
    q[1::2] = (q[1::2].float() / size).to(st.dtype)
    scale = 2.0 ** -33 if dtype == "bf16" else 2.0 ** -11
    out = api.attention(ctx, st.cache, st.seqs, q, scale=scale)
    ctx.check()
    want, bound = st.expected(q, scale=scale)
    assert within(out, want, bound)


def test_attention_window_needs_no_pages_behind_it(ctx):
    """Pages that lie wholly between the sinks and every row's window may be given away (-1 in the block table)."""
    from plm import cache as api

    for e4m3 in (False, True):
        for rows in (1, 20, 200):
            st = Setup(rows=[rows], context=[1000], kv_heads=2, head_dim=128, page=16, dtype="bf16", e4m3=e4m3, seed=6)
            q = st.randn(rows, 4, 128)
            whole = api.attention(ctx, st.cache, st.seqs, q, window=100, sinks=20)
            first = (1000 - 99) // 16  # the page of the first row's first key
            st.seqs.block_tables[0, 2:first] = -1
            assert torch.equal(_bits(api.attention(ctx, st.cache, st.seqs, q, window=100, sinks=20)), _bits(whole))
            ctx.check()


def test_attention_strided_rows_and_streams(ctx):
    """q and out as slices of wider rows, on a stream of the caller's, and replayed from a graph with other lengths."""
    from plm import cache as api

    for e4m3, rows in ((False, [1, 1]), (True, [1, 1]), (False, [33, 60]), (True, [33, 60])):
        st = Setup(rows=rows, context=[90, 200], kv_heads=2, head_dim=128, page=16, dtype="bf16", e4m3=e4m3, seed=8)
        wide = st.randn(st.held, 3, 4, 128)
        q = wide[:, 1]
        plain = api.attention(ctx, st.cache, st.seqs, q.contiguous())
        into = torch.zeros(st.held, 2, 4, 128, dtype=st.dtype, device="cuda")
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        api.attention(ctx, st.cache, st.seqs, q, out=into[:, 1], stream=side)
        fresh = api.attention(ctx, st.cache, st.seqs, q, stream=side)
        torch.cuda.current_stream().wait_stream(side)
        assert torch.equal(_bits(into[:, 1]), _bits(plain)) and torch.equal(_bits(fresh), _bits(plain))
        assert (into[:, 0] == 0).all()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            captured = api.attention(ctx, st.cache, st.seqs, q)
        st.seqs.context.copy_(torch.tensor([70, 150], device="cuda"))
        graph.replay()
        assert torch.equal(_bits(captured), _bits(api.attention(ctx, st.cache, st.seqs, q)))
        st.ctx_host = [70, 150]
        want, bound = st.expected(q)
        assert within(captured, want, bound)
        ctx.check()


def test_attention_device_bounds(ctx):
    """Sequences whose device arrays contradict the host's bounds are skipped and recorded, the others computed."""
    from plm import cache as api
    from plm.native import NativeError

    for rows in ([1, 1, 1], [30, 30, 30]):
        st = Setup(rows=rows, context=[50, 60, 70], kv_heads=2, head_dim=128, page=16, dtype="bf16", e4m3=False, seed=9)
        q = st.randn(st.held, 2, 128)
        good = api.attention(ctx, st.cache, st.seqs, q)
        out = torch.full_like(q, 7.0)
        for bad in (-1, 100000):
            st.seqs.context[1] = bad
            out.fill_(7.0)
            api.attention(ctx, st.cache, st.seqs, q, out=out)
            with pytest.raises(NativeError, match="out of range"):
                ctx.check()
            n = rows[0]
            assert torch.equal(out[:n], good[:n]) and torch.equal(out[2 * n:], good[2 * n:])
            assert (out[n:2 * n] == 7.0).all()
            st.seqs.context[1] = 60
        st.seqs.block_tables[0, 1] = 10000  # a page the pool does not have
        api.attention(ctx, st.cache, st.seqs, q, out=out)
        with pytest.raises(NativeError, match="out of range"):
            ctx.check()


def test_attention_repeats_bit_for_bit(ctx):
    from plm import cache as api

    for rows, context in (([1], [5000]), ([56], [3000]), ([300, 1], [1000, 2000])):
        for e4m3 in (False, True):
            st = Setup(rows=rows, context=context, kv_heads=2, head_dim=128, page=16, dtype="bf16", e4m3=e4m3, seed=10)
            q = st.randn(st.held, 4, 128)
            first = api.attention(ctx, st.cache, st.seqs, q)
            for _ in range(3):
                assert torch.equal(_bits(api.attention(ctx, st.cache, st.seqs, q)), _bits(first))
    ctx.check()


def _cos_sin(head_dim, positions, dtype):
    from plm.model import rope_cache

    return rope_cache(head_dim, positions, 10000.0, dtype).cuda()


def _assert_pages(cache, model):
    assert torch.equal(cache.k.double().cpu().nan_to_num(999.0), model.k.to(cache.dtype).double().nan_to_num(999.0))
    assert torch.equal(cache.v.double().cpu().nan_to_num(999.0), model.v.to(cache.dtype).double().nan_to_num(999.0))
    if cache.k_scale is not None:
        assert torch.equal(cache.k_scale.double().cpu(), model.k_scale)
        assert torch.equal(cache.v_scale.double().cpu(), model.v_scale)


@pytest.mark.parametrize("dtype,e4m3", PAGES)
@pytest.mark.parametrize("rows,context,heads,kv_heads,head_dim,page,block", [
    ([1], [0], 4, 4, 128, 16, 16), ([1], [37], 4, 2, 64, 16, 8), ([56], [100], 4, 4, 128, 16, 16),
    ([1, 0, 7, 1], [15, 3, 30, 64], 6, 2, 128, 32, 32), ([130, 3], [0, 61], 3, 1, 64, 64, 64),
    ([20], [5], 2, 2, 128, 16, 1), ([1] * 40, list(range(40)), 2, 1, 64, 16, 4), ([200], [1000], 2, 1, 128, 128, 64),
])
def test_append(ctx, dtype, e4m3, rows, context, heads, kv_heads, head_dim, page, block):
    from plm import cache as api

    st = Setup(rows=rows, context=context, kv_heads=kv_heads, head_dim=head_dim, page=page, dtype=dtype, e4m3=e4m3,
               block=block, seed=rows[0] + page, spare_rows=5)
    qkv = st.randn(st.held, heads + 2 * kv_heads, head_dim, scale=3.0)
    q, k, v = qkv.split([heads, kv_heads, kv_heads], dim=1)
    v[0, 0] = 0.0
    cos_sin = _cos_sin(head_dim, 1300, st.dtype)
    model = st.model()
    rotated = model.append(st.starts, context, st.tables, k.double().cpu(), v.double().cpu(), q.double().cpu(), cos_sin.cpu())
    q_out = torch.full((st.held, heads, head_dim), 7.0, dtype=st.dtype, device="cuda")
    assert api.append(ctx, st.cache, st.seqs, k, v, q=q, q_out=q_out, cos_sin=cos_sin) is q_out
    ctx.check()
    _assert_pages(st.cache, model)
    want = torch.stack([rotated[r] for r in range(st.total)]).to(st.dtype)
    assert torch.equal(q_out[:st.total].cpu(), want) and (q_out[st.total:] == 7.0).all()


@pytest.mark.parametrize("dtype,e4m3", PAGES)
def test_append_positions_and_no_rotation(ctx, dtype, e4m3):
    from plm import cache as api

    for cos_sin_rows, given in ((500, True), (None, False)):
        st = Setup(rows=[9, 20], context=[40, 3], kv_heads=2, head_dim=64, page=16, dtype=dtype, e4m3=e4m3, seed=4)
        k, v = st.randn(29, 2, 64), st.randn(29, 2, 64)
        cos_sin = None if cos_sin_rows is None else _cos_sin(64, cos_sin_rows, st.dtype)
        positions = torch.randint(0, 500, (29,), generator=st.g, device="cuda").to(torch.int32) if given else None
        model = st.model()
        model.append(st.starts, st.ctx_host, st.tables, k.double().cpu(), v.double().cpu(), None,
                     None if cos_sin is None else cos_sin.cpu(), None if positions is None else positions.tolist())
        assert api.append(ctx, st.cache, st.seqs, k, v, cos_sin=cos_sin, positions=positions) is None
        ctx.check()
        _assert_pages(st.cache, model)


def test_append_extremes(ctx):
    """Infinities saturate at the block's scale, NaN stays NaN, and neither moves the scale; all-zero blocks."""
    from plm import cache as api

    for dtype in (torch.bfloat16, torch.float16):
        name = "bf16" if dtype == torch.bfloat16 else "f16"
        st = Setup(rows=[32], context=[0], kv_heads=2, head_dim=64, page=16, dtype=name, e4m3=True, seed=2)
        k, v = st.randn(32, 2, 64), st.randn(32, 2, 64)
        v[3, 0, 5], v[4, 0, 6], v[5, 1, 7] = float("inf"), float("-inf"), float("nan")
        v[16:, 1] = 0.0
        k[0, 0, 0] = torch.finfo(dtype).max
        k[16:, 0] = torch.finfo(dtype).tiny
        model = st.model()
        model.append(st.starts, [0], st.tables, k.double().cpu(), v.double().cpu())
        api.append(ctx, st.cache, st.seqs, k, v)
        ctx.check()
        _assert_pages(st.cache, model)
        p = st.tables[0][0]
        assert st.cache.v[p, 0, 3, 5].float() == 448 and st.cache.v[p, 0, 4, 6].float() == -448
        assert torch.isnan(st.cache.v[p, 1, 5, 7].float())


def test_append_token_by_token(ctx):
    """Growing values, a token at a time: the block's scale follows them and the older codes with it."""
    from plm import cache as api

    st = Setup(rows=[1, 1], context=[3, 0], kv_heads=2, head_dim=128, page=16, dtype="bf16", e4m3=True, block=8, seed=12)
    model = st.model()
    for step in range(11):
        k, v = st.randn(2, 2, 128, scale=1.5 ** step), st.randn(2, 2, 128, scale=1.7 ** -step)
        context = [3 + step, step]
        st.seqs.context.copy_(torch.tensor(context, device="cuda"))
        model.append(st.starts, context, st.tables, k.double().cpu(), v.double().cpu())
        api.append(ctx, st.cache, st.seqs, k, v)
    ctx.check()
    _assert_pages(st.cache, model)


def test_append_in_place_stream_and_graph(ctx):
    from plm import cache as api

    for e4m3 in (False, True):
        st = Setup(rows=[4, 30], context=[10, 20], kv_heads=2, head_dim=128, page=16, dtype="f16", e4m3=e4m3, seed=13)
        q, k, v = st.randn(34, 4, 128), st.randn(34, 2, 128), st.randn(34, 2, 128)
        cos_sin = _cos_sin(128, 100, st.dtype)
        model = st.model()
        rotated = model.append(st.starts, st.ctx_host, st.tables, k.double().cpu(), v.double().cpu(), q.double().cpu(),
                               cos_sin.cpu())
        side = torch.cuda.Stream()
        graph = torch.cuda.CUDAGraph()
        side.wait_stream(torch.cuda.current_stream())
        into = q.clone()
        with torch.cuda.graph(graph):
            api.append(ctx, st.cache, st.seqs, k, v, q=into, q_out=into, cos_sin=cos_sin)
        graph.replay()
        fresh = api.append(ctx, st.cache, st.seqs, k, v, q=q, cos_sin=cos_sin, stream=side)
        torch.cuda.synchronize()
        ctx.check()
        _assert_pages(st.cache, model)  # twice the same tokens: the same pages
        want = torch.stack([rotated[r] for r in range(34)]).to(st.dtype)
        assert torch.equal(into.cpu(), want) and torch.equal(fresh.cpu(), want)


def test_append_device_bounds(ctx):
    """Bad pages and positions are recorded; the rows of other sequences are written."""
    from plm import cache as api
    from plm.native import NativeError

    for e4m3 in (False, True):
        st = Setup(rows=[2, 2], context=[16, 30], kv_heads=1, head_dim=64, page=16, dtype="bf16", e4m3=e4m3, seed=14)
        k, v = st.randn(4, 1, 64), st.randn(4, 1, 64)
        st.seqs.block_tables[0, 1] = -1
        before = st.cache.k.view(torch.uint8).clone()
        api.append(ctx, st.cache, st.seqs, k, v)
        with pytest.raises(NativeError, match="out of range"):
            ctx.check()
        changed = (st.cache.k.view(torch.uint8) != before).flatten(1).any(dim=1).nonzero().flatten().tolist()
        assert set(changed) <= set(st.tables[1])
        st.seqs.context[0] = 1 << 40
        api.append(ctx, st.cache, st.seqs, k, v)
        with pytest.raises(NativeError, match="out of range"):
            ctx.check()
        st.seqs.context[0] = 0
        api.append(ctx, st.cache, st.seqs, k, v, cos_sin=_cos_sin(64, 8, st.dtype))  # positions up to 31
        with pytest.raises(NativeError, match="out of range"):
            ctx.check()


@pytest.mark.parametrize("dtype,e4m3", PAGES)
def test_prompt_then_tokens(ctx, dtype, e4m3):
    """The operators as a decode loop uses them: a prompt in chunks, then single tokens, with a window, against the
    definition run on the reference's own pages."""
    from plm import cache as api

    heads, kv_heads, hd, page = 8, 2, 128, 16
    st = Setup(rows=[70, 33], context=[0, 0], kv_heads=kv_heads, head_dim=hd, page=page, dtype=dtype, e4m3=e4m3, seed=20)
    pages = 16
    cache = api.PagedCache.allocate(pages, kv_heads, page, hd, dtype="e4m3" if e4m3 else st.dtype, scale_block=8)
    tables = torch.randperm(pages, generator=st.g, device="cuda").to(torch.int32).view(2, 8)
    cos_sin = _cos_sin(hd, 128, st.dtype)
    model = CacheModel(cache.k, cache.v, cache.k_scale, cache.v_scale)
    context = [0, 0]
    for step, rows in enumerate([[70, 33], [20, 1], [1, 1], [1, 1], [1, 1]]):
        starts = [0, rows[0], rows[0] + rows[1]]
        seqs = api.Sequences(torch.tensor(starts, dtype=torch.int32, device="cuda"),
                             torch.tensor(context, dtype=torch.int64, device="cuda"), tables, max_rows=max(rows))
        qkv = st.randn(starts[-1], heads + 2 * kv_heads, hd)
        q, k, v = qkv.split([heads, kv_heads, kv_heads], dim=1)
        rotated = api.append(ctx, cache, seqs, k, v, q=q, cos_sin=cos_sin)
        out = api.attention(ctx, cache, seqs, rotated, window=48, sinks=4)
        ctx.check()
        model.append(starts, context, tables.tolist(), k.double().cpu(), v.double().cpu(), None, cos_sin.cpu())
        if not e4m3:
            model.k, model.v = model.k.to(st.dtype).double(), model.v.to(st.dtype).double()
        _assert_pages(cache, model)
        for s in range(2):
            kk, vv, vs = model.dense(tables[s].tolist(), context[s] + rows[s])
            want, bound = attend(rotated[starts[s]:starts[s + 1]].double().cpu(), kk, vv, vs,
                                 visible(rows[s], context[s], 48, 4), st.dtype)
            assert within(out[starts[s]:starts[s + 1]], want, bound)
        context = [c + n for c, n in zip(context, rows)]
