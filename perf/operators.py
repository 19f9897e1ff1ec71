"""The paged-cache operators as measured workloads: appending rotated keys and values to a paged cache (16-bit, or
e4m3 with a scale per block of tokens and head) and attention over such a cache (causal or under the round mask, with
or without a sliding window and sinks).

``listed()`` names the cases, ``prepare`` makes a case's inputs, ``run`` makes one pass: with ``own`` through
``plm.cache``, otherwise in elementary torch operations in 32 bits. ``exact`` restates the operators in 64 bits.
"""

import math
import sys

import torch

own = False

UNREACHABLE = 1 << 30
E4M3_MAX = 448.0
MIN_EXPONENT = -100
DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16}


def _case(name, op, **kw):
    base = {"name": name, "op": op, "kind": "model", "dtype": "bf16", "heads": 16, "kv_heads": 16, "head_dim": 128,
            "page": 16, "block": 16, "seqs": 1, "rows_lo": 1, "rows_hi": 1, "ctx_lo": 1024, "ctx_hi": 1024,
            "window": 0, "sinks": 0, "round_k": 0, "spare_rows": 0}
    return {**base, **kw}


def listed():
    return [
        # one new token of one request into the 8-bit cache: the smallest call, launch latency
        _case("append e4m3 1 row", "append", kind="e4m3", ctx_lo=1003, ctx_hi=1003),
        # one round's 7 + 49 rows into the 16-bit cache
        _case("append 16-bit round", "append", rows_lo=56, rows_hi=56),
        # a batch of prompts, ragged, grouped heads, the last block of every sequence partly filled, spare rows behind
        _case("append e4m3 prompts", "append", kind="e4m3", dtype="f16", heads=32, kv_heads=8, seqs=7, rows_lo=1500,
              rows_hi=4097, ctx_lo=0, ctx_hi=777, page=64, block=32, spare_rows=24),
        # the same into the 16-bit cache
        _case("append 16-bit prompts", "append", heads=32, kv_heads=8, seqs=7, rows_lo=1500, rows_hi=4097, ctx_lo=0,
              ctx_hi=777, page=64, spare_rows=24),
        # one token against a short 8-bit context: the smallest attention call
        _case("decode e4m3 1024", "attend", kind="e4m3", ctx_lo=1023, ctx_hi=1023),
        # one token against the longest context of the benchmark sweep
        _case("decode e4m3 32768", "attend", kind="e4m3", ctx_lo=32767, ctx_hi=32767, page=32),
        # a serving batch: one token each for many requests of uneven length, grouped heads
        _case("decode e4m3 batch", "attend", kind="e4m3", heads=32, kv_heads=8, seqs=61, ctx_lo=1, ctx_hi=8190,
              page=64, block=32),
        # a round of 7 verify and 49 proposal rows at a 4096-token context
        _case("round e4m3 4096", "attend", kind="e4m3", rows_lo=56, rows_hi=56, ctx_lo=4096, ctx_hi=4096, round_k=7),
        # a prompt chunk behind a long 8-bit context
        _case("prefill e4m3", "attend", kind="e4m3", dtype="f16", rows_lo=2048, rows_hi=2048, ctx_lo=6000,
              ctx_hi=6000, page=64, block=64),
        # one token each, a window of 4096 and 4 sinks over long 16-bit contexts
        _case("window decode", "attend", heads=32, kv_heads=8, seqs=8, ctx_lo=9000, ctx_hi=32700, page=64,
              window=4096, sinks=4),
        # a whole prompt under a window
        _case("window prefill", "attend", heads=16, kv_heads=4, rows_lo=8191, rows_hi=8191, ctx_lo=0, ctx_hi=0,
              page=64, window=1024, sinks=4),
        # prompts and single tokens in one call, odd sizes, heads of 64, spare rows behind the last sequence
        _case("window mixed", "attend", dtype="f16", heads=12, kv_heads=4, head_dim=64, seqs=9, rows_lo=1,
              rows_hi=517, ctx_lo=0, ctx_hi=2999, window=333, sinks=7, spare_rows=5),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    while True:
        case = _draw_any(rng)
        cost = work(case)
        if cost["bytes"] <= 4.5e8 and cost["flops"] <= 1.1e11:
            return case


def _draw_any(rng):
    op = rng.choice(["append", "attend", "attend"])
    kind = rng.choice(["model", "e4m3", "e4m3"])
    kv_heads = rng.choice([1, 2, 4, 8, 16])
    heads = kv_heads * rng.choice([1, 1, 2, 3, 4, 8])
    while heads > 32:
        heads //= 2
    heads = max(heads // kv_heads, 1) * kv_heads
    page = rng.choice([16, 32, 64, 128])
    case = {"op": op, "kind": kind, "dtype": rng.choice(["bf16", "f16"]), "heads": heads, "kv_heads": kv_heads,
            "head_dim": rng.choice([64, 128, 128]), "page": page, "block": rng.choice([16, 32, 64, 128]),
            "window": 0, "sinks": 0, "round_k": 0, "spare_rows": rng.choice([0, 0, 3, 16])}
    case["block"] = min(case["block"], page, 64)
    form = rng.choice(["single", "batch", "round", "prompt", "prompt", "mixed"])
    if form == "single":
        c = _log_int(rng, 1, 32767)
        case.update(seqs=1, rows_lo=1, rows_hi=1, ctx_lo=c, ctx_hi=c)
    elif form == "batch":
        hi = _log_int(rng, 64, 8190)
        case.update(seqs=rng.randint(2, 61), rows_lo=1, rows_hi=1, ctx_lo=rng.randint(0, hi // 2), ctx_hi=hi)
    elif form == "round":
        k, c = rng.choice([4, 6, 7, 8]), _log_int(rng, 64, 16384)
        case.update(seqs=1, rows_lo=k + k * k, rows_hi=k + k * k, ctx_lo=c, ctx_hi=c, round_k=k, spare_rows=0)
    elif form == "prompt":
        n, c = _log_int(rng, 17, 4096), rng.choice([0, _log_int(rng, 1, 3000)])
        case.update(seqs=1, rows_lo=n, rows_hi=n, ctx_lo=c, ctx_hi=c)
    else:
        case.update(seqs=rng.randint(2, 9), rows_lo=1, rows_hi=_log_int(rng, 2, 600), ctx_lo=0,
                    ctx_hi=_log_int(rng, 1, 2999))
    if op == "attend" and rng.random() < 0.5:
        case.update(window=_log_int(rng, 16, 4096), sinks=rng.choice([0, 1, 4, 7]))
    return case


def lengths(case):
    """Rows and context of every sequence: spread over the case's ranges by the golden ratio, both ends included."""
    rows, ctx = [], []
    for s in range(case["seqs"]):
        u = 1.0 if s == 0 else (s * 0.6180339887498949) % 1.0
        w = 0.0 if s == 1 else 1.0 if s == 0 else (s * 0.7548776662466927) % 1.0
        rows.append(case["rows_lo"] + int(round(u * (case["rows_hi"] - case["rows_lo"]))))
        ctx.append(case["ctx_lo"] + int(round(w * (case["ctx_hi"] - case["ctx_lo"]))))
    return rows, ctx


def _round_layout(k):
    depth, own_start = list(range(k)), [UNREACHABLE] * k
    for d in range(k):
        for _ in range(k):
            depth.append(d)
            own_start.append(k + d * k)
    return depth, own_start


def _visible_counts(case):
    """Visible (row, key) pairs, and keys that some row sees, over all sequences."""
    rows, ctx = lengths(case)
    pairs = keys = 0
    w, sinks = case["window"], case["sinks"]
    depth, own_start = _round_layout(case["round_k"]) if case["round_k"] else (None, None)
    for n, c in zip(rows, ctx):
        low = None
        for j in range(n):
            d = j if depth is None else depth[j]
            pos = c + d + (max(0, j - own_start[j]) if depth is not None and own_start[j] <= j else 0)
            first = max(0, pos - w + 1) if w else 0
            pairs += max(0, c + d + 1 - first) + min(first, sinks)
            if depth is not None and own_start[j] <= j:
                pairs += j - own_start[j] + 1
            low = first if low is None else min(low, first)
        keys += c + n - low + min(low, sinks) if n else 0
    return pairs, keys


def work(case):
    rows, _ = lengths(case)
    total, hd, h, hk = sum(rows), case["head_dim"], case["heads"], case["kv_heads"]
    wide = 1 if case["kind"] == "e4m3" else 2
    scale = 4.0 / case["block"] / hd if case["kind"] == "e4m3" else 0.0
    if case["op"] == "append":
        values = total * hk * hd * 2
        return {"bytes": total * h * hd * 4 + values * (2 + wide + scale) + total * hd * 2,
                "flops": total * (h + hk) * hd * 3}
    pairs, keys = _visible_counts(case)
    return {"bytes": total * h * hd * 4 + keys * hk * hd * 2 * (wide + scale), "flops": 4 * pairs * h * hd}


def _exponent(amax):
    """The smallest e with amax <= 448 * 2^e, at least MIN_EXPONENT."""
    mantissa, e = torch.frexp(amax)  # amax = mantissa * 2^e, 0.5 <= mantissa < 1; 448 = 0.875 * 2^9
    e = e - 9 + (mantissa > 0.875).to(e.dtype)
    return torch.where(amax > 0, e, torch.full_like(e, MIN_EXPONENT)).clamp(min=MIN_EXPONENT)


def _quantised_pages(case, pages, g):
    """Random codes with a power-of-two scale per block and head, as an append leaves them."""
    hk, page, hd, block = case["kv_heads"], case["page"], case["head_dim"], case["block"]
    x = torch.empty(pages, hk, page // block, block, hd, device="cuda").normal_(generator=g)
    x = x * torch.empty(pages, hk, page // block, 1, 1, device="cuda").uniform_(0.25, 4.0, generator=g)
    s = torch.exp2(_exponent(x.abs().amax(dim=(-1, -2))).float())
    codes = (x / s[..., None, None]).to(torch.float8_e4m3fn).view(pages, hk, page, hd)
    return codes, s


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    dtype, hd, page, hk, h = DTYPES[case["dtype"]], case["head_dim"], case["page"], case["kv_heads"], case["heads"]
    rows, ctx = lengths(case)
    total = sum(rows)
    held = total + case["spare_rows"]
    need = [-(-(n + c) // page) for n, c in zip(rows, ctx)]
    pages = sum(need) + 3
    st = {"case": case, "rows": rows, "ctx": ctx, "total": total, "max_rows": max(rows),
          "max_keys": max(n + c for n, c in zip(rows, ctx))}
    perm = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)
    tables = torch.full((case["seqs"], max(need)), -1, dtype=torch.int32, device="cuda")
    at = 0
    for s, n in enumerate(need):
        tables[s, :n] = perm[at:at + n]
        at += n
    st["tables"] = tables
    starts = [0]
    for n in rows:
        starts.append(starts[-1] + n)
    st["row_start"] = torch.tensor(starts, dtype=torch.int32, device="cuda")
    st["context"] = torch.tensor(ctx, dtype=torch.int64, device="cuda")
    if case["kind"] == "e4m3":
        st["k_cache"], st["k_scale"] = _quantised_pages(case, pages, g)
        st["v_cache"], st["v_scale"] = _quantised_pages(case, pages, g)
    else:
        st["k_cache"] = torch.empty(pages, hk, page, hd, dtype=dtype, device="cuda").normal_(generator=g)
        st["v_cache"] = torch.empty(pages, hk, page, hd, dtype=dtype, device="cuda").normal_(generator=g)
        st["k_scale"] = st["v_scale"] = None
    if case["op"] == "append":
        # the fused projection's rows: q, k and v side by side
        qkv = torch.empty(held, (h + 2 * hk) * hd, dtype=dtype, device="cuda").normal_(generator=g)
        st["q"], st["k"], st["v"] = (t.unflatten(1, (-1, hd)) for t in qkv.split([h * hd, hk * hd, hk * hd], dim=1))
        st["q_out"] = torch.zeros(held, h, hd, dtype=dtype, device="cuda")
        inv = 1.0 / (10000.0 ** (torch.arange(0, hd, 2, dtype=torch.float64, device="cuda") / hd))
        angle = torch.arange(st["max_keys"], dtype=torch.float64, device="cuda")[:, None] * inv
        st["cos_sin"] = torch.cat((angle.cos(), angle.sin()), dim=1).to(dtype)
    else:
        st["q"] = torch.empty(held, h, hd, dtype=dtype, device="cuda").normal_(generator=g)
        st["out"] = torch.zeros(held, h, hd, dtype=dtype, device="cuda")
        st["depth"] = st["own_start"] = None
        if case["round_k"]:
            depth, own_start = _round_layout(case["round_k"])
            st["depth"] = torch.tensor(depth, dtype=torch.int32, device="cuda")
            st["own_start"] = torch.tensor(own_start, dtype=torch.int32, device="cuda")
    if own:
        if "plm-anon_b200" not in sys.path:
            sys.path.insert(0, "plm-anon_b200")
        from plm import cache, native

        global _context
        if _context is None:
            _context = native.Context()
        st["api"], st["ctx_handle"] = cache, _context
        st["cache"] = cache.PagedCache(st["k_cache"], st["v_cache"], st["k_scale"], st["v_scale"])
        st["seqs"] = cache.Sequences(st["row_start"], st["context"], st["tables"], max_rows=st["max_rows"],
                                     max_keys=st["max_keys"])
    return st


_context = None  # the program's one context


def _row_places(st):
    """Sequence, logical index, page and slot of every row that a sequence holds."""
    row = torch.arange(st["total"], device="cuda")
    seq = torch.searchsorted(st["row_start"][1:].long(), row, right=True)
    logical = st["context"][seq] + row - st["row_start"].long()[seq]
    page = st["case"]["page"]
    return seq, logical, st["tables"].long()[seq, logical // page], logical % page


def _rotate(x, cos_sin, logical, wide):
    cos, sin = cos_sin[logical].to(wide)[:, None, :].chunk(2, dim=-1)
    a, b = x.to(wide).chunk(2, dim=-1)
    return torch.cat((a * cos - b * sin, b * cos + a * sin), dim=-1)


def _store_e4m3(codes, scale, x, case, logical, pages, slots, seq, context):
    """One of K and V into the 8-bit cache: new scales of the blocks that the rows touch, the older tokens of a block
    that was begun earlier brought to the new scale, and the rows' codes."""
    block = case["block"]
    sub = slots // block
    n_sub = scale.shape[2]
    flat = pages * n_sub + sub
    touched, index = torch.unique(flat, return_inverse=True)
    amax = torch.zeros(touched.numel(), x.shape[1], dtype=x.dtype, device="cuda")
    amax.scatter_reduce_(0, index[:, None].expand(-1, x.shape[1]), x.abs().amax(dim=-1), "amax")
    new = torch.exp2(_exponent(amax).float())
    # tokens of the block that the sequence held before this call: logical indices below its context
    begun = torch.zeros(touched.numel(), dtype=torch.int64, device="cuda")
    begun[index] = (context[seq] - logical // block * block).clamp(0, block)
    p, b = touched // n_sub, touched % n_sub
    old = scale[p, :, b]
    new = torch.where(begun[:, None] > 0, torch.maximum(new, old), new)
    place = b[:, None] * block + torch.arange(block, device="cuda")
    kept = torch.arange(block, device="cuda")[None, :] < begun[:, None]
    before = codes[p[:, None], :, place]
    after = (before.float() * (old / new)[:, None, :, None]).to(torch.float8_e4m3fn)
    raw, was = after.view(torch.uint8), before.view(torch.uint8)
    codes.view(torch.uint8)[p[:, None], :, place] = torch.where(kept[:, :, None, None], raw, was)
    scale[p, :, b] = new
    q = (x.float() / new[index][:, :, None]).clamp(-E4M3_MAX, E4M3_MAX).to(torch.float8_e4m3fn)
    codes.view(torch.uint8)[pages, :, slots] = q.view(torch.uint8)


def _append_plain(st):
    case, n = st["case"], st["total"]
    seq, logical, pages, slots = _row_places(st)
    dtype = st["q"].dtype
    st["q_out"][:n] = _rotate(st["q"][:n], st["cos_sin"], logical, torch.float32).to(dtype)
    k = _rotate(st["k"][:n], st["cos_sin"], logical, torch.float32)
    if case["kind"] == "e4m3":
        _store_e4m3(st["k_cache"], st["k_scale"], k, case, logical, pages, slots, seq, st["context"])
        _store_e4m3(st["v_cache"], st["v_scale"], st["v"][:n].float(), case, logical, pages, slots, seq, st["context"])
    else:
        st["k_cache"][pages, :, slots] = k.to(dtype)
        st["v_cache"][pages, :, slots] = st["v"][:n]
    return _append_outputs(st)


def _append_outputs(st):
    out = {"q": st["q_out"], "k": st["k_cache"], "v": st["v_cache"]}  # e4m3 tensors: numbers, in units of the scales
    if st["case"]["kind"] == "e4m3":
        out.update(k_scale=st["k_scale"], v_scale=st["v_scale"])
    return out


def _attend(st, wide, out_dtype):
    """All sequences at once, padded to the longest: gathered keys, masked scores, softmax, weighted values."""
    case = st["case"]
    h, hk, hd, page = case["heads"], case["kv_heads"], case["head_dim"], case["page"]
    n_max, l_max, n_seqs = st["max_rows"], st["max_keys"], case["seqs"]
    start, ctx = st["row_start"].long(), st["context"]
    rows = start[1:] - start[:-1]
    j = torch.arange(n_max, device="cuda")
    kv = torch.arange(l_max, device="cuda")
    table = st["tables"].long().clamp(min=0)[:, kv // page]
    live = (kv[None, :] < (ctx + rows)[:, None])[..., None, None]

    def gather(cache, scale):
        x = cache.view(torch.uint8)[table, :, kv % page].view(torch.float8_e4m3fn) if scale is not None else cache[table, :, kv % page]
        x = x.to(wide)
        if scale is not None:
            x = x * scale[table, :, (kv % page) // case["block"]].to(wide)[..., None]
        return torch.where(live, x, torch.zeros((), dtype=wide, device="cuda"))  # [seq, key, kv head, d]

    keys = gather(st["k_cache"], st["k_scale"]).permute(0, 2, 3, 1)
    values = gather(st["v_cache"], st["v_scale"]).permute(0, 2, 1, 3)
    row = (start[:-1, None] + j).clamp(max=st["total"] - 1)
    q = st["q"][row].to(wide).view(n_seqs, n_max, hk, h // hk, hd).permute(0, 2, 3, 1, 4).reshape(n_seqs, hk, -1, hd)
    scores = torch.matmul(q, keys) * (1.0 / math.sqrt(hd))
    depth, begins = j, torch.full_like(j, UNREACHABLE)
    if st["depth"] is not None:
        depth, begins = st["depth"].long(), st["own_start"].long()
    rel = kv[None, None, :] - ctx[:, None, None]
    pos = ctx[:, None] + depth + torch.where(begins <= j, j - begins, torch.zeros_like(j))
    seen = rel <= depth[None, :, None]
    if case["window"]:
        seen = seen & ((kv < case["sinks"]) | (kv > pos[..., None] - case["window"]))
    seen = seen | ((rel >= begins[None, :, None]) & (rel <= j[None, :, None]))
    seen = seen & (j[None, :, None] < rows[:, None, None]) & live[:, None, :, 0, 0]
    seen = seen[:, None, None].expand(-1, 1, h // hk, -1, -1).reshape(n_seqs, 1, -1, l_max)
    scores.masked_fill_(~seen, float("-inf"))
    top = scores.amax(dim=-1, keepdim=True)
    weights = scores.sub_(torch.where(top == float("-inf"), torch.zeros_like(top), top)).exp_()
    total = weights.sum(dim=-1, keepdim=True)
    out = torch.matmul(weights, values) / torch.where(total > 0, total, torch.ones_like(total))
    out = out.view(n_seqs, hk, h // hk, n_max, hd).permute(0, 3, 1, 2, 4).reshape(n_seqs, n_max, h, hd)
    return out[j[None, :] < rows[:, None]].to(out_dtype)


def run(state):
    case = state["case"]
    if own:
        api, ctx = state["api"], state["ctx_handle"]
        if case["op"] == "append":
            api.append(ctx, state["cache"], state["seqs"], state["k"], state["v"], q=state["q"], q_out=state["q_out"],
                       cos_sin=state["cos_sin"])
            return _append_outputs(state)
        return api.attention(ctx, state["cache"], state["seqs"], state["q"], out=state["out"], window=case["window"],
                             sinks=case["sinks"], depth=state["depth"], own_start=state["own_start"])
    if case["op"] == "append":
        return _append_plain(state)
    state["out"][:state["total"]] = _attend(state, torch.float32, state["out"].dtype)
    return state["out"]


def _exact_codes(x):
    """Nearest e4m3 numbers of 64-bit values, ties to even, saturating at 448."""
    a = x.abs().clamp(max=E4M3_MAX)
    step = torch.exp2(torch.floor(torch.log2(a.clamp(min=2.0 ** -6))) - 3)
    a = torch.round(a / step) * step
    return torch.where(x < 0, -a, a)


def _exact_append(st):
    """Row by row blocks of the definition in 64 bits: the blocks every sequence's new rows fall into."""
    case, n = st["case"], st["total"]
    wide, block, page = torch.float64, case["block"], case["page"]
    row_start, ctx, tables = st["row_start"].tolist(), st["ctx"], st["tables"].tolist()
    out = {"q": st["q_out"].to(wide), "k": st["k_cache"].to(wide), "v": st["v_cache"].to(wide)}
    if case["kind"] == "e4m3":
        out.update(k_scale=st["k_scale"].to(wide), v_scale=st["v_scale"].to(wide))
    for s, c in enumerate(ctx):
        lo, hi = row_start[s], row_start[s + 1]
        angle = st["cos_sin"][c:c + hi - lo].to(wide)[:, None, :]
        half = case["head_dim"] // 2

        def rotated(x):
            a, b, cos, sin = x[..., :half], x[..., half:], angle[..., :half], angle[..., half:]
            return torch.cat((a * cos - b * sin, a * sin + b * cos), dim=-1)

        out["q"][lo:hi] = rotated(st["q"][lo:hi].to(wide))
        new = {"k": rotated(st["k"][lo:hi].to(wide)), "v": st["v"][lo:hi].to(wide)}
        step = block if case["kind"] == "e4m3" else page
        for first in range(c // step * step, c + hi - lo, step):
            a, b = max(first, c), min(first + step, c + hi - lo)
            p, slot = tables[s][first // page], first % page
            for name in ("k", "v"):
                x = new[name][a - c:b - c].transpose(0, 1)
                place = out[name][p, :, slot:slot + step]
                if case["kind"] == "e4m3":
                    scale = out[name + "_scale"][p, :, slot // block]
                    amax = x.abs().amax(dim=(1, 2)).float().to(wide)
                    want = torch.exp2(torch.ceil(torch.log2(amax.clamp(min=2.0 ** -100) / E4M3_MAX)).clamp(min=MIN_EXPONENT))
                    if a > first:
                        want = torch.maximum(want, scale)
                        place[:, :a - first] = _exact_codes(place[:, :a - first] * (scale / want)[:, None, None])
                    scale.copy_(want)
                    x = _exact_codes(x / want[:, None, None])
                place[:, a - first:b - first] = x
    return out


def exact(case, seed):
    st = prepare(case, seed)
    if case["op"] == "append":
        return _exact_append(st)
    out = st["out"].to(torch.float64)
    h, hk, hd, page = case["heads"], case["kv_heads"], case["head_dim"], case["page"]
    at = 0
    for s, (n, c) in enumerate(zip(st["rows"], st["ctx"])):
        pages = st["tables"][s, :-(-(n + c) // page)].long()

        def dense(cache, scale):
            x = cache.view(torch.uint8)[pages].view(torch.float8_e4m3fn).double() if scale is not None else cache[pages].double()
            if scale is not None:
                x = x * scale[pages].double().repeat_interleave(case["block"], dim=2)[..., None]
            return x.transpose(0, 1).reshape(hk, -1, hd)[:, :n + c]

        k, v = dense(st["k_cache"], st["k_scale"]), dense(st["v_cache"], st["v_scale"])
        j, kv = torch.arange(n, device="cuda")[:, None], torch.arange(n + c, device="cuda")[None, :]
        if case["round_k"]:
            depth, begins = st["depth"].long()[:, None], st["own_start"].long()[:, None]
            inside = (kv - c >= begins) & (kv - c <= j)
            place = depth + torch.where(begins <= j, j - begins, 0)
        else:
            depth, inside, place = j, torch.zeros(n, n + c, dtype=torch.bool, device="cuda"), j
        seen = kv <= c + depth
        if case["window"]:
            seen &= (kv < case["sinks"]) | (c + place - kv < case["window"])
        hidden = ~(seen | inside)
        for head in range(h):
            g = head // (h // hk)
            score = st["q"][at:at + n, head].double() @ k[g].T / math.sqrt(hd)
            out[at:at + n, head] = torch.softmax(score.masked_fill_(hidden, float("-inf")), dim=-1) @ v[g]
        at += n
    return out
