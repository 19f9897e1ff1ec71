"""The paged-cache operators restated in 64 bits from their definitions, with the error bounds their tests use."""

from __future__ import annotations

import math

import torch

UNREACHABLE = 1 << 30


def e4m3(x: torch.Tensor) -> torch.Tensor:
    """Nearest e4m3 numbers (ties to even, saturating at 448) of 64-bit values; NaN stays NaN."""
    a = x.abs().clamp(max=448.0)
    step = torch.exp2(torch.floor(torch.log2(a.clamp(min=2.0 ** -6))) - 3)
    return torch.copysign((a / step).round() * step, x)


def block_scale(amax: float) -> float:
    """2^e, e the smallest integer >= -100 with amax <= 448 * 2^e."""
    e = -100
    while amax > 448.0 * 2.0 ** e:
        e += 1
    return 2.0 ** e


def rotate(x: torch.Tensor, cos_sin: torch.Tensor | None, pos: int) -> torch.Tensor:
    """[heads, d] float64, rotated at one position; exact products rounded to fp32 once."""
    if cos_sin is None:
        return x
    half = x.shape[-1] // 2
    cos, sin = cos_sin[pos, :half].double(), cos_sin[pos, half:].double()
    a, b = x[:, :half], x[:, half:]
    return torch.cat((a * cos - b * sin, b * cos + a * sin), dim=-1).float().double()


class CacheModel:
    """A paged cache as plain 64-bit numbers (codes and scales apart), appended to a row at a time per call."""

    def __init__(self, k, v, k_scale=None, v_scale=None):
        self.k, self.v = k.double().cpu(), v.double().cpu()
        self.k_scale = None if k_scale is None else k_scale.double().cpu()
        self.v_scale = None if v_scale is None else v_scale.double().cpu()
        self.page = k.shape[2]
        self.block = 0 if k_scale is None else self.page // k_scale.shape[2]

    def append(self, row_start, context, tables, k, v, q=None, cos_sin=None, positions=None):
        """Returns the rotated queries of the rows the sequences hold ({row: [heads, d]})."""
        rotated = {}
        for s, c in enumerate(context):
            rows = range(row_start[s], row_start[s + 1])
            groups: dict[int, list] = {}
            for j, r in enumerate(rows):
                logical = c + j
                pos = logical if positions is None else positions[r]
                if q is not None:
                    rotated[r] = rotate(q[r], cos_sin, pos)
                new_k = rotate(k[r], cos_sin, pos)
                if not self.block:
                    p, slot = tables[s][logical // self.page], logical % self.page
                    self.k[p, :, slot], self.v[p, :, slot] = new_k, v[r]
                else:
                    groups.setdefault(logical // self.block, []).append((logical, new_k, v[r]))
            for block, tokens in groups.items():
                first = block * self.block
                p, slot = tables[s][first // self.page], first % self.page
                begun = tokens[0][0] - first
                for plane, scales, at in ((self.k, self.k_scale, 1), (self.v, self.v_scale, 2)):
                    for h in range(plane.shape[1]):
                        values = torch.stack([t[at][h] for t in tokens])
                        finite = values[torch.isfinite(values)].abs()
                        now = block_scale(finite.max().item() if finite.numel() else 0.0)
                        old = scales[p, h, slot // self.block].item()
                        if begun:
                            now = max(now, old)
                            kept = plane[p, h, slot:slot + begun]
                            plane[p, h, slot:slot + begun] = e4m3(kept * (old / now))
                        scales[p, h, slot // self.block] = now
                        plane[p, h, slot + begun:slot + begun + len(tokens)] = e4m3(values / now)
        return rotated

    def dense(self, table, keys: int):
        """K, V [keys, heads, d] of a sequence and, for codes, V's scales [keys, heads]."""
        pages = torch.tensor(table[:-(-keys // self.page)], dtype=torch.long).clamp(min=0)

        def flat(x):
            return x[pages].transpose(1, 2).reshape(-1, x.shape[1], *x.shape[3:])[:keys]

        k, v = flat(self.k), flat(self.v)
        if not self.block:
            return k, v, None
        ks, vs = (s[pages].repeat_interleave(self.block, dim=2).transpose(1, 2).reshape(-1, s.shape[1])[:keys]
                  for s in (self.k_scale, self.v_scale))
        return k * ks[..., None], v * vs[..., None], vs


def visible(n, c, window, sinks, depth=None, own_start=None):
    """[n, c + n] mask of one sequence, straight from the definition."""
    mask = torch.zeros(n, c + n, dtype=torch.bool)
    kv = torch.arange(c + n)
    for j in range(n):
        d = j if depth is None else depth[j]
        own = UNREACHABLE if own_start is None else own_start[j]
        p = c + d
        pos = p + (j - own if own <= j else 0)
        a = kv <= p
        if window:
            a &= (kv < sinks) | (kv > pos - window)
        mask[j] = a | ((kv - c >= own) & (kv - c <= j))
    return mask


def within(got, want, bound) -> bool:
    """Whether every element is within its bound of what is wanted, or the same infinity, or NaN where NaN is wanted."""
    got = got.double().cpu()
    same = (got == want) | (torch.isnan(got) & torch.isnan(want))
    ratio = torch.where(same, torch.zeros_like(bound), (got - want).abs() / bound)
    print(f"{ratio.max().item():.3f} of the bound")
    return bool((ratio <= 1.0).all())  # false for NaN


def attend(q, k, v, v_scale, mask, dtype, scale=None):
    """(out, bound) [n, heads, d] in 64 bits. The bound, per element, of a kernel that accumulates in fp32:
    - the output's one rounding, eps/2 |out|;
    - the weights' rounding to the 16-bit type they are multiplied in, eps/2 of A = sum w |v|, and for f16 (also with
      codes) half its smallest subnormal per key, 2^-25 of the largest w (times its scale) times the numbers they meet;
    - scores: fp32 sums of d products err by at most (d + 2) 2^-24 sum |q k|, twice (the maximum's term too), with a
      relative effect of as much on every weight;
    - 2^-14 of A for the exponentials and up to 512 rescalings in fp32 (2^-23 each)."""
    heads, hd = q.shape[1], q.shape[2]
    group = heads // k.shape[1]
    scale = 1.0 / math.sqrt(hd) if scale is None else scale
    kk, vv = k.repeat_interleave(group, dim=1), v.repeat_interleave(group, dim=1)
    # numbers that no row may see never enter: a masked NaN must not reach a product
    hidden = ~mask.any(dim=0)
    kk, vv = kk.clone(), vv.clone()
    kk[hidden], vv[hidden] = 0.0, 0.0
    s = torch.einsum("nhd,khd->hnk", q, kk) * scale
    s = torch.where(mask[None], s, torch.full_like(s, float("-inf")))
    top = s.amax(dim=-1, keepdim=True)
    w = torch.exp(s - torch.where(top == float("-inf"), torch.zeros_like(top), top))
    total = w.sum(dim=-1, keepdim=True)
    w = torch.where(total == 0, torch.zeros_like(w), w / total)  # NaN scores stay NaN
    clean = torch.where(torch.isfinite(vv), vv, torch.zeros_like(vv))
    out = torch.einsum("hnk,khd->nhd", w, clean)
    bad = ~torch.isfinite(vv)
    for key in torch.nonzero(bad.any(dim=(1, 2))).flatten().tolist():
        rows = mask[:, key]
        out[rows] = out[rows] + torch.where(bad[key], vv[key], torch.zeros_like(vv[key]))
    absolute = torch.einsum("hnk,khd->nhd", w, clean.abs())
    products = torch.einsum("nhd,khd->hnk", q.abs(), kk.abs()) * scale
    products = torch.where(mask[None], products, torch.zeros_like(products)).nan_to_num(0.0, 0.0, 0.0)
    delta = 2 * (hd + 2) * 2.0 ** -24 * products.amax(dim=-1).T[..., None]
    eps = torch.finfo(dtype).eps / 2
    weight = 2.0 ** -11 if v_scale is not None or dtype == torch.float16 else eps
    bound = eps * out.abs() + absolute * (weight + delta + 2.0 ** -14)
    if weight == 2.0 ** -11:
        vs = torch.ones(k.shape[:2], dtype=torch.float64) if v_scale is None else v_scale
        vs = vs.repeat_interleave(group, dim=1)
        largest = (w * vs.T[:, None, :]).amax(dim=-1)  # [heads, n]
        numbers = torch.einsum("nk,khd->nhd", mask.double(), clean.abs() / vs[..., None])
        bound = bound + 2.0 ** -25 * largest.T[..., None] * numbers
    return out, bound + torch.finfo(dtype).tiny
