"""The 8-bit paged K/V cache restated on the CPU, token by token (no upstream counterpart).

Codes, scales and means are defined bit for bit: single FP32 operations and sums of whole numbers.  Attention is computed in 64 bits.
A cache is a dict of CPU tensors: k, v [pages, page_size, kv_heads, head_dim] (int8 or float8_e4m3fn), k_scale, v_scale
[pages, kv_heads] float32, k_mean [pages, kv_heads, head_dim] int8.
"""

from __future__ import annotations

import math

import torch

TOP = {torch.int8: 127.0, torch.float8_e4m3fn: 448.0}


def empty(pages, page_size, kv_heads, head_dim, codes):
    shape = (pages, page_size, kv_heads, head_dim)
    return dict(k=torch.zeros(shape, dtype=codes), v=torch.zeros(shape, dtype=codes), k_scale=torch.zeros(pages, kv_heads),
                v_scale=torch.zeros(pages, kv_heads), k_mean=torch.zeros(pages, kv_heads, head_dim, dtype=torch.int8))


def rotate(x, cos, sin, rope_dim, interleaved):
    """One token's heads [heads, dim] in FP32, products and sums rounded one by one."""
    x = x.float()
    out, half = x.clone(), rope_dim // 2
    one, two = (slice(0, rope_dim, 2), slice(1, rope_dim, 2)) if interleaved else (slice(0, half), slice(half, rope_dim))
    a, b, c, s = x[:, one], x[:, two], cos[None, :half], sin[None, :half]
    out[:, one], out[:, two] = a * c - b * s, a * s + b * c
    return out


def _round(x, codes):
    x = x.round() if codes == torch.int8 else x
    return x.clamp(-TOP[codes], TOP[codes]).to(codes)


def _write(codes, scale, rows, values):
    """Rows {row: value [dim]} into one block [page_size, dim] with its scale; returns the new (codes, scale)."""
    kind = codes.dtype
    before = torch.tensor(0.0) if 0 in rows else scale
    most = torch.stack(list(values.values())).abs().max() if values else torch.tensor(0.0)
    if not math.isfinite(float(most)) or not math.isfinite(float(before)):
        now = torch.tensor(float("nan"))
    else:
        now = torch.maximum(before, most * (torch.tensor(1.0) / TOP[kind]))
    codes = codes.clone()
    if 0 not in rows and bool(now > before):
        kept = [r for r in range(codes.shape[0]) if r not in rows]
        codes[kept] = _round(codes[kept].float() * (before / now), kind)
    for row, x in values.items():
        codes[row] = _round(x / now, kind) if bool(now > 0) else torch.zeros_like(x).to(kind)
    return codes, now


def append(q, k, v, cos, sin, positions, page_table, sequence_ids, cache, *, rope_dim, interleaved):
    """Writes into `cache`; returns rotated q."""
    page_size, kind = cache["k"].shape[1], cache["k"].dtype
    out = torch.zeros_like(q)
    blocks: dict = {}  # page -> {row: token}
    for t, pos in enumerate(positions.tolist()):
        if pos < 0:
            continue
        out[t] = rotate(q[t], cos[pos], sin[pos], rope_dim, interleaved).to(q.dtype)
        blocks.setdefault(int(page_table[sequence_ids[t], pos // page_size]), {})[pos % page_size] = t
    for page, rows in blocks.items():
        turned = {row: rotate(k[t], cos[positions[t]], sin[positions[t]], rope_dim, interleaved) for row, t in rows.items()}
        for h in range(cache["k"].shape[2]):
            for name, of in (("k", lambda row: turned[row][h]), ("v", lambda row: v[rows[row], h].float())):
                cache[name][page, :, h], cache[name + "_scale"][page, h] = _write(
                    cache[name][page, :, h], cache[name + "_scale"][page, h].clone(), rows, {row: of(row) for row in rows})
            if page_size - 1 in rows:
                total = cache["k"][page, :, h].double().sum(0)
                if kind == torch.int8:
                    mean = total.float() * torch.tensor(1.0 / page_size)
                else:
                    mean = (total * 512).float() * torch.tensor(127.0 / (448.0 * 512.0 * page_size))
                cache["k_mean"][page, h] = mean.round().clamp(-127, 127).to(torch.int8)
    return out


def attention(q, cache, positions, page_table, sequence_ids, *, scale=None, pages=None):
    """A dict: `result` in 64 bits; for every element of it `bound`, sum_j p_j |v_j|, and `least`, max_j(p_j vs_j) * sum_j |code_j|, vs
    the scales of V; for every head `score`, the largest scale * sum_d |q_d k_d| of a position, `offset`, the largest
    scale * ks * max(|sum of q_d over d >= 16 c|, 2 |q_d|), and `flat`, sum_j p_j vs_j.
    `pages` [tokens, kv_heads, n]: only these."""
    page_size, heads, dim = cache["k"].shape[1:]
    scale = dim ** -0.5 if scale is None else scale
    out = torch.zeros(q.shape, dtype=torch.float64)
    bound, least = torch.zeros_like(out), torch.zeros_like(out)
    score, offset, flat = (torch.zeros(q.shape[:2], dtype=torch.float64) for _ in range(3))
    group = q.shape[1] // heads
    for t, pos in enumerate(positions.tolist()):
        for h in range(heads):
            js = range(pos + 1)
            if pages is not None:
                js, before = [], -1
                for p in pages[t, h].tolist():
                    if p >= 0 and p > before:
                        js += [j for j in range(p * page_size, (p + 1) * page_size) if j <= pos]
                    before = p
            js = torch.tensor(list(js), dtype=torch.int64)
            if js.numel() == 0:
                continue
            at, off = page_table[sequence_ids[t], js // page_size], js % page_size
            k = cache["k"][at, off, h].double() * cache["k_scale"][at, h].double()[:, None]
            v = cache["v"][at, off, h].double() * cache["v_scale"][at, h].double()[:, None]
            mine = slice(h * group, (h + 1) * group)
            x = q[t, mine].double()
            p = torch.softmax(x @ k.T * scale, dim=-1)
            out[t, mine], bound[t, mine] = p @ v, p @ v.abs()
            least[t, mine] = (p * cache["v_scale"][at, h].double().abs()).amax(-1, keepdim=True) * cache["v"][at, off, h].double().abs().sum(0)
            ks, vs = cache["k_scale"][at, h].double().abs(), cache["v_scale"][at, h].double()
            ends = x.unflatten(-1, (dim // 16, 16)).sum(-1).flip(-1).cumsum(-1).abs().amax(-1).maximum(2 * x.abs().amax(-1))
            offset[t, mine], flat[t, mine] = ends * ks.amax() * abs(scale), p @ vs
            score[t, mine] = (x.abs() @ k.abs().T * abs(scale)).amax(-1)
    return dict(result=out, bound=bound, least=least, score=score, offset=offset, flat=flat)


def select(q, cache, positions, page_table, sequence_ids, *, top_pages):
    heads, page_size = cache["k"].shape[2], cache["k"].shape[1]
    group = q.shape[1] // heads
    out = torch.full((q.shape[0], heads, top_pages), -1, dtype=torch.int32)
    for t, pos in enumerate(positions.tolist()):
        if pos < 0:
            continue
        last = pos // page_size
        for h in range(heads):
            chosen = list(range(last))
            if last > top_pages - 1:
                x = q[t, h * group:(h + 1) * group].float()
                unit = x.abs().amax(-1) * (torch.tensor(1.0) / 127.0)
                codes = torch.where(unit[:, None] > 0, (x / unit[:, None]).round(), torch.tensor(0.0))
                at = page_table[sequence_ids[t], :last]
                dots = (codes.double() @ cache["k_mean"][at, h].double().T).float()
                scores = ((dots * unit[:, None]).amax(0) * cache["k_scale"][at, h]).tolist()
                scores = [math.inf if s != s else s for s in scores]
                chosen = sorted(range(last), key=lambda p: (-scores[p], p))[:top_pages - 1]
            out[t, h, :len(chosen) + 1] = torch.tensor(sorted(chosen) + [last], dtype=torch.int32)
    return out
