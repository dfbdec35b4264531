"""The 8-bit paged K/V cache: what its operators are measured on.

Four operators share a cache of 8-bit codes (int8 or e4m3) with an FP32 scale per page and KV head: the rotation and
append that write it, the attention that reads it, the selection of pages by their mean keys, and the attention over the
selected pages.  ``own`` chooses between the framework's calls and the same operators in elementary torch operations.

``listed()`` are the fixed cases, ``draw(rng)`` one more of the same ranges, ``exact`` the results in 64-bit arithmetic.
"""

from __future__ import annotations

import math

import torch

own = False

_DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
_CODES = {"int8": (torch.int8, 127.0), "e4m3": (torch.float8_e4m3fn, 448.0)}
_THETA = 10000.0


def listed() -> list[dict]:
    return [
        # The append of one sequence's decode step, the smallest call: launch and host cost, and a chain of index loads.
        dict(name="append_e4m3_t1", kind="append", tokens=1, sequences=1, capacity=512, q_heads=32, kv_heads=8, head_dim=128,
             rope_dim=128, page_size=16, layout="NHD", interleaved=False, order="runs", codes="e4m3", dtype="f16"),
        # The append of a full decode batch, one token per sequence; the caches are returned as the values they stand for.
        dict(name="append_int8_t16", kind="append", tokens=16, sequences=16, capacity=256, q_heads=32, kv_heads=8, head_dim=128,
             rope_dim=64, page_size=16, layout="NHD", interleaved=False, order="runs", codes="int8", dtype="bf16"),
        # A prefill chunk of several prompts: 4096 tokens that fill whole pages and begin and end inside others.
        dict(name="append_e4m3_t4096", kind="append", tokens=4096, sequences=13, capacity=512, q_heads=32, kv_heads=8, head_dim=128,
             rope_dim=128, page_size=16, layout="HND", interleaved=False, order="runs", codes="e4m3", dtype="bf16"),
        # One sequence with a long context: few rows, so the context has to be split.
        dict(name="attend_int8_t1_ctx8192", kind="attend", tokens=1, context=8192, full=True, q_heads=32, kv_heads=8, head_dim=128,
             page_size=16, layout="NHD", codes="int8", dtype="f16"),
        # An odd small model in FP32: three heads to a group, pages that no tile divides, contexts from one token on.
        dict(name="attend_int8_t5_ctx1001_f32", kind="attend", tokens=5, context=1001, full=False, q_heads=6, kv_heads=2, head_dim=64,
             page_size=7, layout="NHD", codes="int8", dtype="f32"),
        # A larger batch with contexts of every length up to 2048.
        dict(name="attend_int8_t64_ctx2048", kind="attend", tokens=64, context=2048, full=False, q_heads=32, kv_heads=8, head_dim=128,
             page_size=16, layout="HND", codes="int8", dtype="bf16"),
        # The full decode batch at the context of this repository's decode layer.
        dict(name="attend_e4m3_t16_ctx8192", kind="attend", tokens=16, context=8192, full=True, q_heads=32, kv_heads=8, head_dim=128,
             page_size=16, layout="NHD", codes="e4m3", dtype="f16"),
        # The largest read: long contexts for the full batch, a gigabyte of codes.
        dict(name="attend_int8_t16_ctx32768", kind="attend", tokens=16, context=32768, full=True, q_heads=32, kv_heads=8, head_dim=128,
             page_size=32, layout="HND", codes="int8", dtype="bf16"),
        # Selection for one sequence, and for the full batch, from the means of thousands of pages.
        dict(name="select_t1_ctx8192", kind="select", tokens=1, context=8192, full=True, top_pages=64, q_heads=32, kv_heads=8,
             head_dim=128, page_size=16, codes="int8", dtype="f16"),
        dict(name="select_t16_ctx32768", kind="select", tokens=16, context=32768, full=True, top_pages=64, q_heads=32, kv_heads=8,
             head_dim=128, page_size=16, codes="e4m3", dtype="bf16"),
        # Attention over the selected pages of one sequence, and of the full batch.
        dict(name="sparse_int8_t1_64", kind="sparse", tokens=1, context=8192, full=True, top_pages=64, q_heads=32, kv_heads=8,
             head_dim=128, page_size=16, layout="NHD", codes="int8", dtype="f16"),
        dict(name="sparse_e4m3_t16_128", kind="sparse", tokens=16, context=32768, full=True, top_pages=128, q_heads=32, kv_heads=8,
             head_dim=128, page_size=16, layout="HND", codes="e4m3", dtype="bf16"),
    ]


def _log_int(rng, lo: int, hi: int) -> int:
    """An integer spread evenly over its logarithm in [lo, hi]."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng) -> dict:
    kind = rng.choice(["append", "attend", "attend", "select", "sparse"])
    kv_heads, head_dim = rng.choice([1, 2, 4, 8]), rng.choice([64, 128, 128, 256])
    group = rng.choice([1, 2, 3, 4, 4, 5, 8])
    c = dict(kind=kind, q_heads=kv_heads * group, kv_heads=kv_heads, head_dim=head_dim, page_size=rng.choice([5, 8, 16, 16, 32, 64]),
             codes=rng.choice(["int8", "e4m3"]), dtype=rng.choice(["bf16", "f16", "f16", "f32"]))
    if kind == "append":
        tokens = _log_int(rng, 1, 4096 if head_dim * group * kv_heads <= 4096 else 1024)
        sequences = min(tokens, rng.choice([1, 3, 16]))
        need = -(-tokens // sequences)
        return dict(c, tokens=tokens, sequences=sequences, capacity=need + rng.choice([8, 100, 256]),
                    rope_dim=rng.choice([head_dim, head_dim, head_dim // 2, 6]), layout=rng.choice(["NHD", "HND"]),
                    interleaved=rng.random() < 0.3, order=rng.choice(["runs", "runs", "mixed"]))
    tokens = _log_int(rng, 1, 64)
    most = (1 << 19) * 8 // kv_heads * 128 // head_dim  # positions of the largest listed case
    c.update(tokens=tokens, full=rng.random() < 0.5)
    if kind == "attend":
        return dict(c, context=_log_int(rng, 1, min(32768, most // (2 * tokens))), layout=rng.choice(["NHD", "HND"]))
    c["context"] = _log_int(rng, 200, min(32768, most // (2 * tokens)))
    pages = -(-c["context"] // c["page_size"])
    c["top_pages"] = min(_log_int(rng, 1, 128), max(1, pages // 2))
    return c if kind == "select" else dict(c, layout=rng.choice(["NHD", "HND"]))


def _codes(shape, gen, codes):
    """Codes as a quantiser leaves them: normal values whose largest of a block is near the end of the range."""
    dtype, top = _CODES[codes]
    out = torch.empty(shape, dtype=dtype, device="cuda")
    step = max(1, (1 << 27) // max(1, out[0].numel()))
    for at in range(0, shape[0], step):
        part = torch.randn((min(step, shape[0] - at), *shape[1:]), generator=gen, device="cuda").mul_(top / 4).clamp_(-top, top)
        out[at:at + step] = (part.round_() if codes == "int8" else part).to(dtype)
    return out


def prepare(case: dict, seed: int) -> dict:
    gen = torch.Generator(device="cuda").manual_seed(seed)
    kind, dtype = case["kind"], _DTYPES[case["dtype"]]
    tokens, heads, dim, page = case["tokens"], case["kv_heads"], case["head_dim"], case["page_size"]

    def normal(*shape):
        return torch.randn(*shape, generator=gen, device="cuda").to(dtype)

    st = dict(case=case, q=normal(tokens, case["q_heads"], dim))
    sequences = case["sequences"] if kind == "append" else tokens
    per_seq = -(-(case["capacity"] if kind == "append" else case["context"]) // page)
    pages = sequences * per_seq
    st["page_table"] = torch.randperm(pages, generator=gen, device="cuda").reshape(sequences, per_seq)
    if kind == "append":
        at = torch.arange(tokens, device="cuda")
        longest = -(-tokens // sequences)  # consecutive positions of each sequence, from one of its own on
        seq, step = (at // longest, at % longest) if case["order"] == "runs" else (at % sequences, at // sequences)
        start = torch.randint(0, case["capacity"] - longest + 1, (sequences,), generator=gen, device="cuda")
        st["sequence_ids"], st["positions"] = seq, start[seq] + step
        rope = case["rope_dim"]
        inv_freq = _THETA ** (-torch.arange(0, rope, 2, device="cuda").double() / rope)
        angle = torch.arange(case["capacity"], device="cuda").double()[:, None] * inv_freq[None, :]
        # channels of very different size, as keys have them, and values that are small
        st.update(cos=angle.cos().float(), sin=angle.sin().float(), k=normal(tokens, heads, dim).mul_(1 + 3 * torch.rand(dim, generator=gen, device="cuda")).to(dtype),
                  v=(0.2 * normal(tokens, heads, dim)).to(dtype))
    else:
        st["sequence_ids"] = torch.arange(tokens, device="cuda")
        shorter = torch.randint(0, max(1, case["context"] // 100) if case["full"] else case["context"], (tokens,), generator=gen, device="cuda")
        st["positions"] = case["context"] - 1 - shorter
    layout = case.get("layout", "NHD")
    shape = (pages, page, heads, dim) if layout == "NHD" else (pages, heads, page, dim)
    top = _CODES[case["codes"]][1]
    if kind == "select":  # reads the means and the scales of the keys, no codes
        k_codes = v_codes = torch.empty(shape, dtype=_CODES[case["codes"]][0], device="cuda")
    else:
        k_codes, v_codes = _codes(shape, gen, case["codes"]), _codes(shape, gen, case["codes"])

    def scales(size):  # of blocks whose largest value is about `size`, within a factor of two or so
        return size / top * torch.exp(0.3 * torch.randn(pages, heads, generator=gen, device="cuda"))

    # the mean of a block's keys is smaller than its largest by four, and by the root of their number
    means = (torch.randn(pages, heads, dim, generator=gen, device="cuda") * 32 / math.sqrt(page)).round_().clamp_(-127, 127).to(torch.int8)
    st.update(k_cache=k_codes, v_cache=v_codes, k_scale=scales(8.0), v_scale=scales(0.8), k_mean=means)
    if kind == "sparse":
        st["pages"] = _choose(st["positions"] // page, torch.rand(tokens, heads, per_seq, generator=gen, device="cuda"), case["top_pages"])
    if own:
        from cross_dsl_kernels_b200.kv8 import PagedKV8Cache

        v_codes = torch.empty_like(k_codes) if kind == "select" else v_codes  # the tensors of a cache are apart
        st["cache"] = PagedKV8Cache(st["k_cache"], v_codes, st["k_scale"], st["v_scale"], st["k_mean"], kv_layout=layout)
    return st


def run(st: dict):
    return _own(st) if own else _plain(st)


def _own(st: dict):
    from cross_dsl_kernels_b200 import kv8

    case, index = st["case"], (st["positions"], st["page_table"], st["sequence_ids"])
    if case["kind"] == "append":
        q_rot = kv8.rope_gqa_paged_kv8_append(st["q"], st["k"], st["v"], st["cos"], st["sin"], *index, st["cache"],
                                              rope_dim=case["rope_dim"], interleaved=case["interleaved"])
        return _written(st, q_rot)
    if case["kind"] == "attend":
        return kv8.paged_kv8_decode_attention(st["q"], st["cache"], *index, context_hint=case["context"])
    if case["kind"] == "select":
        return kv8.select_kv8_pages(st["q"], st["cache"], *index, top_pages=case["top_pages"])
    return kv8.paged_kv8_sparse_attention(st["q"], st["cache"], st["pages"], *index)


def _written(st: dict, q_rot) -> dict:
    """What an append leaves: e4m3 codes are values in units of their scale; int8 codes are returned as the values they stand for."""
    out = dict(q_rot=q_rot, k_scale=st["k_scale"], v_scale=st["v_scale"], k_mean=st["k_mean"].float())
    if st["case"]["codes"] == "e4m3":
        return dict(out, k=st["k_cache"], v=st["v_cache"])
    per = (slice(None), None, slice(None), None) if st["case"]["layout"] == "NHD" else (slice(None), slice(None), None, None)
    return dict(out, k=st["k_cache"] * st["k_scale"][per], v=st["v_cache"] * st["v_scale"][per])


# ---- the operators in elementary operations, 32 bits -------------------------------------------------------------------


def _plain(st: dict):
    case = st["case"]
    if case["kind"] == "append":
        return _append(st)
    if case["kind"] == "select":
        return _select(st)
    page, width = case["page_size"], st["page_table"].shape[1]
    if case["kind"] == "attend":
        j = torch.arange(width * page, device="cuda").expand(case["tokens"], case["kv_heads"], -1)
        live = j <= st["positions"][:, None, None]
    else:
        first = st["pages"].long()[..., None] * page + torch.arange(page, device="cuda")
        j = first.flatten(2)
        live = (j >= 0) & (j <= st["positions"][:, None, None])
        j = j.clamp_min(0)
    return _attention(st, j, live)


def _attention(st, j, live):
    """Softmax attention over the positions j [tokens, heads, n] of each token's sequence that are `live`."""
    case, q = st["case"], st["q"]
    page, heads, dim = case["page_size"], case["kv_heads"], case["head_dim"]
    at = st["page_table"][st["sequence_ids"][:, None, None], j // page]
    head = torch.arange(heads, device="cuda")[None, :, None]

    def rows(cache, scale):
        raw = cache.view(torch.uint8)
        raw = raw[at, j % page, head] if case["layout"] == "NHD" else raw[at, head, j % page]
        return raw.view(cache.dtype).float() * scale[at, head][..., None]

    qs = q.float().reshape(q.shape[0], heads, -1, dim)
    s = qs @ rows(st["k_cache"], st["k_scale"]).transpose(2, 3) * dim ** -0.5
    s = s.masked_fill(~live[:, :, None, :], -math.inf)
    p = torch.exp(s - s.amax(-1, keepdim=True))
    o = (p @ rows(st["v_cache"], st["v_scale"])) / p.sum(-1, keepdim=True)
    return o.reshape(q.shape).to(q.dtype)


def _choose(last, score, top_pages):
    """The `top_pages - 1` best of the pages in front of the `last` (ties: the lowest), and that one; ascending, padded with -1."""
    width = score.shape[-1]
    page = torch.arange(width, device="cuda")
    score = score.masked_fill(page >= last[:, None, None], -math.inf)
    best = torch.sort(score, dim=-1, descending=True, stable=True).indices[..., :top_pages - 1]
    best = torch.where(best < last[:, None, None], best, width)
    both = torch.cat([best, last[:, None, None].expand(*best.shape[:2], 1)], dim=-1).sort(dim=-1).values
    pad = both.new_full((*both.shape[:2], top_pages - both.shape[-1]), -1)
    return torch.cat([both.masked_fill(both == width, -1), pad], dim=-1).to(torch.int32)


def _select(st):
    case, q = st["case"], st["q"]
    heads, dim = case["kv_heads"], case["head_dim"]
    qs = q.float().reshape(q.shape[0], heads, -1, dim)
    unit = qs.abs().amax(-1, keepdim=True) / 127
    codes = torch.where(unit > 0, torch.round(qs / unit), 0.0)
    at = st["page_table"][st["sequence_ids"]]  # [tokens, pages of a sequence]
    means = st["k_mean"][at].transpose(1, 2).float()  # [tokens, heads, pages, dim]
    dot = codes @ means.transpose(2, 3)  # whole numbers under 2^24: exact in any order
    score = (dot * unit).amax(2) * st["k_scale"][at].transpose(1, 2)
    return _choose(st["positions"] // case["page_size"], score, case["top_pages"])


def _rotate(x, cos, sin, rope, interleaved):
    half = rope // 2
    one, two = (slice(0, rope, 2), slice(1, rope, 2)) if interleaved else (slice(0, half), slice(half, rope))
    out = x.clone()
    a, b, c, s = x[..., one], x[..., two], cos[:, None, :half], sin[:, None, :half]
    out[..., one], out[..., two] = a * c - b * s, a * s + b * c
    return out


def _round(x, codes):
    dtype, top = _CODES[codes]
    return x.round().clamp(-top, top).to(dtype) if codes == "int8" else x.clamp(-top, top).to(dtype)


def _append(st):
    case, pos, page = st["case"], st["positions"], st["case"]["page_size"]
    turn = [_rotate(st[n].float(), st["cos"][pos], st["sin"][pos], case["rope_dim"], case["interleaved"]) for n in ("q", "k")]
    at, off = st["page_table"][st["sequence_ids"], pos // page], pos % page
    kept_k = _store(st, "k", turn[1], at, off)
    _store(st, "v", st["v"].float(), at, off)
    # the means of the blocks whose last row was written
    top = _CODES[case["codes"]][1]
    whole = torch.zeros(st["k_scale"].shape[0], device="cuda").index_add_(0, at, (off == page - 1).float()) > 0
    if case["codes"] == "int8":
        total, unit = kept_k.float().sum(1), 1 / page
    else:
        total, unit = (kept_k.double() * 512).sum(1).float(), 127 / (top * 512 * page)
    mean = torch.round(total * torch.tensor(unit, device="cuda")).clamp(-127, 127).to(torch.int8)
    st["k_mean"].copy_(torch.where(whole[:, None, None], mean, st["k_mean"]))
    return _written(st, turn[0].to(st["q"].dtype))


def _store(st, name, x, at, off):
    """Writes the rows x [tokens, heads, dim] into their blocks; returns all codes as [pages, page, heads, dim]."""
    case, codes, scale = st["case"], st["case"]["codes"], st[name + "_scale"]
    top, page = _CODES[codes][1], case["page_size"]
    cache = st[name + "_cache"]
    old = cache if case["layout"] == "NHD" else cache.transpose(1, 2)
    new = torch.zeros(old.shape, device="cuda")
    new[at, off] = x
    written = torch.zeros(old.shape[:2], dtype=torch.bool, device="cuda")
    written[at, off] = True
    begins, touched = written[:, :1], written.any(1, keepdim=True)
    before = torch.where(begins, 0.0, scale)
    now = torch.where(touched, torch.maximum(before, new.abs().amax((1, 3)) / top), scale)
    now4, grows = now[:, None, :, None], (touched & ~begins & (now > before))[:, None, :, None]
    fresh = _round(torch.where(now4 > 0, new / now4, 0.0), codes)
    moved = _round(old.float() * (before / now)[:, None, :, None], codes)
    kept = torch.where(grows, moved.float(), old.float())
    kept = torch.where(written[:, :, None, None], fresh.float(), kept).to(cache.dtype)
    old.copy_(kept)
    scale.copy_(now)
    return kept


# ---- 64 bits -------------------------------------------------------------------------------------------------------------


def exact(case: dict, seed: int):
    st = prepare(case, seed)
    if case["kind"] == "append":
        return _exact_append(case, st)
    if case["kind"] == "select":
        return None  # whole numbers alone
    page, group = case["page_size"], case["q_heads"] // case["kv_heads"]
    out = torch.zeros(st["q"].shape, dtype=torch.float64, device="cuda")
    for t in range(case["tokens"]):
        last = int(st["positions"][t])
        row = st["page_table"][int(st["sequence_ids"][t])]
        for h in range(case["kv_heads"]):
            if case["kind"] == "attend":
                chosen = range(last // page + 1)
            else:
                chosen = [p for p in st["pages"][t, h].tolist() if p >= 0]
            logical = torch.tensor(list(chosen), device="cuda")
            physical = row[logical]
            live = (logical[:, None] * page + torch.arange(page, device="cuda") <= last).flatten()

            def block(cache, scale):
                part = cache[:, :, h] if case["layout"] == "NHD" else cache[:, h]
                values = part.view(torch.uint8)[physical].view(cache.dtype).double() * scale[physical, h].double()[:, None, None]
                return values.flatten(0, 1)[live]

            k, v = block(st["k_cache"], st["k_scale"]), block(st["v_cache"], st["v_scale"])
            mine = slice(h * group, (h + 1) * group)
            weights = torch.softmax(st["q"][t, mine].double() @ k.T / math.sqrt(case["head_dim"]), dim=-1)
            out[t, mine] = weights @ v
    return out


def _exact_append(case, st):
    """Rotated Q, and the scales; what the codes are rounded to has no value of more bits."""
    half, pos = case["rope_dim"] // 2, st["positions"]
    z = torch.complex(st["cos"][pos].double(), st["sin"][pos].double())[:, None, :half]

    def turned(x):
        x = x.double()
        front = x[..., :case["rope_dim"]]
        pairs = front.unflatten(-1, (half, 2)) if case["interleaved"] else front.unflatten(-1, (2, half)).transpose(-1, -2)
        w = torch.view_as_real(torch.view_as_complex(pairs.contiguous()) * z)
        w = w if case["interleaved"] else w.transpose(-1, -2)
        return torch.cat([w.flatten(-2), x[..., case["rope_dim"]:]], dim=-1)

    page, top = case["page_size"], _CODES[case["codes"]][1]
    seqs, logical, off = st["sequence_ids"].tolist(), (pos // page).tolist(), (pos % page).tolist()
    result = dict(q_rot=turned(st["q"]), k=None, v=None, k_mean=None)
    for name, x in (("k_scale", turned(st["k"])), ("v_scale", st["v"].double())):
        most = (x.abs().amax(-1) / top).cpu()
        scale, begun = st[name].double().cpu(), set()
        table = st["page_table"].cpu()
        where = [int(table[s, p]) for s, p in zip(seqs, logical)]
        for block, row in zip(where, off):
            if row == 0 and block not in begun:
                begun.add(block)
                scale[block] = 0
        for block, value in zip(where, most):
            scale[block] = torch.maximum(scale[block], value)
        result[name] = scale
    return result


def work(case: dict) -> dict:
    """Bytes: every operand that the operator needs read once, every result written once."""
    tokens, hq, hkv, dim, page = (case[n] for n in ("tokens", "q_heads", "kv_heads", "head_dim", "page_size"))
    elt = _DTYPES[case["dtype"]].itemsize
    if case["kind"] == "append":
        rows = elt * tokens * dim * (2 * hq + 2 * hkv) + 2 * tokens * hkv * dim  # q in and out, k and v in, their codes out
        touched = min(tokens, tokens // page + 2 * case["sequences"])
        return dict(bytes=rows + 4 * tokens * case["rope_dim"] + 24 * tokens + 16 * touched * hkv, flops=0)
    context = case["context"] - case["context"] / 200 if case["full"] else (case["context"] + 1) / 2  # in the mean
    blocks = context / page
    ends = 2 * elt * tokens * hq * dim
    if case["kind"] == "select":
        return dict(bytes=ends / 2 + tokens * hkv * (blocks * (dim + 4) + 4 * case["top_pages"]) + 8 * tokens * blocks,
                    flops=2 * tokens * hq * dim * blocks)
    if case["kind"] == "sparse":
        blocks = min(blocks, case["top_pages"])
        context = blocks * page
    nbytes = tokens * hkv * (2 * context * dim + 8 * blocks) + ends
    return dict(bytes=nbytes + (4 * tokens * hkv * case["top_pages"] if case["kind"] == "sparse" else 8 * tokens * blocks),
                flops=4 * tokens * hq * dim * context)
