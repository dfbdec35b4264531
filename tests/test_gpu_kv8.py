"""The 8-bit paged cache on the GPU: append, attention, selection of pages and the attention over them, against the restatement of
oracle/kv8.py (codes, scales, means and choices bit for bit, attention against 64 bits)."""

from __future__ import annotations

import pytest
import torch

from oracle import kv8 as oracle

pytestmark = pytest.mark.gpu

INT8, E4M3 = torch.int8, torch.float8_e4m3fn
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


def _gen(seed):
    return torch.Generator().manual_seed(seed)


def _table(sequences, per_seq, seed):
    return torch.randperm(sequences * per_seq, generator=_gen(seed)).reshape(sequences, per_seq)


def _trig(positions, rope_dim, width=None):
    angle = torch.arange(positions).double()[:, None] * 10000.0 ** (-torch.arange(0, rope_dim, 2).double() / rope_dim)[None]
    pad = torch.zeros(positions, (width or rope_dim // 2) - rope_dim // 2)
    return torch.cat([angle.cos().float(), pad], 1), torch.cat([angle.sin().float(), pad], 1)


def _bits(t):
    return t.view(torch.uint8) if t.element_size() == 1 else t


def _on_gpu(cache, layout):
    from cross_dsl_kernels_b200.kv8 import PagedKV8Cache
    move = (lambda t: t.cuda()) if layout == "NHD" else (lambda t: _bits(t).transpose(1, 2).contiguous().view(t.dtype).cuda())
    return PagedKV8Cache(move(cache["k"]), move(cache["v"]), cache["k_scale"].cuda(), cache["v_scale"].cuda(), cache["k_mean"].cuda(), layout)


def _same(ours, cache):
    """Codes (also of slots that were never written), scales and means, bit for bit."""
    for name in ("k", "v"):
        got = _bits(getattr(ours, name)).cpu()
        assert torch.equal(got if ours.kv_layout == "NHD" else got.transpose(1, 2), _bits(cache[name])), name
    for name in ("k_scale", "v_scale", "k_mean"):
        assert torch.equal(torch.nan_to_num(getattr(ours, name).cpu(), nan=-1.0), torch.nan_to_num(cache[name], nan=-1.0)), name


def _values(tokens, heads, dim, dtype, g, spread=3.0):
    """Values whose size differs from token to token, so that scales grow along a page."""
    return (torch.randn(tokens, heads, dim, generator=g) * torch.exp(spread * torch.randn(tokens, 1, 1, generator=g))).clamp(-3e4, 3e4).to(dtype)


def _filled(pages, page, heads, dim, codes, seed):
    """A cache of normal codes, whose scales lie over a factor of a thousand."""
    g = _gen(seed)
    cache = oracle.empty(pages, page, heads, dim, codes)
    for name in ("k", "v"):
        x = (torch.randn(pages, page, heads, dim, generator=g) * oracle.TOP[codes] / 4).clamp(-oracle.TOP[codes], oracle.TOP[codes])
        cache[name] = (x.round() if codes == INT8 else x).to(codes)
        cache[name + "_scale"] = torch.exp(1.5 * torch.randn(pages, heads, generator=g)) * (0.1 if name == "v" else 2.0) / oracle.TOP[codes]
    cache["k_mean"] = torch.randint(-40, 41, (pages, heads, dim), generator=g).to(torch.int8)
    return cache


def _append(ours, cache, q, k, v, trig, pos, table, seq, **kw):
    """Both sides; returns rotated q, which has to have the same bits."""
    from cross_dsl_kernels_b200.kv8 import rope_gqa_paged_kv8_append
    want = oracle.append(q, k, v, *trig, pos, table, seq, cache, **kw)
    got = rope_gqa_paged_kv8_append(*(t.cuda() for t in (q, k, v, *trig, pos, table, seq)), ours, **kw)
    assert torch.equal(got.cpu(), want)
    _same(ours, cache)
    return got


# (q heads, kv heads), head_dim, page, rope_dim, interleaved
SHAPES = [((8, 2), 128, 16, 128, False), ((6, 2), 64, 7, 32, False), ((2, 1), 256, 5, 256, True), ((4, 4), 64, 1, 64, True),
          ((3, 1), 128, 40, 6, False), ((4, 2), 64, 16, 10, True)]


@pytest.mark.parametrize("codes", [INT8, E4M3])
@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("heads,dim,page,rope,interleaved", SHAPES)
def test_append_step_by_step(codes, dtype, heads, dim, page, rope, interleaved):
    """Three sequences from their first token on, one of which pauses (padding): blocks begin, grow and fill up."""
    g, layout = _gen(dim + page), "HND" if page % 2 else "NHD"
    steps = min(2 * page + 2, 40)
    table, cache = _table(3, -(-steps // page), 1), oracle.empty(3 * -(-steps // page), page, heads[1], dim, codes)
    ours, trig = _on_gpu(cache, layout), _trig(steps, rope)
    seq = torch.tensor([2, 0, 1])
    for step in range(steps):
        pos = torch.tensor([step, step if step % 3 else -1, step])
        _append(ours, cache, *(_values(3, h, dim, dtype, g) for h in (heads[0], heads[1], heads[1])), trig, pos, table, seq, rope_dim=rope,
                interleaved=interleaved)


@pytest.mark.parametrize("codes", [INT8, E4M3])
@pytest.mark.parametrize("tokens", [5, 128, 129, 700])
@pytest.mark.parametrize("order", ["runs", "mixed", "shuffled"])
def test_append_chunks_in_any_order(codes, tokens, order):
    """Prefill chunks of four sequences that begin and end inside pages, in three orders, with padding between: one launch up to
    128 tokens, grouped by page above."""
    heads, dim, page, g = (4, 2), 64, 16, _gen(tokens)
    each = -(-tokens // 4)
    i = torch.arange(tokens)
    seq, step = (i // each, i % each) if order != "mixed" else (i % 4, i // 4)
    pos = torch.tensor([0, 5, 16, 31])[seq] + step
    pos[3::11] = -1
    if order == "shuffled":
        mix = torch.randperm(tokens, generator=g)
        seq, pos = seq[mix], pos[mix]
    per_seq = (each + 31) // page + 1
    table, cache = _table(4, per_seq, 2), _filled(4 * per_seq, page, heads[1], dim, codes, 3)
    ours = _on_gpu(cache, "NHD")
    for _ in range(2):  # the second call writes the same slots again
        _append(ours, cache, *(_values(tokens, h, dim, BF16, g, 1.0) for h in (4, 2, 2)), _trig(each + 40, dim), pos, table, seq, rope_dim=dim,
                interleaved=False)


@pytest.mark.parametrize("codes", [INT8, E4M3])
@pytest.mark.parametrize("heads,dim,page", [((4, 2), 64, 40), ((2, 1), 256, 24), ((9, 3), 128, 64), ((6, 6), 64, 7), ((3, 3), 256, 33)])
def test_append_long_chunks_of_any_page(codes, heads, dim, page):
    """Prompts that fill some pages and end inside others, then their next chunk: pages of few and of many rows."""
    g, lens, layout = _gen(dim + page), [210, 90], "HND" if page % 2 else "NHD"
    per_seq = -(-2 * max(lens) // page)
    table, cache = _table(2, per_seq, 3), oracle.empty(2 * per_seq, page, heads[1], dim, codes)
    ours, trig = _on_gpu(cache, layout), _trig(2 * max(lens), dim)
    seq = torch.cat([torch.full((n,), i) for i, n in enumerate(lens)])
    for chunk in range(2):
        pos = torch.cat([torch.arange(n) + chunk * n for n in lens])
        _append(ours, cache, *(_values(300, h, dim, F16, g, 1.0) for h in (heads[0], heads[1], heads[1])), trig, pos, table, seq, rope_dim=dim,
                interleaved=False)


@pytest.mark.parametrize("tokens", [9, 200])
def test_append_several_tokens_for_one_slot(tokens):
    """Of tokens for the same slot the last one counts, in every launch form."""
    g, page = _gen(tokens), 4
    pos, seq = torch.randint(0, 6, (tokens,), generator=g), torch.randint(0, 2, (tokens,), generator=g)
    table, cache = _table(2, 2, 4), _filled(4, page, 1, 64, INT8, 5)
    _append(_on_gpu(cache, "HND"), cache, *(_values(tokens, 1, 64, F32, g) for _ in range(3)), _trig(8, 64), pos, table, seq, rope_dim=64,
            interleaved=False)


@pytest.mark.parametrize("codes", [INT8, E4M3])
def test_append_extremes(codes):
    """Zeros, values whose scale is subnormal or underflows, the largest of the type, and a block that is given a value that is not
    finite: NaN until its page begins anew."""
    page, table, seq, trig = 4, torch.tensor([[1, 0], [3, 2]]), torch.tensor([0, 1]), _trig(8, 64)
    cache = oracle.empty(4, page, 1, 64, codes)
    ours = _on_gpu(cache, "NHD")

    def put(pos, k, v):
        q = torch.ones(2, 1, 64)
        _append(ours, cache, q, torch.tensor(k).reshape(2, 1, 1).expand(2, 1, 64).contiguous(),
                torch.tensor(v).reshape(2, 1, 1).expand(2, 1, 64).contiguous(), trig, torch.tensor(pos), table, seq, rope_dim=64, interleaved=False)

    put([0, 0], [0.0, 1e-44], [1e-45, 2.8e-43])
    put([1, 1], [1.0, 0.0], [3e38, 1e-40])
    put([2, 2], [float("inf"), 1.0], [1.0, float("nan")])
    assert torch.isnan(ours.k_scale[1]).all() and torch.isnan(ours.v_scale[3]).all()
    put([3, 3], [2.0, 3.0], [2.0, 3.0])
    assert torch.isnan(ours.k_scale[1]).all() and torch.isnan(ours.v_scale[3]).all()
    put([0, 0], [2.0, 3.0], [2.0, 3.0])
    assert torch.isfinite(ours.k_scale).all() and torch.isfinite(ours.v_scale).all()


def test_append_takes_slices_of_a_fused_projection_and_wide_tables():
    g, dim = _gen(8), 64
    qkv = torch.randn(5, 8 * dim + 3, generator=g).half()[:, :8 * dim].view(5, 8, dim).cuda()  # rows that are not 16-byte aligned
    from cross_dsl_kernels_b200.kv8 import rope_gqa_paged_kv8_append
    cache, table, pos, seq = _filled(10, 16, 2, dim, E4M3, 9), _table(5, 2, 9), torch.tensor([0, 3, 15, 16, 31]), torch.arange(5)
    ours, trig = _on_gpu(cache, "NHD"), _trig(32, dim, width=37)
    parts = qkv.split((4, 2, 2), dim=1)
    want = oracle.append(*(p.cpu() for p in parts), *trig, pos, table, seq, cache, rope_dim=dim, interleaved=False)
    got = rope_gqa_paged_kv8_append(*parts, *(t.cuda() for t in (*trig, pos, table, seq)), ours, rope_dim=dim, interleaved=False)
    assert torch.equal(got.cpu(), want)
    _same(ours, cache)


@pytest.mark.parametrize("codes", [INT8, E4M3])
@pytest.mark.parametrize("tokens", [100, 900])
def test_append_quotients(codes, tokens):
    """Quotients on and next to the middle between two codes, for scales from the smallest subnormal to beyond the middle of the
    exponents' range, with significands of all ones among them: the bytes of a division that is rounded once."""
    g, dim, top = _gen(tokens), 256, oracle.TOP[codes]
    most = torch.ldexp(1 + torch.rand(tokens, generator=g), torch.linspace(-149, 126, tokens).round().int())
    most[::7] = torch.ldexp(torch.full_like(most, 2 - 2.0 ** -23), torch.linspace(-149, 126, tokens).round().int())[::7]
    scale = most * (torch.tensor(1.0) / top)
    every = torch.arange(256, dtype=torch.uint8).view(codes).double()
    every = every[every.isfinite()].sort().values
    middle = ((every[1:] + every[:-1]) / 2)[torch.randint(0, every.numel() - 1, (tokens, dim), generator=g)]
    x = (middle * scale.double()[:, None]).float()
    step = torch.randint(-1, 2, x.shape, generator=g)
    x = torch.where(step == 0, x, torch.nextafter(x, step * torch.inf))
    x = x.clamp(-most[:, None], most[:, None])
    x[:, 0] = most
    cache, pos = oracle.empty(tokens, 1, 1, dim, codes), torch.zeros(tokens, dtype=torch.int64)
    _append(_on_gpu(cache, "NHD"), cache, *(t[:, None].contiguous() for t in (x, x, -x)), _trig(1, dim), pos, _table(tokens, 1, 1),
            torch.arange(tokens), rope_dim=dim, interleaved=False)


@pytest.mark.parametrize("tokens", [128, 300])
def test_append_without_means_captured_twice(tokens):
    """Two graphs of one stream, each a prompt's append with what it needs besides, replayed in turn on changed inputs; no mean keys."""
    from dataclasses import replace
    from cross_dsl_kernels_b200.kv8 import rope_gqa_paged_kv8_append
    g, dim, page = _gen(tokens), 64, 16
    trig, pos, seq = _trig(512, dim), torch.arange(tokens) % 150, torch.arange(tokens) // 150
    table = _table(3, 10, 5)
    caches = [_filled(30, page, 2, dim, codes, 6) for codes in (INT8, E4M3)]
    ours = [replace(_on_gpu(cache, "HND"), k_mean=None) for cache in caches]
    inputs = [torch.zeros(tokens, h, dim, dtype=BF16, device="cuda") for h in (4, 2, 2)]
    index, dev = [pos.cuda(), table.cuda(), seq.cuda()], [t.cuda() for t in trig]
    stream, graphs, outs = torch.cuda.Stream(), [], []
    with torch.cuda.stream(stream):
        for cache in ours:
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=stream):
                outs.append(rope_gqa_paged_kv8_append(*inputs, *dev, *index, cache, rope_dim=dim, interleaved=True, dependent_launch=True))
            graphs.append(graph)
    torch.cuda.synchronize()
    for _ in range(3):
        fresh = [_values(tokens, h, dim, BF16, g) for h in (4, 2, 2)]
        for to, x in zip(inputs, fresh):
            to.copy_(x)
        for graph in graphs:
            graph.replay()
        torch.cuda.synchronize()
        for cache, own, out in zip(caches, ours, outs):
            means = cache["k_mean"].clone()
            want = oracle.append(*fresh, *trig, pos, table, seq, cache, rope_dim=dim, interleaved=True)
            cache["k_mean"] = means  # the restatement always keeps them
            assert torch.equal(out.cpu(), want)
            _same(replace(own, k_mean=means.cuda()), cache)


# ---- attention -------------------------------------------------------------------------------------------------------------


def _close(got, exact, dtype, dim):
    """Half a step of the output type, and sum_j p_j |v_j| times what the weights are off by.  16-bit q: it is exact, a weight is rounded
    to FP16 once (2^-11 of it).  FP32 q: two FP16 numbers leave 2^-21 of a weight and of a product of the scores.  Either way FP32 sums:
    a score is off by at most 2^-22 of sum |q_d k_d| per matrix product of its chain (truncation; 2 dim / 16 of them, and its scaling), a
    weight by twice that (exp, and the sum it is divided by), and the accumulators by 2^-18.  Weights are taken relative to the largest,
    times 2^14, so that a step of the smallest FP16 numbers, 2^-24, is 2^-38 of it: a code is off by half of that, wherever the largest
    weight meets codes of 0 and nothing else is left to see.  int8 codes under 16-bit q enter as code + 128: a matrix product
    cuts its 16 terms and its sum at 2^-24 of the largest of them, which is up to 128 * |the sum of q_d behind it| or 256 * |q_d| (17 * 2^-24 < 2^-19 of
    that, dim / 16 products to a score), or 256 * the weights (two products, and their own sum rounded 8 times: 2^-18 of 128 * the sum)."""
    bound, score = exact["bound"], exact["score"]
    chain, lift = 2 * dim // 16 + 4, 0.0 if dtype == F32 else 128.0
    lost = 2 * (score * (chain * 2.0 ** -22 + 2.0 ** -21) + lift * exact["offset"] * dim / 16 * 2.0 ** -19)
    weight = 2.0 ** (-21 if dtype == F32 else -11) + 2.0 ** -18 + lost[..., None]
    info = torch.finfo(dtype)  # half a step of a subnormal result is that of the smallest normal one
    limit = bound * weight * 1.01 + exact["least"] * 2.0 ** -39 + lift * exact["flat"][..., None] * 2.0 ** -18
    limit = limit + torch.clamp(exact["result"].abs(), min=info.smallest_normal) * info.eps / 2
    finite, far = bool(torch.isfinite(got).all()), float(((got.double().cpu() - exact["result"]).abs() / limit).max())
    assert finite and far <= 1.0


def _attend_inputs(heads, dim, page, positions, codes, seed, per_seq=None):
    tokens = len(positions)
    per_seq = per_seq or max(max(positions), 0) // page + 1
    cache = _filled(tokens * per_seq, page, heads[1], dim, codes, seed)
    return cache, torch.tensor(positions), _table(tokens, per_seq, seed), torch.randperm(tokens, generator=_gen(seed))


MIXES = [((8, 2), 128, 16, [0, 1, 15, 16, 31, 32, 127, 128, -1, 300]), ((6, 2), 64, 7, [1000, -1, 0, 6, 7, 500]),
         ((5, 1), 256, 32, [63, 0, 130]), ((8, 1), 128, 1, [0, 200]), ((7, 7), 64, 64, [70, 2]),
         ((4, 1), 128, 16, [5000, 0, 3000, -1, 63, 64, 1, 127, 128, 2047]),  # items inside one CTA, across two, across many
         ((2, 2), 64, 16, [-1] * 3), ((2, 1), 64, 5, [i % 90 - 1 for i in range(300)])]


@pytest.mark.parametrize("codes", [INT8, E4M3])
@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("heads,dim,page,positions", MIXES)
def test_attention(codes, dtype, heads, dim, page, positions):
    """Contexts of every mix and none, groups of any size up to eight, for each bound the caller may name (the split follows it): within the
    rounding of the formula, zeros where there is nothing to attend to, the same bits every time."""
    from cross_dsl_kernels_b200.kv8 import paged_kv8_decode_attention
    cache, pos, table, seq = _attend_inputs(heads, dim, page, positions, codes, seed=dim + len(positions))
    q = torch.randn(len(positions), heads[0], dim, generator=_gen(1)).to(dtype)
    exact = oracle.attention(q, cache, pos, table, seq)
    args = [t.cuda() for t in (pos, table, seq)]
    for layout in ("NHD", "HND"):
        ours = _on_gpu(cache, layout)
        for hint in (0, 1, 100000):
            got = paged_kv8_decode_attention(q.cuda(), ours, *args, context_hint=hint)
            _close(got, exact, dtype, dim)
            assert (got[(pos < 0).cuda()] == 0).all()
            assert torch.equal(got, paged_kv8_decode_attention(q.cuda(), ours, *args, context_hint=hint)), "deterministic"


@pytest.mark.parametrize("codes", [INT8, E4M3])
@pytest.mark.parametrize("dtype", [F16, BF16, F32])
def test_attention_over_scales_of_any_size(codes, dtype):
    """Scales of V over thirty powers of ten, and q from the smallest to the largest of its type: what matters keeps its bits."""
    from cross_dsl_kernels_b200.kv8 import paged_kv8_decode_attention
    cache, pos, table, seq = _attend_inputs((4, 2), 64, 16, [200, 97, 2000], codes, seed=4)
    g = _gen(2)
    cache["v_scale"] = 10.0 ** (30 * torch.rand(cache["v_scale"].shape, generator=g) - 28)
    cache["k_scale"] = cache["k_scale"] * 1e-3
    q = torch.randn(3, 4, 64, generator=g) * torch.tensor([1.0, 1e-6, 3e4]).reshape(3, 1, 1)
    q[2] = (q[2] * 1e-2).clamp(-200, 200)
    q[0, 1] = 0
    q = q.to(dtype)
    exact = oracle.attention(q, cache, pos, table, seq)
    if dtype == F16:  # results beyond the type are infinite
        keep = exact["result"].abs().amax(-1, keepdim=True) < 6e4
        exact = {name: x * (keep if x.dim() == 3 else keep[..., 0]) for name, x in exact.items()}
    got = paged_kv8_decode_attention(q.cuda(), _on_gpu(cache, "NHD"), *(t.cuda() for t in (pos, table, seq)))
    if dtype == F16:
        got = torch.where(keep.cuda(), got, torch.zeros_like(got))
    _close(got, exact, dtype, 64)


def test_attention_not_a_number_shows():
    """A block whose scale is NaN reaches the heads that read it and no others, whether K's or V's."""
    from cross_dsl_kernels_b200.kv8 import paged_kv8_decode_attention
    cache, pos, table, seq = _attend_inputs((8, 2), 128, 16, [4000, 5, 2000], INT8, seed=6)
    cache["k_scale"][int(table[seq[0], 2500 // 16]), 1] = float("nan")
    cache["v_scale"][int(table[seq[2], 100 // 16]), 0] = float("nan")
    q = torch.randn(3, 8, 128, generator=_gen(1)).half().cuda()
    got = paged_kv8_decode_attention(q, _on_gpu(cache, "HND"), *(t.cuda() for t in (pos, table, seq))).cpu()
    assert torch.isnan(got[0, 4:]).all() and torch.isfinite(got[0, :4]).all() and torch.isfinite(got[1]).all()
    assert torch.isnan(got[2, :4]).all() and torch.isfinite(got[2, 4:]).all()


def test_attention_far_into_a_large_cache():
    """Offsets beyond 32 bits: pages at the end of caches of more than 2^32 bytes."""
    from cross_dsl_kernels_b200 import kv8
    pages, page, heads, dim = (1 << 32) // (64 * 4 * 128) + 9, 64, 4, 128
    if torch.cuda.mem_get_info()[0] < 12 << 30:
        pytest.skip("needs 12 GB of device memory")
    ours = kv8.PagedKV8Cache(*(torch.empty(pages, page, heads, dim, dtype=INT8, device="cuda") for _ in range(2)),
                             *(torch.empty(pages, heads, device="cuda") for _ in range(2)), torch.zeros(pages, heads, dim, dtype=INT8, device="cuda"))
    small = _filled(4, page, heads, dim, INT8, 7)
    for name in ("k", "v", "k_scale", "v_scale", "k_mean"):
        getattr(ours, name)[-4:] = small[name].cuda()
    pos, seq, near = torch.tensor([255]), torch.tensor([0]), torch.tensor([[2, 0, 3, 1]])
    q = torch.randn(1, 8, dim, generator=_gen(3)).half()
    far = (near + pages - 4).cuda()
    exact = oracle.attention(q, small, pos, near, seq)
    _close(kv8.paged_kv8_decode_attention(q.cuda(), ours, pos.cuda(), far, seq.cuda()), exact, F16, dim)
    chosen = kv8.select_kv8_pages(q.cuda(), ours, pos.cuda(), far, seq.cuda(), top_pages=2)
    assert torch.equal(chosen.cpu(), oracle.select(q, small, pos, near, seq, top_pages=2))
    exact = oracle.attention(q, small, pos, near, seq, pages=chosen.cpu())
    _close(kv8.paged_kv8_sparse_attention(q.cuda(), ours, chosen, pos.cuda(), far, seq.cuda()), exact, F16, dim)
    k = torch.randn(1, heads, dim, generator=_gen(4)).half()
    trig = _trig(256, dim)
    want = oracle.append(q, k, k, *trig, pos, near, seq, small, rope_dim=dim, interleaved=False)
    got = kv8.rope_gqa_paged_kv8_append(*(t.cuda() for t in (q, k, k, *trig, pos)), far, seq.cuda(), ours, rope_dim=dim, interleaved=False)
    assert torch.equal(got.cpu(), want)
    for name in ("k", "v", "k_scale", "v_scale", "k_mean"):
        assert torch.equal(getattr(ours, name)[-4:].cpu(), small[name]), name


@pytest.mark.parametrize("tokens,heads", [(65535, (2, 1)), (2500, (9, 3))])
def test_many_tokens(tokens, heads):
    """The most tokens a call takes, of few sequences over and over, for all three ops that read the cache."""
    from cross_dsl_kernels_b200 import kv8
    dim, page, few = 64, 8, 61
    cache, pos, table, seq = _attend_inputs(heads, dim, page, [(i * 37) % 100 - 1 for i in range(few)], INT8, seed=17)
    q = torch.randn(few, heads[0], dim, generator=_gen(17)).half()
    of, ours = torch.arange(tokens) % few, _on_gpu(cache, "NHD")
    args = [pos[of].cuda(), table.cuda(), seq[of].cuda()]
    many = lambda exact: {name: x[of] for name, x in exact.items()}  # noqa: E731
    chosen = oracle.select(q, cache, pos, table, seq, top_pages=4)
    assert torch.equal(kv8.select_kv8_pages(q[of].cuda(), ours, *args, top_pages=4).cpu(), chosen[of])
    whole, some = oracle.attention(q, cache, pos, table, seq), oracle.attention(q, cache, pos, table, seq, pages=chosen)
    for hint in (0, 100):
        _close(kv8.paged_kv8_decode_attention(q[of].cuda(), ours, *args, context_hint=hint), many(whole), F16, dim)
    _close(kv8.paged_kv8_sparse_attention(q[of].cuda(), ours, chosen[of].cuda(), *args), many(some), F16, dim)


@pytest.mark.parametrize("dtype", [F16, F32])
def test_q_that_begins_anywhere(dtype):
    """A contiguous q whose first element is not on a 16-byte boundary: the same bits as one on it."""
    from cross_dsl_kernels_b200 import kv8
    cache, pos, table, seq = _attend_inputs((8, 2), 128, 16, [700, 3, -1], E4M3, seed=18)
    q = torch.randn(3, 8, 128, generator=_gen(18)).to(dtype).cuda()
    shifted = torch.empty(q.numel() + 1, dtype=dtype, device="cuda")[1:].view_as(q)
    shifted.copy_(q)
    ours, args = _on_gpu(cache, "HND"), [t.cuda() for t in (pos, table, seq)]
    pages = kv8.select_kv8_pages(q, ours, *args, top_pages=5)
    assert torch.equal(pages, kv8.select_kv8_pages(shifted, ours, *args, top_pages=5))
    assert torch.equal(kv8.paged_kv8_decode_attention(q, ours, *args), kv8.paged_kv8_decode_attention(shifted, ours, *args))
    assert torch.equal(kv8.paged_kv8_sparse_attention(q, ours, pages, *args), kv8.paged_kv8_sparse_attention(shifted, ours, pages, *args))


# ---- selection and the attention over the selected pages -----------------------------------------------------------------------


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("heads,dim,page,positions,top", [
    ((8, 2), 128, 16, [0, 15, 16, 40, -1, 999, 1600], 8), ((3, 1), 64, 7, [3000, 48, 49], 1), ((8, 1), 256, 5, [700, 1], 2),
    ((5, 5), 64, 1, [2000, 511, 512, 513], 300), ((4, 4), 128, 4, [9000], 64), ((1, 1), 64, 8, [100], 1000)])
def test_selection(dtype, heads, dim, page, positions, top):
    """The same pages as the restatement, in order: few candidates and thousands, odd pages, one page, more than there are, none."""
    from cross_dsl_kernels_b200.kv8 import select_kv8_pages
    cache, pos, table, seq = _attend_inputs(heads, dim, page, positions, INT8, seed=top)
    q = torch.randn(len(positions), heads[0], dim, generator=_gen(5)).to(dtype)
    q[0, 0] = 0  # a head without a direction: its scores are all 0
    want = oracle.select(q, cache, pos, table, seq, top_pages=top)
    for layout in ("NHD", "HND"):
        assert torch.equal(select_kv8_pages(q.cuda(), _on_gpu(cache, layout), *(t.cuda() for t in (pos, table, seq)), top_pages=top).cpu(), want)


def test_selection_of_equals_and_of_not_a_number():
    """Equal scores go to the lowest pages, wherever in the order the last one chosen falls; a block that is NaN comes first."""
    from cross_dsl_kernels_b200.kv8 import select_kv8_pages
    cache, pos, table, seq = _attend_inputs((2, 1), 64, 4, [4 * 1500], INT8, seed=8)
    cache["k_mean"][:] = 1
    cache["k_scale"][:] = 0.5
    q = torch.ones(1, 2, 64)
    at = table[seq[0]]
    cache["k_scale"][at[torch.arange(700, 1500, 7)]] = 0.75
    for top in (2, 50, 116, 117, 600, 1500):
        want = oracle.select(q, cache, pos, table, seq, top_pages=top)
        assert torch.equal(select_kv8_pages(q.cuda(), _on_gpu(cache, "NHD"), *(t.cuda() for t in (pos, table, seq)), top_pages=top).cpu(), want)
    cache["k_scale"][at[1234]] = float("nan")
    got = select_kv8_pages(-q.cuda(), _on_gpu(cache, "NHD"), *(t.cuda() for t in (pos, table, seq)), top_pages=3).cpu()
    assert got.flatten().tolist() == [0, 1234, 1500]


@pytest.mark.parametrize("value", [float("inf"), float("-inf"), float("nan")])
def test_selection_by_a_q_that_is_not_finite(value):
    """No choice is better than another then; each is still one of pages of the context, ascending, the last one among them."""
    from cross_dsl_kernels_b200.kv8 import select_kv8_pages
    cache, pos, table, seq = _attend_inputs((4, 2), 64, 4, [1000, 399, 7], INT8, seed=19)
    q = torch.randn(3, 4, 64, generator=_gen(19))
    q[:, 1, 5] = value
    got = select_kv8_pages(q.cuda(), _on_gpu(cache, "NHD"), *(t.cuda() for t in (pos, table, seq)), top_pages=9).cpu()
    assert torch.equal(got[:, 1], oracle.select(q, cache, pos, table, seq, top_pages=9)[:, 1])  # the head that has numbers
    for t, last in ((0, 250), (1, 99)):
        assert (got[t].diff() > 0).all() and (got[t, :, 0] >= 0).all() and (got[t, :, -1] == last).all()
    assert got[2].tolist() == [[0, 1] + [-1] * 7] * 2


@pytest.mark.parametrize("codes", [INT8, E4M3])
@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("heads,dim,page,positions,lists", [
    ((8, 2), 128, 16, [0, 15, 16, 40, -1, 999, 1600], 8), ((3, 1), 64, 7, [3000, 48, 49], 5), ((8, 1), 256, 5, [700, 1], 30),
    ((5, 5), 64, 1, [200, 511], 130), ((4, 4), 128, 64, [9000], 40)])
def test_sparse_attention(codes, dtype, heads, dim, page, positions, lists):
    """Lists with holes, repeats, pages out of order and behind the context: what the documentation says each of them adds."""
    from cross_dsl_kernels_b200.kv8 import paged_kv8_sparse_attention
    cache, pos, table, seq = _attend_inputs(heads, dim, page, positions, codes, seed=lists)
    g, per_seq = _gen(lists), table.shape[1]
    q = torch.randn(len(positions), heads[0], dim, generator=g).to(dtype)
    pages = torch.randint(-1, per_seq + 2, (len(positions), heads[1], lists), generator=g).sort(-1).values
    pages[:, :, lists // 2] = pages[:, :, 0]  # below its neighbours
    pages[0] = -1
    pages = pages.to(torch.int32)
    exact = oracle.attention(q, cache, pos, table, seq, pages=pages)
    args = [t.cuda() for t in (pages, pos, table, seq)]
    for layout in ("NHD", "HND"):
        got = paged_kv8_sparse_attention(q.cuda(), _on_gpu(cache, layout), *args)
        _close(got, exact, dtype, dim)
        assert (got[0] == 0).all()


# ---- together ------------------------------------------------------------------------------------------------------------------


def _step(ours, q, k, v, trig, pos, table, seq, top, **kw):
    from cross_dsl_kernels_b200 import kv8
    q = kv8.rope_gqa_paged_kv8_append(q, k, v, *trig, pos, table, seq, ours, rope_dim=q.shape[2], interleaved=False, **kw)
    pages = kv8.select_kv8_pages(q, ours, pos, table, seq, top_pages=top, **kw)
    return (q, kv8.paged_kv8_decode_attention(q, ours, pos, table, seq, **kw), pages,
            kv8.paged_kv8_sparse_attention(q, ours, pages, pos, table, seq, **kw))


@pytest.mark.parametrize("codes", [INT8, E4M3])
def test_a_prompt_and_the_steps_behind_it(codes):
    """Prefill of two prompts, then decode steps, each op on what the one before it left: eagerly, captured and replayed, with and
    without dependent launches -- the same bits; and against the restatement on its own cache."""
    heads, dim, page, top, dtype = (8, 2), 64, 8, 6, F16
    g, lens = _gen(11), [150, 75]
    table, trig = _table(2, 24, 11).cuda(), _trig(192, dim)
    cache = oracle.empty(48, page, heads[1], dim, codes)
    ours, again = _on_gpu(cache, "NHD"), _on_gpu(cache, "NHD")
    pos = torch.cat([torch.arange(n) for n in lens])
    seq = torch.cat([torch.full((n,), i) for i, n in enumerate(lens)])
    dev = [t.cuda() for t in trig]
    prompt = [torch.randn(225, h, dim, generator=g).to(dtype) for h in (8, 2, 2)]
    _append(ours, cache, *prompt, trig, pos, table.cpu(), seq, rope_dim=dim, interleaved=False)
    from cross_dsl_kernels_b200.kv8 import rope_gqa_paged_kv8_append
    rope_gqa_paged_kv8_append(*(t.cuda() for t in prompt), *dev, pos.cuda(), table, seq.cuda(), again, rope_dim=dim, interleaved=False)

    inputs = [torch.empty(2, h, dim, dtype=dtype, device="cuda") for h in (8, 2, 2)]
    at, both = torch.tensor(lens, device="cuda"), torch.arange(2, device="cuda")
    graph = None
    for step in range(20):
        fresh = [torch.randn(2, h, dim, generator=g).to(dtype) for h in (8, 2, 2)]
        for to, x in zip(inputs, fresh):
            to.copy_(x)
        got = _step(ours, *inputs, dev, at, table, both, top)
        if graph is None:
            stream = torch.cuda.Stream()
            with torch.cuda.stream(stream):  # two layers' worth on one stream; capture runs nothing
                graph = torch.cuda.CUDAGraph()
                with torch.cuda.graph(graph, stream=stream):
                    replayed = _step(again, *inputs, dev, at, table, both, top, dependent_launch=True)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, replayed))
        want_q = oracle.append(*fresh, *trig, at.cpu(), table.cpu(), both.cpu(), cache, rope_dim=dim, interleaved=False)
        assert torch.equal(got[0].cpu(), want_q)
        _same(ours, cache)
        _same(again, cache)
        pages = oracle.select(want_q, cache, at.cpu(), table.cpu(), both.cpu(), top_pages=top)
        assert torch.equal(got[2].cpu(), pages)
        for out, kept in ((got[1], None), (got[3], pages)):
            _close(out, oracle.attention(want_q, cache, at.cpu(), table.cpu(), both.cpu(), pages=kept), dtype, dim)
        at += 1


def test_all_pages_selected_is_the_whole_context():
    from cross_dsl_kernels_b200 import kv8
    cache, pos, table, seq = _attend_inputs((8, 2), 128, 16, [500, 0, -1, 77], E4M3, seed=12)
    ours, q = _on_gpu(cache, "HND"), torch.randn(4, 8, 128, generator=_gen(12)).half()
    args = [t.cuda() for t in (pos, table, seq)]
    pages = kv8.select_kv8_pages(q.cuda(), ours, *args, top_pages=40)
    exact = oracle.attention(q, cache, pos, table, seq)
    _close(kv8.paged_kv8_sparse_attention(q.cuda(), ours, pages, *args), exact, F16, 128)


@pytest.mark.parametrize("tokens", [7, 200])
def test_padding_names_no_sequence(tokens):
    """A padded batch: what stands in the sequence ids of padding, and in the page table behind a context, is nothing that is read."""
    from cross_dsl_kernels_b200 import kv8
    heads, dim, page, g = (4, 2), 128, 16, _gen(21)
    cache, table = _filled(30, page, 2, dim, INT8, 21), torch.full((2, 40), 1 << 40)
    table[:, :15] = torch.randperm(30, generator=g).reshape(2, 15)
    pos, seq = torch.full((tokens,), -1), torch.full((tokens,), 1 << 50)
    pos[2:7:2], seq[2:7:2] = torch.tensor([100, 239, 16]), torch.tensor([0, 1, 1])
    pos[0] = -(1 << 40)
    seq[3] = -9
    ours = _on_gpu(cache, "NHD")
    q, k, v = (torch.randn(tokens, h, dim, generator=g).half() for h in (4, 2, 2))
    q = _append(ours, cache, q, k, v, _trig(256, dim), pos, table, seq, rope_dim=dim, interleaved=False)
    args = [t.cuda() for t in (pos, table, seq)]
    pages = kv8.select_kv8_pages(q, ours, *args, top_pages=3)
    assert torch.equal(pages.cpu(), oracle.select(q.cpu(), cache, pos, table, seq, top_pages=3))
    for got, kept in ((kv8.paged_kv8_decode_attention(q, ours, *args), None), (kv8.paged_kv8_sparse_attention(q, ours, pages, *args), pages.cpu())):
        _close(got, oracle.attention(q.cpu(), cache, pos, table, seq, pages=kept), F16, dim)
        assert (got[(pos < 0).cuda()] == 0).all()


def test_streams_and_a_wider_destination():
    """On a stream that is not the default one, behind work that is still running there; and the output as columns of a wider matrix."""
    from cross_dsl_kernels_b200 import _native, kv8
    cache, pos, table, seq = _attend_inputs((8, 2), 64, 16, [3000, 12], INT8, seed=13)
    ours, args = _on_gpu(cache, "NHD"), [t.cuda() for t in (pos, table, seq)]
    q = torch.randn(2, 8, 64, generator=_gen(13)).half().cuda()
    pages = kv8.select_kv8_pages(q, ours, *args, top_pages=9)
    want = kv8.paged_kv8_decode_attention(q, ours, *args), kv8.paged_kv8_sparse_attention(q, ours, pages, *args)
    torch.cuda.synchronize()
    stream, late = torch.cuda.Stream(), torch.zeros_like(q)
    with torch.cuda.stream(stream):
        torch.cuda._sleep(20_000_000)
        late.copy_(q)
        got = kv8.paged_kv8_decode_attention(late, ours, *args), kv8.paged_kv8_sparse_attention(late, ours, pages, *args)
        chosen = kv8.select_kv8_pages(late, ours, *args, top_pages=9)
    stream.synchronize()
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1]) and torch.equal(chosen, pages)
    for width, col in ((600, 40), (601, 40), (600, 41)):  # rows that begin on any element
        wide = torch.full((2, width), -7.0, dtype=F16, device="cuda")
        dst = _native.PeerOutStruct()
        dst.ptr[0], dst.world, dst.ld, dst.col0 = wide.data_ptr(), 1, width, col
        assert kv8.paged_kv8_decode_attention(q, ours, *args, peer_out=dst) is None
        mine = slice(col, col + 512)
        assert torch.equal(wide[:, mine], want[0].view(2, 512)) and (wide[:, :col] == -7).all() and (wide[:, col + 512:] == -7).all()
        kv8.paged_kv8_sparse_attention(q, ours, pages, *args, peer_out=dst)
        assert torch.equal(wide[:, mine], want[1].view(2, 512)) and (wide[:, :col] == -7).all() and (wide[:, col + 512:] == -7).all()


def test_two_streams_at_once():
    """Steps over two caches on two streams, whose kernels run side by side: what each gives alone."""
    heads, dim, page, top = (8, 2), 64, 16, 12
    g, trig = _gen(20), [t.cuda() for t in _trig(4096, dim)]
    sides = []
    for codes in (INT8, E4M3):
        cache, pos, table, seq = _attend_inputs(heads, dim, page, [4000, 31, 2222, 800], codes, seed=20)
        qkv = [torch.randn(4, h, dim, generator=g).half().cuda() for h in (8, 2, 2)]
        many = [torch.randn(300, h, dim, generator=g).half().cuda() for h in (8, 2, 2)]
        sides.append((cache, qkv, many, [t.cuda() for t in (pos, table, seq)]))

    def run(side, ours):
        from cross_dsl_kernels_b200.kv8 import rope_gqa_paged_kv8_append
        cache, qkv, many, (pos, table, seq) = side
        at, of = torch.arange(300, device="cuda") % 75, torch.arange(300, device="cuda") // 75
        got = []
        for step in range(6):
            got += _step(ours, *qkv, trig, pos + step, table, seq, top)
            got.append(rope_gqa_paged_kv8_append(*many, *trig, at + step, table, of, ours, rope_dim=dim, interleaved=False))
        return got

    alone = []
    for side in sides:
        alone.append(run(side, _on_gpu(side[0], "NHD")))
        torch.cuda.synchronize()
    streams, again, got = [torch.cuda.Stream() for _ in sides], [_on_gpu(side[0], "NHD") for side in sides], []
    torch.cuda.synchronize()
    for side, stream, ours in zip(sides, streams, again):
        with torch.cuda.stream(stream):
            torch.cuda._sleep(5_000_000)
            got.append(run(side, ours))
    torch.cuda.synchronize()
    for a, b in zip(alone, got):
        assert all(torch.equal(x, y) for x, y in zip(a, b))
