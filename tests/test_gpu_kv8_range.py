"""The attention over the 8-bit cache at the ends of its operands' range, against 64 bits."""

from __future__ import annotations

import pytest
import torch

from oracle import kv8 as oracle
from test_gpu_kv8 import BF16, E4M3, F16, F32, INT8, _attend_inputs, _close, _gen, _on_gpu

pytestmark = pytest.mark.gpu


def _reads(q, cache, pos, table, seq, dtype, layout="NHD", hints=(0, 1, 100000)):
    """Both reads, however the batch is split, against the formula."""
    from cross_dsl_kernels_b200 import kv8
    exact, dim = oracle.attention(q, cache, pos, table, seq), q.shape[2]
    assert torch.isfinite(exact["result"].to(dtype)).all()
    ours, args = _on_gpu(cache, layout), [t.cuda() for t in (pos, table, seq)]
    for hint in hints:
        _close(kv8.paged_kv8_decode_attention(q.cuda(), ours, *args, context_hint=hint), exact, dtype, dim)
    every = torch.arange(table.shape[1], dtype=torch.int32, device="cuda").expand(q.shape[0], cache["k"].shape[2], -1).contiguous()
    _close(kv8.paged_kv8_sparse_attention(q.cuda(), ours, every, *args), exact, dtype, dim)


@pytest.mark.parametrize("codes", [INT8, E4M3])
@pytest.mark.parametrize("dtype,exponents", [(F16, (-20, 0, 14)), (BF16, (-125, -60, 119, 120, 125)), (F32, (-125, -60, 119, 120, 125))])
def test_q_of_any_size(codes, dtype, exponents):
    """q from the smallest to the largest of its type, over keys as much smaller or larger, so that the scores are ordinary ones."""
    for exponent in exponents:
        cache, pos, table, seq = _attend_inputs((8, 2), 128, 16, [500, 40, 0], codes, seed=31)
        q = torch.randn(3, 8, 128, generator=_gen(31)).clamp(-3.9, 3.9)
        cache["k_scale"] = torch.ldexp(cache["k_scale"] * 0.2, torch.tensor(-exponent))
        q = torch.ldexp(q, torch.tensor(exponent))
        _reads(q.to(dtype), cache, pos, table, seq, dtype)
        q[:, 1::2] *= 2.0 ** -8  # heads of a group that differ
        _reads(q.to(dtype), cache, pos, table, seq, dtype)


def _scaled(cache, table, seq, rows):
    """`rows`: {slice of a context's pages: exponent, or None for blocks of zeros}; in all contexts."""
    scale = cache["v_scale"]
    for part, exponent in rows.items():
        at = table[seq][:, part].flatten()
        if exponent is None:
            scale[at] = 0
            cache["v"].view(torch.uint8)[at] = 0
        else:
            scale[at] = torch.ldexp(scale[at], torch.tensor(exponent))


FAR = {
    "first far below": {slice(0, 2): -120, slice(2, None): 8}, "first far above": {slice(0, 2): 30, slice(2, None): -100},
    "one far below": {slice(7, 8): -115}, "one far above": {slice(9, 10): 100}, "last far above": {slice(-1, None): 118},
    "first zero, tiny behind": {slice(0, 3): None, slice(3, None): -110}, "one zero": {slice(20, 21): None}, "all zero": {slice(0, None): None},
    "all tiny": {slice(0, None): -116}, "all large": {slice(0, None): 118},
    "steps": {slice(i, i + 1): 100 - 6 * i for i in range(34)}, "steps up": {slice(i, i + 1): -100 + 6 * i for i in range(34)},
}


@pytest.mark.parametrize("codes,dtype", [(INT8, BF16), (E4M3, BF16), (INT8, F32), (E4M3, F32)])
@pytest.mark.parametrize("rows", FAR.values(), ids=FAR.keys())
def test_scales_of_v_far_from_each_other(codes, dtype, rows):
    """Blocks whose V is larger or smaller by up to 2^230 than in the pages in front of them, or nothing: results of ordinary scores, and of
    scores so far apart that the small blocks have the weight."""
    for dim, spread, top in ((128, 1.0, 1.0), (64, 300.0, 1.0), (256, 40.0, 1.0)):
        cache, pos, table, seq = _attend_inputs((6, 2), dim, 16, [540, 300, 543], codes, seed=33)
        _scaled(cache, table, seq, rows)
        cache["k_scale"] *= spread / 10
        q = (torch.randn(3, 6, dim, generator=_gen(33)) * top).to(dtype)
        _reads(q, cache, pos, table, seq, dtype, "HND")


@pytest.mark.parametrize("codes", [INT8, E4M3])
def test_scales_of_zero_over_codes_that_are_not(codes):
    """A scale of 0 makes its block 0, whatever the codes are: alone in a context, in front of others and behind them."""
    cache, pos, table, seq = _attend_inputs((8, 2), 128, 16, [540, 300, 20], codes, seed=34)
    cache["v_scale"][table[seq[0], 3:20]] = 0
    cache["v_scale"][table[seq[1], :4]] = 0
    cache["v_scale"][table[seq[2]]] = 0
    _reads(torch.randn(3, 8, 128, generator=_gen(34)).half(), cache, pos, table, seq, F16)


@pytest.mark.parametrize("position", [-1, 100])
def test_selection_of_as_many_pages_as_there_can_be(position):
    """The largest top_pages: what stands behind the context's pages is -1 up to the end."""
    from cross_dsl_kernels_b200.kv8 import select_kv8_pages
    if torch.cuda.mem_get_info()[0] < 12 << 30:
        pytest.skip("needs 12 GB of device memory")
    cache, pos, table, seq = _attend_inputs((2, 1), 64, 16, [100], INT8, seed=35)
    pos[0] = position
    top = 2 ** 31 - 1
    got = select_kv8_pages(torch.ones(1, 2, 64, device="cuda"), _on_gpu(cache, "NHD"), *(t.cuda() for t in (pos, table, seq)), top_pages=top)
    assert got.shape == (1, 1, top)
    pages = 0 if position < 0 else position // 16 + 1
    assert got[0, 0, :pages].tolist() == list(range(pages))
    for part in got[0, 0, pages:].split(1 << 29):
        assert bool((part == -1).all())


@pytest.mark.parametrize("codes", [INT8, E4M3])
def test_scores_are_near_those_of_exact_means(codes):
    """A chosen page's score by its exact mean key is below that of no page left out by more than what the rounding of q and of the means
    is off by: half a step of each, 1/127 of the largest |value| (of the head of q, of the block)."""
    from cross_dsl_kernels_b200 import kv8
    page, dim, heads, last, top, g = 16, 64, (4, 2), 60, 12, _gen(36)
    table, pos = torch.randperm(last + 1, generator=g)[None], torch.arange((last + 1) * page)
    ours = kv8.PagedKV8Cache.empty(last + 1, page, heads[1], dim, dtype=codes)
    k = torch.randn(last + 1, 1, heads[1], dim, generator=g) + 0.7 * torch.randn((last + 1) * page, heads[1], dim, generator=g).view(last + 1, page, heads[1], dim)
    k = k.flatten(0, 1)
    trig = torch.ones(pos.numel(), 1, device="cuda"), torch.zeros(pos.numel(), 1, device="cuda")  # no rotation
    kv8.rope_gqa_paged_kv8_append(torch.zeros(pos.numel(), heads[0], dim, device="cuda"), k.cuda(), k.cuda(), *trig, pos.cuda(), table.cuda(),
                                  torch.zeros_like(pos).cuda(), ours, rope_dim=2, interleaved=False)
    q = torch.randn(1, heads[0], dim, generator=g)
    at = pos[-1:].cuda(), table.cuda(), torch.zeros(1, dtype=torch.int64, device="cuda")
    pages = kv8.select_kv8_pages(q.cuda(), ours, *at, top_pages=top).cpu()
    means = ours.dequantized()[0].double().cpu()[table[0, :last]].mean(1)  # [pages, heads, dim] of the codes
    step = ours.k_scale.double().cpu()[table[0, :last]][..., None] * (1.0 if codes == INT8 else 448 / 127)
    for h in range(heads[1]):
        x = q[0, h * 2:h * 2 + 2].double()
        unit = x.abs().amax(-1, keepdim=True) / 127
        score = (x @ means[:, h].T).amax(0)
        off = (0.5 * (x.abs()[:, None] * step[None, :, h] + means[None, :, h].abs() * unit[:, None] + 0.5 * step[None, :, h] * unit[:, None])).sum(-1).amax(0)
        off = off + 2.0 ** -21 * score.abs()  # the FP32 steps of a score
        chosen = torch.zeros(last, dtype=torch.bool)
        chosen[pages[0, h, :-1].long()] = True
        assert chosen.sum() == top - 1 and pages[0, h, -1] == last
        assert bool(((score + off)[chosen].min() >= (score - off)[~chosen].max()))


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("heads,dim,page,positions", [((8, 2), 128, 16, [0, 15, 300, 5000, -1]), ((6, 2), 64, 7, [1000, 6, 7]), ((5, 1), 256, 32, [63, 0, 700])])
def test_e4m3_codes_have_no_offset(dtype, heads, dim, page, positions):
    """Codes of e4m3 enter the products as they are: the limit without what int8 codes are granted for theirs, which is
    * of a score, 2^-22 of sum |q_d k_d| for each of the 2 dim / 16 truncating products of its chain and for four steps of its scaling,
    * of a weight, twice that, its rounding to FP16 (2^-11) and FP32 steps of the sums (2^-18),
    * of the smallest FP16 weights half a step, 2^-39 of the largest, and half a step of the result's type."""
    from cross_dsl_kernels_b200 import kv8
    cache, pos, table, seq = _attend_inputs(heads, dim, page, positions, E4M3, seed=37)
    q = torch.randn(len(positions), heads[0], dim, generator=_gen(37)).to(dtype)
    exact, info = oracle.attention(q, cache, pos, table, seq), torch.finfo(dtype)
    weight = 2.0 ** -11 + 2.0 ** -18 + 2 * exact["score"][..., None] * (2 * dim // 16 + 4) * 2.0 ** -22
    limit = exact["bound"] * weight * 1.01 + exact["least"] * 2.0 ** -39 + exact["result"].abs().clamp(min=info.smallest_normal) * info.eps / 2
    got = kv8.paged_kv8_decode_attention(q.cuda(), _on_gpu(cache, "HND"), *(t.cuda() for t in (pos, table, seq)))
    assert bool(((got.double().cpu() - exact["result"]).abs() <= limit).all())


@pytest.mark.parametrize("codes", [INT8, E4M3])
@pytest.mark.parametrize("dtype", [F16, BF16, F32])
def test_one_position_that_has_all_the_weight(codes, dtype):
    """Its weight is rounded to nothing: the result is its value, rounded once to the result's type but for the FP32 steps behind the products."""
    from cross_dsl_kernels_b200 import kv8
    cache, pos, table, seq = _attend_inputs((4, 2), 128, 16, [900, 333, 15], codes, seed=38)
    q = torch.zeros(3, 4, 128)
    q[..., 0] = 1.0
    cache["k"].view(torch.uint8)[:, :, :, 0] = 0
    cache["k_scale"][:] = 40.0
    exact = torch.zeros(3, 2, 128, dtype=torch.float64)
    for t, j in enumerate((411, 332, 0)):
        page, row = int(table[seq[t], j // 16]), j % 16
        cache["k"][page, row, :, 0] = torch.tensor(64.0).to(codes)  # a score of 64 * 40 / 128 ** 0.5 against zeros
        exact[t] = cache["v"][page, row].double() * cache["v_scale"][page].double()[:, None]
    got = kv8.paged_kv8_decode_attention(q.to(dtype).cuda(), _on_gpu(cache, "NHD"), *(t.cuda() for t in (pos, table, seq))).double().cpu()
    exact = exact.repeat_interleave(2, 1)
    info = torch.finfo(dtype)
    assert bool(((got - exact).abs() <= exact.abs().clamp(min=info.smallest_normal) * (info.eps / 2 + 2.0 ** -19)).all())


@pytest.mark.parametrize("codes", [INT8, E4M3])
@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("k_scale", [3e3, 1e5, 1e7, 1e12, 1e30])
def test_scores_of_any_size(codes, dtype, k_scale):
    """Scores between which one step of FP32 is more than the logarithms of V's scales: a position that has all the weight gives its value; where
    its scale of V is 0, nothing."""
    from cross_dsl_kernels_b200 import kv8
    cache, pos, table, seq = _attend_inputs((4, 2), 128, 16, [900, 333, 15], codes, seed=39)
    q = torch.zeros(3, 4, 128)
    q[..., 0] = 1.0
    cache["k"].view(torch.uint8)[:, :, :, 0] = 0
    cache["k_scale"][:] = k_scale
    exact = torch.zeros(3, 2, 128, dtype=torch.float64)
    for t, j in enumerate((411, 332, 0)):
        page, row = int(table[seq[t], j // 16]), j % 16
        for at, code in ((page, 64.0), (int(table[seq[t], 0]), -32.0)):  # the largest score, and one far below the rest's zeros
            cache["k"][at, row if code > 0 else 3, :, 0] = torch.tensor(code).to(codes)
        exact[t] = cache["v"][page, row].double() * cache["v_scale"][page].double()[:, None]
    info = torch.finfo(dtype)

    def read(kept):
        got = kv8.paged_kv8_decode_attention(q.to(dtype).cuda(), _on_gpu(cache, "NHD"), *(t.cuda() for t in (pos, table, seq))).double().cpu()
        want = (exact * kept).repeat_interleave(2, 1)
        assert bool(((got - want).abs() <= want.abs().clamp(min=info.smallest_normal) * (info.eps / 2 + 2.0 ** -19)).all())

    read(1.0)
    for t, j in enumerate((411, 332, 0)):
        cache["v_scale"][table[seq[t], j // 16]] = 0
    read(0.0)
