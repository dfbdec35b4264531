"""Sizes that the ops of the 8-bit cache do not take: a ValueError that names them, like every other refusal."""

from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu


def _reads(q, cache, **kw):
    from cross_dsl_kernels_b200 import kv8
    tokens = q.shape[0]
    index = (torch.zeros(tokens, dtype=torch.int64, device="cuda"), torch.zeros(1, 1, dtype=torch.int64, device="cuda"),
             torch.zeros(tokens, dtype=torch.int64, device="cuda"))
    pages = torch.zeros(tokens, cache.kv_heads, 1, dtype=torch.int32, device="cuda")
    scale = {} if kw else dict(top_pages=1)
    calls = [lambda: kv8.paged_kv8_decode_attention(q, cache, *index, **kw), lambda: kv8.paged_kv8_sparse_attention(q, cache, pages, *index, **kw)]
    return calls + ([lambda: kv8.select_kv8_pages(q, cache, *index, **scale)] if scale else [])


def test_more_tokens_than_a_read_takes():
    from cross_dsl_kernels_b200 import kv8
    cache = kv8.PagedKV8Cache.empty(1, 16, 1, 64)
    for call in _reads(torch.zeros(65536, 1, 64, device="cuda", dtype=torch.float16), cache):
        with pytest.raises(ValueError, match="65535 tokens"):
            call()
    for call in _reads(torch.zeros(65535, 1, 64, device="cuda", dtype=torch.float16), cache):
        call()


@pytest.mark.parametrize("scale", [1e39, -1e300, float("inf"), float("nan"), 10 ** 39])
def test_scales_that_are_not_finite_in_float32(scale):
    from cross_dsl_kernels_b200 import kv8
    for call in _reads(torch.zeros(1, 1, 64, device="cuda"), kv8.PagedKV8Cache.empty(1, 16, 1, 64), scale=scale):
        with pytest.raises(ValueError, match="scale must be finite"):
            call()


def test_more_heads_than_an_append_takes():
    from cross_dsl_kernels_b200 import kv8
    cache, zero = kv8.PagedKV8Cache.empty(1, 16, 1, 64), torch.zeros(1, dtype=torch.int64, device="cuda")
    q, kv, trig = torch.zeros(1, 65536, 64, device="cuda"), torch.zeros(1, 1, 64, device="cuda"), torch.zeros(1, 32, device="cuda")
    with pytest.raises(ValueError, match="q_heads"):
        kv8.rope_gqa_paged_kv8_append(q, kv, kv, trig, trig.clone(), zero, zero[None], zero, cache, rope_dim=64, interleaved=False)
