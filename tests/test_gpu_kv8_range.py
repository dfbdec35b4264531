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
