"""The decode layer on an 8-bit cache: every op on what the layer itself gave it, eagerly and captured, and beside the 16-bit layer."""

from __future__ import annotations

import pytest
import torch

from conftest import rel_l2
from oracle import kv8 as oracle
from test_gpu_kv8 import _close

CODES = {"int8": torch.int8, "e4m3": torch.float8_e4m3fn}


def _config(**kw):
    from cross_dsl_kernels_b200.chain import ChainConfig
    return ChainConfig(**{**dict(tokens=5, hidden=1024, q_heads=8, kv_heads=2, mlp=1536, context=256), **kw})


@pytest.mark.gpu
@pytest.mark.parametrize("kv_cache,top_pages", [("int8", 0), ("e4m3", 0), ("int8", 3), ("e4m3", 3)])
def test_layer_matches_the_restatement(kv_cache, top_pages):
    from cross_dsl_kernels_b200.chain import DecodeLayerChain
    cfg = _config()
    chain = DecodeLayerChain(cfg, attention=True, kv_cache=kv_cache, top_pages=top_pages)
    g = torch.Generator().manual_seed(1)
    cache = oracle.empty(chain.cache8.pages, cfg.page_size, cfg.kv_heads, cfg.head_dim, CODES[kv_cache])
    top = oracle.TOP[CODES[kv_cache]]
    for name in ("k", "v"):
        x = (torch.randn(cache[name].shape, generator=g) * top / 4).clamp(-top, top)
        cache[name] = (x.round() if kv_cache == "int8" else x).to(CODES[kv_cache])
        cache[name + "_scale"] = 4 / top * torch.exp(0.3 * torch.randn(cache[name + "_scale"].shape, generator=g))
    cache["k_mean"] = torch.randint(-40, 41, cache["k_mean"].shape, generator=g).to(torch.int8)
    for name in ("k", "v", "k_scale", "v_scale") + (("k_mean",) if top_pages else ()):
        getattr(chain.cache8, name).copy_(cache[name].cuda())
    out = chain.step()
    t, d, hq, hkv = cfg.tokens, cfg.head_dim, cfg.q_heads, cfg.kv_heads
    q, k, v = out["qkv"].cpu().view(t, hq + 2 * hkv, d).split((hq, hkv, hkv), dim=1)
    index = (chain.positions, chain.page_table, chain.sequence_ids)
    want = oracle.append(q, k, v, chain.cos, chain.sin, *index, cache, rope_dim=d, interleaved=False)
    assert torch.equal(out["q_rot"].cpu(), want)
    assert torch.equal(chain.cache8.k.cpu().view(torch.uint8), cache["k"].view(torch.uint8))
    assert torch.equal(chain.cache8.v_scale.cpu(), cache["v_scale"])
    pages = oracle.select(want, cache, *index, top_pages=top_pages) if top_pages else None
    _close(out["attn"].view(t, hq, d), oracle.attention(want, cache, *index, pages=pages), torch.float16, d)


@pytest.mark.gpu
@pytest.mark.parametrize("kv_cache,step", [("int8", 1 / 127), ("e4m3", 2.0 ** -4)])
def test_layer_is_near_the_16_bit_one(kv_cache, step):
    """Contexts that both layers are given through their appends, so the caches hold the same values to a rounding: half a step of the
    codes (int8: of the block's largest value, 127 steps; e4m3: 2^-4 of each value).  Softmax weights are off by e^(2 x) - 1 where scores
    are off by x, values by the same half step, so the outputs' rounding errors average to well below one whole step of what is summed."""
    from cross_dsl_kernels_b200.chain import DecodeLayerChain
    cfg = _config(tokens=4, context=64)
    layers = {name: DecodeLayerChain(cfg, attention=True, kv_cache=name) for name in ("f16", kv_cache)}
    outs = {}
    for name, chain in layers.items():
        last = chain.positions.clone()
        for pos in range(int(last.max()) + 1):
            chain.dev["positions"].copy_(torch.minimum(torch.full_like(last, pos), last).cuda())
            g = torch.Generator(device="cuda").manual_seed(pos)
            outs[name] = chain.step(h=torch.randn(cfg.tokens, cfg.hidden, generator=g, device="cuda").half())
    for stage in ("attn", "act"):
        assert torch.isfinite(outs[kv_cache][stage]).all()
    values = outs["f16"]["qkv"].float().abs().amax()
    assert float((outs[kv_cache]["attn"].float() - outs["f16"]["attn"].float()).abs().max()) <= 4 * step * float(values)
    assert rel_l2(outs[kv_cache]["attn"], outs["f16"]["attn"]) <= 8 * step


@pytest.mark.gpu
@pytest.mark.parametrize("top_pages", [0, 4])
def test_captured_layers_with_dependent_launches(top_pages):
    """Two layers captured with dependent launches give the bits of the eager ones; the launches are counted."""
    from cross_dsl_kernels_b200.chain import DecodeLayerChain
    from cross_dsl_kernels_b200.timing import capture
    kw = dict(layers=2, attention=True, kv_cache="e4m3", top_pages=top_pages)
    eager, chain = DecodeLayerChain(_config(), **kw), DecodeLayerChain(_config(), dependent_launch=True, **kw)
    assert chain.launches_per_layer == (9 if top_pages else 8)
    want = eager.run_layers()
    outputs: list = []
    graph = capture([chain.run_layers], outputs=outputs)
    for t in (chain.cache8.k_scale, chain.cache8.v_scale):
        t.zero_()
    for t in (chain.cache8.k, chain.cache8.v):
        t.view(torch.uint8).zero_()
    for name in ("attn", "act", "n2"):
        outputs[0][name].fill_(float("nan"))
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(outputs[0][name], want[name]) for name in ("q_rot", "attn", "act", "n2"))
    assert all(torch.equal(a, b) for a, b in zip(eager.cache8.tensors(), chain.cache8.tensors()))


@pytest.mark.gpu
def test_kernel_bench_rows_of_the_cache():
    from cross_dsl_kernels_b200 import kernel_bench
    for op in ("append", "attention", "select", "sparse"):
        row = kernel_bench.one(["kv8", op, "512", "2"])
        assert row["us"] > 0 and row["bytes"] > 0 and op in row["kernel"]


@pytest.mark.parametrize("kw", [dict(kv_cache="int4", attention=True), dict(kv_cache="int8"), dict(top_pages=4, attention=True),
                                dict(kv_cache="int8", attention=True, top_pages=-1), dict(kv_cache="int8", attention=True, top_pages=2.0)])
def test_layer_refuses(kw):
    from cross_dsl_kernels_b200.chain import DecodeLayerChain
    with pytest.raises(ValueError):
        DecodeLayerChain(_config(), device="cpu", **kw)
