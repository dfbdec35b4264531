"""The 8-bit cache sharded by KV head: results stored to several destinations, and the decode layer of two ranks, one after the other on one
GPU (no kernel waits for another rank's)."""

from __future__ import annotations

import pytest
import torch

from oracle import kv8 as oracle
from test_gpu_kv8 import BF16, E4M3, F16, F32, INT8, _attend_inputs, _close, _gen, _on_gpu
from test_gpu_kv8_chain import CODES, _config

pytestmark = pytest.mark.gpu


def _destination(matrices, col):
    from cross_dsl_kernels_b200 import _native
    out = _native.PeerOutStruct()
    for i, m in enumerate(matrices):
        out.ptr[i] = m.data_ptr()
    out.world, out.ld, out.col0 = len(matrices), matrices[0].shape[1], col
    return out


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("width,col", [(600, 40), (601, 40), (600, 41)])
@pytest.mark.parametrize("codes,positions", [(INT8, [3000, 12, -1]), (E4M3, [i % 90 for i in range(300)])])
def test_several_destinations(dtype, width, col, codes, positions):
    """Whole items, items of many warps and rows that begin on any element: every copy has the bits of the only one."""
    from cross_dsl_kernels_b200 import kv8
    cache, pos, table, seq = _attend_inputs((8, 2), 64, 16, positions, codes, seed=41)
    tokens, ours, args = len(positions), _on_gpu(cache, "NHD"), [t.cuda() for t in (pos, table, seq)]
    q = torch.randn(tokens, 8, 64, generator=_gen(41)).to(dtype).cuda()
    pages = kv8.select_kv8_pages(q, ours, *args, top_pages=9)
    for want, call in ((kv8.paged_kv8_decode_attention(q, ours, *args), lambda to: kv8.paged_kv8_decode_attention(q, ours, *args, peer_out=to)),
                       (kv8.paged_kv8_sparse_attention(q, ours, pages, *args), lambda to: kv8.paged_kv8_sparse_attention(q, ours, pages, *args, peer_out=to))):
        for copies in (2, 3):
            every = [torch.full((tokens, width), -7.0, dtype=dtype, device="cuda") for _ in range(copies)]
            assert call(_destination(every, col)) is None
            for one in every:
                assert torch.equal(one[:, col:col + 512], want.view(tokens, 512))
                assert (one[:, :col] == -7).all() and (one[:, col + 512:] == -7).all()


class _Matrix:
    def __init__(self, arena, number, rows, cols, dtype):
        self.arena, self.number, self.local = arena, number, torch.full((rows, cols), float("nan"), dtype=dtype, device="cuda")

    def out_for(self, col0):
        return _destination([a.matrices[self.number].local for a in self.arena.ranks], col0)


class _Arena:
    """The ranks' matrices as tensors of this process; its barrier is the order in which the test runs the ranks."""

    def __init__(self, ranks):
        self.ranks, self.matrices = ranks, []
        ranks.append(self)

    def matrix(self, rows, cols, dtype):
        self.matrices.append(_Matrix(self, len(self.matrices), rows, cols, dtype))
        return self.matrices[-1]

    def new_site(self):
        return 0

    def barrier(self, site, **kw):
        pass


@pytest.mark.parametrize("kv_cache,top_pages", [("int8", 0), ("e4m3", 3)])
def test_layer_of_two_ranks(monkeypatch, kv_cache, top_pages):
    """Each rank's columns of the attention are what the restatement makes of that rank's own projections and cache, in both ranks' matrices, and
    its columns of the activation are SwiGLU of its own."""
    from cross_dsl_kernels_b200 import peer
    from cross_dsl_kernels_b200.chain import DecodeLayerChain
    from cross_dsl_kernels_b200.ops import swiglu
    ranks: list = []
    monkeypatch.setattr(peer, "PeerArena", lambda *a, **kw: _Arena(ranks))
    cfg = _config(tokens=4)
    chains = [DecodeLayerChain(cfg, rank=r, world=2, attention=True, kv_cache=kv_cache, top_pages=top_pages) for r in range(2)]
    t, d, hq, hkv = cfg.tokens, cfg.head_dim, cfg.q_heads // 2, cfg.kv_heads // 2
    for chain in chains:
        chain.step()  # both ranks' columns are there behind this
    outs = [chain.step() for chain in chains]
    outs[0] = chains[0].step()  # with the activation of rank 1, whose attention was whole
    for r, (chain, out) in enumerate(zip(chains, outs)):
        cache = oracle.empty(chain.cache8.pages, cfg.page_size, hkv, d, CODES[kv_cache])
        q, k, v = out["qkv"].cpu().view(t, hq + 2 * hkv, d).split((hq, hkv, hkv), dim=1)
        index = (chain.positions, chain.page_table, chain.sequence_ids)
        want = oracle.append(q, k, v, chain.cos, chain.sin, *index, cache, rope_dim=d, interleaved=False)
        assert torch.equal(out["q_rot"].cpu(), want)
        assert torch.equal(chain.cache8.k.cpu().view(torch.uint8), cache["k"].view(torch.uint8))
        pages = oracle.select(want, cache, *index, top_pages=top_pages) if top_pages else None
        exact = oracle.attention(want, cache, *index, pages=pages)
        _close(out["attn"][:, r * hq * d:(r + 1) * hq * d].reshape(t, hq, d), exact, F16, d)
        mine = cfg.mlp // 2
        assert torch.equal(out["act"][:, r * mine:(r + 1) * mine], swiglu(out["up"]))
    assert torch.equal(outs[0]["attn"], outs[1]["attn"]) and torch.isfinite(outs[0]["attn"]).all()
    assert torch.equal(outs[0]["n2"], outs[1]["n2"]) and torch.equal(outs[0]["act"], outs[1]["act"])
    assert all(chain.launches_per_layer == (11 if top_pages else 10) for chain in chains)
