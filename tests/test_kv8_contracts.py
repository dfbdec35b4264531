"""What the 8-bit paged cache and its ops refuse, and what the C entry points do: before anything is launched."""

from __future__ import annotations

import pytest
import torch

from cross_dsl_kernels_b200 import _native, kv8
from cross_dsl_kernels_b200.kv8 import PagedKV8Cache


def _cache(device="cpu", pages=4, page=8, heads=2, dim=64, dtype=torch.int8, layout="NHD", means=True):
    return PagedKV8Cache.empty(pages, page, heads, dim, dtype=dtype, kv_layout=layout, means=means, device=device)


@pytest.mark.parametrize("layout", ["NHD", "HND", "hnd"])
@pytest.mark.parametrize("dtype", [torch.int8, torch.float8_e4m3fn])
def test_cache_shape(layout, dtype):
    c = _cache(layout=layout, dtype=dtype, means=False)
    assert (c.pages, c.page_size, c.kv_heads, c.head_dim, c.kv_layout) == (4, 8, 2, 64, layout.upper())
    assert c.k_mean is None and len(c.tensors()) == 4 and c.dequantized()[0].shape == c.k.shape


def test_cache_dequantizes_by_block():
    c = _cache(layout="HND", dtype=torch.float8_e4m3fn)
    c.k[1, 1] = torch.full((8, 64), 1.5).to(torch.float8_e4m3fn)
    c.k_scale[1, 1] = 4.0
    k, v = c.dequantized()
    assert (k[1, 1] == 6).all() and float(k.sum()) == 6 * 8 * 64 and not v.any()


@pytest.mark.parametrize("change", [
    dict(k=torch.zeros(4, 8, 2, 64)), dict(v=torch.zeros(4, 8, 2, 64, dtype=torch.float8_e4m3fn)), dict(v=torch.zeros(4, 8, 1, 64, dtype=torch.int8)),
    dict(k=torch.zeros(4, 8, 128, dtype=torch.int8)), dict(k_scale=torch.zeros(4, 8)), dict(v_scale=torch.zeros(4, 2, dtype=torch.float64)),
    dict(k_mean=torch.zeros(4, 2, 64)), dict(k_mean=torch.zeros(2, 4, 64, dtype=torch.int8)), dict(kv_layout="NDH"), dict(kv_layout="HND"),
    dict(k_scale=torch.zeros(2, 4).t()), dict(v_scale=torch.zeros(4, 2, requires_grad=True)),
    dict(k=torch.zeros(4 * 8 * 2 * 64 + 1, dtype=torch.int8)[1:].view(4, 8, 2, 64))])
def test_cache_refuses(change):
    c = _cache()
    parts = dict(k=c.k, v=c.v, k_scale=c.k_scale, v_scale=c.v_scale, k_mean=c.k_mean, kv_layout="NHD")
    with pytest.raises(ValueError):
        PagedKV8Cache(**{**parts, **change})
    with pytest.raises(ValueError, match="overlap"):
        PagedKV8Cache(**{**parts, "v": c.k})
    with pytest.raises(ValueError, match="overlap"):
        PagedKV8Cache(**{**parts, "v_scale": c.k_scale})


@pytest.mark.parametrize("size", [dict(dim=96), dict(page=1025), dict(pages=0), dict(heads=0)])
def test_cache_sizes(size):
    with pytest.raises(ValueError):
        _cache(**size)


def test_there_is_no_cpu_path():
    c, q, index = _cache(), torch.zeros(1, 4, 64), (torch.zeros(1, dtype=torch.int64), torch.zeros(1, 1, dtype=torch.int64), torch.zeros(1, dtype=torch.int64))
    kv, trig = torch.zeros(1, 2, 64), torch.zeros(8, 32)
    for call in (lambda: kv8.rope_gqa_paged_kv8_append(q, kv, kv, trig, trig, *index, c, rope_dim=64, interleaved=False),
                 lambda: kv8.paged_kv8_decode_attention(q, c, *index), lambda: kv8.select_kv8_pages(q, c, *index, top_pages=2),
                 lambda: kv8.paged_kv8_sparse_attention(q, c, torch.zeros(1, 2, 1, dtype=torch.int32), *index)):
        with pytest.raises(ValueError, match="CUDA"):
            call()
        with pytest.raises(ValueError, match="PagedKV8Cache"):
            kv8.paged_kv8_decode_attention(q, (c.k, c.v), *index)


def test_c_entry_points_check_sizes_before_they_touch_a_gpu():
    """Pointers are never followed here: each call has one argument that the entry point refuses."""
    lib, p = _native.lib(), 4096
    dst = _native.PeerOutStruct()
    dst.ptr[0], dst.world, dst.ld, dst.col0 = p, 1, 4 * 64, 0
    import ctypes
    out = ctypes.byref(dst)
    good = dict(tokens=1, hq=4, hkv=2, dim=64, width=4, page=8)

    def attend(q=p, k=p, codes=0, dtype=0, scale=1.0, flags=0, dst=out, **kw):
        s = {**good, **kw}
        return lib.xdk_kv8_decode_attention(q, k, p, p, p, p, p, p, dst, s["tokens"], s["hq"], s["hkv"], s["dim"], s["width"], s["page"], 0, scale, 0,
                                            dtype, codes, kw.get("scratch"), kw.get("nbytes", 0), flags, None)

    def sparse(n=1, pages=p, **kw):
        s = {**good, **kw}
        return lib.xdk_kv8_sparse_attention(p, p, p, p, p, pages, p, p, p, out, s["tokens"], s["hq"], s["hkv"], s["dim"], s["width"], s["page"], n, 0, 1.0,
                                            0, 0, kw.get("scratch"), kw.get("nbytes", 0), 0, None)

    def select(top=1, mean=p, **kw):
        s = {**good, **kw}
        return lib.xdk_kv8_select_pages(p, mean, p, p, p, p, p, s["tokens"], s["hq"], s["hkv"], s["dim"], s["width"], s["page"], top, 0, 0, None)

    def append(cache=p, mean=None, rope=64, cw=32, qs=256, codes=0, dtype=0, scratch=None, nbytes=0, flags=0, **kw):
        s = {**good, **kw}
        return lib.xdk_kv8_append(p, p, p, p, p, p, p, p, p, cache, p, p, p, mean, s["tokens"], s["hq"], s["hkv"], s["dim"], cw, s["width"], s["page"],
                                  rope, qs, 128, 128, 0, 0, dtype, codes, scratch, nbytes, flags, None)

    wrong, limit = -1, -4
    for kw in (dict(q=None), dict(k=None), dict(k=p + 8), dict(codes=2), dict(codes=-1), dict(dtype=3), dict(scale=float("nan")),
               dict(scale=float("inf")), dict(flags=1), dict(dst=None), dict(tokens=0), dict(hq=3), dict(page=0), dict(width=0), dict(hq=8),
               dict(), dict(scratch=p, nbytes=64), dict(scratch=p + 8, nbytes=1 << 40)):
        assert attend(**kw) == wrong, kw
    for kw in (dict(tokens=65536), dict(dim=32), dict(page=1025), dict(width=1 << 31)):
        assert attend(**kw) == limit, kw
    dst.ld = 18 * 64
    assert attend(hq=18) == limit  # nine heads to a group
    dst.ld = 4 * 64
    assert sparse() == wrong and sparse(scratch=p, nbytes=64) == wrong and sparse(n=0) == wrong and sparse(pages=None) == wrong and sparse(n=1 << 22) == limit
    assert select(top=0) == wrong and select(mean=None) == wrong and select(mean=p + 4) == wrong and select(width=51201) == limit and select(hq=18) == limit
    for kw in (dict(cache=None), dict(cache=p + 1), dict(mean=p + 4), dict(rope=3), dict(rope=66), dict(rope=0), dict(cw=31), dict(qs=255), dict(codes=2),
               dict(dtype=7), dict(flags=1), dict(tokens=129), dict(tokens=129, scratch=p, nbytes=64), dict(tokens=-1)):
        assert append(**kw) == wrong, kw
    for kw in (dict(dim=192, qs=768), dict(page=2000), dict(tokens=(1 << 26) + 1)):
        assert append(**kw) in (limit, wrong), kw
    assert lib.xdk_kv8_append_scratch_bytes(128, 2) == 0 and lib.xdk_kv8_append_scratch_bytes(129, 2) >= 512 * 20
    size = lib.xdk_kv8_decode_attention_scratch_bytes
    assert 0 < size(1, 4, 2, 64, 1024) < size(1, 4, 2, 64, 8192) <= size(1, 4, 2, 64, 0) == size(1, 4, 2, 64, 1 << 62) == size(1, 4, 2, 64, (1 << 63) - 1)
    assert size(1, 18, 2, 64, 8192) == size(0, 4, 2, 64, 64) == size(1, 4, 2, 96, 64) == size(1, 4, 3, 64, 64) == 0
    assert lib.xdk_kv8_sparse_attention_scratch_bytes(1, 4, 2, 64, 16, 8) > 0 == lib.xdk_kv8_sparse_attention_scratch_bytes(1, 4, 2, 64, 16, 0)


def _inputs():
    g = torch.Generator(device="cuda").manual_seed(0)

    def normal(*shape):
        return torch.randn(*shape, generator=g, device="cuda").half()

    trig = torch.rand(64, 32, generator=g, device="cuda")
    return dict(q=normal(3, 4, 64), k=normal(3, 2, 64), v=normal(3, 2, 64), cos=trig, sin=trig.clone(), pos=torch.tensor([0, 9, 15], device="cuda"),
                table=torch.tensor([[0, 1], [2, 3], [4, 5]], device="cuda"), seq=torch.arange(3, device="cuda"),
                cache=_cache("cuda", pages=6), pages=torch.tensor([[0, 1]], device="cuda", dtype=torch.int32).repeat(3, 2, 1))


def _calls(i, **kw):
    index = (i["pos"], i["table"], i["seq"])
    return dict(append=lambda: kv8.rope_gqa_paged_kv8_append(i["q"], i["k"], i["v"], i["cos"], i["sin"], *index, i["cache"],
                                                             **{"rope_dim": 64, "interleaved": False, **kw}),
                attend=lambda: kv8.paged_kv8_decode_attention(i["q"], i["cache"], *index, **kw),
                select=lambda: kv8.select_kv8_pages(i["q"], i["cache"], *index, **{"top_pages": 2, **kw}),
                sparse=lambda: kv8.paged_kv8_sparse_attention(i["q"], i["cache"], i["pages"], *index, **kw))


class _Declines:
    def __getattr__(self, name):
        return lambda *args: None


@pytest.mark.gpu
def test_native_and_python_paths_give_the_same_bits(monkeypatch):
    one, two = _inputs(), _inputs()
    kept = {}
    for i, native in ((one, True), (two, False)):
        with monkeypatch.context() as m:
            if native:  # the Python half may not be reached
                m.setattr(kv8, "_indices", lambda *a: pytest.fail("the native half declined an ordinary call"))
            else:
                m.setattr(_native, "host", lambda: _Declines())
            kept[native] = [call() for call in _calls(i).values()]
    assert all(torch.equal(a, b) for a, b in zip(kept[True], kept[False]))
    assert all(torch.equal(a, b) for a, b in zip(one["cache"].tensors(), two["cache"].tensors()))


@pytest.mark.gpu
@pytest.mark.parametrize("op,change,match", [
    ("all", dict(q=lambda i: i["q"].double()), "q must be"), ("all", dict(q=lambda i: i["q"][:, :3]), "divisible"),
    ("all", dict(q=lambda i: i["q"][0]), "q must be"), ("all", dict(q=lambda i: i["q"].float().requires_grad_()), "gradient"),
    ("all", dict(q=lambda i: torch.cat([i["q"]] * 2, -1)), "head_dim"), ("all", dict(q=lambda i: i["q"][:0]), "q must be"),
    ("all", dict(pos=lambda i: i["pos"].int()), "positions must be int64"), ("all", dict(pos=lambda i: i["pos"].cpu()), "positions must be on"),
    ("all", dict(pos=lambda i: i["pos"][:2]), "one entry per token"), ("all", dict(table=lambda i: i["table"][:, ::2]), "contiguous"),
    ("all", dict(table=lambda i: i["table"][:, :0]), "at least one page"), ("all", dict(seq=lambda i: i["seq"][:1]), "one entry per token"),
    ("all", dict(cache=lambda i: _cache()), "same CUDA device"), ("all", dict(cache=lambda i: None), "PagedKV8Cache"),
    ("append", dict(k=lambda i: i["k"].float()), "unexpected dtype"), ("append", dict(v=lambda i: i["v"][:, :1]), "k and v must be"),
    ("append", dict(k=lambda i: i["k"].transpose(0, 1).contiguous().transpose(0, 1)), "column slice"),
    ("append", dict(cos=lambda i: i["cos"][:, :31]), "cos"), ("append", dict(sin=lambda i: i["sin"].double()), "unexpected dtype"),
    ("append", dict(rope_dim=66), "exceed"), ("append", dict(rope_dim=5), "even"), ("append", dict(rope_dim=True), "even"),
    ("append", dict(k=lambda i: i["cache"].k_scale.view(torch.float16).view(-1)[:0].new_zeros(3, 2, 64)[:2]), "k and v must be"),
    ("append", dict(k=lambda i: i["cache"].k.view(torch.float16).view(-1)[:384].view(3, 2, 64)), "overlap"),
    ("attend", dict(scale=float("nan")), "finite"), ("attend", dict(q=lambda i: i["q"].transpose(0, 1).contiguous().transpose(0, 1)), "contiguous"),
    ("attend", dict(q=lambda i: torch.cat([i["q"]] * 5, 1)[:, :18].contiguous()), "at most 8"), ("select", dict(top_pages=0), "top_pages"),
    ("select", dict(top_pages=2.0), "top_pages"), ("select", dict(cache=lambda i: _cache("cuda", pages=6, means=False)), "mean keys"),
    ("select", dict(table=lambda i: i["table"].repeat(1, 25601)), "at most 51200"), ("sparse", dict(pages=lambda i: i["pages"].long()), "int32"),
    ("sparse", dict(pages=lambda i: i["pages"][:, :1]), "pages must be"), ("sparse", dict(pages=lambda i: i["pages"].cpu()), "pages must be on"),
    ("sparse", dict(scale=float("inf")), "finite")])
def test_ops_refuse(op, change, match):
    """Each refusal is a ValueError that names what is wrong, and nothing was written."""
    i = _inputs()
    before = [t.clone() for t in i["cache"].tensors()]
    cache = i["cache"]
    kw = {n: x for n, x in change.items() if not callable(x)}
    i.update({n: x(i) for n, x in change.items() if callable(x)})
    for name, call in _calls(i, **kw).items():
        if op in (name, "all"):
            with pytest.raises(ValueError, match=match):
                call()
    assert all(torch.equal(a, b) for a, b in zip(cache.tensors(), before))
