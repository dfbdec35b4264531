"""Two host threads that call an op at the same time, with sizes that take different amounts of shared memory."""

from __future__ import annotations

import threading

import pytest
import torch

pytestmark = pytest.mark.gpu


def _side_by_side(calls, rounds=4000):
    """Each of `calls` in a thread and on a stream of its own, over and over; every result is that of the call alone."""
    alone = [call() for call in calls]
    torch.cuda.synchronize()
    wrong, start = [], threading.Barrier(len(calls))

    def run(call, want):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                start.wait()
                for i in range(rounds):
                    got = call()
                    if i % 500 == 499 and not torch.equal(got, want):
                        wrong.append("another result")
        except Exception as error:  # a thread's own would be lost
            wrong.append(repr(error))

    threads = [threading.Thread(target=run, args=pair) for pair in zip(calls, alone)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    assert not wrong, wrong[0]


def test_selections_from_tables_of_different_widths():
    from cross_dsl_kernels_b200 import kv8

    def call(width):
        g = torch.Generator(device="cuda").manual_seed(width)
        cache = kv8.PagedKV8Cache.empty(width, 1, 1, 64)
        cache.k_mean.copy_(torch.randint(-60, 61, cache.k_mean.shape, generator=g, device="cuda", dtype=torch.int8))
        cache.k_scale.fill_(1.0)
        q = torch.randn(1, 2, 64, generator=g, device="cuda")
        index = (torch.tensor([width - 1], device="cuda"), torch.randperm(width, generator=g, device="cuda")[None], torch.zeros(1, dtype=torch.int64, device="cuda"))
        return lambda: kv8.select_kv8_pages(q, cache, *index, top_pages=9)

    _side_by_side([call(51200), call(9000)])


@pytest.mark.parametrize("m", [1, 4, 16])
def test_first_call_of_a_thread(m):
    """A thread that has not used the GPU before: the same bits as in the main thread, for projections of each kind."""
    from cross_dsl_kernels_b200.ops import decode_linear
    from cross_dsl_kernels_b200.w4a16 import w4a16_linear
    g = torch.Generator(device="cuda").manual_seed(m)
    x, w = (torch.randn(*shape, generator=g, device="cuda") for shape in ((m, 1024), (1024, 4096)))
    packed = torch.randint(0, 256, (4096, 512), generator=g, device="cuda", dtype=torch.uint8)
    scales, half = torch.rand(4096, 8, generator=g, device="cuda").half(), x.half()
    for call in (lambda: w4a16_linear(half, packed, scales, None, group_size=128), lambda: decode_linear(x, w, None, weight_layout="KN"),
                 lambda: decode_linear(x, w.view(4096, 1024), None, weight_layout="NK")):
        want, got = call(), []

        def run():
            try:
                got.append(call())
            except Exception as error:  # a thread's own would be lost
                got.append(error)

        thread = threading.Thread(target=run)
        thread.start()
        thread.join()
        torch.cuda.synchronize()
        assert isinstance(got[0], torch.Tensor), got[0]
        assert torch.equal(got[0], want)


@pytest.mark.parametrize("one,two", [((1, 96000), (1, 1600)), ((8, 8192), (8, 2048)), ((16, 6080), (16, 160))])
def test_projections_of_different_depths(one, two):
    """x stays in shared memory, as much as there is of it."""
    from cross_dsl_kernels_b200.w4a16 import w4a16_linear

    def call(m, k):
        g = torch.Generator(device="cuda").manual_seed(k)
        x = torch.randn(m, k, generator=g, device="cuda").half()
        packed = torch.randint(0, 256, (64, k // 2), generator=g, device="cuda", dtype=torch.uint8)
        scales = torch.rand(64, k // 32, generator=g, device="cuda").half()
        return lambda: w4a16_linear(x, packed, scales, None, group_size=32)

    _side_by_side([call(*one), call(*two)])
