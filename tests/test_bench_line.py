"""What bench.py prints: one short JSON line on standard output, whatever the size of the per-kernel table."""

from __future__ import annotations

import json

import bench


def test_the_line_is_one_and_short(capsys):
    line = dict(metric=bench.METRIC, value=1.0, config=bench.workload_config(1, "peer"))
    table = [dict(kernel=f"gemv_f32_KN_m16_k4096_n14336_s{i}", us=1.0, gbps=2.0, gated=True, cpu_us=3.0) for i in range(200)]
    bench.report(line, table)
    got = capsys.readouterr()
    assert got.out.count("\n") == 1 and len(got.out) < 4096
    assert json.loads(got.out) == dict(line, kernels=200)
    assert [json.loads(row) for row in got.err.splitlines()] == table
    bench.report(line, [])
    assert json.loads(capsys.readouterr().out) == line
