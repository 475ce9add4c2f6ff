"""bench.py's HBM traffic figure: reported for the kernels that it was measured on, and for no others."""

from __future__ import annotations

import json
import re
import shutil

import pytest

import bench

DEC = {"launches_per_step": json.loads(bench.PROFILE_TRAFFIC.read_text())["calls"]}


def test_the_sweeps_sources_are_whole():
    """Every local header that one of them includes is among them, but for the public one; every launch of the two
    decode GEMMs' kernels lies in them."""
    for name in bench.SWEEP_SOURCES:
        text = (bench.CSRC / name).read_text()
        assert set(re.findall(r'#include "(\w+\.h)"', text)) <= {*bench.SWEEP_SOURCES, "lse_int8.h"}
    for f in bench.CSRC.glob("*.hip"):
        if f.name not in bench.SWEEP_SOURCES:
            assert not re.search(r"__global__[^;{]*\b(skinny_\w+|tiled_gemm_kernel|xs_kernel)\(", f.read_text()), f.name


@pytest.mark.parametrize("name", ["attn_fp8.hip", "new.hip", "new.h", *bench.SWEEP_SOURCES])
def test_only_the_sweeps_own_sources_count(name, tmp_path):
    shutil.copytree(bench.CSRC, tmp_path / "csrc")
    assert bench.sweep_sources_digest(tmp_path / "csrc") == bench.sweep_sources_digest()
    with open(tmp_path / "csrc" / name, "a") as f:
        f.write("// one more line\n")
    same = bench.sweep_sources_digest(tmp_path / "csrc") == bench.sweep_sources_digest()
    assert same == (name not in bench.SWEEP_SOURCES)


def test_another_build_and_other_launches_are_told(tmp_path, monkeypatch):
    summary = json.loads(bench.PROFILE_TRAFFIC.read_text())
    at = tmp_path / "traffic.json"
    monkeypatch.setattr(bench, "PROFILE_TRAFFIC", at)
    assert bench.measured_traffic(DEC)[0] is None
    at.write_text(json.dumps({**summary, "sweep_sources_sha16": bench.sweep_sources_digest()}))
    assert bench.measured_traffic(DEC) == (summary["hbm_bytes_per_call"], "")
    assert bench.measured_traffic({"launches_per_step": DEC["launches_per_step"] + 1})[0] is None
    at.write_text(json.dumps({**summary, "sweep_sources_sha16": "0" * 16}))
    traffic, why = bench.measured_traffic(DEC)
    assert traffic is None and "another build" in why
