"""What the bench's counters are tied to: the step's own kernels and how they are compiled, not the library's other operators."""
import json
import os
import shutil

import bench
from gossipnet_amd import build


def test_the_hash_is_of_the_step(tmp_path, monkeypatch):
    at = tmp_path / "gossipnet_amd"
    shutil.copytree(build.CSRC, at / "csrc", ignore=shutil.ignore_patterns("build"))
    here = bench.kernel_source_hash()
    monkeypatch.setattr(bench, "ROOT", str(tmp_path))
    assert bench.kernel_source_hash() == here
    for f in ("vocab.hip", "vocab_gemm.hpp", "embed.hip", "roi_pool.hip"):
        (at / "csrc" / f).write_text("changed")
    (at / "csrc" / "another_operator.hip").write_text("new")
    assert bench.kernel_source_hash() == here
    monkeypatch.setattr(build, "FLAGS", build.FLAGS + ["-another-flag"])
    assert bench.kernel_source_hash() != here
    monkeypatch.undo()
    monkeypatch.setattr(bench, "ROOT", str(tmp_path))
    for f in ("forward.hip", "backward_edge.hpp"):
        (at / "csrc" / f).write_text("changed")
        assert bench.kernel_source_hash() != here


def test_every_source_of_a_step_is_there_and_includes_nothing_else():
    for f in bench.STEP_SOURCES:
        text = open(os.path.join(build.CSRC, f)).read()
        for line in text.splitlines():
            if line.startswith('#include "'):
                name = line.split('"')[1]
                assert name in bench.STEP_SOURCES or name.endswith("gossipnet_hip.h"), (f, name)


def test_the_counters_name_what_they_were_collected_from():
    tf = json.load(open(bench.TRAFFIC_FILE))
    assert len(tf["kernel_source_hash"]) == 16 and tf["workload"][:3] == [2000, 8, 80] and tf["kernels"]
