"""The DRAM traffic figures recorded for bench.py belong to the kernels as they are."""
import importlib
import json
import os

import pytest

from conftest import ROOT

P = "tensor-compiler-webgpu_b200"


def _launch_sources(pkg, name):
    wl, cg = importlib.import_module(P + ".workloads"), importlib.import_module(P + ".codegen")
    W = {"c2": lambda: wl.c2_graph(8192, 8192), "c3": lambda: wl.c3_graph(4096, 4096, 4096, "relu"),
         "c4": lambda: wl.c4_graph(65536, 4096, "softmax")}[name]()
    f = pkg.fuse.fuse(W["graph"], keep=W["keep"])
    kept = [f.index[i] for i in W["keep"]]
    for kw in ({}, {"keep": kept, "fold": True, "colfuse": True, "mofuse": True}):
        for lau in cg.lower_fused(f.graph, matmul="tiled", **kw)["launches"]:
            yield lau.code


@pytest.mark.parametrize("name", ["c2", "c3", "c4"])
def test_recorded_traffic_is_of_a_current_kernel(pkg, name):
    """Otherwise the bench line has no traffic for it: a template moved to a header of its own orphaned C3's."""
    bench = importlib.import_module("bench")
    with open(os.path.join(ROOT, "profiles", "traffic.json")) as f:
        recorded = json.load(f)[name]
    assert recorded["code_hash"] in {bench._code_hash(code) for code in _launch_sources(pkg, name)}


def test_the_hash_covers_what_a_template_includes(pkg, tmp_path, monkeypatch):
    bench = importlib.import_module("bench")
    d = tmp_path / P / "csrc" / "templates"
    d.mkdir(parents=True)
    (d / "outer1.cuh").write_text('#include "tcb/inner.cuh"\nint a;\n')
    (d / "inner.cuh").write_text("int b;   // one\n")
    monkeypatch.setattr(bench, "ROOT", str(tmp_path))
    code = '#include "tcb/outer1.cuh"\n'
    first = bench._code_hash(code)
    (d / "inner.cuh").write_text("int b;   // another comment\n\n")
    assert bench._code_hash(code) == first
    (d / "inner.cuh").write_text("int c;\n")
    assert bench._code_hash(code) != first
