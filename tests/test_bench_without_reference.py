"""bench.py where the reference's sources, and so oracle/_ref, are not there (CPU): the reference arm says so and ends well, and
this repository's own lines go without a CPU baseline."""
import argparse
import importlib.util
import os
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture
def bench(monkeypatch):
    sys.path.insert(0, ROOT)
    from oracle import refvm
    monkeypatch.setattr(refvm, "lib", lambda: None)
    spec = importlib.util.spec_from_file_location("bench_alone", os.path.join(ROOT, "bench.py"))
    b = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(b)
    return b


@pytest.mark.parametrize("workload", ["all", "decode", "decode_small", "prefill", "ssm"])
def test_the_reference_arm_is_unavailable(bench, workload):
    args = argparse.Namespace(workload=workload, steps=1, warmup=3, seqs=0, prompt=0, new=0, layers=0, bits=4, m=[1])
    line, = bench.reference_arm(args)
    assert line["impl"] == "reference" and line["unavailable"] and "value" not in line


def test_own_lines_have_no_cpu_baseline(bench):
    assert bench.cpu_baseline_decode() is None and bench.cpu_baseline_prefill() is None and bench.cpu_baseline_ssm() is None
