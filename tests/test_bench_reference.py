"""CPU: bench.py where the reference's compiled operator is absent."""

import argparse
import json

import pytest

import bench
from oracle import oracle as O
from torchsoftdtw_b200.workloads import WORKLOADS


@pytest.fixture
def no_reference(monkeypatch, tmp_path):
    monkeypatch.setattr(O, "REF_SO", str(tmp_path / "missing.so"))
    monkeypatch.setattr(O, "build", lambda: None)


def test_reference_arm_says_that_it_is_unavailable(no_reference, capsys):
    args = argparse.Namespace(cpu_sample=1, steps=1, warmup=1)
    bench.run_reference_arm(args, WORKLOADS["medium"], 0, 1)
    line = json.loads(capsys.readouterr().out)
    assert line["impl"] == "reference" and "oracle/_ref" in line["unavailable"]


def test_the_measurement_names_what_is_missing(no_reference):
    with pytest.raises(bench.ReferenceUnavailable):
        bench.cpu_reference_measure(WORKLOADS["medium"], 1, 1, 1)
