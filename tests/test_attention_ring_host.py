"""The 16-row attention kernel's query ring, with the kernel's own turns, against every order of its sides."""

import os
import subprocess
from pathlib import Path

import pytest

ROOT = Path(__file__).resolve().parents[1]


@pytest.fixture(scope="module")
def model(tmp_path_factory):
    exe = tmp_path_factory.mktemp("ring") / "model"
    subprocess.run([os.environ.get("CXX") or "g++", "-O2", "-std=c++17", "-x", "c++",
                    f"-I{ROOT / 'vllm_ascend_hust_latchmoe_b200/csrc'}",
                    str(ROOT / "tests/attention_ring_model.cpp"), "-o", str(exe)], check=True)

    def run(protocol):
        out = subprocess.run([str(exe), protocol], check=True, capture_output=True, text=True, timeout=300).stdout
        return tuple(map(int, out.split()))

    return run


def test_turns_hold_for_every_pattern_of_segments_without_keys(model):
    patterns, broken = model("turns")
    assert patterns == 2 ** 11 - 2 and broken == 0


def test_the_model_tells_turns_by_segment_number_apart(model):
    _, broken = model("segments")
    assert broken > 0
