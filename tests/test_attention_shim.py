"""Runs tests/cpp/attention_check.cpp: attention and the token log probabilities through the C++ shim."""
import os
import subprocess

import pytest

BIN = os.path.join(os.path.dirname(os.path.abspath(__file__)), "cpp", "build", "attention_check")


def run(*args):
    assert os.path.exists(BIN), "build it with `make -C tests/cpp` (done by __graft_entry__.build())"
    r = subprocess.run([BIN, *args], capture_output=True, text=True, timeout=100)
    print(r.stdout[-3000:], r.stderr[-2000:])
    assert r.returncode == 0 and "RESULT: PASS" in r.stdout


def test_shim_refusals():
    run("host")


@pytest.mark.gpu
def test_shim_calls():
    run()
