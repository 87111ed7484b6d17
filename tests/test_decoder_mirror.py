"""The decoder block's methods of the C++ operator mirror, called from compiled engine-style code
(tests/decoder_mirror_driver.cpp, built by tests/Makefile)."""
import os
import subprocess

import pytest

from util import ROOT

HERE = os.path.join(ROOT, "tests")
DRIVER = os.path.join(HERE, "decoder_mirror_driver")


def run(mode, checks):
    if not os.path.exists(DRIVER):
        subprocess.check_call(["make", "-C", HERE, "-s", "decoder_mirror_driver"])
    r = subprocess.run([DRIVER, mode], stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True, timeout=110)
    assert r.returncode == 0 and "all checks passed" in r.stdout and r.stdout.count("ok  ") == checks, r.stdout


def test_mirror_raises_the_error_codes():
    run("cpu", 7)


@pytest.mark.gpu
def test_mirror_results():
    run("gpu", 6)
