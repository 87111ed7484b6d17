"""Which scratch buffers a wait for the device releases (csrc/scratch_book.h), checked on the host, and a call whose buffer is
outgrown while it runs beside another thread that waits for the device all the time."""
import os
import subprocess
import threading

import numpy as np
import pytest

from util import ROOT

HERE = os.path.join(ROOT, "tests")


def test_books_of_the_scratch(tmp_path):
    program = str(tmp_path / "scratch_book")
    subprocess.check_call(["g++", "-std=c++17", "-O1", "-Wall", "-Wextra", "-I", os.path.join(ROOT, "deep_learning_framework_amd", "csrc"),
                           "-o", program, os.path.join(HERE, "scratch_book_driver.cpp")])
    r = subprocess.run([program], stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True, timeout=60)
    assert r.returncode == 0 and "all checks passed" in r.stdout and r.stdout.count("ok  ") == 11, r.stdout


@pytest.mark.gpu
def test_a_held_buffer_outlives_another_threads_wait():
    """Gradients of few rows hold their scratch while the products inside ask for more; each size is new, so each call grows."""
    from deep_learning_framework_amd import kai
    from deep_learning_framework_amd.kai import ACT, DeviceBuffer, VMath
    rng = np.random.default_rng(3)
    done = threading.Event()

    def wait():
        while not done.is_set():
            kai.synchronize()

    cases = []
    for ndat, xvec, yvec in ((24, 4096, 700), (32, 5000, 1000), (64, 300, 20000), (300, 700, 9000)):
        x, gy, gate, up = (rng.standard_normal(s).astype(np.float32) for s in ((ndat, xvec), (ndat, yvec), (ndat, yvec), (ndat, yvec)))
        w = (rng.standard_normal((yvec, xvec)) / 64).astype(np.float32)
        cases.append((ndat, xvec, yvec, [DeviceBuffer.from_numpy(a) for a in (gy, w, w, x, gate, up)]))

    def run(ndat, xvec, yvec, given, work):
        out = [DeviceBuffer(4 * n) for n in (ndat * xvec, yvec * xvec, yvec * xvec, yvec, yvec)]
        VMath.gated_backward(0, *out, work, *given, yvec, ndat, xvec, ACT["swish"], None, False)
        return [b.to_numpy(b.nbytes // 4) for b in out]

    kai.synchronize()
    kai.shutdown()
    want = [run(*c, DeviceBuffer(8 * c[0] * c[2])) for c in cases]
    kai.synchronize()
    kai.shutdown()
    thread = threading.Thread(target=wait)
    thread.start()
    try:
        got = [run(*c, None) for c in cases]
    finally:
        done.set()
        thread.join()
    for a, b in zip(want, got):
        assert all(np.array_equal(x, y) for x, y in zip(a, b))
    kai.synchronize()
    assert kai.scratch_info()[2] == 0, "and goes back afterwards"
