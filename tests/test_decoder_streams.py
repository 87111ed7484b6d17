"""Two threads, each with a stream of its own, run a decoding step (rotary, append, attention over the cache with its joined
parts, gated projection) and a training step at once, and two decoding steps at once: every result equals the one computed alone.

PyTorch supplies streams and memory.  The body runs in a process of its own that imports torch before the library touches the GPU
(torch brings its own copy of the HIP runtime)."""
import os
import subprocess
import sys

import pytest

HERE = os.path.dirname(os.path.abspath(__file__))


@pytest.mark.gpu
def test_decoding_steps_on_two_streams_at_once():
    out = subprocess.run([sys.executable, "-u", os.path.abspath(__file__)], capture_output=True, text=True, timeout=110)
    assert out.returncode == 0, out.stdout[-3000:] + out.stderr[-3000:]
    assert "streams equal alone" in out.stdout


def _body():
    import threading
    import torch
    sys.path[:0] = [os.path.dirname(HERE), HERE]
    torch.zeros(1, device="cuda")
    from deep_learning_framework_amd import kai
    from test_decoder_graph import Decode, Train
    kai.load()
    kai.set_device(0)
    plan = kai.VMath.cache_attention_plan(3, 5, 8, 2, 64, 32, 40)
    assert plan.startswith("tiles of 16 rows, 10 parts"), plan            # its parts meet in the scratch
    same = lambda a, b: all(torch.equal(x, y) for x, y in zip(a, b))
    works = [Decode(torch, kai, 1), Decode(torch, kai, 7), Train(torch, kai, 2)]
    want = {}
    for i, w in enumerate(works):
        for seed in range(1, 5):
            w.inputs(seed)
            w.step()
            torch.cuda.synchronize()
            want[i, seed] = w.outputs()
    for pair in ((0, 2), (0, 1)):
        bad, go = [], threading.Barrier(2, timeout=60)

        def run(k):
            try:
                s = torch.cuda.Stream()
                kai.set_stream(s.cuda_stream)
                with torch.cuda.stream(s):
                    for n in range(12):
                        seed = 1 + n % 4
                        works[k].inputs(seed)
                        s.synchronize()
                        go.wait()
                        works[k].step()
                        s.synchronize()
                        if not same(works[k].outputs(), want[k, seed]):
                            bad.append((k, seed))
            except Exception as e:
                bad.append((k, repr(e)))
                go.abort()

        threads = [threading.Thread(target=run, args=(k,)) for k in pair]
        for t in threads:
            t.start()
        for t in threads:
            t.join()
        torch.cuda.synchronize()
        assert not bad, (pair, bad)
        print("ok", pair, flush=True)
    print("streams equal alone", flush=True)


if __name__ == "__main__":
    _body()
