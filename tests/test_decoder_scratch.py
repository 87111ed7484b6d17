"""A caller reserves what the header says and records: no call of the gated projection asks for more.

PyTorch supplies streams, graphs and memory.  The body runs in a process of its own that imports torch before the library
touches the GPU (torch brings its own copy of the HIP runtime)."""
import os
import subprocess
import sys

import pytest


@pytest.mark.gpu
def test_reserved_scratch_is_enough_for_a_capture():
    out = subprocess.run([sys.executable, "-u", os.path.abspath(__file__)], capture_output=True, text=True, timeout=110)
    assert out.returncode == 0, out.stdout[-3000:] + out.stderr[-3000:]
    assert "reserved scratch is enough" in out.stdout


def _body():
    import torch
    sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
    dev = torch.device("cuda:0")
    torch.zeros(1, device=dev)
    from deep_learning_framework_amd import kai
    kai.load()
    kai.set_device(0)
    P, V = lambda a: a.data_ptr(), kai.VMath
    stream = torch.cuda.Stream()
    # the small one takes 16 parts of 16 tiles, the large one cut its rest into 192 MiB of parts; 24 rows run as separate products,
    # 64 x 20000 has wide bias sums, and those of 9 million columns would pass 64 MiB: they are taken from the gradients
    for ndat, xvec, yvec in ((193, 4096, 193), (4096, 1024, 11008), (24, 4096, 11008), (64, 300, 20000), (2, 1, 9000000)):
        gen = torch.Generator(device=dev).manual_seed(ndat)
        r = lambda *s: torch.empty(s, device=dev).normal_(generator=gen).mul_(0.05)
        x, wg, wu, gate, up, gy = r(ndat, xvec), r(yvec, xvec), r(yvec, xvec), r(ndat, yvec), r(ndat, yvec), r(ndat, yvec)
        outs = [r(ndat, yvec), r(ndat, xvec), r(yvec, xvec), r(yvec, xvec), r(yvec), r(yvec)]

        def step():
            V.gated_forward(0, P(outs[0]), None, None, P(wg), P(wu), None, None, P(x), yvec, ndat, xvec, 8, None)
            V.gated_backward(0, *(P(o) for o in outs[1:]), None, P(gy), P(wg), P(wu), P(x), P(gate), P(up), yvec, ndat, xvec, 8,
                             None, False)

        torch.cuda.synchronize()
        kai.shutdown()
        kai.set_stream(stream.cuda_stream)
        kai.reserve_scratch((64 << 20) + (2 * ndat * yvec * 4 + 255) // 256 * 256)
        with torch.cuda.stream(stream):
            graph = torch.cuda.CUDAGraph()
            torch.cuda.synchronize()
            with torch.cuda.graph(graph, stream=stream):
                step()
            torch.cuda.synchronize()
            assert kai.scratch_info()[1] == 1, "the reserved buffer, and no other"
            step()                                   # eager, through the same buffer
            torch.cuda.synchronize()
            want = [o.clone() for o in outs]
            for _ in range(3):
                for o in outs:
                    o.fill_(float("nan"))
                graph.replay()
                torch.cuda.synchronize()
                assert all(torch.equal(a, b) for a, b in zip(outs, want))
            assert kai.scratch_info()[1] == 1
        sg = torch.sigmoid(gate.double())
        for got, each in ((outs[4], gy * up * (sg + gate * sg * (1 - sg))), (outs[5], gy * gate * sg)):
            # of ndat numbers below 0.05^2 * 6^2: as many roundings as there are terms, and some for the slope
            assert (got - each.sum(0)).abs().max() <= (ndat + 20) * 2.0 ** -24 * each.abs().sum(0).max()
        del graph
        kai.set_stream(None)
        torch.cuda.synchronize()
        print("ok", ndat, xvec, yvec, flush=True)
    print("reserved scratch is enough", flush=True)


if __name__ == "__main__":
    _body()
