"""The operators of a decoder block recorded into HIP graphs and run on several streams: a step of decoding and a training
step of the gated projection are captured once and replayed on new inputs between eager calls, two recorded graphs of one
stream take turns with the library scratch, and two threads work on streams of their own at once.  Every result must equal
the eager call's bit for bit.

PyTorch supplies streams, graphs and memory.  The body runs in a process of its own that imports torch before the library
touches the GPU (torch brings its own copy of the HIP runtime)."""
import os
import subprocess
import sys

import pytest


@pytest.mark.gpu
def test_decoder_graphs_and_streams_equal_eager():
    out = subprocess.run([sys.executable, "-u", os.path.abspath(__file__)], capture_output=True, text=True, timeout=110)
    assert out.returncode == 0, out.stdout[-3000:] + out.stderr[-3000:]
    assert "decoder graphs and streams equal eager" in out.stdout


class Decode:
    """Rotary, append, attention over the cache and the gated projection of one step, in buffers of its own."""

    def __init__(self, torch, kai, seed):
        self.kai, self.dev = kai, torch.device("cuda:0")
        self.gen = torch.Generator(device=self.dev).manual_seed(seed)
        self.nbat, self.nt, self.nh, self.nkv, self.np, self.page, self.most = 3, 5, 8, 2, 64, 32, 40
        t = lambda *s: torch.empty(s, device=self.dev)
        width, nvec = self.nkv * self.np, self.nh * self.np
        self.ck, self.cv = t(self.nbat * self.most, self.page, width), t(self.nbat * self.most, self.page, width)
        self.ck.normal_(generator=self.gen)
        self.cv.normal_(generator=self.gen)
        self.before = self.ck.clone(), self.cv.clone()
        self.q, self.k, self.v = t(self.nbat, self.nt, nvec), t(self.nbat, self.nt, width), t(self.nbat, self.nt, width)
        self.y, self.h = t(self.nbat, self.nt, nvec), t(self.nbat * self.nt, 320)
        self.wg, self.wu = t(320, nvec), t(320, nvec)
        self.wg.normal_(generator=self.gen).mul_(0.05)
        self.wu.normal_(generator=self.gen).mul_(0.05)
        self.table = torch.randperm(self.nbat * self.most).view(self.nbat, self.most).to(torch.int32).to(self.dev)
        self.len = torch.zeros(self.nbat, dtype=torch.int32, device=self.dev)
        self.count = torch.full((self.nbat,), self.nt, dtype=torch.int32, device=self.dev)
        self.pos = torch.zeros(self.nbat, self.nt, dtype=torch.int32, device=self.dev)
        self.coef = torch.full((1,), 0.125, device=self.dev)
        self.desc = kai.rotary_desc(64, layout="pairs")
        self.torch = torch

    def inputs(self, seed):
        self.gen.manual_seed(seed)
        for a in (self.q, self.k, self.v):
            a.normal_(generator=self.gen)
        self.y.fill_(0)
        self.ck.copy_(self.before[0])
        self.cv.copy_(self.before[1])
        self.len.copy_(self.torch.tensor([1000 - seed, 37 * seed, 3], dtype=self.torch.int32))
        self.count.copy_(self.torch.tensor([self.nt, 1 + seed % 4, 2], dtype=self.torch.int32))
        self.pos.copy_(self.len[:, None] + self.torch.arange(self.nt, device=self.dev))

    def step(self):
        P, V = lambda a: a.data_ptr(), self.kai.VMath
        nvec, width, npage = self.nh * self.np, self.nkv * self.np, self.nbat * self.most
        V.rotary(0, P(self.q), P(self.q), P(self.pos), self.nbat, self.nt, nvec, self.nh, self.np, self.desc)
        V.cache_append(0, P(self.ck), P(self.cv), P(self.k), P(self.v), P(self.table), P(self.len), P(self.count), None, self.nbat,
                       self.nt, width, self.nkv, self.np, npage, self.page, self.most, self.desc)
        V.cache_attention(0, P(self.y), P(self.q), P(self.ck), P(self.cv), P(self.table), P(self.len), P(self.count), None,
                          self.nbat, self.nt, nvec, self.nh, self.nkv, self.np, npage, self.page, self.most, P(self.coef))
        V.gated_forward(0, P(self.h), None, None, P(self.wg), P(self.wu), None, None, P(self.y), 320, self.nbat * self.nt, nvec, 8,
                        None)

    def outputs(self):
        return [a.clone() for a in (self.q, self.ck, self.cv, self.y, self.h)]


class Train:
    """Forward and all gradients of the gated projection: parts of a reduction and bias sums in the library scratch."""

    def __init__(self, torch, kai, seed, ndat=200, xvec=520, yvec=300):
        self.kai, self.size = kai, (yvec, ndat, xvec)
        self.dev = torch.device("cuda:0")
        self.gen = torch.Generator(device=self.dev).manual_seed(seed)
        t = lambda *s: torch.empty(s, device=self.dev)
        self.x, self.gy = t(ndat, xvec), t(ndat, yvec)
        self.wg, self.wu, self.bg, self.bu = t(yvec, xvec), t(yvec, xvec), t(yvec), t(yvec)
        self.y, self.gate, self.up = t(ndat, yvec), t(ndat, yvec), t(ndat, yvec)
        self.gx, self.gwg, self.gwu, self.gbg, self.gbu = t(ndat, xvec), t(yvec, xvec), t(yvec, xvec), t(yvec), t(yvec)

    def inputs(self, seed):
        self.gen.manual_seed(seed)
        for a in (self.x, self.gy, self.wg, self.wu, self.bg, self.bu):
            a.normal_(generator=self.gen).mul_(0.1)

    def step(self):
        P, V = lambda a: a.data_ptr(), self.kai.VMath
        V.gated_forward(0, P(self.y), P(self.gate), P(self.up), P(self.wg), P(self.wu), P(self.bg), P(self.bu), P(self.x),
                        *self.size, 8, None)
        V.gated_backward(0, P(self.gx), P(self.gwg), P(self.gwu), P(self.gbg), P(self.gbu), None, P(self.gy), P(self.wg),
                         P(self.wu), P(self.x), P(self.gate), P(self.up), *self.size, 8, None, False)

    def outputs(self):
        return [a.clone() for a in (self.y, self.gate, self.up, self.gx, self.gwg, self.gwu, self.gbg, self.gbu)]


def _body():
    import threading
    import torch
    sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
    torch.zeros(1, device="cuda")
    from deep_learning_framework_amd import kai
    kai.load()
    kai.set_device(0)
    same = lambda a, b: all(torch.equal(x, y) for x, y in zip(a, b))

    def eager(work, seed):
        work.inputs(seed)
        work.step()
        torch.cuda.synchronize()
        return work.outputs()

    works = [Decode(torch, kai, 1), Train(torch, kai, 2), Train(torch, kai, 3, ndat=90, xvec=1030, yvec=64)]
    want = {(i, seed): eager(w, seed) for i, w in enumerate(works) for seed in range(1, 5)}

    # graphs, all of one stream and so of one scratch buffer, replayed in turn with eager calls between them
    stream = torch.cuda.Stream()
    graphs = []
    with torch.cuda.stream(stream):
        kai.set_stream(stream.cuda_stream)
        for w in works:
            w.inputs(9)
            w.step()
        torch.cuda.synchronize()
        for w in works:
            g = torch.cuda.CUDAGraph()
            w.inputs(9)
            torch.cuda.synchronize()
            with torch.cuda.graph(g, stream=stream):
                w.step()
            graphs.append(g)
        torch.cuda.synchronize()
        for seed in range(1, 5):
            for i, (w, g) in enumerate(zip(works, graphs)):
                w.inputs(seed)
                g.replay()
                torch.cuda.synchronize()
                assert same(w.outputs(), want[i, seed]), (i, seed)
                assert same(eager(works[i - 1], seed), want[(i - 1) % 3, seed]), (i, seed, "eager between replays")
    kai.set_stream(None)
    torch.cuda.synchronize()
    print("graphs ok", flush=True)

    # two threads, a stream each, at once
    bad = []

    def run(work, key):
        s = torch.cuda.Stream()
        kai.set_stream(s.cuda_stream)
        with torch.cuda.stream(s):
            for n in range(12):
                seed = 1 + n % 4
                work.inputs(seed)
                work.step()
                s.synchronize()
                if not same(work.outputs(), want[key, seed]):
                    bad.append((key, seed))

    threads = [threading.Thread(target=run, args=(works[k], k)) for k in (1, 2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    assert not bad, bad
    # a capture that the scratch is too small for is refused, not recorded wrong
    kai.shutdown()
    s = torch.cuda.Stream()
    kai.set_stream(s.cuda_stream)
    refused = False
    g = torch.cuda.CUDAGraph()
    with torch.cuda.stream(s):
        torch.cuda.synchronize()
        g.capture_begin()
        try:
            works[0].step()
        except kai.KaiError as e:
            refused = e.code == 50002 and "scratch" in e.message
        g.capture_end()
    kai.set_stream(None)
    assert refused
    assert same(eager(works[1], 2), want[1, 2])
    print("decoder graphs and streams equal eager", flush=True)


if __name__ == "__main__":
    _body()
