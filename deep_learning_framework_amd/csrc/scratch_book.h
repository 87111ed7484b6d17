// The books of a device's scratch memory (kai_common.h: workspace()), apart from the runtime's calls, so that they can be
// checked without a GPU.  Whoever uses them holds the lock.
//
// Per device: one scratch buffer per STREAM that calls of the library have been enqueued on (the stream a thread
// set with kai_set_stream; the null stream counts as one), so that calls on different streams of a device never
// share partial sums, and the smaller buffers that grown ones replaced.  A replaced buffer is only retired: kernels
// already enqueued that use it stay valid, and growing needs neither a wait for the device nor a hipFree (which
// waits for the device, too).  Retired buffers are released at the library's own synchronisation points, when the
// device is idle anyway (kai_device_synchronize, kai_shutdown) -- except those that were handed out while a stream
// capture was active: a recorded graph keeps the address and may be replayed at any later time, so they stay until
// kai_shutdown.  Growth at least doubles the size, so the retired buffers of a stream together are smaller than
// its current one.
//
// A call that holds data in the scratch across inner calls (ScratchHold) may have its buffer retired by an inner one and
// enqueue kernels on it afterwards, while another thread waits for the device: `holds` counts such calls of a stream, and
// what is retired there stays until a wait that begins when none is left.
#pragma once

#include <stdint.h>

#include <vector>

namespace kai {

struct StreamScratch {
    const void* stream = nullptr;
    void* ptr = nullptr;
    int64_t bytes = 0;
    bool in_graph = false;     // handed out during a capture
    int holds = 0;             // calls in progress that keep data in it
};
struct RetiredScratch {
    void* ptr;
    int64_t bytes;
    bool in_graph;
    const void* stream;
};
struct DeviceScratch {
    std::vector<StreamScratch> streams;
    std::vector<RetiredScratch> retired;
    int64_t retired_bytes = 0;
    int64_t growths = 0;

    StreamScratch* find(const void* stream) {
        for (StreamScratch& e : streams)
            if (e.stream == stream) return &e;
        return nullptr;
    }
    void put_back(const RetiredScratch& r) {
        retired.push_back(r);
        retired_bytes += r.bytes;
    }
    void replace(StreamScratch& s, void* fresh, int64_t bytes) {
        if (s.ptr) put_back(RetiredScratch{s.ptr, s.bytes, s.in_graph, s.stream});
        s.ptr = fresh;
        s.bytes = bytes;
        s.in_graph = false;
        growths++;
    }
    void hold(const void* stream, int more) {
        StreamScratch* s = find(stream);
        if (s == nullptr) return;                  // the buffers were released meanwhile (kai_shutdown)
        s->holds += more;
        if (s->holds < 0) s->holds = 0;
    }
    // Takes the retired buffers that no kernel will name any more once a wait for the device that begins NOW has ended.
    // What is retired during that wait is the next one's.
    std::vector<RetiredScratch> take_idle() {
        std::vector<RetiredScratch> idle, kept;
        for (const RetiredScratch& r : retired) {
            const StreamScratch* s = find(r.stream);
            if (r.in_graph || (s && s->holds > 0)) {
                kept.push_back(r);
            } else {
                idle.push_back(r);
                retired_bytes -= r.bytes;
            }
        }
        retired.swap(kept);
        return idle;
    }
};

}  // namespace kai
