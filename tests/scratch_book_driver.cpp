// Checks the books of the scratch memory (csrc/scratch_book.h) on the host: which retired buffers a wait for the device may
// release.  Built and run by tests/test_scratch_book.py.
#include <cstdio>

#include "scratch_book.h"

static int g_failed = 0;
static void check(bool ok, const char* what) {
    std::printf("%s %s\n", ok ? "ok  " : "FAIL", what);
    if (!ok) g_failed++;
}

int main() {
    char buffers[8];
    int s1, s2;
    kai::DeviceScratch d;
    for (const void* st : {(const void*)&s1, (const void*)&s2}) {
        d.streams.push_back(kai::StreamScratch{});
        d.streams.back().stream = st;
    }
    d.replace(*d.find(&s1), buffers, 10);
    check(d.retired.empty() && d.growths == 1, "a first buffer replaces none");
    d.replace(*d.find(&s1), buffers + 1, 20);
    d.replace(*d.find(&s2), buffers + 2, 10);
    check(d.retired_bytes == 10 && d.growths == 3, "a grown buffer retires the smaller one");

    // A call on s1 holds buffer 1; an inner call of it outgrows it; another thread begins to wait; only then does the call
    // enqueue its next kernel on buffer 1.
    d.hold(&s1, 1);
    d.replace(*d.find(&s1), buffers + 3, 40);
    std::vector<kai::RetiredScratch> idle = d.take_idle();
    check(idle.empty() && d.retired_bytes == 30, "what a call in progress holds is not released");
    d.hold(&s1, 1);        // calls may nest
    d.hold(&s1, -1);
    check(d.take_idle().empty(), "nor while the outer call still runs");
    d.replace(*d.find(&s2), buffers + 4, 20);
    idle = d.take_idle();
    check(idle.size() == 1 && idle[0].ptr == buffers + 2 && d.retired_bytes == 30, "another stream's goes back meanwhile");
    // A wait that began while the call still ran releases nothing of it, though the call ends during the wait.
    idle = d.take_idle();
    d.hold(&s1, -1);
    check(idle.empty(), "a wait that began during the call releases nothing of it");
    idle = d.take_idle();
    check(idle.size() == 2 && d.retired_bytes == 0 && d.retired.empty(), "the next wait does");

    // recorded graphs keep their buffers, and what could not be freed stays on the books
    d.find(&s1)->in_graph = true;
    d.replace(*d.find(&s1), buffers + 5, 80);
    check(d.take_idle().empty() && !d.find(&s1)->in_graph, "a recorded buffer stays");
    d.replace(*d.find(&s2), buffers + 6, 40);
    idle = d.take_idle();
    check(idle.size() == 1, "one is idle");
    d.put_back(idle[0]);
    check(d.take_idle().size() == 1 && d.retired_bytes == 40, "put back, and taken again");

    // the buffers of all streams are gone (kai_shutdown) while a call still holds one
    d = kai::DeviceScratch();
    d.hold(&s1, -1);
    d.streams.push_back(kai::StreamScratch{});
    d.streams.back().stream = &s1;
    d.hold(&s1, -1);
    check(d.find(&s1)->holds == 0, "a hold that outlived its books counts for nothing");
    if (g_failed == 0) std::printf("all checks passed\n");
    return g_failed;
}
