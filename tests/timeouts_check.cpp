// Host check of ReportedTimeouts (csrc/timeouts.cuh): prints "ok" or the first failure.
#include <cstdio>
#include <thread>
#include <vector>

#include "timeouts.cuh"

static int fail(const char *what) {
    std::printf("%s\n", what);
    return 1;
}

int main() {
    hct::ReportedTimeouts r;
    if (r.report(0, 0)) return fail("nothing counted, yet reported");
    if (!r.report(0, 3)) return fail("a timeout was lost");
    if (r.report(0, 3)) return fail("reported twice");
    if (!r.report(0, 4)) return fail("one that expired after the last reading was lost");
    if (r.report(0, 3)) return fail("an older reading reported again");
    if (r.report(0, 4)) return fail("an older reading brought back the later one");
    if (r.report(1, 0) || !r.report(1, 1) || !r.report(63, 1)) return fail("devices share a count");
    if (!r.report(64, 1) || r.report(64, 0) || !r.report(-1, 1)) return fail("a device past the table");
    // the count passes 2^32
    hct::ReportedTimeouts w;
    if (!w.report(0, 0x7fffffffu) || !w.report(0, 0xfffffffeu) || !w.report(0, 2)) return fail("wrap");

    // threads that count and read at once: after each expiry some later call reports, and
    // there are no more reports than expiries
    for (int round = 0; round < 50; round++) {
        hct::ReportedTimeouts t;
        std::atomic<uint32_t> count{0}, reports{0};
        std::vector<std::thread> threads;
        for (int i = 0; i < 4; i++)
            threads.emplace_back([&] {
                for (int j = 0; j < 500; j++) {
                    count.fetch_add(1);
                    if (t.report(0, count.load())) reports.fetch_add(1);
                }
            });
        for (auto &th : threads) th.join();
        if (t.report(0, count.load())) return fail("the last expiry had not been reported");
        if (reports.load() == 0 || reports.load() > count.load()) return fail("too many reports");
    }
    std::printf("ok\n");
    return 0;
}
