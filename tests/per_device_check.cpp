// Host check of PerDevice (csrc/per_device.cuh): prints "ok" or the first failure.
#include <cstdio>
#include <thread>
#include <vector>

#include "per_device.cuh"

int main() {
    hct::PerDevice p;
    int asked = 0;
    const auto say = [&](uint32_t v) { return [&asked, v] { return asked++, v; }; };
    if (p.get(0, say(0)) != 0 || p.get(0, say(148)) != 148) return std::puts("a failure was remembered"), 1;
    if (p.get(1, say(132)) != 132) return std::puts("devices share an answer"), 1;
    if (p.get(0, say(7)) != 148 || p.get(1, say(7)) != 132 || asked != 3) return std::puts("asked again"), 1;
    if (p.get(64, say(5)) != 5 || p.get(64, say(6)) != 6 || p.get(-1, say(9)) != 9)
        return std::puts("devices past the table"), 1;
    hct::PerDevice q;
    std::atomic<int> wrong{0};
    std::vector<std::thread> threads;
    for (int i = 0; i < 8; i++)
        threads.emplace_back([&, i] {
            for (int j = 0; j < 20000; j++) {
                const int dev = (i + j) % 64;
                if (q.get(dev, [dev] { return 100u + dev; }) != 100u + dev) wrong++;
            }
        });
    for (auto &t : threads) t.join();
    if (wrong) return std::puts("threads disagree"), 1;
    std::puts("ok");
    return 0;
}
