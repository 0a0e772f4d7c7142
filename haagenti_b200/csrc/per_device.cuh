// A property of each device, asked for once.  Host code without CUDA.
#pragma once

#include <atomic>
#include <cstdint>

namespace hct {

class PerDevice {
  public:
    // `ask`()'s answer for `device`, remembered (of the first 64 devices) unless it is
    // 0, which is no answer.  Threads that ask at once store the same.
    template <class Ask>
    uint32_t get(int device, const Ask &ask) {
        if (device < 0 || device >= DEVICES) return ask();
        uint32_t v = known_[device].load(std::memory_order_relaxed);
        if (!v) {
            v = ask();
            known_[device].store(v, std::memory_order_relaxed);
        }
        return v;
    }

  private:
    static constexpr int DEVICES = 64;
    std::atomic<uint32_t> known_[DEVICES] = {};
};

}  // namespace hct
