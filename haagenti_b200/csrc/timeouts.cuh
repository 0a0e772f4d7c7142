// Which device-side timeouts have been reported.  Host code without CUDA.
#pragma once

#include <atomic>
#include <cstdint>

namespace hct {

// A device counts its expired waits and never clears the count, so that a wait
// that expires while the count is being read is in the next reading and cannot be
// lost.  The host remembers how far each device's count has been reported.
class ReportedTimeouts {
  public:
    // Whether `count`, read from `device`, holds a timeout that no call has reported.
    // Readings may arrive in another order than they were made: an older one is
    // covered by the later one's report.  Devices past the table report again what
    // they have counted.
    bool report(int device, uint32_t count) {
        if (device < 0 || device >= DEVICES) return count != 0;
        std::atomic<uint32_t> &seen = seen_[device];
        uint32_t before = seen.load();
        while ((int32_t)(count - before) > 0)
            if (seen.compare_exchange_weak(before, count)) return true;
        return false;
    }

  private:
    static constexpr int DEVICES = 64;
    std::atomic<uint32_t> seen_[DEVICES] = {};
};

}  // namespace hct
