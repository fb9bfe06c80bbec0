// wc_once.h -- an action that has to have happened once per device before a launch (the opt-in to more than 64 KB of LDS, which
// hipFuncSetAttribute makes for the current device).  No HIP in here.
#pragma once
#include <atomic>
#include <mutex>

namespace wc {

struct OncePerKey {
    static constexpr int kKeys = 64;
    std::mutex m;
    std::atomic<bool> done[kKeys] = {};
    // True once `action` has succeeded for `key`; it runs under the lock, so that a second thread does not go on before it has,
    // and again in the next call if it fails.  Keys outside the table: in every call.
    template <class Action>
    bool run(int key, Action&& action) {
        if (key < 0 || key >= kKeys) return action();
        if (done[key].load(std::memory_order_acquire)) return true;
        std::lock_guard<std::mutex> lock(m);
        if (done[key].load(std::memory_order_relaxed)) return true;
        if (!action()) return false;
        done[key].store(true, std::memory_order_release);
        return true;
    }
};

}  // namespace wc
