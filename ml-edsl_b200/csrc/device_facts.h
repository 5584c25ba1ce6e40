// What the host asks the driver about a device and a kernel before it launches.
// No CUDA in here: the queries are the callers'.
#pragma once
#include <atomic>
#include <mutex>

namespace b200 {

// A value for each device, made when it is first asked for there; once, also when
// several threads ask at the same time. Devices differ, and what one gives must
// not decide how another one runs.
template <class T>
class PerDevice {
 public:
  template <class Make>
  T of(int device, Make make) {
    if (device < 0 || device >= kDevices) return make();
    Slot& s = slots_[device];
    if (!s.made.load(std::memory_order_acquire)) {
      std::lock_guard<std::mutex> lock(making_);
      if (!s.made.load(std::memory_order_relaxed)) {
        s.value = make();
        s.made.store(true, std::memory_order_release);
      }
    }
    return s.value;
  }

 private:
  static constexpr int kDevices = 64;
  struct Slot {
    std::atomic<bool> made{false};
    T value{};
  };
  Slot slots_[kDevices];
  std::mutex making_;
};

// What `ask(&n)` gives (true: the query went well), or `otherwise` where it fails
// or gives nothing. `forget` takes the error of a failing query back, so that the
// next launch's check does not report it.
template <class Ask, class Forget>
int ask_or(int otherwise, Ask ask, Forget forget) {
  int n = 0;
  if (!ask(&n)) {
    forget();
    return otherwise;
  }
  return n > 0 ? n : otherwise;
}

}  // namespace b200
