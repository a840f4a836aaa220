// How much dynamic shared memory a kernel may be launched with: an attribute of (kernel, device), so what has been set is remembered for each device.
// Plain C++ without CUDA.
#pragma once
#include <atomic>
#include <mutex>
#include <stddef.h>

#define IFB_MAX_DEVICES 64

// One of a kernel's.  Calls of host threads may meet here (ctypes lets go of the interpreter's lock): it is raised by one at a time, so that no
// thread's smaller size comes behind another's larger one and the launches after it fail.
struct IfbSmemLimit {
  std::atomic<size_t> allowed[IFB_MAX_DEVICES] = {};
  std::mutex lock;
  // set(): sets the attribute to `bytes`; 0, or an error, which is returned.
  template <typename Set> int raise(int device, size_t bytes, Set set) {
    if (bytes <= 48 * 1024 || bytes <= allowed[device].load(std::memory_order_acquire)) return 0;      // (48 KB need no leave)
    std::lock_guard<std::mutex> turn(lock);
    if (bytes <= allowed[device].load(std::memory_order_relaxed)) return 0;
    const int error = set();
    if (error == 0) allowed[device].store(bytes, std::memory_order_release);
    return error;
  }
};
