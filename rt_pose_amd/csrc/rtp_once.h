// One-time set-up for each device (hipFuncSetAttribute is per device: a process-wide flag would leave a second GPU of the same process without its
// LDS limit).  Host code without HIP, so that it is tested by itself.
#pragma once
#include <atomic>

#define RTP_MAX_DEVICES 16

// True once `set` has succeeded for this device; false if it fails now, and the next call then tries again.  `done`: static, one flag for each device.
// Threads that come here together each run `set`, which has to allow it: the flag is only raised behind a set-up that is complete, so that no thread
// goes on to a launch in front of it.  Devices without a flag (or unknown ones) are set up every time.
template <typename F>
static inline bool rtp_once(std::atomic<bool>* done, int device, F set) {
  const bool known = device >= 0 && device < RTP_MAX_DEVICES;
  if (known && done[device].load(std::memory_order_acquire)) return true;
  if (!set()) return false;
  if (known) done[device].store(true, std::memory_order_release);
  return true;
}
