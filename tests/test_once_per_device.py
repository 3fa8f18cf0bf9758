"""csrc/rtp_once.h, the one-time set-up of a kernel on a device: built and run on the CPU."""
import os
import subprocess

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "rt_pose_amd", "csrc")

PROGRAM = r"""
#include <cassert>
#include <chrono>
#include <thread>
#include <vector>

#include "rtp_once.h"

int main() {
  // threads that arrive during the first one's set-up do not go on in front of its end
  static std::atomic<bool> done[RTP_MAX_DEVICES];
  std::atomic<int> inside{0}, complete{0}, early{0};
  std::vector<std::thread> threads;
  auto user = [&] {
    const bool ok = rtp_once(done, 3, [&] {
      inside = 1;
      std::this_thread::sleep_for(std::chrono::milliseconds(100));
      complete = 1;
      return true;
    });
    if (!ok || !complete) early = 1;
  };
  threads.emplace_back(user);
  while (!inside) std::this_thread::yield();
  for (int i = 0; i < 4; ++i) threads.emplace_back(user);
  for (auto& t : threads) t.join();
  assert(!early);

  int calls = 0;
  auto count = [&] { ++calls; return true; };
  assert(rtp_once(done, 3, count) && calls == 0);        // done
  assert(rtp_once(done, 4, count) && calls == 1);        // another device
  assert(rtp_once(done, 4, count) && calls == 1);

  // a set-up that fails is tried again
  static std::atomic<bool> other[RTP_MAX_DEVICES];
  assert(!rtp_once(other, 0, [&] { return false; }));
  assert(rtp_once(other, 0, count) && calls == 2);
  assert(rtp_once(other, 0, count) && calls == 2);

  // devices without a flag are set up every time, and never in another one's name
  for (int d : {-1, RTP_MAX_DEVICES, RTP_MAX_DEVICES + 48}) {
    const int before = calls;
    assert(rtp_once(other, d, count) && rtp_once(other, d, count) && calls == before + 2);
  }
  return 0;
}
"""


def test_nothing_goes_on_in_front_of_a_complete_set_up(tmp_path):
    src, exe = tmp_path / "once.cpp", tmp_path / "once"
    src.write_text(PROGRAM)
    subprocess.run(["g++", "-std=c++17", "-O1", "-pthread", "-I", CSRC, str(src), "-o", str(exe)], check=True)
    subprocess.run([str(exe)], check=True, timeout=60)
