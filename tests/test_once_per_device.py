"""CPU: what a kernel's first launch on a device sets up is there for every thread that launches it, also while it is being set up."""
import shutil
import subprocess

import pytest

from conftest import PKG

PROGRAM = r"""
#include <chrono>
#include <cstdio>
#include <thread>
#include <vector>
#include "b2g_once.h"

int main() {
  // many threads at once: one of them sets up, slowly, and none returns before it is done
  for (int dev : {0, 1, 63}) {
    b2g::OncePerDevice once;
    std::atomic<int> calls{0}, ready{0}, early{0};
    std::vector<std::thread> all;
    for (int i = 0; i < 16; ++i)
      all.emplace_back([&] {
        const int rc = b2g::once_on(once, dev, [&] {
          ++calls;
          std::this_thread::sleep_for(std::chrono::milliseconds(50));
          ready = 1;
          return 0;
        });
        if (rc != 0 || !ready) ++early;
      });
    for (auto& t : all) t.join();
    if (early || calls != 1) { std::printf("device %d: %d early, %d calls\n", dev, early.load(), calls.load()); return 1; }
  }
  // devices are apart; a failure is reported and tried again; an unknown device is set up every time
  b2g::OncePerDevice once;
  int calls = 0;
  auto set = [&] { return ++calls == 1 ? -2 : 0; };
  if (b2g::once_on(once, 3, set) != -2 || b2g::once_on(once, 3, set) != 0 || b2g::once_on(once, 3, set) != 0 || calls != 2) return 2;
  if (b2g::once_on(once, 4, set) != 0 || calls != 3) return 3;
  if (b2g::once_on(once, -1, set) != 0 || b2g::once_on(once, -1, set) != 0 || calls != 5) return 4;
  return 0;
}
"""


def test_once_per_device(tmp_path):
    gxx = shutil.which("g++")
    if gxx is None:
        pytest.skip("no host compiler")
    src, exe = tmp_path / "once.cpp", tmp_path / "once"
    src.write_text(PROGRAM)
    subprocess.run([gxx, "-std=c++17", "-O1", "-pthread", "-I", str(PKG / "csrc"), str(src), "-o", str(exe)], check=True, timeout=120)
    r = subprocess.run([str(exe)], capture_output=True, text=True, timeout=60)
    assert r.returncode == 0, (r.returncode, r.stdout)
