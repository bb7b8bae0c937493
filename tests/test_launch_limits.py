"""The launch limits that handles on several host threads share (csrc/
launch_limits.h), with fakes for the CUDA calls (no GPU)."""

import os
import shutil
import subprocess

import pytest

from conftest import PKG

# A fake attribute whose setting takes a while: slower the smaller it is, so
# that a small one which began first ends last.
PROGRAM = r"""
#include <chrono>
#include <cstdio>
#include <thread>
#include <vector>
#include "launch_limits.h"

static std::atomic<size_t> attribute{0};
static std::atomic<int> firsts{0}, lowered{0};

static void set(size_t bytes, bool first) {
  if (first) firsts++;
  std::this_thread::sleep_for(std::chrono::milliseconds(bytes < 1000 ? 40 : 5));
  if (attribute.exchange(bytes) > bytes) lowered++;
}

int main() {
  std::atomic<int> bad{0};
  for (int round = 0; round < 10; round++) {
    attribute = 0;
    firsts = lowered = 0;
    iec::SmemLimit limit;
    std::vector<std::thread> threads;
    for (int t = 0; t < 8; t++)
      threads.emplace_back([&, t] {
        const size_t bytes = t % 2 ? 200 * 1024 : 100;
        limit.raise(0, bytes, set);
        if (attribute < bytes) bad++;  // a launch with `bytes` would fail here
      });
    for (auto& t : threads) t.join();
    if (attribute != 200 * 1024 || firsts != 1 || lowered) bad++;
  }
  // zero bytes are set once too; devices are kept apart
  iec::SmemLimit limit;
  int calls = 0;
  for (int i = 0; i < 3; i++) limit.raise(1, 0, [&](size_t, bool) { calls++; });
  limit.raise(2, 0, [&](size_t, bool first) { calls += first; });
  if (calls != 2) bad++;
  iec::Residency found;
  int looked = 0;
  auto find = [&] { return ++looked * 10; };
  if (found.get(0, 2, 1000, find) != 10 || found.get(0, 2, 2000, find) != 10 || found.get(0, 16, 1000, find) != 20 ||
      found.get(0, 2, 17000, find) != 30 || found.get(1, 2, 1000, find) != 40 || looked != 4)
    bad++;
  // no room is an answer too, and kept
  for (int i = 0; i < 2; i++)
    if (found.get(0, 8, 0, [&] { looked++; return 0; }) != 0 || looked != 5) bad++;
  std::printf("%d\n", bad.load());
  return bad != 0;
}
"""


@pytest.mark.skipif(shutil.which("g++") is None, reason="no g++")
def test_limits_never_go_down_between_threads(tmp_path):
    src, exe = tmp_path / "limits.cpp", tmp_path / "limits"
    src.write_text(PROGRAM)
    subprocess.run(["g++", "-std=c++17", "-O1", "-pthread", "-I", os.path.join(PKG, "csrc"), str(src), "-o", str(exe)], check=True)
    done = subprocess.run([str(exe)], capture_output=True, text=True, timeout=60)
    assert done.returncode == 0, done.stdout


@pytest.mark.gpu
def test_handles_on_two_threads():
    """Two handles, each on its own host thread and stream, with maps of
    sizes that need different amounts of shared memory in turn."""
    import threading

    import torch

    from iec.ops import Ops

    maps = [torch.randn(1, px, 512, device="cuda").half() for px in (16, 100, 300, 700, 1300, 2500, 3600, 12000)]
    with_one = Ops()
    want = [with_one.group_norm(x, 32) for x in maps]
    codes = [with_one.group_norm_fp8(x, 32)[0].view(torch.uint8) for x in maps]
    torch.cuda.synchronize()
    wrong = []

    def work(order):
        try:
            ops, stream = Ops(), torch.cuda.Stream()
            with torch.cuda.stream(stream):
                for _ in range(20):
                    for i in order:
                        if not torch.equal(ops.group_norm(maps[i], 32), want[i]):
                            wrong.append(i)
                        if not torch.equal(ops.group_norm_fp8(maps[i], 32)[0].view(torch.uint8), codes[i]):
                            wrong.append(-i)
            stream.synchronize()
            ops.close()
        except Exception as e:  # noqa: BLE001 (shown by the assertion)
            wrong.append(e)

    threads = [threading.Thread(target=work, args=(o,)) for o in (range(8), range(7, -1, -1))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong
    with_one.close()
