"""The control flow of warps that meet at a barrier in every step, run on host threads: whichever of them gives up, and at
whichever step, all of them leave.  On the device a warp that waits at the barrier for one that has left never ends."""
import os
import subprocess

from conftest import ROOT

PROGRAM = r"""
#include <chrono>
#include <condition_variable>
#include <cstdio>
#include <mutex>
#include <thread>
#include <vector>
#include "ql_together.cuh"

constexpr int kWarps = 4;
struct Barrier { // with a vote, and a limit in place of waiting for good
  std::mutex m;
  std::condition_variable cv;
  int arrived = 0, generation = 0;
  bool all = true, result = false, stuck = false;
  bool meet(bool go) {
    std::unique_lock<std::mutex> lock(m);
    all = all && go;
    const int mine = generation;
    if (++arrived == kWarps) {
      result = all, all = true, arrived = 0, generation++;
      cv.notify_all();
      return result;
    }
    if (!cv.wait_for(lock, std::chrono::seconds(5), [&] { return generation != mine; })) stuck = true;
    return !stuck && result;
  }
};

int main() {
  int cases = 0;
  for (int n = 0; n <= 5; n++) {
    int at[kWarps]; // the step a warp gives up at; n: it never does
    for (int code = 0; code < (n + 1) * (n + 1) * (n + 1) * (n + 1); code++, cases++) {
      int first = n;
      for (int w = 0, c = code; w < kWarps; w++, c /= n + 1) {
        at[w] = c % (n + 1);
        if (at[w] < first) first = at[w];
      }
      Barrier barrier;
      std::vector<int> met(kWarps), taken(kWarps), wrong(kWarps);
      std::vector<std::thread> warps;
      for (int w = 0; w < kWarps; w++)
        warps.emplace_back([&, w] {
          ql::steps_together(
              n, [&](auto slot, int i, bool go) { wrong[w] += slot != i % 2 || i != met[w]; met[w]++; return barrier.meet(go); },
              [&](auto slot, int i) { wrong[w] += slot != i % 2 || i != taken[w]; taken[w]++; return i != at[w]; });
        });
      for (auto &t : warps) t.join();
      // all take the same steps: up to the first one that any gives up at, and meet once more behind it
      const int steps = first < n ? first + 1 : n, meetings = first + 1 < n ? first + 2 : n;
      for (int w = 0; w < kWarps; w++)
        if (barrier.stuck || wrong[w] || taken[w] != steps || met[w] != meetings) {
          printf("n %d, gives up at %d %d %d %d: warp %d took %d steps, met %d times%s\n", n, at[0], at[1], at[2], at[3], w, taken[w], met[w], barrier.stuck ? ", stuck" : "");
          return 1;
        }
    }
  }
  printf("%d cases\n", cases);
  return 0;
}
"""


def test_every_warp_leaves_when_one_gives_up(tmp_path):
    source, program = tmp_path / "together.cc", tmp_path / "together"
    source.write_text(PROGRAM)
    subprocess.run(["g++", "-std=c++17", "-O1", "-pthread", "-Wall", "-Werror", "-I", os.path.join(ROOT, "tensorrt-incubator_b200", "csrc"), "-o", str(program), str(source)], check=True)
    r = subprocess.run([str(program)], capture_output=True, text=True, timeout=120)
    assert r.returncode == 0, r.stdout
    assert r.stdout == f"{sum((n + 1) ** 4 for n in range(6))} cases\n"
