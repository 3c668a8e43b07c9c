"""The library's cache of what it asks the device (known.h): an answer is kept,
a failed query is reported and asked again, and no exception leaves it.  Compiled and run on the host, with
a query that fails where the device's would."""
import os
import subprocess

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

PROGRAM = r"""
#include <cstdio>
#include <cstdlib>
#include <new>
#include <utility>
#include "known.h"

static bool memory = true;
void* operator new(std::size_t n) {
  if (!memory) throw std::bad_alloc();
  return std::malloc(n);
}
void operator delete(void* p) noexcept { std::free(p); }
void operator delete(void* p, std::size_t) noexcept { std::free(p); }

enum Error { kNone = 0, kBusy = 7 };

int main() {
  det::Known<std::pair<int, int>, int> known;
  int asked = 0, value = -1;
  auto answer = [&](int* v) { ++asked; *v = 42; return kNone; };
  auto fails = [&](int* v) { ++asked; *v = 1; return kBusy; };
  auto never = [&](int* v) { ++asked; *v = 99; return kBusy; };
  if (known.get({1, 2}, &value, fails) != kBusy || value != -1 || asked != 1) return 1;
  if (known.get({1, 2}, &value, fails) != kBusy || value != -1 || asked != 2) return 2;
  if (known.get({1, 2}, &value, answer) != kNone || value != 42 || asked != 3) return 3;
  value = 0;
  if (known.get({1, 2}, &value, never) != kNone || value != 42 || asked != 3) return 4;
  if (known.get({2, 1}, &value, fails) != kBusy || value != 42 || asked != 4) return 5;
  // no memory to keep it: handed out all the same, and asked again
  memory = false;
  value = 0;
  for (int i = 0; i < 2; i++)
    if (known.get({3, 3}, &value, answer) != kNone || value != 42 || asked != 5 + i) return 6;
  std::puts("kept");
  return 0;
}
"""


def test_only_answers_are_kept(tmp_path):
    src, exe = tmp_path / "known.cpp", tmp_path / "known"
    src.write_text(PROGRAM)
    subprocess.run(["g++", "-std=c++17", "-Wall", "-Werror", "-I", os.path.join(ROOT, "detllm_b200", "csrc"), str(src),
                    "-o", str(exe), "-lpthread"], check=True)
    r = subprocess.run([str(exe)], capture_output=True, text=True, timeout=60)
    assert r.returncode == 0 and r.stdout == "kept\n"


def test_occupancy_answers_go_through_it():
    """No answer about the device is kept by hand in the scoring calls, and none
    of its queries' errors is turned into a number."""
    text = open(os.path.join(ROOT, "detllm_b200", "csrc", "scoring.cu"), encoding="utf-8").read()
    assert "std::map" not in text and "std::mutex" not in text
    for query in ("cudaOccupancyMaxActiveBlocksPerMultiprocessor(", "cudaOccupancyMaxActiveClusters("):
        assert text.count(query) == 1
        line = next(x for x in text.split("\n") if query in x)
        assert "cudaError_t e = " in line, line
