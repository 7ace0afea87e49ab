"""Host state that threads share (csrc/host_state.h), against fakes of what lies
on the device: compiled and run here, without a GPU."""

import ctypes
import shutil
import subprocess
from pathlib import Path

import pytest

CSRC = Path(__file__).resolve().parents[1] / "burn_automata_b200" / "csrc"

SOURCE = r"""
#include <atomic>
#include <chrono>
#include <thread>
#include <vector>
#include "host_state.h"

extern "C" {
void* watermarks_new() { return new npa::Watermarks; }
int watermarks_grown(void* w, int device, uint64_t now) {
  return static_cast<npa::Watermarks*>(w)->grown(device, now);
}
// Eight threads see one growth: how many report it.
int watermarks_race(void* w, int device, uint64_t now) {
  int reports[8] = {};
  std::vector<std::thread> threads;
  for (int i = 0; i < 8; ++i)
    threads.emplace_back([&, i] {
      for (int k = 0; k < 1000; ++k) reports[i] += static_cast<npa::Watermarks*>(w)->grown(device, now);
    });
  for (auto& t : threads) t.join();
  int n = 0;
  for (int r : reports) n += r;
  return n;
}

// Two threads plan one kernel with different amounts, the smaller one slow to
// set its limit; the limit that the kernel is left with, and each plan's answer.
size_t plans_race(size_t slow, size_t fast, int* found) {
  npa::LaunchPlans plans;
  std::atomic<size_t> attribute{0};  // the device's side
  std::atomic<bool> started{false};
  int kernel = 0, ctx = 0;
  auto plan = [&](size_t smem, int ms) {
    npa::LaunchPlan p{0, &ctx, &kernel, 256, smem, 0, 0};
    if (plans.find(&p)) return;
    plans.add(&p, [&](size_t limit, npa::LaunchPlan* q) {
      started = true;
      std::this_thread::sleep_for(std::chrono::milliseconds(ms));
      attribute = limit;
      q->per_sm = int(smem / 1000);
      return 0;
    });
  };
  std::thread a([&] { plan(slow, 100); });
  while (!started) std::this_thread::yield();
  std::thread b([&] { plan(fast, 0); });
  a.join();
  b.join();
  npa::LaunchPlan p{0, &ctx, &kernel, 256, slow, 0, 0}, q{0, &ctx, &kernel, 256, fast, 0, 0};
  npa::LaunchPlan other{0, &ctx, &kernel, 128, fast, 0, 0}, device{1, &ctx, &kernel, 256, fast, 0, 0};
  *found = plans.find(&p) && plans.find(&q) && p.per_sm == int(slow / 1000) &&
           q.per_sm == int(fast / 1000) && !plans.find(&other) && !plans.find(&device);
  return attribute;
}
// A plan that could not be set is not kept.
int plans_failed() {
  npa::LaunchPlans plans;
  int kernel = 0, ctx = 0;
  npa::LaunchPlan p{0, &ctx, &kernel, 256, 1000, 0, 0};
  const int status = plans.add(&p, [](size_t, npa::LaunchPlan*) { return 5; });
  return status == 5 && !plans.find(&p);
}
}
"""


@pytest.fixture(scope="module")
def lib(tmp_path_factory):
    gxx = shutil.which("g++")
    if gxx is None:
        pytest.skip("no C++ compiler")
    folder = tmp_path_factory.mktemp("host_state")
    source, out = folder / "t.cpp", folder / "t.so"
    source.write_text(SOURCE)
    subprocess.run([gxx, "-std=c++17", "-O1", "-pthread", "-shared", "-fPIC", f"-I{CSRC}",
                    str(source), "-o", str(out)], check=True)
    lib = ctypes.CDLL(str(out))
    lib.watermarks_new.restype = ctypes.c_void_p
    lib.watermarks_grown.argtypes = lib.watermarks_race.argtypes = [
        ctypes.c_void_p, ctypes.c_int, ctypes.c_uint64]
    lib.plans_race.restype = ctypes.c_size_t
    lib.plans_race.argtypes = [ctypes.c_size_t, ctypes.c_size_t, ctypes.POINTER(ctypes.c_int)]
    return lib


def test_a_grown_count_is_reported_once_per_device(lib):
    w = lib.watermarks_new()
    assert not lib.watermarks_grown(w, 0, 0)
    assert lib.watermarks_grown(w, 0, 2)
    assert not lib.watermarks_grown(w, 0, 2)
    assert not lib.watermarks_grown(w, 3, 0)
    assert lib.watermarks_grown(w, 3, 1)
    assert lib.watermarks_grown(w, 0, 3)
    assert not lib.watermarks_grown(w, 3, 1)


def test_threads_report_one_growth_once(lib):
    assert lib.watermarks_race(lib.watermarks_new(), 1, 7) == 1


@pytest.mark.parametrize("slow,fast", [(100000, 200000), (200000, 100000), (50000, 50000)])
def test_threads_that_plan_one_kernel_leave_the_largest_limit(lib, slow, fast):
    found = ctypes.c_int(0)
    assert lib.plans_race(slow, fast, ctypes.byref(found)) == max(slow, fast)
    assert found.value == 1


def test_a_plan_that_failed_is_not_kept(lib):
    assert lib.plans_failed() == 1


def test_the_layers_waits_are_reported_by_an_entry_point(npa_lib):
    """The check exists, and npa_bulk_copy_timeouts' comment names it for these
    waits instead of calls that do not look at them."""
    assert hasattr(npa_lib, "npa_dev_check_layer_waits")
    text = (CSRC.parents[1] / "include" / "npa_b200.h").read_text()
    comment = text[:text.index("uint64_t npa_bulk_copy_timeouts")].rsplit("/*", 1)[1]
    assert "npa_dev_check_layer_waits" in comment
