"""The paged decode kernel's bounded wait on the CPU: its own source over 32 threads for a warp's lanes,
with a scripted barrier and clock.  The lanes go on to warp-wide instructions together, so they must all
get one verdict, whatever each of them saw at the limit."""

import os
import re
import subprocess

import pytest

from kvboost_b200 import _build

STUBS = r"""
#include <atomic>
#include <barrier>
#include <cstdint>
#include <cstdio>
#include <cstdlib>
#include <thread>
#include <vector>
#include "kvb_attn.h"
#define __device__
#define __forceinline__ inline
static std::barrier<> meet(32);
static std::atomic<int> ayes[3];
static thread_local int lane, votes, tries;
static thread_local uint64_t clock_ns;
static int lands[32];            // a lane's barrier has landed from this try on
static uint64_t pace[32];        // a lane's clock advances by this at each look
static int count(bool x) {       // lanes that say yes
  std::atomic<int>& n = ayes[votes % 3];
  if (x) ++n;
  meet.arrive_and_wait();
  const int y = n;
  ayes[(votes + 2) % 3] = 0;     // the vote before this one has been read by all
  ++votes;
  meet.arrive_and_wait();
  return y;
}
static bool __all_sync(uint32_t, bool x) { return count(x) == 32; }
static bool __any_sync(uint32_t, bool x) { return count(x) > 0; }
static uint64_t globaltimer_ns() { return clock_ns += pace[lane]; }
static bool mbar_try_wait(uint32_t, uint32_t) { return ++tries > lands[lane]; }
static void atomicOr(int32_t* p, int v) { __atomic_fetch_or(p, v, __ATOMIC_RELAXED); }
"""

MAIN = r"""
int main(int, char** a) {
  const int script = atoi(a[1]);
  for (int i = 0; i < 32; ++i) {
    lands[i] = script == 0 ? i % 3 : script == 1 ? (i == 7 ? 1 << 30 : 2) : script == 2 ? 40 : i;
    pace[i] = script == 2 ? 1000000 + (uint64_t)i * 10000000 : script == 3 ? 100000000ull * (1 + i % 2) : 300000000;
  }
  int32_t status = 0;
  bool got[32];
  std::vector<std::thread> warp;
  for (int i = 0; i < 32; ++i)
    warp.emplace_back([&, i] { lane = i; got[i] = wait_full(0, 0, &status); });
  for (auto& t : warp) t.join();
  int yes = 0;
  for (bool g : got) yes += g;
  std::printf("%d %d\n", yes, status);
}
"""


@pytest.fixture(scope="module")
def program(tmp_path_factory):
    src = open(os.path.join(_build.CSRC, "kvb_paged_decode_sm100.cu")).read()
    limit = re.search(r"^constexpr uint64_t kWaitNs = .*?;", src, re.M).group()
    body = re.search(r"^__device__ __forceinline__ bool wait_full\(.*?^}", src, re.M | re.S).group()
    tmp = tmp_path_factory.mktemp("waits")
    (tmp / "w.cc").write_text("\n".join([STUBS, limit, body, MAIN]))
    subprocess.run(["g++", "-std=c++20", "-O1", "-pthread", "-I", _build.INCLUDE, "-o", str(tmp / "w"),
                    str(tmp / "w.cc")], check=True)
    return str(tmp / "w")


LOAD_WAIT = 1


@pytest.mark.parametrize("script,yes", [(0, 32),    # landed within the first tries
                                        (1, 0),     # one lane's never lands: no lane goes on
                                        (2, None),  # clocks that pass the limit at different tries
                                        (3, None)]) # lanes whose loads land one after another at the limit
def test_the_lanes_agree(program, script, yes):
    out = subprocess.run([program, str(script)], capture_output=True, text=True, check=True, timeout=60).stdout
    n, status = map(int, out.split())
    assert n in ((0, 32) if yes is None else (yes,))
    assert status == (0 if n == 32 else LOAD_WAIT)
