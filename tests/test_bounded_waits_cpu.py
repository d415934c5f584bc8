"""CPU: the bounded waits of converged warps in the kernels for several requests.

Where a whole warp waits and then issues instructions that need all of its lanes (elect.sync, votes,
tcgen05 loads, barriers), its lanes must leave an expired wait with one answer: otherwise some go on to
an instruction that waits for lanes which have left, without a bound. The wait's code is compiled here
for the host, with 32 threads as lanes whose clocks and polls differ, and the kernels are read for waits
that each lane ends alone and for barriers between warps that may leave their loops one by one."""
import os
import re
import subprocess

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "stablediffusion-cpp_b200", "csrc")


def source(name):
    with open(os.path.join(CSRC, name)) as f:
        return f.read()


def function(text, head):
    """The definition that starts with `head`, to its closing brace."""
    at = text.index(head)
    depth = 0
    for i in range(text.index("{", at), len(text)):
        depth += {"{": 1, "}": -1}.get(text[i], 0)
        if depth == 0:
            return text[at:i + 1]
    raise ValueError(head)


HARNESS = r"""
#include <sched.h>
#include <stdint.h>
#include <stdio.h>
#include <stdlib.h>
#include <atomic>
#include <thread>
#include <vector>
#define __device__
#define __forceinline__ inline
constexpr uint64_t kWaitLimitNs = 1000000;
constexpr int kLanes = 32;
struct { int x; } threadIdx = {5 * 32 + 7};  // of warp 5
static std::atomic<int> word;
static std::atomic<uint64_t> polls;
static std::atomic<bool> over;  // the barrier's phase is complete, and stays so
static thread_local int lane;
static thread_local uint64_t looks;
struct Plan {
  uint64_t over_at;   // the poll of all lanes' that ends the phase
  bool after_late;    // the first poll of the upper half after a lane was late ends it
  uint64_t late[kLanes];  // the look at the clock from which a lane is past the limit
};
static Plan plan;
static uint64_t globaltimer_ns() { return looks++ >= plan.late[lane] ? 10 * kWaitLimitNs : 0; }
static bool mbar_try_wait(uint64_t*, uint32_t) {
  if (polls++ % 7 == 0) sched_yield();
  if (plan.after_late && lane >= 16) {
    while (!word.load()) sched_yield();
    over = true;
  }
  if (polls >= plan.over_at) over = true;
  return over;
}
static void atomicOr(int*, int v) { word.fetch_or(v); }
static int atomicAdd(int* p, int v) { return __atomic_fetch_add(p, v, __ATOMIC_SEQ_CST); }
static int atomicCAS(int* p, int want, int v) {
  __atomic_compare_exchange_n(p, &want, v, false, __ATOMIC_SEQ_CST, __ATOMIC_SEQ_CST);
  return want;
}
@CODE@
int main() {
  srand(7);
  int disagreements = 0, unreported = 0, wrong = 0;
  for (int trial = 0; trial < 400; ++trial) {
    const uint64_t never = 1ull << 60;
    int abort[1 + 12] = {}, err = 0;
    word = 0;
    polls = 0;
    over = false;
    plan.over_at = never;
    plan.after_late = trial == 0;
    for (int i = 0; i < kLanes; ++i) plan.late[i] = trial == 0 ? (i < 16 ? 1 : 50) : trial == 1 ? never : 1;
    if (trial == 1) plan.over_at = 0;                  // complete at once
    if (trial > 2) {                                   // trial 2: nobody ever sees the end
      plan.over_at = 1500 + rand() % 3000;             // 64 polls of 32 lanes are 2048
      for (int i = 0; i < kLanes; ++i) plan.late[i] = 1 + rand() % 3;
    }
    std::vector<std::thread> warp;
    std::vector<int> answer(kLanes);
    for (int i = 0; i < kLanes; ++i)
      warp.emplace_back([&, i] {
        lane = i;
        looks = 0;
        uint64_t bar = 0;
        answer[i] = @CALL@(&bar, 0u, abort, &err, 4);
      });
    for (auto& t : warp) t.join();
    bool same = true;
    for (int a : answer) same = same && a == answer[0];
    disagreements += !same;
    if (trial == 1) wrong += !answer[0] || abort[0];
    if (trial == 2) wrong += answer[0];
    if (same && !answer[0]) unreported += !(abort[0] == 1 && (word.load() & 4));
  }
  printf("%d %d %d\n", disagreements, unreported, wrong);
}
"""


def run(tmp_path, code, call):
    src, exe = tmp_path / "w.cpp", tmp_path / "w"
    src.write_text(HARNESS.replace("@CODE@", code).replace("@CALL@", call))
    subprocess.run(["g++", "-O1", "-std=c++17", "-pthread", "-o", str(exe), str(src)], check=True, capture_output=True)
    out = subprocess.run([str(exe)], check=True, capture_output=True, text=True, timeout=120).stdout
    return [int(x) for x in out.split()]


def test_lanes_of_a_warp_leave_a_wait_with_one_answer(tmp_path):
    text = source("ptx.cuh")
    code = "\n".join(("" if f == "mbar_wait_warp" else "template <class Done>\n")
                     + function(text, f"__device__ __forceinline__ bool {f}(") for f in ("give_up_warp", "wait_warp", "mbar_wait_warp"))
    disagreements, unreported, wrong = run(tmp_path, code, "mbar_wait_warp")
    assert disagreements == 0 and unreported == 0 and wrong == 0


def test_the_harness_sees_lanes_that_decide_alone(tmp_path):
    """The wait of a single thread, run by 32 of them, is told apart."""
    disagreements, _, _ = run(tmp_path, function(source("ptx.cuh"), "__device__ __forceinline__ bool mbar_wait("), "mbar_wait")
    assert disagreements > 0


@pytest.mark.parametrize("name", ["lora.cu", "attention_ragged_tc.cuh"])
def test_whole_warps_wait_together(name):
    """Every bounded wait in these kernels is a whole warp's."""
    text = source(name)
    assert not re.findall(r"\bmbar_wait\(", text)
    assert re.findall(r"\bmbar_wait_warp\(", text)


def test_the_counter_of_h_is_waited_for_together():
    assert "wait_warp(" in function(source("lora.cu"), "__device__ __forceinline__ bool wait_count(")


def test_no_barrier_between_warps_that_may_leave_their_loop():
    """Warps of the adapter GEMM leave their loops by themselves when a wait expires; until the end of the
    kernel, where all meet, none may wait for another at a named barrier."""
    body = function(source("lora.cu"), "k_lora_gemm(const __grid_constant__ CUtensorMap tmX")
    assert "bar.sync" not in body and "barrier.sync" not in body
    assert body.count("__syncthreads()") == 2  # set-up and end
