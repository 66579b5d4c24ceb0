"""The waits of a CTA that stops early (csrc/drain.cuh), compiled for the host against a simulated clock, copies and
abort flag."""

from __future__ import annotations

import re
import shutil
import subprocess
from pathlib import Path

import pytest

CSRC = Path(__file__).resolve().parent.parent / "cute-moe-train_b200" / "csrc"

PROGRAM = r"""
#include <cstdio>
#include "drain.cuh"
using namespace mgf::drain;

static uint64_t clock_ns = 0;
static int polls = 0;
static uint64_t now() { return clock_ns; }

int main() {
  // a copy that lands after 5000 polls of 10 us (50 ms), far behind the polls at which a running wait looks at its flag
  auto done = [] { clock_ns += 10000; return ++polls >= 5000; };
  const bool ended = wait_until(done, now, clock_ns + kLimitNs);
  std::printf("%d %d\n", ended, polls);
  // one that never lands: given up at the deadline, not before and not long after
  clock_ns = 7; polls = 0;
  const bool got = wait_until([] { clock_ns += 10000; ++polls; return false; }, now, clock_ns + kLimitNs);
  std::printf("%d %d\n", got, polls);
  // stages: the parity of the last phase of each one that was armed, all under one deadline
  Copies c;
  c.arm(0, 0); c.arm(2, 0); c.arm(2, 1); c.arm(7, 1); c.arm(7, 0);
  unsigned seen = 0, parities = 0;
  clock_ns = 0;
  auto landed = [&](uint32_t s, uint32_t parity) { seen |= 1u << s; parities |= parity << s; return true; };
  const bool all = wait_copies(c, landed, now, kLimitNs);
  std::printf("%d %u %u\n", all, seen, parities);
  clock_ns = 0; polls = 0;
  auto never = [](uint32_t s, uint32_t) { clock_ns += 10000; ++polls; return s == 7; };
  const bool some = wait_copies(c, never, now, kLimitNs);
  std::printf("%d %d\n", some, polls);
  std::printf("%d\n", wait_copies(Copies(), never, now, 0));
}
"""


@pytest.mark.skipif(shutil.which("g++") is None, reason="needs a host compiler")
def test_drain_waits_end_with_what_they_wait_for_or_at_their_limit(tmp_path):
    src = tmp_path / "drain.cpp"
    src.write_text(PROGRAM)
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-Werror", f"-I{CSRC}", str(src), "-o", str(tmp_path / "drain")], check=True)
    out = subprocess.run([str(tmp_path / "drain")], capture_output=True, text=True, check=True, timeout=60).stdout.split("\n")
    assert out[0] == "1 5000"
    assert out[1] == "0 10001"          # 100 ms of polls of 10 us, and the one past them
    assert out[2] == f"1 {1 | 4 | 128} 4"
    assert out[3] == "0 10003"          # one deadline for all: the second wait ends at its first poll, stage 7 has landed
    assert out[4] == "1"


def _tail(source: str, kernel: str) -> str:
    """The kernel's end: from the barrier behind its roles to the release of its tensor memory."""
    body = source[source.index(kernel):]
    dealloc = body.index("tmem_dealloc")
    return body[body.rindex("__syncthreads();\n  if (*abort_flag)", 0, dealloc):dealloc]


@pytest.mark.parametrize("name,kernel", [("fp8_block_gemm.cu", "gemm_kernel(const"), ("fp8_block_gemm.cu", "mx_kernel(const")])
def test_kernels_drain_behind_their_roles_and_before_they_leave(name, kernel):
    source = (CSRC / name).read_text()
    tail = _tail(source, kernel)
    order = [tail.index(s) for s in ("drain::copies<CG>", "drain::products<CG>", "cluster_sync")]
    assert order == sorted(order)
    assert "CG == 1" not in tail  # a pair drains too
    # no wait that looks at the abort flag has a limit of its own any more
    assert not re.search(r"wait_bounded\([^;]*kDrain", source)


def test_the_bf16_kernel_drains_too():
    source = (CSRC / "moe_gemm_sm100.cu").read_text()
    tail = _tail(source, "grouped_gemm_kernel(const")
    order = [tail.index(s) for s in ("drain::copies<CG>", "drain::products<CG>", "cluster_sync")]
    assert order == sorted(order) and "CG == 1" not in tail
    assert not re.search(r"wait_bounded\([^;]*kDrain", source)
