"""The notes by which runs of attention tiles tell the merge of a shared stream
(csrc/run_tail.h), on the CPU: what the merge takes addresses from is in range even
where a run failed before it wrote its note and the workspace holds anything."""

import os
import re
import shutil
import subprocess

import pytest

from helpers import PKG_NAME

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), PKG_NAME, "csrc")

MAIN = r"""
#include <cstdio>
#include <cstdint>
#include <cstring>
#include "run_tail.h"
using i4kv::RunTail;

static uint64_t state = 88172645463325252ull;
static uint32_t next() { state ^= state << 13; state ^= state >> 7; state ^= state << 17; return (uint32_t)(state >> 16); }

int main() {
  const int runs = 148, total = 96, kv = 8, group = 4;
  auto ok = [&](RunTail n, int run) { return i4kv::tail_in_range(n, run, runs, total, kv, group); };
  // notes that runs leave
  const RunTail good[] = {{128, 0, 0, 0, 0, 1, {}}, {384, 0, 7, 256, 5, 147, {}}, {4, 95, 3, 0, 292, 147, {}},
                          {128, 64, 2, 64, 21, 11, {}}};
  const int run_of[] = {0, 2, 146, 10};
  for (int i = 0; i < 4; ++i)
    if (!ok(good[i], run_of[i])) return printf("refused a note (%d)\n", i), 1;
  // one field wrong
  const RunTail n = good[3];
  auto bad = [&](int RunTail::*f, int v) { RunTail m = n; m.*f = v; return !ok(m, 10); };
  const int lows = INT32_MIN, highs = INT32_MAX;
  const bool all = bad(&RunTail::rows, 0) && bad(&RunTail::rows, lows) && bad(&RunTail::rows, highs) && bad(&RunTail::rows, 129) &&
                   bad(&RunTail::row0, -1) && bad(&RunTail::row0, 65) && bad(&RunTail::row0, highs) && bad(&RunTail::row0, lows) &&
                   bad(&RunTail::head, -1) && bad(&RunTail::head, 8) && bad(&RunTail::head, highs) &&
                   bad(&RunTail::first_row, -1) && bad(&RunTail::first_row, 128) && bad(&RunTail::first_row, lows) &&
                   bad(&RunTail::slot, 19) && bad(&RunTail::slot, 22) && bad(&RunTail::slot, -2) &&
                   bad(&RunTail::last, 10) && bad(&RunTail::last, -1) && bad(&RunTail::last, 148) && bad(&RunTail::last, highs);
  if (!all) return printf("a wrong field went through\n"), 1;
  if (ok(RunTail{}, 0)) return printf("the empty note counts\n"), 1;
  // leftover bytes: floats, small integers, anything; what goes through is in range
  long through = 0;
  for (long i = 0; i < 4000000; ++i) {
    RunTail m;
    for (int k = 0; k < 8; ++k) {
      uint32_t w = next();
      if (i % 3 == 0) w %= 300;
      if (i % 3 == 1) w = 0x3f000000u + (w & 0xffffff);
      memcpy((char*)&m + 4 * k, &w, 4);
    }
    const int run = (int)(next() % (runs - 1));
    if (!ok(m, run)) continue;
    ++through;
    const bool in = m.rows >= 1 && m.row0 >= 0 && (long long)m.row0 * group + m.rows <= (long long)total * group &&
                    m.head >= 0 && m.head < kv && m.first_row >= 0 && m.first_row < m.rows && m.slot / 2 == run && m.last < runs;
    if (!in) return printf("out of range\n"), 1;
  }
  printf("notes ok\n");
  return 0;
}
"""


def test_notes_out_of_range_are_not_followed(tmp_path):
    cc = shutil.which("g++") or shutil.which("c++")
    if not cc:
        pytest.skip("no C++ compiler")
    src, exe = tmp_path / "tails.cpp", tmp_path / "tails"
    src.write_text(MAIN)
    res = subprocess.run([cc, "-std=c++17", "-O2", "-Wall", "-Werror", "-fsanitize=undefined", "-fno-sanitize-recover", "-I", CSRC,
                          str(src), "-o", str(exe)], capture_output=True, text=True)
    assert res.returncode == 0, res.stderr
    run = subprocess.run([str(exe)], capture_output=True, text=True, timeout=120)
    assert run.returncode == 0 and "notes ok" in run.stdout, run.stdout + run.stderr


@pytest.mark.parametrize("source", ["multi_query_tc.cu", "multi_query_f32.cu"])
def test_every_run_leaves_an_empty_note_before_it_waits(source):
    """The order in the kernels' text: an unconditional empty note first, then the roles that may
    leave early, then the note of the last tile; and the merge asks before it follows one."""
    text = open(os.path.join(CSRC, source)).read()
    kernel = text[text.index("__global__"):]
    empty = [m.start() for m in re.finditer(r"a\.tails\[cta\] = RunTail\{\}", kernel)]
    assert len(empty) == 1
    line = kernel[kernel.rindex("\n", 0, empty[0]) + 1:empty[0]]
    assert "tiles" not in line  # (of every run, not of the empty ones alone)
    waits = [m.start() for m in re.finditer(r"\b(tc_wait|wait|mbar_wait_bounded)\(", kernel[empty[0]:])]
    before = re.findall(r"\b(tc_wait|mbar_wait_bounded|mbar_try_wait)\(", kernel[:empty[0]])
    assert waits and not before
    assert kernel.index("note_tail(a, cta") > empty[0]
    merge = open(os.path.join(CSRC, "multi_query.cuh")).read()
    merge = merge[merge.index("merge_records_kernel"):]
    assert merge.index("if (!tail_in_range(") < merge.index("record(i)")
