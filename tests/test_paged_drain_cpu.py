"""A warp whose wait ran out waits again for every copy that it still has in flight (no GPU).

The schedule of the paged attention's stage is played through on the host: for each tile
at which the wait for its keys or its values runs out, the copies requested and not
yet arrived must be exactly those that the drain waits for.
"""

import shutil
import subprocess

import pytest

from conftest import native_build_module

PROGRAM = r"""
#include <cstdio>
#include <set>
#include <utility>
#include "rkv_drain.h"

using Copies = std::set<std::pair<int, int>>;  // (barrier, tile)

int main() {
  int checked = 0;
  for (int count = 1; count <= 6; ++count) {
    for (int fail = 0; fail < count; ++fail) {
      for (int which = 0; which < 2; ++which) {  // the keys' wait or the values'
        Copies flying = {{0, 0}, {1, 0}};
        bool out = false;
        for (int j = 0; j < count && !out; ++j) {
          const bool more = j + 1 < count;
          Copies waited;
          // a barrier's phase of that parity: the copy on it that is in flight
          auto wait = [&](int barrier, int parity) {
            for (const auto& copy : flying) {
              if (copy.first == barrier && (copy.second & 1) == parity) waited.insert(copy);
            }
          };
          if (j == fail && which == 0) {
            rkv::drain_keys_and_values(j, wait);
            out = true;
          } else {
            flying.erase({0, j});
            if (more) flying.insert({0, j + 1});
            if (j == fail) {
              rkv::drain_values(j, more, wait);
              out = true;
            } else {
              flying.erase({1, j});
              if (more) flying.insert({1, j + 1});
            }
          }
          if (out) {
            ++checked;
            if (waited != flying) {
              std::printf("tile %d of %d, barrier %d\n", j, count, which);
              return 1;
            }
          }
        }
      }
    }
  }
  return checked == 42 ? 0 : 2;
}
"""


@pytest.mark.skipif(shutil.which("g++") is None, reason="needs a host compiler")
def test_every_copy_in_flight_is_waited_for(tmp_path):
    source, program = tmp_path / "drain.cpp", tmp_path / "drain"
    source.write_text(PROGRAM)
    csrc = native_build_module().CSRC
    subprocess.run(["g++", "-std=c++17", f"-I{csrc}", str(source), "-o", str(program)], check=True)
    done = subprocess.run([str(program)], capture_output=True, text=True)
    assert done.returncode == 0, done.stdout


def test_the_kernel_drains_by_that_schedule():
    """Both waits of the kernel's loop end in the drain when they run out."""
    kernel = (native_build_module().CSRC / "rkv_paged.cu").read_text()
    for wait, drain in (("!warp_wait(&bars[warp][0], j & 1)", "drain_keys_and_values(j,"),
                        ("!warp_wait(&bars[warp][1], j & 1)", "drain_values(j, more,")):
        at = kernel.index(wait)
        assert drain in kernel[at:kernel.index("aborted = true", at)]


def test_rows_left_short_by_a_timeout_are_nan():
    """Where a row's or a part's sum is taken, an aborted warp's is NaN before any use of it."""
    kernel = (native_build_module().CSRC / "rkv_paged.cu").read_text()
    after = kernel[kernel.index("reduce_l<NT>(l);"):]
    poison = after.index("l[nt][0] = l[nt][1] = NAN")
    assert "aborted" in after[:poison]
    assert poison < after.index("1.f / l[nt][c]") and poison < after.index("seg_l[i][g] = l[nt][c]")
