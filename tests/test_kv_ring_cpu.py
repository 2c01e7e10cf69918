"""The bookkeeping by which the quantised cache's kernels wait for their own
copies before they leave, against a model of the barriers, without a GPU."""
import os
import shutil
import subprocess

import pytest

from conftest import ROOT

CUDA = "/usr/local/cuda/include"

MODEL = r"""
#include <stdio.h>
#include "%s"
// a barrier: phases that have ended; a wait for a parity returns at once when
// the phase that runs has the other one
struct Barrier { int ended; bool passes(unsigned parity) const { return (unsigned)(ended & 1) != parity; } };
int main() {
  for (int stages = 1; stages <= 5; stages++)
    for (int issued = 0; issued < 40; issued++)
      for (int landed = kv_ring_first(issued, stages); landed <= issued; landed++) {
        // copies land in order here: buffer s has seen those of its copies that are before `landed`
        Barrier b[5];
        for (int s = 0; s < stages; s++) b[s].ended = landed > s ? (landed - s - 1) / stages + 1 : 0;
        for (int i = kv_ring_first(issued, stages); i < issued; i++)
          if (b[i %% stages].passes(kv_ring_parity(i, stages)) != (i < landed)) {
            printf("stages %%d issued %%d landed %%d copy %%d\n", stages, issued, landed, i);
            return 1;
          }
        for (int i = 0; i < kv_ring_first(issued, stages); i++)   // the others have landed: their buffers were filled again
          if (i >= landed) return 2;
      }
  return 0;
}
"""


@pytest.mark.skipif(not shutil.which("g++") or not os.path.exists(CUDA), reason="needs a C++ compiler and CUDA's headers")
def test_a_wait_for_a_copy_passes_exactly_when_it_has_landed(tmp_path):
    src = tmp_path / "m.cpp"
    src.write_text(MODEL % os.path.join(ROOT, "chonklm_b200", "csrc", "ck_kv.h"))
    exe = str(tmp_path / "m")
    subprocess.check_call(["g++", "-std=c++17", "-I", CUDA, str(src), "-o", exe])
    done = subprocess.run([exe], capture_output=True, text=True)
    assert done.returncode == 0, done.stdout
