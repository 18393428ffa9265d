"""The shared-memory opt-in of the kernels (csrc/smem_opt_in.h), compiled for the host with a stand-in for the CUDA call."""
import os
import shutil
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

PROGRAM = r"""
#include <cstdio>
#include <thread>
#include <vector>
#include "smem_opt_in.h"

#define EXPECT(c) if (!(c)) { std::printf("line %d: %s\n", __LINE__, #c); return 1; }

int main() {
  pan::SmemOptIn opted;
  int calls = 0;
  auto ok = [&] { ++calls; return true; };
  EXPECT(opted.once(0, ok) && calls == 1);
  EXPECT(opted.once(0, ok) && calls == 1);                   // set once for a device
  EXPECT(opted.once(1, ok) && calls == 2);                   // and again for another one
  EXPECT(opted.once(0, ok) && opted.once(1, ok) && calls == 2);
  EXPECT(!opted.once(2, [] { return false; }));              // a refusal is not remembered
  EXPECT(opted.once(2, ok) && calls == 3);
  EXPECT(opted.once(63, ok) && opted.once(63, ok) && calls == 4);
  EXPECT(opted.once(64, ok) && opted.once(64, ok) && calls == 6);  // past the flags: set every time
  EXPECT(opted.once(-1, ok) && calls == 7);
  for (int round = 0; round < 200; ++round) {                // nobody passes before the value is set
    pan::SmemOptIn shared;
    std::atomic<int> value{0}, wrong{0};
    std::vector<std::thread> threads;
    for (int t = 0; t < 8; ++t)
      threads.emplace_back([&] {
        if (!shared.once(3, [&] { value.store(225280); return true; }) || value.load() != 225280) ++wrong;
      });
    for (auto& t : threads) t.join();
    EXPECT(wrong == 0);
  }
  return 0;
}
"""


@pytest.mark.skipif(shutil.which("g++") is None, reason="needs a host compiler")
def test_opt_in_is_made_once_for_every_device(tmp_path):
    source, program = tmp_path / "opt_in.cpp", tmp_path / "opt_in"
    source.write_text(PROGRAM)
    subprocess.run(["g++", "-std=c++17", "-O1", "-pthread", "-I", os.path.join(ROOT, "csrc"), str(source), "-o", str(program)],
                   check=True, timeout=120)
    done = subprocess.run([str(program)], capture_output=True, text=True, timeout=60)
    assert done.returncode == 0, done.stdout


def test_launches_use_it():
    """No launch of these files remembers its opt-in in a plain static, which knows neither devices nor threads."""
    for name in ("norm_ops.cu", "wgrad_sm100.cu", "gemm_sm100.cu"):
        with open(os.path.join(ROOT, "csrc", name)) as f:
            text = f.read()
        assert "cudaFuncSetAttribute" not in text and "SmemOptIn opted" in text, name
