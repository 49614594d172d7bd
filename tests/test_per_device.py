"""CPU: a kernel's setup runs once on each device, not once in a process."""
from __future__ import annotations

import re
import subprocess
from pathlib import Path

CSRC = Path(__file__).resolve().parents[1] / "minixmax_h3_b200" / "csrc"

PROGRAM = """
#include "per_device.hpp"
#include <cstdio>
#include <thread>
#include <vector>
int main() {
  h3b::OncePerDevice once;
  int runs[70] = {0};
  auto on = [&](int dev, int rc) { return once.run(dev, [&] { ++runs[dev]; return rc; }); };
  if (on(0, 0) != 0 || on(0, 0) != 0 || on(1, 0) != 0 || on(63, 0) != 0 || on(1, 0) != 0 || on(63, 0) != 0) return 1;
  if (runs[0] != 1 || runs[1] != 1 || runs[63] != 1) return 2;
  if (on(5, 4) != 4 || on(5, 4) != 4 || on(5, 0) != 0 || on(5, 4) != 0 || runs[5] != 3) return 3;  // a failure is not kept
  if (on(64, 0) != 0 || on(64, 0) != 0 || runs[64] != 2) return 4;
  h3b::OncePerDevice other;
  std::atomic<int> n{0};
  std::vector<std::thread> ts;
  for (int i = 0; i < 8; ++i) ts.emplace_back([&, i] { other.run(i % 4, [&] { ++n; return 0; }); });
  for (auto& t : ts) t.join();
  if (n < 4 || n > 8) return 5;
  std::puts("ok");
  return 0;
}
"""


def test_setup_runs_once_on_each_device(tmp_path):
    (tmp_path / "t.cpp").write_text(PROGRAM)
    subprocess.run(["g++", "-std=c++17", "-O1", "-pthread", "-I", str(CSRC), "-o", str(tmp_path / "t"), str(tmp_path / "t.cpp")],
                   check=True)
    assert subprocess.run([str(tmp_path / "t")], check=True, capture_output=True, text=True).stdout == "ok\n"


def test_kernel_attributes_are_set_on_each_device():
    """Kernels take their shared memory through allow_smem, always in a OncePerDevice."""
    found = 0
    for path in sorted(CSRC.glob("*.cu")):
        text = path.read_text()
        assert "cudaFuncSetAttribute(" not in text, path.name
        for m in re.finditer(r"allow_smem\(", text):
            assert "OncePerDevice" in text[max(0, m.start() - 800):m.start()], path.name
            found += 1
    assert found == len(re.findall("<<<.*smem", "".join(p.read_text() for p in CSRC.glob("*.cu")), re.I))
