"""Kernel attributes are set on every GPU, not once for the process."""
import os
import re
import subprocess

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "kraken-infer_b200", "csrc")

PROGRAM = r"""
#include "per_device.hpp"
#include <cstdio>
int main() {
  static kib::PerDevice once;
  int set[3] = {0, 0, 0};
  bool works = true;
  auto call = [&](int device) { return once.once(device, [&] { ++set[device < 2 ? device : 2]; return works; }); };
  for (int i = 0; i < 3; ++i)
    if (!call(0)) return 1;
  works = false;
  if (call(1)) return 2;  // an attempt that failed is made again
  works = true;
  for (int i = 0; i < 3; ++i)
    if (!call(1) || !call(0) || !call(200)) return 3;
  std::printf("%d %d %d", set[0], set[1], set[2]);
}
"""


def test_once_for_every_device(tmp_path):
    src, exe = tmp_path / "t.cpp", tmp_path / "t"
    src.write_text(PROGRAM)
    subprocess.check_call(["g++", "-std=c++17", "-I", CSRC, str(src), "-o", str(exe)])
    assert subprocess.check_output([str(exe)], text=True) == "1 2 3"


@pytest.mark.parametrize("source", ["kvq8.cu", "sample.cu"])
def test_the_paged_cache_and_sampling_set_their_attributes_per_device(source):
    text = open(os.path.join(CSRC, source)).read()
    assert "cudaFuncSetAttribute" in text
    assert not re.search(r"static bool", text)
