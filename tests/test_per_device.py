"""Kernel attributes are set once for every device (csrc/per_device.h)."""
import os
import shutil
import subprocess

import pytest
import torch

from cascadia_b200 import ops

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

PROGRAM = r"""
#include <cassert>
#include <stdexcept>
#include <thread>
#include <vector>
#include "per_device.h"
int main() {
  // As a launch uses it: the limit of the current device, from a fake of the CUDA runtime.
  static int limit[70];
  static std::atomic<int> calls[70];
  static cb::PerDevice set;
  auto launch = [&](int device, int bytes) {
    set.once(device, [&] { limit[device] = 100; ++calls[device]; });
    if (bytes > limit[device]) throw std::runtime_error("launch refused");
  };
  launch(0, 60);
  launch(0, 100);
  launch(3, 60);   // another device of the same process
  launch(3, 100);
  launch(0, 10);   // a small launch lowers nothing
  launch(0, 100);
  assert(calls[0] == 1 && calls[3] == 1 && calls[1] == 0);
  launch(69, 100);  // past the devices it remembers: set every time
  launch(69, 100);
  assert(calls[69] == 2);
  std::vector<std::thread> t;
  for (int i = 0; i < 8; ++i)
    t.emplace_back([&, i] { for (int k = 0; k < 1000; ++k) launch(5 + k % 3, 1 + (i + k) % 100); });
  for (auto& x : t) x.join();
  // A failure is not remembered.
  static cb::PerDevice other;
  int tries = 0;
  for (int k = 0; k < 2; ++k) {
    try { other.once(1, [&] { ++tries; throw 1; }); } catch (int) {}
  }
  assert(tries == 2);
  return 0;
}
"""


def test_once_for_every_device(tmp_path):
    cxx = shutil.which("g++") or shutil.which("c++")
    if cxx is None:
        pytest.skip("no C++ compiler")
    src, exe = tmp_path / "p.cpp", tmp_path / "p"
    src.write_text("#include <atomic>\n" + PROGRAM)
    subprocess.check_call([cxx, "-std=c++17", "-pthread", "-I", os.path.join(ROOT, "csrc"),
                           str(src), "-o", str(exe)])
    subprocess.check_call([str(exe)], timeout=60)


@pytest.mark.gpu
def test_attention_on_the_second_device_of_a_process():
    if torch.cuda.device_count() < 2:
        pytest.skip("needs two GPUs")
    outs = []
    for dev in ("cuda:0", "cuda:1"):
        g = torch.Generator().manual_seed(0)
        i32 = dict(dtype=torch.int32, device=dev)
        k = torch.randn(1, 8, 2, 16, 128, generator=g).to(torch.bfloat16).to(dev)
        q = torch.randn(40, 1024, generator=g).to(torch.bfloat16).to(dev)
        for nodes in (1, 40):
            with torch.cuda.device(dev):
                o = ops.attn_tree(q[:nodes], k, k, torch.arange(8, **i32).view(1, 8),
                                  torch.tensor([128], **i32), torch.tensor([0, nodes], **i32),
                                  torch.empty_like(q[:nodes]), 0, 0.1, max_nodes=nodes)
            outs.append(o.cpu())
    assert torch.equal(outs[0], outs[2]) and torch.equal(outs[1], outs[3])
