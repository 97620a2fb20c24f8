"""Attributes and occupancies of kernels are per device (csrc/wp_once.h): on the
CPU against a cudaGetDevice of the test's own, and, where there are two GPUs,
every operator with a kernel above 48 KB of shared memory on both of them in
one process."""

import shutil
import subprocess

import pytest
import torch

from adapterslotsplusplus_b200.build import CSRC

MAIN = r"""
#include <cassert>
#include <initializer_list>
#include "wp_once.h"

static int device = 0, asked = 0;
static cudaError_t status = cudaSuccess;
extern "C" cudaError_t cudaGetDevice(int* d) { *d = device; return status; }

static int per_sm() {
  static wp::PerDevice known;
  return known.get([] { ++asked; return device + 1; });
}
static bool failing(bool ok) {
  static wp::PerDevice ready;
  return ready.get([&] { ++asked; return ok; });
}

int main() {
  for (int round = 0; round < 3; ++round)
    for (int dev : {0, 3, 7, 63}) {
      device = dev;
      assert(per_sm() == dev + 1);
    }
  assert(asked == 4);
  device = 64;  // more devices than places: asked each time
  assert(per_sm() == 65 && per_sm() == 65 && asked == 6);
  device = 1;
  assert(!failing(false) && !failing(false) && failing(true) && failing(false) && asked == 9);  // a failure is not kept
  status = cudaErrorInvalidDevice;
  assert(per_sm() == 0);
  return 0;
}
"""


def test_each_device_is_asked_once(tmp_path):
    cxx, nvcc = shutil.which("g++"), shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc"
    if cxx is None:
        pytest.skip("no C++ compiler")
    include = subprocess.run(["realpath", nvcc], capture_output=True, text=True, check=True).stdout.rsplit("/bin/", 1)[0] + "/include"
    (tmp_path / "main.cpp").write_text(MAIN)
    subprocess.run([cxx, "-std=c++17", "-I", str(CSRC), "-I", include, str(tmp_path / "main.cpp"), "-o", str(tmp_path / "main")],
                   check=True)
    subprocess.run([str(tmp_path / "main")], check=True)


@pytest.mark.gpu
def test_operators_on_two_gpus_of_one_process():
    if torch.cuda.device_count() < 2:
        pytest.skip("needs 2 GPUs")
    from adapterslotsplusplus_b200 import KvCache4, WarpPipeConfig, WarpPipeEngine

    got = []
    for dev in (0, 1):
        with torch.cuda.device(dev):
            eng = WarpPipeEngine(WarpPipeConfig(max_tokens=1024), device=dev)
            g = torch.Generator().manual_seed(0)
            q, k, v = (torch.randn(300, h, 128, generator=g).to(f"cuda:{dev}", torch.bfloat16) for h in (8, 2, 2))
            i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=f"cuda:{dev}")
            out = [eng.prompt_attention(q, k, v, i32([0, 300]), max_q=m) for m in (1, 300)]
            cache = KvCache4(eng, 8, 2, 128)
            table, lens = i32([[3, 1, 0, 5, 2]]), i32([300])
            cache.append(k, v, table, lens, i32([0, 300]))
            out += [cache.attention(q[:n], table, lens, i32([0, n]), n) for n in (1, 5)]
            got.append([x.cpu() for x in out])
            assert eng.device_error(clear=True) == 0
    assert all(torch.equal(a, b) for a, b in zip(*got))
