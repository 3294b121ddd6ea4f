"""How many clusters run at once is asked of each device, once, and again where the answer could not be had: the launch header against a runtime
of two devices that counts its calls."""
import os
import subprocess
from pathlib import Path

import pytest

CSRC = Path(__file__).resolve().parent.parent / "flagdnn_b200" / "csrc"
CUDA = Path(os.environ.get("CUDA_HOME", "/usr/local/cuda"))

PROGRAM = r"""
#include <stdio.h>
#include "sequence_launch.h"
static int device = 0, asked = 0, fails = 0;
extern "C" cudaError_t cudaGetDevice(int* d) { *d = device; return cudaSuccess; }
extern "C" cudaError_t cudaGetLastError() { return cudaSuccess; }
extern "C" cudaError_t cudaOccupancyMaxActiveClusters(int* n, const void*, const cudaLaunchConfig_t* c) {
  ++asked;
  if (fails) return cudaErrorUnknown;
  *n = device == 1 ? 0 : 16 / int(c->attrs[0].val.clusterDim.x);
  return cudaSuccess;
}
void kernel() {}
static fdnn::ClusterCounts two, eight;
static int ask(int d, int cluster, fdnn::ClusterCounts& known) { device = d; return fdnn::clusters_at_once(&kernel, 128, 1000, cluster, known); }
int main() {
  fails = 1;
  int a = ask(0, 2, two);
  fails = 0;
  int b = ask(0, 2, two), c = ask(0, 2, two), d = ask(1, 2, two), e = ask(1, 2, two), f = ask(0, 8, eight), g = ask(200, 8, eight), h = ask(200, 8, eight);
  printf("%d %d %d %d %d %d %d %d, asked %d\n", a, b, c, d, e, f, g, h, asked);
}
"""


def test_each_device_answers_for_itself(tmp_path):
    if not (CUDA / "include" / "cuda_runtime.h").exists():
        pytest.skip("no CUDA headers")
    source, program = tmp_path / "counts.cpp", tmp_path / "counts"
    source.write_text(PROGRAM)
    subprocess.run(["g++", "-std=c++17", "-O1", f"-I{CSRC}", f"-I{CUDA / 'include'}", str(source), "-o", str(program)], check=True)
    out = subprocess.run([str(program)], check=True, capture_output=True, text=True).stdout
    assert out.strip() == "0 8 8 0 0 2 2 2, asked 6"
