"""Attention over packed sequences at the sizes where its index arithmetic and
its workspace could go wrong: more workgroups than 31 bits hold threads, many
heads on few tokens."""
import ctypes
import subprocess
from pathlib import Path

import pytest

REPO = Path(__file__).resolve().parent.parent


@pytest.fixture(scope="module")
def nat():
    from jax_mlx_amd import native

    native.load()
    return native


def run_cpp(tmp_path, text):
    src, exe = tmp_path / "t.cpp", tmp_path / "t"
    src.write_text(text)
    subprocess.run(["g++", "-std=c++17", "-Wall", "-I", str(REPO / "jax-mlx-plugin_amd/csrc/kernels"), str(src), "-o",
                    str(exe)], check=True)
    r = subprocess.run([str(exe)], capture_output=True, text=True)
    assert r.returncode == 0, r.stdout


def test_cleared_counts_stay_inside(tmp_path):
    """The backward's workgroups clear the counts of its shares, each thread
    the one of its number: none outside them, whatever the grid (2^23
    workgroups of 256 threads and more), and each of them once."""
    run_cpp(tmp_path, r"""
#include "packed_index.h"
#include <cstdio>
#include <vector>
using namespace mfx;
int main() {
  int bad = 0;
  for (int64_t counts : {int64_t(0), int64_t(1), int64_t(255), int64_t(57344), (int64_t(1) << 31) + 5})
    for (uint32_t id : {0u, 1u, 224u, (1u << 23) - 1, 1u << 23, 8388831u, (1u << 24) - 1, 1u << 24, 0xffffffffu})
      for (int tid : {0, 1, 255}) {
        const int64_t i = packed_cleared(id, tid, 256, counts), want = int64_t(id) * 256 + tid;
        bad += want < counts ? i != want : i != -1;
        bad += i < -1 || i >= counts;
      }
  std::vector<int> hits(1000);
  for (uint32_t id = 0; id < 9; ++id)
    for (int tid = 0; tid < 256; ++tid) {
      const int64_t i = packed_cleared(id, tid, 256, 1000);
      if (i >= 0) ++hits[i];
    }
  for (int h : hits) bad += h != 1;
  std::printf("%d\n", bad);
  return bad != 0;
}
""")


MANY = [0] * 131072 + [600] + [0] * 131070 + [400]


@pytest.mark.gpu
def test_more_workgroups_than_threads_fit_31_bits(cuda, nat):
    """262144 sequences of 32 heads, all but two empty: 8388832 workgroups.
    Nothing before or behind the workspace is written, and the gradients are
    those of the two sequences."""
    torch = cuda
    from test_sdpa_packed import check_all, make

    q, k, v, g, off = make(torch, "bf16", MANY, 32, 8, 64)
    lse = torch.zeros(32, 1000, device="cuda")
    out = nat.sdpa_packed(q, k, v, off, lse=lse)
    dq, dk, dv = (torch.zeros_like(t) for t in (q, k, v))
    a = nat.sdpa_packed_bwd_args(q, k, v, g, out, lse, dq, dk, dv, off)
    need = int(nat.load().mfx_sdpa_packed_bwd_workspace_size(ctypes.byref(a)))
    big = torch.full(((8 << 30) + (64 << 20),), 7, dtype=torch.uint8, device="cuda")
    at = (8 << 30) + (32 << 20)
    nat.sdpa_packed_bwd(q, k, v, g, out, lse, off, dq=dq, dk=dk, dv=dv, workspace=big[at:at + need])
    assert bool((big[:at] == 7).all()) and bool((big[at + need:] == 7).all())
    del big
    check_all(torch, nat, "bf16", MANY, 32, 8, 64)
