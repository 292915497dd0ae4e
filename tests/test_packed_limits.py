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


def test_blocks_are_shared_only_where_shares_are_planned(tmp_path):
    """Batches of up to three sequences: whenever packed_share would share a
    block (its arithmetic, in 64 bits here), the plan has shares."""
    run_cpp(tmp_path, r"""
#include "packed_index.h"
#include <algorithm>
#include <cstdio>
using namespace mfx;
int main() {
  int bad = 0, shared = 0, without = 0;
  const int room = 256, least = 8, BM = 128;
  for (int quarters : {3, 4})
    for (int64_t heads = 1; heads <= 1024; heads += heads < 40 ? 1 : 13)
      for (int64_t tiles : {2, 4, 6, 8, 10, 16, 64})
        for (int64_t a = 1; a <= 40; a += 3)
          for (int64_t b : {0, 1, 7, 40})
            for (int64_t c : {0, 2}) {
              const int64_t all = (a * (a + 1) / 2 + b * (b + 1) / 2 + c * (c + 1) / 2) * tiles * heads * quarters;
              const int64_t most = std::max<int64_t>((all + 4 * room - 1) / (4 * room), least);
              const bool shares = std::max(a, b) - most / tiles > 0;  // blocks of two shares or more
              // The fewest tokens with so many blocks.
              const int64_t total = (a - 1) * BM + 1 + (b ? (b - 1) * BM + 1 : 0) + (c ? (c - 1) * BM + 1 : 0);
              const bool planned = packed_shares_possible(total, BM, heads, quarters, room, tiles, least);
              bad += shares && !planned;
              shared += shares;
              without += !planned;
            }
  std::printf("%d %d %d\n", bad, shared, without);
  return bad != 0 || shared < 1000 || without < 1000;
}
""")


def _workspace(nat, T, n, Hq, Hkv, D):
    a = nat.SdpaPackedBwdArgs()
    for i, f in enumerate(("q", "k", "v", "dout", "out", "lse", "dq", "dk", "dv", "seq_offsets")):
        setattr(a, f, 0x100000 * (i + 1))
    a.T, a.num_seqs, a.Hq, a.Hkv, a.D = T, n, Hq, Hkv, D
    for f, _ in a._fields_:
        if f.endswith("_strides"):
            getattr(a, f)[:] = [D, (Hkv if f[:2] in ("k_", "v_", "dk", "dv") else Hq) * D, 1]
    a.scale, a.causal, a.dtype = 0.125, 1, nat.MFX_BF16
    return int(nat.load().mfx_sdpa_packed_bwd_workspace_size(ctypes.byref(a)))


def test_no_workspace_for_shares_that_cannot_be(nat):
    """Few tokens of many heads: no block has more tiles than a share, or all
    heads' blocks are more than the CUs.  The workspace is the row sums then."""
    for T, n, Hq, Hkv in ((100, 1, 512, 512), (100, 1, 1024, 1024), (100, 3, 300, 300), (500, 1, 128, 128),
                          (100, 1, 5120, 1024), (128, 2, 1600, 320), (50, 1, 64, 16)):
        rows = (Hq * T * 4 + 255) // 256 * 256
        assert _workspace(nat, T, n, Hq, Hkv, 128) == rows, (T, n, Hq, Hkv)
    # Where blocks are shared there is room for it.
    for T, n, Hq, Hkv in ((1411, 1, 8, 1), (2000, 3, 32, 8), (2536, 3, 8, 1), (100, 1, 80, 8)):
        assert _workspace(nat, T, n, Hq, Hkv, 128) > Hq * T * 4 + (1 << 20)


def test_workspace_for_shares_is_bounded(nat):
    """All head counts and lengths that shares are planned for, at D 128."""
    most = 0
    for Hkv in (*range(1, 40), *range(40, 1100, 7)):
        for group in (1, 2, 4, 5, 8, 16):
            for T in (100, 128, 129, 500, 513, 640, 1000, 2049, 4096, 8192, 16384, 65536, 131000):
                for n in (1, 8, 64, 512):
                    if Hkv * group <= 65535 and T * Hkv * group < 1 << 31:
                        most = max(most, _workspace(nat, T, n, Hkv * group, Hkv, 128) - Hkv * group * T * 4)
    assert most <= 180e6, most


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
