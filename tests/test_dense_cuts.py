"""How the dense attention calls are cut (ssa_amd/csrc/ssa_cuts.h, compiled for the host): the
cases of tests/test_gpu_dense_long.py reach the kernels that they are there for."""

import os
import shutil
import subprocess

import pytest
import torch

from ssa_amd import _lib
from tests.test_gpu_dense_long import MASKED, PAGED

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

SOURCE = r"""
#include <stdio.h>
#include "ssa_cuts.h"
using namespace ssa;
int main() {
  char op;
  int dtype, h_q, h_kv, d;
  long long a, b, c, e;
  while (scanf(" %c %d %lld %lld %lld %lld %d %d %d", &op, &dtype, &a, &b, &c, &e, &h_q, &h_kv, &d) == 9) {
    if (op == 'm') {  // batch n n_q -
      const DenseSplit f = dense_split(c * (h_q / h_kv), a * h_kv, b, c, dtype == SSA_DTYPE_F32, d > 64, false);
      const BwdCut l = bwd_cut(dtype, a, b, c, h_q, h_kv, d);
      printf("%d %d %d %d %d\n", f.kw, f.parts, l.kw, l.key_groups, l.splits);
    } else {  // tokens batch max_new max_len
      const PagedPlan l = paged_plan(dtype, a, b, h_q, h_kv, d, c, e);
      printf("%d %d\n", l.row_kw, l.row_splits);
    }
  }
}
"""


@pytest.fixture(scope="module")
def cuts(tmp_path_factory):
    cxx = shutil.which("g++")
    if cxx is None:
        pytest.skip("no g++")
    at = tmp_path_factory.mktemp("cuts")
    (at / "cuts.cpp").write_text(SOURCE)
    subprocess.run([cxx, "-std=c++17", "-Wall", "-Werror", f"-I{ROOT}/ssa_amd/csrc", f"-I{ROOT}/include", "-o", str(at / "cuts"),
                    str(at / "cuts.cpp")], check=True)

    def ask(op, dtype, *sizes):
        code = _lib.DTYPE_F32 if dtype == torch.float32 else _lib.DTYPE_BF16
        line = f"{op} {code} " + " ".join(str(x) for x in sizes)
        res = subprocess.run([str(at / "cuts")], input=line, capture_output=True, text=True, check=True)
        return tuple(int(x) for x in res.stdout.split())

    return ask


@pytest.mark.parametrize("case,want", MASKED, ids=str)
def test_masked(cuts, case, want):
    dtype, B, n, n_q, h_kv, g, d = case
    assert cuts("m", dtype, B, n, n_q, 0, h_kv * g, h_kv, d) == want


@pytest.mark.parametrize("case,want,own", PAGED, ids=str)
def test_paged(cuts, case, want, own):
    dtype, seqs, h_kv, g, d = case
    new, keys = max(m for m, _ in seqs), max(m + c for m, c in seqs)
    assert cuts("p", dtype, sum(m for m, _ in seqs), len(seqs), new, keys, h_kv * g, h_kv, d) == want
    assert (3 * new >= keys) == own


def test_every_kernel_is_reached():
    """Of both types and both widths: the forward's and dQ's waves that share rows, dK/dV's
    key groups, the paged chunks with and without their own rows read as contiguous ones.  Four
    waves, and the smallest key groups, are what the small cases of the other tests take."""
    wide = lambda d: d > 64  # noqa: E731
    for dtype in (torch.float32, torch.bfloat16):
        for w in (False, True):
            masked = [want for c, want in MASKED if c[0] == dtype and wide(c[6]) == w]
            assert {1, 2} <= {x[0] for x in masked} and {1, 2} <= {x[2] for x in masked} and 4 in {x[3] for x in masked}
            assert w or 2 in {x[3] for x in masked}
            paged = [(want[0], own) for c, want, own in PAGED if c[0] == dtype and wide(c[4]) == w]
            assert {(1, True), (1, False), (2, True), (2, False)} <= set(paged)
    assert {1} < {want[4] for _, want in MASKED}
