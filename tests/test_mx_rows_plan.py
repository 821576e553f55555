"""The memory of the 4-bit kernel for few rows, for every length of K that it takes: what it asks for is what it uses, and fits.
No GPU: the arithmetic of csrc/mx_rows_plan.h, compiled for the host."""
import os
import subprocess

import pytest

HERE = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(HERE)


@pytest.fixture(scope="module")
def plan(tmp_path_factory):
  exe = str(tmp_path_factory.mktemp("plan") / "plan")
  cc = subprocess.run(["g++", "-std=c++17", "-O1", "-I", os.path.join(ROOT, "cache_dit_amd", "csrc"),
                       os.path.join(HERE, "native", "mx_rows_plan.cc"), "-o", exe], capture_output=True, text=True)
  assert cc.returncode == 0, cc.stderr

  def run(problems):
    r = subprocess.run([exe], input="\n".join(" ".join(map(str, p)) for p in problems), capture_output=True, text=True)
    assert r.returncode == 0
    return [tuple(map(int, line.split())) for line in r.stdout.splitlines()]

  return run


def used(weight_only, M, groups, chunk, waves):
  """Bytes the kernel indexes: partial sums, the weight's scales, the activation's rows, their scales."""
  rows = min(M, 16)
  x, s = (1024 if weight_only else 256) * chunk + 16, 16 * chunk + 4
  return 1024 * groups * waves + 16 * groups * s + rows * (x + s)


def test_every_length_of_k_fits(plan):
  problems = [(wo, M, N, K, 256) for wo in (0, 1) for M in (1, 2, 3, 8, 15, 16, 500) for N in (1, 16, 8193, 2**31 - 600)
              for K in (0, 32, 512, 544, 5120, 16384, 65568, 2**20, 2**26 - 32, 2**26, 2**26 + 32, 140000032, 250000032, 2**28 - 32)]
  for (wo, M, N, K, cus), (groups, chunk, waves, lds) in zip(problems, plan(problems)):
    case = (wo, M, N, K, groups, chunk, waves, lds)
    items = max(1, -(-K // 512))
    assert groups == (2 if -(-N // 16) > 2 * cus else 1), case
    assert 1 <= chunk <= items and 1 <= waves <= 8 and waves * -(-chunk // waves) >= chunk, case
    assert lds == used(wo, M, groups, chunk, waves), case
    # two workgroups to a CU, and no smaller piece of K than need be
    activation = lds - 1024 * groups * waves
    assert activation <= 64 * 1024 and lds <= 80 * 1024, case
    assert chunk == items or used(wo, M, groups, chunk + 1, 0) > 64 * 1024, case
