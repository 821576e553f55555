"""The block norm, the 4-bit quantizer and the products of few rows as the compiler made them (gfx950 assembly, no GPU needed): rows
that one piece a lane holds stay in registers, and no others spill than is known; no packed fp32."""
import os
import re
import subprocess

import pytest

from test_mxfp4_isa import CSRC, ROOT, _hipcc


def kernels(tmp_path, source):
  hipcc = _hipcc()
  if hipcc is None:
    pytest.skip("hipcc not found")
  from cache_dit_amd.csrc import build
  out = tmp_path / "k.s"
  r = subprocess.run([hipcc, *build.DEVICE_FLAGS, "-I", os.path.join(ROOT, "include"), "-I", CSRC, "--cuda-device-only", "-S",
                      os.path.join(CSRC, source), "-o", str(out)], capture_output=True, text=True)
  assert r.returncode == 0, r.stderr[-2000:]
  found = dict(re.findall(r"^(_ZN\S+):[^\n]*\n(.*?)s_endpgm", out.read_text(), re.S | re.M))
  for name, body in found.items():
    assert "v_pk_fma_f32" not in body and "v_pk_mul_f32" not in body and "v_pk_add_f32" not in body, name
  return found


def test_block_norm(tmp_path):
  found = kernels(tmp_path, "block_norm.hip")
  rows = {tuple(map(int, re.search(r"rowsILi(\d+)ELi(\d+)ELi(\d+)ELi(\d+)ELb(\d)ELb(\d)E", n).groups())): "scratch_" in body
          for n, body in found.items() if "gate_residual_norm_rows" in n}
  assert len(rows) == 5 * (7 + 12) + 4 * 12, len(rows)  # types: unaligned, aligned; non-temporal where the branch has 16 bits
  for (stream, _, waves, pieces, _, _), spills in rows.items():
    # rows above 8192: 128 registers a lane at 16 wavefronts, 168 at 12, where an fp32 stream is too much
    assert not spills or (pieces == 2 and (waves == 16 or stream == 2)), (stream, waves, pieces)
  assert not any("scratch_" in body for n, body in found.items() if "gate_residual_norm_rows" not in n)


@pytest.mark.parametrize("source,kernel,instances", [("mxfp4_quant.hip", "quant_rows", 10), ("gemm_mx_rows.hip", "gemm_mx_rows", 5)])
def test_no_spills(tmp_path, source, kernel, instances):
  found = {n: body for n, body in kernels(tmp_path, source).items() if kernel in n}
  assert len(found) == instances, sorted(found)
  assert not any("scratch_" in body for body in found.values())
