"""The 4-bit GEMM kernels as the compiler made them (gfx950 assembly, no GPU needed): nothing is spilled, and the sums that the
256 x 256 kernels read from accumulation registers through inline assembly, which the compiler's hazard recognizer does not
see, are read behind a wait of more than the 18 states that the last matrix instruction asks for."""
import os
import re
import shutil
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CSRC = os.path.join(ROOT, "cache_dit_amd", "csrc")


def _hipcc():
  for cand in (os.environ.get("HIPCC"), shutil.which("hipcc"), "/opt/rocm/bin/hipcc"):
    if cand and os.path.exists(cand):
      return cand
  return None


@pytest.mark.parametrize("source,kernel,instances", [("gemm_mxfp4.hip", "gemm_mxfp4_tile", 23), ("gemm_w4a16.hip", "gemm_w4a16_", 9)])
def test_spills_and_waits(tmp_path, source, kernel, instances):
  hipcc = _hipcc()
  if hipcc is None:
    pytest.skip("hipcc not found")
  from cache_dit_amd.csrc import build
  out = tmp_path / "k.s"
  r = subprocess.run([hipcc, *build.DEVICE_FLAGS, "-I", os.path.join(ROOT, "include"), "-I", CSRC, "--cuda-device-only", "-S",
                      os.path.join(CSRC, source), "-o", str(out)], capture_output=True, text=True)
  assert r.returncode == 0, r.stderr[-2000:]
  kernels = dict(re.findall(r"^(_ZN\S*" + kernel + r"\S*):[^\n]*\n(.*?)s_endpgm", out.read_text(), re.S | re.M))
  assert len(kernels) == instances, sorted(kernels)
  large = 0
  for name, body in kernels.items():
    assert "scratch_" not in body, name
    assert "v_pk_fma_f32" not in body and "v_pk_mul_f32" not in body and "v_pk_add_f32" not in body, name
    if "Li256ELi256E" not in name:
      continue
    large += 1
    wait = [m.start() for m in re.finditer(r"ASMSTART\n\s*s_nop 15\n\s*s_nop 15\n", body)]
    reads = [m.start() for m in re.finditer(r"ASMSTART\n\s*v_accvgpr_read_b32", body)]
    assert len(wait) == 1 and len(reads) == 4 * 256, (name, len(wait), len(reads))  # with and without GELU, whole and cut
    assert wait[0] < reads[0] and "mfma" not in body[wait[0]:reads[-1]], name
  assert large >= 1
