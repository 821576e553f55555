"""Bounds of lora.hip's buffer accesses (gfx950 assembly, no GPU needed). A buffer compares the vector offset with its size less the scalar
offset. Where a tile has few rows, or the columns end in it, rows and columns that do not exist lie further than the size is: as a scalar
offset they would make that difference negative, and an access that is meant to find nothing would reach memory behind the tensor."""
import os
import re
import shutil
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CSRC = os.path.join(ROOT, "cache_dit_amd", "csrc")


def scalar_offset(line):
  """The scalar offset of a buffer access, as it is written."""
  return re.match(r"buffer_(?:load|store)_\w+ (?:\S+, )?\S+, s\[\d+:\d+\], (\S+)", line)[1]


def test_forms_of_an_access():
  assert scalar_offset("buffer_load_dwordx4 v[4:7], v1, s[8:11], s3 offen") == "s3"
  assert scalar_offset("buffer_load_dwordx4 v1, s[8:11], 0 offen offset:16 lds") == "0"
  assert scalar_offset("buffer_store_dwordx4 v[4:7], v1, s[8:11], 0 offen") == "0"


def test_no_scalar_offsets(tmp_path):
  hipcc = next((c for c in (os.environ.get("HIPCC"), shutil.which("hipcc"), "/opt/rocm/bin/hipcc") if c and os.path.exists(c)), None)
  if hipcc is None:
    pytest.skip("hipcc not found")
  from cache_dit_amd.csrc import build
  out = tmp_path / "k.s"
  r = subprocess.run([hipcc, *build.DEVICE_FLAGS, "-I", os.path.join(ROOT, "include"), "-I", CSRC, "--cuda-device-only", "-S",
                      os.path.join(CSRC, "lora.hip"), "-o", str(out)], capture_output=True, text=True)
  assert r.returncode == 0, r.stderr[-2000:]
  lines = [line.split(";")[0].strip() for line in out.read_text().split("\n")]
  accesses = [line for line in lines if line.startswith("buffer_")]
  kinds = {"lds" if line.endswith("lds") else line.split("_")[1] for line in accesses}
  assert kinds == {"lds", "load", "store"}
  assert not [line for line in accesses if scalar_offset(line) != "0"]
