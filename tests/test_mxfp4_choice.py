"""The kernels that the 4-bit products choose by shape, at shapes where the rules were measured on both sides (figures beside the
rules in csrc/gemm_mx_rows.hip and csrc/mx_tile.h) and at the timed cases. No GPU: the choice of 256 compute units."""
import pytest

DIRECT, ROWS = 0, 100


@pytest.fixture(scope="module")
def choice():
  from cache_dit_amd import _native
  if not _native.is_built():
    pytest.skip("libcdit_hip.so not built")
  return _native.load().cdit_debug_mxfp4_choice


@pytest.mark.parametrize("M,N,K,want", [
    # few rows: while rows times columns are few
    (1, 30720, 5120, ROWS), (4, 13824, 5120, ROWS), (8, 13824, 5120, ROWS), (16, 13824, 5120, 8), (16, 5120, 5120, ROWS),
    (16, 30720, 5120, 8),
    # more rows: where the tiles leave CUs idle
    (294, 16, 9248, ROWS), (502, 128, 5856, ROWS), (32, 1024, 15360, ROWS), (17, 5120, 5120, 8),
    # tiles
    (64, 5120, 4096, 8), (600, 1024, 2560, 4), (512, 5120, 4096, 2), (1357, 4463, 2208, 2), (32760, 13824, 5120, 1),
    (8192, 10240, 2560, 1),
    # rows of codes that 256 of do not fit 32-bit offsets
    (300, 64, 2**24, DIRECT), (16, 16, 2**28, DIRECT), (16, 16, 2**28 - 32, ROWS)])
def test_w4a4(choice, M, N, K, want):
  assert choice(0, M, N, K) == want


@pytest.mark.parametrize("M,N,K,want", [
    (1, 13824, 5120, ROWS), (8, 13824, 5120, ROWS), (16, 13824, 5120, ROWS), (16, 30720, 5120, 4),
    (294, 16, 9248, ROWS), (502, 128, 5856, ROWS), (32, 1024, 15360, ROWS), (17, 5120, 5120, 8),
    (77, 5120, 4096, 8), (4608, 5120, 5120, 6), (16384, 5120, 5120, 1), (300, 64, 2**24, DIRECT)])
def test_w4a16(choice, M, N, K, want):
  assert choice(1, M, N, K) == want


def test_no_such_problem(choice):
  for M, N, K in ((0, 1, 32), (1, 0, 32), (1, 1, 48), (1, 1, 0), (1, 1, 2**29 + 32), (2**31, 1, 32)):
    assert choice(0, M, N, K) == -1 and choice(1, M, N, K) == -1
