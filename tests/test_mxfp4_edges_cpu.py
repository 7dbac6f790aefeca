"""MXFP4 entry points without a GPU: sizes at the end of the int range and operands that overlap come back as FW_E_BADARG before anything is
launched, and one row may have any stride."""
import ctypes

import pytest
import torch

from fantasy_world_amd import hip_ops
from test_mxfp4_cpu import lib, p, refused  # noqa: F401

TOP = 0x7fffffff


@pytest.mark.parametrize("K", [TOP, TOP - 254, TOP - 255])
def test_rows_too_long_for_32_bit_columns(lib, p, K):
    """Up to 2^31 - 257 values a row: past that the padded row's columns do not fit an int."""
    refused(lib, lib.fw_mxfp4_quant_rows(p(), K, 1, p(), 1 << 31, p(), 1, K, None), "fw_mxfp4_quant_rows: bf16")
    refused(lib, lib.fw_mxfp4_dequant_rows(p(), 1 << 31, p(), p(), K, 1, 1, K, None), "fw_mxfp4_dequant_rows: bf16")
    refused(lib, lib.fw_gemm_mxfp4(p(), 128, p(), p(), 128, p(), p(), 64, 1, None, 4, 64, K, None, 0, None, None, None, 0, 0, None), "fw_gemm_mxfp4")
    refused(lib, lib.fw_linear_mxfp4(p(), K, p(), 128, p(), p(), 64, 1, None, 4, 64, K, None, 0, None, None, None, 0, 0, p(), 1 << 40, None), "fw_gemm_mxfp4")
    assert lib.fw_linear_mxfp4_workspace_bytes(1, K) == (K + 255) // 256 * (128 + 256)


def test_more_rows_or_columns_than_tiles_can_count(lib, p):
    for M, N in ((TOP, 64), (TOP - 200, 64), (4, TOP), (4, TOP - 200)):
        refused(lib, lib.fw_gemm_mxfp4(p(), 128, p(), p(), 128, p(), p(), 1 << 31, 1, None, M, N, 64, None, 0, None, None, None, 0, 0, None), "2^31 - 256")
    assert lib.fw_linear_mxfp4_workspace_bytes(TOP, 64) == TOP * 128 + (1 << 26) * 256
