"""Grouped products divide a routed row's number by top_k in 32 bits: one that does not fit is refused, ahead of a
launch."""
import pytest

from sglite_amd import _lib

PAST = [1 << 31, 1 << 32, (1 << 32) + 2, (1 << 63) - 1]  # 2^32 would be 0 in 32 bits, 2^32 + 2 would be 2


@pytest.mark.parametrize("top_k", PAST)
def test_refused(top_k):
    lib, inv = _lib.load(), _lib.AWQ_STATUS_INVALID_ARGUMENT
    rows = (64, 100, 128, 256, 8, top_k, 0, 1, 65536)  # sorted ids and their count, offsets, weights, routed rows
    assert lib.awq_moe_w4a16_gemm(4096, 4, 8192, 8192, 8192, 8, 256, 256, 128, 0, *rows, None) == inv
    assert "top_k" in _lib.last_error()
    assert lib.awq_moe_dense_gemm(4096, 4, 8192, 3, 64, 64, 0, *rows, None) == inv
    assert "top_k" in _lib.last_error()
    assert lib.awq_mx4_moe_workspace_bytes(8, top_k, 3, 64, 64, 0) == inv
    assert lib.awq_mx4_moe_gemm(4096, 4, 8192, 128, 3, 64, 64, 0, *rows, 1 << 20, 1 << 20, None) == inv
    assert "top_k" in _lib.last_error()


def test_the_largest_is_planned_for():
    assert _lib.load().awq_mx4_moe_workspace_bytes(8, (1 << 31) - 1, 3, 64, 64, 0) >= 0
