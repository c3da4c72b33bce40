"""Sizes of calls on drafted tokens: workspaces that serve smaller calls."""

import pytest

from falcon_perception_amd import ops


@pytest.mark.parametrize("V", [1, 500, 4096, 32000, 65536, 150001, 1 << 24])
def test_a_verification_workspace_serves_every_smaller_call(native_lib, V):
    """Fewer requests, fewer rows, a smaller vocabulary: of what a program asks for its largest call it can run all others."""
    largest = 0
    for B in range(1, 65):
        n = ops.verify_workspace_bytes(B, 16, V)
        assert n >= largest, (B, n, largest)
        largest = n
    for S in (1, 2, 7, 16, 33, 64):
        sizes = [ops.verify_workspace_bytes(B, S, V) for B in (1, 2, 3, 5, 6, 9, 24, 25, 64, 130)]
        assert sizes == sorted(sizes), (S, sizes)
    for B in (1, 6, 24, 64):
        sizes = [ops.verify_workspace_bytes(B, S, V) for S in range(1, 65)]
        assert sizes == sorted(sizes), (B, sizes)
    sizes = [ops.verify_workspace_bytes(6, 16, v) for v in sorted({1, 7, 1000, 4096, 4097, 32000, 32769, 65536, V})]
    assert sizes == sorted(sizes)


def test_a_workspace_is_not_much_larger_than_its_call(native_lib):
    assert ops.verify_workspace_bytes(1, 1, 1) < 1 << 17
    # 512 requests of 33 rows of 65536: 4 chunks of 16384 a row, 256 pieces of 256 a request
    assert ops.verify_workspace_bytes(512, 33, 65536) < 512 * (33 * 4 * 16 + 256 * 32) + (1 << 18)
