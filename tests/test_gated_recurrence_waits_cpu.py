"""Limits of the gated recurrence's waits, without a GPU."""
import pytest

from tensoroperations_b200 import abi


@pytest.mark.parametrize("maps,tiles,want", [
    (0, 0, abi.TO_OK), (100, 5, abi.TO_OK), (-1, 3600000000, abi.TO_OK), (3600000001, 0, abi.TO_ERR_INVALID_ARGUMENT),
    (0, 2 ** 62, abi.TO_ERR_INVALID_ARGUMENT), (-2 ** 62, -1, abi.TO_OK)])
def test_limits(maps, tiles, want):
    try:
        assert abi.lib.to_gated_recurrence_wait_limits(maps, tiles) == want
        assert want == abi.TO_OK or b"wait_limits" in abi.lib.to_last_error()
    finally:
        abi.lib.to_gated_recurrence_wait_limits(-1, -1)
