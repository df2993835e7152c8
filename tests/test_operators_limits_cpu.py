"""The limit of the operators' device-side waits, as far as it needs no GPU."""
import pytest


@pytest.mark.parametrize("milliseconds,status", [(float("nan"), -1), (60001.0, -1), (float("inf"), -1), (60000.0, 0), (2.5, 0), (-1.0, 0), (0.0, 0)])
def test_wait_limit_is_a_minute_at_most(built_library, milliseconds, status):
    from deepity_b200 import _lib
    lib = _lib.load()
    try:
        assert lib.dpc_operators_set_wait_limit(milliseconds, 0) == status
        assert status == 0 or b"minute" in lib.dpc_last_error()
    finally:
        assert lib.dpc_operators_set_wait_limit(0.0, 0) == 0
