"""Sizes that the categorical-head operators refuse before anything is launched: no GPU is needed."""
import ctypes as C

import pytest

from lvd_pg_b200 import _lib, build

INVALID = 1


@pytest.fixture(scope="module")
def lib():
    build.build()
    return _lib.lib()


@pytest.mark.parametrize("variables", [1 << 31, (1 << 32) - 1])
def test_more_variables_than_tiles_are_counted(lib, variables):
    """A tile of one variable each: a block's count of them, 65535 at a time, would pass 2^32 and begin anew."""
    b = C.create_string_buffer(80)
    assert lib.pcb_soft_evidence(b, 0, 1, variables, 1, 0, 0, None, 0, 0, 1.0, b, None, None) == INVALID
    assert b"variables" in lib.pcb_last_error()
    assert lib.pcb_soft_evidence_backward(b, 0, 1, variables, 1, 0, 0, None, 0, 0, 1.0, b, b, b, None) == INVALID
    assert b"variables" in lib.pcb_last_error()
