"""The dense operators at their edges, as far as no GPU is needed."""
import pytest


def test_wait_limit_refuses(built_lib):
    assert built_lib.fv_ops_wait_limit(-2) == 1 and b"cycles" in built_lib.fv_last_error()
    assert built_lib.fv_ops_wait_limit(-1) == 0
