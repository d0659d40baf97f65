"""Further refusals of the stand-alone operators: checked before anything is enqueued, so they need no GPU."""
import ctypes

import pytest

import sparsemoe_b200 as sm

FAKE = 1 << 20   # never dereferenced: every call below is refused first


def test_int8_selftest_refusals():
    for ns, written in ((0, FAKE), (-5, FAKE), (10_000_000_001, FAKE), (50_000_000, None), (50_000_000, FAKE + 2)):
        assert sm.lib.moe_selftest_int8_wait_timeout(ns, written, None) == sm.MOE_ERR_INVALID_ARG
        assert b"selftest" in sm.lib.moe_last_error()
