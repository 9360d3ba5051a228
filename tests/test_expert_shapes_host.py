"""Which form of the experts' product a call takes, seen from the host: the tests of each form reach it."""
import ctypes

import pytest

import rxmet_lib
import test_expert_large_tiles_gpu as large

FEW_SHARED, FEW, T128X64, T128X128, T256X256 = range(5)


def form(rows, experts, weight_rows):
    return rxmet_lib.load().rxmet_selftest_experts_form(rows, experts, weight_rows)


def test_forms():
    assert form(8, 4, 512) == FEW_SHARED
    assert form(16, 16, 2048) == FEW
    assert form(128, 64, 2048) == T128X64
    assert form(65536, 32, 2048) == T256X256


@pytest.mark.parametrize("less", [0, 1, 2])
def test_large_tiles_are_tested(less):
    for (T, k, E, out), want in ((large.MIDDLE, T128X128), (large.LARGE, T256X256)):
        assert form(T * k, E, out - less) == want


def test_small_batches_of_them_take_another():
    for T, k, E, out in (large.MIDDLE, large.LARGE):
        assert form(4 * k, E, out) in (FEW_SHARED, FEW)
