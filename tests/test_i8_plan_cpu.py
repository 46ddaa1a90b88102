"""Refusals of bbh_linear_i8_plan, which need no GPU."""
import ctypes

import pytest
import torch

ARG, CUDA, UNSUPPORTED = -1, -3, -6


@pytest.mark.parametrize("M,N,K", [(0, 8, 16), (8, 0, 16), (8, 8, 0), (-1, 8, 16), (8, -1, 16), (8, 8, 131072)])
def test_bad_sizes(M, N, K):
    import bbh

    assert bbh.lib().bbh_linear_i8_plan(M, N, K, 0, (ctypes.c_int * 3)()) == ARG
    assert b"bbh_linear_i8_plan" in bbh.lib().bbh_last_error()
    with pytest.raises(bbh.BBHError):
        bbh.linear_i8_plan(M, N, K)


def test_null_result():
    import bbh

    assert bbh.lib().bbh_linear_i8_plan(8, 8, 16, 0, None) == ARG


@pytest.mark.skipif(torch.cuda.is_available(), reason="there is a device")
def test_without_a_device():
    import bbh

    plan = (ctypes.c_int * 3)(7, 7, 7)
    assert bbh.lib().bbh_linear_i8_plan(8, 8, 16, 0, plan) in (CUDA, UNSUPPORTED)
    assert list(plan) == [7, 7, 7]
