"""Calls of the microscaled operators that tests/test_microscale.py does not make."""
import ctypes as C

import numpy as np
import pytest
import torch

import gemm_zoo_b200 as gz
from gemm_zoo_b200 import api, microscale as ms
from tests import mx_oracle as orc
from tests.test_microscale import (ACTS, FORMATS, FP4, HALF, NV, _check_quantised, _guards_intact, _mx, _out, _tolerance,
                                   _values)

gpu = pytest.mark.gpu


# ------------------------------------------------------------------------------------------- shuffles
def test_shuffle_masks_do_not_depend_on_convergence():
    """Which lanes happen to be together (__activemask) says nothing about which lanes share a scale word."""
    for f in (api.PKG / "csrc").rglob("*.cu*"):
        assert "__activemask" not in f.read_text(), f


@gpu
@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_rows_whose_words_end_inside_a_warp(fmt, dtype):
    """Every number of scale words of a row up to a whole block of threads, and rows in several pieces."""
    word = 64 if fmt == NV else 128
    for words in [1, 2, 3, 5, 6, 7, 9, 11, 13, 21, 31, 32, 33, 43, 63, 65]:
        for k in (words * word, words * word - 17):
            x = _values(5, k, dtype, 11)
            _check_quantised(x.double().numpy(), gz.mx_quantize(x.cuda(), fmt), fmt)
