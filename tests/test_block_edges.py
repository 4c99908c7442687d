"""Refusals of the operators for blocks of language models (include/qcnn.h) at the largest sizes; no GPU."""
import ctypes as C

import pytest

from qcnn_gpu_amd import capi
from test_block_ops import E_UNSUPPORTED, grouped

BIG = 2 ** 31 - 1


@pytest.mark.parametrize("make,kw", ((grouped, dict(rows=BIG, n=512, ldy=512)), (grouped, dict(rows=1024, experts=1024, n=1 << 28, ldy=1 << 28)),
                                     (grouped, dict(rows=1 << 20, n=1 << 20, ldy=1 << 20))), ids=str)
def test_more_tiles_than_a_launch_takes(make, kw):
    fn, a = make(**kw)
    assert fn(C.byref(a), None) == E_UNSUPPORTED
    assert b"tiles" in capi.load().qcnn_last_error()
