"""Refusals of the operators for blocks of language models (include/qcnn.h) and their 64-bit oracle; no GPU."""
import ctypes as C

import numpy as np
import pytest

from oracle import np_blocks
from qcnn_gpu_amd import capi

E_ARG, E_UNSUPPORTED = -1, -6
A = 1 << 20  # an address that no refused call may look at


def w4(**kw):
    f = dict(x=A, y=A, w=A, scale=A, ldx=64, ldy=8, ldw=32, rows=1, n=8, k=64, group=32, type=capi.BF16, scale_type=capi.BF16, out_type=capi.BF16)
    return capi.load().qcnn_op_matvec_w4, capi.MatvecW4(**{**f, **kw})


def grouped(**kw):
    f = dict(x=A, y=A, w=A, offsets=A, ldx=64, ldy=8, ldw=64, w_stride=512, rows=4, x_rows=4, experts=2, n=8, k=64, type=capi.F16, out_type=capi.F32)
    return capi.load().qcnn_op_grouped_matmul, capi.GroupedMatmul(**{**f, **kw})


def norm(**kw):
    f = dict(x=A, y=A, h=2 * A, n=3 * A, ldx=64, ldy=64, ldg=64, ldh=64, ldn=64, rows=4, y_rows=4, d=64, parts=1, gate_rows=1, type=capi.F16,
             w_type=capi.F16, post=1, pre=1, act=0, alpha=1, beta=1, post_eps=1e-6, pre_eps=1e-6)
    return capi.load().qcnn_op_norm_res, capi.NormRes(**{**f, **kw})


REFUSED = [
    (w4, dict(type=3), E_UNSUPPORTED), (w4, dict(scale_type=9), E_UNSUPPORTED), (w4, dict(out_type=-1), E_UNSUPPORTED),
    (w4, dict(rows=-1), E_ARG), (w4, dict(n=0), E_ARG), (w4, dict(k=0), E_ARG), (w4, dict(n=(1 << 26) + 1, ldy=1 << 29), E_UNSUPPORTED), (w4, dict(ldx=(1 << 24) + 1), E_UNSUPPORTED), (w4, dict(ldw=(1 << 25) + 1), E_UNSUPPORTED), (w4, dict(group=0), E_ARG), (w4, dict(group=48), E_ARG),
    (w4, dict(group=-32), E_ARG), (w4, dict(ldx=63), E_ARG), (w4, dict(ldy=7), E_ARG), (w4, dict(ldw=31), E_ARG), (w4, dict(ldw=1 << 62), E_UNSUPPORTED),
    (w4, dict(k=63, ldx=63, ldw=31), E_ARG), (w4, dict(x=None), E_ARG), (w4, dict(y=None), E_ARG), (w4, dict(w=None), E_ARG), (w4, dict(scale=None), E_ARG),
    (w4, dict(x=A + 1), E_ARG), (w4, dict(scale=A + 1), E_ARG), (w4, dict(bias=A + 2), E_ARG), (w4, dict(y=A + 2, out_type=capi.F32), E_ARG),
    (grouped, dict(type=4), E_UNSUPPORTED), (grouped, dict(out_type=capi.I8), E_UNSUPPORTED), (grouped, dict(act=3), E_ARG), (grouped, dict(act=-1), E_ARG),
    (grouped, dict(rows=-1), E_ARG), (grouped, dict(x_rows=-1, src=A), E_ARG), (grouped, dict(n=0), E_ARG),
    (grouped, dict(k=0), E_ARG), (grouped, dict(experts=0), E_UNSUPPORTED), (grouped, dict(experts=1025), E_UNSUPPORTED),
    (grouped, dict(k=(1 << 28) + 1, ldx=1 << 29, ldw=1 << 29), E_UNSUPPORTED), (grouped, dict(n=(1 << 28) + 1, ldy=1 << 29), E_UNSUPPORTED), (grouped, dict(type=capi.I8, k=131072, ldx=131072, ldw=131072), E_UNSUPPORTED), (grouped, dict(ldx=63), E_ARG), (grouped, dict(ldy=7), E_ARG),
    (grouped, dict(ldw=63), E_ARG), (grouped, dict(w_stride=1 << 62), E_ARG), (grouped, dict(x=None), E_ARG), (grouped, dict(w=None), E_ARG),
    (grouped, dict(y=None), E_ARG), (grouped, dict(offsets=None), E_ARG), (grouped, dict(offsets=A + 2), E_ARG), (grouped, dict(src=A + 1), E_ARG),
    (grouped, dict(x=A + 1), E_ARG), (grouped, dict(bias=A + 2), E_ARG), (grouped, dict(row_scale=A + 2), E_ARG),
    (norm, dict(type=3), E_UNSUPPORTED), (norm, dict(w_type=capi.BF16), E_UNSUPPORTED), (norm, dict(post=3), E_ARG), (norm, dict(pre=-1), E_ARG),
    (norm, dict(gate=A, act=4), E_ARG), (norm, dict(rows=-1), E_ARG), (norm, dict(d=0), E_ARG), (norm, dict(d=65537), E_UNSUPPORTED),
    (norm, dict(post_eps=-1), E_ARG), (norm, dict(x=None), E_ARG), (norm, dict(h=None, n=None), E_ARG), (norm, dict(y=None, index=A), E_ARG),
    (norm, dict(y=None, gate=A), E_ARG), (norm, dict(gate=A, gate_rows=0), E_ARG), (norm, dict(y_rows=3), E_ARG), (norm, dict(parts=2), E_ARG),
    (norm, dict(index=A, parts=0), E_ARG), (norm, dict(index=A, parts=65), E_ARG), (norm, dict(index=A, y_rows=0), E_ARG), (norm, dict(ldx=63), E_ARG),
    (norm, dict(ldy=63), E_ARG), (norm, dict(gate=A, ldg=63), E_ARG), (norm, dict(ldh=63), E_ARG), (norm, dict(ldn=63), E_ARG),
    (norm, dict(ldx=1 << 62), E_ARG), (norm, dict(n=2 * A), E_ARG), (norm, dict(x=A + 1), E_ARG), (norm, dict(pre_w=A + 1), E_ARG),
    (norm, dict(h=A, index=A), E_ARG), (norm, dict(h=A, ldh=65), E_ARG),
]


@pytest.mark.parametrize("make,kw,code", REFUSED, ids=lambda v: getattr(v, "__name__", None) or str(v).replace(" ", ""))
def test_refusals(make, kw, code):
    fn, a = make(**kw)
    assert fn(C.byref(a), None) == code
    assert capi.load().qcnn_last_error()


@pytest.mark.parametrize("make", (w4, grouped, norm))
def test_null_and_empty_calls(make):
    fn, a = make(rows=0, x=None, y=None, **({"y_rows": 0} if make is norm else {}))
    assert fn(C.byref(a), None) == 0  # no rows: nothing to do, no pointer looked at
    assert fn(None, None) == E_ARG


def test_structures_have_the_sizes_of_the_header():
    """The C compiler lays out pointers, then size_t, then int, then float without holes; so does ctypes."""
    assert C.sizeof(capi.MatvecW4) == 6 * 8 + 3 * 8 + 8 * 4  # seven ints, padded to eight bytes
    assert C.sizeof(capi.GroupedMatmul) == 9 * 8 + 4 * 8 + 8 * 4
    assert C.sizeof(capi.NormRes) == 10 * 8 + 5 * 8 + 16 * 4  # ten ints and five floats, padded


def test_oracle_on_values_done_by_hand():
    # two outputs of three inputs: codes 1, 9, 15 and 8, 8, 0; scale 0.5 and 2; zero point 8
    w = np.array([[0x91, 0x0F], [0x88, 0xF0]], np.uint8)  # the high half of the last byte belongs to no input
    y, b = np_blocks.matvec_w4(np.array([[1.0, 2.0, 3.0]]), w, np.array([[0.5, 2.0]]), None, None, 3, 32)
    assert y.tolist() == [[0.5 * (-7 + 2 + 21), 2 * -24.0]] and (b > 0).all()
    x = np.array([[1, 2], [3, 4]], np.int8)
    wt = np.array([[[1, 0]], [[0, -1]]], np.int8)
    out, b = np_blocks.grouped_matmul(x, wt, [0, 1, 2], np.array([1, 7, 0]), None, None, None, np.array([2, 2, 2.0]), 0, np.full((3, 1), 5.0))
    assert out[:, 0].tolist() == [6.0, 0.0, 5.0] and b[2, 0] == 0  # an index outside reads zeros, a row behind stays
    h, _, n, _ = np_blocks.norm_res(np.zeros((1, 2)), np.array([[3.0, 5.0], [1.0, 1.0]]), np.array([[0, 1, 9]]), None, 1, 0, None, None, 2, None,
                                    np.array([0.0, 1.0]), 0, 0.5, 1.0, 0.0, 0.0, 0.0)
    assert h.tolist() == [[2.0, 3.0]] and n.tolist() == [[-1.0, 2.0]]
