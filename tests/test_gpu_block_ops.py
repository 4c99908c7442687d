"""GPU parity of the operators for blocks of language models against the 64-bit oracle (oracle/np_blocks.py).

Tolerance: the oracle's first-order bound of a float32 evaluation plus half a step of the output type; integer data pins
the element order exactly."""
import ctypes as C
import pathlib
import subprocess
import sys
import threading

import numpy as np
import pytest
import torch

from oracle import np_blocks
from qcnn_gpu_amd import capi

pytestmark = pytest.mark.gpu
T = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16, "i8": torch.int8}
KIND = {"f32": capi.F32, "f16": capi.F16, "bf16": capi.BF16, "i8": capi.I8}
TINY = {"f32": 2.0 ** -149, "f16": 2.0 ** -24, "bf16": 2.0 ** -133}
PAD = 77.0  # stands between the rows of an output and must stay


def ptr(t):
    return None if t is None else t.data_ptr()


def np64(t):
    return None if t is None else t.double().cpu().numpy() if t.is_floating_point() else t.cpu().numpy()


def close(got, want, bound, kind, what=""):
    got = got.double().cpu().numpy()
    tol = bound + np_blocks.half_step(np.abs(want) + bound, torch.finfo(T[kind]).eps, TINY[kind])
    # a value from max + half a step on rounds to infinity (half: 65504 + 16): the infinity of its sign is the right answer there
    top = float(torch.finfo(T[kind]).max) * (1 + torch.finfo(T[kind]).eps / 4)
    with np.errstate(invalid="ignore"):
        over = (np.abs(want) + bound >= top) & (got == np.sign(want) * np.inf)
        bad = ~(np.abs(got - want) <= tol) & ~over
    assert not bad.any(), (what, int(bad.sum()), [(tuple(i), got[tuple(i)], want[tuple(i)], tol[tuple(i)]) for i in np.argwhere(bad)[:3]])


def rows_of(values, kind, pad, shift=0):
    """values [r][c] on the GPU in rows of c + pad elements, `shift` elements into an allocation."""
    r, c = values.shape
    buf = torch.full((r * (c + pad) + shift + 64,), PAD if kind != "i8" else 77, dtype=T[kind], device="cuda")
    v = buf[shift:shift + r * (c + pad)].view(r, c + pad)
    v[:, :c] = values.to(T[kind]).cuda()
    return v, buf


def call(fn, a, stream=None):
    s = torch.cuda.current_stream().cuda_stream if stream is None else stream
    capi.check(fn(C.byref(a), s))


# ---- 4-bit products --------------------------------------------------------------------------------------
def w4_data(rows, n, k, group, kind, zeros, bias, seed, ints=False):
    g = torch.Generator().manual_seed(seed)
    ng = -(-k // group)
    x = torch.randint(-3, 4, (rows, k), generator=g).double() if ints else torch.randn(rows, k, generator=g, dtype=torch.float64)
    w = torch.randint(0, 256, (n, (k + 1) // 2), generator=g, dtype=torch.uint8)
    scale = 2.0 ** torch.randint(-2, 2, (ng, n), generator=g).double() if ints else torch.rand(ng, n, generator=g, dtype=torch.float64) / k ** 0.5 + 1e-3
    zero = torch.randint(0, 16, (ng, n), generator=g, dtype=torch.uint8) if zeros else None
    b = (torch.randint(-8, 9, (n,), generator=g).float() if ints else torch.randn(n, generator=g)) if bias else None
    return x, w, scale, zero, b


def w4_run(x, w, scale, zero, b, group, kind, skind=None, okind=None, pads=(0, 0, 0), shift=0, stream=None):
    skind, okind = skind or kind, okind or kind
    rows, k = x.shape
    n = w.shape[0]
    xv, xb = rows_of(x, kind, pads[0], shift)
    wbuf = torch.full((n * (w.shape[1] + pads[1]) + shift + 64,), 0xA5, dtype=torch.uint8, device="cuda")
    wv = wbuf[shift:shift + n * (w.shape[1] + pads[1])].view(n, -1)
    wv[:, :w.shape[1]] = w.cuda()
    sv = scale.to(T[skind]).cuda()
    zv, bv = (None if zero is None else zero.cuda()), (None if b is None else b.float().cuda())
    yv, yb = rows_of(torch.full((rows, n), PAD), okind, pads[2], shift)
    a = capi.MatvecW4(x=ptr(xv), y=ptr(yv), w=ptr(wv), scale=ptr(sv), zero=ptr(zv), bias=ptr(bv), ldx=xv.stride(0), ldy=yv.stride(0),
                      ldw=wv.stride(0), rows=rows, n=n, k=k, group=group, type=KIND[kind], scale_type=KIND[skind], out_type=KIND[okind])
    call(capi.load().qcnn_op_matvec_w4, a, stream)
    torch.cuda.synchronize()
    assert (yb.double() == PAD).sum() >= yb.numel() - rows * n and (yv[:, n:].double() == PAD).all()
    assert (yb[:shift].double() == PAD).all() and (yb[shift + rows * yv.stride(0):].double() == PAD).all()
    want, bound = np_blocks.matvec_w4(np64(xv[:, :k]), w.numpy(), np64(sv), None if zero is None else zero.numpy(), np64(bv), k, group)
    return yv[:, :n], want, bound


W4_SHAPES = [(1, 1, 1, 32), (1, 16, 32, 32), (1, 17, 33, 32), (2, 5, 31, 64), (3, 64, 128, 64), (1, 100, 257, 128), (16, 48, 256, 128),
             (17, 33, 384, 96), (32, 70, 130, 32), (33, 16, 1000, 256), (64, 20, 512, 4096), (65, 130, 63, 32), (130, 31, 200, 64), (1, 512, 4096, 128),
             (4, 2000, 96, 32), (8, 40, 9001, 128), (1, 3, 20000, 32)]


@pytest.mark.parametrize("kind", ("f32", "f16", "bf16"))
@pytest.mark.parametrize("zeros", (False, True))
@pytest.mark.parametrize("shape", W4_SHAPES, ids=str)
def test_w4_against_the_definition(shape, zeros, kind):
    rows, n, k, group = shape
    d = w4_data(rows, n, k, group, kind, zeros, rows % 2 == 1, 11 * n + k)
    close(*w4_run(*d, group, kind), kind)


@pytest.mark.parametrize("kind", ("f32", "f16", "bf16"))
@pytest.mark.parametrize("rows", (1, 4, 5, 16, 17, 33, 64, 70))
@pytest.mark.parametrize("n,k,group", ((4096, 384, 64), (4100, 256, 32), (8200, 300, 128), (4097, 1000, 96), (150, 5000, 64)))
def test_w4_many_outputs(n, k, group, rows, kind):
    """Both sides of every border of the launch rules, groups of all three kinds, a last workgroup that is not full."""
    d = w4_data(rows, n, k, group, kind, True, True, n + rows)
    close(*w4_run(*d, group, kind), kind)


@pytest.mark.parametrize("kind", ("f32", "f16", "bf16"))
@pytest.mark.parametrize("zeros", (False, True))
def test_w4_integers_are_exact(kind, zeros):
    """Integer inputs and scales that are powers of two: every sum is exact in float32."""
    for rows, n, k, group in ((1, 37, 77, 32), (5, 64, 512, 64), (20, 50, 300, 128), (64, 18, 1031, 32)):
        d = w4_data(rows, n, k, group, kind, zeros, True, n + k, ints=True)
        y, want, _ = w4_run(*d, group, kind, okind="f32")
        assert np.array_equal(y.double().cpu().numpy(), want), (rows, n, k)


@pytest.mark.parametrize("kind,skind,okind", (("f32", "f16", "bf16"), ("bf16", "f32", "f32"), ("f16", "bf16", "f32"), ("bf16", "f16", "f16")))
@pytest.mark.parametrize("pads,shift", (((0, 0, 0), 1), ((1, 1, 1), 0), ((3, 5, 7), 3), ((8, 16, 8), 8)))
def test_w4_types_strides_and_addresses(kind, skind, okind, pads, shift):
    for rows, n, k in ((1, 33, 129), (7, 64, 256), (19, 21, 511)):
        d = w4_data(rows, n, k, 64, kind, True, True, 5 + k)
        close(*w4_run(*d, 64, kind, skind, okind, pads, shift), okind, (rows, n, k))


def test_w4_large_and_small_values():
    """float32 inputs over many powers of two keep float32 precision; half outputs overflow to infinity as the rounding says."""
    g = torch.Generator().manual_seed(3)
    x = torch.randn(3, 256, generator=g, dtype=torch.float64) * 10.0 ** torch.randint(-20, 20, (3, 1), generator=g)
    _, w, scale, zero, b = w4_data(3, 24, 256, 64, "f32", True, False, 4)
    close(*w4_run(x, w, scale, zero, None, 64, "f32"), "f32")
    y, want, _ = w4_run(torch.full((1, 256), 60000.0, dtype=torch.float64), w, scale * 100, zero, None, 64, "f16")
    y = y.double().cpu().numpy()
    big = np.abs(want) > 66000
    assert big.any() and np.isinf(y[big]).all()


# ---- products grouped by expert ---------------------------------------------------------------------------
def grouped_run(sizes, n, k, kind, okind, seed, gather=False, scales=False, bias=False, rs=False, act=0, behind=0, before=0, pads=(0, 0, 0),
                shift=0, ints=False, bad_src=False, short_x=0, offsets=None, stream=None):
    g = torch.Generator().manual_seed(seed)
    e = len(sizes)
    rows = before + sum(sizes) + behind
    off = torch.tensor([0] + sizes).cumsum(0) + before if offsets is None else torch.tensor(offsets)
    xrows = max(1, rows // 3) if gather else rows - short_x
    if kind == "i8":
        x, w = (torch.randint(-127, 128, s, generator=g) for s in ((xrows, k), (e * n, k)))
    elif ints:
        x, w = (torch.randint(-4, 5, s, generator=g).double() for s in ((xrows, k), (e * n, k)))
    else:
        x, w = torch.randn(xrows, k, generator=g, dtype=torch.float64), torch.randn(e * n, k, generator=g, dtype=torch.float64) / k ** 0.5
    xv, _ = rows_of(x, kind, pads[0], shift)
    wv, _ = rows_of(w, kind, pads[1], shift)
    yv, yb = rows_of(torch.full((rows, n), PAD), okind, pads[2], shift)
    y0 = yb.clone()
    src = torch.randint(-2 if bad_src else 0, xrows + (2 if bad_src else 0), (rows,), generator=g, dtype=torch.int32).cuda() if gather else None
    xs = torch.rand(xrows, generator=g).cuda() if scales else None
    ws = torch.rand(e, n, generator=g).cuda() if scales else None
    b = (torch.randint(-9, 10, (e, n), generator=g).float() if ints else torch.randn(e, n, generator=g)).cuda() if bias else None
    r = torch.randn(rows, generator=g).cuda() if rs else None
    ov = off.to(torch.int32).cuda()
    a = capi.GroupedMatmul(x=ptr(xv), y=ptr(yv), w=ptr(wv), offsets=ptr(ov), src=ptr(src), x_scale=ptr(xs), w_scale=ptr(ws), bias=ptr(b), row_scale=ptr(r),
                           ldx=xv.stride(0), ldy=yv.stride(0), ldw=wv.stride(0), w_stride=n * wv.stride(0), rows=rows, x_rows=xrows, experts=e, n=n, k=k,
                           type=KIND[kind], out_type=KIND[okind], act=act)
    call(capi.load().qcnn_op_grouped_matmul, a, stream)
    torch.cuda.synchronize()
    inside = torch.zeros_like(yb, dtype=torch.bool)
    inside[shift:shift + rows * yv.stride(0)].view(rows, -1)[:, :n] = True
    assert torch.equal(yb[~inside], y0[~inside])  # nothing outside the output's rows
    want, bound = np_blocks.grouped_matmul(np64(xv[:, :k]), np64(wv[:, :k]).reshape(e, n, k), off.numpy(), np64(src), np64(xs), np64(ws), np64(b), np64(r), act,
                                           np.full((rows, n), PAD))
    y = yv[:, :n].double().cpu().numpy()
    lo, hi = max(0, int(off[0])), min(rows, int(off[-1]))
    if (off[1:] >= off[:-1]).all():
        assert (y[:lo] == PAD).all() and (y[max(lo, hi):] == PAD).all()  # rows of no expert stay
    return yv[:, :n], want, bound


SIZES = {"one": [1], "none": [0, 0, 0], "few": [1, 0, 2, 5, 0], "mixed": [17, 0, 64, 3, 130, 1], "ragged": [300, 129, 0, 33], "many": [(i * 7) % 5 for i in range(90)]}


@pytest.mark.parametrize("kind", ("f32", "f16", "bf16", "i8"))
@pytest.mark.parametrize("nk", ((1, 1), (32, 48), (17, 33), (64, 64), (130, 200), (256, 128), (100, 513)), ids=str)
@pytest.mark.parametrize("load", SIZES)
def test_grouped_against_the_definition(load, nk, kind):
    n, k = nk
    s = n % 2 == 0
    okind = "f32" if kind == "i8" else kind
    close(*grouped_run(SIZES[load], n, k, kind, okind, n + k, gather=s, scales=kind == "i8", bias=not s, rs=s, act=n % 3, behind=3 * s, before=2 * (not s)), okind)


@pytest.mark.parametrize("kind", ("f32", "f16", "bf16", "i8"))
def test_grouped_integers_are_exact(kind):
    for sizes, n, k in (([5, 0, 40], 33, 100), ([200, 100], 128, 192), ([1] * 20, 64, 1000), ([1000], 72, 64)):
        y, want, _ = grouped_run(sizes, n, k, kind, "f32", n + k, ints=True, bias=True, gather=True)
        assert np.array_equal(y.double().cpu().numpy(), want), (sizes, n, k)


@pytest.mark.parametrize("kind", ("f32", "f16", "bf16", "i8"))
@pytest.mark.parametrize("sizes,n,k", (([1] * 200 + [0, 3], 700, 96), ([20] * 30, 600, 256), ([70, 0, 95, 81], 1100, 200), ([60] * 40, 500, 72),
                                       ([300, 180, 500], 4000, 64), ([2000, 1777, 0, 2600], 4200, 128), ([2100, 1, 1900, 2500], 4100, 130)), ids=str)
def test_grouped_every_kernel(sizes, n, k, kind):
    """Loads on both sides of the launch rules' borders: single rows, a few, dozens and thousands of rows an expert."""
    okind = "bf16" if kind == "i8" else kind
    g = sum(sizes) > 6000
    close(*grouped_run(sizes, n, k, kind, okind, n + k, gather=g, scales=kind == "i8", bias=True, rs=not g, act=1 + g, behind=2, before=3), okind)


@pytest.mark.parametrize("kind,okind", (("f32", "f32"), ("f16", "f16"), ("bf16", "f32"), ("i8", "f32"), ("i8", "bf16")))
@pytest.mark.parametrize("n,k,pads,shift", ((32, 48, (0, 0, 0), 0), (1, 1, (0, 0, 0), 0), (17, 13, (3, 1, 2), 1), (33, 60, (0, 0, 0), 3), (64, 64, (16, 16, 16), 16), (50, 31, (1, 0, 1), 0)))
def test_grouped_many_short_rows(n, k, pads, shift, kind, okind):
    """The 1x1 layers of an image network: many rows of few values."""
    for sizes, act in (([1500, 0, 700, 513], 1), ([2100], 2)):
        for gather in (False, True):
            close(*grouped_run(sizes, n, k, kind, okind, n + k, gather=gather, scales=kind == "i8", bias=True, rs=gather, act=act, behind=5, before=1, pads=pads,
                               shift=shift, bad_src=gather), okind)


@pytest.mark.parametrize("kind,okind", (("i8", "bf16"), ("i8", "f16"), ("f32", "bf16"), ("bf16", "f32"), ("f16", "bf16"), ("f16", "f16")))
@pytest.mark.parametrize("pads,shift", (((0, 0, 0), 1), ((1, 1, 1), 0), ((3, 5, 7), 3), ((16, 16, 16), 16)))
@pytest.mark.parametrize("load", ("few", "mixed"))
def test_grouped_types_strides_and_addresses(load, kind, okind, pads, shift):
    for n, k in ((48, 96), (65, 131), (128, 256)):
        close(*grouped_run(SIZES[load], n, k, kind, okind, n, gather=True, scales=True, bias=True, rs=True, act=2, behind=2, pads=pads, shift=shift), okind, (n, k))


@pytest.mark.parametrize("kind", ("bf16", "i8"))
def test_grouped_rows_outside_x_read_zeros(kind):
    for sizes in ([4, 9, 0, 30], [200, 150]):
        close(*grouped_run(sizes, 40, 128, kind, "f32", 9, gather=True, bad_src=True, bias=True, scales=True), "f32")
        close(*grouped_run(sizes, 40, 128, kind, "f32", 9, bias=True, scales=True, short_x=7), "f32")


@pytest.mark.parametrize("offsets", ([0, 10, 10, 40], [-5, 10, 30, 90], [7, 7, 7, 7], [0, 20, 20, 20], [50, 50, 60, 70], [-9, -8, -3, 0]), ids=str)
def test_grouped_offsets_are_cut_to_the_rows(offsets):
    """sizes give 40 rows; offsets outside are cut off, rows of no expert stay."""
    for kind in ("bf16", "f32"):
        close(*grouped_run([13, 13, 14], 36, 64, kind, "f32", 1, offsets=offsets), "f32")


@pytest.mark.parametrize("kind,n,k", (("i8", 4300, 96), ("f16", 8300, 64), ("bf16", 2304, 96), ("bf16", 2300, 50), ("f32", 6300, 40)))
@pytest.mark.parametrize("sizes", ([1500, 129, 128, 1, 900, 300, 256], [64, 2000, 65, 0, 127, 640, 128]))
def test_grouped_halves_of_tiles(sizes, kind, n, k):
    """Tiles of at most half of their rows, and a last round of few tiles, are made in halves."""
    close(*grouped_run(sizes, n, k, kind, "f32", n + k, gather=True, bias=True, scales=True), "f32")


@pytest.mark.parametrize("kind", ("bf16", "i8", "f32"))
def test_grouped_decreasing_offsets_touch_nothing_else(kind):
    """Offsets that break the contract: rows may hold anything, nothing outside y's rows is written (grouped_run looks)."""
    for sizes, n, k in (([40] * 5, 70, 64), ([700] * 3, 300, 64), ([900] * 3, 30, 48)):
        rows = sum(sizes)
        for off in ([0, rows, 5, rows, 0, rows], [rows, 0, rows, 0, rows, 0], [7, 3, 1, 0, -5, -9]):
            grouped_run(sizes, n, k, kind, "f32", 3, offsets=off[:len(sizes) + 1])


@pytest.mark.parametrize("experts", (64, 65, 300, 1024))
def test_grouped_many_experts(experts):
    """The offsets are summed up 64 experts at a time."""
    sizes = [(i * 7 + 3) % 4 if i % 5 else 0 for i in range(experts)]
    close(*grouped_run(sizes, 40, 32, "bf16", "f32", experts, gather=True, bias=True), "f32")
    sizes = [0] * experts
    sizes[-1], sizes[experts // 2] = 300, 200
    close(*grouped_run(sizes, 136, 64, "f16", "f32", experts, bias=True), "f32")


def test_grouped_nan_stays_in_its_row_and_its_output():
    """A NaN or infinity in a row of x or of w reaches that row's or that output's values alone, whatever kernel runs."""
    for sizes, n, k in (([3, 2], 40, 96), ([70, 90], 200, 64), ([300, 900], 60, 40)):
        g = torch.Generator().manual_seed(n)
        rows, e = sum(sizes), len(sizes)
        x, w = torch.randn(rows, k, generator=g).bfloat16().cuda(), torch.randn(e, n, k, generator=g).bfloat16().cuda()
        x[1, 5], x[rows - 1, k - 1], w[1, 7, 3] = float("nan"), float("inf"), float("nan")
        y = torch.zeros(rows, n, device="cuda")
        off = torch.tensor([0] + sizes).cumsum(0).to(torch.int32).cuda()
        call(capi.load().qcnn_op_grouped_matmul, capi.GroupedMatmul(x=ptr(x), y=ptr(y), w=ptr(w), offsets=ptr(off), ldx=k, ldy=n, ldw=k, w_stride=n * k, rows=rows,
             x_rows=rows, experts=e, n=n, k=k, type=capi.BF16, out_type=capi.F32))
        bad = ~torch.isfinite(y)
        want = torch.zeros_like(bad)
        want[1], want[rows - 1] = True, True
        want[sizes[0]:, 7] = True
        assert torch.equal(bad, want)


def test_half_subnormals_are_multiplied():
    """Half inputs below 2^-14 keep their value in the matrix instructions."""
    x = torch.full((4, 64), 3e-6, dtype=torch.float64)
    w = torch.full((33, 32), 0x99, dtype=torch.uint8)  # codes of 1
    y, want, bound = w4_run(x, w, torch.ones(1, 33, dtype=torch.float64), None, None, 64, "f16", okind="f32")
    close(y, want, bound, "f32")
    assert (y > 1.8e-4).all()
    xh, wh = x.half().cuda(), torch.ones(1, 40, 64, dtype=torch.float16, device="cuda")
    out, off = torch.zeros(4, 40, device="cuda"), torch.tensor([0, 4], dtype=torch.int32, device="cuda")
    call(capi.load().qcnn_op_grouped_matmul, capi.GroupedMatmul(x=ptr(xh), y=ptr(out), w=ptr(wh), offsets=ptr(off), ldx=64, ldy=40, ldw=64, w_stride=40 * 64, rows=4,
         x_rows=4, experts=1, n=40, k=64, type=capi.F16, out_type=capi.F32))
    assert torch.allclose(out, xh.float().sum(1, keepdim=True).expand(4, 40), rtol=1e-5, atol=0)


# ---- addresses beyond 32 bits -----------------------------------------------------------------------------
def test_w4_far_addresses():
    n, k, rows = 70000, 131072, 2  # 4.6 GB of codes
    g = torch.Generator().manual_seed(1)
    w = torch.empty(n, k // 2, dtype=torch.uint8, device="cuda")
    last = torch.randint(0, 256, (3, k // 2), generator=g, dtype=torch.uint8)
    w[-3:] = last.cuda()
    x, s = torch.randn(rows, k, generator=g).bfloat16().cuda(), (torch.rand(k // 128, n, generator=g) / 512).cuda()
    y = torch.zeros(rows, n, device="cuda")
    call(capi.load().qcnn_op_matvec_w4, capi.MatvecW4(x=ptr(x), y=ptr(y), w=ptr(w), scale=ptr(s), ldx=k, ldy=n, ldw=k // 2, rows=rows, n=n, k=k, group=128,
         type=capi.BF16, scale_type=capi.F32, out_type=capi.F32))
    want, bound = np_blocks.matvec_w4(np64(x), last.numpy(), np64(s[:, -3:]), None, None, k, 128)
    close(y[:, -3:], want, bound, "f32")


def test_grouped_far_addresses():
    e, n, k = 40, 8192, 8192  # 5.4 GB of weights; and rows of x and y 2.2 GB apart
    g = torch.Generator().manual_seed(2)
    w = torch.empty(e, n, k, dtype=torch.bfloat16, device="cuda")
    w[-1, -2:] = (torch.randn(2, k, generator=g) / 64).bfloat16().cuda()
    x = torch.empty(3, 1 << 30, dtype=torch.bfloat16, device="cuda")
    x[:, :k] = torch.randn(3, k, generator=g).bfloat16().cuda()
    y = torch.empty(3, 1 << 30, dtype=torch.bfloat16, device="cuda")
    off = torch.zeros(e + 1, dtype=torch.int32, device="cuda")
    off[-1] = 3
    call(capi.load().qcnn_op_grouped_matmul, capi.GroupedMatmul(x=ptr(x), y=ptr(y), w=ptr(w), offsets=ptr(off), ldx=1 << 30, ldy=1 << 30, ldw=k, w_stride=n * k, rows=3,
         x_rows=3, experts=e, n=n, k=k, type=capi.BF16, out_type=capi.BF16))
    want, bound = np_blocks.grouped_matmul(np64(x[:, :k]), np64(w[-1:, -2:]), [0, 3], None, None, None, None, None, 0, np.zeros((3, 2)))
    close(y[:, n - 2:n], want, bound, "bf16")


def test_norm_far_addresses():
    rows, d = 40000, 65536  # 5.2 GB a buffer
    x, n = (torch.empty(rows, d, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    x[-1] = torch.randn(d, generator=torch.Generator().manual_seed(3)).bfloat16().cuda()
    call(capi.load().qcnn_op_norm_res, capi.NormRes(x=ptr(x), n=ptr(n), ldx=d, ldn=d, rows=rows, d=d, parts=1, type=capi.BF16, w_type=capi.F32, pre=1, beta=1.0,
         pre_eps=1e-6))
    _, _, want, bound = np_blocks.norm_res(np64(x[-1:]), None, None, None, 1, 0, None, None, 1, None, None, 0, 0, 1, 0, 1e-6, 0)
    close(n[-1:], want, bound, "bf16")


# ---- the two ends of a residual block ---------------------------------------------------------------------
def norm_run(rows, d, kind, wkind, post, pre, seed, gate=0, act=0, parts=0, alpha=0.8, beta=1.0, w_offset=0.0, eps=1e-6, pads=0, shift=0, weights=True,
             with_y=True, out="hn", bad=False, over="", stream=None, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    normal = lambda *s: torch.randn(*s, generator=g, dtype=torch.float64)  # noqa: E731
    yrows = rows * max(1, parts)
    xv, xb = rows_of(normal(rows, d) * scale, kind, pads, shift)
    yv, _ = rows_of(normal(yrows, d) * scale, kind, pads, shift) if with_y else (None, None)
    gv, _ = rows_of(normal(-(-rows // gate), d), kind, pads, shift) if gate else (None, None)
    index = torch.randint(-1 if bad else 0, yrows + (1 if bad else 0), (rows, parts), generator=g, dtype=torch.int32).cuda() if parts else None
    vec = lambda at: (1 + 0.3 * normal(d) if at == "w" else 0.3 * normal(d)).to(T[wkind]).cuda() if weights else None  # noqa: E731
    pw, pb, nw, nb = vec("w"), vec("b"), vec("w"), vec("b")
    want = np_blocks.norm_res(np64(xv[:, :d]), np64(yv[:, :d]) if with_y else None, np64(index), np64(gv[:, :d]) if gate else None, max(1, gate), post, np64(pw),
                              np64(pb), pre, np64(nw), np64(nb), act, alpha, beta, eps, eps, w_offset)
    outs = {o: rows_of(torch.full((rows, d), PAD), kind, pads, shift) for o in out}
    for o, at in zip(over[0::2], over[1::2]):  # "hx": h over x
        outs[o] = (xv, xb) if at == "x" else (yv, None)
    h, n = (outs.get(o, (None, None))[0] for o in "hn")
    a = capi.NormRes(x=ptr(xv), y=ptr(yv), index=ptr(index), gate=ptr(gv), post_w=ptr(pw), post_b=ptr(pb), pre_w=ptr(nw), pre_b=ptr(nb), h=ptr(h), n=ptr(n),
                     ldx=d + pads, ldy=d + pads, ldg=d + pads, ldh=d + pads, ldn=d + pads, rows=rows, y_rows=yrows, d=d, parts=max(1, parts),
                     gate_rows=max(1, gate), type=KIND[kind], w_type=KIND[wkind], post=post, pre=pre, act=act, alpha=alpha, beta=beta, post_eps=eps,
                     pre_eps=eps, w_offset=w_offset)
    call(capi.load().qcnn_op_norm_res, a, stream)
    torch.cuda.synchronize()
    for v, buf in outs.values():
        if buf is not None:
            assert (v[:, d:].double() == PAD).all() and (buf[:shift].double() == PAD).all() and (buf[shift + v.numel():].double() == PAD).all()
    for o, (w, b) in zip("hn", (want[:2], want[2:])):
        if o in out:
            close(outs[o][0][:, :d], w, b, kind, o)
    return a


ROW_LENGTHS = (1, 2, 7, 8, 15, 16, 33, 64, 100, 128, 255, 257, 512, 768, 1001, 1024, 2048, 2500, 4096, 5000, 8192, 10000, 16384, 20001, 32768, 65536)


@pytest.mark.parametrize("kind", ("f32", "f16", "bf16"))
@pytest.mark.parametrize("d", ROW_LENGTHS)
def test_norm_row_lengths(d, kind):
    """Layer norms of one value or equal values divide by sqrt(eps): eps is 1e-2 there."""
    eps = 1e-2 if d < 8 else 1e-6
    for i, (post, pre) in enumerate(((1, 1), (2, 2), (0, 1), (1, 0))):
        norm_run((1, 3, 5, 9)[i], d, kind, ("f32", kind)[i % 2], post, pre, d + i, gate=(0, 1, 2, 100)[i], act=i, parts=(0, 0, 3, 0)[i], eps=eps)


@pytest.mark.parametrize("kind", ("f32", "bf16"))
@pytest.mark.parametrize("rows", (1, 2, 31, 32, 33, 512, 513, 1000))
def test_norm_row_counts(rows, kind):
    """512 rows, and with them outputs of 8 MB, are borders of the launch rules."""
    for d in (40, 130, 600, 1025, 3000, 6001):
        norm_run(rows, d, kind, "f32", 2, 1, rows + d, gate=3, act=1, parts=2)


@pytest.mark.parametrize("kind", ("f32", "f16", "bf16"))
@pytest.mark.parametrize("pads,shift", ((0, 1), (1, 0), (3, 5), (8, 8)))
def test_norm_strides_and_addresses(kind, pads, shift):
    for d in (63, 64, 515, 1024, 3000):
        norm_run(6, d, kind, kind, 1, 2, d, gate=1, act=3, parts=0, pads=pads, shift=shift)
        norm_run(6, d, kind, "f32", 1, 2, d, gate=4, act=2, parts=5, pads=pads, shift=shift, bad=True)


@pytest.mark.parametrize("kind", ("f32", "bf16"))
def test_norm_parts_left_out(kind):
    for d in (24, 1000):
        norm_run(5, d, kind, kind, 1, 1, 1, weights=False)                        # no weights
        norm_run(5, d, kind, kind, 1, 1, 2, w_offset=1.0)                         # weights stored as a distance from 1
        norm_run(5, d, kind, kind, 1, 2, 3, with_y=False, beta=0.5)               # no block: scale and norm alone
        norm_run(5, d, kind, kind, 2, 0, 4, out="h")                              # the residual alone
        norm_run(5, d, kind, kind, 0, 1, 5, out="n")                              # the norm alone
        norm_run(5, d, kind, kind, 0, 0, 6, alpha=-0.25, beta=2.0)                # no norms
        norm_run(5, d, kind, kind, 2, 1, 7, parts=64, bad=True)                   # many parts, some outside


@pytest.mark.parametrize("over", ("hx", "hy", "hxny", "nxhy", "nx", "ny"))
def test_norm_in_place(over):
    for d in (64, 777, 4096, 30000):
        norm_run(7, d, "bf16", "f32", 1, 1, d, gate=2, act=1, over=over)


def test_norm_far_from_zero():
    """Rows far from zero: the variance comes from the distances, not from a difference of large numbers."""
    for d in (100, 4096):
        g = torch.Generator().manual_seed(d)
        x = (1000 + torch.randn(4, d, generator=g)).float().cuda()
        n = torch.empty_like(x)
        a = capi.NormRes(x=ptr(x), n=ptr(n), ldx=d, ldn=d, rows=4, d=d, parts=1, type=capi.F32, w_type=capi.F32, pre=2, beta=1.0, pre_eps=1e-5)
        call(capi.load().qcnn_op_norm_res, a)
        _, _, want, bound = np_blocks.norm_res(np64(x), None, None, None, 1, 0, None, None, 2, None, None, 0, 0, 1, 0, 1e-5, 0)
        close(n, want, bound, "f32")
        if d == 100:  # the mean's error d U 1000 counts about four times: 0.024; the bound is far below the values there
            assert bound.max() < 0.2


# ---- streams, graphs, a block of all three -----------------------------------------------------------------
def block_state(seed, tokens=6, d=256, hid=192, experts=5, top=2):
    """An expert block and the 4-bit projection behind it: norm -> up -> down -> sum, gate, residual, norm -> projection."""
    g = torch.Generator().manual_seed(seed)
    n = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    s = {"x": n(tokens, d).bfloat16().cuda(), "v": (0.1 * n(tokens, d)).bfloat16().cuda()}
    s["w1"], s["w2"] = (n(experts, hid, d) / d ** 0.5).bfloat16().cuda(), (n(experts, d, hid) / hid ** 0.5).bfloat16().cuda()
    pick = torch.stack([torch.randperm(experts, generator=g)[:top] for _ in range(tokens)])
    order = pick.flatten().argsort(stable=True)
    s["offsets"] = torch.cat((torch.zeros(1), torch.bincount(pick.flatten(), minlength=experts).cumsum(0))).to(torch.int32).cuda()
    s["src"] = (order // top).to(torch.int32).cuda()
    place = torch.empty(tokens * top, dtype=torch.int32)
    place[order] = torch.arange(tokens * top, dtype=torch.int32)
    s["place"] = place.view(tokens, top).cuda()
    s["prob"] = torch.rand(tokens * top, generator=g).cuda()
    s["nw"], s["gate"] = (1 + 0.1 * n(d)).cuda(), n(1, d).bfloat16().cuda()
    s["q"] = torch.randint(0, 256, (130, d // 2), generator=g, dtype=torch.uint8).cuda()
    s["qs"] = (torch.rand(d // 64, 130, generator=g) / 64).bfloat16().cuda()
    for name, shape in (("h0", (tokens, d)), ("n0", (tokens, d)), ("u", (tokens * top, hid)), ("o", (tokens * top, d)), ("h", (tokens, d)), ("n", (tokens, d)),
                        ("y", (tokens, 130))):
        s[name] = torch.zeros(shape, dtype=torch.bfloat16, device="cuda")
    s["dims"] = (tokens, d, hid, experts, top)
    return s


def block_calls(s, stream):
    lib = capi.load()
    tokens, d, hid, experts, top = s["dims"]
    rows = tokens * top
    b = capi.BF16
    call(lib.qcnn_op_norm_res, capi.NormRes(x=ptr(s["x"]), y=ptr(s["v"]), pre_w=ptr(s["nw"]), h=ptr(s["h0"]), n=ptr(s["n0"]), ldx=d, ldy=d, ldh=d, ldn=d, rows=tokens,
         y_rows=tokens, d=d, parts=1, type=b, w_type=capi.F32, pre=1, alpha=1.0, beta=1.0, pre_eps=1e-6), stream)
    call(lib.qcnn_op_grouped_matmul, capi.GroupedMatmul(x=ptr(s["n0"]), y=ptr(s["u"]), w=ptr(s["w1"]), offsets=ptr(s["offsets"]), src=ptr(s["src"]), ldx=d, ldy=hid,
         ldw=d, w_stride=hid * d, rows=rows, x_rows=tokens, experts=experts, n=hid, k=d, type=b, out_type=b, act=capi.ACT_SILU), stream)
    call(lib.qcnn_op_grouped_matmul, capi.GroupedMatmul(x=ptr(s["u"]), y=ptr(s["o"]), w=ptr(s["w2"]), offsets=ptr(s["offsets"]), row_scale=ptr(s["prob"]), ldx=hid,
         ldy=d, ldw=hid, w_stride=hid * d, rows=rows, x_rows=rows, experts=experts, n=d, k=hid, type=b, out_type=b), stream)
    call(lib.qcnn_op_norm_res, capi.NormRes(x=ptr(s["h0"]), y=ptr(s["o"]), index=ptr(s["place"]), gate=ptr(s["gate"]), pre_w=ptr(s["nw"]), post_w=ptr(s["nw"]),
         h=ptr(s["h"]), n=ptr(s["n"]), ldx=d, ldy=d, ldg=d, ldh=d, ldn=d, rows=tokens, y_rows=rows, d=d, parts=top, gate_rows=tokens, type=b, w_type=capi.F32, post=1,
         pre=1, act=1, alpha=0.5, beta=1.0, post_eps=1e-6, pre_eps=1e-6), stream)
    call(lib.qcnn_op_matvec_w4, capi.MatvecW4(x=ptr(s["n"]), y=ptr(s["y"]), w=ptr(s["q"]), scale=ptr(s["qs"]), ldx=d, ldy=130, ldw=d // 2, rows=tokens, n=130, k=d,
         group=64, type=b, scale_type=b, out_type=b), stream)


def block_check(s):
    """Each step against the definition on the step's own inputs."""
    tokens, d, hid, experts, top = s["dims"]
    v = {k: np64(t) for k, t in s.items() if k != "dims"}
    h, bh, n, bn = np_blocks.norm_res(v["x"], v["v"], None, None, 1, 0, None, None, 1, v["nw"], None, 0, 1, 1, 0, 1e-6, 0)
    close(s["h0"], h, bh, "bf16", "h0"), close(s["n0"], n, bn, "bf16", "n0")
    close(s["u"], *np_blocks.grouped_matmul(v["n0"], v["w1"], v["offsets"], v["src"], None, None, None, None, 2, v["u"]), "bf16", "up")
    close(s["o"], *np_blocks.grouped_matmul(v["u"], v["w2"], v["offsets"], None, None, None, None, v["prob"], 0, v["o"]), "bf16", "down")
    h, bh, n, bn = np_blocks.norm_res(v["h0"], v["o"], v["place"], v["gate"], tokens, 1, v["nw"], None, 1, v["nw"], None, 1, 0.5, 1, 1e-6, 1e-6, 0)
    close(s["h"], h, bh, "bf16", "h"), close(s["n"], n, bn, "bf16", "n")
    close(s["y"], *np_blocks.matvec_w4(v["n"], v["q"], v["qs"], None, None, d, 64), "bf16", "y")


def test_a_block_of_all_three():
    for seed, tokens in ((1, 1), (2, 6), (3, 200)):
        s = block_state(seed, tokens)
        block_calls(s, None)
        torch.cuda.synchronize()
        block_check(s)


def test_a_block_on_two_streams_at_once():
    states = [block_state(20 + i, 40) for i in range(2)]
    streams = [torch.cuda.Stream() for _ in states]
    torch.cuda.synchronize()
    for _ in range(5):
        for s, st in zip(states, streams):
            block_calls(s, st.cuda_stream)
    torch.cuda.synchronize()
    for s in states:
        block_check(s)


def test_a_block_captured_and_replayed():
    """Replays see new inputs, other offsets among them, and give the eager call's bits; eager work runs in between."""
    s = block_state(30, 12)
    block_calls(s, None)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        block_calls(s, torch.cuda.current_stream().cuda_stream)
    for seed in (31, 32, 33):
        other = block_state(seed, 12)
        for k, t in other.items():
            if k in ("x", "v", "offsets", "src", "place", "prob", "gate"):
                s[k].copy_(t)
            elif k not in ("dims", "h0", "n0", "u", "o", "h", "n", "y"):
                other[k] = s[k]  # the graph's own weights
        g.replay()
        torch.cuda.synchronize()
        block_check(s)
        block_calls(other, None)
        torch.cuda.synchronize()
        for k in ("h0", "n0", "u", "o", "h", "n", "y"):
            assert torch.equal(other[k], s[k]), k


def test_a_block_from_threads_at_once():
    """Four host threads, each with a stream and buffers of its own, also through the kernels that ask for more LDS."""
    states = [block_state(50 + i, 400 if i % 2 else 9) for i in range(4)]
    streams, errors = [torch.cuda.Stream() for _ in states], []
    torch.cuda.synchronize()

    def work(s, st):
        try:
            for _ in range(10):
                block_calls(s, st.cuda_stream)
            st.synchronize()
        except Exception as e:
            errors.append(e)

    threads = [threading.Thread(target=work, args=a) for a in zip(states, streams)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors
    for s in states:
        block_check(s)


def test_two_graphs_replayed_at_once():
    states, graphs, streams = [block_state(60 + i, 60) for i in range(2)], [], [torch.cuda.Stream() for _ in range(2)]
    for s in states:
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            block_calls(s, torch.cuda.current_stream().cuda_stream)
    torch.cuda.synchronize()
    for _ in range(4):
        for g, st in zip(graphs, streams):
            with torch.cuda.stream(st):
                g.replay()
        block_calls(block_state(70, 5), None)  # eager work between the replays
    torch.cuda.synchronize()
    for s in states:
        block_check(s)


def test_the_first_call_of_a_process_may_be_captured():
    code = ("import sys, torch; sys.path[:0] = ['tests', '.']; import test_gpu_block_ops as t; s = t.block_state(80, 7); g = torch.cuda.CUDAGraph()\n"
            "with torch.cuda.graph(g): t.block_calls(s, torch.cuda.current_stream().cuda_stream)\n"
            "for _ in range(3): g.replay(); torch.cuda.synchronize(); t.block_check(s); t.block_calls(s, None); torch.cuda.synchronize(); t.block_check(s)\n"
            "print('checked')")
    done = subprocess.run([sys.executable, "-c", code], cwd=pathlib.Path(__file__).resolve().parents[1], capture_output=True, text=True, timeout=100)
    assert done.returncode == 0 and done.stdout.strip().endswith("checked"), done.stderr[-2000:]


def test_the_same_call_gives_the_same_bits():
    s = block_state(40, 300)
    block_calls(s, None)
    first = {k: s[k].clone() for k in ("u", "o", "h", "n", "y")}
    for _ in range(3):
        block_calls(s, None)
        assert all(torch.equal(first[k], s[k]) for k in first)
