"""GPU parity of the operators for blocks of language models at their borders.  Inputs, oracle and tolerances as in
test_gpu_block_ops.py unless a test says otherwise."""
import numpy as np
import pytest
import torch

from oracle import np_blocks
from qcnn_gpu_amd import capi
from test_gpu_block_ops import KIND, T, call, close, grouped_run, np64, ptr, w4_run

pytestmark = pytest.mark.gpu
NAN, INF = float("nan"), float("inf")


# ---- the end of a row between two norms ------------------------------------------------------------------
@pytest.mark.parametrize("kind", ("f32", "f16", "bf16"))
@pytest.mark.parametrize("d", (9, 63, 100, 515, 777, 1001, 4099, 20001))
def test_layer_norm_behind_layer_norm(d, kind):
    """What the first norm makes of the registers behind a row's end (with no weights, or weights as a distance from 1, not zero)
    must not reach the mean of the second.  Inputs far from zero; gates whose value at 0 is not 0 among them."""
    rows = 3
    for seed, (weights, offset, gate, act) in enumerate(((False, 0.0, 0, 0), (False, 0.0, 2, 1), (True, 1.0, 0, 0), (True, 1.0, 1, 1), (True, -0.5, 1, 3))):
        g = torch.Generator().manual_seed(100 * d + seed)
        x, y = (torch.randn(rows, d, generator=g) + m for m in (1.0, 5.0))
        x, y = (v.to(T[kind]).cuda() for v in (x, y))
        gv = torch.randn(-(-rows // gate), d, generator=g).to(T[kind]).cuda() if gate else None
        v = [(0.3 * torch.randn(d, generator=g)).cuda() if weights else None for _ in range(4)]
        h, n = torch.empty_like(x), torch.empty_like(x)
        a = capi.NormRes(x=ptr(x), y=ptr(y), gate=ptr(gv), post_w=ptr(v[0]), post_b=ptr(v[1]), pre_w=ptr(v[2]), pre_b=ptr(v[3]), h=ptr(h), n=ptr(n), ldx=d, ldy=d,
                         ldg=d, ldh=d, ldn=d, rows=rows, y_rows=rows, d=d, parts=1, gate_rows=max(1, gate), type=KIND[kind], w_type=capi.F32,
                         post=capi.NORM_LAYER, pre=capi.NORM_LAYER, act=act, alpha=0.8, beta=1.0, post_eps=1e-5, pre_eps=1e-5, w_offset=offset)
        call(capi.load().qcnn_op_norm_res, a)
        want = np_blocks.norm_res(np64(x), np64(y), None, np64(gv), max(1, gate), 2, *map(np64, v[:2]), 2, *map(np64, v[2:]), act, 0.8, 1.0, 1e-5, 1e-5, offset)
        close(h, want[0], want[1], kind, ("h", seed))
        close(n, want[2], want[3], kind, ("n", seed))


# ---- rows that are not there, scales that are not finite -------------------------------------------------
@pytest.mark.parametrize("kind", ("bf16", "i8"))
@pytest.mark.parametrize("sizes,n,k", (([3, 5], 40, 96), ([4] * 40, 300, 700), ([20] * 30, 600, 256), ([20] * 30, 600, 600), ([300, 200], 200, 130), ([300, 200, 400], 900, 130), ([600], 32, 48)), ids=str)
def test_grouped_rows_outside_x_whatever_the_scales_hold(sizes, n, k, kind):
    """Of a row whose src is outside x, activation and row scale of the bias are left, in every kernel: infinite or NaN weights and
    scales are not multiplied with its zeros."""
    g = torch.Generator().manual_seed(n)
    e, rows = len(sizes), sum(sizes)
    draw = (lambda *s: torch.randint(-9, 10, s, generator=g).to(torch.int8)) if kind == "i8" else (lambda *s: torch.randn(*s, generator=g).bfloat16())
    x, w, bias = draw(rows, k).cuda(), draw(e, n, k), torch.randn(e, n, generator=g)
    ws, rs = torch.rand(e, n, generator=g), torch.rand(rows, generator=g)
    ws[:, 2], ws[:, 7] = INF, NAN
    if kind == "bf16":
        w[:, 4] = NAN
    src = torch.arange(rows, dtype=torch.int32)
    src[::3] = torch.tensor([-1, rows, 2 ** 31 - 1], dtype=torch.int32)[torch.arange(len(src[::3])) % 3]
    of = torch.repeat_interleave(torch.arange(e), torch.tensor(sizes))
    w, src, ws, bias_d, rs_d = (t.cuda() for t in (w, src, ws, bias, rs))
    xs, off = torch.rand(rows, generator=g).cuda(), torch.tensor([0] + sizes).cumsum(0).to(torch.int32).cuda()
    y = torch.zeros(rows, n, device="cuda")
    call(capi.load().qcnn_op_grouped_matmul, capi.GroupedMatmul(x=ptr(x), y=ptr(y), w=ptr(w), offsets=ptr(off), src=ptr(src), x_scale=ptr(xs), w_scale=ptr(ws),
         bias=ptr(bias_d), row_scale=ptr(rs_d), ldx=k, ldy=n, ldw=k, w_stride=n * k, rows=rows, x_rows=rows, experts=e, n=n, k=k, type=KIND[kind],
         out_type=capi.F32, act=capi.ACT_RELU))
    assert torch.equal(y[::3].cpu(), (bias[of].clamp_min(0) * rs[:, None])[::3])
    assert torch.isfinite(y[1::3][:, :2]).all() and torch.isnan(y[1::3][:, 7]).all()


@pytest.mark.parametrize("kind", ("f32", "bf16", "i8"))
@pytest.mark.parametrize("sizes,n,k", (([3, 5], 40, 96), ([300, 200, 400], 900, 130), ([300, 200, 400], 900, 128), ([600], 32, 48)), ids=str)
def test_grouped_without_any_row_of_x(sizes, n, k, kind):
    """x_rows = 0: x is not looked at."""
    e, rows = len(sizes), sum(sizes)
    w, bias = torch.ones(e, n, k, device="cuda").to(T[kind]), torch.randn(e, n, device="cuda")
    off, y = torch.tensor([0] + sizes).cumsum(0).to(torch.int32).cuda(), torch.zeros(rows, n, device="cuda")
    call(capi.load().qcnn_op_grouped_matmul, capi.GroupedMatmul(y=ptr(y), w=ptr(w), offsets=ptr(off), bias=ptr(bias), ldx=k, ldy=n, ldw=k, w_stride=n * k,
         rows=rows, experts=e, n=n, k=k, type=KIND[kind], out_type=capi.F32))
    assert torch.equal(y, bias.repeat_interleave(torch.tensor(sizes, device="cuda"), 0))


@pytest.mark.parametrize("kind", ("f32", "f16", "bf16"))
@pytest.mark.parametrize("zeros", (False, True))
@pytest.mark.parametrize("rows,k,group", ((1, 40, 32), (3, 33, 32), (2, 170, 64), (18, 330, 96), (40, 65, 64)))
def test_w4_infinite_scale_of_the_last_group(rows, k, group, zeros, kind):
    """The groups that a run of 128 k has behind the last one add nothing, also where the last one's scale is infinite."""
    n, ng = 21, -(-k // group)
    g = torch.Generator().manual_seed(k)
    x = torch.randint(1, 4, (rows, k), generator=g).double()
    codes = torch.randint(9, 16, (n, k + 1), generator=g, dtype=torch.uint8)
    w = codes[:, 0:(k + 1) // 2 * 2:2] | codes[:, 1:(k + 1) // 2 * 2:2] << 4
    scale = torch.ones(ng, n, dtype=torch.float64)
    scale[-1, ::2], scale[-1, 1] = INF, -INF
    zero = torch.full((ng, n), 7, dtype=torch.uint8) if zeros else None
    y, want, _ = w4_run(x, w, scale, zero, None, group, kind, okind="f32")
    assert np.array_equal(y.double().cpu().numpy(), want)


# ---- more workgroups than a launch, or a row of its grid, takes --------------------------------------------
def test_w4_rows_beyond_one_launch():
    """2^28 rows make 2^23 workgroups of 512 threads."""
    rows, n = (1 << 28) + 77, 1
    x = torch.randint(-8, 9, (rows, 1), generator=torch.Generator("cuda").manual_seed(5), device="cuda", dtype=torch.int8).to(torch.bfloat16)
    y = torch.full((rows + 64, n), 77.0, dtype=torch.bfloat16, device="cuda")
    w, s = torch.full((1, 1), 13, dtype=torch.uint8, device="cuda"), torch.full((1, 1), 0.5, device="cuda")
    call(capi.load().qcnn_op_matvec_w4, capi.MatvecW4(x=ptr(x), y=ptr(y), w=ptr(w), scale=ptr(s), ldx=1, ldy=1, ldw=1, rows=rows, n=n, k=1, group=32,
         type=capi.BF16, scale_type=capi.F32, out_type=capi.BF16))
    assert torch.equal(y[:rows], x * 2.5) and (y[rows:] == 77).all()


def test_norm_rows_beyond_one_launch():
    """2^29 rows of one value make 2^24 workgroups of 256 threads."""
    rows = (1 << 29) + 77
    x = torch.randint(-8, 9, (rows,), generator=torch.Generator("cuda").manual_seed(6), device="cuda", dtype=torch.int8).to(torch.bfloat16)
    h = torch.full((rows + 64,), 77.0, dtype=torch.bfloat16, device="cuda")
    call(capi.load().qcnn_op_norm_res, capi.NormRes(x=ptr(x), h=ptr(h), ldx=1, ldh=1, rows=rows, d=1, parts=1, type=capi.BF16, w_type=capi.F32, beta=0.5))
    assert torch.equal(h[:rows], x * 0.5) and (h[rows:] == 77).all()


@pytest.mark.parametrize("gate_rows", (7, (1 << 29) - 5, 1 << 30))
def test_norm_gates_and_indices_beyond_one_launch(gate_rows):
    """A launch takes 2^29 - 32 rows of one value: rows of gate that end before its end, behind it and never."""
    rows = (1 << 29) + 77
    g = torch.Generator("cuda").manual_seed(gate_rows)
    x, y = (torch.randint(-8, 9, (rows,), generator=g, device="cuda", dtype=torch.int8).to(torch.bfloat16) for _ in range(2))
    gate = torch.randint(-4, 5, (-(-rows // gate_rows),), generator=g, device="cuda", dtype=torch.int8).to(torch.bfloat16)
    index = torch.arange(rows - 1, -1, -1, device="cuda", dtype=torch.int32)
    n = torch.empty_like(x)
    want = x + y.flip(0) * gate.repeat_interleave(gate_rows)[:rows]
    call(capi.load().qcnn_op_norm_res, capi.NormRes(x=ptr(x), y=ptr(y), index=ptr(index), gate=ptr(gate), h=ptr(x), n=ptr(n), ldx=1, ldy=1, ldg=1, ldh=1, ldn=1, rows=rows,
         y_rows=rows, d=1, parts=1, gate_rows=gate_rows, type=capi.BF16, w_type=capi.F32, alpha=1.0, beta=1.0))
    assert torch.equal(x, want) and torch.equal(n, want)
    y0 = y.clone()
    call(capi.load().qcnn_op_norm_res, capi.NormRes(x=ptr(x), y=ptr(y), h=ptr(y), n=ptr(n), ldx=1, ldy=1, ldh=1, ldn=1, rows=rows, y_rows=rows, d=1, parts=1,
         type=capi.BF16, w_type=capi.F32, alpha=1.0, beta=0.0, pre=capi.NORM_LAYER, pre_eps=1.0))
    assert torch.equal(y, y0) and (n == 0).all()


def test_grouped_tiles_beyond_one_launch():
    """One row for each of 32 experts with 2^25 outputs: 2^24 and more workgroups of 256 threads."""
    e, n = 32, 1 << 25
    g = torch.Generator("cuda").manual_seed(7)
    w = torch.randint(-8, 9, (e, n), generator=g, device="cuda", dtype=torch.int8)
    x = torch.arange(1, e + 1, device="cuda", dtype=torch.int8).view(e, 1)
    y, off = torch.full((e + 1, n), 77.0, dtype=torch.float16, device="cuda"), torch.arange(e + 1, dtype=torch.int32, device="cuda")
    call(capi.load().qcnn_op_grouped_matmul, capi.GroupedMatmul(x=ptr(x), y=ptr(y), w=ptr(w), offsets=ptr(off), ldx=1, ldy=n, ldw=1, w_stride=n, rows=e, x_rows=e,
         experts=e, n=n, k=1, type=capi.I8, out_type=capi.F16))
    assert torch.equal(y[:e], w.half() * x.half()) and (y[e:] == 77).all()


# ---- the loops of the tile kernels -----------------------------------------------------------------------
def tile_of(sizes, n, k, kind, aligned=True):
    """The launch rules of kernels_grouped.hip for calls that reach a tile kernel: its height and width (None: another kernel)."""
    z = T[kind].itemsize
    rows, e = sum(sizes), len(sizes)
    avg = rows // e

    def tiles(t):
        return (rows // t + min(rows, e)) * -(-n // t)
    if (n <= 64 and k * z <= 256 and avg >= 512) or tiles(32) < 128 or avg <= 24 or tiles(64) < (160 if z == 4 else 64):
        return None
    if tiles(128) < (1024 if z == 4 else 256):
        return 64
    if z < 4 and aligned and k * z % 16 == 0 and avg >= 256 and tiles(256) >= (240 if k >= 2048 else 512):
        return 256
    return 128


def tile_run(sizes, n, k, kind, seed, gather):
    """Small whole numbers, sums below 2^24: every kernel's result is exact and equal to the product in 64 bits."""
    g = torch.Generator("cuda").manual_seed(seed)
    e, rows = len(sizes), sum(sizes)
    whole = lambda *s: torch.randint(-3, 4, s, generator=g, device="cuda", dtype=torch.int8)  # noqa: E731
    xrows = rows // 2 if gather else rows
    x, w = whole(xrows, k), whole(e, n, k)
    src = torch.randint(0, xrows, (rows,), generator=g, device="cuda", dtype=torch.int32) if gather else None
    xt, wt = x.to(T[kind]), w.to(T[kind])
    off = torch.tensor([0] + sizes).cumsum(0).to(torch.int32).cuda()
    y = torch.full((rows + 5, n), 77.0, device="cuda")
    call(capi.load().qcnn_op_grouped_matmul, capi.GroupedMatmul(x=ptr(xt), y=ptr(y), w=ptr(wt), offsets=ptr(off), src=ptr(src), ldx=k, ldy=n, ldw=k, w_stride=n * k,
         rows=rows, x_rows=xrows, experts=e, n=n, k=k, type=KIND[kind], out_type=capi.F32))
    at = 0
    for i, c in enumerate(sizes):
        if c:
            v = x[src[at:at + c].long()] if gather else x[at:at + c]
            assert torch.equal(y[at:at + c].double(), v.double() @ w[i].double().t()), (i, kind, n, k)
        at += c
    assert (y[rows:] == 77).all()


# by float32 rows and tile: rows of the experts, outputs; and bytes of k: fewer steps of 64 than the loop begins with, the loop once, its end with one and two steps over, an unfinished step
LOADS = {(False, 64): ([150, 0, 33, 260, 64], 420), (False, 128): ([700, 129, 0, 1200, 64, 128], 2100), (False, 256): ([3000, 257, 1, 4200, 0, 900, 128], 4100),
         (True, 64): ([150, 0, 33, 260, 64], 1000), (True, 128): ([3000, 129, 0, 3100, 64, 128], 2450)}
STEPS = (64, 320, 384, 448, 512, 528, 1024, 1040)


@pytest.mark.parametrize("kind", ("f32", "f16", "bf16", "i8"))
@pytest.mark.parametrize("tile", (64, 128, 256))
@pytest.mark.parametrize("gather", (False, True))
def test_grouped_tile_loops(tile, kind, gather):
    """Every length of the loop over k in every tile kernel; loads that leave short tiles, halves, and several tiles to a workgroup."""
    if tile == 256 and kind == "f32":
        assert tile_of([9000], 9000, 512, kind) == 128  # float32 has no such tiles
        return
    sizes, n = LOADS[kind == "f32", tile]
    z = T[kind].itemsize
    for i, bytes_ in enumerate(STEPS):
        k = bytes_ // z
        assert tile_of(sizes, n, k, kind) == tile, (k, tile_of(sizes, n, k, kind))
        tile_run(sizes, n, k, kind, 10 * tile + i, gather)


@pytest.mark.parametrize("kind", ("f16", "bf16", "i8"))
def test_grouped_large_tiles_by_long_k(kind):
    """240 tiles are enough for 256 x 256 from k = 2048 on; below, 128 x 128."""
    sizes, n = [1000, 2000, 300, 700], 3100
    assert [tile_of(sizes, n, k, kind) for k in (2032, 2048, 2080)] == [128, 256, 256]
    for k in (2032, 2048, 2080):
        tile_run(sizes, n, k, kind, k, False)


@pytest.mark.parametrize("kind", ("f32", "f16", "bf16", "i8"))
def test_grouped_tile_loops_of_unaligned_rows(kind):
    """Rows that are no whole chunks go through registers: 64 x 64 and 128 x 128 tiles alone."""
    z = T[kind].itemsize
    for tile in (64, 128):
        sizes, n = LOADS[kind == "f32", tile]
        for k in (1, 63 // z, 64 // z + 1, 130 // z + 1, 200 // z + 1, 600 // z + 1):
            if k * z % 16 == 0:
                k += 1
            assert tile_of(sizes, n, k, kind) == tile
            tile_run(sizes, n, k, kind, 7 * k, k % 2 == 0)


# ---- the size of the rounding error at a model's row lengths ---------------------------------------------
# The bound that holds for every input grows with k times the sum of the magnitudes, far above what random inputs show.  These
# tests look at the root mean square over the outputs.  An addition in float32 is off by at most U of its result, U / sqrt(3) at
# most in the mean; of N additions in a row of terms of rms t the j-th result is about sqrt(j) t, so that the sum is off by
# U t sqrt(sum j / 3) <= U sqrt(N / 6) * (sqrt(N) t): U sqrt(N / 6) times the L2 norm of the terms.  Other orders of the sum have
# shorter chains.  Twice that is allowed, and one rounding of the result.
U = np_blocks.U


def rms(v):
    return float(np.sqrt(np.mean(np.square(v))))


@pytest.mark.parametrize("kind", ("f32", "f16", "bf16"))
@pytest.mark.parametrize("rows,n,k,group", ((1, 512, 4096, 128), (16, 300, 4096, 64), (48, 200, 8192, 32), (4, 400, 16384, 16384)))
def test_w4_error_of_long_rows(rows, n, k, group, kind):
    g = torch.Generator().manual_seed(k + rows)
    x = torch.randn(rows, k, generator=g, dtype=torch.float64)
    w = torch.randint(0, 256, (n, k // 2), generator=g, dtype=torch.uint8)
    scale = (0.5 + torch.rand(k // group, n, generator=g, dtype=torch.float64)) / k ** 0.5
    zero = torch.randint(0, 16, (k // group, n), generator=g, dtype=torch.uint8)
    y, want, _ = w4_run(x, w, scale, zero, None, group, kind, skind="f32", okind="f32")
    x = x.to(T[kind]).double().numpy()
    q = np.stack((w.numpy() & 15, w.numpy() >> 4), -1).reshape(n, k).astype(np.float64)
    s = np.repeat(scale.float().double().numpy(), group, 0).T
    z = np.repeat(zero.numpy().astype(np.float64), group, 0).T

    def l2(of):  # of the terms of each output
        return np.sqrt(np.square(x) @ np.square(s * of).T)
    add = -8.0 if kind == "f32" else 16.0  # what the codes are summed with, and what is taken off again
    chain = group * (3 if kind == "f32" else 1)  # float32 rows: three parts of each value
    tol = 2 * U * (np.sqrt(chain / 6) * np.hypot(l2(q + add), l2(z + add)) + np.sqrt(k / group / 6) * l2(q - z)) + U * np.abs(want) + 2 * U * l2(q + add)
    assert rms(y.double().cpu().numpy() - want) <= rms(tol)


@pytest.mark.parametrize("kind", ("f32", "f16", "bf16"))
@pytest.mark.parametrize("sizes,n,k", (([2, 1, 0, 3], 300, 4096), ([20] * 8, 256, 8192), ([300, 200], 500, 4096), ([1200, 848], 1100, 2048)), ids=str)
def test_grouped_error_of_long_rows(sizes, n, k, kind):
    y, want, _ = grouped_run(sizes, n, k, kind, "f32", k + n)
    g = torch.Generator().manual_seed(k + n)  # the inputs that grouped_run made
    rows, e = sum(sizes), len(sizes)
    x, w = torch.randn(rows, k, generator=g, dtype=torch.float64), torch.randn(e * n, k, generator=g, dtype=torch.float64) / k ** 0.5
    x, w = (t.to(T[kind]).double().square() for t in (x, w.view(e, n, k)))
    l2 = torch.cat([p @ v.t() for p, v in zip(x.split(sizes), w)]).sqrt().numpy()
    assert rms(y.double().cpu().numpy() - want) <= rms(2 * U * np.sqrt(k / 6) * l2 + U * np.abs(want))


def test_w4_float32_rows_of_small_values():
    """A float32 value goes in as three bfloat16 parts, so as a multiple of 2^-133: full precision from 2^-109 on, below that off by
    at most 2^-133 of every value times what it is multiplied with."""
    for shift in (-100, -108, -115, -122, -130):
        g = torch.Generator().manual_seed(-shift)
        x = torch.randn(4, 256, generator=g, dtype=torch.float64)
        x = torch.where(x.abs() < 0.5, x.sign() * 0.5 + x / 2, x) * 2.0 ** shift  # at least 2^(shift - 1)
        w = torch.randint(0, 256, (48, 128), generator=g, dtype=torch.uint8)
        scale, zero = (torch.rand(4, 48, generator=g) + 0.5).double(), torch.randint(0, 16, (4, 48), generator=g, dtype=torch.uint8)
        y, want, bound = w4_run(x, w, scale, zero, None, 64, "f32")
        q = np.stack((w.numpy() & 15, w.numpy() >> 4), -1).reshape(48, 256).astype(np.float64)
        size = (scale.float().double().repeat_interleave(64, 0).T.numpy() * (np.abs(q - 8) + np.abs(zero.repeat_interleave(64, 0).T.double().numpy() - 8))).sum(1)
        close(y, want, bound + (2.0 ** -133 * size[None, :] if shift < -108 else 0), "f32", shift)


# ---- the largest values and sizes of single arguments ----------------------------------------------------
def test_grouped_int8_sums_at_the_end_of_int32():
    """k = 131071 times 128 * 128 is the largest sum an int32 holds; in the kernels that split k and in those that do not."""
    k = 131071
    for sizes, n in (([2], 5), ([130, 120], 300), ([700], 1200)):
        e, rows = len(sizes), sum(sizes)
        x, w = torch.full((rows, k), -128, dtype=torch.int8, device="cuda"), torch.full((e, n, k), -128, dtype=torch.int8, device="cuda")
        w[:, 1] = 127
        off, y = torch.tensor([0] + sizes).cumsum(0).to(torch.int32).cuda(), torch.zeros(rows, n, device="cuda")
        call(capi.load().qcnn_op_grouped_matmul, capi.GroupedMatmul(x=ptr(x), y=ptr(y), w=ptr(w), offsets=ptr(off), ldx=k, ldy=n, ldw=k, w_stride=n * k, rows=rows,
             x_rows=rows, experts=e, n=n, k=k, type=capi.I8, out_type=capi.F32))
        want = torch.full((n,), float(k * 128 * 128), device="cuda")
        want[1] = float(-k * 128 * 127)
        assert torch.equal(y, want.expand(rows, n))


@pytest.mark.parametrize("kind", ("f32", "bf16"))
def test_w4_one_group_longer_than_any_row_and_the_longest_row(kind):
    for rows, n, k, group in ((2, 20, 200, 1 << 30), (1, 3, 1 << 24, 1 << 24), (6, 2, (1 << 23) + 77, 96)):
        g = torch.Generator().manual_seed(k)
        x = torch.randint(-1, 2, (rows, k), generator=g, dtype=torch.int8).to(T[kind]).cuda()
        w = torch.randint(0, 256, (n, (k + 1) // 2), generator=g, dtype=torch.uint8).cuda()
        s = torch.ones(-(-k // group), n, device="cuda")
        y = torch.zeros(rows, n, device="cuda")
        call(capi.load().qcnn_op_matvec_w4, capi.MatvecW4(x=ptr(x), y=ptr(y), w=ptr(w), scale=ptr(s), ldx=k, ldy=n, ldw=(k + 1) // 2, rows=rows, n=n, k=k, group=group,
             type=KIND[kind], scale_type=capi.F32, out_type=capi.F32))
        codes = torch.stack((w & 15, w >> 4), -1).view(n, -1)[:, :k].double() - 8
        assert torch.equal(y.double(), x.double() @ codes.t())  # whole numbers below 2^24


@pytest.mark.parametrize("kind,d,rows", (("f32", 1001, 3000), ("bf16", 4099, 2000), ("f16", 77, 60000)))
def test_norm_in_place_past_the_caches(kind, d, rows):
    """Outputs of 8 MB and more are written past the caches, also over the inputs that a thread has just read."""
    g = torch.Generator("cuda").manual_seed(d)
    x, y = (torch.randn(rows, d, generator=g, device="cuda").to(T[kind]) for _ in range(2))
    out = []
    for over in (False, True):
        xs, ys = x.clone(), y.clone()
        h, n = (xs, ys) if over else (torch.empty_like(x), torch.empty_like(x))
        call(capi.load().qcnn_op_norm_res, capi.NormRes(x=ptr(xs), y=ptr(ys), h=ptr(h), n=ptr(n), ldx=d, ldy=d, ldh=d, ldn=d, rows=rows, y_rows=rows, d=d, parts=1,
             type=KIND[kind], w_type=capi.F32, post=capi.NORM_RMS, pre=capi.NORM_LAYER, alpha=0.5, beta=1.0, post_eps=1e-6, pre_eps=1e-6))
        out.append((h, n))
    assert torch.equal(out[0][0], out[1][0]) and torch.equal(out[0][1], out[1][1])
    v = y.double()
    want = x.double() + 0.5 * v / (v.square().mean(1, keepdim=True) + 1e-6).sqrt()
    assert (out[1][0].double() - want).abs().max() <= 8 * torch.finfo(T[kind]).eps + 1e-5
