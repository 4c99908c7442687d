"""GPU parity of the operators for blocks of language models at their borders.  Inputs, oracle and tolerances as in
test_gpu_block_ops.py unless a test says otherwise."""
import pytest
import torch

from oracle import np_blocks
from qcnn_gpu_amd import capi
from test_gpu_block_ops import KIND, T, call, close, np64, ptr

pytestmark = pytest.mark.gpu


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
