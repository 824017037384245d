"""hip_ops.fp8_linear on values at the ends of their types, against its formulas in float64 on the 8-bit values (act8_ref.held8);
tolerances as tests/test_fp8_linear_gpu.py derives them."""
import pytest
import torch

from act8_ref import held8

pytestmark = pytest.mark.gpu

DEV = 'cuda:0'
U = 2.0 ** -24
TYPES = [torch.float32, torch.bfloat16, torch.float16]


def _same_or_close(got, want, err, what):
    got = got.double().cpu()
    assert torch.equal(got.isnan(), want.isnan()), what
    assert torch.equal(got.isinf(), want.isinf()) and torch.equal(got[got.isinf()], want[want.isinf()]), what
    ok = want.isfinite()
    bad = ((got - want).abs() - err - 2.0 ** -24 * want.abs())[ok]
    assert bad.max() <= 0, (what, float(bad.max()))


@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('M,N,K', [(3, 20, 40), (40, 130, 270), (600, 300, 500), (2100, 2001, 1800), (2100, 2048, 1800)])
def test_infinite_and_largest_gradients(M, N, K, dtype):
    """dW = dy^T Q(x) with infinities, NaN and the type's largest values in dy: every tile of the weight's gradient, all pieces of dy."""
    from hcmoco_amd import hip_ops
    g = torch.Generator().manual_seed(M)
    x = (torch.rand(M, K, generator=g) * 2.0 ** -7 + 2.0 ** -8) * torch.sign(torch.randn(M, 1, generator=g))
    x = x.to(dtype)
    x[0, 1] = 0
    dy = torch.randn(M, N, generator=g).to(dtype)
    top = torch.finfo(dtype).max
    dy[0, 1], dy[M - 1, 3], dy[1, 4], dy[2, N - 1] = float('inf'), float('-inf'), float('nan'), float('inf')
    dy[1, 6], dy[2, 7], dy[0, 8], dy[0, 9], dy[1, 9] = top, -top, top * 0.999, float('inf'), float('-inf')
    w = torch.zeros(N, K, device=DEV, requires_grad=True)
    b = torch.zeros(N, device=DEV, requires_grad=True)
    y = hip_ops.fp8_linear(x.to(DEV), w, b)
    dw, db = torch.autograd.grad(y, (w, b), dy.to(DEV))
    xq, d = held8(x)[0], dy.double()
    rows = (32 + 3 * M / 32 + M / 512) * U
    fine = torch.where(d.isfinite(), d, torch.zeros_like(d))
    # by columns of dy, so that no other column's infinity enters a sum through a zero
    want = torch.stack([(d[:, n, None] * xq).sum(0) if not bool(d[:, n].isfinite().all()) else d[:, n] @ xq for n in range(N)])
    _same_or_close(dw, want, rows * (fine.abs().t() @ xq.abs()), 'dw')
    total = d.sum(0)
    total = torch.where(total.abs() > 3.4028235e38, torch.sign(total) * float('inf'), total)
    _same_or_close(db, total, rows * fine.abs().sum(0), 'db')
