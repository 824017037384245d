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


def _small(M, N, K, ex, ew, seed):
    g = torch.Generator().manual_seed(seed)
    x = (torch.randn(M, K, generator=g).double() * 2.0 ** ex).float()
    w = (torch.randn(N, K, generator=g).double() * 2.0 ** ew).float()
    return x, w


@pytest.mark.parametrize('M', [20, 200])
@pytest.mark.parametrize('ex,ew', [(-114, 60), (-118, 60), (-126, 60), (-140, 60), (0, -126), (20, -130), (115, -20)])
def test_ends_of_the_range_of_scales(M, ex, ew):
    """y in fp32 is computed on the blocks' values in bf16, whose steps are 2^-133 at their smallest: a value of x (of w) is off by at most
    half of one, and nothing else is lost.  With a 16-bit y the 8-bit instructions take the scales as they are."""
    from hcmoco_amd import hip_ops
    K = 256
    x, w = _small(M, 140, K, ex, ew, M)
    xq, wq = held8(x)[0], held8(w, 128)[0]
    mag = xq.abs() @ wq.abs().t()
    y = hip_ops.fp8_linear(x.to(DEV), hip_ops.fp8_weight(w.to(DEV)))
    lost = 2.0 ** -134 * (xq.abs().sum(1, keepdim=True) + wq.abs().sum(1)[None] + K * 2.0 ** -134)
    err = (128 + K / 128 + 16) * U * (mag + lost) + lost
    assert bool(((y.double().cpu() - xq @ wq.t()).abs() <= err + U * mag + 2.0 ** -149).all())
    x16 = x.to(torch.bfloat16)
    xq = held8(x16)[0]
    mag = xq.abs() @ wq.abs().t()
    y = hip_ops.fp8_linear(x16.to(DEV), hip_ops.fp8_weight(w.to(DEV)))
    err = ((128 + K / 128 + 16) * U + 7 * 2.0 ** -13) * mag
    assert bool(((y.double().cpu() - xq @ wq.t()).abs() <= err + 2.0 ** -8 * (mag + err) + 2.0 ** -133).all())


@pytest.mark.parametrize('e', [-100, -118, -126])
def test_smallest_gradients(e):
    """fp32 dy in three bf16 pieces: what is under 2^-110 is held to half a step of 2^-133."""
    from hcmoco_amd import hip_ops
    M, N, K = 200, 140, 256
    x, dy = _small(M, N, K, 30, 0, 5)[0], (_small(M, 1, N, 0, 0, 6)[0].double() * 2.0 ** e).float()
    w = torch.zeros(N, K, device=DEV, requires_grad=True)
    dw, = torch.autograd.grad(hip_ops.fp8_linear(x.to(DEV), w), w, dy.to(DEV))
    xq, d = held8(x)[0], dy.double()
    err = (32 + 3 * M / 32 + M / 512) * U * (d.abs().t() @ xq.abs()) + 2.0 ** -134 * xq.abs().sum(0)[None]
    assert bool(((dw.double().cpu() - d.t() @ xq).abs() <= err + 2.0 ** -149).all())
