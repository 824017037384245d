"""Every tile, ring and split of the products behind hip_ops.fp8_linear, at contractions long enough to use it, with scales that differ
from block to block along every axis.

The data are small whole numbers times powers of two that depend on the block of the contraction (and cancel between the two operands) and
on the row or column: products of eight neighbours stay within 2^13 of each other and sums under 2^24 units (64 * 16 a term; sums of 20001 of
them, of either sign, come to 2^17), so that every result is exact, in any order, and a scale that is taken from another block is off by
a power of two."""
import re

import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = 'cuda:0'

# M, N, K -> columns (= rows) of a tile of y, stages of its ring, whether the contraction is split
FORWARD = [
    (2048, 2048, 2051, 128, 4, False),
    (1800, 1900, 800, 128, 4, False),
    (2100, 1800, 2001, 128, 2, True),
    (1000, 5000, 1000, 128, 2, False),
    (3500, 1300, 300, 128, 2, False),
    (3000, 3000, 1700, 256, 2, False),
    (3000, 3000, 1025, 256, 2, False),
    (300, 500, 2300, 64, 4, True),
    (1000, 1200, 900, 64, 4, False),
    (640, 1280, 1601, 64, 2, True),
    (1500, 1900, 700, 64, 2, False),
    (500, 700, 300, 64, 2, False),
]


def _data(M, N, K, dtype, seed):
    """x, w, dy; every exponent but the operands' own cancels in a product's sum."""
    g = torch.Generator().manual_seed(seed)
    whole = lambda *s: torch.randint(-8, 9, s, generator=g).double()
    blocks = lambda n, top: torch.exp2(torch.randint(-top, top + 1, ((n + 127) // 128,), generator=g).double()).repeat_interleave(128)[:n]
    small = dtype == torch.float16
    ek, en, em = blocks(K, 8 if small else 20), blocks(N, 2 if small else 12), torch.exp2(torch.randint(-2, 3, (M,), generator=g).double())
    x = whole(M, K) * ek * em[:, None]
    w = whole(N, K) / ek * en[:, None]
    dy = whole(M, N) / en
    return x.to(dtype), w.float(), dy.to(dtype)


def _kernels(call):
    from torch.profiler import ProfilerActivity, profile
    with profile(activities=[ProfilerActivity.CUDA]) as prof:
        out = call()
        torch.cuda.synchronize()
    return out, [e.key for e in prof.key_averages()]


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize('M,N,K,tile,stages,split', FORWARD)
def test_exact_with_scales_of_every_block(M, N, K, tile, stages, split, dtype):
    from hcmoco_amd import hip_ops
    x, w, dy = _data(M, N, K, dtype, M + N)
    leaves = [x.to(DEV).requires_grad_(), w.to(DEV).requires_grad_()]
    y, names = _kernels(lambda: hip_ops.fp8_linear(*leaves))
    want = r'fp8_tile_kernel<%d, %d, \d, \d, %d, %s>' % (tile, tile, stages, str(dtype == torch.float32).lower())
    assert any(re.search(want, n) for n in names), (want, names)
    assert any('join_kernel' in n for n in names) == split, names
    dx, dw = torch.autograd.grad(y, leaves, dy.to(DEV))
    xd, wd, dyd = (t.double().to(DEV) for t in (x, w, dy))
    assert torch.equal(y.double(), (xd @ wd.t()).to(dtype).double())
    assert torch.equal(dx.double(), (dyd @ wd).to(dtype).double())
    assert torch.equal(dw.double(), dyd.t() @ xd)


# M, N, K, type of dy -> columns k and n of a tile of dW, whether dy goes to LDS directly
GRADIENT = [
    (2500, 2048, 2300, torch.bfloat16, 256, 256, True),
    (2500, 2001, 2300, torch.bfloat16, 256, 256, False),
    (2500, 2048, 2300, torch.float16, 256, 256, False),
    (2500, 2048, 2300, torch.float32, 384, 128, False),
    (20001, 128, 270, torch.bfloat16, 384, 128, False),
    (20001, 130, 270, torch.float32, 384, 128, False),
    (20001, 130, 270, torch.float16, 384, 128, False),
    (5000, 200, 500, torch.float32, 256, 128, False),
    (5000, 200, 500, torch.bfloat16, 256, 128, False),
    (5000, 200, 500, torch.float16, 256, 128, False),
    (5000, 333, 100, torch.float32, 128, 128, False),
    (5000, 333, 100, torch.bfloat16, 128, 128, False),
    (5000, 333, 100, torch.float16, 128, 128, False),
]


@pytest.mark.parametrize('M,N,K,dtype,tk,tn,direct', GRADIENT)
def test_weight_gradient_is_exact_in_every_tile(M, N, K, dtype, tk, tn, direct):
    from hcmoco_amd import hip_ops
    x, w, dy = _data(M, N, K, dtype, N)
    leaves = [x.to(DEV), w.to(DEV).requires_grad_(), torch.zeros(N, device=DEV, requires_grad=True)]
    y = hip_ops.fp8_linear(*leaves)
    (dw, db), names = _kernels(lambda: torch.autograd.grad(y, leaves[1:], dy.to(DEV)))
    # how the profiler prints a kernel's name depends on the type: plain, as the compiler mangled it, or with the type garbled
    want = r'fp8_wgrad_kernel(<.*, {0}, {1}, \d+, \d, \d, {2}>|I\w+?Li\dELi{0}ELi{1}ELi\d+ELi\dELi\dELb{3:d}E)'.format(
        tk, tn, str(direct).lower(), direct)
    assert any(re.search(want, n) for n in names), (want, names)
    xd, dyd = x.double().to(DEV), dy.double().to(DEV)
    assert torch.equal(dw.double(), dyd.t() @ xd)
    assert torch.equal(db.double(), dyd.sum(0))
