"""Products of 8-bit blocks (hip_ops.fp8_weight / fp8_matmul / fp8_linear) against their formulas in float64 on the 8-bit values,
which the format defines exactly (act8_ref.held8).

Tolerances: u = 2^-24.  A product of two 8-bit values is exact in fp32, and so are the power-of-two scales.  In fp32 one
matrix instruction adds its products in some order of fp32 additions, blocks and splits follow one after the other: a sum over K
is off by at most (128 + K / 128 + 16) u sum|x||w|.  A 16-bit y or dx comes from the 8-bit instructions, whose arithmetic (measured
on single products) aligns groups of eight products to the group's largest and drops what is under 2^-13 of it: seven such losses
of at most 2^-13 of a product each, so at most 7 * 2^-13 sum|x||w| more; their fp32 sums err as before.  The weight's gradient multiplies exact values too (dy as up to three bf16 pieces):
(32 + 3 M / 32 + M / 512) u sum|dy||x|.  One addition of the bias, and half a step of the output's type."""
import pytest
import torch

from act8_ref import held8

pytestmark = pytest.mark.gpu

DEV = 'cuda:0'
U = 2.0 ** -24
TYPES = [torch.float32, torch.bfloat16, torch.float16]


def _inputs(M, N, K, dtype, seed, wdtype=torch.float32):
    g = torch.Generator().manual_seed(seed)
    x = (torch.randn(M, K, generator=g) * torch.exp(torch.randn(1, K, generator=g))).clamp(-3e4, 3e4).to(dtype)
    w = (torch.randn(N, K, generator=g) / K ** 0.5 * torch.exp(torch.randn(N, 1, generator=g))).to(wdtype)
    b = torch.randn(N, generator=g)
    dy = (torch.randn(M, N, generator=g) * torch.exp(torch.randn(M, 1, generator=g)) * 0.1).to(dtype)
    return x, w, b, dy


def _close(got, want, err, dtype, what):
    assert got.dtype == dtype and got.shape == want.shape, what
    got = got.double().cpu()
    tol = err + torch.finfo(dtype).eps / 2 * (want.abs() + err) + torch.finfo(dtype).tiny
    assert got.isfinite().all(), what
    bad = (got - want).abs() - tol
    assert bad.max() <= 0, (what, float((got - want).abs().max()), float(bad.max()))


def _mm(a, b):
    """a b^T and the sum of the products' magnitudes."""
    return a @ b.t(), a.abs() @ b.abs().t()


def _sum_tol(K, dtype):
    return (128 + K / 128 + 16) * U + (0 if dtype == torch.float32 else 7 * 2.0 ** -13)


def _check_step(x, w, b, dy, got):
    """got: y, dx, dw[, db] of one training step from x, w, b and dy (CPU tensors)."""
    M, K = x.shape
    N = w.shape[0]
    xq, wq, gq = held8(x)[0], held8(w, 128)[0], held8(dy)[0]
    want, mag = _mm(xq, wq)
    err = _sum_tol(K, x.dtype) * mag
    if b is not None:
        want = want + b.double()
        err = err + U * want.abs()
    _close(got[0], want, err, x.dtype, 'y')
    want, mag = _mm(gq, wq.t())
    _close(got[1], want, _sum_tol(N, x.dtype) * mag, x.dtype, 'dx')
    rows = (32 + 3 * M / 32 + M / 512) * U
    want, mag = _mm(dy.double().t(), xq.t())
    _close(got[2], want, rows * mag, w.dtype, 'dw')
    if b is not None:
        _close(got[3], dy.double().sum(0), rows * dy.double().abs().sum(0), b.dtype, 'db')


def _run(x, w, b, dy):
    from hcmoco_amd import hip_ops
    leaves = [t.to(DEV).requires_grad_() for t in ((x, w, b) if b is not None else (x, w))]
    y = hip_ops.fp8_linear(*leaves)
    return [y.detach()] + list(torch.autograd.grad(y, leaves, dy.to(DEV)))


@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('M,N,K', [(1, 1, 1), (32, 128, 270), (5, 3, 17), (1, 300, 1000), (16, 130, 129), (17, 64, 128), (200, 257, 640),
                                   (700, 40, 2049), (130, 1500, 96), (64, 64, 5000)])
def test_training_step(M, N, K, dtype):
    x, w, b, dy = _inputs(M, N, K, dtype, M + N + K)
    _check_step(x, w, b, dy, _run(x, w, b, dy))


@pytest.mark.parametrize('M,N,K', [(3500, 3600, 300), (1800, 1900, 200), (3000, 100, 1300), (40, 4000, 700), (1000, 2040, 2049), (333, 2100, 2300),
                                   (4200, 264, 1900)])
def test_every_tile_and_split(M, N, K):
    for dtype in (torch.bfloat16, torch.float32):
        x, w, b, dy = _inputs(M, N, K, dtype, 7)
        _check_step(x, w, None, dy, _run(x, w, None, dy))


@pytest.mark.parametrize('dtype', [torch.float16, torch.bfloat16])
@pytest.mark.parametrize('M,N,K', [(2100, 2001, 1800), (2049, 2901, 2889)])
def test_wide_gradient_through_registers(M, N, K, dtype):
    x, w, b, dy = _inputs(M, N, K, dtype, 8)
    _check_step(x, w, b, dy, _run(x, w, b, dy))


def test_gradient_that_begins_anywhere():
    from hcmoco_amd import hip_ops
    x, w, b, dy = _inputs(300, 96, 200, torch.bfloat16, 6)
    leaves = [t.to(DEV).requires_grad_() for t in (x, w, b)]
    y = hip_ops.fp8_linear(*leaves)
    room = torch.zeros(300 * 96 + 1, dtype=torch.bfloat16, device=DEV)
    room[1:] = dy.flatten().to(DEV)
    _check_step(x, w, b, dy, [y.detach()] + list(torch.autograd.grad(y, leaves, room[1:].view(300, 96))))


def test_many_rows_few_columns():
    x, w, b, dy = _inputs(20001, 128, 270, torch.float32, 11)
    _check_step(x, w, b, dy, _run(x, w, b, dy))


@pytest.mark.parametrize('wdtype', [torch.bfloat16, torch.float16])
def test_weights_of_another_type(wdtype):
    x, w, b, dy = _inputs(100, 200, 300, torch.bfloat16, 3, wdtype)
    _check_step(x, w, b.to(wdtype), dy, _run(x, w, b.to(wdtype), dy))


@pytest.mark.parametrize('M', [1, 2, 7, 16, 17, 33, 250])
@pytest.mark.parametrize('N,K', [(128, 270), (1000, 4096), (77, 8000), (4100, 130)])
def test_kept_weight(M, N, K):
    from hcmoco_amd import hip_ops
    for dtype in TYPES:
        x, w, b, _ = _inputs(M, N, K, dtype, M + N, dtype)
        kept = hip_ops.fp8_weight(w.to(DEV))
        want, mag = _mm(held8(x)[0], held8(w, 128)[0])
        y = hip_ops.fp8_linear(x.to(DEV), kept, b.to(DEV))
        _close(y, want + b.double(), _sum_tol(K, dtype) * mag + U * (want + b.double()).abs(), dtype, 'y')
        y2 = hip_ops.fp8_matmul(hip_ops.act8_pack(x.to(DEV)), kept, dtype=torch.float32)
        _close(y2, want, _sum_tol(K, torch.float32) * mag, torch.float32, 'y2')


@pytest.mark.parametrize('M,N,K', [(1, 200, 384), (12, 300, 515), (40, 70, 1111), (300, 520, 900), (3000, 3500, 260)])
def test_whole_numbers_are_exact(M, N, K):
    """Small integers are 8-bit values at any scale, products of eight neighbours stay within 2^13 of each other and the sums under
    2^24: every output has to be equal, a 16-bit one to the rounded sum."""
    g = torch.Generator().manual_seed(M)
    x, w, dy = (torch.randint(-8, 9, s, generator=g).float() for s in ((M, K), (N, K), (M, N)))
    b = torch.randint(-50, 50, (N,), generator=g).float()
    y, dx, dw, db = _run(x, w, b, dy)
    assert torch.equal(y.cpu(), x @ w.t() + b) and torch.equal(dx.cpu(), dy @ w)
    assert torch.equal(dw.cpu(), dy.t() @ x) and torch.equal(db.cpu(), dy.sum(0))
    for t in (torch.bfloat16, torch.float16):
        y16, dx16, dw16, _ = _run(x.to(t), w, b, dy.to(t))
        assert torch.equal(y16.cpu(), (x @ w.t() + b).to(t)) and torch.equal(dx16.cpu(), (dy @ w).to(t)) and torch.equal(dw16.cpu(), dy.t() @ x)
    # and the gradients are the slopes: L = sum(dy * y) along whole directions
    for k, (p, grad) in enumerate(((x, dx), (w, dw), (b, db))):
        v = torch.randint(-1, 2, p.shape, generator=g).float()
        ends = []
        for sign in (1, -1):
            q = [x, w, b]
            q[k] = (p + sign * v)
            ends.append((_run(*q, dy)[0].double().cpu() * dy.double()).sum())
        assert float(ends[0] - ends[1]) == 2 * float((grad.double().cpu() * v.double()).sum())


def test_scales_span_the_range():
    from hcmoco_amd import hip_ops
    g = torch.Generator().manual_seed(1)
    x = torch.randn(20, 512, generator=g)
    w = torch.randn(140, 512, generator=g)
    x[:, 128:256] *= 2.0 ** 60
    x[:, 256:384] *= 2.0 ** -60
    w[:, 128:256] *= 2.0 ** -70
    w[128:] *= 2.0 ** 20
    x[3] = 0
    for rows in (20, 200):                              # the kernel for a few rows, and the tiles
        x = x.repeat(rows // 20, 1)
        want, mag = _mm(held8(x)[0], held8(w, 128)[0])
        y = hip_ops.fp8_linear(x.to(DEV), hip_ops.fp8_weight(w.to(DEV)))
        _close(y, want, _sum_tol(512, torch.float32) * mag, torch.float32, 'y')
        assert (y[3] == 0).all()
        x16 = x.to(torch.bfloat16)                      # (bf16 has fp32's range)
        want, mag = _mm(held8(x16)[0], held8(w, 128)[0])
        _close(hip_ops.fp8_linear(x16.to(DEV), hip_ops.fp8_weight(w.to(DEV))), want, _sum_tol(512, torch.bfloat16) * mag, torch.bfloat16, 'y16')


def test_rows_that_are_not_finite_stay_by_themselves():
    from hcmoco_amd import hip_ops
    for M in (9, 200):
        x, w, b, dy = _inputs(M, 150, 300, torch.float32, 4)
        kept = hip_ops.fp8_weight(w.to(DEV))
        clean = hip_ops.fp8_linear(x.to(DEV), kept)
        x2 = x.clone()
        x2[2, 7], x2[8, 299] = float('inf'), float('nan')
        y = hip_ops.fp8_linear(x2.to(DEV), kept)
        keep = torch.ones(M, dtype=torch.bool)
        keep[[2, 8]] = False
        assert torch.equal(y[keep], clean[keep]) and y[~keep].isnan().all()


def test_packed_rows_are_the_checkpoint():
    """A few rows are packed inside the product's kernel, more of them by act8_pack: the weight's gradient reads the same bytes."""
    from hcmoco_amd import hip_ops
    for M, K in ((3, 270), (32, 1024), (32, 1025), (33, 270)):
        x, w, b, dy = _inputs(M, 40, K, torch.bfloat16, M + K)
        xs, ws = x.to(DEV).requires_grad_(), w.to(DEV).requires_grad_()
        y = hip_ops.fp8_linear(xs, ws)
        p = hip_ops.act8_pack(xs)
        assert torch.equal(y, hip_ops.fp8_matmul(p, hip_ops.fp8_weight(w.to(DEV))))
        got = torch.autograd.grad(y, ws, dy.to(DEV))[0]
        want, mag = _mm(dy.double().t(), held8(x)[0].t())
        _close(got, want, (32 + 3 * M / 32 + M / 512) * U * mag, torch.float32, 'dw')


def test_two_streams_at_once():
    from hcmoco_amd import hip_ops
    data = [_inputs(300, 500, 1200, torch.bfloat16, 60 + k) for k in range(2)]
    alone = [_run(*d) for d in data]
    streams = [torch.cuda.Stream() for _ in range(2)]
    inputs = [[t.to(DEV) for t in d] for d in data]
    torch.cuda.synchronize()
    outs = [[], []]
    for rep in range(5):
        for k in range(2):
            with torch.cuda.stream(streams[k]):
                leaves = [t.clone().requires_grad_() for t in inputs[k][:3]]
                y = hip_ops.fp8_linear(*leaves)
                outs[k].append([y.detach()] + list(torch.autograd.grad(y, leaves, inputs[k][3])))
    torch.cuda.synchronize()
    for k in range(2):
        for got in outs[k]:
            assert all(torch.equal(p, q) for p, q in zip(got, alone[k]))


def test_one_tensor_in_two_places():
    from hcmoco_amd import hip_ops
    x, _, _, dy = _inputs(130, 130, 130, torch.float32, 70)
    a = x.to(DEV).requires_grad_()
    y = hip_ops.fp8_linear(a, a)
    y.backward(dy.to(DEV))
    xq, wq, gq = held8(x)[0], held8(x, 128)[0], held8(dy)[0]
    d1, m1 = _mm(gq, wq.t())
    d2, m2 = _mm(dy.double().t(), xq.t())
    _close(a.grad, d1 + d2, _sum_tol(130, torch.float32) * (m1 + m2) + U * (d1 + d2).abs(), torch.float32, 'dx + dw')


def test_shapes_views_frozen_and_empty():
    from hcmoco_amd import hip_ops
    x, w, b, dy = _inputs(60, 90, 140, torch.float32, 5)
    xd, wd, bd = x.to(DEV), w.to(DEV), b.to(DEV)
    flat = hip_ops.fp8_linear(xd, wd, bd)
    assert torch.equal(hip_ops.fp8_linear(xd.view(3, 4, 5, 140), wd, bd).view(60, 90), flat)
    assert torch.equal(hip_ops.fp8_linear(xd[0], wd, bd), hip_ops.fp8_linear(xd[:1], wd, bd)[0])
    wide = torch.zeros(60, 301, device=DEV)
    wide[:, 3:143] = xd
    wt = wd.t().contiguous().t()
    assert torch.equal(hip_ops.fp8_linear(wide[:, 3:143], wt, bd), flat)
    # a frozen weight kept in 8 bits: the gradient of x and of the bias only, the same bits
    kept = hip_ops.fp8_weight(wd)
    a, c = xd.clone().requires_grad_(), bd.clone().requires_grad_()
    y = hip_ops.fp8_linear(a, kept, c)
    y.backward(dy.to(DEV).expand_as(y))
    full = _run(x, w, b, dy)
    assert torch.equal(y, full[0]) and torch.equal(a.grad, full[1]) and torch.equal(c.grad, full[3])
    a = xd.clone().requires_grad_()
    y = hip_ops.fp8_linear(a, wd, bd)
    y.sum().backward()                              # an expanded dy
    assert a.grad.shape == a.shape
    e = torch.empty(0, 140, device=DEV, requires_grad=True)
    wl, bl = wd.clone().requires_grad_(), bd.clone().requires_grad_()
    y = hip_ops.fp8_linear(e, wl, bl)
    y.sum().backward()
    assert y.shape == (0, 90) and e.grad.shape == (0, 140) and (wl.grad == 0).all() and (bl.grad == 0).all()
    assert kept.nbytes() < 3 * w.numel()


@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('M,N', [(5, 3), (40, 130), (3000, 257), (20000, 1000)])
def test_bias_alone(M, N, dtype):
    """A frozen weight: nothing of x is kept, the bias's gradient is the sum of dy's rows."""
    from hcmoco_amd import hip_ops
    x, w, b, dy = _inputs(M, N, 70, dtype, M)
    bias = b.to(DEV).requires_grad_()
    y = hip_ops.fp8_linear(x.to(DEV), hip_ops.fp8_weight(w.to(DEV)), bias)
    got, = torch.autograd.grad(y, bias, dy.to(DEV))
    _close(got, dy.double().sum(0), (32 + 3 * M / 32 + M / 512) * U * dy.double().abs().sum(0), torch.float32, 'db')


def test_a_block_of_layers():
    """layer norm -> linear -> layer norm (8-bit checkpoint) -> linear, forward and backward in one graph: every stage against its
    formulas on the tensors that it was really given."""
    from hcmoco_amd import hip_ops
    from test_layer_norm_gpu import _check, _truth
    g = torch.Generator().manual_seed(9)
    M, C, H = 544, 270, 384
    dtype = torch.bfloat16
    x = torch.randn(M, C, generator=g).to(dtype)
    p = [1 + 0.1 * torch.randn(C, generator=g), 0.1 * torch.randn(C, generator=g), torch.randn(H, C, generator=g) / C ** 0.5,
         torch.randn(H, generator=g), 1 + 0.1 * torch.randn(H, generator=g), 0.1 * torch.randn(H, generator=g),
         torch.randn(128, H, generator=g) / H ** 0.5]
    dy = (0.01 * torch.randn(M, 128, generator=g)).to(dtype)
    leaves = [t.to(DEV).requires_grad_() for t in [x] + p]
    xs, w1, b1, W1, B1, w2, b2, W2 = leaves
    h1 = hip_ops.layer_norm(xs, w1, b1)
    h2 = hip_ops.fp8_linear(h1, W1, B1)
    h3 = hip_ops.layer_norm(h2, w2, b2, act8=True)
    y = hip_ops.fp8_linear(h3, W2)
    for t in (h1, h2, h3):
        t.retain_grad()
    y.backward(dy.to(DEV))
    c = lambda t: t.detach().cpu()
    _check_step(c(h3), p[6], None, dy, [y.detach(), h3.grad, W2.grad])
    want, err = _truth(c(h2), p[4], p[5], c(h3.grad), 1e-5, held8(c(h2))[0])
    for got, t, e, n, d in zip((h3.detach(), h2.grad, w2.grad, b2.grad), want, err, 'yxwb', (dtype, dtype, torch.float32, torch.float32)):
        _check(got, t, e, (n, d))
    _check_step(c(h1), p[2], p[3], c(h2.grad), [h2.detach(), h1.grad, W1.grad, B1.grad])
    want, err = _truth(x, p[0], p[1], c(h1.grad), 1e-5)
    for got, t, e, n, d in zip((h1.detach(), xs.grad, w1.grad, b1.grad), want, err, 'yxwb', (dtype, dtype, torch.float32, torch.float32)):
        _check(got, t, e, (n, d))


def test_same_bits_twice_other_stream_and_graph():
    from hcmoco_amd import hip_ops
    x, w, b, dy = _inputs(600, 384, 1300, torch.bfloat16, 50)
    one, two = _run(x, w, b, dy), _run(x, w, b, dy)
    assert all(torch.equal(p, q) for p, q in zip(one, two))
    xs, ws, bs, ds = (t.to(DEV) for t in (x, w, b, dy))
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        leaves = [t.clone().requires_grad_() for t in (xs, ws, bs)]
        y = hip_ops.fp8_linear(*leaves)
        other = [y.detach()] + list(torch.autograd.grad(y, leaves, ds))
    st.synchronize()
    assert all(torch.equal(p, q) for p, q in zip(one, other))
    leaves = [t.clone().requires_grad_() for t in (xs, ws, bs)]
    st.wait_stream(torch.cuda.current_stream())
    graphs = []
    for _ in range(2):                                  # two graphs of the same call: neither may use the other's workspace
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=st):
            y = hip_ops.fp8_linear(*leaves)
            outs = [y.detach()] + list(torch.autograd.grad(y, leaves, ds))
        graphs.append((graph, outs))
    for k in range(4):
        with torch.no_grad():
            leaves[0].copy_(xs * (k + 1))
        for graph, _ in graphs:
            graph.replay()
        torch.cuda.synchronize()
        eager = _run(x * (k + 1), w, b, dy)
        for _, outs in graphs:
            assert all(torch.equal(p, q) for p, q in zip(outs, eager))


def test_refuses():
    from hcmoco_amd import hip_ops
    x, w, b = torch.zeros(4, 8, device=DEV), torch.zeros(6, 8, device=DEV), torch.zeros(6, device=DEV)
    for bad in ((x.double(), w), (x, w.double()), (x, w, b.double())):
        with pytest.raises(TypeError):
            hip_ops.fp8_linear(*bad)
    for bad in ((x, w[:, :7]), (x, w, b[:5]), (x, w, b.view(1, 6)), (x, w.view(6, 8, 1)), (x, w[:0])):
        with pytest.raises(ValueError):
            hip_ops.fp8_linear(*bad)
    with pytest.raises(RuntimeError, match='no CPU fallback'):
        hip_ops.fp8_linear(x, w.cpu())
    with pytest.raises(ValueError):
        hip_ops.fp8_weight(w[0])
    kept, a = hip_ops.fp8_weight(w), hip_ops.act8_pack(x)
    with pytest.raises(TypeError):
        hip_ops.fp8_matmul(x, kept)
    with pytest.raises(TypeError):
        hip_ops.fp8_matmul(a, w)
    with pytest.raises(TypeError):
        hip_ops.fp8_matmul(a, kept, dtype=torch.int32)
    for call in (lambda: hip_ops.fp8_matmul(hip_ops.act8_pack(x[:, :5]), kept), lambda: hip_ops.fp8_linear(x[:, :5], kept),
                 lambda: hip_ops.fp8_linear(x, kept, b[:5]), lambda: hip_ops.fp8_matmul(a, kept, b[:5])):
        with pytest.raises(ValueError):
            call()
    y = hip_ops.fp8_linear(x.requires_grad_(), w)
    g, = torch.autograd.grad(y, x, torch.ones_like(y).requires_grad_(), create_graph=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(g.sum(), x)                 # no second derivative
