"""hip_ops.layer_norm against its formulas in float64.

Tolerances, before any run: u = 2^-24 is the rounding of one fp32 operation.  No sum here is a chain of more than 64 additions
(a lane's values, then a tree of lanes and waves; for the columns, a workgroup's rows, its side-by-side rows, the partial rows), so
a sum is off by at most 64 u sum|terms|; that bounds the mean (64 u mean|x|), the variance and 1/sqrt (40 u), and every
gradient term by term, as written in _bounds().  The output's own rounding is half a step of its type."""
import pytest
import torch

from act8_ref import held8

pytestmark = pytest.mark.gpu

DEV = 'cuda:0'
U = 2.0 ** -24
TYPES = [torch.float32, torch.bfloat16, torch.float16]
COLS = [1, 2, 3, 8, 127, 128, 129, 270, 384, 385, 513, 1000, 2048, 2049, 5000, 8193, 16384, 16385, 20001]


def _inputs(rows, cols, dtype, seed, wdtype=torch.float32):
    g = torch.Generator().manual_seed(seed)
    x = (torch.randn(rows, cols, generator=g) * torch.exp(0.5 * torch.randn(1, cols, generator=g)) + torch.randn(rows, 1, generator=g)).to(dtype)
    w = (1 + 0.3 * torch.randn(cols, generator=g)).to(wdtype)
    b = torch.randn(cols, generator=g).to(wdtype)
    dy = (torch.randn(rows, cols, generator=g) * 0.1).to(dtype)
    return x, w, b, dy


def _truth(x, w, b, dy, eps, x8=None):
    """y, dx, dw, db in float64 and how far fp32 arithmetic may be from them, before the outputs' own rounding."""
    x, w, b, dy = (t.double() for t in (x, w, b, dy))
    mean = x.mean(1, keepdim=True)
    rstd = 1 / torch.sqrt(((x - mean) ** 2).mean(1, keepdim=True) + eps)
    n = (x - mean) * rstd
    src = x if x8 is None else x8
    h = (src - mean) * rstd
    # normalised value: the mean's error and the subtraction's, scaled; the scale's own error
    off = lambda v, hv: 64 * U * x.abs().mean(1, keepdim=True) * rstd + U * v.abs() * rstd + 48 * U * hv.abs()
    en, eh = off(x, n), off(src, h)
    # the variance feels the mean's error through the scale as well where the row is nearly constant
    dm = 64 * U * x.abs().mean(1, keepdim=True) * rstd
    en, eh = en + n.abs() * dm ** 2, eh + h.abs() * dm ** 2
    y = n * w + b
    ey = en * w.abs() + 2 * U * (n * w).abs() + U * y.abs()
    g = dy * w
    mg, mgh = g.mean(1, keepdim=True), (g * h).mean(1, keepdim=True)
    emg = 66 * U * g.abs().mean(1, keepdim=True)
    emgh = 67 * U * (g * h).abs().mean(1, keepdim=True) + (g.abs() * eh).mean(1, keepdim=True)
    inner = g - mg - h * mgh
    dx = rstd * inner
    edx = rstd * (4 * U * (g.abs() + mg.abs() + (h * mgh).abs()) + emg + h.abs() * emgh + eh * mgh.abs()) + (48 * U + dm ** 2) * dx.abs()
    dw, db = (dy * h).sum(0), dy.sum(0)
    edw = 66 * U * (dy * h).abs().sum(0) + (dy.abs() * eh).sum(0)
    edb = 66 * U * dy.abs().sum(0)
    return (y, dx, dw, db), (ey, edx, edw, edb)


def _check(got, want, err, what):
    got = got.double().cpu()
    tol = err + (torch.finfo(what[1]).eps / 2) * (want.abs() + err) + torch.finfo(what[1]).tiny
    bad = (got - want).abs() - tol
    assert got.isfinite().all() and bad.max() <= 0, (what[0], float((got - want).abs().max()), float(bad.max()))


def _run(x, w, b, dy, eps, act8):
    from hcmoco_amd import hip_ops
    xs, ws, bs = (t.to(DEV).requires_grad_() for t in (x, w, b))
    y = hip_ops.layer_norm(xs, ws, bs, eps, act8=act8)
    return [y.detach()] + list(torch.autograd.grad(y, (xs, ws, bs), dy.to(DEV)))


def _case(rows, cols, dtype, act8, seed, wdtype=torch.float32, eps=1e-5):
    x, w, b, dy = _inputs(rows, cols, dtype, seed, wdtype)
    got = _run(x, w, b, dy, eps, act8)
    want, err = _truth(x, w, b, dy, eps, held8(x)[0] if act8 else None)
    for g, t, e, n, d in zip(got, want, err, ('y', 'dx', 'dw', 'db'), (dtype, dtype, wdtype, wdtype)):
        assert g.dtype == d
        _check(g, t, e, (n, d))


@pytest.mark.parametrize('act8', [False, True])
@pytest.mark.parametrize('cols', COLS)
def test_matches_the_formulas(cols, act8):
    _case(5, cols, torch.float32, act8, cols)


@pytest.mark.parametrize('act8', [False, True])
@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('rows,cols', [(1, 1024), (544, 128), (97, 270), (1300, 40), (70, 2048), (33, 4096), (9, 7777)])
def test_types_and_rows(rows, cols, dtype, act8):
    _case(rows, cols, dtype, act8, rows + cols)


@pytest.mark.parametrize('wdtype', [torch.bfloat16, torch.float16])
def test_parameters_of_another_type(wdtype):
    _case(50, 270, torch.float32, False, 3, wdtype)
    _case(50, 270, torch.bfloat16, True, 4, wdtype)


def test_eps_is_inside_the_root_and_constant_rows_give_the_bias():
    x, w, b, dy = _inputs(6, 256, torch.float32, 8)
    x[1] = 3.0
    x[2] = 0.0
    x[3] *= 1e-4
    got = _run(x, w, b, dy, 1e-2, False)
    want, err = _truth(x, w, b, dy, 1e-2)
    for g, t, e, n in zip(got, want, err, ('y', 'dx', 'dw', 'db')):
        _check(g, t, e, (n, torch.float32))
    assert torch.equal(got[0][1].cpu(), b) and torch.equal(got[0][2].cpu(), b)


def test_optional_parameters_and_inference():
    from hcmoco_amd import hip_ops
    x, w, b, dy = _inputs(40, 300, torch.float32, 12)
    one, zero = torch.ones(300), torch.zeros(300)
    for ww, bb in ((None, None), (w, None), (None, b)):
        want, err = _truth(x, ww if ww is not None else one, bb if bb is not None else zero, dy, 1e-5)
        leaves = [t.to(DEV).requires_grad_() if t is not None else None for t in (x, ww, bb)]
        y = hip_ops.layer_norm(*leaves)
        grads = torch.autograd.grad(y, [t for t in leaves if t is not None], dy.to(DEV))
        it = iter(grads)
        for t, k, n in zip(leaves, (1, 2, 3), ('dx', 'dw', 'db')):
            if t is not None:
                _check(next(it), want[k], err[k], (n, torch.float32))
        with torch.no_grad():
            assert torch.equal(hip_ops.layer_norm(*leaves), y)
    frozen = hip_ops.layer_norm(x.to(DEV), w.to(DEV).requires_grad_(), b.to(DEV))
    frozen.backward(dy.to(DEV))                        # x itself needs no gradient


def test_rows_that_are_not_finite_stay_by_themselves():
    from hcmoco_amd import hip_ops
    x, w, b, dy = _inputs(64, 270, torch.float32, 13)
    clean = _run(x, w, b, dy, 1e-5, False)
    x2 = x.clone()
    x2[3, 5], x2[40, 269] = float('nan'), float('inf')
    got = _run(x2, w, b, dy, 1e-5, False)
    keep = torch.ones(64, dtype=torch.bool)
    keep[[3, 40]] = False
    for k in (0, 1):
        assert torch.equal(got[k][keep], clean[k][keep]) and got[k][~keep].isnan().all()
    assert hip_ops.layer_norm(x2.to(DEV))[keep].isfinite().all()


@pytest.mark.parametrize('act8', [False, True])
def test_views_shapes_and_misaligned_rows(act8):
    from hcmoco_amd import hip_ops
    base = _inputs(30, 701, torch.bfloat16, 21)[0]
    for v in (base[:, 1:271], base[:, 3:4], base[::3], base.t(), base[:, ::7], base.flatten()[1:1 + 30 * 700].view(3, 10, 700), base[2]):
        cols = v.shape[-1]
        x2 = v.reshape(-1, cols)
        _, w, b, dy = _inputs(x2.shape[0], cols, torch.bfloat16, cols)
        xs = base.to(DEV)
        xv = torch.as_strided(xs, v.shape, v.stride(), v.storage_offset()).requires_grad_()
        ws, bs = w.to(DEV).requires_grad_(), b.to(DEV).requires_grad_()
        y = hip_ops.layer_norm(xv, ws, bs, act8=act8)
        got = [y] + list(torch.autograd.grad(y, (xv, ws, bs), dy.view(v.shape).to(DEV)))
        want, err = _truth(x2, w, b, dy, 1e-5, held8(x2)[0] if act8 else None)
        assert y.shape == v.shape and got[1].shape == v.shape
        for g, t, e, n, d in zip(got, want, err, ('y', 'dx', 'dw', 'db'), (torch.bfloat16, torch.bfloat16, torch.float32, torch.float32)):
            _check(g.reshape(t.shape), t, e, (n, d))


def test_gradients_of_broadcast_and_empty_inputs():
    from hcmoco_amd import hip_ops
    x, w, b, dy = _inputs(12, 200, torch.float32, 30)
    row = x[:1].to(DEV).requires_grad_()
    y = hip_ops.layer_norm(row.expand(12, 200), w.to(DEV), b.to(DEV))
    y.backward(dy.to(DEV))
    want, err = _truth(x[:1].expand(12, 200), w, b, dy, 1e-5)
    _check(row.grad, want[1].sum(0, keepdim=True), err[1].sum(0, keepdim=True) + 12 * U * want[1].abs().sum(0, keepdim=True), ('dx', torch.float32))
    e = torch.empty(0, 200, device=DEV, requires_grad=True)
    ws, bs = w.to(DEV).requires_grad_(), b.to(DEV).requires_grad_()
    y = hip_ops.layer_norm(e, ws, bs, act8=True)
    y.sum().backward()
    assert y.shape == (0, 200) and e.grad.shape == (0, 200) and (ws.grad == 0).all() and (bs.grad == 0).all()


def test_gradient_against_differences():
    """L = sum(c * y): (L(p + s v) - L(p - s v)) / 2 s for a random direction v of x, w and b.  y is off by at most 2^-20 of its
    size, so the quotient by sum|c| 2^-20 |y| / s, and the third derivative adds s^2: both under 2e-3 of sum|c||dy| here."""
    from hcmoco_amd import hip_ops
    x, w, b, c = _inputs(8, 64, torch.float32, 44)
    got = _run(x, w, b, c, 1e-5, False)
    g = torch.Generator().manual_seed(3)
    s = 2.0 ** -7
    for k, p in enumerate((x, w, b)):
        v = torch.randn(p.shape, generator=g)
        ends = []
        for sign in (1, -1):
            q = [t.clone() for t in (x, w, b)]
            q[k] = p + sign * s * v
            ends.append((hip_ops.layer_norm(*[t.to(DEV) for t in q]).double().cpu() * c.double()).sum())
        slope = (ends[0] - ends[1]) / (2 * s)
        scale = (got[k + 1].double().cpu() * v.double()).abs().sum()
        assert abs(float(slope - (got[k + 1].double().cpu() * v.double()).sum())) < 2e-3 * float(scale)


def test_same_bits_twice_other_stream_and_graph():
    from hcmoco_amd import hip_ops
    x, w, b, dy = _inputs(3000, 270, torch.float32, 50)
    one, two = _run(x, w, b, dy, 1e-5, True), _run(x, w, b, dy, 1e-5, True)
    assert all(torch.equal(p, q) for p, q in zip(one, two))
    xs, ws, bs, ds = (t.to(DEV) for t in (x, w, b, dy))
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        leaves = [t.clone().requires_grad_() for t in (xs, ws, bs)]
        y = hip_ops.layer_norm(*leaves, act8=True)
        other = [y.detach()] + list(torch.autograd.grad(y, leaves, ds))
    st.synchronize()
    assert all(torch.equal(p, q) for p, q in zip(one, other))
    leaves = [t.clone().requires_grad_() for t in (xs, ws, bs)]
    st.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=st):
        y = hip_ops.layer_norm(*leaves, act8=True)
        outs = [y.detach()] + list(torch.autograd.grad(y, leaves, ds))
    for k in range(4):
        with torch.no_grad():
            leaves[0].copy_(xs * (k + 1))
        graph.replay()
        torch.cuda.synchronize()
        eager = _run(x * (k + 1), w, b, dy, 1e-5, True)
        assert all(torch.equal(p, q) for p, q in zip(outs, eager))


def test_refuses():
    from hcmoco_amd import hip_ops
    x, w = torch.zeros(4, 8, device=DEV), torch.ones(8, device=DEV)
    for bad in (dict(x=x.double()), dict(x=x.int())):
        with pytest.raises(TypeError):
            hip_ops.layer_norm(**bad)
    with pytest.raises(RuntimeError, match='no CPU fallback'):
        hip_ops.layer_norm(x, w.cpu())
    for bad in (w[:7], w.view(1, 8), torch.ones(16, device=DEV)[::2]):
        with pytest.raises(ValueError):
            hip_ops.layer_norm(x, bad)
        with pytest.raises(ValueError):
            hip_ops.layer_norm(x, w, bad)
    with pytest.raises(ValueError):
        hip_ops.layer_norm(x, eps=-1.0)
    with pytest.raises(ValueError):
        hip_ops.layer_norm(x[:, :0])
    y = hip_ops.layer_norm(x.requires_grad_())
    g, = torch.autograd.grad(y, x, torch.ones_like(y).requires_grad_(), create_graph=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(g.sum(), x)                     # no second derivative
