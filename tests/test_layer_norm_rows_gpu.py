"""hip_ops.layer_norm at the sizes where its sums get long: very long rows, and more rows than its workgroups hold at once.

Tolerances: u = 2^-24.  No sum in the kernels is a chain of more than 256 additions of terms, and what those make is added up again
(at most 64 of them here, then 22 more in a tree of lanes, waves and slices): a sum is off by at most 350 u sum|terms|."""
import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = 'cuda:0'
U = 2.0 ** -24
SUM = 350 * U


@pytest.fixture(autouse=True)
def _memory_goes_back():
    yield
    torch.cuda.empty_cache()


def _needs(gigabytes):
    if torch.cuda.mem_get_info()[0] < gigabytes << 30:
        pytest.skip('needs %d GB of device memory' % gigabytes)


def test_sums_along_a_very_long_row():
    """Equal values, just above a power of two: a running sum of 16384 of them (2^24 columns on 1024 lanes) would round each one down and
    lose 2e-4 of itself.  With eps = 1: y = x - mean = 0 up to the mean's error, and dx = dy - mean(dy) = 0 likewise."""
    from hcmoco_amd import hip_ops
    C = 1 << 24
    x = torch.full((1, C), 1 + 0.9 * 2.0 ** -11, device=DEV, requires_grad=True)
    y = hip_ops.layer_norm(x, eps=1.0)
    assert float(y.detach().abs().max()) <= 2 * SUM
    dx, = torch.autograd.grad(y, x, torch.full_like(y, 1 + 0.9 * 2.0 ** -11))
    assert float(dx.abs().max()) <= 2 * SUM
    # and the variance: (x - mean)^2 = (1 + 0.9 * 2^-11)^2 in every column
    s = (1 + 0.9 * 2.0 ** -11) * (1 - 2 * (torch.arange(C, device=DEV) & 1).float())
    y = hip_ops.layer_norm(s[None], eps=0.0)
    assert float((y.abs() - 1).abs().max()) <= 2 * SUM


@pytest.mark.parametrize('rows,cols,memory', [(200000, 16385, 100), (1000000, 4100, 110), (3000000, 400, 40)])
def test_sums_over_very_many_rows(rows, cols, memory):
    """dy of one value whose running sum, over 2048 long, would round each addition down (7e-5 of the sum at 200000 rows).  x is +1 and
    -1 in turn along every row, so that h is +-1/2 and dw sums equal terms too."""
    from hcmoco_amd import hip_ops
    _needs(memory)
    eps = 3.0                                               # sqrt(1 + 3) = 2: h is exactly +-1/2
    cols += cols & 1
    v = 1 + 0.9 * 2.0 ** -13
    x = torch.ones(rows, cols, device=DEV)
    x[:, 1::2] = -1
    w, b = torch.ones(cols, device=DEV, requires_grad=True), torch.zeros(cols, device=DEV, requires_grad=True)
    y = hip_ops.layer_norm(x, w, b, eps=eps)
    assert torch.equal(y[-1], 0.5 * x[-1]) and torch.equal(y[rows // 2], 0.5 * x[0])
    dw, db = torch.autograd.grad(y, (w, b), torch.full((1, 1), v, device=DEV).expand(rows, cols))
    vf = float(torch.tensor(v))
    assert float((db.double() - rows * vf).abs().max()) <= (SUM + U) * rows * vf
    assert float((dw.double() - 0.5 * rows * vf * x[0].double()).abs().max()) <= (SUM + 4 * U) * 0.5 * rows * vf


@pytest.mark.parametrize('act8', [False, True])
@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
def test_the_longest_row(dtype, act8):
    """2^27 - 1 columns, both directions, at the values of a sample of columns; the sums of all in float64."""
    from hcmoco_amd import hip_ops
    _needs(30)
    C = (1 << 27) - 1
    g = torch.Generator(device=DEV).manual_seed(2)
    x, dy = (torch.randint(-4, 5, (1, C), generator=g, device=DEV, dtype=torch.int8).to(dtype) for _ in range(2))     # 8-bit values: act8 keeps them
    w, b = (torch.randint(-4, 5, (C,), generator=g, device=DEV, dtype=torch.int8).float() for _ in range(2))
    leaves = [t.requires_grad_() for t in (x, w, b)]
    y = hip_ops.layer_norm(*leaves, act8=act8)
    dx, dw, db = torch.autograd.grad(y, leaves, dy)
    x, dy, w, b = (t.detach().double().view(-1) for t in (x, dy, w, b))
    mean = x.mean()
    rstd = 1 / torch.sqrt(((x - mean) ** 2).mean() + 1e-5)
    gr = dy * w
    mg, mgh = gr.mean(), (gr * (x - mean)).mean() * rstd
    # |h|, |g|, |y| <= 2, 16, 12 and a sum's error of 2 * 256 + 22 additions on mean, variance and both means of the gradient
    err = 600 * U
    half = torch.finfo(dtype).eps / 2
    for at in (slice(0, 5000), slice(C // 2, C // 2 + 5000), slice(C - 5000, C)):
        h = (x[at] - mean) * rstd
        want = h * w[at] + b[at]
        assert float(((y.detach().view(-1)[at].double() - want).abs() - 12 * err - half * want.abs()).max()) <= 0
        want = rstd * (gr[at] - mg - h * mgh)
        assert float(((dx.view(-1)[at].double() - want).abs() - 100 * err - half * want.abs()).max()) <= 0
        assert float((dw[at].double() - dy[at] * h).abs().max()) <= 8 * err
    assert torch.equal(db.double(), dy)


def test_too_many_long_rows_are_refused():
    from hcmoco_amd import hip_ops
    for train in (False, True):
        with pytest.raises(ValueError):
            hip_ops.layer_norm(torch.zeros(1, 1, device=DEV, dtype=torch.bfloat16, requires_grad=train).expand(1 << 22, 16385))


# (rows, cols): each of the kernels' widths, with three trips of the forward pass's workgroups and five to nine of the backward pass's, the last
# one not full.  One trip is 32768 and 16384 rows up to 384 columns, 4096 and 2048 up to 2048, 1024 and 512 up to 4096, 1024 and 256 up to
# 8192, 512 and 256 up to 16384.
TRIPS = [(65543, 100), (65601, 270), (81001, 384), (8195, 500), (12200, 1000), (8501, 2000), (2051, 4096), (2900, 3001), (2051, 8000), (1031, 16384)]


@pytest.mark.parametrize('act8', [False, True])
@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize('rows,cols', TRIPS)
def test_workgroups_that_take_many_rows(rows, cols, dtype, act8):
    """Every row's y and dx and both column sums against float64 (tests/test_layer_norm_gpu.py derives the tolerances: its sums of at
    most 64 additions hold here too, 9 trips + 16 rows side by side + 1024 partial rows by 64 + 20)."""
    from act8_ref import held8
    from test_layer_norm_gpu import _check, _inputs, _run, _truth
    x, w, b, dy = _inputs(rows, cols, dtype, rows)
    x8 = held8(x)[0].to(DEV) if act8 else None
    got = _run(x, w, b, dy, 1e-5, act8)
    want, err = _truth(*(t.to(DEV) for t in (x, w, b, dy)), 1e-5, x8)
    for g, t, e, n, d in zip(got, want, err, ('y', 'dx', 'dw', 'db'), (dtype, dtype, torch.float32, torch.float32)):
        _check(g, t.cpu(), e.cpu(), (n, d))


@pytest.mark.parametrize('rows,cols', [(65543, 100), (8195, 500), (2051, 4096)])
def test_many_rows_of_a_column_slice(rows, cols):
    """The rows that are loaded ahead lie a pitch apart, and what lies between them is NaN."""
    from test_layer_norm_gpu import _check, _inputs, _truth
    from hcmoco_amd import hip_ops
    x, w, b, dy = (t.to(DEV) for t in _inputs(rows, cols, torch.bfloat16, cols))
    wide = torch.full((rows, cols + 13), float('nan'), dtype=torch.bfloat16, device=DEV)
    wide[:, 5:5 + cols] = x
    leaves = [t.requires_grad_() for t in (wide[:, 5:5 + cols].detach(), w, b)]
    y = hip_ops.layer_norm(*leaves)
    got = [y.detach()] + list(torch.autograd.grad(y, leaves, dy))
    want, err = _truth(x, w.detach(), b.detach(), dy, 1e-5)
    for g, t, e, n, d in zip(got, want, err, ('y', 'dx', 'dw', 'db'), (torch.bfloat16, torch.bfloat16, torch.float32, torch.float32)):
        _check(g, t.cpu(), e.cpu(), (n, d))


@pytest.mark.parametrize('act8', [False, True])
@pytest.mark.parametrize('rows,cols,dtype', [(4200007, 8, torch.float32), (2 * 4194304, 5, torch.bfloat16), (131077, 2049, torch.float16)])
def test_more_rows_than_one_launch_takes(rows, cols, dtype, act8):
    """256 rows of each workgroup of a launch (4194304 rows up to 384 columns, 131072 of 2049..4096), then the next launch: eager, and captured
    and replayed.  The column sums: chains of 256 + 16 side by side + at most 2048 partial rows by 64 + 20 < 350, where _truth() has 66."""
    from act8_ref import held8
    from hcmoco_amd import hip_ops
    from test_layer_norm_gpu import _check, _inputs, _run, _truth
    x, w, b, dy = _inputs(rows, cols, dtype, cols)
    x8 = held8(x)[0].to(DEV) if act8 else None
    got = _run(x, w, b, dy, 1e-5, act8)
    want, err = _truth(*(t.to(DEV) for t in (x, w, b, dy)), 1e-5, x8)
    for g, t, e, n, d, long in zip(got, want, err, ('y', 'dx', 'dw', 'db'), (dtype, dtype, torch.float32, torch.float32), (1, 1, 6, 6)):
        _check(g, t.cpu(), long * e.cpu(), (n, d))
    leaves = [t.to(DEV).requires_grad_() for t in (x, w, b)]
    dy = dy.to(DEV)
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=st):
        y = hip_ops.layer_norm(*leaves, act8=act8)
        outs = [y.detach()] + list(torch.autograd.grad(y, leaves, dy))
    for _ in range(3):
        for o in outs:
            o.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(outs, got))
