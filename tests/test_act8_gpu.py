"""8-bit activation checkpoints (hip_ops.act8_pack / act8_unpack) against the format's definition in float64.  The format is
exact arithmetic (a power of two, one rounding), so every comparison is for equality."""
import pytest
import torch

from act8_ref import held8

pytestmark = pytest.mark.gpu

DEV = 'cuda:0'
TYPES = [torch.float32, torch.bfloat16, torch.float16]


def _x(rows, cols, dtype, seed, spread=3.0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(rows, cols, generator=g) * torch.exp(spread * torch.randn(rows, 1, generator=g))
    return x.clamp(-6e4, 6e4).to(dtype)


def _same(a, b):
    a, b = a.double().cpu(), b.double()
    assert torch.equal(a.isnan(), b.isnan())
    assert torch.equal(a.nan_to_num(), b.nan_to_num())


@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('rows,cols', [(1, 1), (3, 7), (1, 128), (2, 129), (544, 128), (33, 270), (5, 1000), (1, 4096), (700, 257),
                                       (4099, 16), (64, 8192), (3, 20001)])
def test_round_trip_is_the_format(rows, cols, dtype):
    from hcmoco_amd import hip_ops
    x = _x(rows, cols, dtype, rows * 31 + cols)
    p = hip_ops.act8_pack(x.to(DEV))
    want, e = held8(x)
    back = hip_ops.act8_unpack(p, torch.float32)
    _same(back, want)
    kb = (cols + 127) // 128
    assert torch.equal(p.scale.cpu()[:, :kb].long(), e.long() + 127)
    assert (p.scale.cpu()[:, kb:] == 127).all() and (p.q.cpu()[:, cols:] == 0).all()
    # the bytes are e4m3: torch reads the same values out of them
    bytes_ = p.q.cpu().view(torch.float8_e4m3fn).double()[:, :cols]
    _same(bytes_ * torch.repeat_interleave(torch.exp2(e.double()), 128, 1)[:, :cols], want)
    own = hip_ops.act8_unpack(p)
    assert own.dtype == dtype and own.shape == x.shape
    top = torch.finfo(dtype).max
    _same(own, want.clamp(-top, top).to(dtype).double())


def test_borders_of_the_scale_and_of_the_rounding():
    from hcmoco_amd import hip_ops
    rows = []
    for e in (-130, -126, -100, -20, -1, 0, 1, 30, 118, 119):
        for f in (448.0, 448.0 * (1 + 2.0 ** -23), 448.0 * (1 - 2.0 ** -24), 224.0, 256.0, 1.0):
            v = f * 2.0 ** e
            if abs(v) < 3.4e38:
                rows.append([v, -v / 2, v * 17 / 32, v * 2.0 ** -9, v * 2.0 ** -18, 0.0, -0.0, v / 3])
    # every tie between neighbouring e4m3 values, next to a 448 that fixes the scale
    grid = torch.arange(127, dtype=torch.uint8).view(torch.float8_e4m3fn).double()
    mids = ((grid[1:] + grid[:-1]) / 2).tolist()
    rows += [[448.0] + mids[i:i + 7] for i in range(0, len(mids), 7)]
    rows[-1] += [0.0] * (8 - len(rows[-1]))
    x = torch.tensor(rows, dtype=torch.float64).float()
    _same(hip_ops.act8_unpack(hip_ops.act8_pack(x.to(DEV))), held8(x)[0].clamp(-3.4028234663852886e38, 3.4028234663852886e38))


@pytest.mark.parametrize('dtype', TYPES)
def test_values_that_are_not_finite_stay_where_they_are(dtype):
    from hcmoco_amd import hip_ops
    x = _x(4, 300, dtype, 5)
    x[0, 3], x[0, 130], x[1, 299], x[2] = float('nan'), float('inf'), float('-inf'), float('nan')
    got = hip_ops.act8_unpack(hip_ops.act8_pack(x.to(DEV)), torch.float32)
    _same(got, held8(x)[0])
    assert int(got.isnan().sum()) == 3 + 300


def test_largest_values_stay_finite():
    from hcmoco_amd import hip_ops
    for dtype in TYPES:
        top = torch.finfo(dtype).max
        x = torch.tensor([[top, -top, top / 2, 1.0]], dtype=dtype, device=DEV)
        y = hip_ops.act8_unpack(hip_ops.act8_pack(x))
        assert torch.isfinite(y).all() and y[0, 0] == top and y[0, 1] == -top


def test_views_shapes_and_empty():
    from hcmoco_amd import hip_ops
    x = _x(37, 700, torch.bfloat16, 9).to(DEV)
    for v in (x[:, 3:303], x[::2], x[5:6], x.t(), x.reshape(37, 7, 100), x[0], x[:, ::2], x.flatten()[1:1 + 37 * 18].view(37, 18)):
        p = hip_ops.act8_pack(v)
        got = hip_ops.act8_unpack(p)
        assert got.shape == v.shape
        _same(got.reshape(-1, v.shape[-1]), held8(v.reshape(-1, v.shape[-1]))[0])
    e = hip_ops.act8_pack(x[:0])
    assert hip_ops.act8_unpack(e).shape == (0, 700) and e.nbytes() == 0


def test_checkpoint_is_a_quarter_of_float32():
    from hcmoco_amd import hip_ops
    x = torch.zeros(1024, 512, device=DEV)
    assert hip_ops.act8_pack(x).nbytes() == 1024 * (512 + 4)


def test_on_a_side_stream_and_in_a_graph():
    from hcmoco_amd import hip_ops
    a, b = _x(64, 270, torch.float32, 1), _x(64, 270, torch.float32, 2)
    st = torch.cuda.Stream()
    x = a.to(DEV)
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        y = hip_ops.act8_unpack(hip_ops.act8_pack(x))
    st.synchronize()
    _same(y, held8(a)[0])
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        y = hip_ops.act8_unpack(hip_ops.act8_pack(x))
    for src in (b, a, b, a):
        x.copy_(src)
        g.replay()
        eager = hip_ops.act8_unpack(hip_ops.act8_pack(x))
        torch.cuda.synchronize()
        assert torch.equal(y, eager)
        _same(y, held8(src)[0])


def test_refuses():
    from hcmoco_amd import hip_ops
    x = torch.zeros(4, 8, device=DEV)
    with pytest.raises(TypeError):
        hip_ops.act8_pack(x.double())
    with pytest.raises(ValueError):
        hip_ops.act8_pack(x[:, :0])
    with pytest.raises(TypeError):
        hip_ops.act8_unpack(x)
    p = hip_ops.act8_pack(x)
    with pytest.raises(TypeError):
        hip_ops.act8_unpack(p, torch.int8)
    with pytest.raises(ValueError):
        hip_ops.act8_unpack(hip_ops.Act8(p.q[:2], p.scale, p.shape, p.dtype))
    with pytest.raises(ValueError):
        hip_ops.act8_unpack(hip_ops.Act8(p.q, p.scale, (4, 400), p.dtype))


def test_offsets_past_32_bits():
    """Tensors of more than 2^32 values: the last rows come out as they do by themselves.  Whole numbers, whose products' sums are
    exact in any order."""
    from hcmoco_amd import hip_ops
    M, C, last = (1 << 20) + 3001, 4096, 300
    if torch.cuda.mem_get_info()[0] < 110 << 30:
        pytest.skip('needs 110 GB of device memory')
    x = torch.randint(-3, 4, (M, C), device=DEV, dtype=torch.bfloat16)
    tail = x[-last:].clone()
    packed, small = hip_ops.act8_pack(x), hip_ops.act8_pack(tail)
    assert torch.equal(packed.q[-last:], small.q) and torch.equal(packed.scale[-last:], small.scale)
    assert torch.equal(hip_ops.act8_unpack(packed)[-last:], tail)
    del packed

    w = torch.randint(-2, 3, (C, C), device=DEV, dtype=torch.bfloat16)
    b = torch.randint(-2, 3, (C,), device=DEV, dtype=torch.bfloat16)
    dy = torch.zeros_like(x)
    dy[-last:] = torch.randint(-2, 3, (last, C), device=DEV, dtype=torch.bfloat16)

    def grads(op, *leaves):
        leaves = [t.detach().requires_grad_() for t in leaves]
        y = op(*leaves)
        return [y.detach()] + list(torch.autograd.grad(y, leaves, dy[-leaves[0].shape[0]:]))
    for act8 in (False, True, None):
        op = hip_ops.fp8_linear if act8 is None else (lambda *a: hip_ops.layer_norm(*a, act8=act8))
        p = (w if act8 is None else w[0].contiguous(), b)
        big, little = grads(op, x, *p), grads(op, tail, *p)
        for k in (0, 1):
            assert torch.equal(big[k][-last:], little[k]), (act8, k)
        for k in (2, 3):
            if act8 is None:
                assert torch.equal(big[k], little[k]), k
            else:       # sums of 300 rows in another order (2^-24 a step), then bf16
                mag = dy[-last:].double().abs().sum(0) * (1 if k == 3 else 4096 ** 0.5)
                err = 300 * 2.0 ** -24 * mag + 2.0 ** -8 * little[k].double().abs() * 2
                assert bool(((big[k].double() - little[k].double()).abs() <= err).all()), (act8, k)
        del big, little
    del x, dy, tail
    torch.cuda.empty_cache()
