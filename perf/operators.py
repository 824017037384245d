"""Measured cases of the 8-bit training operators: layer norm, 8-bit activation checkpoints, block-scaled 8-bit products.

The number format they share: the values of 128 neighbours of a row (of a 128 x 128 block, for a weight) are held as e4m3
numbers times ONE power of two 2^E, with E the smallest exponent for which the block's largest magnitude is at most 448 * 2^E.
Multiplying by a power of two is exact, so an 8-bit value does not depend on how it was computed.

  norm      y = (x - mean) / sqrt(var + eps) * w + b over the last axis; its backward pass from x, or from x's 8-bit checkpoint
  pack      x -> checkpoint -> x
  product   y = Q(x) Q(W)^T + b with a weight laid out once (serving)
  linear    one training step of the same layer: y, dx = Q(dy) Q(W), dW = dy^T Q(x), db = sum dy; Q(x) is the checkpoint

``own`` selects the framework's operators (hcmoco_amd.hip_ops); otherwise the same in elementary torch operations.
"""
import math

import torch

own = False

EPS = 1e-5
TYPES = {'fp32': torch.float32, 'bf16': torch.bfloat16, 'fp16': torch.float16}


# --------------------------------------------------------------------------- #
# cases
# --------------------------------------------------------------------------- #
def listed():
    return [
        # the joint features of one training batch: 32 skeletons x 17 joints, 128 channels (latency counts)
        dict(name='norm_joints', op='norm', rows=544, cols=128, dtype='fp32', train=True, act8=False),
        # one row, no gradient: a feature vector answered by itself
        dict(name='norm_row', op='norm', rows=1, cols=1024, dtype='fp16', train=False, act8=False),
        # the merged HRNet-w18 maps of a batch, normalised per pixel: 32 x 64 x 64 pixels, 18 + 36 + 72 + 144 channels
        dict(name='norm_pixels', op='norm', rows=131072, cols=270, dtype='fp32', train=True, act8=False),
        # a long batch of wide rows whose input is kept in 8 bits until the backward pass
        dict(name='norm_wide_act8', op='norm', rows=16384, cols=4096, dtype='bf16', train=True, act8=True),
        # a checkpoint of the joint features, written and read back
        dict(name='pack_joints', op='pack', rows=544, cols=128, dtype='fp32'),
        # a checkpoint of half a gigabyte of activations
        dict(name='pack_wide', op='pack', rows=65536, cols=4096, dtype='bf16'),
        # a single row through a laid-out weight: bound by reading the weight
        dict(name='product_row', op='product', rows=1, outs=4096, cols=4096, dtype='bf16', bias=False),
        # no size a multiple of anything
        dict(name='product_ragged', op='product', rows=997, outs=1501, cols=1290, dtype='fp16', bias=True),
        # a product that the matrix cores bound
        dict(name='product_large', op='product', rows=8192, outs=8192, cols=8192, dtype='bf16', bias=False),
        # the projection head of one batch, pooled channels of HRNet-w18 -> 128 features, one training step
        dict(name='linear_heads', op='linear', rows=32, outs=128, cols=270, dtype='fp32', bias=True),
        # the same projection at every pixel of the merged maps
        dict(name='linear_pixels', op='linear', rows=131072, outs=128, cols=270, dtype='fp32', bias=True),
        # a wide layer on many rows, fp32 weights under bf16 activations
        dict(name='linear_wide', op='linear', rows=8192, outs=4096, cols=4096, dtype='bf16', bias=True),
    ]


def _log_size(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))


def draw(rng):
    op = rng.choice(['norm', 'norm', 'pack', 'product', 'product', 'linear', 'linear'])
    dtype = rng.choice(['fp32', 'bf16', 'fp16'])
    if op in ('norm', 'pack'):
        # under 8 columns the gradient of a norm is the rounding error of its own cancellation: not a measurement
        cols = _log_size(rng, 8 if op == 'norm' else 1, 8192)
        rows = _log_size(rng, 1, min(1 << 17, (1 << 26) // cols))
        if op == 'pack':
            return dict(op=op, rows=rows, cols=cols, dtype=dtype)
        train = rng.random() < 0.7
        return dict(op=op, rows=rows, cols=cols, dtype=dtype, train=train, act8=train and rng.random() < 0.5)
    cols, outs = _log_size(rng, 16, 8192), _log_size(rng, 1, 8192)
    most = (1 << 39) if op == 'product' else (1 << 37)
    rows = _log_size(rng, 1, max(1, min(1 << 13 if op == 'product' else 1 << 17, most // (cols * outs), (1 << 28) // max(cols, outs))))
    return dict(op=op, rows=rows, outs=outs, cols=cols, dtype=dtype, bias=rng.random() < 0.5)


# --------------------------------------------------------------------------- #
# inputs
# --------------------------------------------------------------------------- #
def _activations(gen, rows, cols, dtype):
    """Features with channels of different strength and offset, and a few channels far above the others."""
    spread = torch.exp(0.5 * torch.randn(cols, generator=gen, device='cuda'))
    spread = torch.where(torch.rand(cols, generator=gen, device='cuda') < 0.01, spread * 20, spread)
    offset = 0.3 * torch.randn(cols, generator=gen, device='cuda')
    return torch.randn(rows, cols, generator=gen, device='cuda').mul_(spread).add_(offset).to(dtype)


def _gradients(gen, rows, cols, dtype):
    """Loss gradients: small, and rows of very different size."""
    size = 1e-2 * torch.exp(torch.randn(rows, 1, generator=gen, device='cuda'))
    return (torch.randn(rows, cols, generator=gen, device='cuda') * size).to(dtype)


def _weights(gen, outs, cols, dtype):
    return (torch.randn(outs, cols, generator=gen, device='cuda') / math.sqrt(cols)).to(dtype)


def _tensors(case, seed):
    gen = torch.Generator(device='cuda').manual_seed(int(seed))
    dtype = TYPES[case['dtype']]
    rows, cols, op = case['rows'], case['cols'], case['op']
    s = {'x': _activations(gen, rows, cols, dtype)}
    if op == 'norm':
        s['w'] = 1 + 0.2 * torch.randn(cols, generator=gen, device='cuda')
        s['b'] = 0.2 * torch.randn(cols, generator=gen, device='cuda')
        if case['train']:
            s['dy'] = _gradients(gen, rows, cols, dtype)
    elif op != 'pack':
        outs = case['outs']
        s['w'] = _weights(gen, outs, cols, torch.float32 if op == 'linear' else dtype)
        s['b'] = 0.1 * torch.randn(outs, generator=gen, device='cuda') if case['bias'] else None
        if op == 'linear':
            s['dy'] = _gradients(gen, rows, outs, dtype)
    return s


def prepare(case, seed):
    s = _tensors(case, seed)
    s['case'] = case
    if case['op'] == 'product':
        # a serving program keeps the weight as it laid it out, not the weight that it was laid out from
        if own:
            from hcmoco_amd import hip_ops
            s['kept'] = hip_ops.fp8_weight(s.pop('w'))
        else:
            s['kept'] = _held_in_8_bits(s.pop('w').float(), 128)
    elif case['op'] == 'linear' or case.get('train'):
        for k in ('x', 'w', 'b'):
            if s[k] is not None:
                s[k].requires_grad_(own)
    return s


# --------------------------------------------------------------------------- #
# one pass
# --------------------------------------------------------------------------- #
def run(s):
    return _run_own(s) if own else _run_plain(s)


def _run_own(s):
    from hcmoco_amd import hip_ops
    case, x, b = s['case'], s['x'], s.get('b')
    if case['op'] == 'pack':
        return hip_ops.act8_unpack(hip_ops.act8_pack(x))
    if case['op'] == 'product':
        return hip_ops.fp8_linear(x, s['kept'], b)
    if case['op'] == 'norm':
        y = hip_ops.layer_norm(x, s['w'], b, EPS, act8=case['act8'])
        if not case['train']:
            return y
    else:
        y = hip_ops.fp8_linear(x, s['w'], b)
    leaves = [s['x'], s['w']] + ([b] if b is not None else [])
    return [y.detach()] + list(torch.autograd.grad(y, leaves, s['dy']))


def _power_of_two(e):
    """2^e in float32, by its bits: -126 <= e <= 127."""
    return ((e + 127) << 23).view(torch.float32)


def _held_in_8_bits(x, block_rows):
    """The float32 values that the 8-bit blocks of x [rows, cols] stand for."""
    rows, cols = x.shape
    br = min(block_rows, rows)
    pr, pc = -rows % br, -cols % 128
    v = torch.nn.functional.pad(x, (0, pc, 0, pr)).reshape((rows + pr) // br, br, (cols + pc) // 128, 128)
    amax = v.abs().amax(dim=(1, 3), keepdim=True)
    m, e = torch.frexp(amax)                                    # amax = m 2^e, 1/2 <= m < 1;  448 = 0.875 * 2^9
    e = torch.where(amax > 0, torch.where(m > 0.875, e - 8, e - 9).clamp(-126, 127), torch.zeros_like(e)).int()
    q = (v * _power_of_two(-e)).to(torch.float8_e4m3fn).float()
    return (q * _power_of_two(e)).reshape(rows + pr, cols + pc)[:rows, :cols]


def _run_plain(s):
    case, x, b = s['case'], s['x'].detach(), s.get('b')
    dtype, xf = x.dtype, x.detach().float()
    if case['op'] == 'pack':
        top = torch.finfo(dtype).max
        return _held_in_8_bits(xf, 1).clamp(-top, top).to(dtype)
    if case['op'] == 'product':
        y = _held_in_8_bits(xf, 1) @ s['kept'].t()
        return (y if b is None else y + b).to(dtype)
    w = s['w'].detach()
    if case['op'] == 'norm':
        mean = xf.mean(1, keepdim=True)
        centred = xf - mean
        rstd = torch.rsqrt((centred * centred).mean(1, keepdim=True) + EPS)
        y = (centred * rstd * w + b).to(dtype)
        if not case['train']:
            return y
        xhat = ((_held_in_8_bits(xf, 1) - mean) if case['act8'] else centred) * rstd
        dy = s['dy'].float()
        g = dy * w
        dx = rstd * (g - g.mean(1, keepdim=True) - xhat * (g * xhat).mean(1, keepdim=True))
        return [y, dx.to(dtype), (dy * xhat).sum(0), dy.sum(0)]
    dy = s['dy'].float()
    xq, wq = _held_in_8_bits(xf, 1), _held_in_8_bits(w, 128)
    y = xq @ wq.t()
    y = (y if b is None else y + b).to(dtype)
    out = [y, (_held_in_8_bits(dy, 1) @ wq).to(dtype), dy.t() @ xq]
    return out + [dy.sum(0)] if b is not None else out


# --------------------------------------------------------------------------- #
# what a pass cannot do without
# --------------------------------------------------------------------------- #
def work(case):
    size = {'fp32': 4, 'bf16': 2, 'fp16': 2}[case['dtype']]
    rows, cols, op = case['rows'], case['cols'], case['op']
    n = rows * cols
    if op == 'pack':              # the checkpoint (a byte a value, a byte a block) is written and read: it outlives the pass
        return dict(bytes=2 * n * size + 2 * (n + rows * -(-cols // 128)), flops=4 * n)
    if op == 'norm':
        return dict(bytes=n * size * (4 if case['train'] else 2) + 4 * cols * (4 if case['train'] else 2),
                    flops=n * (20 if case['train'] else 8))
    outs = case['outs']
    if op == 'product':
        return dict(bytes=n * size + outs * cols + rows * outs * size, flops=2 * n * outs)
    return dict(bytes=2 * (n + rows * outs) * size + 8 * outs * cols, flops=6 * n * outs)


# --------------------------------------------------------------------------- #
# the same in 64 bits, from the definitions
# --------------------------------------------------------------------------- #
def _two64(e):
    return ((e.long() + 1023) << 52).view(torch.float64)


def _q64(x, tall):
    """Blocks one after the other along the columns: the largest magnitude, the exponent, round to 4 significant bits (ties to
    even) above 2^-6 and to multiples of 2^-9 below."""
    out = torch.empty(x.shape, dtype=torch.float64, device=x.device)
    for c in range(0, x.shape[1], 128):
        part = x[:, c:c + 128].double()
        top = part.abs().amax(1)
        if tall:
            top = torch.cat([t.max().expand(len(t)) for t in top.split(128)])
        # 2^E >= top / 448: the ratio is exact to 2^-53, and a power of two exactly where top is 448 2^E
        m, e = torch.frexp(top / 448)
        e = torch.where(m == 0.5, e - 1, e)
        e = torch.where(top > 0, e, torch.zeros_like(e)).clamp(-126, 127)[:, None]
        v = part * _two64(-e)
        step = _two64((torch.frexp(v)[1] - 4).clamp(min=-9))
        out[:, c:c + 128] = torch.round(v / step) * step * _two64(e)
    return out


def exact(case, seed):
    s = _tensors(case, seed)
    x = s['x']
    b = s['b'].double() if s.get('b') is not None else None
    if case['op'] == 'pack':
        top = torch.finfo(x.dtype).max
        return _q64(x, False).clamp(-top, top)
    if case['op'] == 'product':
        y = torch.mm(_q64(x, False), _q64(s['w'], True).t().contiguous())
        return y if b is None else y + b
    w, x64 = s['w'].double(), x.double()
    if case['op'] == 'norm':
        var, mean = torch.var_mean(x64, dim=1, unbiased=False, keepdim=True)
        sd = torch.sqrt(var + EPS)
        y = (x64 - mean) / sd * w + b
        if not case['train']:
            return y
        if case['act8']:
            x64 = _q64(x, False)
        h = (x64 - mean) / sd
        dy = s['dy'].double()
        dh = dy * w
        dx = (dh - dh.mean(1, keepdim=True) - h * (dh * h).mean(1, keepdim=True)) / sd
        return [y, dx, (dy * h).sum(0), dy.sum(0)]
    dy, xq, wq = s['dy'].double(), _q64(x, False), _q64(s['w'], True)
    y = torch.mm(xq, wq.t().contiguous())
    out = [y if b is None else y + b, torch.mm(_q64(s['dy'], False), wq), torch.mm(dy.t().contiguous(), xq)]
    return out + [dy.sum(0)] if b is not None else out
