"""The backward passes of hip_ops.layer_norm and hip_ops.fp8_linear on saved tensors that come back from a saved-tensor hook in another
layout or on other memory.  The values are the same, so the gradients have to be, bit for bit; what is not the tensor that was
saved is refused."""
import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = 'cuda:0'
TYPES = [torch.float32, torch.bfloat16, torch.float16]


def _room(t, skip):
    """t's values on memory that begins ``skip`` elements into another tensor."""
    r = torch.empty(t.numel() + skip, dtype=t.dtype, device=t.device)
    r[skip:] = t.reshape(-1)
    return r[skip:].view(t.shape)


def _strided(t):
    """t's values with gaps between the elements of every axis."""
    r = torch.empty([2 * n for n in t.shape], dtype=t.dtype, device=t.device)
    v = r[tuple(slice(None, None, 2) for _ in t.shape)]
    v.copy_(t)
    return v


# what a hook may hand back for a saved tensor
BACK = {
    'save_on_cpu': lambda: torch.autograd.graph.save_on_cpu(),
    'contiguous': lambda: torch.autograd.graph.saved_tensors_hooks(lambda t: t.detach().clone(memory_format=torch.contiguous_format), lambda t: t),
    'strided': lambda: torch.autograd.graph.saved_tensors_hooks(lambda t: t.detach().clone(), _strided),
    'begins_anywhere': lambda: torch.autograd.graph.saved_tensors_hooks(lambda t: t.detach().clone(), lambda t: _room(t, 1)),
    'as_it_is': lambda: torch.autograd.graph.saved_tensors_hooks(lambda t: t.detach(), lambda t: t),
}


def _views(dtype):
    g = torch.Generator().manual_seed(5)
    wide = torch.randn(40, 333, generator=g).to(dtype).to(DEV)
    return {
        'whole': wide, 'columns': wide[:, 3:273], 'rows': wide[::3], 'columns_of_rows': wide[5:38, 1:130], 'transposed': wide.t(),
        'three_axes': wide[:, :300].reshape(40, 3, 100), 'every_second': wide[:, ::2],
    }


def _grads(op, leaves, dy):
    y = op(*leaves)
    return torch.autograd.grad(y, [t for t in leaves if t.requires_grad], dy)


@pytest.mark.parametrize('back', sorted(BACK))
@pytest.mark.parametrize('act8', [False, True])
@pytest.mark.parametrize('dtype', TYPES)
def test_layer_norm(dtype, act8, back):
    from hcmoco_amd import hip_ops
    for name, v in _views(dtype).items():
        C = v.shape[-1]
        g = torch.Generator().manual_seed(C)
        leaves = [v.detach().requires_grad_()] + [torch.randn(C, generator=g).to(DEV).requires_grad_() for _ in range(2)]
        assert leaves[0].stride() == v.stride()
        dy = torch.randn(v.shape, generator=g).to(dtype).to(DEV)
        op = lambda *a: hip_ops.layer_norm(*a, act8=act8)
        want = _grads(op, leaves, dy)
        with BACK[back]():
            got = _grads(op, leaves, dy)
        for a, b in zip(got, want):
            assert torch.equal(a, b), name


@pytest.mark.parametrize('back', sorted(BACK))
@pytest.mark.parametrize('dtype', TYPES)
def test_linear(dtype, back):
    from hcmoco_amd import hip_ops
    for name, v in _views(dtype).items():
        K, N = v.shape[-1], 90
        g = torch.Generator().manual_seed(K)
        w, b = torch.randn(N, K, generator=g).to(DEV), torch.randn(N, generator=g).to(DEV)
        dy = torch.randn(tuple(v.shape[:-1]) + (N,), generator=g).to(dtype).to(DEV)
        kept = hip_ops.fp8_weight(w)
        for op, leaves in ((hip_ops.fp8_linear, [v, w, b]), (lambda x, c: hip_ops.fp8_linear(x, kept, c), [v, b])):
            leaves = [t.detach().requires_grad_() for t in leaves]
            want = _grads(op, leaves, dy)
            with BACK[back]():
                got = _grads(op, leaves, dy)
            for p, q in zip(got, want):
                assert torch.equal(p, q), name


@pytest.mark.parametrize('wrong', ['short', 'flat', 'type', 'device'])
def test_something_else_is_refused(wrong):
    """Each of the saved tensors in turn."""
    from hcmoco_amd import hip_ops
    change = {'short': lambda t: t[:-1], 'flat': lambda t: t.reshape(-1, 1), 'device': lambda t: t.cpu(),
              'type': lambda t: t.to(torch.int16 if t.dtype == torch.uint8 else torch.float64)}[wrong]
    x, w, b = torch.randn(40, 333, device=DEV), torch.randn(90, 333, device=DEV), torch.randn(90, device=DEV)
    kept = hip_ops.fp8_weight(w)
    ops = {'norm': (lambda x, w: hip_ops.layer_norm(x, w), [x, w[0]]), 'norm8': (lambda x, w: hip_ops.layer_norm(x, w, act8=True), [x, w[0]]),
           'linear': (hip_ops.fp8_linear, [x, w, b]), 'kept': (lambda x: hip_ops.fp8_linear(x, kept), [x])}
    for name, (op, leaves) in ops.items():
        leaves = [t.detach().clone().requires_grad_() for t in leaves]
        plain = []
        with torch.autograd.graph.saved_tensors_hooks(lambda t: plain.append(t) or t, lambda t: t):
            op(*leaves)
        assert plain, name
        for k in range(len(plain)):
            seen = []
            with torch.autograd.graph.saved_tensors_hooks(lambda t: (t.detach(), seen.append(t) or len(seen) - 1),
                                                          lambda p: change(p[0]) if p[1] == k else p[0]):
                y = op(*leaves)
                with pytest.raises(RuntimeError):
                    torch.autograd.grad(y, leaves, torch.ones_like(y))


@pytest.mark.parametrize('reentrant', [False, True])
def test_under_activation_checkpointing(reentrant):
    from hcmoco_amd import hip_ops
    from torch.utils.checkpoint import checkpoint
    g = torch.Generator().manual_seed(8)
    wide = torch.randn(60, 333, generator=g).to(DEV)
    p = [torch.randn(s, generator=g).to(DEV) for s in ((270,), (270,), (90, 270), (90,), (90,), (40, 90))]
    dy = torch.randn(60, 40, generator=g).to(DEV)

    def block(x, w1, b1, W1, B1, w2, W2):
        h = hip_ops.fp8_linear(hip_ops.layer_norm(x, w1, b1), W1, B1)
        return hip_ops.fp8_linear(hip_ops.layer_norm(h, w2, act8=True), W2)
    leaves = [t.detach().requires_grad_() for t in [wide[:, 3:273]] + p]
    want = _grads(block, leaves, dy)
    y = checkpoint(block, *leaves, use_reentrant=reentrant)
    y.backward(dy)
    assert all(torch.equal(t.grad, q) for t, q in zip(leaves, want))
