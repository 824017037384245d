"""hip_ops.layer_norm and hip_ops.fp8_linear under ways of differentiating that they have no rule for: they raise, and never hand back
a result whose derivative is silently missing."""
import pytest
import torch
import torch.autograd.forward_ad as fw

pytestmark = pytest.mark.gpu

DEV = 'cuda:0'


def _ops():
    from hcmoco_amd import hip_ops
    g = torch.Generator().manual_seed(0)
    x, w, b = (torch.randn(s, generator=g).to(DEV) for s in ((20, 140), (90, 140), (90,)))
    kept = hip_ops.fp8_weight(w)
    return [('norm', lambda x, w, b: hip_ops.layer_norm(x, w, b), [x, w[0].contiguous(), w[1].contiguous()]),
            ('norm8', lambda x, w, b: hip_ops.layer_norm(x, w, b, act8=True), [x, w[0].contiguous(), w[1].contiguous()]),
            ('linear', hip_ops.fp8_linear, [x, w, b]), ('kept', lambda x, b: hip_ops.fp8_linear(x, kept, b), [x, b])]


@pytest.mark.parametrize('needs', [False, True])
@pytest.mark.parametrize('record', [False, True])
def test_a_tangent_is_refused_in_every_place(record, needs):
    for name, op, args in _ops():
        clean = op(*args)
        for k in range(len(args)):
            leaves = [t.detach().requires_grad_(needs) for t in args]
            with fw.dual_level(), torch.set_grad_enabled(record):
                leaves[k] = fw.make_dual(leaves[k], torch.ones_like(leaves[k]))
                with pytest.raises(NotImplementedError, match='forward-mode'):
                    op(*leaves)
                # the primal by itself is an ordinary tensor
                leaves[k] = fw.unpack_dual(leaves[k]).primal.detach()
                assert torch.equal(op(*leaves), clean), (name, k)
            assert torch.equal(op(*args), clean), (name, k)


def test_where_torch_itself_propagates_no_tangent():
    for name, op, args in _ops():
        with fw.dual_level():
            duals = [fw.make_dual(t, torch.ones_like(t)) for t in args]
            with torch.inference_mode():
                assert torch.equal(op(*duals), op(*args)), name


def test_function_transforms():
    """jvp and grad raise; vmap is torch's loop over the calls, its results those of the calls, and differentiable."""
    for name, op, args in _ops():
        rest = args[1:]
        with pytest.raises(RuntimeError):
            torch.func.jvp(lambda t: op(t, *rest), (args[0],), (torch.ones_like(args[0]),))
        with pytest.raises(RuntimeError):
            torch.func.grad(lambda t: op(t, *rest).sum())(args[0])
        x = args[0].detach().requires_grad_()
        y = torch.func.vmap(lambda t: op(t[None], *rest))(x)[:, 0]
        want = torch.cat([op(x[i:i + 1], *rest) for i in range(len(x))])
        assert torch.equal(y, want), name
        dy = torch.randn_like(y)
        assert torch.equal(*[torch.autograd.grad(t, x, dy)[0] for t in (y, want)]), name
