"""GPU: gradients of the rotation through autograd."""
import pytest
import torch

from tests import kv_reference as R
from tests.test_gpu_kv_operators import BF, FP, _close, _gen, _randn

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("t,h,d,rot,dtype,interleaved", [(5, 3, 64, 64, BF, False), (33, 8, 128, 64, FP, True), (1, 1, 66, 18, BF, False),
                                                         (700, 4, 128, 128, FP, False)])
def test_gradient(cuda_device, t, h, d, rot, dtype, interleaved):
    """The gradient is the transposed rotation of the result's gradient, for heads of a packed leaf too; the values are those of
    a call without gradients; the gradient's gradient is the rotation again."""
    from unified_cache_management_b200 import ops
    g = _gen(t)
    f, _ = ops.rotary_frequencies(rot, device="cuda")
    pos = torch.randint(0, 100000, (t,), device="cuda", generator=g)
    kw = dict(interleaved=interleaved, mscale=1.25)
    packed = _randn((t, h + 2, d), g, dtype).requires_grad_()
    dy = _randn((t, h, d), g, dtype)
    y = ops.rotary(packed[:, 1:h + 1], pos, f, **kw)
    assert y.requires_grad and torch.equal(y, ops.rotary(packed.detach()[:, 1:h + 1], pos, f, **kw))
    y.backward(dy)
    want = R.rotate(dy, pos, f, interleaved, 1.25, True)
    _close(packed.grad[:, 1:h + 1], want, R.half_step(dtype, want) + R.rotate_slack(dy, f, interleaved, 1.25), "gradient")
    assert int(packed.grad[:, 0].count_nonzero()) == int(packed.grad[:, h + 1].count_nonzero()) == 0
    x, w = packed.detach()[:, 1:h + 1].clone().requires_grad_(), dy.clone().requires_grad_()
    grad, = torch.autograd.grad(ops.rotary(x, pos, f, transpose=True, **kw), x, w, create_graph=True)
    assert torch.equal(grad, ops.rotary(w.detach(), pos, f, **kw))
    again, = torch.autograd.grad(grad, w, x.detach())
    assert torch.equal(again, ops.rotary(x.detach(), pos, f, transpose=True, **kw))


def test_gradient_of_a_sum_and_without_grad(cuda_device):
    from unified_cache_management_b200 import ops
    f, _ = ops.rotary_frequencies(32, device="cuda")
    pos = torch.arange(9, device="cuda")
    x = _randn((9, 2, 64), _gen(1), BF).requires_grad_()
    ops.rotary(x, pos, f).sum().backward()                     # (the gradient comes with strides of 0)
    one = torch.ones((9, 2, 64), device="cuda", dtype=BF)
    assert torch.equal(x.grad, ops.rotary(one, pos, f, transpose=True))
    with torch.no_grad():
        assert not ops.rotary(x, pos, f).requires_grad
    empty = torch.empty((0, 2, 64), device="cuda", dtype=BF, requires_grad=True)
    ops.rotary(empty, pos[:0], f).sum().backward()
    assert empty.grad.shape == (0, 2, 64)


def test_refusals(cuda_device):
    from unified_cache_management_b200 import ops
    f, _ = ops.rotary_frequencies(32, device="cuda")
    pos = torch.arange(3, device="cuda")
    x = torch.zeros((3, 2, 64), device="cuda", dtype=BF, requires_grad=True)
    for kw in (dict(out=torch.empty_like(x)), dict(out=x)):
        with pytest.raises(ValueError):
            ops.rotary(x, pos, f, **kw)
        with torch.no_grad():
            ops.rotary(x, pos, f, **kw)
    with pytest.raises(ValueError):
        ops.rotary(x.detach(), pos, f.clone().requires_grad_())
    # positions that have changed since are not used
    y = ops.rotary(x, pos, f)
    pos += 1
    with pytest.raises(RuntimeError):
        y.sum().backward()
