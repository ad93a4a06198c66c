"""Weights and biases of qk_norm_rope in other shapes and types."""
import pytest
import torch

import trinix_b200 as T
from tests.test_gpu_qk_norm_rope import angles, check_forward, make, tables

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("shape", [(64,), (1, 64), (1, 1, 64), (8, 8)], ids=str)
def test_gradients_have_the_parameters_shapes(cuda, shape):
    q, k, w, b = make(2, 5, 4, 2, 64, torch.bfloat16, cuda, "layernorm")
    cos, sin = tables(5, 64, cuda)
    grads = []
    for how in ((64,), shape):
        leaves = [t.clone().view(how).requires_grad_() for t in (*w, *b)]
        y = T.QKNormRoPEKernel.apply(q, k, leaves[0], leaves[1], cos, sin, leaves[2], leaves[3], 1e-5, "layernorm", False)
        (y[0].float().square().sum() + y[1].float().sum()).backward()
        assert all(t.grad.shape == t.shape and t.grad.dtype == t.dtype for t in leaves)
        grads.append([t.grad.flatten() for t in leaves])
    assert all(torch.equal(x, y) for x, y in zip(*grads))


@pytest.mark.parametrize("which", [(2,), (3,), (2, 3)], ids=str)
def test_one_bias_alone(cuda, which):
    q, k, w, b = make(1, 5, 2, 2, 64, torch.bfloat16, cuda, "layernorm")
    cos, sin = tables(5, 64, cuda)
    leaves = [t.clone().view(1, 64).requires_grad_() if i in which or i < 2 else None for i, t in enumerate((*w, *b))]
    y = T.QKNormRoPEKernel.apply(q, k, leaves[0], leaves[1], cos, sin, leaves[2], leaves[3], 1e-5, "layernorm")
    (y[0].float().square().sum() + y[1].float().sum()).backward()
    assert all(t.grad.shape == t.shape for t in leaves if t is not None)


BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


@pytest.mark.parametrize("types", [(BF16, F32, BF16, BF16), (BF16, BF16, F32, F32), (F32, BF16, F16, BF16), (F16, BF16, F16, BF16)],
                         ids=str)
@pytest.mark.parametrize("first", [True, False], ids=["first", "last"])
def test_parameters_of_several_types(cuda, first, types):
    """Each is read with all its digits, and its gradient is rounded to its own type once."""
    q, k, w, b = make(2, 7, 4, 2, 64, F32, cuda, "layernorm")
    cos, sin = tables(7, 64, cuda)
    params = [(t + 1 / 3).to(x).requires_grad_() for t, x in zip((*w, *b), types)]
    y = T.QKNormRoPEKernel.apply(q, k, params[0], params[1], cos, sin, params[2], params[3], 1e-5, "layernorm", first)
    dy = [torch.randn(t.shape, generator=torch.Generator().manual_seed(3)).to(cuda) for t in (q, k)]
    torch.autograd.backward(y, dy)
    c, s = angles(cos, sin, 7, None)
    for i, x in enumerate((q, k)):
        pw, pb = params[i], params[2 + i]
        check_forward(y[i].detach(), x, pw.detach(), pb.detach(), c, s, 1e-5, "layernorm", first)
        assert pw.grad.dtype == pw.dtype and pb.grad.dtype == pb.dtype
    alike = [t.detach().float().requires_grad_() for t in params]
    z = T.QKNormRoPEKernel.apply(q, k, alike[0], alike[1], cos, sin, alike[2], alike[3], 1e-5, "layernorm", first)
    torch.autograd.backward(z, dy)
    for u, v in zip(y, z):
        assert torch.equal(u, v)
    for t, u in zip(params, alike):
        assert torch.equal(t.grad, u.grad.to(t.dtype))
