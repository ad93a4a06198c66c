"""Weights and biases of qk_norm_rope in other shapes and types."""
import pytest
import torch

import trinix_b200 as T
from tests.test_gpu_qk_norm_rope import make, tables

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
