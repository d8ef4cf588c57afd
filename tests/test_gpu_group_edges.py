"""Calls at the edges of what the product with groups allows."""
import importlib

import pytest
import torch

from tests.test_gpu_group_matmul import matrix

pytestmark = pytest.mark.gpu


@pytest.fixture(scope='module')
def G():
    return importlib.import_module('jax_gptq_b200')


@pytest.mark.parametrize('M', [1, 40])
def test_trainable_scales_and_zero_points_are_refused(G, M):
    qm, w, size = matrix(G, 128, 64, 32)
    x = torch.randn((M, 128), device='cuda')
    for which in ('scale', 'zero'):
        for leaf in (x, x.clone().requires_grad_()):
            for transpose_b in (False, True):
                parts = dict(zero=qm.zero, scale=qm.scale)
                parts[which] = parts[which].clone().requires_grad_()
                trained = G.QuantizedMatrix(qm.int_weight, parts['zero'], parts['scale'], group_size=32)
                a = leaf if not transpose_b else leaf[:, :64].contiguous()
                with pytest.raises(ValueError, match='gradient'):
                    G.quantized_matmul(a, trained, transpose_b)
                with torch.no_grad():
                    assert torch.equal(G.quantized_matmul(a, trained, transpose_b), G.quantized_matmul(a, qm, transpose_b))
