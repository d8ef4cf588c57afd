"""Calls at the edges of what the products with groups, and per channel, allow."""
import importlib

import pytest
import torch

from tests.test_gpu_group_matmul import DT, matrix

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


@pytest.mark.parametrize('x', ['f16', 'f32'])
@pytest.mark.parametrize('M', [1, 12, 48, 300])
def test_captured_products_per_channel_have_their_own_workspaces(G, M, x):
    """Two graphs captured on one stream, the second replayed before the first ever was, then both at once beside eager calls."""
    mats = []
    for seed in (1, 2):
        qm, _, _ = matrix(G, 2048, 256, 128, seed=seed)
        mats.append(G.QuantizedMatrix(qm.int_weight, qm.zero[0].contiguous(), qm.scale[0].contiguous()))
    xs = [torch.randn((M, 2048), device='cuda').to(DT[x]) for _ in mats]
    dys = [torch.randn((M, 256), device='cuda').to(DT[x]) for _ in mats]
    want = [(G.quantized_matmul(a, m), G.quantized_matmul(b, m, transpose_b=True)) for a, b, m in zip(xs, dys, mats)]
    graphs, outs = [], []
    for a, b, m in zip(xs, dys, mats):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            G.quantized_matmul(a, m)
            outs.append((G.quantized_matmul(a, m), G.quantized_matmul(b, m, transpose_b=True)))
        graphs.append(g)
    graphs[1].replay()
    torch.cuda.synchronize()
    assert all(torch.equal(o, w) for o, w in zip(outs[1], want[1]))
    streams = [torch.cuda.Stream() for _ in graphs]
    torch.cuda.synchronize()
    for _ in range(20):
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
        eager = G.quantized_matmul(xs[0], mats[0])
    torch.cuda.synchronize()
    assert torch.equal(eager, want[0][0])
    for o, w in zip(outs, want):
        assert all(torch.equal(a, b) for a, b in zip(o, w))
