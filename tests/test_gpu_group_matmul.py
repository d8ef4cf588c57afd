"""Packed-int4 matmul with a scale and a zero point per group, its gradient, and the path that makes such matrices, against
plain computations in 64 bits."""
import importlib

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

DT = {'f16': torch.float16, 'bf16': torch.bfloat16, 'f32': torch.float32}


@pytest.fixture(scope='module')
def G():
    return importlib.import_module('jax_gptq_b200')


def matrix(G, K, N, group, zs='f32', seed=0, spread=1.0, fractional=False):
    """A grouped matrix and its dense form in 64 bits, with s (c + |z|), the size of what is summed up."""
    gen = torch.Generator(device='cuda').manual_seed(seed + 7 * K + N)
    groups = -(-K // group)
    packed = torch.randint(0, 256, (K // 2, N), generator=gen, dtype=torch.uint8, device='cuda')
    scale = (0.001 + 0.019 * torch.rand((groups, N), generator=gen, device='cuda'))
    if spread != 1.0:
        scale = scale * torch.exp(np.log(spread) * (torch.rand((groups, N), generator=gen, device='cuda') - 0.5))
    zero = torch.randint(0, 16, (groups, N), generator=gen, device='cuda').float()
    if fractional:
        zero = zero + torch.rand((groups, N), generator=gen, device='cuda')
    scale, zero = scale.to(DT[zs]), zero.to(DT[zs])
    codes = torch.stack((packed & 15, packed >> 4), 1).reshape(K, N).double()
    of = torch.arange(K, device='cuda') // group
    s, z = scale.double()[of], zero.double()[of]
    return G.QuantizedMatrix(packed, zero, scale, group_size=group), s * (codes - z), s * (codes + z.abs())


def allowed(exact, size, depth, dtype):
    """Per element: the result's rounding; in the products of 16-bit activations the weights' rounding to that type (half a
    step of each term); fp32 sums of `depth` terms, 16 at a time, truncated: depth / 8 steps of 2^-23 of what is summed."""
    u = torch.finfo(dtype).eps / 2
    return u * exact.abs() + ((u if dtype != torch.float32 else 0.0) + (depth / 8 + 64) * 2.0 ** -23) * 1.01 * size


def check(got, x, w, size, dtype):
    exact = x.double() @ w
    tol = allowed(exact, x.double().abs() @ size, w.shape[0], dtype)
    off = (got.double() - exact).abs()
    assert got.dtype == dtype and got.shape == exact.shape
    assert bool((off <= tol).all()), f'{float((off / tol).max())} of the tolerance'


SHAPES = [(1, 4096, 4096, 128), (1, 256, 16, 32), (2, 64, 8, 64), (3, 130, 909, 32), (4, 1024, 1536, 64), (5, 272, 48, 32), (8, 512, 272, 96), (8, 2048, 512, 128),
          (16, 1000, 640, 64), (17, 768, 2304, 128), (31, 320, 77, 32), (32, 4096, 1024, 128), (32, 96, 256, 4096), (33, 512, 512, 128), (64, 1024, 400, 64),
          (100, 2, 33, 32), (137, 272, 909, 32), (129, 640, 1040, 128), (256, 4096, 768, 128), (300, 1056, 2000, 96), (520, 384, 1024, 32), (1030, 512, 512, 128)]


@pytest.mark.parametrize('M,K,N,group', SHAPES)
@pytest.mark.parametrize('x', ['f16', 'bf16', 'f32'])
def test_product_and_gradient(G, M, K, N, group, x):
    dtype = DT[x]
    qm, w, size = matrix(G, K, N, group, zs='f16' if (M + K) % 3 == 0 else 'f32')
    gen = torch.Generator(device='cuda').manual_seed(M)
    xs = (torch.randn((M, K), generator=gen, device='cuda') + 0.25).to(dtype)
    check(G.quantized_matmul(xs, qm), xs, w, size, dtype)
    leaf = xs.clone().requires_grad_()
    y = G.quantized_matmul(leaf, qm)
    check(y.detach(), xs, w, size, dtype)
    dy = torch.randn((M, N), generator=gen, device='cuda').to(dtype)
    dx, = torch.autograd.grad(y, leaf, dy)
    check(dx, dy, w.T, size.T, dtype)


@pytest.mark.parametrize('M,K,N,group', [(33, 5002, 272, 96), (40, 11008, 256, 32), (64, 2998, 1008, 64), (96, 1030, 4096, 128), (130, 4096, 4112, 128),
                                         (257, 3000, 528, 32), (300, 2050, 2064, 160), (512, 8200, 256, 8224), (700, 1536, 1536, 64),
                                         (1000, 8200, 4112, 128), (1024, 4110, 8208, 32), (1001, 4104, 11008, 96), (390, 11008, 2064, 64), (17, 4096, 4112, 64), (32, 11008, 2064, 32)])
@pytest.mark.parametrize('x', ['f16', 'bf16'])
def test_tiles_shared_along_the_contraction(G, M, K, N, group, x):
    """Few tiles and a long contraction in either direction: odd numbers of stages per slice, groups that straddle the slices,
    rows that are no multiple of four, token columns that are not full; the same bits every time."""
    dtype = DT[x]
    qm, w, size = matrix(G, K, N, group, seed=1)
    gen = torch.Generator(device='cuda').manual_seed(K)
    xs, dy = (torch.randn((M, d), generator=gen, device='cuda').to(dtype) for d in (K, N))
    for a, flip in ((xs, False), (dy, True)):
        got = G.quantized_matmul(a, qm, transpose_b=flip)
        check(got, a, w.T if flip else w, size.T if flip else size, dtype)
        assert torch.equal(G.quantized_matmul(a, qm, transpose_b=flip), got)


@pytest.mark.parametrize('M', [1, 7, 40, 260])
@pytest.mark.parametrize('x', ['f16', 'bf16', 'f32'])
def test_scales_over_many_magnitudes_and_fractional_zero_points(G, M, x):
    """Scales of a channel between 1e-6 and 1 (weights below the normal range of f16), zero points that are no whole
    numbers, activations with a mean: a rounded zero point would show in every element."""
    qm, w, size = matrix(G, 512, 256, 64, spread=1e6, fractional=True, seed=3)
    xs = (1 + 0.1 * torch.randn((M, 512), device='cuda', generator=torch.Generator(device='cuda').manual_seed(M))).to(DT[x])
    check(G.quantized_matmul(xs, qm), xs, w, size, DT[x])
    dy = (1 + 0.1 * torch.randn((M, 256), device='cuda')).to(DT[x])
    got = G.quantized_matmul(dy, qm, transpose_b=True)
    # a weight far below the largest of its group may be lost below f16's range: 2^-24 of that largest
    exact = dy.double() @ w.T
    tol = allowed(exact, dy.double().abs() @ size.T, 256, DT[x]) + 2.0 ** -23 * dy.double().abs().sum(1, keepdim=True) * float(size.max())
    assert bool(((got.double() - exact).abs() <= tol).all())


@pytest.mark.parametrize('magnitude', [1e-30, 1e-12, 1e6, 1e20])
@pytest.mark.parametrize('M', [1, 40])
def test_scales_outside_the_range_of_f16(G, M, magnitude):
    qm, w, size = matrix(G, 256, 128, 32, seed=4)
    qm.scale = qm.scale * magnitude
    w, size = w / w.abs().max(), size / w.abs().max()
    of = torch.arange(256, device='cuda') // 32
    packed = qm.int_weight
    codes = torch.stack((packed & 15, packed >> 4), 1).reshape(256, 128).double()
    w = qm.scale.double()[of] * (codes - qm.zero.double()[of])
    size = qm.scale.double()[of] * (codes + qm.zero.double()[of])
    for dtype in (torch.bfloat16, torch.float32):
        xs = torch.randn((M, 256), device='cuda').to(dtype)
        check(G.quantized_matmul(xs, qm), xs, w, size, dtype)
        dy = torch.randn((M, 128), device='cuda').to(dtype)
        check(G.quantized_matmul(dy, qm, transpose_b=True), dy, w.T, size.T, dtype)
    if magnitude < 1:
        xs = (torch.randn((M, 256), device='cuda') / 16).half()
        big = G.QuantizedMatrix(packed, qm.zero, qm.scale / magnitude * 1e-12, group_size=32)
        y = G.quantized_matmul(xs, big)                        # far below f16's range: zero, not NaN
        assert bool((y == 0).all())


def test_same_groups_equal_the_product_per_channel(G):
    """One scale and zero per channel repeated for every group: the ungrouped product's values, to the types' rounding."""
    K, N, M = 512, 320, 24
    qm, w, size = matrix(G, K, N, K)
    xs = torch.randn((M, K), device='cuda').half()
    plain = G.quantized_matmul(xs, G.QuantizedMatrix(qm.int_weight, qm.zero[0], qm.scale[0]))
    rep = G.QuantizedMatrix(qm.int_weight, qm.zero.expand(4, N).contiguous(), qm.scale.expand(4, N).contiguous(), group_size=128)
    exact = xs.double() @ w
    tol = 2 * allowed(exact, xs.double().abs() @ size, K, torch.float16)
    for got in (G.quantized_matmul(xs, qm), G.quantized_matmul(xs, rep)):
        assert bool(((got.double() - plain.double()).abs() <= tol).all())


@pytest.mark.parametrize('M', [1, 24, 70, 300])
@pytest.mark.parametrize('x', ['f16', 'bf16', 'f32'])
def test_repeated_calls_give_the_same_bits_and_unaligned_pointers_work(G, M, x):
    dtype = DT[x]
    qm, w, size = matrix(G, 1024, 528, 128)
    xs = torch.randn((M, 1024), device='cuda').to(dtype)
    first = G.quantized_matmul(xs, qm)
    for _ in range(3):
        assert torch.equal(G.quantized_matmul(xs, qm), first)
    # the same values one element (one byte) off every alignment
    off = torch.empty(xs.numel() + 1, dtype=dtype, device='cuda')[1:].view_as(xs).copy_(xs)
    wo = torch.empty(qm.int_weight.numel() + 1, dtype=torch.uint8, device='cuda')[1:].view_as(qm.int_weight).copy_(qm.int_weight)
    so = torch.empty(qm.scale.numel() + 1, dtype=qm.scale.dtype, device='cuda')[1:].view_as(qm.scale).copy_(qm.scale)
    zo = torch.empty(qm.zero.numel() + 1, dtype=qm.zero.dtype, device='cuda')[1:].view_as(qm.zero).copy_(qm.zero)
    for a, b in ((off, qm), (xs, G.QuantizedMatrix(wo, qm.zero, qm.scale, group_size=128)), (xs, G.QuantizedMatrix(qm.int_weight, zo, so, group_size=128))):
        check(G.quantized_matmul(a, b), xs, w, size, dtype)
        dy = torch.randn((M, 528), device='cuda').to(dtype)
        check(G.quantized_matmul(dy, b, transpose_b=True), dy, w.T, size.T, dtype)


def test_shapes_strides_streams_and_empty_calls(G):
    qm, w, size = matrix(G, 256, 144, 64)
    x = torch.randn((2, 3, 512), device='cuda').half()[..., ::2]          # strided, three axes
    y = G.quantized_matmul(x, qm)
    assert y.shape == (2, 3, 144)
    check(y.reshape(6, 144), x.reshape(6, 256), w, size, torch.float16)
    assert G.quantized_matmul(x.new_empty((0, 256)), qm).shape == (0, 144)
    assert G.quantized_matmul(x.new_empty((0, 144)), qm, transpose_b=True).shape == (0, 256)
    s = torch.cuda.Stream()
    xs = torch.randn((5, 256), device='cuda').half()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        y = G.quantized_matmul(xs, qm)
    torch.cuda.current_stream().wait_stream(s)
    check(y, xs, w, size, torch.float16)
    got = G.quantized_matmul(xs.cpu().numpy(), qm)
    assert isinstance(got, np.ndarray) and np.array_equal(got, y.cpu().numpy())
    dy = torch.ones((1, 1), device='cuda').half().expand(5, 144)          # a gradient that is broadcast
    leaf = xs.clone().requires_grad_()
    G.quantized_matmul(leaf, qm).backward(dy)
    check(leaf.grad, dy, w.T, size.T, torch.float16)


@pytest.mark.parametrize('M', [1, 48])
def test_gradient_agrees_with_differences(G, M):
    qm, w, _ = matrix(G, 96, 40, 32)
    x = torch.randn((M, 96), device='cuda', requires_grad=True)
    v = torch.randn((M, 40), device='cuda')
    dx, = torch.autograd.grad((G.quantized_matmul(x, qm) * v).sum(), x)
    step = torch.randn_like(x)
    f = lambda a: (G.quantized_matmul(x.detach() + a * step, qm).double() * v.double()).sum()      # noqa: E731
    # linear: the difference of two fp32 results of size S has an error of about 2^-22 S; the step is of size one
    size = float((x.detach().abs().double() @ w.abs() * v.double().abs()).sum() + (step.abs().double() @ w.abs() * v.double().abs()).sum())
    assert abs(float(f(1.0) - f(-1.0)) / 2 - float((dx.double() * step.double()).sum())) <= 96 * 2.0 ** -22 * size


def test_gradient_of_the_gradient(G):
    """The product is linear: differentiating its gradient with respect to the incoming one is the product again."""
    qm, w, size = matrix(G, 128, 64, 32)
    x = torch.randn((3, 128), device='cuda', requires_grad=True)
    dy = torch.randn((3, 64), device='cuda', requires_grad=True)
    dx, = torch.autograd.grad(G.quantized_matmul(x, qm), x, dy, create_graph=True)
    v = torch.randn((3, 128), device='cuda')
    again, = torch.autograd.grad(dx, dy, v)
    check(again, v, w, size, torch.float32)


@pytest.mark.parametrize('M', [1, 12, 48])
def test_two_captured_graphs_do_not_share_a_workspace(G, M):
    """Graphs captured on one stream, replayed on two at once, beside eager calls."""
    qms = [matrix(G, 2048, 256, 128, seed=i) for i in (1, 2)]
    xs = [torch.randn((M, 2048), device='cuda').half() for _ in qms]
    want = [G.quantized_matmul(x, q[0]) for x, q in zip(xs, qms)]
    graphs, outs = [], []
    for x, q in zip(xs, qms):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            y = G.quantized_matmul(x, q[0])
            y = G.quantized_matmul(x, q[0]) + (y - y)
        graphs.append(g)
        outs.append(y)
    streams = [torch.cuda.Stream() for _ in graphs]
    torch.cuda.synchronize()
    for _ in range(20):
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
        eager = G.quantized_matmul(xs[0], qms[0][0])
    torch.cuda.synchronize()
    assert torch.equal(eager, want[0])
    for o, y in zip(outs, want):
        assert torch.equal(o, y)


def test_backward_captured_into_a_graph(G):
    qm, w, size = matrix(G, 512, 256, 128)
    x = torch.randn((40, 512), device='cuda').half().requires_grad_()
    dy = torch.randn((40, 256), device='cuda').half()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        torch.autograd.grad(G.quantized_matmul(x, qm), x, dy)
    torch.cuda.current_stream().wait_stream(s)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        dx, = torch.autograd.grad(G.quantized_matmul(x, qm), x, dy)
    g.replay()
    torch.cuda.synchronize()
    check(dx, dy, w.T, size.T, torch.float16)


def test_refusals(G):
    qm, _, _ = matrix(G, 256, 48, 64)
    x = torch.randn((2, 256), device='cuda')
    with pytest.raises(AssertionError, match='Inner dim mismatch'):
        G.quantized_matmul(x[:, :128], qm)
    with pytest.raises(ValueError, match='must have shape'):
        G.quantized_matmul(x, G.QuantizedMatrix(qm.int_weight, qm.zero, qm.scale, group_size=128))
    with pytest.raises(ValueError, match='must have shape'):
        G.quantized_matmul(x, G.QuantizedMatrix(qm.int_weight, qm.zero[0], qm.scale[0], group_size=64))
    with pytest.raises(ValueError):
        G.gptq.gptq(torch.randn((256, 8), device='cuda'), [torch.randn((512, 256), device='cuda')], actorder=True, group_size=64)


# ---- the path that makes such matrices ----
@pytest.mark.parametrize('K,N,group', [(256, 40, 64), (128, 33, 32), (272, 16, 32), (96, 8, 128)])
@pytest.mark.parametrize('bits', [4, 3])
def test_params_pack_and_unpack(G, K, N, group, bits):
    rng = np.random.default_rng(K + N)
    W = (0.02 * rng.standard_normal((K, N))).astype(np.float32)
    p = G.get_col_quantize_params(W, bits=bits, group_size=group)
    groups = -(-K // group)
    assert p['group_size'] == group and p['scale'].shape == p['zero'].shape == (groups, N)
    of = np.arange(K) // group
    for i in range(groups):
        ref = G.get_col_quantize_params(W[of == i], bits=bits)
        assert np.array_equal(p['scale'][i], ref['scale']) and np.array_equal(p['zero'][i], ref['zero'])
    codes = np.clip(np.round(W / p['scale'][of]) + p['zero'][of], 0, p['maxq'])
    Q = (p['scale'][of] * (codes - p['zero'][of])).astype(np.float32)
    if bits == 3 and K % 8:
        return
    qm = G.pack_matrix(Q, p, bits=bits)
    assert qm.group_size == group and qm.shape == (K, N)
    assert np.array_equal(np.asarray(G.unpack_along_axis(0, qm.int_weight)) if bits == 4 else codes, codes)
    assert np.array_equal(G.gptq.unpack_matrix(qm), Q)
    x = rng.standard_normal((5, K)).astype(np.float32)
    y = G.quantized_matmul(x, qm)
    size = np.abs(x) @ (p['scale'][of] * (codes + p['zero'][of]))
    assert np.all(np.abs(y - x.astype(np.float64) @ Q.astype(np.float64)) <= ((K / 8 + 64) * 2.0 ** -23 + 2.0 ** -23) * size + 2.0 ** -24 * np.abs(y))


def test_pack_refuses_params_of_another_shape(G):
    W = torch.randn((128, 8), device='cuda')
    p = G.get_col_quantize_params(W, group_size=32)
    with pytest.raises(ValueError, match='must have shape'):
        G.pack_matrix(W, {**p, 'group_size': 64})
    with pytest.raises(ValueError, match='axis 0'):
        G.pack_matrix(W, p, contraction_axis=1)


@pytest.mark.parametrize('K,N,group,block', [(256, 64, 128, 128), (256, 40, 32, 128), (384, 24, 192, 128), (256, 32, 256, 64), (256, 8, 512, 128)])
def test_gptq_with_groups(G, K, N, group, block):
    """The loop against the oracle's, block by block with the block's group: codes from the same factor may differ only where
    the lazy update's last bits decide a rounding (at most 0.1 %, the bar of the layer tests)."""
    import math
    from oracle import ref_gptq as R
    g = importlib.import_module('jax_gptq_b200.gptq')
    rng = np.random.default_rng(K + N + group)
    W = (0.02 * rng.standard_normal((K, N))).astype(np.float32)
    xs = [rng.standard_normal((4 * K, K)).astype(np.float32) for _ in range(2)]
    Q, params, qm, codes = g.gptq(W, xs, block_size=block, group_size=group, return_packed=True, return_codes=True)
    assert params['group_size'] == group and qm.group_size == group
    _, L, _ = R.damp_and_invert(W, R.accumulate_H(xs), 0.01)
    L, bs = L.astype(np.float32), math.gcd(block, group)
    Wr, want = W.copy(), []
    for s in range(0, K, bs):
        i = s // group
        ref = R.get_col_quantize_params(W[i * group:(i + 1) * group])
        assert np.array_equal(ref['scale'], params['scale'][i]) and np.array_equal(ref['zero'], params['zero'][i])
        q, err = R.process_block(Wr, L, s, ref, bs)
        Wr[s + bs:] -= (L[s + bs:, s:s + bs] @ err).astype(np.float32)
        want.append(np.round(q / ref['scale'] + ref['zero']).astype(np.uint8))
    want = np.concatenate(want)
    # the factor is this library's own here, the oracle's above: the layer tests' bar for that is 99.9 % as well
    assert (codes != want).mean() <= 2e-3
    of = np.arange(K) // group
    assert np.array_equal(Q, (params['scale'][of] * (codes.astype(np.float32) - params['zero'][of])).astype(np.float32))
    assert np.array_equal(G.gptq.unpack_matrix(qm), Q)


def test_gptq_many_with_groups(G):
    g = importlib.import_module('jax_gptq_b200.gptq')
    gen = torch.Generator(device='cuda').manual_seed(9)
    jobs = [(0.02 * torch.randn((256, n), generator=gen, device='cuda'), [torch.randn((1024, 256), generator=gen, device='cuda')]) for n in (48, 96)]
    many = g.gptq_many(jobs, group_size=64, streams=2)
    again = g.gptq_many(jobs, group_size=64, streams=2)
    third = g.gptq_many(jobs, group_size=128, streams=2)                 # other groups do not replay the sequence of these
    for (W, xs), a, b, c in zip(jobs, many, again, third):
        _, _, one = g.gptq(W, xs, group_size=64, return_packed=True)
        _, _, wide = g.gptq(W, xs, group_size=128, return_packed=True)
        for got, ref in ((a, one), (b, one), (c, wide)):
            assert torch.equal(got.int_weight, ref.int_weight) and torch.equal(got.scale, ref.scale) and got.group_size == ref.group_size


@pytest.mark.parametrize('M,K,N,group', [(1, 4096, 4096, 128), (5, 272, 909, 32), (17, 4096, 512, 32), (24, 2048, 1024, 64), (32, 8192, 272, 128), (40, 11008, 256, 32),
                                         (130, 4096, 528, 128), (300, 512, 2064, 96), (700, 384, 1040, 32)])
@pytest.mark.parametrize('x', ['f16', 'bf16', 'f32'])
def test_a_workspace_of_the_stated_size_is_enough(G, M, K, N, group, x):
    """Both directions, also with a pointer that keeps the call from the kernels that want alignment; nothing behind it changes."""
    lib, code = G._lib.lib, {'f16': G._lib.F16, 'bf16': G._lib.BF16, 'f32': G._lib.F32}[x]
    qm, w, size = matrix(G, K, N, group)
    stream = torch.cuda.current_stream().cuda_stream
    for flags, depth, rows in ((0, K, N), (1, N, K)):
        xs = torch.randn((M, depth), device='cuda').to(DT[x])
        off = torch.empty(xs.numel() + 1, dtype=xs.dtype, device='cuda')[1:].view_as(xs).copy_(xs)
        need = lib.jgq_w4_group_matmul_workspace_bytes(M, N, K, group, flags)
        for a in (xs, off):
            ws = torch.zeros(need + 4096, dtype=torch.uint8, device='cuda')
            ws[need:] = 171
            out = torch.empty((M, rows), dtype=xs.dtype, device='cuda')
            rc = lib.jgq_w4_group_matmul(a.data_ptr(), code, qm.int_weight.data_ptr(), qm.zero.data_ptr(), qm.scale.data_ptr(), G._lib.F32, out.data_ptr(),
                                         M, N, K, group, flags, ws.data_ptr(), need, stream)
            assert rc == 0, lib.jgq_last_error()
            check(out, xs, w.T if flags else w, size.T if flags else size, DT[x])
            assert bool((ws[need:] == 171).all()) and not bool(ws[:16384].any())


@pytest.mark.parametrize('M', [1, 40])
def test_in_inference_mode(G, M):
    with torch.inference_mode():
        qm, w, size = matrix(G, 256, 64, 64)
        xs = torch.randn((M, 256), device='cuda').half()
        for _ in range(2):
            check(G.quantized_matmul(xs, qm), xs, w, size, torch.float16)


def test_scales_changed_just_before_a_call(G):
    """Decode products with scales and zero points that a kernel on the same stream has just written."""
    qm, w, size = matrix(G, 4096, 2048, 64)
    xs = torch.randn((1, 4096), device='cuda').half() / 8
    base, ones = G.quantized_matmul(xs, qm), torch.ones_like(qm.scale)
    scale = qm.scale.clone()
    for i in range(30):
        for _ in range(i % 3):
            G.quantized_matmul(xs, qm)
        f = 2.0 ** ((i % 7) - 3)
        torch.mul(scale, ones * f, out=qm.scale)
        assert torch.equal(G.quantized_matmul(xs, qm), (base.float() * f).half()) or f < 1      # subnormals round
        if f < 1:
            assert float((G.quantized_matmul(xs, qm).float() - base.float() * f).abs().max()) <= float(base.abs().max()) * f * 2.0 ** -10
