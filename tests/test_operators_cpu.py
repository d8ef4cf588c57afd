"""Refusals of the grouped matmul and of the paged cache, without a GPU: the C ABI's argument checks and the Python ones."""
import pytest

from tests.test_abi import jlib  # noqa: F401  (fixture: the built library)


def test_grouped_entry_points_refuse(jlib):  # noqa: F811
    lib, F16, F32 = jlib.lib, jlib.F16, jlib.F32
    ws = 1 << 30
    good = dict(x=256, xd=F16, w=256, z=256, s=256, zd=F32, out=256, M=4, N=64, K=128, g=32, flags=0, ws=256, n=ws)

    def call(**kw):
        a = {**good, **kw}
        return lib.jgq_w4_group_matmul(a['x'], a['xd'], a['w'], a['z'], a['s'], a['zd'], a['out'], a['M'], a['N'], a['K'], a['g'],
                                       a['flags'], a['ws'], a['n'], None)
    for bad in (dict(g=0), dict(g=-32), dict(g=48), dict(g=16), dict(K=127), dict(K=0), dict(N=0), dict(M=-1), dict(xd=jlib.U8),
                dict(zd=jlib.BF16), dict(flags=4), dict(x=None), dict(out=None), dict(s=None), dict(z=None), dict(w=None)):
        assert call(**bad) == -1, bad
    assert call(M=0) == 0
    assert call(n=16) == -3 and call(ws=None) == -3
    assert call(ws=8) == -2 and call(x=257) == -2 and call(s=258) == -2
    assert call(M=1 << 30) == -5
    assert lib.jgq_w4_group_matmul_workspace_bytes(0, 64, 128, 32, 0) == 0
    assert lib.jgq_group_params(256, 64, 8, 48, 15, 256, 256, None) == -1
    assert lib.jgq_group_params(256, 0, 8, 32, 15, 256, 256, None) == -1
    # a block of the loop must lie in one group
    assert lib.jgq_gptq_quantize_groups(256, 256, 256, 256, 256, 8, 32, 128, 15, 256, F32, None, 256, ws, None) == -1
    assert lib.jgq_gptq_quantize_groups(256, 256, 256, 256, 100, 8, 32, 32, 15, 256, F32, None, 256, ws, None) == -1


def test_scales_that_changed_are_not_fetched_early(jlib):  # noqa: F811
    """The decode kernel may read weights, scales and zero points ahead of the stream's previous kernel only if none of them
    changed since the matmul before."""
    import torch
    from jax_gptq_b200.op import _settled_groups
    w, zero, scale = torch.zeros((64, 16), dtype=torch.uint8), torch.zeros((4, 16)), torch.ones((4, 16))
    assert not _settled_groups(w, zero, scale) and _settled_groups(w, zero, scale)
    for changed in (w, zero, scale):
        changed.add_(1)
        assert not _settled_groups(w, zero, scale) and _settled_groups(w, zero, scale)
    scale[0].mul_(2)                                                     # through a view
    assert not _settled_groups(w, zero, scale) and _settled_groups(w, zero, scale)
    assert not _settled_groups(w, zero, scale.clone()) and not _settled_groups(w, zero.clone(), scale)
    with torch.inference_mode():                                         # no version counter: never early
        made = torch.ones((4, 16))
    assert not _settled_groups(w, zero, made) and not _settled_groups(w, zero, made)


def test_cache_entry_points_refuse(jlib):  # noqa: F811
    lib, F16 = jlib.lib, jlib.F16

    def attend(q=256, dt=F16, pages=8, page=64, width=4, cu=None, tokens=2, requests=2, most=1, hq=8, hkv=2, D=64, flags=0, ws=256, n=1 << 30, table=256):
        return lib.jgq_kv_attend(q, dt, hq * D, D, 256, None, 256, 256, 256, 256, pages, page, table, width, width, 256, cu, tokens, requests, most,
                                 hq, hkv, D, 1.0, flags, ws, n, None)
    for bad in (dict(dt=jlib.U8), dict(page=32), dict(page=96), dict(D=0), dict(D=257), dict(hq=7), dict(hkv=0), dict(tokens=3), dict(most=0),
                dict(pages=0), dict(width=-1), dict(flags=2), dict(q=None), dict(table=None)):
        assert attend(**bad) == -1, bad
    assert attend(tokens=0, requests=0) == 0
    assert attend(n=64) == -3 and attend(ws=None) == -3
    assert attend(ws=128) == -2 and attend(q=257) == -2
    assert attend(width=1 << 26, page=256) == -5
    assert attend(tokens=1 << 22, cu=256, hq=1024, hkv=1) == -5            # rows per kv head are counted in 32 bits

    def write(k=256, dt=F16, slots=256, tokens=4, pages=8, page=64, H=2, D=64, codes=256):
        return lib.jgq_kv_write(k, 256, dt, H * D, D, H * D, D, slots, tokens, codes, 256, 256, 256, pages, page, H, D, None)
    for bad in (dict(dt=jlib.U8), dict(page=16), dict(D=300), dict(H=0), dict(tokens=-1), dict(k=None), dict(slots=None), dict(pages=0)):
        assert write(**bad) == -1, bad
    assert write(tokens=0) == 0
    assert write(codes=264) == -2 and write(k=257) == -2
    assert lib.jgq_kv_read(256, 256, 256, 256, 8, 64, 2, 64, None, 1, 256, 256, F16, None) == -1
    assert lib.jgq_kv_read(256, 256, 256, 256, 8, 64, 2, 64, None, 0, None, None, F16, None) == 0
    assert lib.jgq_kv_read(256, 256, 256, 256, 8, 64, 2, 64, 256, 1, 256, 256, jlib.I32, None) == -1

    def reserve(table=256, width=4, pages=8, page=64, lengths=256, B=2, tokens=8, slots=256, out=512, status=256):
        return lib.jgq_kv_reserve(table, width, width, 256, 256, 256, pages, page, lengths, 256, None, B, slots, 256, tokens, 256, out, status, None)
    for bad in (dict(table=None), dict(width=-1), dict(pages=0), dict(page=0), dict(lengths=None), dict(B=-1), dict(tokens=-1), dict(slots=None),
                dict(out=None), dict(status=None), dict(out=256)):
        assert reserve(**bad) == -1, bad
    assert reserve(tokens=1 << 25) == -5 and reserve(B=1 << 21) == -5


def test_python_refusals_without_a_gpu(jlib):  # noqa: F811
    import torch
    import jax_gptq_b200 as G
    w = torch.zeros((64, 16), dtype=torch.uint8)
    for g in (0, -32, 16, 48, 33):
        with pytest.raises(ValueError, match='multiple of 32'):
            G.QuantizedMatrix(w, None, None, group_size=g)
    qm = G.QuantizedMatrix(w, torch.zeros(4, 16), torch.zeros(4, 16), group_size=32)
    assert qm.shape == (128, 16)
    children, aux = qm.tree_flatten()
    again = G.QuantizedMatrix.tree_unflatten(aux, children)
    assert again.group_size == 32 and again.contraction_axis == 0
    plain = G.QuantizedMatrix(w, None, None)
    assert plain.group_size is None and plain.tree_flatten()[1] == 0
    for kw in (dict(page_size=32), dict(page_size=100), dict(head_dim=0), dict(head_dim=257), dict(num_pages=0), dict(kv_heads=0)):
        with pytest.raises(ValueError):
            G.KVCache(**{**dict(num_pages=4, kv_heads=2, head_dim=64, page_size=64, device='cuda:0'), **kw})
    with pytest.raises(ValueError):
        G.PageTable(0, 4, 8, 64, device='cuda:0')
    with pytest.raises(ValueError, match='CUDA device'):
        G.PageTable(1, 4, 8, 64, device='cpu')


def test_group_parts_cover_every_row():
    from jax_gptq_b200.gptq import _group_parts
    for K, g in ((128, 32), (272, 32), (32, 64), (96, 96), (4096, 128), (100, 32)):
        rows = []
        for r0, i, n, per in _group_parts(K, g):
            for j in range(n):
                rows += [(r0 + j * per + x, i + j) for x in range(per)]
        assert rows == [(k, k // g) for k in range(K)]


def test_grouped_workspaces(jlib):  # noqa: F811
    """Workspaces without room for the tickets, none at all and misaligned ones are refused, whichever kernel the call is for."""
    lib = jlib.lib
    for M in (1, 5, 16, 17, 31, 32, 33, 200):
        for K, N in ((4096, 4096), (272, 909), (11008, 256), (256, 8192)):
            for g in (32, 128):
                for flags in (0, 1):
                    need = lib.jgq_w4_group_matmul_workspace_bytes(M, N, K, g, flags)
                    assert need >= 16384
                    for xd in (jlib.F32, jlib.F16, jlib.BF16):
                        call = lambda ws, n: lib.jgq_w4_group_matmul(256, xd, 256, 256, 256, jlib.F32, 256, M, N, K, g, flags, ws, n, None)
                        assert call(256, 16383) == -3 and call(None, need) == -3
                        assert call(8, need) == -2


def test_rows_with_a_tangent_are_refused(jlib):  # noqa: F811
    """Keys, values and queries of the cache have no derivative; a forward-mode one would be lost."""
    import types

    import torch
    import torch.autograd.forward_ad as fwAD
    from jax_gptq_b200.cache import KVCache
    cache = KVCache.__new__(KVCache)
    cache.device, cache.head_dim = types.SimpleNamespace(index=-1), 8    # -1: what CPU tensors answer
    t = torch.zeros((3, 2, 8))
    assert cache._rows(t, 'q', None)[1] == (3, 2, 8)
    with fwAD.dual_level():
        assert cache._rows(t, 'q', 2)[0] is t
        with pytest.raises(ValueError, match='tangent'):
            cache._rows(fwAD.make_dual(t, torch.ones_like(t)), 'q', None)
        with torch.no_grad(), pytest.raises(ValueError, match='tangent'):
            cache._rows(fwAD.make_dual(t, torch.ones_like(t)).transpose(0, 1), 'q', None)
    with pytest.raises(ValueError, match='gradient'):
        cache._rows(t.clone().requires_grad_(), 'q', None)


def test_trainable_scales_of_groups_are_refused(jlib):  # noqa: F811
    import torch
    from jax_gptq_b200.op import _group_matmul
    w, x = torch.zeros((32, 16), dtype=torch.uint8), torch.zeros((3, 64))
    for trained in range(2):
        parts = [torch.zeros((2, 16)), torch.ones((2, 16))]
        parts[trained].requires_grad_()
        for flip in (False, True):
            with pytest.raises(ValueError, match='no gradient'):
                _group_matmul(x[:, :16] if flip else x, w, *parts, 32, flip)
