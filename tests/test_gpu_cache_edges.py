"""Calls at the edges of what the paged cache allows: rows that are not finite inside longer runs, scales below the normal range
and below zero."""
import importlib

import numpy as np
import pytest
import torch
import torch.autograd.forward_ad as fwAD

from tests.test_gpu_cache import DT, codes_of, filled, i32, write_reference
from tests.test_gpu_prompt_attention import reference

pytestmark = pytest.mark.gpu


@pytest.fixture(scope='module')
def G():
    return importlib.import_module('jax_gptq_b200')


def check_write(G, k, v, slots, pages, page):
    """Codes and scales are whole numbers and fp32 quotients by definition: every bit is compared."""
    heads, dim = k.shape[1:]
    cache = G.KVCache(pages, heads, dim, page)
    cache.write(k, v, torch.tensor(slots, device='cuda'))
    for got, scale, x in zip(codes_of(cache), (cache.k_scale, cache.v_scale), (k, v)):
        codes, want = np.zeros_like(got), np.zeros((pages, heads), np.float32)
        write_reference(codes, want, x.float().cpu().numpy(), slots, page)
        assert np.array_equal(scale.cpu().numpy(), want)
        assert np.array_equal(got, codes)                                 # the padding behind the head dimension too


@pytest.mark.parametrize('x', ['f16', 'bf16', 'f32'])
@pytest.mark.parametrize('heads,dim', [(2, 64), (1, 80), (1, 33), (1, 256)])
@pytest.mark.parametrize('page', [64, 256])
def test_runs_with_values_that_are_not_finite(G, x, heads, dim, page):
    """Tokens and channels that are NaN throughout, infinities among other values, a page of nothing but NaN."""
    gen = torch.Generator(device='cuda').manual_seed(dim)
    slots = list(range(page)) + [page + i for i in range(5, 29)] + [2 * page + i for i in range(9)] + [3 * page + 7, 3 * page + 8]
    k, v = torch.randn((2, len(slots), heads, dim), generator=gen, device='cuda').unbind(0)
    nan, inf = float('nan'), float('inf')
    for t in (k, v):
        t[3] = nan                                                        # a token; four of them, and a whole block of sixteen
        t[8:12] = nan
        t[32:48] = nan
        t[20, :, :3] = torch.tensor([inf, -inf, nan], device='cuda')
        t[page + 2:page + 20, :, 4:20] = nan                              # channels
        t[page + 21, 0, 0] = -inf
        t[page + 24:page + 33] = nan                                      # a run without a number
        t[page + 33, 0] = inf                                             # infinities alone
        t[page + 34, 0] = nan
    check_write(G, k.to(DT[x]), v.to(DT[x]), slots, 4, page)


@pytest.mark.parametrize('x', ['bf16', 'f32'])
@pytest.mark.parametrize('heads,dim', [(2, 64), (1, 80), (1, 200)])
@pytest.mark.parametrize('top', [1e-36, 1e-37, 3e-38, 1e-39])
def test_runs_whose_scale_has_no_reciprocal(G, x, heads, dim, top):
    """Scales (a 127th of `top`) around and below 2^-126: zeros stay zeros, also behind the head dimension."""
    gen = torch.Generator(device='cuda').manual_seed(dim)
    slots = list(range(64)) + [64 + i for i in range(3, 24)]
    k, v = (torch.randn((2, len(slots), heads, dim), generator=gen, device='cuda').clamp(-1, 1) * top).unbind(0)
    for t in (k, v):
        t[5:14] = 0
        t[:, :, 16:32] = 0
    check_write(G, k.to(DT[x]), v.to(DT[x]), slots, 2, 64)


@pytest.mark.parametrize('x', ['f16', 'bf16', 'f32'])
@pytest.mark.parametrize('new', [1, 20, 100, 300])
@pytest.mark.parametrize('D', [64, 128])
@pytest.mark.parametrize('scale', [None, -0.2])
def test_negative_scales_of_keys(G, x, new, D, scale):
    """A page with a negative scale is one with a positive scale and negated codes, whatever the scores' range in its tiles is."""
    lengths = [700, 400]
    cache, table, gen = filled(G, lengths, 2, D, 64, D + new)
    cache.k.clamp_(min=1)                                                 # every code has a negative
    cache.k_scale[::2] *= 4                                               # scores some 50 powers of two apart
    same = G.KVCache(cache.num_pages, 2, D, 64)
    for name in ('k', 'v', 'k_scale', 'v_scale'):
        getattr(same, name).copy_(getattr(cache, name))
    cache.k_scale[::3] *= -1
    same.k[::3] = (256 - same.k[::3].int()).to(torch.uint8)
    q = (2 * torch.randn((2 * new, 4, D), generator=gen, device='cuda')).to(DT[x])
    out, lse = cache.attend(q, table, i32(lengths), i32([0, new, 2 * new]), new, scale=scale, return_lse=True)
    want, wl, tol, tl = reference(same, table, q, lengths, [new, new], D ** -0.5 if scale is None else scale)
    off = (out.double() - want).abs()
    assert bool((off <= tol).all()), f'{float((off / tol).max())} of the tolerance'
    assert bool(((lse.double() - wl).abs() <= tl).all())


@pytest.mark.parametrize('new', [3, 90])
def test_lse_behind_the_last_request_beside_a_given_result(G, new):
    lengths = [200, 100]
    cache, table, gen = filled(G, lengths, 2, 64, 64, 3)
    q = torch.randn((2 * new + 40, 4, 64), generator=gen, device='cuda').half()
    cu = i32([0, new, 2 * new])
    _, want = cache.attend(q, table, i32(lengths), cu, new, return_lse=True)
    out = torch.full_like(q, 7.0)
    used = torch.full(want.shape, 3.0, device='cuda')                  # what the allocator hands out next
    del used
    _, lse = cache.attend(q, table, i32(lengths), cu, new, out=out, return_lse=True)
    assert torch.equal(lse, want) and bool((lse[2 * new:] == -float('inf')).all()) and bool((out[2 * new:] == 7).all())


@pytest.mark.parametrize('new', [1, 90])
def test_rows_of_no_request(G, new):
    """A step without requests: all rows lie behind the last one."""
    cache, _, gen = filled(G, [10], 2, 64, 64, 3)
    q = torch.randn((5, 4, 64), generator=gen, device='cuda').half()
    none, table = i32([]), torch.zeros((0, 4), dtype=torch.int32, device='cuda')
    got, lse = cache.attend(q, table, none, i32([0]), new, return_lse=True)
    assert bool((got == 0).all()) and bool((lse == -float('inf')).all())
    out = torch.full_like(q, 7.0)
    assert bool((cache.attend(q, table, none, i32([0]), new, out=out) == 7).all())


@pytest.mark.parametrize('x', ['f16', 'f32'])
@pytest.mark.parametrize('new', [3, 90])
def test_rows_in_front_of_the_first_request(G, new, x):
    lengths = [200, 100]
    cache, table, gen = filled(G, lengths, 2, 64, 64, 3)
    q = torch.randn((2 * new + 7, 4, 64), generator=gen, device='cuda').to(DT[x])
    want, wl = cache.attend(q[5:], table, i32(lengths), i32([0, new, 2 * new]), new, return_lse=True)
    used = torch.full_like(q, 3.0)                                        # what the allocator hands out next
    del used
    got, lse = cache.attend(q, table, i32(lengths), i32([5, new + 5, 2 * new + 5]), new, return_lse=True)
    assert torch.equal(got[5:], want) and torch.equal(lse[5:], wl)
    assert bool((got[:5] == 0).all()) and bool((lse[:5] == -float('inf')).all())
    out = torch.full_like(q, 7.0)
    cache.attend(q, table, i32(lengths), i32([5, new + 5, 2 * new + 5]), new, out=out)
    assert torch.equal(out[5:-2], want[:-2]) and bool((out[:5] == 7).all()) and bool((out[-2:] == 7).all())


def test_forward_mode_tangents_are_refused(G):
    cache, table, gen = filled(G, [10], 2, 64, 64, 3)
    q = torch.randn((1, 4, 64), generator=gen, device='cuda')
    kv, slots = torch.randn((1, 2, 64), generator=gen, device='cuda'), torch.tensor([3], device='cuda')
    with fwAD.dual_level():
        dual = fwAD.make_dual(q, torch.ones_like(q))
        with pytest.raises(ValueError, match='tangent'):
            cache.attend(dual, table, i32([10]))
        with pytest.raises(ValueError, match='tangent'):
            cache.write(kv, fwAD.make_dual(kv, torch.ones_like(kv)), slots)
        cache.attend(q, table, i32([10]))                                 # nothing depends on these
        cache.write(kv, kv, slots)


def test_a_refused_step_has_taken_back_what_finished_requests_held(G):
    """Nothing is handed out, but the pages of those who left are free; the same call again, then one that fits."""
    table = G.PageTable(3, 4, 6, 64)
    table.reserve(i32([0, 0, 0]), i32([100, 60, 128]), 300)
    held = table.block_table.tolist()
    gone = torch.tensor([False, True, True], device='cuda')
    for _ in range(2):
        got = table.reserve(i32([100, 0, 0]), i32([1, 256, 256]), 600, finished=gone)         # eight pages of four
        assert got.slots.tolist() == [-1] * 600 and got.cu_seqlens.tolist() == [0] * 4 and got.lengths.tolist() == [100, 0, 0]
        assert table.held.tolist() == [2, 0, 0] and int(table.free_count) == 4
        assert table.block_table.tolist() == [held[0], [-1] * 4, [-1] * 4]
        with pytest.raises(RuntimeError, match='too few free pages'):
            table.check()
    got = table.reserve(i32([100, 0, 0]), i32([1, 64, 65]), 130)
    table.check()
    assert table.held.tolist() == [2, 1, 2] and got.lengths.tolist() == [101, 64, 65]
    pages = [p for row in table.block_table.tolist() for p in row if p >= 0]
    assert sorted(pages + table.free[:int(table.free_count)].tolist()) == list(range(6))
