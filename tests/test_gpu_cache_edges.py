"""Calls at the edges of what the paged cache allows: rows that are not finite inside longer runs, scales below the normal range."""
import importlib

import numpy as np
import pytest
import torch

from tests.test_gpu_cache import DT, codes_of, write_reference

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
