"""Attention of prompts and chunks over the paged 8-bit cache: many rows per sequence, scores that keep rising, scales of the
pages that lie orders of magnitude apart, zero and negative ones, items that many blocks share; against 64 bits."""
import importlib
import math

import numpy as np
import pytest
import torch

from tests.test_gpu_cache import DT, filled, i32, rows_of

pytestmark = pytest.mark.gpu


@pytest.fixture(scope='module')
def G():
    return importlib.import_module('jax_gptq_b200')


def reference(cache, table, q, lengths, new, scale):
    """(output, lse, tolerance of the output, of lse) in 64 bits.

    Rounded are: a score, an fp32 sum in ceil(D / 16) steps (plus a few for the factor and the exponent's argument) of terms of
    sum |q| |k| (and 128 scale |q| where codes keep their excess), `d` below, with the argument of 2^x at 2^-23 of the largest
    numbers in it; 2^x itself (2^-22); p v_scale as f16: half a step of 2^-11, or 2^-25 below 2^-14 of the row's largest (fp32
    calls: 2^-21); sums of the values, four steps of 2^-22 per 64 tokens, plus, where codes keep their excess, 2^-22 of the sum of p times
    256 scales (the numbers that are subtracted from one another reach that, tile by tile);
    the result once (f16: by half a step of 2^-24 below 2^-14, where its steps stop shrinking: an output of 3e-8 may come back
    as zero).  What lies below 2^-60 of the row's largest p v_scale may count as that."""
    Hq, D, H = q.shape[1], q.shape[2], cache.kv_heads
    g, P = Hq // H, cache.page_size
    f32 = q.dtype == torch.float32
    u = torch.finfo(q.dtype).eps / 2
    outs, lses, tols, tls = [], [], [], []
    at = 0
    for r, (L, n) in enumerate(zip(lengths, new)):
        k, v = rows_of(cache, table, r, L)
        pages = table[r, :-(-L // P)].long()
        ks = cache.k_scale[pages].double().T.repeat_interleave(P, 1)[:, :L]          # [H, L]
        vs = cache.v_scale[pages].double().T.repeat_interleave(P, 1)[:, :L].abs()
        see = (L - n + 1 + torch.arange(n, device='cuda')).clamp(0, L)
        mask = torch.arange(L, device='cuda')[None] < see[:, None]                   # [n, L]
        for h in range(Hq):
            qr, kh, vh = q[at:at + n, h].double(), k[h // g], v[h // g]
            s = (qr @ kh.T) * scale
            s = s.masked_fill(~mask, -math.inf)
            m = s.max(1, keepdim=True).values if L else torch.full((n, 1), -math.inf, device='cuda', dtype=torch.float64)
            m0 = m.masked_fill(m.isinf(), 0.0)
            e = torch.exp(s - m0)
            tot = e.sum(1, keepdim=True)
            p = e / tot.clamp(min=1e-300)
            o = p @ vh
            big = (qr.abs() @ kh.abs().T + 128 * qr.abs().sum(1, keepdim=True) * ks[h // g][None]) * abs(scale)
            big = big.masked_fill(~mask, 0.0)
            lv = torch.log(vs[h // g].clamp(min=1e-30)).abs().max() if L else 0.0
            d = (D / 16 + 6) * 2.0 ** -22 * big.amax(1, keepdim=True) + 2.0 ** -21 * (m0.abs() + lv + 60) if L else torch.zeros_like(m0)
            rp = (2.0 ** -21 if f32 else 2.0 ** -11) + 2.0 ** -20
            weight = (p * vs[h // g][None]).amax(1, keepdim=True) if L else torch.zeros_like(m0)
            spread = (p * vs[h // g][None]).sum(1, keepdim=True) if L else torch.zeros_like(m0)
            tiles = see[:, None] / 64 + 2
            tol = ((2 * (d + rp) + tiles * 2.0 ** -20) * (p @ vh.abs()) + see[:, None] * 2.0 ** (-35 if f32 else -25) * 2 * 128 * weight
                   + 2.0 ** -22 * 256 * spread + u * o.abs() + (2.0 ** -25 if q.dtype == torch.float16 else 0.0))
            outs.append(o), lses.append((m + torch.log(tot))[:, 0]), tols.append(tol)
            tls.append((d + rp + tiles * 2.0 ** -22 + see[:, None] * 2.0 ** -25)[:, 0] + 2.0 ** -22 * m0[:, 0].abs())
        at += n
    def whole(parts):
        rows, i = [], 0
        for n in new:
            rows.append(torch.stack(parts[i:i + Hq], 1))
            i += Hq
        return torch.cat(rows)
    return whole(outs), whole(lses), whole(tols), whole(tls)


def check(cache, table, q, lengths, new, scale=None):
    cu = i32(np.concatenate([[0], np.cumsum(new)]).tolist())
    kw = dict(scale=scale, cu_seqlens=cu, max_new=max(new))
    out, lse = cache.attend(q, table, i32(lengths), return_lse=True, **kw)
    want, wl, tol, tl = reference(cache, table, q, lengths, new, q.shape[2] ** -0.5 if scale is None else scale)
    assert out.dtype == q.dtype and bool(out.isfinite().all())
    off = (out.double() - want).abs()
    close = bool((off <= tol).all())
    assert close, f'{float((off / tol.clamp(min=1e-300)).max())} of the tolerance'
    fin = torch.isfinite(wl)
    assert torch.equal(torch.isfinite(lse), fin)
    assert bool(((lse.double() - wl).abs()[fin] <= tl[fin]).all())
    assert torch.equal(cache.attend(q, table, i32(lengths), **kw), out)              # the same bits again, without lse
    return out


@pytest.mark.parametrize('x', ['f16', 'bf16'])
@pytest.mark.parametrize('lengths,new', [([65], [65]), ([127], [100]), ([500, 3], [128, 3]), ([256, 255, 31], [256, 255, 40]), ([3000], [70]),
                                         ([9000, 700], [300, 129]), ([1, 64, 1024], [1, 64, 513])])
@pytest.mark.parametrize('Hq,H,D,page', [(2, 2, 64, 64), (6, 2, 128, 256), (8, 1, 96, 128), (1, 1, 33, 64)])
def test_rows_of_many_tokens(G, x, lengths, new, Hq, H, D, page):
    cache, table, gen = filled(G, lengths, H, D, page, sum(lengths))
    q = torch.randn((sum(new), Hq, D), generator=gen, device='cuda').to(DT[x])
    out = check(cache, table, q, lengths, new)
    at = 0
    for L, n in zip(lengths, new):
        assert bool((out[at:at + max(0, n - L)] == 0).all())
        at += n


@pytest.mark.parametrize('x', ['f16', 'bf16', 'f32'])
@pytest.mark.parametrize('new', [1, 20, 100, 300])
@pytest.mark.parametrize('D', [64, 128])
def test_scores_that_rise_from_page_to_page(G, x, new, D):
    """Every page outweighs the ones before it by far, so that a row's reference moves all the time; then the other way round."""
    lengths = [640]
    for order in (1, -1):
        cache, table, gen = filled(G, lengths, 1, D, 64, D + new)
        n = torch.arange(10, device='cuda', dtype=torch.float32)
        cache.k_scale[table[0, :10].long(), 0] = 0.004 * (1 + n if order == 1 else 10 - n)
        cache.k[table[0, :10].long(), :, :, :D] = cache.k[table[0, :10].long(), :, :, :D] // 2 + 128
        q = (torch.randn((new, 2, D), generator=gen, device='cuda').abs() * 2).to(DT[x])
        check(cache, table, q, lengths, [new])


@pytest.mark.parametrize('x', ['f16', 'bf16', 'f32'])
@pytest.mark.parametrize('new', [1, 20, 100, 300])
@pytest.mark.parametrize('large', ['first', 'last', 'mixed'])
@pytest.mark.parametrize('unit', [1.0, 2.0 ** 14])
def test_faint_pages_of_large_values(G, x, new, large, unit):
    """Pages whose values are a million times larger and whose weights are next to nothing: the others keep their precision."""
    lengths, D = [64 * 8 + 300], 64
    cache, table, gen = filled(G, lengths, 1, D, 64, new)
    pages = table[0, :13].long()
    where = {'first': [0, 1], 'last': [6, 7], 'mixed': [1, 4, 5]}[large]
    cache.v_scale[pages] *= 2.0 ** -20 * unit
    cache.k[pages, :, :, :D] = 128 + cache.k[pages, :, :, :D] % 16
    for i in where:
        cache.v_scale[pages[i]] *= 2.0 ** 20
        cache.k[pages[i], :, :, :D] = 0                                   # -128 in every channel
    cache.k_scale[pages] = 0.06
    q = torch.randn((new, 2, D), generator=gen, device='cuda').abs().to(DT[x])
    check(cache, table, q, lengths, [new])


@pytest.mark.parametrize('x', ['f16', 'bf16', 'f32'])
@pytest.mark.parametrize('new', [1, 20, 100, 300])
def test_zero_negative_and_scattered_scales(G, x, new):
    lengths, D = [700, 400], 128
    cache, table, gen = filled(G, lengths, 2, D, 64, 5)
    pages = table[0, :11].long()
    cache.v_scale[pages[:3]] = 0.0                                        # before any other
    cache.v_scale[pages[5]] = 0.0
    cache.k_scale[pages[4]] = 0.0
    cache.v_scale[pages[6]] *= -1.0
    cache.v_scale[pages[7:]] *= torch.tensor([2.0 ** -30, 1.0, 2.0 ** 12, 2.0 ** -9], device='cuda')[:, None]
    cache.v_scale[table[1, :7].long(), 0] = 0.0                           # a head whose values are all zero
    q = torch.randn((2 * new, 4, D), generator=gen, device='cuda').to(DT[x])
    out = check(cache, table, q, lengths, [new, new])
    assert bool((out[new:, :2] == 0).all())
    for scale in (-0.2, 0.0):
        check(cache, table, q, lengths, [new, new], scale)


@pytest.mark.parametrize('x', ['f16', 'bf16'])
@pytest.mark.parametrize('what', ['k', 'v'])
@pytest.mark.parametrize('value', [math.nan, math.inf])
@pytest.mark.parametrize('new', [80, 300])
def test_scales_that_are_not_finite(G, x, what, value, new):
    """Rows that see the page become NaN, wherever it lies, and no others do."""
    lengths = [400, 500]
    for page in (0, 3, 6):
        cache, table, gen = filled(G, lengths, 1, 64, 64, page)
        q = torch.randn((2 * new, 2, 64), generator=gen, device='cuda').to(DT[x])
        cu = i32([0, new, 2 * new])
        good = cache.attend(q, table, i32(lengths), cu_seqlens=cu, max_new=new)
        (cache.k_scale if what == 'k' else cache.v_scale)[table[0, page].long()] = value
        got = cache.attend(q, table, i32(lengths), cu_seqlens=cu, max_new=new)
        first = min(new, max(0, 64 * page - (lengths[0] - new)))              # row i sees lengths - new + i + 1 tokens
        assert torch.equal(got[:first], good[:first]) and torch.equal(got[new:], good[new:])
        assert not bool(got[first:new].isfinite().any())


@pytest.mark.parametrize('x', ['f16', 'bf16'])
@pytest.mark.parametrize('new', [70, 300])
def test_rows_behind_and_strided_rows_and_a_wrong_guess(G, x, new):
    lengths, news = [new + 900, 90], [new, 66]
    cache, table, gen = filled(G, lengths, 2, 128, 128, 9)
    T = new + 66
    q = torch.randn((T + 50, 4, 128), generator=gen, device='cuda').to(DT[x])
    q[T:] = float('nan')
    cu = i32([0, new, T])
    check(cache, table, q[:T], lengths, news)
    out = torch.full_like(q, 7.0)
    for guess in (new, 1, 5, None):
        out.fill_(7.0)
        cache.attend(q, table, i32(lengths), cu_seqlens=cu, max_new=guess, out=out)
        want, _, tol, _ = reference(cache, table, q[:T], lengths, news, 128 ** -0.5)
        assert bool(((out[:T].double() - want).abs() <= tol).all()) and bool((out[T:] == 7).all())
    fresh = cache.attend(q, table, i32(lengths), cu_seqlens=cu, max_new=new)
    assert bool((fresh[T:] == 0).all())
    wide = torch.zeros((T + 50, 9, 136), dtype=q.dtype, device='cuda')
    wide[:, 3:7, 1:129] = q
    again = cache.attend(wide[:, 3:7, 1:129], table, i32(lengths), cu_seqlens=cu, max_new=new)
    assert torch.equal(again, fresh)


@pytest.mark.parametrize('new', [100, 320])
def test_a_captured_chunk_replayed_with_other_lengths(G, new):
    """Two graphs of a padded chunk, replayed at once on two streams with lengths that change between replays."""
    cache, table, gen = filled(G, [2000, 2000], 2, 64, 64, 10)
    lengths, cu = i32([2000, 700]), i32([0, new, new + 50])
    qs = [torch.randn((new + 128, 4, 64), generator=gen, device='cuda').half() for _ in range(2)]
    for q in qs:
        cache.attend(q, table, lengths, cu_seqlens=cu, max_new=new)
    graphs, outs = [], []
    for q in qs:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(cache.attend(q, table, lengths, cu_seqlens=cu, max_new=new))
        graphs.append(g)
    streams = [torch.cuda.Stream() for _ in graphs]
    for L, rows in (([2000, 700], [0, new, new + 50]), ([40, 2000], [0, 17, 17 + new]), ([0, 1], [0, 0, 1]), ([300, 2000], [0, 1, 128])):
        lengths.copy_(i32(L))
        cu.copy_(i32(rows))
        torch.cuda.synchronize()
        for _ in range(5):
            for g, s in zip(graphs, streams):
                with torch.cuda.stream(s):
                    g.replay()
        torch.cuda.synchronize()
        for q, o in zip(qs, outs):
            assert torch.equal(o, cache.attend(q, table, lengths, cu_seqlens=cu, max_new=new))
            assert bool((o[rows[-1]:] == 0).all())


@pytest.mark.parametrize('x', ['f16', 'bf16', 'f32'])
@pytest.mark.parametrize('new', [1, 30, 100, 300])
@pytest.mark.parametrize('Hq,H,D', [(4, 4, 64), (8, 1, 128), (2, 2, 256)])
def test_a_workspace_of_the_stated_size_is_enough(G, x, new, Hq, H, D):
    """Sequences that many blocks share; nothing behind the workspace changes, its tickets are left zero."""
    lib, code = G._lib.lib, {'f16': G._lib.F16, 'bf16': G._lib.BF16, 'f32': G._lib.F32}[x]
    lengths = [5000, new, 3000]
    cache, table, gen = filled(G, lengths, H, D, 64, new)
    q = torch.randn((3 * new, Hq, D), generator=gen, device='cuda').to(DT[x])
    n, cu = i32(lengths), i32([0, new, 2 * new, 3 * new])
    need = lib.jgq_kv_attend_workspace_bytes(Hq, H, D, new, code)
    ws = torch.zeros(need + 4096, dtype=torch.uint8, device='cuda')
    ws[need:] = 171
    out = torch.empty_like(q)
    rc = lib.jgq_kv_attend(q.data_ptr(), code, q.stride(0), q.stride(1), out.data_ptr(), 0, cache.k.data_ptr(), cache.v.data_ptr(), cache.k_scale.data_ptr(),
                           cache.v_scale.data_ptr(), cache.num_pages, 64, table.data_ptr(), table.stride(0), table.shape[1], n.data_ptr(), cu.data_ptr(),
                           3 * new, 3, new, Hq, H, D, D ** -0.5, 0, ws.data_ptr(), need, torch.cuda.current_stream().cuda_stream)
    assert rc == 0, lib.jgq_last_error()
    assert torch.equal(out, cache.attend(q, table, n, cu_seqlens=cu, max_new=new))
    assert bool((ws[need:] == 171).all()) and not bool(ws[:16384].any())


@pytest.mark.parametrize('new', [1, 90])
def test_requests_that_share_pages_and_calls_on_two_streams(G, new):
    """A prefix that two requests have in common lies in the same pages; calls on two streams at once do not meet."""
    lengths = [640, 700, 64 * 9]
    cache, table, gen = filled(G, lengths, 2, 64, 64, 12)
    table[1, :8] = table[0, :8]
    table[2, :9] = table[0, 3]                                            # one page nine times
    q = torch.randn((3 * new, 8, 64), generator=gen, device='cuda').half()
    out = check(cache, table, q, lengths, [new] * 3)
    cu, n = i32([0, new, 2 * new, 3 * new]), i32(lengths)
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(20):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(cache.attend(q, table, n, cu_seqlens=cu, max_new=new))
    torch.cuda.synchronize()
    assert all(torch.equal(o, out) for part in got for o in part)
