"""Paged cache of 8-bit keys and values: block tables and slot maps, quantization of new tokens into their pages, attention
over the pages, and the three together, against plain computations in 64 bits."""
import importlib
import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

DT = {'f16': torch.float16, 'bf16': torch.bfloat16, 'f32': torch.float32}


@pytest.fixture(scope='module')
def G():
    return importlib.import_module('jax_gptq_b200')


def i32(v):
    return torch.tensor(v, dtype=torch.int32, device='cuda')


# --------------------------------------------------------------------------
# tables: whole numbers, against a plain simulation
# --------------------------------------------------------------------------
class Simulated:
    def __init__(self, requests, width, pages, page):
        self.rows, self.width, self.page = [[] for _ in range(requests)], width, page
        self.stack = list(range(pages - 1, -1, -1))

    def reserve(self, lengths, added, most, finished=None):
        if finished is not None:
            for r in reversed(range(len(self.rows))):
                if finished[r]:
                    self.stack += reversed(self.rows[r])
                    self.rows[r] = []
        want = [-(-(a + n) // self.page) for a, n in zip(lengths, added)]
        lack = sum(max(0, w - len(row)) for w, row in zip(want, self.rows))
        fits = lack <= len(self.stack) and max(want) <= self.width and sum(added) <= most and min(list(lengths) + list(added)) >= 0
        if not fits:
            return [-1] * most, [0] * most, [0] * (len(self.rows) + 1), list(lengths)
        slots, pos, cu = [], [], [0]
        for row, a, n, w in zip(self.rows, lengths, added, want):
            while len(row) < w:
                row.append(self.stack.pop())
            for p in range(a, a + n):
                slots.append(row[p // self.page] * self.page + p % self.page)
                pos.append(p)
            cu.append(len(slots))
        return slots + [-1] * (most - len(slots)), pos + [0] * (most - len(pos)), cu, [a + n for a, n in zip(lengths, added)]

    def compare(self, table):
        want = [row + [-1] * (self.width - len(row)) for row in self.rows]
        assert table.block_table.tolist() == want
        assert table.held.tolist() == [len(r) for r in self.rows]
        n = int(table.free_count)
        assert n == len(self.stack) and table.free[:n].tolist() == self.stack


@pytest.mark.parametrize('requests,page,longest,most_new', [(1, 64, 300, 1), (3, 16, 50, 7), (37, 64, 1000, 40), (256, 128, 4000, 1),
                                                            (1023, 64, 500, 3), (1025, 5, 60, 4), (2500, 64, 700, 30), (40, 64, 3000, 900)])
def test_tables_over_many_steps(G, requests, page, longest, most_new):
    rng = np.random.default_rng(requests + page)
    width = -(-(longest + most_new) // page) + 1
    pages = requests * width
    table, sim = G.PageTable(requests, width, pages, page), Simulated(requests, width, pages, page)
    lengths = [0] * requests
    for step in range(6):
        finished = rng.random(requests) < 0.2 if step % 2 else np.zeros(requests, bool)
        lengths = [0 if f else n for f, n in zip(finished, lengths)]
        added = [int(rng.integers(0, most_new + 1)) if n else int(rng.integers(0, min(longest, 4 * most_new) + 1)) for n in lengths]
        added = [min(a, width * page - n) for a, n in zip(added, lengths)]
        most = sum(added) + int(rng.integers(0, 5))
        got = table.reserve(i32(lengths), i32(added), most, torch.tensor(finished, device='cuda') if step % 2 else None)
        slots, pos, cu, after = sim.reserve(lengths, added, most, finished)
        assert got.slots.tolist() == slots and got.positions.tolist() == pos
        assert got.cu_seqlens.tolist() == cu and got.lengths.tolist() == after
        sim.compare(table)
        lengths = after
    table.check()
    table.release(torch.ones(requests, dtype=torch.bool, device='cuda'))
    assert int(table.free_count) == pages and sorted(table.free.tolist()) == list(range(pages))
    assert table.held.sum() == 0 and bool((table.block_table == -1).all())


@pytest.mark.parametrize('why,lengths,added,most', [('too few free pages', [0, 0, 0], [64, 65, 1], 200), ('longer than its row', [0, 0, 193], [0, 0, 64], 64),
                                                    ('more tokens', [0, 0, 0], [2, 2, 2], 5), ('negative length', [0, -1, 0], [1, 1, 1], 9),
                                                    ('negative length', [0, 0, 0], [1, -1, 1], 9), ('negative length', [0, 0, 2 ** 31 - 1], [1, 1, 1], 9)])
def test_tables_all_or_nothing(G, why, lengths, added, most):
    table = G.PageTable(3, 4, 3 if 'pages' in why else 12, 64)
    before = [t.clone() for t in (table.block_table, table.held, table.free_count)]
    got = table.reserve(i32(lengths), i32(added), most)
    assert got.slots.tolist() == [-1] * most and got.cu_seqlens.tolist() == [0] * 4 and got.lengths.tolist() == lengths
    for a, b in zip(before, (table.block_table, table.held, table.free_count)):
        assert torch.equal(a, b)
    with pytest.raises(RuntimeError, match=why):
        table.check()
    table.check()
    got = table.reserve(i32([0, 0, 0]), i32([1, 1, 1]), 3)               # the table goes on
    assert got.slots.tolist() == [0, 64, 128]


def test_tables_keep_pages_of_shortened_requests_and_take_tampered_tables(G):
    table = G.PageTable(2, 8, 16, 64)
    table.reserve(i32([0, 0]), i32([300, 10]), 400)
    held = table.held.tolist()
    got = table.reserve(i32([100, 10]), i32([2, 0]), 2)                  # set back: the pages stay
    assert table.held.tolist() == held == [5, 1]
    row = table.block_table[0].tolist()
    assert got.slots.tolist() == [row[1] * 64 + 36, row[1] * 64 + 37]
    table.held[0] = 99                                                    # more than the row has
    table.reserve(i32([0, 0]), i32([1, 1]), 2)
    with pytest.raises(RuntimeError, match='inconsistent'):
        table.check()
    with pytest.raises(TypeError):
        table.reserve(torch.zeros(2, dtype=torch.int64, device='cuda'), i32([1, 1]), 2)
    with pytest.raises(ValueError):
        table.reserve(i32([0]), i32([1, 1]), 2)
    with pytest.raises(TypeError):
        table.reserve(i32([0, 0]).cpu(), i32([1, 1]), 2)


# --------------------------------------------------------------------------
# write and read: exact
# --------------------------------------------------------------------------
def codes_of(cache):
    """(keys, values) as [pages, heads, token, width] whole numbers."""
    v = cache.v.cpu().numpy().astype(np.int64).transpose(0, 1, 2, 4, 3).reshape(cache.k.shape)
    return cache.k.cpu().numpy().astype(np.int64) - 128, v - 128


def write_reference(codes, scale, x, slots, page):
    """Page by page, quotients in fp32 as the format says, everything else exact."""
    i = 0
    while i < len(slots):
        if slots[i] < 0 or slots[i] >= codes.shape[0] * page:
            i += 1
            continue
        j = i + 1
        while j < len(slots) and slots[j] == slots[j - 1] + 1 and slots[j] // page == slots[i] // page:
            j += 1
        p, o = slots[i] // page, slots[i] % page
        for h in range(codes.shape[1]):
            rows = x[i:j, h].astype(np.float32)
            finite = np.abs(rows[np.isfinite(rows)])
            need = np.float32(finite.max() if finite.size else 0) / np.float32(127)
            s = scale[p, h]
            if o == 0 or not s > 0:
                s = need
            else:
                n = 0
                while s < need:
                    s, n = s * np.float32(2), n + 1
                if n:
                    codes[p, h] = np.round(codes[p, h] / 2.0 ** n)
            scale[p, h] = s
            with np.errstate(all='ignore'):
                q = np.round(np.where(np.isnan(rows), 0, rows) / (s if s > 0 else np.float32(1)))
            codes[p, h, o:o + j - i, :rows.shape[1]] = np.clip(q, -127, 127)
        i = j


@pytest.mark.parametrize('page', [64, 128, 256])
@pytest.mark.parametrize('heads,dim,x', [(2, 64, 'f16'), (1, 128, 'bf16'), (3, 80, 'f32'), (2, 256, 'f16'), (1, 1, 'f32'), (2, 33, 'bf16'), (1, 200, 'f32')])
def test_write_and_read_are_exact(G, page, heads, dim, x):
    rng = np.random.default_rng(page + dim)
    pages = 7
    cache = G.KVCache(pages, heads, dim, page)
    k, v = codes_of(cache)
    ks, vs = cache.k_scale.cpu().numpy(), cache.v_scale.cpu().numpy()
    order = rng.permutation(pages)
    # whole pages, a run that ends inside one, a run that begins inside one, single tokens of growing size, rewritten tokens
    runs = [[(0, page), (1, page), (2, 37)], [(2, 37, 41), (3, 1)], [(3, 1, 2), (2, 41, page)]] + [[(3, i, i + 1), (4, i - 2, i - 1)] for i in range(2, 12)]
    runs += [[(0, 5, 9)], [(5, 17), (6, page - 1)], [(6, page - 1, page)], [(0, 0, 1)]]
    for n, run in enumerate(runs):
        slots = []
        for part in run:
            a, b = (0, part[1]) if len(part) == 2 else part[1:]
            slots += [int(order[part[0]]) * page + o for o in range(a, b)]
            if rng.random() < 0.3:
                slots += [-1, pages * page + 3]                           # nowhere
        new = [torch.tensor(rng.standard_normal((len(slots), heads, dim)) * 1.6 ** n, dtype=torch.float32).to(DT[x]).cuda() for _ in range(2)]
        cache.write(new[0], new[1], torch.tensor(slots, device='cuda'))
        for c, s, t in ((k, ks, new[0]), (v, vs, new[1])):
            write_reference(c, s, t.float().cpu().numpy(), slots, page)
        got_k, got_v = codes_of(cache)
        assert np.array_equal(cache.k_scale.cpu().numpy(), ks) and np.array_equal(cache.v_scale.cpu().numpy(), vs)
        assert np.array_equal(got_k[..., :dim], k[..., :dim]) and np.array_equal(got_v[..., :dim], v[..., :dim])
        assert not got_k[..., dim:].any() and not got_v[..., dim:].any()
    index = [3, 0, 3, pages - 1]
    for dtype in (torch.float32, torch.float16, torch.bfloat16):
        rk, rv = cache.read(torch.tensor(index, device='cuda'), dtype)
        for got, c, s in ((rk, k, ks), (rv, v, vs)):
            want = torch.tensor((c[index][..., :dim].astype(np.float32) * s[index][:, :, None, None])).to(dtype)
            assert got.dtype == dtype and torch.equal(got.cpu(), want)
    rk, rv = cache.read(torch.tensor([-1, pages, 1], device='cuda'))
    assert bool(rk[:2].isnan().all()) and bool(rv[:2].isnan().all()) and bool(rk[2].isfinite().all())


def test_a_token_loses_at_most_a_step_of_its_pages_final_scale(G):
    """Half a step when it is stored, then half a step of every later scale it is rounded to: below one final step."""
    cache = G.KVCache(1, 1, 64, 64)
    x = torch.randn((64, 1, 64), device='cuda') * torch.exp(torch.arange(64, device='cuda') / 8.0)[:, None, None]
    for i in range(64):
        cache.write(x[i:i + 1], -x[i:i + 1], torch.tensor([i], device='cuda'))
    k, v = cache.read(torch.tensor([0], device='cuda'))
    for got, want, s in ((k, x, cache.k_scale), (v, -x, cache.v_scale)):
        assert float((got[0, 0] - want[:, 0]).abs().max()) <= float(s) * (1 + 127 * 2.0 ** -23)


def test_write_of_special_values(G):
    cache = G.KVCache(2, 1, 64, 64)
    x = torch.zeros((3, 1, 64), device='cuda')
    cache.write(x, x, torch.tensor([0, 1, 2], device='cuda'))             # only zeros: scale zero
    assert float(cache.k_scale[0]) == 0 and bool((cache.k[0] == 128).all())
    x[0, 0, :4] = torch.tensor([float('nan'), float('inf'), -float('inf'), 2.0])
    cache.write(x[:1], x[:1], torch.tensor([3], device='cuda'))
    k, v = cache.read(torch.tensor([0], device='cuda'))
    for got in (k, v):
        assert got[0, 0, 3, :4].tolist() == [0.0, 2.0, -2.0, 2.0]          # 127 steps of 2 / 127
    tiny = torch.full((1, 1, 64), 1e-42, device='cuda')
    cache.write(tiny, tiny, torch.tensor([64], device='cuda'))
    cache.write(tiny * 0 + 3e38, tiny, torch.tensor([65], device='cuda'))  # grows over the whole range of fp32
    k, v = cache.read(torch.tensor([1], device='cuda'))
    assert bool(k.isfinite().all()) and abs(float(k[0, 0, 1, 0]) / 3e38 - 1) < 1 / 127 and float(k[0, 0, 0, 0]) == 0
    cache.write(x[:0], x[:0], torch.zeros(0, dtype=torch.int64, device='cuda'))


def test_write_takes_strided_rows(G):
    qkv = torch.randn((10, 3, 4, 72), device='cuda').half()
    k, v = qkv[:, 1, :, :64], qkv[:, 2, 1:3].transpose(0, 1).contiguous().transpose(0, 1)[..., 3:67]
    slots = torch.arange(10, device='cuda')
    a, b = G.KVCache(1, 4, 64), G.KVCache(1, 4, 64)
    a.write(k, k, slots)
    b.write(k.contiguous(), k.contiguous(), slots)
    assert torch.equal(a.k, b.k) and torch.equal(a.v, b.v)
    a, b = G.KVCache(1, 2, 64), G.KVCache(1, 2, 64)
    a.write(v, v, slots)
    b.write(v.contiguous(), v.contiguous(), slots)
    assert torch.equal(a.k, b.k) and torch.equal(a.v, b.v)


# --------------------------------------------------------------------------
# attention
# --------------------------------------------------------------------------
def filled(G, lengths, kv_heads, dim, page, seed, spare=3, spread=4.0):
    """A cache with random codes everywhere (also behind the sequences), random scales, pages in random order."""
    gen = torch.Generator(device='cuda').manual_seed(seed)
    counts = [-(-n // page) for n in lengths]
    pages = max(1, sum(counts) + spare)
    cache = G.KVCache(pages, kv_heads, dim, page)
    cache.k.copy_(torch.randint(0, 256, cache.k.shape, generator=gen, device='cuda', dtype=torch.uint8))
    cache.v.copy_(torch.randint(0, 256, cache.v.shape, generator=gen, device='cuda', dtype=torch.uint8))
    cache.k[..., dim:] = 128
    cache.v[..., dim:, :] = 128
    for s, unit in ((cache.k_scale, 0.02), (cache.v_scale, 0.02)):
        s.copy_(unit * torch.exp(math.log(spread) * (torch.rand(s.shape, generator=gen, device='cuda') - 0.5)))
    order = torch.randperm(pages, generator=gen, device='cuda').to(torch.int32)
    width = max([1] + counts) + 1
    table = torch.full((len(lengths), width), -1, dtype=torch.int32, device='cuda')
    at = 0
    for r, n in enumerate(counts):
        table[r, :n] = order[at:at + n]
        at += n
    return cache, table, gen


def rows_of(cache, table, r, length):
    """Keys and values of a sequence in 64 bits: [heads, length, dim]."""
    D, P = cache.head_dim, cache.page_size
    n = -(-length // P)
    if n == 0:
        z = torch.zeros((cache.kv_heads, 0, D), dtype=torch.float64, device='cuda')
        return z, z
    idx = table[r, :n].long()
    k = (cache.k[idx].double() - 128) * cache.k_scale[idx].double()[:, :, None, None]
    v = (cache.v[idx].double() - 128) * cache.v_scale[idx].double()[:, :, None, None, None]
    v = v.transpose(3, 4).reshape(k.shape)
    return [t.transpose(0, 1).reshape(cache.kv_heads, n * P, -1)[:, :length, :D] for t in (k, v)]


def attend_reference(cache, table, q, lengths, new, scale):
    """(output, lse, tolerance of the output, of lse) in 64 bits, row by row of the formula.

    What the kernel rounds: scores are fp32 sums of exact products of q (f16: exact; fp32: 22 bits) and codes in excess 128, at most
    DW / 16 + 2 truncated additions of terms that reach |q| (|k| + 128 scale), so a score is off by `d` below; p is rounded to f16
    (2^-11; with fp32 calls in two parts, 2^-21) or lost below 2^-25, and p's numerator and denominator use the same values; the
    values' sums in excess 128 lose 2^-22 of 256 scales per 64 tokens, and running fp32 sums 2^-23 per tile; out is rounded once."""
    Hq, D, H = q.shape[1], q.shape[2], cache.kv_heads
    f32 = q.dtype == torch.float32
    out = torch.zeros(q.shape, dtype=torch.float64, device='cuda')
    lse = torch.full(q.shape[:2], -math.inf, dtype=torch.float64, device='cuda')
    tol, tol_lse = torch.zeros_like(out), torch.zeros_like(lse)
    u = torch.finfo(q.dtype).eps / 2
    at = 0
    for r, (L, n) in enumerate(zip(lengths, new)):
        k, v = rows_of(cache, table, r, L)
        for i in range(n):
            see = max(0, min(L, L - n + i + 1))
            if see == 0:
                continue
            for h in range(Hq):
                kh, vh = k[h // (Hq // H)][:see], v[h // (Hq // H)][:see]
                qr = q[at + i, h].double()
                s = (kh @ qr) * scale
                m = s.max()
                e = torch.exp(s - m)
                p = e / e.sum()
                out[at + i, h] = p @ vh
                lse[at + i, h] = m + torch.log(e.sum())
                ks = cache.k_scale[table[r, :-(-see // cache.page_size)].long(), h // (Hq // H)].double().repeat_interleave(cache.page_size)[:see]
                big = ((kh.abs() @ qr.abs()) + 128 * ks * qr.abs().sum()) * abs(scale)
                d = float(((D / 16 + 6) * 2.0 ** -23 * big).max()) + 2.0 ** -21 * float(s.abs().max() + 1)
                rp = (2.0 ** -21 if f32 else 2.0 ** -11) + 2.0 ** -21
                tiles = see / 64 + 2
                vmax = float(vh.abs().max())
                vs = float(cache.v_scale.max())
                tol[at + i, h] = (2 * (d + rp) * (p @ vh.abs()) + see * 2.0 ** (-35 if f32 else -25) * 2 * vmax
                                  + 2.0 ** -22 * 256 * vs * 2 + tiles * 2.0 ** -23 * vmax + u * out[at + i, h].abs())
                tol_lse[at + i, h] = d + rp + tiles * 2.0 ** -23 + see * 2.0 ** -25 + 2.0 ** -22 * lse[at + i, h].abs()
        at += n
    return out, lse, tol, tol_lse


def run_attend(G, lengths, new, Hq, H, D, page, dtype, seed=0, scale=None, **kw):
    cache, table, gen = filled(G, lengths, H, D, page, seed)
    T = sum(new)
    q = (torch.randn((T, Hq, D), generator=gen, device='cuda')).to(dtype)
    cu = i32(np.concatenate([[0], np.cumsum(new)]).tolist())
    single = all(n == 1 for n in new) and not kw.get('force_cu')
    args = dict(scale=scale, return_lse=True)
    if not single:
        args.update(cu_seqlens=cu, max_new=max(new))
    out, lse = cache.attend(q, table, i32(lengths), **args)
    want, wl, tol, tl = attend_reference(cache, table, q, lengths, new, D ** -0.5 if scale is None else scale)
    off = (out.double() - want).abs()
    assert out.dtype == dtype and out.shape == q.shape and bool(out.isfinite().all())
    assert bool((off <= tol).all()), f'{float((off / tol.clamp(min=1e-300)).max())} of the tolerance'
    fin = torch.isfinite(wl)
    assert torch.equal(torch.isfinite(lse), fin)
    assert bool(((lse.double() - wl).abs()[fin] <= tl[fin]).all())
    return cache, table, q, cu, out


@pytest.mark.parametrize('x', ['f16', 'bf16', 'f32'])
@pytest.mark.parametrize('Hq,H,D', [(12, 12, 64), (8, 1, 128), (6, 2, 256), (4, 2, 80), (3, 1, 33), (20, 4, 96), (16, 1, 64), (24, 1, 128), (2, 2, 1), (10, 2, 200)])
@pytest.mark.parametrize('page', [64, 256])
def test_single_tokens(G, x, Hq, H, D, page):
    run_attend(G, [1, 64, 0, 65, 300, 63, 577], [1] * 7, Hq, H, D, page, DT[x], seed=D)


@pytest.mark.parametrize('x', ['f16', 'bf16', 'f32'])
@pytest.mark.parametrize('lengths,new', [([5], [5]), ([1], [1]), ([130, 64, 7], [3, 64, 7]), ([200, 0, 90], [70, 0, 1]), ([65, 128, 129, 40], [1, 2, 65, 17]),
                                         ([3, 500], [5, 9]), ([0, 2], [4, 2])])
@pytest.mark.parametrize('Hq,H,D', [(4, 4, 64), (8, 1, 128), (5, 1, 96), (2, 1, 256)])
def test_several_tokens_per_sequence(G, x, lengths, new, Hq, H, D):
    """Prompts, chunks behind a prefix, speculation; more rows than tokens: the first ones see nothing and are zero."""
    cache, table, q, cu, out = run_attend(G, lengths, new, Hq, H, D, 128, DT[x], seed=sum(lengths), force_cu=True)
    at = 0
    for L, n in zip(lengths, new):
        hidden = max(0, n - L)
        assert bool((out[at:at + hidden] == 0).all())
        at += n


@pytest.mark.parametrize('x', ['f16', 'f32'])
@pytest.mark.parametrize('B,L,Hq,H,D', [(1, 20000, 8, 8, 64), (1, 9000, 8, 1, 128), (3, 5000, 4, 2, 128), (150, 130, 4, 4, 64), (700, 3, 2, 1, 64)])
def test_long_sequences_and_large_batches(G, x, B, L, Hq, H, D):
    """Items shared by many CTAs and CTAs with many items."""
    rng = np.random.default_rng(B)
    lengths = [int(L * (0.2 + 0.8 * rng.random())) for _ in range(B)]
    run_attend(G, lengths, [1] * B, Hq, H, D, 64, DT[x], seed=B)


@pytest.mark.parametrize('scale', [0.0, -0.3, 1.5, 1e-3])
def test_other_scales(G, scale):
    run_attend(G, [200, 31], [1, 1], 4, 2, 64, 64, torch.float32, scale=scale)


@pytest.mark.parametrize('new', [1, 40])
@pytest.mark.parametrize('x', ['f16', 'bf16', 'f32'])
def test_results_do_not_depend_on_the_run_or_on_what_lies_behind(G, new, x):
    """The same bits every time, also with other codes, NaN scales and bad page numbers in places that no row sees."""
    lengths, news = [1000, 77, 3000], [new] * 3
    cache, table, q, cu, out = run_attend(G, lengths, news, 4, 2, 64, 64, DT[x], force_cu=new > 1)
    kw = dict(cu_seqlens=cu, max_new=new) if new > 1 else {}
    for _ in range(3):
        assert torch.equal(cache.attend(q, table, i32(lengths), **kw), out)
    used = torch.zeros(cache.num_pages, dtype=torch.bool, device='cuda')
    for r, L in enumerate(lengths):
        n = -(-L // 64)
        used[table[r, :n].long()] = True
        table[r, n:] = 10 ** 9
        if L % 64:
            cache.k[table[r, n - 1].long(), :, L % 64:] = 255
            cache.v[table[r, n - 1].long(), :, 0, :, L % 64:] = 0
    cache.k_scale[~used] = float('nan')
    cache.v_scale[~used] = float('inf')
    assert torch.equal(cache.attend(q, table, i32(lengths), **kw), out)
    wide = torch.full((3, 100), -7, dtype=torch.int32, device='cuda')
    wide[:, :table.shape[1]] = table
    assert torch.equal(cache.attend(q, wide[:, :table.shape[1]], i32(lengths), **kw), out)
    # q, a slice of a wider tensor
    packed = torch.zeros((q.shape[0], 7, 72), dtype=q.dtype, device='cuda')
    packed[:, 2:6, 5:69] = q
    assert torch.equal(cache.attend(packed[:, 2:6, 5:69], table, i32(lengths), **kw), out)
    assert torch.equal(cache.attend(q, table, i32(lengths), out=torch.empty_like(q), **kw), out)


@pytest.mark.parametrize('bad', [-1, 10 ** 9, 'length', 'scale'])
@pytest.mark.parametrize('new', [1, 30])
def test_a_bad_page_makes_its_rows_nan_and_no_others(G, bad, new):
    lengths = [100, 200, 300]
    cache, table, gen = filled(G, lengths, 2, 64, 64, 1)
    q = torch.randn((3 * new, 4, 64), device='cuda').half()
    kw = dict(cu_seqlens=i32([0, new, 2 * new, 3 * new]), max_new=new) if new > 1 else {}
    good = cache.attend(q, table, i32(lengths), **kw)
    if bad == 'length':
        lengths[1] = 10 ** 6                                              # more than its row of the table holds: -1 there
    elif bad == 'scale':
        cache.k_scale[table[1, 0].long()] = float('nan')
    else:
        table[1, 0] = bad
    got = cache.attend(q, table, i32(lengths), **kw)
    assert bool(got[new:2 * new].isnan().all())
    assert torch.equal(got[:new], good[:new]) and torch.equal(got[2 * new:], good[2 * new:])


def test_a_causal_row_takes_nothing_of_a_page_it_does_not_see(G):
    """A later page with NaN scales: the rows before it are what they are without it."""
    cache, table, gen = filled(G, [128], 1, 64, 64, 2)
    q = torch.randn((100, 2, 64), device='cuda').half()
    kw = dict(cu_seqlens=i32([0, 100]), max_new=100)
    good = cache.attend(q, table, i32([128]), **kw)
    cache.k_scale[table[0, 1].long()] = float('nan')
    cache.v_scale[table[0, 1].long()] = float('nan')
    got = cache.attend(q, table, i32([128]), **kw)
    first = 64 - 28                                                       # row i sees 28 + i + 1 tokens
    assert torch.equal(got[:first], good[:first]) and bool(got[first:].isnan().all())


def test_rows_behind_the_last_sequence(G):
    lengths, new = [70, 5], [3, 2]
    cache, table, gen = filled(G, lengths, 2, 64, 64, 3)
    q = torch.randn((9, 4, 64), device='cuda').half()
    q[5:] = float('nan')
    cu = i32([0, 3, 5])
    fresh = cache.attend(q, table, i32(lengths), cu_seqlens=cu, max_new=3)
    assert bool((fresh[5:] == 0).all()) and bool(fresh[:5].isfinite().all())
    out = torch.full_like(q, 7.0)
    cache.attend(q, table, i32(lengths), cu_seqlens=cu, max_new=3, out=out)
    assert torch.equal(out[:5], fresh[:5]) and bool((out[5:] == 7).all())
    # a wrong guess of max_new costs nothing but time
    for guess in (1, 2, 100, None):
        again = cache.attend(q, table, i32(lengths), cu_seqlens=cu, max_new=guess)
        assert float((again[:5].float() - fresh[:5].float()).abs().max()) <= 2.0 ** -8 * float(fresh[:5].abs().max())
    none = cache.attend(q[:0], table[:0], i32([]), cu_seqlens=i32([0]))
    assert none.shape == (0, 4, 64)
    assert bool((cache.attend(q, table, i32([0, 0]), cu_seqlens=cu) [:5] == 0).all())
    assert bool((cache.attend(q, table, i32(lengths), cu_seqlens=i32([0, 0, 0])) == 0).all())


def test_special_values_of_q(G):
    cache, table, gen = filled(G, [90], 1, 64, 64, 4)
    q = torch.randn((1, 4, 64), device='cuda')
    q[0, 0] = 0
    q[0, 1] *= 1e-30
    q[0, 2, 3] = float('nan')
    q[0, 3] *= 1e4
    for dtype in (torch.float32, torch.bfloat16):
        out = cache.attend(q.to(dtype), table, i32([90]))
        assert bool(out[0, [0, 1, 3]].isfinite().all()) and bool(out[0, 2].isnan().all())
        k, v = rows_of(cache, table, 0, 90)
        mean = v[0].mean(0)                                                # all weights equal
        for h in (0, 1):
            assert float((out[0, h].double() - mean).abs().max()) <= 2.0 ** -7 * float(v.abs().max())
        top = v[0, int((k[0] @ q[0, 3].double()).argmax())]               # one weight
        assert float((out[0, 3].double() - top).abs().max()) <= 2.0 ** -7 * float(v.abs().max())


def test_attend_refusals(G):
    cache, table, gen = filled(G, [10], 2, 64, 64, 5)
    q = torch.randn((1, 4, 64), device='cuda').half()
    n = i32([10])
    for bad in (dict(q=q[:, :3]), dict(q=q[..., :32]), dict(q=q.expand(2, 4, 64)), dict(block_table=table.long()), dict(lengths=i32([1, 2])),
                dict(out=torch.empty((1, 4, 32), device='cuda').half()), dict(out=torch.empty((1, 4, 64), device='cuda')), dict(cu_seqlens=i32([0])),
                dict(q=q.clone().requires_grad_())):
        with pytest.raises(ValueError):
            cache.attend(**{**dict(q=q, block_table=table, lengths=n), **bad})
    for bad in (dict(q=q.double()), dict(q=q.cpu()), dict(lengths=n.long()), dict(lengths=n.cpu())):
        with pytest.raises(TypeError):
            cache.attend(**{**dict(q=q, block_table=table, lengths=n), **bad})
    with pytest.raises(TypeError):
        cache.write(q[:, :2], q[:, :2], i32([0]))
    with pytest.raises(ValueError):
        cache.write(q[:, :2], q[:, :2].float(), torch.tensor([0], device='cuda'))
    with pytest.raises(ValueError):
        cache.write(q, q, torch.tensor([0], device='cuda'))
    with pytest.raises(TypeError):
        cache.read(i32([0]))


# --------------------------------------------------------------------------
# together
# --------------------------------------------------------------------------
def test_a_serving_loop(G):
    """Prompts, decode steps, a request that leaves and one that takes its place: linears with grouped weights around the
    attention, all of it against the same loop in 64 bits on the dequantized values."""
    from tests.test_gpu_group_matmul import matrix
    B, H, Hq, D, page, hidden = 3, 2, 4, 64, 64, 128
    qkv, wq, _ = matrix(G, hidden, (Hq + 2 * H) * D, 64, seed=1)
    proj, wo, _ = matrix(G, Hq * D, hidden, 32, seed=2)
    table, cache = G.PageTable(B, 8, 20, page), G.KVCache(20, H, D, page)
    gen = torch.Generator(device='cuda').manual_seed(0)
    lengths, kept = i32([0, 0, 0]), [[], [], []]
    steps = [([70, 3, 129], None)] + [([1, 1, 1], None)] * 3 + [([1, 40, 2], [False, True, False])] + [([1, 1, 1], None)] * 2
    for added, finished in steps:
        if finished:
            lengths = torch.where(torch.tensor(finished, device='cuda'), 0, lengths).int()
            kept = [[] if f else r for f, r in zip(finished, kept)]
        T = sum(added)
        step = table.reserve(lengths, i32(added), T, torch.tensor(finished, device='cuda') if finished else None)
        x = torch.randn((T, hidden), generator=gen, device='cuda')
        y = G.quantized_matmul(x, qkv).view(T, Hq + 2 * H, D)
        cache.write(y[:, Hq:Hq + H], y[:, Hq + H:], step.slots)
        out = cache.attend(y[:, :Hq], table.block_table, step.lengths, step.cu_seqlens, max(added))
        z = G.quantized_matmul(out.view(T, Hq * D), proj)
        lengths = step.lengths
        # in 64 bits, keys and values as the cache has them now
        y64 = (x.double() @ wq).view(T, Hq + 2 * H, D)
        assert float((y.double() - y64).abs().max()) <= 1e-4 * float(y64.abs().max())
        want, _, tol, _ = attend_reference(cache, table.block_table, y[:, :Hq].contiguous(), lengths.tolist(), added, D ** -0.5)
        assert bool(((out.double() - want).abs() <= tol).all())
        at = 0
        for r, n in enumerate(added):
            kept[r].append(y[at:at + n, Hq:])
            at += n
            rows = torch.cat(kept[r]).double()
            k, v = rows_of(cache, table.block_table, r, int(lengths[r]))
            pages = table.block_table[r, :-(-int(lengths[r]) // page)].long()
            for got, ref, sc in ((k, rows[:, :H], cache.k_scale), (v, rows[:, H:], cache.v_scale)):
                step_of = sc[pages].double().repeat_interleave(page, 0)[:got.shape[1]].transpose(0, 1)[:, :, None]
                assert bool(((got - ref.transpose(0, 1)).abs() <= 1.001 * step_of).all())
        assert float((z.double() - want.reshape(T, -1) @ wo).abs().max()) <= 1e-3 * float(z.abs().max()) + float(tol.max()) * float(wo.abs().sum(0).max())
    table.check()


@pytest.mark.parametrize('x', ['f16', 'f32'])
def test_a_captured_step_replayed_with_new_lengths(G, x):
    """A decode step for a padded batch in one graph: replays follow the lengths on the device; a second graph and an eager
    call beside it."""
    dtype = DT[x]
    B, H, Hq, D = 4, 2, 8, 128
    table, cache = G.PageTable(B, 6, 24, 64), G.KVCache(24, H, D, 64)
    lengths, added = i32([0] * B), i32([0] * B)
    y = torch.zeros((B, Hq + 2 * H, D), dtype=dtype, device='cuda')

    def step():
        s = table.reserve(lengths, added, B)
        cache.write(y[:, Hq:Hq + H], y[:, Hq + H:], s.slots)
        return s, cache.attend(y[:, :Hq], table.block_table, s.lengths, s.cu_seqlens, 1)
    step()
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            s, out = step()
        graphs.append((g, s, out))
    other_table, other = G.PageTable(B, 6, 24, 64), G.KVCache(24, H, D, 64)
    ol = i32([0] * B)
    gen = torch.Generator(device='cuda').manual_seed(1)
    for i in range(70):
        n = [1, int(i % 2 == 0), 1, int(i > 60)]
        added.copy_(i32(n))
        y.copy_(torch.randn(y.shape, generator=gen, device='cuda'))
        g, s, out = graphs[i % 2]
        g.replay()
        es = other_table.reserve(ol, i32(n), B)
        other.write(y[:, Hq:Hq + H], y[:, Hq + H:], es.slots)
        want = other.attend(y[:, :Hq], other_table.block_table, es.lengths, es.cu_seqlens, 1)
        assert torch.equal(s.slots, es.slots) and torch.equal(s.lengths, es.lengths) and torch.equal(out, want)
        assert bool((out[sum(n):] == 0).all())
        lengths.copy_(s.lengths)
        ol = es.lengths
    table.check()
    assert torch.equal(cache.k, other.k) and torch.equal(cache.v_scale, other.v_scale)


def test_two_graphs_of_one_stream_replayed_at_once(G):
    cache, table, gen = filled(G, [4000, 100], 1, 128, 64, 6)
    qs = [torch.randn((2, 8, 128), device='cuda').half() for _ in range(2)]
    n = i32([4000, 100])
    want = [cache.attend(q, table, n) for q in qs]
    graphs, outs = [], []
    for q in qs:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            for _ in range(4):
                o = cache.attend(q, table, n)
        graphs.append(g)
        outs.append(o)
    streams = [torch.cuda.Stream() for _ in graphs]
    torch.cuda.synchronize()
    for _ in range(30):
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    for o, w in zip(outs, want):
        assert torch.equal(o, w)


def test_offsets_beyond_32_bits(G):
    """A pool of more than 4 GB: pages at its end are written, read and attended."""
    free, _ = torch.cuda.mem_get_info()
    pages = 66000                                                         # 66000 * 8 * 64 * 128 = 4.3 GB each for k and v
    if free < 12e9:
        pytest.skip('needs 12 GB')
    cache = G.KVCache(pages, 8, 128, 64)
    k, v = (torch.randn((64, 8, 128), device='cuda').half() for _ in range(2))
    last = pages - 1
    cache.write(k, v, torch.arange(64, device='cuda') + last * 64)
    rk, rv = cache.read(torch.tensor([last], device='cuda'))
    for got, want, s in ((rk, k, cache.k_scale), (rv, v, cache.v_scale)):
        assert float((got[0].transpose(0, 1) - want.float()).abs().max()) <= 0.51 * float(s[last].max())
    assert bool((cache.k[:last] == 128).all())
    table = i32([[last]])
    q = torch.randn((1, 8, 128), device='cuda').half()
    out = cache.attend(q, table, i32([64]))
    want, _, tol, _ = attend_reference(cache, table, q, [64], [1], 128 ** -0.5)
    assert bool(((out.double() - want).abs() <= tol).all())
