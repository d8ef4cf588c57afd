"""Measured operators of a quantized model's serving and fine-tuning step, and their plain forms.

  matmul, grad  `quantized_matmul` on int4 weights with a scale and a zero point per group of the contraction axis and
                output channel, and the gradient of its input.
  attend        attention over a paged cache of 8-bit keys and values with one scale per page and head: single tokens
                and several tokens per sequence.
  write         new keys and values quantized into their pages; the pages' values read back.
  tables        block tables, slot maps and positions from request lengths, pages of finished requests given back first.

`listed()` holds the fixed cases, `draw(rng)` more of the same ranges; `prepare` makes what a program has in hand before
the call, `run` is one pass, `exact` the same outputs in 64 bits.  With `own` false `run` computes the operators from
elementary torch operations, with `own` true it calls the framework.
"""
from __future__ import annotations

import math
import random

import torch

own = False

_DTYPES = {'f32': torch.float32, 'f16': torch.float16, 'bf16': torch.bfloat16}
_BYTES = {'f32': 4, 'f16': 2, 'bf16': 2}


# --------------------------------------------------------------------------
# the cases
# --------------------------------------------------------------------------
def listed():
    return [
        # One token through one linear of a 7B-sized model, groups of 128: the smallest product, launches and latency count.
        dict(name='decode_m1_4096x4096_g128_f16', kind='matmul', M=1, K=4096, N=4096, group=128, x='f16', zs='f16'),
        # One token through the widest linear of a 70B-sized block: the packed weights stream once from HBM.
        dict(name='decode_m1_8192x28672_g128_bf16', kind='matmul', M=1, K=8192, N=28672, group=128, x='bf16', zs='f16'),
        # A prompt of 2048 tokens.
        dict(name='prefill_m2048_4096x11008_g128_bf16', kind='matmul', M=2048, K=4096, N=11008, group=128, x='bf16', zs='f32'),
        # Fine-tuning around a frozen quantized linear: the product and the gradient of its input, small groups.
        dict(name='tune_m1024_11008x4096_g64_bf16', kind='grad', M=1024, K=11008, N=4096, group=64, x='bf16', zs='f32'),
        # Odd channel count, ragged token count, a last group that is not full, fp32 activations, with the gradient.
        dict(name='ragged_m137_272x909_g32_f32', kind='grad', M=137, K=272, N=909, group=32, x='f32', zs='f32'),
        # One sequence of a GPT-2-small-shaped model, fp32: the smallest attention call.
        dict(name='attend_b1_gpt2_f32', kind='attend', B=1, new=1, longest=700, heads=12, kv_heads=12, dim=64, page=64, x='f32'),
        # A decode step of 64 sequences of very different lengths, 70B-shaped heads.
        dict(name='attend_b64_decode_bf16', kind='attend', B=64, new=1, longest=32768, heads=64, kv_heads=8, dim=128, page=64, x='bf16'),
        # Chunks of four prompts over what is cached of them already, 7B-shaped heads.
        dict(name='attend_b4_chunk512_f16', kind='attend', B=4, new=512, longest=4096, heads=32, kv_heads=32, dim=128, page=128, x='f16'),
        # The keys and values of one decode step of 256 sequences: one row each into pages that are partly full.
        dict(name='write_b256_decode_bf16', kind='write', B=256, new=1, kv_heads=8, dim=128, page=64, x='bf16'),
        # The keys and values of a batch of prompts.
        dict(name='write_b6_prompt_f16', kind='write', B=6, new=2000, kv_heads=32, dim=128, page=128, x='f16'),
        # A decode step's bookkeeping: one token each, a few sequences replaced by new ones.
        dict(name='tables_b256_decode', kind='tables', B=256, new=1, longest=8192, page=64, finished=0.03),
        # Prompts admitted to a large batch at once.
        dict(name='tables_b1024_prompts', kind='tables', B=1024, new=400, longest=4096, page=64, finished=0.25),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


_HEADS = ((12, 12, 64), (32, 32, 128), (64, 8, 128), (32, 8, 128), (24, 3, 64), (16, 1, 256), (20, 4, 96), (14, 2, 80))


def draw(rng):
    kind = rng.choice(['matmul', 'matmul', 'matmul', 'grad', 'grad', 'attend', 'attend', 'attend', 'attend', 'write', 'write', 'tables'])
    if kind in ('matmul', 'grad'):
        while True:
            M = _log_int(rng, 1, 2048)
            align = rng.choice([1, 16, 128])         # a third of the shapes as they fall, K even because two codes share a byte
            K, N = _log_int(rng, 256, 11008), _log_int(rng, 256, 28672)
            K, N = K // max(2, align) * max(2, align), N // align * align
            if M * K * N * (2 if kind == 'grad' else 1) <= 2048 * 4096 * 11008:
                break
        return dict(kind=kind, M=M, K=K, N=N, group=rng.choice([32, 64, 128, 128]), x=rng.choice(['f16', 'bf16', 'f32']),
                    zs=rng.choice(['f16', 'f32']))
    if kind == 'attend':
        heads, kv_heads, dim = rng.choice(_HEADS)
        while True:
            new = 1 if rng.random() < 0.6 else _log_int(rng, 2, 512)
            B, longest = _log_int(rng, 1, 128), _log_int(rng, new, 32768)
            if B * longest * kv_heads * dim <= 1 << 29 and B * new * longest * heads * dim <= 1 << 35:
                break
        return dict(kind=kind, B=B, new=new, longest=longest, heads=heads, kv_heads=kv_heads, dim=dim,
                    page=rng.choice([64, 64, 128, 256]), x=rng.choice(['f16', 'bf16', 'bf16', 'f32']))
    if kind == 'write':
        _, kv_heads, dim = rng.choice(_HEADS)
        while True:
            new, B = 1 if rng.random() < 0.5 else _log_int(rng, 2, 2048), _log_int(rng, 1, 256)
            if B * new * kv_heads * dim <= 1 << 26:
                break
        return dict(kind=kind, B=B, new=new, kv_heads=kv_heads, dim=dim, page=rng.choice([64, 64, 128, 256]),
                    x=rng.choice(['f16', 'bf16', 'f32']))
    new = 1 if rng.random() < 0.5 else _log_int(rng, 2, 512)
    return dict(kind=kind, B=_log_int(rng, 1, 1024), new=new, longest=_log_int(rng, new, 8192), page=rng.choice([16, 64, 128]),
                finished=rng.choice([0.0, 0.05, 0.3]))


# --------------------------------------------------------------------------
# sizes that follow from a case
# --------------------------------------------------------------------------
def _rng(case):
    return random.Random(repr(sorted((k, v) for k, v in case.items() if k != 'name')))


def _pages(tokens, page):
    return (tokens + page - 1) // page


def _sequences(case):
    """(lengths with the new tokens, new tokens) of every sequence: lengths spread over their logarithm, the first one the
    longest; where several tokens are new, some sequences bring fewer."""
    rng = _rng(case)
    lengths, new = [], []
    for i in range(case['B']):
        n = case['new'] if i == 0 or case['new'] == 1 else rng.randint(max(1, case['new'] // 2), case['new'])
        lengths.append(case['longest'] if i == 0 else max(n, _log_int(rng, max(1, case['longest'] // 128), case['longest'])))
        new.append(n)
    return lengths, new


def _writes(case):
    """(tokens that are there, new tokens) of every sequence of a write."""
    rng = _rng(case)
    start, new = [], []
    for i in range(case['B']):
        start.append(rng.randrange(case['page']) if case['new'] == 1 else rng.choice([0, 0, rng.randrange(case['page'])]))
        new.append(case['new'] if i == 0 or case['new'] == 1 else rng.randint(max(1, case['new'] // 2), case['new']))
    return start, new


def _requests(case):
    """(tokens that are there, new tokens, left) of every request; where one left, another one begins."""
    rng = _rng(case)
    start, new, left = [], [], []
    for _ in range(case['B']):
        gone = rng.random() < case['finished']
        start.append(0 if gone else _log_int(rng, 1, case['longest']))
        new.append(_log_int(rng, 1, case['longest']) if gone else rng.randint(1, case['new']))
        left.append(gone)
    return start, new, left


def _width(dim):
    """Bytes of a stored row: head dimensions are padded to 64, 128 or 256."""
    return 64 if dim <= 64 else 128 if dim <= 128 else 256


# --------------------------------------------------------------------------
# inputs
# --------------------------------------------------------------------------
def _generator(seed):
    return torch.Generator(device='cuda').manual_seed(seed)


def _randn(gen, shape, dtype):
    return torch.randn(shape, generator=gen, device='cuda').to(_DTYPES[dtype])


def _int32(values):
    return torch.tensor(values, dtype=torch.int32, device='cuda')


def _weights(case, gen):
    """Uniform codes, scales ~ U(0.001, 0.02), whole zeros in [0, 15], per group and channel; activations."""
    K, N = case['K'], case['N']
    groups = (K + case['group'] - 1) // case['group']
    packed = torch.randint(0, 256, (K // 2, N), generator=gen, dtype=torch.uint8, device='cuda')
    scale = (0.001 + 0.019 * torch.rand((groups, N), generator=gen, device='cuda')).to(_DTYPES[case['zs']])
    zero = torch.randint(0, 16, (groups, N), generator=gen, device='cuda').to(_DTYPES[case['zs']])
    s = dict(packed=packed, scale=scale, zero=zero, group=case['group'], x=_randn(gen, (case['M'], K), case['x']))
    if case['kind'] == 'grad':
        s['dy'] = _randn(gen, (case['M'], N), case['x'])
    return s


def _codes(gen, shape):
    """8-bit codes, excess 128, of normally distributed values whose largest come near the range's end."""
    c = torch.empty(shape, dtype=torch.uint8, device='cuda')
    for part in c.split(max(1, (1 << 26) // max(1, c[0].numel()))):
        part.copy_((torch.randn(part.shape, generator=gen, device='cuda') * 36).round_().clamp_(-127, 127) + 128)
    return c


def _pool(case, gen, count):
    """The cache's tensors: codes of keys [pages, heads, page, width], of values [pages, heads, page / 64, width, 64], and
    a scale per page and head.  The columns behind the head dimension hold zeros (code 128)."""
    H, D, P, W = case['kv_heads'], case['dim'], case['page'], _width(case['dim'])
    k, v = _codes(gen, (count, H, P, W)), _codes(gen, (count, H, P // 64, W, 64))
    k[..., D:] = 128
    v[..., D:, :] = 128
    ks, vs = (0.01 + 0.03 * torch.rand((2, count, H), generator=gen, device='cuda')).unbind(0)
    return dict(k=k, v=v, k_scale=ks.contiguous(), v_scale=vs.contiguous())


def _table(gen, counts, spare):
    """Pages handed out at random: (block table, pages in all)."""
    total = sum(counts) + spare
    order = torch.randperm(total, generator=gen, device='cuda').tolist()
    rows, at = [], 0
    for c in counts:
        rows.append(order[at:at + c])
        at += c
    width = max(1, max(counts))
    return _int32([r + [-1] * (width - len(r)) for r in rows]), total, rows


def _attend_inputs(case, gen):
    lengths, new = _sequences(case)
    table, total, rows = _table(gen, [_pages(n, case['page']) for n in lengths], 3)
    s = _pool(case, gen, total)
    cu = [0]
    for n in new:
        cu.append(cu[-1] + n)
    s.update(table=table, rows=rows, lengths=lengths, new=new, most=max(new), lengths_gpu=_int32(lengths),
             cu_gpu=_int32(cu), dim=case['dim'], page=case['page'],
             q=_randn(gen, (cu[-1], case['heads'], case['dim']), case['x']) * 2)
    return s


def _write_inputs(case, gen):
    start, new = _writes(case)
    table, total, rows = _table(gen, [_pages(a + n, case['page']) for a, n in zip(start, new)], 0)
    s = _pool(case, gen, total)
    slots = [rows[r][p // case['page']] * case['page'] + p % case['page'] for r, (a, n) in enumerate(zip(start, new)) for p in range(a, a + n)]
    shape = (len(slots), case['kv_heads'], case['dim'])
    # a token's magnitude varies: some of the new ones go beyond their page's range
    size = torch.exp(0.5 * torch.randn((2, len(slots), 1, 1), generator=gen, device='cuda'))
    k, v = (torch.randn((2,) + shape, generator=gen, device='cuda') * size).to(_DTYPES[case['x']]).unbind(0)
    s.update(k_new=k.contiguous(), v_new=v.contiguous(), slots_host=slots, slots=torch.tensor(slots, device='cuda'),
             pages=torch.arange(total, device='cuda'), dim=case['dim'], page=case['page'])
    return s


def _tables_inputs(case, gen):
    start, new, left = _requests(case)
    P = case['page']
    held = [_pages(new[r], P) if left[r] else _pages(start[r], P) for r in range(case['B'])]      # who left had as many
    need = [_pages(a + n, P) for a, n in zip(start, new)]
    width = max(need + held)
    total = sum(max(h, n) for h, n in zip(held, need)) + 7
    order = torch.randperm(total, generator=gen, device='cuda').tolist()
    rows, at = [], 0
    for h in held:
        rows.append(order[at:at + h] + [-1] * (width - h))
        at += h
    return dict(B=case['B'], page=P, width=width, total=total, table=_int32(rows), held=_int32(held),
                free=_int32(order[at:] + [-1] * at), free_count=_int32([total - at]), start=_int32(start), new=_int32(new),
                left=torch.tensor(left, device='cuda'), tokens=sum(new))


_INPUTS = {'matmul': _weights, 'grad': _weights, 'attend': _attend_inputs, 'write': _write_inputs, 'tables': _tables_inputs}


def prepare(case, seed):
    s = _INPUTS[case['kind']](case, _generator(seed))
    s['kind'] = case['kind']
    if case['kind'] == 'grad':
        s['x'].requires_grad_()
    if own:
        import jax_gptq_b200 as G
        if case['kind'] in ('matmul', 'grad'):
            s['qm'] = G.QuantizedMatrix(s['packed'], s['zero'], s['scale'], group_size=s['group'])
        elif case['kind'] == 'tables':
            s['pages'] = G.PageTable(s['B'], s['width'], s['total'], s['page'])
            for name in ('held', 'free', 'free_count'):
                getattr(s['pages'], name).copy_(s[name])
            s['pages'].block_table.copy_(s['table'])
        else:
            s['cache'] = G.KVCache(s['k'].shape[0], s['k'].shape[1], s['dim'], s['page'])
            for name in ('k', 'v', 'k_scale', 'v_scale'):
                getattr(s['cache'], name).copy_(s[name])
                s[name] = getattr(s['cache'], name)
    return s


# --------------------------------------------------------------------------
# one pass
# --------------------------------------------------------------------------
def run(state):
    return (_OWN if own else _PLAIN)[state['kind']](state)


def _own_matmul(s):
    import jax_gptq_b200 as G
    return G.quantized_matmul(s['x'], s['qm'])


def _own_grad(s):
    import jax_gptq_b200 as G
    y = G.quantized_matmul(s['x'], s['qm'])
    dx, = torch.autograd.grad(y, s['x'], s['dy'])
    return y.detach(), dx


def _own_attend(s):
    if s['most'] == 1:
        return s['cache'].attend(s['q'], s['table'], s['lengths_gpu'])
    return s['cache'].attend(s['q'], s['table'], s['lengths_gpu'], cu_seqlens=s['cu_gpu'], max_new=s['most'])


def _own_write(s):
    c = s['cache']
    c.write(s['k_new'], s['v_new'], s['slots'])
    k, v = c.read(s['pages'], s['k_new'].dtype)
    return k, v, c.k_scale, c.v_scale


def _own_tables(s):
    p = s['pages']
    step = p.reserve(s['start'], s['new'], s['tokens'], finished=s['left'])
    return step.slots, step.positions, step.cu_seqlens, step.lengths, p.block_table, p.held, p.free_count


_OWN = dict(matmul=_own_matmul, grad=_own_grad, attend=_own_attend, write=_own_write, tables=_own_tables)


def _dense(s, dtype):
    packed, g = s['packed'], s['group']
    K, N = 2 * packed.shape[0], packed.shape[1]
    codes = torch.stack((packed & 15, packed >> 4), 1).reshape(K, N).to(dtype)
    group = torch.arange(K, device='cuda') // g
    return (codes - s['zero'].to(dtype)[group]) * s['scale'].to(dtype)[group]


def _plain_matmul(s):
    return (s['x'].float() @ _dense(s, torch.float32)).to(s['x'].dtype)


def _plain_grad(s):
    w = _dense(s, torch.float32)
    x = s['x'].detach()
    return (x.float() @ w).to(x.dtype), (s['dy'].float() @ w.T).to(x.dtype)


def _values(s, pages):
    """Keys and values of some pages in fp32, [pages, heads, page, dim]."""
    k = (s['k'][pages].float() - 128) * s['k_scale'][pages][:, :, None, None]
    v = (s['v'][pages].float() - 128) * s['v_scale'][pages][:, :, None, None, None]
    v = v.transpose(3, 4).reshape(k.shape)
    return k[..., :s['dim']], v[..., :s['dim']]


def _plain_attend(s):
    q, out, at = s['q'], torch.empty_like(s['q']), 0
    Hq, D = q.shape[1:]
    for r, (L, n) in enumerate(zip(s['lengths'], s['new'])):
        k, v = _values(s, s['table'][r, :_pages(L, s['page'])].long())
        H = k.shape[1]
        k, v = (t.transpose(0, 1).reshape(H, 1, -1, D)[:, :, :L] for t in (k, v))
        qr = q[at:at + n].float().transpose(0, 1).reshape(H, Hq // H, n, D)
        score = (qr @ k.transpose(2, 3)) * D ** -0.5
        if n > 1:
            seen = torch.arange(L, device='cuda')[None] <= torch.arange(L - n, L, device='cuda')[:, None]
            score = torch.where(seen, score, -math.inf)
        p = torch.exp(score - score.amax(-1, keepdim=True))
        o = (p @ v) / p.sum(-1, keepdim=True)
        out[at:at + n] = o.reshape(Hq, n, D).transpose(0, 1).to(q.dtype)
        at += n
    return out


def _plain_write_one(new, codes, scale, slots, page, values):
    """`codes` viewed as [pages, heads, page, width] (keys) or the values' layout; both are updated in place."""
    pages, heads = scale.shape
    at, offset = slots // page, slots % page
    x = new.float()
    top = torch.zeros_like(scale).scatter_reduce(0, at[:, None].expand(-1, heads), x.abs().amax(2), 'amax')
    need = top / torch.full_like(top, 127.0)
    fresh = torch.zeros(pages, dtype=torch.bool, device='cuda')
    fresh[at[offset == 0]] = True
    touched = torch.zeros_like(fresh)
    touched[at] = True
    fresh = fresh[:, None] | (scale == 0)
    m, e = torch.frexp(need / scale)
    shift = torch.where(m == 0.5, e - 1, e)                               # ceil(log2), but for the quotient's rounding
    shift = shift + (torch.ldexp(scale, shift) < need).int() - (torch.ldexp(scale, shift - 1) >= need).int()
    shift = torch.where(touched[:, None] & ~fresh, shift.clamp(min=0), 0)
    scale.copy_(torch.where(touched[:, None], torch.where(fresh, need, torch.ldexp(scale, shift)), scale))
    tail = (slice(None), slice(None)) + (None,) * (codes.dim() - 2)
    codes.copy_(torch.ldexp(codes.float() - 128, -shift[tail]).round() + 128)
    row = torch.where(scale > 0, scale, 1.0)[at][:, :, None]
    c = ((x / row).round().clamp(-127, 127) + 128).to(torch.uint8)
    D = x.shape[2]
    if values:
        codes[at, :, offset // 64, :D, offset % 64] = c
    else:
        codes[at, :, offset, :D] = c


def _plain_write(s):
    _plain_write_one(s['k_new'], s['k'], s['k_scale'], s['slots'], s['page'], False)
    _plain_write_one(s['v_new'], s['v'], s['v_scale'], s['slots'], s['page'], True)
    k, v = _values(s, s['pages'])
    return k.to(s['k_new'].dtype), v.to(s['k_new'].dtype), s['k_scale'], s['v_scale']


def _plain_tables(s):
    B, P, W = s['B'], s['page'], s['width']
    table, held, free, count = s['table'], s['held'].long(), s['free'], s['free_count'].long()
    column = torch.arange(W, device='cuda')
    # pages of those who left: the first page of the first of them ends up on top of the stack
    back = s['left'][:, None] & (column[None] < held[:, None])
    freed = table[back]
    free[count + torch.arange(freed.numel(), device='cuda').flip(0)] = freed
    count = count + freed.numel()
    table[back] = -1
    held = torch.where(s['left'], 0, held)
    need = torch.maximum((s['start'].long() + s['new'] + P - 1) // P, held)
    taken = (column[None] >= held[:, None]) & (column[None] < need[:, None])
    index = torch.cumsum(taken.reshape(-1), 0).reshape(B, W) - 1
    table[taken] = free[count - 1 - index[taken]]
    s['held'].copy_(need)
    s['free_count'].copy_(count - taken.sum())
    cu = torch.zeros(B + 1, dtype=torch.int32, device='cuda')
    cu[1:] = torch.cumsum(s['new'], 0)
    request = torch.repeat_interleave(torch.arange(B, device='cuda'), s['new'], output_size=s['tokens'])
    position = s['start'][request] + torch.arange(s['tokens'], device='cuda') - cu[request]
    slots = table[request, position // P].long() * P + position % P
    return slots, position.int(), cu, s['start'] + s['new'], table, s['held'], s['free_count']


_PLAIN = dict(matmul=_plain_matmul, grad=_plain_grad, attend=_plain_attend, write=_plain_write, tables=_plain_tables)


# --------------------------------------------------------------------------
# what a pass cannot do without
# --------------------------------------------------------------------------
def work(case):
    kind = case['kind']
    if kind in ('matmul', 'grad'):
        M, K, N, b = case['M'], case['K'], case['N'], _BYTES[case['x']]
        groups = (K + case['group'] - 1) // case['group']
        by, fl = K * N / 2 + 2 * groups * N * _BYTES[case['zs']] + M * (K + N) * b, 2.0 * M * K * N
        return {'bytes': by + M * (K + N) * b, 'flops': 2 * fl} if kind == 'grad' else {'bytes': by, 'flops': fl}
    if kind == 'attend':
        lengths, new = _sequences(case)
        pairs = sum(n * L - n * (n - 1) // 2 for L, n in zip(lengths, new))
        by = sum(lengths) * case['kv_heads'] * case['dim'] * 2 + 2 * sum(new) * case['heads'] * case['dim'] * _BYTES[case['x']]
        return {'bytes': by, 'flops': 4.0 * pairs * case['heads'] * case['dim']}
    if kind == 'write':
        start, new = _writes(case)
        values, b = case['kv_heads'] * case['dim'], _BYTES[case['x']]
        held = sum(_pages(a + n, case['page']) for a, n in zip(start, new)) * case['page']
        return {'bytes': 2 * values * (sum(new) * (b + 1) + held * (1 + b)), 'flops': 2.0 * values * (sum(new) + held)}
    start, new, left = _requests(case)
    held = sum(_pages(a + n, case['page']) for a, n in zip(start, new))
    return {'bytes': 12 * sum(new) + 4 * held + 24 * case['B'], 'flops': 4.0 * sum(new)}


# --------------------------------------------------------------------------
# the same outputs in 64 bits
# --------------------------------------------------------------------------
def exact(case, seed):
    gen = _generator(seed)
    return _EXACT[case['kind']](_INPUTS[case['kind']](case, gen))


def _exact_matmul(s):
    x, packed = s['x'].double(), s['packed']
    w = torch.empty((2 * packed.shape[0], packed.shape[1]), dtype=torch.float64, device='cuda')
    w[0::2], w[1::2] = packed & 15, packed >> 4
    for i, (sc, z) in enumerate(zip(s['scale'].double(), s['zero'].double())):
        w[i * s['group']:(i + 1) * s['group']].sub_(z).mul_(sc)
    return (x @ w, s['dy'].double() @ w.T) if 'dy' in s else x @ w


def _exact_attend(s):
    out, at, P, D = [], 0, s['page'], s['dim']
    for r, (L, n) in enumerate(zip(s['lengths'], s['new'])):
        pages = s['rows'][r]
        H = s['k'].shape[1]
        rows = []
        for h in range(H):
            k = torch.cat([(s['k'][p, h, :, :D].double() - 128) * s['k_scale'][p, h].double() for p in pages])[:L]
            v = torch.cat([(s['v'][p, h].transpose(1, 2).reshape(P, -1)[:, :D].double() - 128) * s['v_scale'][p, h].double() for p in pages])[:L]
            per = s['q'].shape[1] // H
            q = s['q'][at:at + n, h * per:(h + 1) * per].double()
            score = torch.einsum('nhd,ld->nhl', q, k) / math.sqrt(D)
            late = torch.arange(L, device='cuda') > torch.arange(L - n, L, device='cuda')[:, None]
            score.masked_fill_(late[:, None], -math.inf)
            rows.append(torch.einsum('nhl,ld->nhd', torch.softmax(score, -1), v))
        out.append(torch.cat(rows, 1))
        at += n
    return torch.cat(out)


def _exact_write_one(new, codes, scale, slots, page):
    """Page by page.  The scale and the quotient are fp32 by definition; a 64-bit quotient rounded to 32 bits is that."""
    value = codes.double() - 128
    i = 0
    while i < len(slots):
        j = i + 1
        while j < len(slots) and slots[j] // page == slots[i] // page:
            j += 1
        p, o = slots[i] // page, slots[i] % page
        x = new[i:j].double().transpose(0, 1)                               # heads, rows, dim
        need = (x.abs().amax((1, 2)) / 127).float().double()
        old = scale[p].double()
        grown = old.clone()
        for h in range(len(grown)) if o else ():
            while 0 < grown[h] < need[h]:
                grown[h] *= 2
        begins = (old == 0) | (o == 0)
        scale[p] = torch.where(begins, need, grown).float()
        factor = torch.where(begins, torch.ones_like(old), old / torch.where(begins, 1.0, grown))
        value[p] = torch.round(value[p] * factor[:, None, None])
        by = torch.where(scale[p] > 0, scale[p], 1.0).double()[:, None, None]
        value[p, :, o:o + j - i, :x.shape[2]] = (x / by).float().double().round().clamp(-127, 127)
        i = j
    return value * scale.double()[:, :, None, None]


def _exact_write(s):
    if len(s['slots_host']) // s['page'] + s['pages'].numel() > 1500:
        return None
    D = s['dim']
    scales = s['k_scale'].clone(), s['v_scale'].clone()
    rows = s['v'].transpose(3, 4).reshape(s['k'].shape)
    k = _exact_write_one(s['k_new'], s['k'], scales[0], s['slots_host'], s['page'])[..., :D]
    v = _exact_write_one(s['v_new'], rows, scales[1], s['slots_host'], s['page'])[..., :D]
    return k, v, scales[0].double(), scales[1].double()


def _exact_tables(s):
    table, held, stack = s['table'].tolist(), s['held'].tolist(), s['free'].tolist()[:int(s['free_count'])]
    start, new, left, P = s['start'].tolist(), s['new'].tolist(), s['left'].tolist(), s['page']
    for r in reversed(range(len(held))):
        if left[r]:
            for j in reversed(range(held[r])):
                stack.append(table[r][j])
                table[r][j] = -1
            held[r] = 0
    slots, positions, cu = [], [], [0]
    for r in range(len(held)):
        while held[r] * P < start[r] + new[r]:
            table[r][held[r]] = stack.pop()
            held[r] += 1
        for p in range(start[r], start[r] + new[r]):
            positions.append(p)
            slots.append(table[r][p // P] * P + p % P)
        cu.append(len(slots))
    return (torch.tensor(slots, device='cuda'), _int32(positions), _int32(cu), _int32([a + n for a, n in zip(start, new)]),
            _int32(table), _int32(held), _int32([len(stack)]))


_EXACT = dict(matmul=_exact_matmul, grad=_exact_matmul, attend=_exact_attend, write=_exact_write, tables=_exact_tables)
