"""Paged cache of 8-bit keys and values for serving a quantized model: block tables and slot maps from request lengths
(`PageTable`), quantization of new tokens into their pages and attention over the pages (`KVCache`).

The reference stops at the packed weights and their product (op.py:11-81) and has no counterpart of this module.  One step
of a serving loop, for every layer between two `quantized_matmul`s:

    step = table.reserve(lengths, added, max_tokens)                    # once per step: pages, slots, positions
    cache.write(k, v, step.slots)                                       # per layer
    out = cache.attend(q, table.block_table, step.lengths, step.cu_seqlens, max_new=...)

Everything is enqueued on the current stream, nothing synchronises, and the arguments stay on the device, so a step can be
captured into a CUDA graph (its outputs and workspaces then belong to the graph).  All tensors are CUDA tensors of one
device; the call makes that device current for its launches.  Calls may come from several host threads: those on one stream run one
after the other.
"""
from __future__ import annotations

import math
from collections import namedtuple

import torch
from torch.autograd import forward_ad

from . import _lib
from ._lib import lib, check
from .gptq import _DT, _dev, _ptr, _scratch, _stream_locks

PAGE_SIZES = (64, 128, 256)

Step = namedtuple('Step', 'slots positions cu_seqlens lengths')
Step.__doc__ = """What `PageTable.reserve` returns: slots (int64) and positions (int32) of the added tokens, -1 and 0 behind the
last one; cu_seqlens (int32, requests + 1), the requests' first rows; lengths (int32) with the added tokens."""


def _cuda(t, name, device):
    if not isinstance(t, torch.Tensor) or not t.is_cuda:
        raise TypeError(f'{name} must be a CUDA tensor')
    if t.get_device() != device.index:
        raise ValueError(f'{name} is on {t.device}, not on {device}')
    return t


def _vector(t, name, dtype, n, device):
    if type(t) is torch.Tensor and t.dtype == dtype and t.get_device() == device.index and t.dim() == 1 and (n is None or t.numel() == n) and t.is_contiguous():
        return t
    t = _cuda(t, name, device)                       # what is wrong, or a copy
    if t.dtype != dtype:
        raise TypeError(f'{name} must be {dtype}, not {t.dtype}')
    if t.dim() != 1 or (n is not None and t.shape[0] != n):
        raise ValueError(f'{name} must have shape ({"n" if n is None else n},), not {tuple(t.shape)}')
    return t if t.is_contiguous() else t.contiguous()


def _device_of(device):
    d = _dev() if device is None else torch.device(device)
    if d.type != 'cuda':
        raise ValueError(f'the cache lives on a CUDA device, not on {d}')
    return torch.device('cuda', torch.cuda.current_device()) if d.index is None else d


_raw_stream, _current_device = torch._C._cuda_getCurrentRawStream, torch._C._cuda_getDevice


def _launch(index, call, *args):
    """`call` with the current stream of device `index`, on which it runs, behind its arguments."""
    stream = _raw_stream(index)
    with _stream_locks[index, stream]:
        if _current_device() == index:
            rc = call(*args, stream)
        else:
            with torch.cuda.device(index):
                rc = call(*args, stream)
    if rc:
        check(rc)


def stored_width(head_dim):
    """Channels of a stored row: the head dimension padded to 64, 128 or 256."""
    if not 1 <= head_dim <= 256:
        raise ValueError(f'head_dim must be in [1, 256], not {head_dim}')
    return 64 if head_dim <= 64 else 128 if head_dim <= 128 else 256


class PageTable:
    """Which pages the requests' tokens lie in: `block_table` (requests, max_pages) int32, -1 where there is none; `held`
    (requests,) pages per request; `free`, `free_count`: the stack of free pages (the next one is free[free_count - 1]).

    One table serves the caches of all layers.  `status` (int32) collects why steps were refused; `check()` reads it."""

    def __init__(self, requests, max_pages, num_pages, page_size=64, device=None):
        if requests < 1 or max_pages < 1 or num_pages < 1 or page_size < 1:
            raise ValueError('requests, max_pages, num_pages and page_size must be positive')
        self.device = d = _device_of(device)
        self.requests, self.max_pages, self.num_pages, self.page_size = int(requests), int(max_pages), int(num_pages), int(page_size)
        self.block_table = torch.full((self.requests, self.max_pages), -1, dtype=torch.int32, device=d)
        self.held = torch.zeros(self.requests, dtype=torch.int32, device=d)
        self.free = torch.arange(self.num_pages - 1, -1, -1, dtype=torch.int32, device=d)
        self.free_count = torch.full((1,), self.num_pages, dtype=torch.int32, device=d)
        self.status = torch.zeros(1, dtype=torch.int32, device=d)

    def reserve(self, lengths, added, max_tokens, finished=None):
        """Pages for `added[r]` tokens behind the `lengths[r]` that request r has (int32, on the device), and their slots.

        Requests with `finished[r]` (bool) first give back what they hold; their lengths are those of the request
        that takes the place.  Pages that a request already holds are kept, also when its length is set back.
        `max_tokens` bounds the sum of `added` and is the length of the slot map.  All or nothing: a step that does not fit
        (too few pages or columns, too many tokens, a negative length) takes no page, its slots are all -1, cu_seqlens
        is zero, the lengths stay, and `status` says why.  What finished requests held goes back to the stack all the
        same, before the step is weighed: the call may be made again, with the same `finished` or without."""
        d, n = self.device, self.requests
        lengths, added = _vector(lengths, 'lengths', torch.int32, n, d), _vector(added, 'added', torch.int32, n, d)
        if finished is not None:
            if isinstance(finished, torch.Tensor) and finished.dtype == torch.uint8:
                finished = finished.view(torch.bool) if finished.is_contiguous() else finished.bool()
            finished = _vector(finished, 'finished', torch.bool, n, d)
        max_tokens = int(max_tokens)
        if max_tokens < 0:
            raise ValueError('max_tokens must not be negative')
        slots = torch.empty(max_tokens, dtype=torch.int64, device=d)
        small = torch.empty(max_tokens + 2 * n + 1, dtype=torch.int32, device=d)
        positions, cu, out = small.split_with_sizes((max_tokens, n + 1, n))
        _launch(d.index, lib.jgq_kv_reserve, self.block_table.data_ptr(), self.block_table.stride(0), self.max_pages, self.held.data_ptr(),
                self.free.data_ptr(), self.free_count.data_ptr(), self.num_pages, self.page_size, lengths.data_ptr(), added.data_ptr(),
                _ptr(finished), n, slots.data_ptr(), positions.data_ptr(), max_tokens, cu.data_ptr(), out.data_ptr(), self.status.data_ptr())
        return Step(slots, positions, cu, out)

    def release(self, finished):
        """The pages of finished requests go back to the stack."""
        zero = torch.zeros(self.requests, dtype=torch.int32, device=self.device)
        self.reserve(zero, zero, 0, finished)

    def check(self):
        """Raises RuntimeError if a step was refused since the last check (waits for the device)."""
        st = int(self.status.item())
        if st:
            self.status.zero_()
            why = [text for bit, text in ((_lib.KV_NO_PAGES, 'too few free pages'), (_lib.KV_ROW_FULL, 'a request is longer than its row of the table'),
                                          (_lib.KV_TOO_MANY_TOKENS, 'more tokens than max_tokens'), (_lib.KV_BAD_LENGTH, 'a negative length'),
                                          (_lib.KV_BAD_TABLE, 'inconsistent table')) if st & bit]
            raise RuntimeError('a step was refused: ' + ', '.join(why))


class KVCache:
    """Keys and values of one layer as 8-bit codes, one fp32 scale per page and kv head.

    `k` (num_pages, kv_heads, page_size, width) and `v` (num_pages, kv_heads, page_size / 64, width, 64) hold code + 128 in
    bytes, `k_scale`, `v_scale` (num_pages, kv_heads) the scales; width is head_dim padded to 64, 128 or 256.  The value of a
    code is (byte - 128) * scale."""

    def __init__(self, num_pages, kv_heads, head_dim, page_size=64, device=None):
        if page_size not in PAGE_SIZES:
            raise ValueError(f'page_size must be one of {PAGE_SIZES} (scales are per page, values lie 64 tokens side by side), not {page_size}')
        if num_pages < 1 or kv_heads < 1:
            raise ValueError('num_pages and kv_heads must be positive')
        w = stored_width(head_dim)
        self.device = d = _device_of(device)
        self.num_pages, self.kv_heads, self.head_dim, self.page_size = int(num_pages), int(kv_heads), int(head_dim), int(page_size)
        self.k = torch.full((num_pages, kv_heads, page_size, w), 128, dtype=torch.uint8, device=d)
        self.v = torch.full((num_pages, kv_heads, page_size // 64, w, 64), 128, dtype=torch.uint8, device=d)
        self._ws_bytes = {}          # workspace bytes of `attend`, a function of the sizes and the device
        self.k_scale = torch.zeros((num_pages, kv_heads), dtype=torch.float32, device=d)
        self.v_scale = torch.zeros((num_pages, kv_heads), dtype=torch.float32, device=d)

    def _rows(self, t, name, heads):
        """(tensor with a contiguous last axis, its shape, its strides) of (tokens, heads, head_dim) rows."""
        if type(t) is not torch.Tensor or t.get_device() != self.device.index:
            t = _cuda(t, name, self.device)
        if t.dtype not in _DT:
            raise TypeError(f'{name} must be float32, float16 or bfloat16, not {t.dtype}')
        shape = t.shape
        if len(shape) != 3 or (heads is not None and shape[1] != heads) or shape[2] != self.head_dim:
            raise ValueError(f'{name} must have shape (tokens, {"heads" if heads is None else heads}, {self.head_dim}), not {tuple(shape)}')
        if t.requires_grad:
            if torch.is_grad_enabled():
                raise ValueError(f'{name} requires a gradient; the cache has none (detach it)')
            t = t.detach()
        if forward_ad._current_level >= 0 and forward_ad.unpack_dual(t).tangent is not None:
            raise ValueError(f'{name} has a tangent; the cache has none (detach it)')
        strides = t.stride()
        if strides[2] != 1 and shape[2] != 1:
            t = t.contiguous()
            strides = t.stride()
        return t, shape, strides

    def write(self, k, v, slots):
        """Quantizes row t of `k` and `v` (tokens, kv_heads, head_dim) into token slot `slots[t]` (int64; page * page_size +
        offset; negative or outside the cache: nowhere).

        The rows of one page must be consecutive rows whose slots follow one another without a gap, as `PageTable.reserve` gives
        them (runs of one page that lie apart in one call spoil each other's codes; two calls do not).  Where a
        page's first token is written its scale is set anew; later tokens that need more make it grow by a power of two,
        and the codes that are there are rounded to it.  NaN is stored as 0, infinities as the largest code."""
        k, shape, ks = self._rows(k, 'k', self.kv_heads)
        v, v_shape, vs = self._rows(v, 'v', self.kv_heads)
        if shape != v_shape or k.dtype != v.dtype:
            raise ValueError(f'k {tuple(shape)} {k.dtype} and v {tuple(v_shape)} {v.dtype} differ')
        tokens = shape[0]
        slots = _vector(slots, 'slots', torch.int64, tokens, self.device)
        _launch(self.device.index, lib.jgq_kv_write, k.data_ptr(), v.data_ptr(), _DT[k.dtype], ks[0], ks[1], vs[0], vs[1],
                slots.data_ptr(), tokens, self.k.data_ptr(), self.v.data_ptr(), self.k_scale.data_ptr(), self.v_scale.data_ptr(),
                self.num_pages, self.page_size, self.kv_heads, self.head_dim)

    def read(self, pages, dtype=torch.float32):
        """Keys and values of the pages `pages` (int64), each (len(pages), kv_heads, page_size, head_dim) in `dtype`; NaN
        where there is no such page."""
        if dtype not in _DT:
            raise TypeError(f'dtype must be float32, float16 or bfloat16, not {dtype}')
        pages = _vector(pages, 'pages', torch.int64, None, self.device)
        shape = (pages.shape[0], self.kv_heads, self.page_size, self.head_dim)
        k = torch.empty(shape, dtype=dtype, device=self.device)
        v = torch.empty_like(k)
        _launch(self.device.index, lib.jgq_kv_read, self.k.data_ptr(), self.v.data_ptr(), self.k_scale.data_ptr(), self.v_scale.data_ptr(),
                self.num_pages, self.page_size, self.kv_heads, self.head_dim, pages.data_ptr(), shape[0], k.data_ptr(), v.data_ptr(), _DT[dtype])
        return k, v

    def attend(self, q, block_table, lengths, cu_seqlens=None, max_new=None, scale=None, out=None, return_lse=False):
        """softmax(scale * q k^T) v over the cached tokens of every request; q (tokens, heads, head_dim), heads a multiple of
        kv_heads (query head h reads kv head h // (heads / kv_heads)).

        Request r has `lengths[r]` tokens, in the pages `block_table[r]`.  Without `cu_seqlens` row r of q is the last
        of them; with it (int32, requests + 1) rows cu_seqlens[r] .. cu_seqlens[r + 1] - 1 are the last ones, and each sees the
        tokens up to its own.  `max_new` is the largest number of rows of a request that is expected (default: all of q); it
        only steers the choice of kernel.  Rows that see nothing are zero.  Rows of no request (behind the
        last one, or in front of cu_seqlens[0]) are zero in a new result and left as they were in `out`.  A page number outside the cache makes its rows NaN (scales
        that are not finite spoil the rows that see their page, and no others).  `scale` defaults to
        head_dim ** -0.5.  With `return_lse` also the logarithm of the sum of exponentials, fp32 (tokens, heads), -inf in rows that
        see nothing and in those of no request."""
        q, shape, strides = self._rows(q, 'q', None)
        d, tokens, heads = self.device, shape[0], shape[1]
        if block_table.dim() != 2 or block_table.dtype != torch.int32:
            raise ValueError('block_table must be a 2-D int32 tensor')
        table = block_table if type(block_table) is torch.Tensor and block_table.get_device() == d.index else _cuda(block_table, 'block_table', d)
        n, width = table.shape
        pitch = table.stride()
        if pitch[1] != 1 and width > 1:
            table = table.contiguous()
            pitch = table.stride()
        if heads < 1 or heads % self.kv_heads:
            raise ValueError(f'{heads} query heads are no multiple of {self.kv_heads} kv heads')
        lengths = _vector(lengths, 'lengths', torch.int32, n, d)
        if cu_seqlens is None:
            if tokens != n:
                raise ValueError(f'{tokens} rows of q for {n} requests without cu_seqlens')
            most = 1
        else:
            cu_seqlens = _vector(cu_seqlens, 'cu_seqlens', torch.int32, n + 1, d)
            most = max(1, tokens if max_new is None else int(max_new))
        fresh = out is None
        if fresh:
            out = torch.empty_like(q) if q.is_contiguous() else q.new_empty(shape)
        else:
            _cuda(out, 'out', d)
            if out.shape != q.shape or out.dtype != q.dtype or not out.is_contiguous():
                raise ValueError(f'out must be a contiguous {q.dtype} tensor of shape {tuple(q.shape)}')
        lse = None
        if return_lse:                   # new in either case: KV_ZERO_REST, which sets the rows of no request, goes with a new result
            lse = torch.empty(shape[:2], dtype=torch.float32, device=d) if fresh else torch.full(shape[:2], -math.inf, dtype=torch.float32, device=d)
        index, code = d.index, _DT[q.dtype]
        args = (q.data_ptr(), code, strides[0], strides[1], out.data_ptr(), _ptr(lse), self.k.data_ptr(), self.v.data_ptr(), self.k_scale.data_ptr(),
                self.v_scale.data_ptr(), self.num_pages, self.page_size, table.data_ptr(), pitch[0], width, lengths.data_ptr(), _ptr(cu_seqlens),
                tokens, n, most, heads, self.kv_heads, self.head_dim, float(self.head_dim ** -0.5 if scale is None else scale),
                _lib.KV_ZERO_REST if fresh else 0)
        if _current_device() == index:
            self._attend(args, heads, most, code, index)
        else:
            with torch.cuda.device(index):
                self._attend(args, heads, most, code, index)
        return (out, lse) if return_lse else out

    def _attend(self, args, heads, most, code, index):
        need = self._ws_bytes.get((heads, most, code))
        if need is None:
            if len(self._ws_bytes) >= 1024:
                self._ws_bytes.clear()
            need = self._ws_bytes[heads, most, code] = lib.jgq_kv_attend_workspace_bytes(heads, self.kv_heads, self.head_dim, most, code)
        stream = _raw_stream(index)
        with _stream_locks[index, stream]:
            rc = lib.jgq_kv_attend(*args, _scratch(need, 'kv', index, stream), need, stream)
        if rc:
            check(rc)
