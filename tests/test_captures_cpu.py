"""Workspaces under capture, without a GPU: the library is a stand-in that looks at the workspace it is given."""
import ctypes
import importlib
import types

import pytest
import torch

from tests.test_abi import jlib  # noqa: F401  (fixture: the built library)
from tests.test_threads_cpu import attention, grouped, per_channel


@pytest.mark.parametrize('calls', [grouped, per_channel, attention])
def test_no_two_captures_share_a_workspace(jlib, monkeypatch, calls):  # noqa: F811
    """Eager calls, a capture, calls in between, a second capture on the same stream: each has a workspace of its own, whose
    tickets were cleared in the same capture, as the first graph's clearing is not part of the second."""
    gptq, op, cache = (importlib.import_module('jax_gptq_b200.' + n) for n in ('gptq', 'op', 'cache'))
    capture, made, seen = 0, [], []

    def buffer(n, dtype, device):
        made.append((capture, torch.full((n,), 171, dtype=dtype)))
        return made[-1][1]

    def call(ws, need):
        where = [(c, t) for c, t in made if t.data_ptr() == ws and t.numel() >= need]
        assert len(where) == 1 and where[0][0] == capture, 'a workspace of another capture'
        tickets = (ctypes.c_uint8 * min(need, 16384)).from_address(ws)
        assert not any(tickets)
        seen.append((capture, ws))
        return 0

    lib = types.SimpleNamespace(jgq_w4_group_matmul=lambda *a: call(*a[-3:-1]), jgq_w4_matmul=lambda *a: call(*a[-3:-1]),
                                jgq_kv_attend=lambda *a: call(*a[-3:-1]), jgq_capture_id=lambda stream: capture)
    for module in (op, cache):
        monkeypatch.setattr(module, 'lib', lib)
        monkeypatch.setattr(module, '_raw_stream', lambda dev: 7)
        monkeypatch.setattr(module, '_current_device', lambda: 0)
    fake = types.SimpleNamespace(zeros=lambda n, dtype, device: buffer(n, dtype, device).zero_(), empty=buffer, uint8=torch.uint8, device=torch.device,
                                 cuda=types.SimpleNamespace(current_device=lambda: 0), _C=types.SimpleNamespace(_cuda_getCurrentRawStream=lambda dev: 7))
    monkeypatch.setattr(gptq, 'torch', fake)
    monkeypatch.setattr(gptq, 'lib', lib)
    monkeypatch.setattr(gptq, '_dev', lambda: torch.device('cpu'))
    monkeypatch.setattr(gptq, '_capturing', lambda: capture != 0)
    for name in ('_ws_cache', '_scratch_ws', '_capture_ws'):
        monkeypatch.setattr(gptq, name, {})
    small, large = calls(op, cache, monkeypatch, None)
    for capture in (0, 11, 0, 12, 13, 0):
        for run in (small, large, small):
            run()
    assert all(len({at for c, at in seen if c == k}) <= 2 for k in (0, 11, 12, 13))          # grown once at most
