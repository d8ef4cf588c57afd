"""Two host threads on one stream, without a GPU: the library is a stand-in that looks at the workspace it is given."""
import threading
import types
import weakref

import pytest
import torch

from tests.test_abi import jlib  # noqa: F401  (fixture: the built library)


class StandIn:
    """A library call that, the first time, lets another thread try to get in, and then looks whether its workspace is still there."""

    def __init__(self):
        self.made, self.inside, self.met, self.alive = [], 0, False, []
        self.first_is_in, self.other_is_done = threading.Event(), threading.Event()

    def zeros(self, n, dtype, device):
        t = torch.zeros(n, dtype=dtype)
        self.made.append((weakref.ref(t), t.data_ptr()))
        return t

    def call(self, ws, need):
        self.met |= self.inside > 0
        self.inside += 1
        if not self.first_is_in.is_set():
            self.first_is_in.set()
            self.other_is_done.wait(1.0)
        self.alive.append(any(ref() is not None and at == ws and ref().numel() >= need for ref, at in self.made))
        self.inside -= 1
        return 0


def grouped(op, cache, monkeypatch, stand_in):
    monkeypatch.setattr(op, '_ws_bytes', {(0, 4, 16, 64, False, 32): 4 << 20, (0, 1, 16, 64, False, 32): 64})
    w, z, s = torch.zeros((32, 16), dtype=torch.uint8), torch.zeros((2, 16)), torch.ones((2, 16))

    def run(M):
        x, out = torch.zeros((M, 64)), torch.zeros((M, 16))
        op._enqueue_groups(x, w, z, s, out, M, 16, 64, 32, False, 0)
    return lambda: run(1), lambda: run(4)


def per_channel(op, cache, monkeypatch, stand_in):
    monkeypatch.setattr(op, '_ws_bytes', {(0, 4, 16, 64, False, None): 4 << 20, (0, 1, 16, 64, False, None): 64})
    w, z, s = torch.zeros((32, 16), dtype=torch.uint8), torch.zeros(16), torch.ones(16)
    return lambda: op._launch(torch.zeros((1, 64)), w, z, s, False), lambda: op._launch(torch.zeros((4, 64)), w, z, s, False)


def attention(op, cache, monkeypatch, stand_in):
    c = cache.KVCache.__new__(cache.KVCache)
    c._ws_bytes = {(8, 1, 0): 64, (8, 100, 0): 4 << 20}
    return lambda: c._attend((), 8, 1, 0, 0), lambda: c._attend((), 8, 100, 0, 0)


@pytest.mark.parametrize('calls', [grouped, per_channel, attention])
@pytest.mark.parametrize('small_first', [True, False])
def test_a_call_keeps_its_workspace_to_itself(jlib, monkeypatch, calls, small_first):  # noqa: F811
    """One needs a larger workspace than the other: what one of them is about to launch on is neither freed nor entered."""
    import importlib
    gptq, op, cache = (importlib.import_module('jax_gptq_b200.' + n) for n in ('gptq', 'op', 'cache'))
    stand_in = StandIn()
    lib = types.SimpleNamespace(jgq_w4_group_matmul=lambda *a: stand_in.call(*a[-3:-1]), jgq_w4_matmul=lambda *a: stand_in.call(*a[-3:-1]),
                                jgq_kv_attend=lambda *a: stand_in.call(*a[-3:-1]))
    for module in (op, cache):
        monkeypatch.setattr(module, 'lib', lib)
        monkeypatch.setattr(module, '_raw_stream', lambda dev: 7)
        monkeypatch.setattr(module, '_current_device', lambda: 0)
    fake = types.SimpleNamespace(zeros=stand_in.zeros, empty=stand_in.zeros, uint8=torch.uint8, device=torch.device,
                                 cuda=types.SimpleNamespace(current_device=lambda: 0), _C=types.SimpleNamespace(_cuda_getCurrentRawStream=lambda dev: 7))
    monkeypatch.setattr(gptq, 'torch', fake)
    monkeypatch.setattr(gptq, '_dev', lambda: torch.device('cpu'))
    monkeypatch.setattr(gptq, '_capturing', lambda: False)
    for name in ('_ws_cache', '_scratch_ws', '_capture_ws'):
        monkeypatch.setattr(gptq, name, {})
    first, second = calls(op, cache, monkeypatch, stand_in)
    if not small_first:
        first, second = second, first
    failed = []

    def guarded(call, before, after):
        try:
            before()
            call()
        except Exception as e:                                            # noqa: BLE001
            failed.append(e)
        after()
    threads = [threading.Thread(target=guarded, args=a) for a in ((first, lambda: None, lambda: None),
                                                                  (second, lambda: stand_in.first_is_in.wait(10), stand_in.other_is_done.set))]
    for t in threads:
        t.start()
    for t in threads:
        t.join(20)
    assert not failed and stand_in.alive == [True, True] and not stand_in.met
