"""Host threads that call the same operators on the same stream: each gets what it gets alone."""
import importlib
import threading

import pytest
import torch

from tests.test_gpu_cache import DT, filled, i32
from tests.test_gpu_group_matmul import matrix

pytestmark = pytest.mark.gpu


@pytest.fixture(scope='module')
def G():
    return importlib.import_module('jax_gptq_b200')


def at_once(G, calls, rounds):
    """Every list of calls in a thread of its own, starting without workspaces; results compared bit by bit."""
    want = [[c() for c in part] for part in calls]
    torch.cuda.synchronize()
    for cache in (G.gptq._scratch_ws, G.gptq._ws_cache):
        cache.clear()
    got, failed, gate = [[] for _ in calls], [], threading.Barrier(len(calls))

    def run(i):
        try:
            gate.wait(30)
            for _ in range(rounds):
                got[i].append([c() for c in calls[i]])
        except Exception as e:                                            # noqa: BLE001
            failed.append(e)
    threads = [threading.Thread(target=run, args=(i,)) for i in range(len(calls))]
    for t in threads:
        t.start()
    for t in threads:
        t.join(120)
    torch.cuda.synchronize()
    assert not failed
    for g, w in zip(got, want):
        assert len(g) == rounds and all(torch.equal(a, b) for part in g for a, b in zip(part, w))


@pytest.mark.parametrize('x', ['f16', 'bf16', 'f32'])
def test_products_of_two_threads(G, x):
    """Tables of one matrix are not multiplied with by the other's product; sizes that grow the workspace among small ones."""
    calls = []
    for seed, sizes in ((1, (1, 300, 40)), (2, (40, 3, 700))):
        qm, _, _ = matrix(G, 1024, 528, 64, seed=seed)
        per_channel = G.QuantizedMatrix(qm.int_weight, qm.zero[0], qm.scale[0])
        part = []
        for M in sizes:
            a, b = torch.randn((M, 1024), device='cuda').to(DT[x]), torch.randn((M, 528), device='cuda').to(DT[x])
            for m in (qm, per_channel):
                part += [lambda a=a, m=m: G.quantized_matmul(a, m), lambda b=b, m=m: G.quantized_matmul(b, m, transpose_b=True)]
        calls.append(part)
    at_once(G, calls, 30)


@pytest.mark.parametrize('x', ['bf16', 'f32'])
def test_attention_of_two_threads(G, x):
    calls = []
    for seed, news in ((1, (1, 300)), (2, (20, 80))):
        cache, table, gen = filled(G, [2000, 900], 2, 64, 64, seed)
        part = []
        for new in news:
            q = torch.randn((2 * new, 8, 64), generator=gen, device='cuda').to(DT[x])
            part.append(lambda q=q, new=new, cache=cache, table=table: cache.attend(q, table, i32([2000, 900]), i32([0, new, 2 * new]), new))
        calls.append(part)
    at_once(G, calls, 30)
