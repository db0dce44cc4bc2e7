"""Decode-step operators of several launches, called at once on the library's scratch."""
import threading

import numpy as np
import pytest

from tests._util import rng

pytestmark = pytest.mark.gpu


def _cg():
    import clove_compute_amd as cg
    return cg


def _cache(g, lens, Hk, D, P):
    """Random pages, each sequence's in a shuffled order."""
    import torch
    per = [-(-n // P) for n in lens]
    order = g.permutation(sum(per)).astype(np.int32)
    table, at = np.full((len(lens), max(per)), -1, np.int32), 0
    for b, n in enumerate(per):
        table[b, :n] = order[at:at + n]
        at += n
    k, v = (torch.from_numpy(g.standard_normal((sum(per), Hk, P, D)).astype(np.float16)).cuda() for _ in range(2))
    return k, v, torch.from_numpy(table).cuda(), torch.tensor(lens, dtype=torch.int32, device="cuda")


class Evict:
    """Selection, then the moves in a second launch."""

    def __init__(self, cg, seed, lens, budget, Hk, D, P):
        import torch
        g = rng("concurrent-evict", seed)
        self.cg, self.budget, self.L, self.B = cg, budget, max(lens), len(lens)
        self.k, self.v, self.table, self.lens = _cache(g, lens, Hk, D, P)
        self.kept = self.k.clone(), self.v.clone()
        self.cache = cg.KVCache(self.k, self.v)
        self.weights = torch.from_numpy(g.uniform(0, 1, (self.B, self.L)).astype(np.float32)).cuda()
        self.positions = torch.from_numpy(np.stack([g.permutation(self.L) for _ in lens]).astype(np.int32)).cuda()
        self.out = torch.empty_like(self.weights), torch.empty_like(self.positions), torch.empty_like(self.lens)

    def __call__(self):
        self.k.copy_(self.kept[0])
        self.v.copy_(self.kept[1])
        self.cg.cache_evict(self.cache, self.table, self.lens, self.weights, self.positions, *self.out, self.B, self.L, self.budget,
                            sinks=4, recent=16)
        return [x.clone() for x in (self.k, self.v, *self.out)]


class Attend:
    """Scores and statistics, then the weights added up in a second launch."""

    def __init__(self, cg, seed, lens, Hq, Hk, D, P):
        import torch
        g = rng("concurrent-attend", seed)
        self.cg, self.Hq, self.L, self.B = cg, Hq, max(lens), len(lens)
        k, v, self.table, self.lens = _cache(g, lens, Hk, D, P)
        self.cache = cg.KVCache(k, v)
        self.q = torch.from_numpy(g.standard_normal((self.B, Hq, D)).astype(np.float16)).cuda()
        self.out, self.weights = torch.empty_like(self.q), torch.zeros(self.B, self.L, device="cuda")

    def __call__(self):
        self.weights.zero_()
        self.cg.paged_attention(self.q, self.cache, self.table, self.lens, self.out, self.B, self.Hq, self.L, weights=self.weights)
        return [self.out.clone(), self.weights.clone()]


def _jobs(cg):
    return [Evict(cg, 0, [3000, 2500, 1800], 700, 4, 64, 16), Evict(cg, 1, [900, 4000], 1100, 2, 128, 32),
            Attend(cg, 0, [700, 30, 2000], 8, 2, 64, 16), Attend(cg, 1, [5000], 16, 2, 128, 64)]


def _at_once(jobs, rounds, stream_of):
    """What each job gave in each round, one thread a job."""
    import torch
    got, failed = [[] for _ in jobs], []
    gate = threading.Barrier(len(jobs), timeout=60)

    def work(i):
        try:
            with torch.cuda.stream(stream_of(i)):
                for _ in range(rounds):
                    gate.wait()
                    got[i].append(jobs[i]())
        except Exception as e:  # (a thread's exception does not end the test by itself)
            failed.append(e)
            gate.abort()

    threads = [threading.Thread(target=work, args=(i,)) for i in range(len(jobs))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    assert not failed, failed
    return got


def _same(jobs, got, want):
    import torch
    for i, runs in enumerate(got):
        for run in runs:
            assert all(torch.equal(x, y) for x, y in zip(run, want[i])), (i, type(jobs[i]).__name__)


def test_threads_on_one_stream():
    """Each call's launches follow one another: no other thread's come between them."""
    import torch
    cg = _cg()
    jobs = _jobs(cg)
    want = [job() for job in jobs]
    torch.cuda.synchronize()
    one = torch.cuda.current_stream()
    _same(jobs, _at_once(jobs, 40, lambda i: one), want)


def test_two_streams_on_library_scratch():
    """Each stream has buffers and counters of its own: calls that run beside each other
    on the device do not meet in them."""
    import torch
    cg = _cg()
    jobs = _jobs(cg)
    want = [job() for job in jobs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = [[] for _ in jobs]
    for _ in range(10):  # one thread, the streams in turn
        for i, job in enumerate(jobs):
            with torch.cuda.stream(streams[i % 2]):
                got[i].append(job())
    torch.cuda.synchronize()
    _same(jobs, got, want)
    _same(jobs, _at_once(jobs, 10, lambda i: streams[i % 2]), want)
