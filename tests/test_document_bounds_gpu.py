"""laya_op_document_bounds on sequences long enough to take its linear passes (above 4,096 rows), against NumPy."""
import numpy as np
import pytest

import attend_reference as A
from laya_cuda import _lib

pytestmark = pytest.mark.gpu


def torch():
    import torch as t
    return t


class Bounds:
    def __init__(self, gpu, lengths, mean, gap=2, seed=0):
        t, rng = torch(), np.random.default_rng(seed)
        self.lengths = np.array(lengths, np.int32)
        self.starts = (np.cumsum(self.lengths + gap) - self.lengths).astype(np.int32)
        self.rows = int(self.starts[-1] + self.lengths[-1] + gap)
        self.ids = np.full(self.rows, 7, np.int32)
        for s, n in zip(self.starts, self.lengths):
            # Few ids, which come again: the lowest and highest of the type, and those that mark an open run, among them.
            self.ids[s:s + n] = np.array([-1, 2 ** 31 - 1, -2 ** 31, 0, 5], np.int32)[np.cumsum(rng.random(n) < 1 / mean) % 5]
        self.d, self.s, self.n = (t.from_numpy(x).to(gpu) for x in (self.ids, self.starts, self.lengths))
        self.out = t.full((self.rows, 2), -9, dtype=t.int32, device=gpu)

    def run(self, max_length, rows=None, stream=None):
        at = lambda x: x.data_ptr()  # noqa: E731
        stream = stream or torch().cuda.current_stream()
        _lib.check(_lib.load().laya_op_document_bounds(at(self.d), at(self.s), at(self.n), len(self.starts), self.rows if rows is None else rows,
                                                       max_length, at(self.out), stream.cuda_stream))
        return self

    def check(self, lengths):
        torch().cuda.synchronize()
        want = np.full((self.rows, 2), -9, np.int32)
        for s, n in zip(self.starts, lengths):
            want[s:s + n] = A.document_bounds(self.ids[s:s + n])
        np.testing.assert_array_equal(self.out.cpu().numpy(), want)


MIXED = [1, 0, 64, 65, 5000, 63, 128, 2049, 70001, 131072, 65536, 65537, 9]


@pytest.mark.parametrize("mean", [1, 3, 64, 900, 40000, 10 ** 9])
@pytest.mark.parametrize("most", [131072, 70000, 4097])
def test_long_sequences(gpu, mean, most):
    """One row to two steps of the carrying pass; sequences longer than the call says are cut, and rows behind them left."""
    b = Bounds(gpu, MIXED, mean, seed=mean % 1000)
    b.run(most).check(np.minimum(MIXED, most))


def test_sequences_are_cut_to_the_array(gpu):
    b = Bounds(gpu, [100, 9000, 300], 50, seed=3)
    rows = int(b.starts[1]) + 6000
    b.s[2] = -4
    b.run(9000, rows).check([100, 6000, 0])


def test_one_document_of_16_million_rows(gpu):
    """Linear in the rows: about a millisecond.  Steps of 512 rows from every 64 of them would be 2^18 waves of 2^15 steps, which no
    second holds."""
    t = torch()
    b = Bounds(gpu, [1 << 24], 10 ** 12)
    b.d.fill_(3)
    b.run(1 << 24)
    t.cuda.synchronize()
    a, e = t.cuda.Event(enable_timing=True), t.cuda.Event(enable_timing=True)
    a.record()
    b.run(1 << 24)
    e.record()
    t.cuda.synchronize()
    assert a.elapsed_time(e) < 500
    s = int(b.starts[0])
    assert (b.out[s:s + (1 << 24), 0] == 0).all() and (b.out[s:s + (1 << 24), 1] == 1 << 24).all()
    assert (b.out[:s] == -9).all() and (b.out[s + (1 << 24):] == -9).all()


def test_replays_with_other_lengths_and_documents(gpu):
    t = torch()
    b = Bounds(gpu, [9000, 300, 70000], 700)
    graph = t.cuda.CUDAGraph()
    t.cuda.synchronize()
    with t.cuda.graph(graph):
        b.run(70000)
    rng = np.random.default_rng(5)
    for lengths, mean in (([9000, 300, 70000], 700), ([4, 0, 65000], 10 ** 9), ([8999, 299, 1], 3)):
        b.ids[:] = np.cumsum(rng.random(b.rows) < 1 / mean) % 3
        b.d.copy_(t.from_numpy(b.ids))
        b.n.copy_(t.from_numpy(np.array(lengths, np.int32)))
        b.out.fill_(-9)
        graph.replay()
        b.check(lengths)
