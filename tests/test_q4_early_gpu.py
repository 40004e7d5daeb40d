"""Token steps that ask for cached pages before they have waited for the kernels in front of them, which steps behind Q8 projections do."""
import numpy as np
import pytest

from deepj_b200 import _lib
from deepj_b200 import compute_graph as cg
from test_q4_cache_gpu import dev, rows, tables  # noqa: F401

pytestmark = pytest.mark.gpu


class Steps:
    """One layer of B sequences of G heads, and a projection whose outputs nobody needs."""

    def __init__(self, dev, B, G, S, hd, seed):  # noqa: F811
        self.dev, self.B, self.G, self.S, self.hd, self.rng = dev, B, G, S, hd, np.random.default_rng(seed)
        cos, sin = tables(S, hd)
        self.kv = dev.cache(1, B, G, S, hd)
        self.x, self.out, self.len, self.cos, self.sin = (dev.buf(a) for a in (rows(self.rng, B, 3 * G * hd), np.zeros(B * G * hd), np.zeros(B), cos, sin))
        w = dev.id()
        _lib.check(dev.rt.lib.deepj_cuda_q8_alloc(w, 1024, 1024))
        px, po = dev.buf(np.ones(1024)), dev.buf(np.zeros(1024))
        self.q8 = [cg.OP_Q8_LINEAR, px, 0, 1024, -1, 0, w, -1, -1, 0, 0, po, 0, 1024, 1]
        self.step = [cg.OP_ATTN_DECODE_Q4, self.x, 0, G * hd, 2 * G * hd, 3 * G * hd, self.kv, 0, self.len, self.len, self.cos, self.sin, S, self.out, 0, G * hd, B, G, -1, -1]

    def results(self):
        return self.dev.get(self.out, (self.B * self.G * self.hd,)).copy()

    def source(self):
        T = self.S - 1
        return self.dev.buf(rows(self.rng, self.B * T, 2 * self.G * self.hd)), T


@pytest.mark.parametrize("B,G,S,hd", [(1, 2, 4000, 128), (3, 4, 900, 64), (16, 2, 500, 32)])
def test_rows_written_right_before_are_read(dev, B, G, S, hd):  # noqa: F811
    """Two sets of rows are stored in turn, an op without work and a projection between them and the step."""
    t = Steps(dev, B, G, S, hd, 1)
    at = dev.buf(np.zeros(B))
    dev.rt.upload_buffer(t.len, np.full(B, S - 1, np.float32))
    stores = []
    for _ in range(2):
        src, T = t.source()
        stores.append([cg.OP_KV_STORE_Q4, src, 0, G * hd, 2 * G * hd, t.kv, 0, at, B, T])
    alone = []
    for s in stores:
        dev.flush(*s)
        dev.flush(*t.step)
        alone.append(t.results())
    assert not np.array_equal(*alone)
    nothing = [cg.OP_COPY, t.x, 0, t.out, 0, 0]
    outs = [dev.buf(np.zeros(B * G * hd)) for _ in range(2)]
    words = []
    for s, o in zip(stores, outs):
        words += s + nothing + t.q8 + t.step + [cg.OP_COPY, t.out, 0, o, 0, B * G * hd]
    for _ in range(12):
        dev.flush(*words)
        for o, want in zip(outs, alone):
            assert np.array_equal(dev.get(o, want.shape), want)


@pytest.mark.parametrize("B,G,S,hd,a,b", [(1, 2, 4000, 128, [3999], [100]), (3, 4, 900, 64, [10, 899, 300], [700, -1, 301]), (16, 2, 500, 32, range(16), range(480, 496))])
def test_lengths_written_right_before_are_followed(dev, B, G, S, hd, a, b):  # noqa: F811
    """The lengths change while pages of the old ones are on their way: those are dropped."""
    t = Steps(dev, B, G, S, hd, 2)
    src, T = t.source()
    dev.flush(cg.OP_KV_STORE_Q4, src, 0, G * hd, 2 * G * hd, t.kv, 0, dev.buf(np.zeros(B)), B, T)
    held, fresh = [dev.buf(np.asarray(list(n), np.float32)) for n in (a, b)], dev.buf(rows(t.rng, B, G * hd))
    set_to = [[cg.OP_COPY, fresh, 0, t.out, 0, B * G * hd, cg.OP_COPY, n, 0, t.len, 0, B] for n in held]
    alone = []
    for _ in range(2):                                               # the second time every row is the one that steps write
        alone = []
        for s in set_to:
            dev.flush(*s)
            dev.flush(*t.step)
            alone.append(t.results())
    outs = [dev.buf(np.zeros(B * G * hd)) for _ in range(2)]
    words = []
    for s, o in zip(set_to, outs):
        words += s + t.q8 + t.step + [cg.OP_COPY, t.out, 0, o, 0, B * G * hd]
    for _ in range(12):
        dev.flush(*words)
        for o, want in zip(outs, alone):
            assert np.array_equal(dev.get(o, want.shape), want)
