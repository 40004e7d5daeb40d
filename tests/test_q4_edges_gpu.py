"""Corners of the 4-bit cache's operators on the GPU: many sequences, keys shared by blocks, long sums, wide scales, rows of NaN, repeated streams, far offsets."""
import ctypes

import numpy as np
import pytest

import q4_ref as ref
from deepj_b200 import _lib
from deepj_b200 import compute_graph as cg
from test_q4_cache_gpu import FILL, dev, rows, run_attention, tables  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def no_wait_ran_out(dev):  # noqa: F811
    yield
    stats = (ctypes.c_int64 * 8)()
    _lib.check(dev.rt.lib.deepj_cuda_stats(stats, 8))
    assert stats[5] == 0


class Attention:
    """One op 87 or 88 over caches and rows of the test's making."""

    def __init__(self, dev, K, V, qkv, lens, new, packed, R, window=0):  # noqa: F811
        B, G, S, hd = K.shape
        self.dev, self.H, self.hd, self.shape, self.window = dev, G * R, hd, K.shape, window
        self.lens, self.starts = np.asarray(lens, np.float32), np.concatenate(([0], np.cumsum(new)))
        self.M = int(self.starts[-1])
        self.cos, self.sin = tables(S + 1, hd)
        self.K, self.V, self.qkv = ref.stored(K), ref.stored(V), qkv
        kv = dev.cache(1, B, G, S, hd)
        dev.store(kv, 0, K, V)
        self.x = dev.buf(qkv)
        self.out = dev.buf(np.full(max(1, self.M * self.H * hd), FILL))
        self.acc = np.random.default_rng(1).random((B, G, S)).astype(np.float32)
        a, self.ao = (dev.buf(self.acc), dev.buf(np.full(self.acc.size, FILL))) if window else (-1, -1)
        where = [self.x, 0, self.H * hd, (self.H + G) * hd, qkv.shape[1], kv, 0]
        rest = [dev.buf(self.lens), dev.buf(self.lens), dev.buf(self.cos), dev.buf(self.sin), S + 1, self.out, 0, self.H * hd, B, self.H]
        self.words = ([cg.OP_ATTN_PACKED_Q4] + where + [dev.buf(self.starts)] + rest + [self.M, a, self.ao, window] if packed
                      else [cg.OP_ATTN_DECODE_Q4] + where + rest + [a, self.ao])

    def run(self):
        self.dev.flush(*self.words)
        return self.dev.get(self.out, (self.M, self.H * self.hd))

    def want(self):
        return ref.attend(self.K.copy(), self.V.copy(), self.qkv, self.starts, self.lens, self.lens, self.cos, self.sin, self.H, self.window, self.acc if self.window else None)

    def check(self):
        want, tol, weights, wtol = self.want()
        got = self.run()
        err = np.abs(got - want)
        assert np.all(err <= tol), (float((err / tol).max()), np.argwhere(err > tol)[:5].tolist())
        if self.window:
            got, written = self.dev.get(self.ao, self.shape[:3]), ~np.isnan(weights)
            err = np.abs(np.where(written, got - np.where(written, weights, 0.0), 0.0))
            assert np.all(err <= wtol) and np.all(got[~written] == FILL)


def drawn(rng, B, G, R, S, hd, M):
    return rows(rng, B, G, S, hd), rows(rng, B, G, S, hd), rows(rng, M, (G * R + 2 * G) * hd)


def test_more_sequences_than_a_warp_has_lanes(dev):  # noqa: F811
    rng = np.random.default_rng(1)
    new = [int(n) for n in rng.integers(0, 9, 71)]
    run_attention(dev, rng, 32, 2, 2, 60, [int(n) for n in rng.integers(0, 60, 71)], new, 3, packed=True)
    run_attention(dev, rng, 32, 1, 1, 400, [int(n) for n in rng.integers(-1, 401, 71)], [1] * 71, 1, packed=False)


@pytest.mark.parametrize("hd,G,R,S,lens,new", [
    (64, 2, 1, 9000, [8000], [40]),                                  # blocks of a cluster with more than 16 tiles of keys each
    (128, 1, 4, 5000, [4300, 70], [5, 3]),
    (32, 3, 2, 2500, [2300, 0, 1100], [70, 300, 1]),                 # some tiles of queries shared, some not
    (128, 2, 1, 1400, [1100], [130]),
])
def test_blocks_that_share_a_tile_of_queries(dev, hd, G, R, S, lens, new):  # noqa: F811
    run_attention(dev, np.random.default_rng(hd + S), hd, G, R, S, lens, new, 3, packed=True)


@pytest.mark.parametrize("G,n", [(2, 7000), (160, 2100)])
def test_maxima_that_grow_all_the_way(dev, G, n):  # noqa: F811
    """Keys that grow with their row: sums that have left tensor memory are multiplied again and again."""
    rng = np.random.default_rng(2)
    K, V, qkv = drawn(rng, 1, G, 1, n + 40, 32, 3)
    K *= np.linspace(0.02, 20.0, n + 40, dtype=np.float32)[:, None]
    Attention(dev, K, V, qkv, [n], [3], True, 1).check()


@pytest.mark.parametrize("G", [2, 160])
def test_values_of_one_sign_over_many_keys(dev, G):  # noqa: F811
    rng = np.random.default_rng(3)
    K, V, qkv = drawn(rng, 1, G, 1, 6010, 32, 2)
    V[:] = 7.0
    qkv[:, 2 * G * 32:] = 7.0
    Attention(dev, K, V, qkv, [6000], [2], True, 1).check()


@pytest.mark.parametrize("packed", [False, True])
@pytest.mark.parametrize("hd", [32, 64, 128])
def test_scales_that_leave_the_fp16_products(dev, hd, packed):  # noqa: F811
    rng = np.random.default_rng(hd)
    new = [60, 3] if packed else [1, 1]
    K, V, qkv = drawn(rng, 2, 2, 2, 300, hd, sum(new))
    K *= 8e3
    V *= 8e3
    qkv[:, :4 * hd] *= 1e-4
    qkv[:, 4 * hd:] *= 8e3
    Attention(dev, K, V, qkv, [230, 77], new, packed, 2, 1).check()


@pytest.mark.parametrize("value", [np.nan, np.inf, -np.inf])
@pytest.mark.parametrize("packed,G,S,lens,new", [(True, 2, 300, [40, 100], [150, 7]), (True, 1, 1500, [1300], [9]), (False, 2, 300, [40, 100, 7], [1, 1, 1]),
                                                 (False, 1, 5000, [4900, 3], [1, 1])])
def test_a_query_that_is_no_number_spoils_its_own_output(dev, packed, G, S, lens, new, value):  # noqa: F811
    rng = np.random.default_rng(4)
    K, V, qkv = drawn(rng, len(lens), G, 3, S, 64, sum(new))
    clean = Attention(dev, K, V, qkv, lens, new, packed, 3).run()
    spoilt = qkv.copy()
    spoilt[1, 64 + 5] = value                                        # row 1, head 1
    got = Attention(dev, K, V, spoilt, lens, new, packed, 3).run()
    assert np.all(np.isnan(got[1, 64:128]))
    got[1, 64:128] = clean[1, 64:128]
    assert np.array_equal(got, clean)


@pytest.mark.parametrize("packed", [False, True])
def test_new_rows_that_are_no_numbers_are_kept_as_the_format_says(dev, packed):  # noqa: F811
    rng = np.random.default_rng(5)
    new = [5, 40] if packed else [1, 1]
    K, V, qkv = drawn(rng, 2, 1, 1, 90, 64, sum(new))
    qkv[0, 64:70] = np.nan
    qkv[1, 128:131] = [np.nan, 3e30, -3e30]                          # a value beyond the largest scale: 7 · 2^13 of it is kept
    Attention(dev, K, V, qkv, [33, 7], new, packed, 1).check()


def test_weights_alone_where_there_are_no_tokens(dev):  # noqa: F811
    rng = np.random.default_rng(6)
    K, V, qkv = drawn(rng, 3, 2, 1, 50, 32, 0)
    a = Attention(dev, K, V, np.zeros((1, 6 * 32), np.float32), [0, 17, 50], [0, 0, 0], True, 1, 2)
    dev.flush(*a.words)
    got = dev.get(a.ao, (3, 2, 50))
    assert np.array_equal(got[1, :, :17], a.acc[1, :, :17]) and np.all(got[1, :, 17:] == FILL) and np.all(got[[0, 2]] == FILL)


def test_streams_that_share_the_workspace_repeat_their_bits(dev):  # noqa: F811
    """Eager, captured and replayed, in turn with each other: every operator that uses the workspace gives the same bits every time."""
    rng = np.random.default_rng(7)
    many = Attention(dev, *drawn(rng, 40, 4, 3, 2500, 64, 40)[:2], rows(rng, 40, 20 * 64), [int(n) for n in rng.integers(0, 2500, 40)], [1] * 40, False, 3, 1)
    few = Attention(dev, *drawn(rng, 1, 2, 1, 9000, 128, 90)[:2], rows(rng, 90, 6 * 128), [8000], [90], True, 1, 20)
    long = Attention(dev, *drawn(rng, 1, 80, 1, 2300, 32, 300)[:2], rows(rng, 300, 240 * 32), [2000], [300], True, 1)
    first = {}
    for turn in range(5):
        for a in (many, few, long):
            got = a.run().tobytes() + (dev.get(a.ao, a.shape[:3]).tobytes() if a.window else b"")
            assert first.setdefault(id(a), got) == got, turn
    # and all in one stream
    dev.flush(*many.words, *few.words, *long.words)
    for a in (many, few, long):
        got = dev.get(a.out, (a.M, a.H * a.hd)).tobytes() + (dev.get(a.ao, a.shape[:3]).tobytes() if a.window else b"")
        assert first[id(a)] == got


def test_rows_behind_four_gigabytes(dev):  # noqa: F811
    """The last sequence's rows lie more than 2^32 bytes into the layer.  All its rows but the last 40 are zeros: every one of them has weight exp(0)."""
    rng = np.random.default_rng(8)
    B, G, S, hd, n = 32, 16, 65536, 128, 65000
    kv = dev.cache(1, B, G, S, hd)
    at = np.full(B, -1.0)
    at[-1] = n - 40
    k, v = rows(rng, G, 40, hd), rows(rng, G, 40, hd)
    src = np.zeros((B, 40, 2, G, hd), np.float32)
    src[-1] = np.stack((k, v)).transpose(2, 0, 1, 3)
    dev.flush(cg.OP_KV_STORE_Q4, dev.buf(src), 0, G * hd, 2 * G * hd, kv, 0, dev.buf(at), B, 40)
    cos, sin = tables(S, hd)
    lens = np.full(B, -1.0, np.float32)
    lens[-1] = n
    k, v = ref.stored(k).astype(np.float64), ref.stored(v).astype(np.float64)
    for packed in (False, True):
        M = 3 if packed else B
        qkv = rows(rng, M, 3 * G * hd)
        starts = np.zeros(B + 1)
        starts[-1] = M
        out = dev.buf(np.full(M * G * hd, FILL))
        tail = [dev.buf(lens), dev.buf(lens), dev.buf(cos), dev.buf(sin), S, out, 0, G * hd, B, G]
        head = [dev.buf(qkv), 0, G * hd, 2 * G * hd, 3 * G * hd, kv, 0]
        dev.flush(*([cg.OP_ATTN_PACKED_Q4] + head + [dev.buf(starts)] + tail + [M, -1, -1, 0] if packed else [cg.OP_ATTN_DECODE_Q4] + head + tail + [-1, -1]))
        got = dev.get(out, (M, G, hd))
        x = qkv.reshape(M, 3, G, hd)[M - 3:] if packed else qkv.reshape(M, 3, G, hd)[-1:]
        assert packed or np.all(got[:-1] == FILL)
        got = got[-len(x):]
        c, s = cos[n:n + len(x), None], sin[n:n + len(x), None]
        q = ref.rotate64(x[:, 0], c, s)
        nk, nv = ref.stored(ref.rotate32(x[:, 1], c, s)).astype(np.float64), ref.stored(x[:, 2]).astype(np.float64)
        for t in range(len(x)):
            for g in (0, G - 1):
                kk, vv = np.concatenate((k[g], nk[:t + 1, g])), np.concatenate((v[g], nv[:t + 1, g]))
                sc = kk @ q[t, g] / np.sqrt(hd)
                A = (np.abs(kk) @ np.abs(q[t, g]) / np.sqrt(hd)).max()
                p = np.exp(sc)
                want = p @ vv / (p.sum() + n - 40)
                # as in q4_ref.attend, of the 43 values that are not zero: their weights add up to p.sum() / (p.sum() + n - 40)
                tol = (2 * 2.0 ** -21 * A + 2.0 ** -20) * np.abs(vv).max() * p.sum() / (p.sum() + n - 40)
                assert np.abs(got[t, g] - want).max() <= tol


@pytest.mark.parametrize("place", ["same", "other"])
def test_eviction_of_many_sequences(dev, place):  # noqa: F811
    rng = np.random.default_rng(9)
    B, G, S, hd, budget, recent = 300, 3, 70, 32, 33, 4
    K, V = rows(rng, B, G, S, hd), rows(rng, B, G, S, hd)
    w = (rng.integers(0, 6, (B, G, S)) / 4.0).astype(np.float32)      # many ties
    n = rng.integers(-2, S + 3, B)
    kv = dev.cache(2, B, G, S, hd)
    dst = kv if place == "same" else dev.cache(2, B, G, budget, hd)
    dev.store(kv, 1, K, V)
    acc, lens = dev.buf(w), dev.buf(n)
    size = S if place == "same" else budget
    ao, lo = (acc if place == "same" else dev.buf(np.full(B * G * size, FILL))), dev.buf(np.zeros(B))
    dev.flush(cg.OP_KV_EVICT_Q4, kv, dst, 1, lens, acc, budget, recent, B, ao, lo, -1)
    gk, gv = dev.load(dst, 1, B, G, size, hd, end=lo)
    got, left = dev.get(ao, (B, G, size)), dev.get(lo, (B,))
    sk, sv = ref.stored(K), ref.stored(V)
    for b in range(B):
        rows_of = min(max(int(n[b]), 0), S)
        assert left[b] == min(rows_of, budget)
        for g in range(G):
            stay = ref.evict(w[b, g], rows_of, budget, recent)
            assert np.array_equal(gk[b, g, :len(stay)], sk[b, g, stay]) and np.array_equal(gv[b, g, :len(stay)], sv[b, g, stay])
            assert np.array_equal(got[b, g, :len(stay)], w[b, g, stay])


@pytest.mark.parametrize("layers,B,G,S,hd,message", [
    (1, 65536, 1, 32, 32, "too many"),
    (1, 1, 32769, 32, 32, "too many"),
    (1, 1, 1 << 30, 32, 128, "too many"),
    (1 << 30, 65535, 8192, 1 << 24, 128, "larger than any memory"),
    ((1 << 31) - 1, 1, 1, (1 << 24) - 1, 32, "larger than any memory"),
])
def test_sizes_that_no_cache_has_are_refused(dev, layers, B, G, S, hd, message):  # noqa: F811
    with pytest.raises(RuntimeError, match=message):
        dev.cache(layers, B, G, S, hd)


@pytest.mark.parametrize("op", [cg.OP_ATTN_DECODE_Q4, cg.OP_ATTN_PACKED_Q4])
def test_an_output_among_the_rows_is_refused(dev, op):  # noqa: F811
    kv = dev.cache(1, 1, 1, 32, 32)
    x, one, t = dev.buf(np.zeros(4 * 96)), dev.buf(np.zeros(2)), dev.buf(np.zeros(32 * 16))
    head = [x, 0, 32, 64, 96, kv, 0] + ([one] if op == cg.OP_ATTN_PACKED_Q4 else [])
    tail = [one, one, t, t, 32, x, 0, 32, 1, 1] + ([1, -1, -1, 0] if op == cg.OP_ATTN_PACKED_Q4 else [-1, -1])
    with pytest.raises(RuntimeError, match="another buffer"):
        dev.flush(op, *head, *tail)


@pytest.mark.parametrize("packed,hd,G,R,S,lens,new", [(True, 64, 2, 8, 700, [650, 0], [50, 300]), (True, 128, 8, 4, 400, [0, 100, 0], [300, 260, 129]),
                                                      (True, 32, 3, 2, 900, [800], [60]), (False, 64, 6, 4, 900, [800, 3, 400], [1, 1, 1])])
def test_every_repeat_gives_the_same_bits(dev, packed, hd, G, R, S, lens, new):  # noqa: F811
    """Rows that are read while the copy of the next ones comes over them would show as an output that changes."""
    rng = np.random.default_rng(11)
    a = Attention(dev, *drawn(rng, len(lens), G, R, S, hd, sum(new)), lens, new, packed, R)
    a.check()
    first = a.run()
    for _ in range(40):
        assert np.array_equal(a.run(), first)


@pytest.mark.parametrize("packed,G,R,S,lens,new,window", [(True, 2, 1, 300, [0, 40], [33, 130], 8), (True, 8, 4, 600, [0, 100, 7], [200, 260, 129], 0), (True, 1, 2, 3000, [2500, 0], [40, 9], 20),
                                                          (False, 4, 2, 600, [500, 3, 77], [1, 1, 1], 1)])
def test_inputs_that_change_right_before_the_op(dev, packed, G, R, S, lens, new, window):  # noqa: F811
    """Rows, tables, lengths, positions, starts and weights of two problems are copied in turn into one set of buffers by the ops before: a block that starts
    before the kernel in front of it has ended has to see all of them."""
    rng = np.random.default_rng(12)
    hd, H, B, M = 64, G * R, len(lens), sum(new)
    width, parts = (H + 2 * G) * hd, []
    for turn in range(2):
        n = np.asarray(lens, np.float32) if turn == 0 else np.maximum(np.asarray(lens, np.float32) - 3, 0)
        cos, sin = tables(S + 50, hd)
        if turn:
            cos, sin = np.ascontiguousarray(cos[::-1]), np.ascontiguousarray(sin[::-1])
        order = new if turn == 0 else new[::-1]
        parts.append([rows(rng, M, width), np.concatenate(([0], np.cumsum(order))).astype(np.float32), n, n + 5 * turn, cos, sin, rng.random((B, G, S)).astype(np.float32)])
    kv = dev.cache(1, B, G, S, hd)
    dev.store(kv, 0, rows(rng, B, G, S, hd), rows(rng, B, G, S, hd))
    shared = [dev.buf(np.zeros(a.size)) for a in parts[0]]
    held = [[dev.buf(a) for a in p] for p in parts]
    outs, weights = [dev.buf(np.zeros(M * H * hd)) for _ in parts], [dev.buf(np.zeros(B * G * S)) for _ in parts]

    def words(turn):
        x, starts, n, pos, cos, sin, acc = shared
        copies = [w for to, of, a in zip(shared, held[turn], parts[turn]) for w in (cg.OP_COPY, of, 0, to, 0, a.size)]
        tail = [n, pos, cos, sin, S + 50, outs[turn], 0, H * hd, B, H]
        seen = [acc, weights[turn]] if window else [-1, -1]
        where = [x, 0, H * hd, (H + G) * hd, width, kv, 0]
        return copies + ([cg.OP_ATTN_PACKED_Q4] + where + [starts] + tail + [M] + seen + [window] if packed else [cg.OP_ATTN_DECODE_Q4] + where + tail + seen)

    def results():
        return [dev.get(i, (M * H * hd,)).tobytes() for i in outs] + [dev.get(i, (B * G * S,)).tobytes() for i in weights]

    for _ in range(2):                                               # the rows that both write are the same again before each of them
        for turn in range(2):
            for w in np.split(np.arange(0, 7 * 6), 7):
                dev.flush(*[words(turn)[i] for i in w])              # a copy to a flush: nothing is close behind anything
            dev.flush(*words(turn)[42:])
    alone = results()
    for _ in range(12):
        dev.flush(*words(0), *words(1))
        assert results() == alone
