"""The 4-bit K/V cache on the GPU against 64 bits: rows in and out, a token step, packed prompts, eviction, and a run of them together."""
import ctypes

import numpy as np
import pytest

import q4_ref as ref
from deepj_b200 import _lib
from deepj_b200 import compute_graph as cg

pytestmark = pytest.mark.gpu
FILL = 12345.0


class Device:
    """Buffers and streams of one test."""
    _next = 1 << 27

    def __init__(self):
        self.rt = cg.CudaGpuRuntime()
        self.ids = []

    def id(self):
        Device._next += 1
        self.ids.append(Device._next)
        return Device._next

    def buf(self, data):
        a = np.ascontiguousarray(data, dtype=np.float32)
        i = self.id()
        self.rt.alloc_buffers([i], [a.size], 1)
        if a.size:
            self.rt.upload_buffer(i, a)
        return i

    def get(self, i, shape):
        out = np.empty(int(np.prod(shape)), dtype=np.float32)
        self.rt.download_buffer(i, out)
        return out.reshape(shape)

    def cache(self, layers, B, G, S, hd):
        i = self.id()
        _lib.check(self.rt.lib.deepj_cuda_kv_alloc_q4(i, layers, B, G, S, hd))
        return i

    def flush(self, *words):
        s = cg.stream(words)
        self.rt.flush_ops(s, s.size)

    def store(self, kv, layer, k, v, at=None):
        """k, v [B][G][T][hd] from row at[b] on."""
        B, G, T, hd = k.shape
        rows = np.concatenate((k.transpose(0, 2, 1, 3).reshape(B * T, G * hd), v.transpose(0, 2, 1, 3).reshape(B * T, G * hd)), 1)
        self.flush(cg.OP_KV_STORE_Q4, self.buf(rows), 0, G * hd, 2 * G * hd, kv, layer, self.buf(np.zeros(B) if at is None else at), B, T)

    def load(self, kv, layer, B, G, T, hd, at=-1, end=-1):
        k, v = self.buf(np.full(B * G * T * hd, FILL)), self.buf(np.full(B * G * T * hd, FILL))
        self.flush(cg.OP_KV_LOAD_Q4, kv, layer, at, end, T, k, v, B)
        return self.get(k, (B, G, T, hd)), self.get(v, (B, G, T, hd))

    def close(self):
        self.rt.release_buffers(self.ids, len(self.ids))


@pytest.fixture
def dev():
    d = Device()
    yield d
    d.close()


def rows(rng, *shape):
    return (rng.standard_normal(shape) * (1.0 + 3.0 * (rng.random(shape[-1]) < 0.1))).astype(np.float32)


def tables(n, hd):
    a = np.arange(n)[:, None] * 10000.0 ** (-np.arange(hd // 2) * 2.0 / hd)
    return np.cos(a).astype(np.float32), np.sin(a).astype(np.float32)


# ───────────── rows in and out ─────────────

@pytest.mark.parametrize("hd", [32, 64, 128])
@pytest.mark.parametrize("T", [1, 31, 32, 33, 100])
def test_rows_read_back_as_their_nearest_codes(dev, hd, T):
    rng = np.random.default_rng(hd + T)
    B, G, S = 2, 3, 100
    k, v = rows(rng, B, G, T, hd), rows(rng, B, G, T, hd)
    k[0, 0, 0, :32] = 0.0                                            # a block of zeros
    k[0, 1, 0, :5] = [np.nan, np.inf, -np.inf, 1e30, -3.0]           # saturates, NaN reads back as 0
    v[0, 0, 0, :32] = rng.standard_normal(32) * 1e-7                 # below the least scale
    v[1, 2, 0, :32] = rng.standard_normal(32) * 5e4                  # above the largest
    v[1, 1, 0] = np.arange(hd) % 15 - 7                              # every code
    kv = dev.cache(2, B, G, S, hd)
    dev.store(kv, 1, k, v)
    gk, gv = dev.load(kv, 1, B, G, T, hd)
    assert np.array_equal(gk, ref.stored(k)) and np.array_equal(gv, ref.stored(v))
    gk, gv = dev.load(kv, 0, B, G, T, hd)                            # the other layer was not touched
    assert not gk.any() and not gv.any()


def test_rows_go_where_they_are_sent_and_nowhere_else(dev):
    rng = np.random.default_rng(3)
    B, G, S, hd = 4, 2, 70, 64
    base_k, base_v = rows(rng, B, G, S, hd), rows(rng, B, G, S, hd)
    kv = dev.cache(1, B, G, S, hd)
    dev.store(kv, 0, base_k, base_v)
    k, v = rows(rng, B, G, 9, hd), rows(rng, B, G, 9, hd)
    at = np.array([0, 65, -1, 70], dtype=np.float32)                 # the second runs over the end, the last two are outside
    dev.store(kv, 0, k, v, at)
    want_k, want_v = ref.stored(base_k), ref.stored(base_v)
    want_k[0, :, :9], want_v[0, :, :9] = ref.stored(k)[0], ref.stored(v)[0]
    want_k[1, :, 65:], want_v[1, :, 65:] = ref.stored(k)[1, :, :5], ref.stored(v)[1, :, :5]
    gk, gv = dev.load(kv, 0, B, G, S, hd)
    assert np.array_equal(gk, want_k) and np.array_equal(gv, want_v)
    gk, _ = dev.load(kv, 0, B, G, 20, hd, at=dev.buf([3, 60, -2, 70]), end=dev.buf([10, 200, 5, 90]))
    assert np.array_equal(gk[0, :, :7], want_k[0, :, 3:10]) and np.all(gk[0, :, 7:] == FILL)
    assert np.array_equal(gk[1, :, :10], want_k[1, :, 60:]) and np.all(gk[1, :, 10:] == FILL)
    assert np.all(gk[2:] == FILL)


# ───────────── attention ─────────────

def run_attention(dev, rng, hd, G, R, S, lens, new, window, packed, pos=None, spread=1.0, in_place=False, behind=0, offsets=0, layers=1, layer=0, B_extra=0):
    """One op 87 or 88 against the reference; rows of no sequence, stale cache rows and weights hold values that must not matter."""
    B, H = len(lens), G * R
    starts = np.concatenate(([0], np.cumsum(new)))
    M = int(starts[-1]) + behind
    lens = np.asarray(lens, dtype=np.float32)
    pos = lens if pos is None else np.asarray(pos, dtype=np.float32)
    max_pos = int(max(S, pos.max() + max(new) + 1, 1))
    cos, sin = tables(max_pos, hd)
    width = (H + 2 * G) * hd
    qkv = (rows(rng, M, width) * spread).astype(np.float32)
    if behind:
        qkv[-behind:] = np.nan
    K0, V0 = rows(rng, B + B_extra, G, S, hd), rows(rng, B + B_extra, G, S, hd)
    acc = rng.random((B, G, S)).astype(np.float32)
    for b in range(B):
        acc[b, :, max(0, int(lens[b])):] = np.nan                    # weights of rows that are not there are not read
    kv = dev.cache(layers, B + B_extra, G, S, hd)
    dev.store(kv, layer, K0, V0)
    ld = width + offsets
    wide = np.full((M, ld), np.nan, dtype=np.float32)
    wide[:, offsets:] = qkv
    x = dev.buf(wide)
    ldo = H * hd + offsets
    out = dev.buf(np.full(M * ldo + 4, FILL))
    a = dev.buf(acc) if window else -1
    ao = a if in_place else dev.buf(np.full(acc.size, FILL)) if window else -1
    where = [x, offsets, offsets + H * hd, offsets + (H + G) * hd, ld, kv, layer]
    rest = [dev.buf(lens), dev.buf(pos), dev.buf(cos), dev.buf(sin), max_pos, out, offsets, ldo, B, H]
    if packed:
        words = [cg.OP_ATTN_PACKED_Q4] + where + [dev.buf(starts)] + rest + [M, a, ao, window]
    else:
        words = [cg.OP_ATTN_DECODE_Q4] + where + rest + [a, ao]
    K, V = ref.stored(K0), ref.stored(V0)
    want, tol, weights, wtol = ref.attend(K[:B], V[:B], qkv, starts, lens, pos, cos, sin, H, window, acc if window else None)
    times = 1 if in_place else 3                                     # eager, captured, replayed: the same rows are written again
    for _ in range(times):
        dev.flush(*words)
        got = dev.get(out, (M * ldo + 4,))[:M * ldo].reshape(M, ldo)
        assert np.all(got[:, :offsets] == FILL)
        got = got[:, offsets:]
        written = ~np.isnan(want)
        assert np.all(got[~written] == FILL)
        err = np.abs(np.where(written, got - np.where(written, want, 0.0), 0.0))
        assert np.all(err <= tol), (float((err / np.maximum(tol, 1e-30)).max()), np.argwhere(err > tol)[:5].tolist())
        if window:
            g = dev.get(ao, acc.shape)
            written = ~np.isnan(weights)
            assert np.all(np.isnan(g[~written]) if in_place else g[~written] == FILL)
            err = np.abs(np.where(written, g - np.where(written, weights, 0.0), 0.0))
            assert np.all(err <= wtol), (float((err / np.maximum(wtol, 1e-30)).max()), np.argwhere(err > wtol)[:5].tolist())
    gk, gv = dev.load(kv, layer, B + B_extra, G, S, hd)
    assert np.array_equal(gk, K) and np.array_equal(gv, V)


STEPS = [
    # hd, G, R, S, lens
    (128, 2, 1, 64, [0]),
    (128, 1, 1, 40, [1, 30, 31, 32, 33, 39]),
    (64, 3, 2, 200, [199, 0, 64, 127]),
    (32, 5, 3, 97, [96, 5, 33]),
    (128, 2, 4, 1100, [1099, 640]),
    (64, 1, 8, 777, [776, 1, 300]),
    (128, 4, 7, 130, [129, 128]),
    (64, 2, 16, 300, [299, 64]),
    (128, 1, 2, 4000, [3999, 2500, 0]),
    (32, 2, 1, 9000, [8999]),
    (128, 1, 1, 20000, [19999, 77]),
    (64, 12, 1, 260, [200 - i for i in range(40)]),
]


@pytest.mark.parametrize("tracked", [0, 1])
@pytest.mark.parametrize("hd,G,R,S,lens", STEPS)
def test_token_step(dev, hd, G, R, S, lens, tracked):
    run_attention(dev, np.random.default_rng(hd * G + S), hd, G, R, S, lens, [1] * len(lens), tracked, packed=False)


def test_token_step_leaves_sequences_outside_their_range_alone(dev):
    run_attention(dev, np.random.default_rng(1), 64, 2, 2, 100, [-1, 100, 99, 12, 50], [1] * 5, 1, packed=False, pos=[3, 4, 99, -1, 7])


@pytest.mark.parametrize("spread", [1e-3, 30.0])
def test_token_step_with_flat_and_with_peaked_scores(dev, spread):
    run_attention(dev, np.random.default_rng(2), 128, 2, 2, 600, [599, 311], [1, 1], 1, packed=False, spread=spread)


def test_token_step_behind_an_eviction_in_place_in_a_layer_with_strides(dev):
    run_attention(dev, np.random.default_rng(4), 64, 2, 3, 90, [40, 89], [1, 1], 1, packed=False, pos=[400, 89], in_place=True, offsets=8, layers=3, layer=2, B_extra=2)


PROMPTS = [
    # hd, G, R, S, lens, new
    (128, 2, 1, 40, [0], [1]),
    (64, 1, 1, 300, [0, 0, 0], [127, 128, 45]),
    (128, 1, 4, 600, [0, 17, 300], [200, 33, 257]),
    (32, 2, 3, 200, [31, 0, 5, 199], [1, 0, 64, 1]),
    (64, 2, 8, 700, [650, 0], [50, 300]),
    (128, 1, 7, 300, [100, 3], [130, 20]),
    (64, 1, 40, 100, [10, 0], [7, 60]),
    (128, 2, 2, 1500, [1000, 1490, 0, 600], [4, 9, 0, 700]),
    (32, 3, 1, 5000, [4500], [16]),
]


@pytest.mark.parametrize("window", [0, 1, 20])
@pytest.mark.parametrize("hd,G,R,S,lens,new", PROMPTS)
def test_packed_prompts(dev, hd, G, R, S, lens, new, window):
    run_attention(dev, np.random.default_rng(hd * G + S + window), hd, G, R, S, lens, new, window, packed=True)


def test_packed_prompts_that_do_not_fit_are_cut(dev):
    run_attention(dev, np.random.default_rng(5), 64, 2, 2, 100, [90, 100, -1, 0], [30, 5, 5, 40], 8, packed=True)


def test_packed_prompts_leave_rows_behind_the_last_sequence(dev):
    run_attention(dev, np.random.default_rng(6), 128, 1, 2, 200, [0, 50], [70, 33], 16, packed=True, behind=37, offsets=4, layers=2, layer=1)


@pytest.mark.parametrize("spread", [1e-3, 30.0])
def test_packed_prompts_with_flat_and_with_peaked_scores(dev, spread):
    run_attention(dev, np.random.default_rng(7), 64, 1, 2, 500, [100, 0], [300, 129], 8, packed=True, spread=spread)


def test_no_rows_at_all(dev):
    kv = dev.cache(1, 2, 1, 64, 32)
    cos, sin = tables(64, 32)
    z, x = dev.buf(np.zeros(2)), dev.buf(np.zeros(0))
    dev.flush(cg.OP_ATTN_PACKED_Q4, x, 0, 32, 64, 96, kv, 0, dev.buf(np.zeros(3)), z, z, dev.buf(cos), dev.buf(sin), 64, x, 0, 32, 2, 1, 0, -1, -1, 0)


# ───────────── eviction ─────────────

@pytest.mark.parametrize("place", ["same", "other"])
@pytest.mark.parametrize("hd,G,S,lens,budget,recent", [
    (128, 2, 100, [100, 50, 49, 0, 7], 50, 10),
    (64, 1, 700, [700, 513], 256, 0),
    (32, 3, 300, [299, 300, 31], 30, 30),
    (64, 2, 40, [40, 39], 1, 0),
    (128, 1, 3000, [3000], 2900, 64),
    (32, 1, 20000, [20000, 12345], 5001, 129),
])
def test_eviction(dev, hd, G, S, lens, budget, recent, place):
    rng = np.random.default_rng(S + budget)
    B = len(lens)
    K0, V0 = rows(rng, B, G, S, hd), rows(rng, B, G, S, hd)
    acc = np.round(rng.random((B, G, S)) ** 4 * 20).astype(np.float32) / 4          # many ties
    acc[rng.random(acc.shape) < 0.05] = -0.0
    acc[rng.random(acc.shape) < 0.02] = np.inf
    acc[rng.random(acc.shape) < 0.02] = np.nan
    acc[rng.random(acc.shape) < 0.02] = -1.5
    kv = dev.cache(2, B, G, S, hd)
    dev.store(kv, 1, K0, V0)
    D = S if place == "same" else budget + 5
    dst = kv if place == "same" else dev.cache(2, B, G, D, hd)
    a = dev.buf(acc)
    ao = a if place == "same" else dev.buf(np.full(B * G * D, FILL))
    n = dev.buf(lens)
    n_out, kept = dev.buf(np.full(B, FILL)), dev.buf(np.full(B * G * budget, FILL))
    dev.flush(cg.OP_KV_EVICT_Q4, kv, dst, 1, n, a, budget, recent, B, ao, n_out, kept)
    assert np.array_equal(dev.get(n_out, (B,)), np.minimum(lens, budget)) and np.array_equal(dev.get(n, (B,)), np.asarray(lens, dtype=np.float32))
    K, V = ref.stored(K0), ref.stored(V0)
    gk, gv = dev.load(dst, 1, B, G, D, hd)
    ga, gi = dev.get(ao, (B, G, D)), dev.get(kept, (B, G, budget))
    for b in range(B):
        for g in range(G):
            stay = ref.evict(acc[b, g], lens[b], budget, recent)
            m = len(stay)
            assert np.array_equal(gi[b, g, :m], stay) and np.all(gi[b, g, m:] == FILL)
            assert np.array_equal(gk[b, g, :m], K[b, g, stay]) and np.array_equal(gv[b, g, :m], V[b, g, stay])
            assert np.array_equal(ga[b, g, :m], acc[b, g, stay], equal_nan=True)
            if place == "same":                                                       # rows behind the kept ones stay as they were
                assert np.array_equal(gk[b, g, m:], K[b, g, m:]) and np.array_equal(ga[b, g, m:], acc[b, g, m:], equal_nan=True)
            else:
                assert not gk[b, g, m:].any() and np.all(ga[b, g, m:] == FILL)


# ───────────── refusals ─────────────

def test_refusals(dev):
    lib = dev.rt.lib
    for args in ((1, 1, 1, 64, 48), (1, 1, 1, 64, 256), (0, 1, 1, 64, 64), (1, 1, 1, 0, 64), (1, 1, 1, (1 << 24) + 1, 64)):
        assert lib.deepj_cuda_kv_alloc_q4(dev.id(), *args) != 0
    kv, small, odd = dev.cache(1, 2, 2, 64, 64), dev.cache(1, 2, 2, 32, 64), dev.cache(1, 2, 2, 64, 32)
    cos, sin = tables(64, 64)
    x, out = dev.buf(np.zeros((2, 6 * 64))), dev.buf(np.zeros((2, 128)))
    z, c, s, st = dev.buf(np.zeros(2)), dev.buf(cos), dev.buf(sin), dev.buf([0, 1, 2])
    w, w2 = dev.buf(np.zeros(2 * 2 * 64)), dev.buf(np.zeros(2 * 2 * 32))
    z2 = dev.buf(np.zeros(2))
    step = [cg.OP_ATTN_DECODE_Q4, x, 0, 128, 256, 384, kv, 0, z, z, c, s, 64, out, 0, 128, 2, 2, w, w]
    pack = [cg.OP_ATTN_PACKED_Q4, x, 0, 128, 256, 384, kv, 0, st, z, z, c, s, 64, out, 0, 128, 2, 2, 2, w, w, 1]
    evict = [cg.OP_KV_EVICT_Q4, kv, small, 0, z, w, 16, 4, 2, w2, z2, -1]
    store = [cg.OP_KV_STORE_Q4, x, 0, 128, 384, kv, 0, z, 2, 1]
    load = [cg.OP_KV_LOAD_Q4, kv, 0, z, -1, 1, out, out, 1]
    for good in (step, pack, evict, store, load):
        dev.flush(*good)

    def bad(words, at, value):
        words = list(words)
        words[at] = value
        with pytest.raises(_lib.DeepJCudaError):
            dev.flush(*words)

    for at, value in ((1, z), (2, 2), (3, -4), (5, 380), (5, 386), (6, w), (7, 1), (7, -1), (8, -1), (10, z), (12, 65), (12, 0), (13, z), (14, 2), (15, 124), (16, 3),
                      (16, 0), (17, 3), (17, 0), (17, 6), (18, -1), (19, -1), (19, z)):
        bad(step, at, value)
    for at, value in ((8, z), (8, -1), (17, 3), (19, 3), (19, -1), (20, -1), (22, 0), (22, -1), (21, z), (6, x)):
        bad(pack, at, value)
    for at, value in ((1, w), (2, odd), (2, w), (3, 1), (6, 0), (6, 33), (7, -1), (7, 17), (8, 3), (9, z), (9, w2 + 1000), (10, z), (11, z)):
        bad(evict, at, value)
    bad(evict, 9, w)                                                                   # in place needs one cache size
    for at, value in ((1, z), (2, 2), (4, 252), (4, 258), (5, x), (6, 1), (7, -1), (8, 3), (9, 2), (9, -1)):
        bad(store, at, value)
    for at, value in ((1, w), (2, 1), (5, 3), (5, -1), (6, z), (8, 3), (3, w2 + 1000)):
        bad(load, at, value)
    with pytest.raises(_lib.DeepJCudaError):
        dev.rt.device_view(kv, (1,))
    with pytest.raises(ValueError):
        dev.rt.device_view(z, (3,))


def test_another_cache_kind_is_refused(dev):
    kv = dev.id()
    _lib.check(dev.rt.lib.deepj_cuda_kv_alloc(kv, 1, 1, 1, 64, 64))
    with pytest.raises(_lib.DeepJCudaError):
        dev.load(kv, 0, 1, 1, 1, 64)


# ───────────── together ─────────────

def test_prompts_steps_and_evictions_in_a_row(dev):
    """A server's life: packed prompts, steps, an eviction in place, more steps, the next turn's prompt, replayed streams throughout."""
    rng = np.random.default_rng(11)
    hd, G, R, S, B = 64, 2, 2, 96, 3
    H, width = G * R, (G * R + 2 * G) * hd
    cos, sin = tables(400, hd)
    kv = dev.cache(1, B, G, S, hd)
    K, V, acc = np.zeros((B, G, S, hd), np.float32), np.zeros((B, G, S, hd), np.float32), np.zeros((B, G, S), np.float32)
    lens, pos = np.zeros(B, np.float32), np.zeros(B, np.float32)
    n, n2, p, a, c, s = dev.buf(lens), dev.buf(lens), dev.buf(pos), dev.buf(acc), dev.buf(cos), dev.buf(sin)
    most = 60
    x, out, st = dev.buf(np.zeros((B * most, width))), dev.buf(np.zeros((B * most, H * hd))), dev.buf(np.zeros(B + 1))

    def prompt(new):
        starts = np.concatenate(([0], np.cumsum(new))).astype(np.float32)
        M = int(starts[-1])
        qkv = rows(rng, M, width)
        dev.rt.upload_buffer(x, qkv)
        dev.rt.upload_buffer(st, starts)
        dev.flush(cg.OP_ATTN_PACKED_Q4, x, 0, H * hd, (H + G) * hd, width, kv, 0, st, n, p, c, s, 400, out, 0, H * hd, B, H, M, a, a, 8)
        want, tol, w, wtol = ref.attend(K, V, qkv, starts, lens, pos, cos, sin, H, 8, acc)
        assert np.all(np.abs(dev.get(out, (B * most, H * hd))[:M] - want) <= tol)
        follow(w, np.asarray(new, np.float32))

    def follow(w, new):
        got = dev.get(a, acc.shape)
        there = ~np.isnan(w)
        assert np.allclose(got[there], w[there], rtol=1e-4, atol=1e-5)
        acc[:] = got                                                  # the device's own sums decide the next eviction
        lens[:] += new
        pos[:] += new
        dev.rt.upload_buffer(n, lens)
        dev.rt.upload_buffer(p, pos)

    def step():
        qkv = rows(rng, B, width)
        dev.rt.upload_buffer(x, qkv)
        dev.flush(cg.OP_ATTN_DECODE_Q4, x, 0, H * hd, (H + G) * hd, width, kv, 0, n, p, c, s, 400, out, 0, H * hd, B, H, a, a)
        want, tol, w, wtol = ref.attend(K, V, qkv, np.arange(B + 1), lens, pos, cos, sin, H, 1, acc)
        assert np.all(np.abs(dev.get(out, (B * most, H * hd))[:B] - want) <= tol)
        follow(w, np.ones(B, np.float32))

    def evict():
        dev.flush(cg.OP_KV_EVICT_Q4, kv, kv, 0, n, a, 40, 12, B, a, n2, -1, cg.OP_COPY, n2, 0, n, 0, B)
        for b in range(B):
            for g in range(G):
                stay = ref.evict(acc[b, g], int(lens[b]), 40, 12)
                K[b, g, :len(stay)], V[b, g, :len(stay)], acc[b, g, :len(stay)] = K[b, g, stay], V[b, g, stay], acc[b, g, stay]
        lens[:] = np.minimum(lens, 40)
        assert np.array_equal(dev.get(n, (B,)), lens)

    prompt([50, 60, 7])
    for _ in range(5):
        step()
    evict()
    for _ in range(4):
        step()
    prompt([3, 0, 45])
    evict()
    for _ in range(3):
        step()
    assert dev.rt.lib.deepj_cuda_synchronize() == 0


def test_a_buffer_seen_from_another_library(dev):
    torch = pytest.importorskip("torch")
    i = dev.buf(np.arange(6))
    view = torch.as_tensor(dev.rt.device_view(i, (2, 3)), device="cuda")
    assert view.data_ptr() % 256 == 0 and torch.equal(view.cpu(), torch.arange(6.0).view(2, 3))
    view += 1
    torch.cuda.synchronize()
    assert np.array_equal(dev.get(i, (6,)), np.arange(6) + 1)
