"""Lengths, positions and places of the 4-bit cache's ops that are no numbers, or far outside: sequences that are left out, never rows that are not there.  As many
sequences times heads as there may be."""
import numpy as np
import pytest

import q4_ref as ref
from deepj_b200 import compute_graph as cg
from test_q4_cache_gpu import FILL, dev, rows, tables  # noqa: F401

pytestmark = pytest.mark.gpu
OUT = [np.nan, -0.5, -1.0, np.inf, -np.inf, 3e9, -3e9, 1e38, -1e38]
S, HD, G = 70, 32, 2


def cache(dev, rng, B):  # noqa: F811
    k, v = rows(rng, B, G, S, HD), rows(rng, B, G, S, HD)
    kv = dev.cache(1, B, G, S, HD)
    dev.store(kv, 0, k, v)
    return kv


@pytest.mark.parametrize("what", ["at", "end"])
def test_row_loads(dev, what):  # noqa: F811
    B = len(OUT) + 1
    kv = cache(dev, np.random.default_rng(1), B)
    want, _ = dev.load(kv, 0, B, G, S, HD)
    at, end = [5.0] * B, [60.0] * B
    (at if what == "at" else end)[:-1] = OUT
    got, gv = dev.load(kv, 0, B, G, S, HD, at=dev.buf(at), end=dev.buf(end))
    for b in range(B - 1):
        if what == "end" and OUT[b] > 0:                             # beyond the cache: to its end
            assert np.array_equal(got[b, :, :S - 5], want[b, :, 5:]) and np.all(got[b, :, S - 5:] == FILL)
        else:
            assert np.all(got[b] == FILL) and np.all(gv[b] == FILL)
    assert np.array_equal(got[-1, :, :55], want[-1, :, 5:60])


def test_row_stores(dev):  # noqa: F811
    B, rng = len(OUT) + 1, np.random.default_rng(2)
    kv = cache(dev, rng, B)
    before = dev.load(kv, 0, B, G, S, HD)
    k = rows(rng, B, G, 3, HD)
    dev.store(kv, 0, k, k, OUT + [4.0])
    for x, y in zip(before, dev.load(kv, 0, B, G, S, HD)):
        assert np.array_equal(x[:-1], y[:-1]) and not np.array_equal(x[-1], y[-1])


def run(dev, rng, B, packed, lens, pos, starts, M):  # noqa: F811
    kv = cache(dev, rng, B)
    cos, sin = tables(S, HD)
    acc, out = dev.buf(np.full(B * G * S, FILL)), dev.buf(np.full(M * G * HD, FILL))
    head = [dev.buf(rows(rng, M, 3 * G * HD)), 0, G * HD, 2 * G * HD, 3 * G * HD, kv, 0]
    tail = [dev.buf(lens), dev.buf(pos), dev.buf(cos), dev.buf(sin), S, out, 0, G * HD, B, G]
    old = dev.buf(np.zeros(B * G * S))
    if packed:
        dev.flush(cg.OP_ATTN_PACKED_Q4, *head, dev.buf(starts), *tail, M, old, acc, 3)
    else:
        dev.flush(cg.OP_ATTN_DECODE_Q4, *head, *tail, old, acc)
    return [dev.get(out, (M * G * HD,)), dev.get(acc, (B * G * S,)), *dev.load(kv, 0, B, G, S, HD)]


@pytest.mark.parametrize("packed", [False, True])
@pytest.mark.parametrize("what", ["len", "pos"])
def test_attention(dev, packed, what):  # noqa: F811
    B = len(OUT) + 2
    M = 2 * B if packed else B
    starts = np.arange(B + 1) * 2
    got = []
    for bad in (OUT, [-1.0] * len(OUT)):                             # the same as sequences that are left out
        lens, pos = [10.0] * B, [12.0] * B
        (lens if what == "len" else pos)[1:-1] = bad
        got.append(run(dev, np.random.default_rng(3), B, packed, lens, pos, starts, M))
    for a, b in zip(*got):
        assert np.array_equal(a, b)
    out = got[0][0].reshape(M, -1)
    n = M // B
    assert np.all(out[n:-n] == FILL) and np.all(out[:n] != FILL) and np.all(out[-n:] != FILL)


def test_starts(dev):  # noqa: F811
    """Sequence 0 has rows 0 … 3; what lies between two others' places is empty, or cut to the rows there are."""
    starts = [0.0, 4.0, 3e9, -3e9, np.nan, -7.0, -np.inf]
    got = run(dev, np.random.default_rng(4), 6, True, [10.0] * 6, [10.0] * 6, starts, 4)
    want = run(dev, np.random.default_rng(4), 6, True, [10.0] * 6, [10.0] * 6, [0.0] + [4.0] * 6, 4)
    for a, b in zip(got, want):
        assert np.array_equal(a, b)


def test_eviction(dev):  # noqa: F811
    B, budget = len(OUT) + 1, 20
    rng = np.random.default_rng(5)
    kv, small = cache(dev, rng, B), dev.cache(1, B, G, budget, HD)
    acc, new, n = dev.buf(rng.random(B * G * S)), dev.buf(np.full(B * G * budget, FILL)), dev.buf(np.full(B, FILL))
    dev.flush(cg.OP_KV_EVICT_Q4, kv, small, 0, dev.buf(OUT + [30.0]), acc, budget, 5, B, new, n, -1)
    assert np.array_equal(dev.get(n, (B,)), [20.0 if x > 0 else 0.0 for x in OUT] + [20.0])
    k, _ = dev.load(small, 0, B, G, budget, HD)
    for b, x in enumerate(OUT):
        assert np.any(k[b]) == (x > 0)


def test_rows_of_as_many_heads_as_a_cache_has(dev):  # noqa: F811
    """More than 65535 sequences times heads: stored, loaded, moved."""
    B, heads, rows_of = 2060, 32, 2
    k, v = (np.random.default_rng(6 + i).standard_normal((B, heads, rows_of, HD)).astype(np.float32) for i in range(2))
    kv, other = dev.cache(1, B, heads, rows_of, HD), dev.cache(1, B, heads, 1, HD)
    dev.store(kv, 0, k, v)
    gk, gv = dev.load(kv, 0, B, heads, rows_of, HD)
    assert np.array_equal(gk, ref.stored(k)) and np.array_equal(gv, ref.stored(v))
    w = np.random.default_rng(8).random((B, heads, rows_of)).astype(np.float32)
    dev.flush(cg.OP_KV_EVICT_Q4, kv, other, 0, dev.buf(np.full(B, rows_of)), dev.buf(w), 1, 0, B, dev.buf(np.zeros(B * heads)), dev.buf(np.zeros(B)), -1)
    ok, ov = dev.load(other, 0, B, heads, 1, HD)
    at = w.argmax(2)[..., None, None]
    assert np.array_equal(ok, np.take_along_axis(gk, at, 2)) and np.array_equal(ov, np.take_along_axis(gv, at, 2))
