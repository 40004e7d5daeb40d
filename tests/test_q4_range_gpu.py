"""Attention over the 4-bit cache where the numbers are far apart: a key that takes nearly all of the weight above thousands that share the rest, sums of
thousands of equal weights, queries and scores of any finite size."""
import ctypes

import numpy as np
import pytest

import q4_ref as ref
from deepj_b200 import _lib
from deepj_b200 import compute_graph as cg
from test_q4_cache_gpu import FILL, dev, rows, tables  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def no_wait_ran_out(dev):  # noqa: F811
    yield
    stats = (ctypes.c_int64 * 8)()
    _lib.check(dev.rt.lib.deepj_cuda_stats(stats, 8))
    assert stats[5] == 0


def attend(dev, K, V, qkv, n, packed, R=1, window=0):  # noqa: F811
    """One sequence of n cached rows and M new tokens (a step: one) → outputs [M][H][hd], accumulated weights [G][n + M] or None.  Positions are 0: the tables'
    first rows do not rotate."""
    G, _, hd = K.shape
    M, H, S = qkv.shape[0], K.shape[0] * R, n + qkv.shape[0]
    kv = dev.cache(1, 1, G, S, hd)
    dev.store(kv, 0, K[None], V[None])
    out = dev.buf(np.full(M * H * hd, FILL))
    a, ao = (dev.buf(np.zeros(G * S)), dev.buf(np.full(G * S, FILL))) if window else (-1, -1)
    ones, none = dev.buf(np.ones(max(M, 1) * hd // 2)), dev.buf(np.zeros(max(M, 1) * hd // 2))
    head = [dev.buf(qkv), 0, H * hd, (H + G) * hd, qkv.shape[1], kv, 0]
    tail = [dev.buf([n]), dev.buf([0]), ones, none, M, out, 0, H * hd, 1, H]
    if packed:
        dev.flush(cg.OP_ATTN_PACKED_Q4, *head, dev.buf([0, M]), *tail, M, a, ao, window)
    else:
        dev.flush(cg.OP_ATTN_DECODE_Q4, *head, *tail, a, ao)
    return dev.get(out, (M, H, hd)), dev.get(ao, (G, S)) if window else None


def one_above(G, n, hd, M, nats, sink, others):
    """n cached rows: the first one's score is `nats` above those of all others, which are 0; values `sink` and `others`.  Returns K, V, qkv and the score."""
    K, V = np.zeros((G, n, hd), np.float32), np.full((G, n, hd), others, np.float32)
    K[:, 0], V[:, 0] = 7.0, sink                                     # scale 1, code 7: stored as they are
    qkv = np.zeros((M, 3 * G * hd), np.float32)
    qkv[:, :G * hd] = nats / (7.0 * np.sqrt(hd))                     # times 7, hd of them, over the root of hd
    qkv[:, 2 * G * hd:] = others
    score = float(qkv[0, 0]) * 7.0 * np.sqrt(hd)
    return K, V, qkv, score


def relative(score):
    """What a weight, a sum of weights and a product with values may be off, relative to themselves.  Operands carry 22 bits: a score is off by 2^-21 of its
    terms' magnitudes, twice (two weights of a quotient); exponential and quotient 2^-20.  The tensor cores cut an fp32 sum off once for 16 keys and each half of the
    weights, 128 times 2^-23 until it is added up rounded; the sums of weights are 64 additions of 2^-24 one behind the other at most."""
    return 2 * 2.0 ** -21 * abs(score) + 2.0 ** -20 + 128 * 2.0 ** -23 + 64 * 2.0 ** -24


@pytest.mark.parametrize("packed", [True, False])
@pytest.mark.parametrize("G,n", [(2, 4000), (2, 16000), (160, 4000), (160, 16000)])
@pytest.mark.parametrize("nats", [10.0, 17.4, 18.0])
def test_many_small_weights_below_a_large_one(dev, packed, G, n, nats):  # noqa: F811
    """The large weight's value is zero, the others' are equal: the output is what is left of the small weights."""
    hd, M = 32, 3 if packed else 1
    K, V, qkv, score = one_above(G, n, hd, M, nats, 0.0, 7.0)
    got, weights = attend(dev, K, V, qkv, n, packed, window=1)
    for t in range(M):
        rest = (n - 1 + t + 1) * np.exp(-score)
        want = 7.0 * rest / (1.0 + rest)
        # in prompts a weight is two fp16 halves of 2^9 times it, whose steps end at 2^-24
        tol = want * relative(score) + 7.0 * (n + t) * 2.0 ** -33
        assert np.all(np.abs(got[t] - want) <= tol), (t, float(np.abs(got[t] - want).max() / tol), float(got[t].flat[0]), want)
    rest = (n + M - 1) * np.exp(-score)
    assert np.all(np.abs(weights[:, 0] * (1.0 + rest) - 1.0) <= relative(score))
    assert np.all(np.abs(weights[:, 1:] * (1.0 + rest) * np.exp(score) - 1.0) <= relative(score))


@pytest.mark.parametrize("packed", [True, False])
@pytest.mark.parametrize("G,n", [(2, 16000), (160, 16000)])
@pytest.mark.parametrize("nats", [0.3, 0.7, 2.9])
def test_sums_of_equal_weights(dev, packed, G, n, nats):  # noqa: F811
    """All values are equal, so the output is that value: sums that drift apart show.  The weights of a chain of equal ones are all rounded the same way."""
    hd, M = 32, 2 if packed else 1
    K, V, qkv, score = one_above(G, n, hd, M, nats, 7.0, 7.0)
    got, weights = attend(dev, K, V, qkv, n, packed, window=1)
    assert np.all(np.abs(got / 7.0 - 1.0) <= relative(score)), float(np.abs(got / 7.0 - 1.0).max() / relative(score))
    rest = (n + M - 1) * np.exp(-score)
    assert np.all(np.abs(weights[:, 1:] * (1.0 + rest) * np.exp(score) - 1.0) <= relative(score)), float(np.abs(weights[:, 1:] * (1.0 + rest) * np.exp(score) - 1.0).max())


@pytest.mark.parametrize("packed", [True, False])
@pytest.mark.parametrize("value", [1e30, 1e32, 3e38])
@pytest.mark.parametrize("hd,G,n", [(32, 2, 100), (64, 1, 3000), (128, 3, 70)])
def test_large_queries_against_keys_of_zero(dev, packed, hd, G, n, value):  # noqa: F811
    rng = np.random.default_rng(hd)
    M = 5 if packed else 1
    K, V, qkv = np.zeros((G, n, hd), np.float32), rows(rng, G, n, hd), rows(rng, M, 3 * G * hd)
    qkv[:, :G * hd] = np.clip(qkv[:, :G * hd], -1, 1) * np.float32(value)
    qkv[:, G * hd:2 * G * hd] = 0.0
    got, _ = attend(dev, K, V, qkv, n, packed)
    old, new = ref.stored(V).astype(np.float64), ref.stored(qkv[:, 2 * G * hd:]).reshape(M, G, hd).astype(np.float64)
    for t in range(M):
        want = (old.sum(1) + new[:t + 1].sum(0)) / (n + t + 1)
        assert np.all(np.abs(got[t] - want) <= 2.0 ** -20 * np.abs(V).max() + 1e-12)


@pytest.mark.parametrize("packed", [True, False])
@pytest.mark.parametrize("scale", [1e4, 1e7, 1e9, 1e12, 1e20])
@pytest.mark.parametrize("hd,G,n", [(64, 2, 300), (128, 1, 3000)])
def test_scores_of_any_size_choose_a_key(dev, packed, hd, G, n, scale):  # noqa: F811
    """Scores so far apart that one weight is left: the output is that key's value, whatever the scores' size."""
    rng = np.random.default_rng(hd + n)
    M = 4 if packed else 1
    K, V, qkv = rows(rng, G, n, hd), rows(rng, G, n, hd), rows(rng, M, 3 * G * hd)
    qkv[:, :G * hd] *= np.float32(scale)
    got, weights = attend(dev, K, V, qkv, n, packed, window=M)
    assert np.all(np.abs(weights.astype(np.float64).sum(1) / M - 1.0) <= 2.0 ** -18)         # every token's weights add up to one
    k64, v64 = ref.stored(K).astype(np.float64), ref.stored(V).astype(np.float64)
    new = qkv.reshape(M, 3, G, hd)
    for t in range(M):
        for g in range(G):
            k = np.concatenate((k64[g], ref.stored(new[:t + 1, 1, g]).astype(np.float64)))
            v = np.concatenate((v64[g], ref.stored(new[:t + 1, 2, g]).astype(np.float64)))
            q = new[t, 0, g].astype(np.float64)
            sc, A = k @ q / np.sqrt(hd), (np.abs(k) @ np.abs(q) / np.sqrt(hd)).max()
            order = np.argsort(sc)
            gap = sc[order[-1]] - sc[order[-2]]
            if gap < 30.0 + 4 * 2.0 ** -21 * A:                      # two keys the operands' 22 bits do not tell apart
                continue
            assert np.all(np.abs(got[t, g] - v[order[-1]]) <= 2.0 ** -20 * np.abs(v).max()), (t, g, got[t, g][:4], v[order[-1]][:4])


@pytest.mark.parametrize("packed", [True, False])
@pytest.mark.parametrize("channel", [5, 70])
@pytest.mark.parametrize("G,R,n", [(2, 1, 200), (1, 4, 900), (1, 1, 9000)])
def test_queries_with_one_large_value(dev, packed, channel, G, R, n):  # noqa: F811
    """One value of each query is 2^12 times the others, and no key has anything there: the scores are the other values' alone.  Operands of 30 bits and more of the
    largest value (steps: half a step is 2^-30 of it, prompts: 2^-33) hold these to 18."""
    hd, M = 128, 4 if packed else 1
    rng = np.random.default_rng(channel + n)
    K, V, q, k_new, v_new = rows(rng, G, n, hd), rows(rng, G, n, hd), rng.standard_normal((M, G * R, hd)).astype(np.float32), rows(rng, M, G, hd), rows(rng, M, G, hd)
    K[..., channel], k_new[..., channel], q[..., channel] = 0.0, 0.0, 4096.0 * np.abs(q).max()
    got, weights = attend(dev, K, V, np.concatenate((q, k_new, v_new), 1).reshape(M, -1), n, packed, R, window=M)
    k_new, v_new = ref.stored(k_new).astype(np.float64), ref.stored(v_new).astype(np.float64)
    want_w, tol_w = np.zeros((G, n + M)), np.zeros((G, n + M))
    for t in range(M):
        for h in range(G * R):
            g = h // R
            k = np.concatenate((ref.stored(K[g]).astype(np.float64), k_new[:t + 1, g]))
            v = np.concatenate((ref.stored(V[g]).astype(np.float64), v_new[:t + 1, g]))
            x = q[t, h].astype(np.float64)
            sc = k @ x / np.sqrt(hd)
            off = 2.0 ** -30 * np.abs(x).max() * np.abs(k).sum(1).max() / np.sqrt(hd) + 2.0 ** -21 * (np.abs(k) @ np.abs(x) / np.sqrt(hd)).max()
            p = np.exp(sc - sc.max())
            p /= p.sum()
            rel = 2 * off + 2.0 ** -19                               # the sums of weights among it, as above
            assert np.all(np.abs(got[t, h] - p @ v) <= rel * np.abs(v).max())
            want_w[g, :n + t + 1] += p
            tol_w[g, :n + t + 1] += rel * p
    err = np.abs(weights - want_w) / tol_w
    assert np.all(err <= 1.0), float(err.max())


@pytest.mark.parametrize("R,M", [(1, 3000), (8, 2000), (33, 300)])
def test_weights_of_many_tokens_add_up(dev, R, M):  # noqa: F811
    """All weights of a token are equal, one over its keys: an old row gets a sum of R · M of them, whose roundings all go the same way for long stretches."""
    hd, n = 32, 5
    qkv = np.zeros((M, (R + 2) * hd), np.float32)
    qkv[:, (R + 1) * hd:] = 7.0
    K = np.full((1, n, hd), 7.0, np.float32)                         # stored as they are
    got, weights = attend(dev, K, K, qkv, n, True, R, window=M)
    each = R / (n + 1.0 + np.arange(M))
    tail = np.cumsum(each[::-1])[::-1]
    want = np.concatenate((np.full(n, tail[0]), tail))
    # exponential and quotient 2^-20; additions one behind the other, half a step each: a token's sum 64, then 64 of a tile of 128 query rows, and the tiles
    rel = 2.0 ** -20 + (64 + 64 + (R * M + 127) // 128) * 2.0 ** -25
    err = np.abs(weights[0] / want - 1.0).max()
    assert err <= rel, (float(err), rel)
    assert np.all(np.abs(got / 7.0 - 1.0) <= relative(0.0))
