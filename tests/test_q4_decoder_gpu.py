"""A decoder over the 4-bit K/V cache: against the same model written out in 64 bits over the cache's own values, with prompts
of one length and of several, and past the end of its rows."""
import numpy as np
import pytest

import oracle
import q4_ref as ref
from deepj_b200.decoder import DecoderConfig, Q8Decoder, rope_tables
from test_decoder_gpu import weight_getter

pytestmark = pytest.mark.gpu


class Model:
    """One sequence of a Llama-shaped model in 64 bits; its cache holds what a 4-bit cache would and may be evicted from."""

    def __init__(self, om, cfg, rows=None, budget=None, recent=None, window=32):
        self.om, self.c, self.rows, self.budget, self.recent, self.window = om, cfg, rows, budget, recent, window
        self.cos, self.sin = rope_tables(cfg.head_dim, cfg.max_seq_len)
        H, hd = cfg.n_heads, cfg.head_dim
        self.K = [[np.zeros((0, hd), np.float32) for _ in range(H)] for _ in range(cfg.n_layers)]
        self.V = [[np.zeros((0, hd), np.float32) for _ in range(H)] for _ in range(cfg.n_layers)]
        self.seen = [[np.zeros(0) for _ in range(H)] for _ in range(cfg.n_layers)]
        self.pos = 0

    def w(self, name, layer=-1):
        c = self.c
        shapes = {n: (k, w) for n, k, w in c.matmul_shapes()}
        shapes.update(emb=(c.vocab_size, c.d_model), Wlm=(c.d_model, c.vocab_size))
        a = self.om.weight(name, layer) if layer >= 0 else self.om.weight(name)
        return a.reshape(shapes[name]).astype(np.float64) if name in shapes else a.astype(np.float64)

    @staticmethod
    def norm(x, g):
        return x / np.sqrt((x * x).mean(-1, keepdims=True) + 1e-6) * g

    def run(self, tokens):
        """Logits behind the last of `tokens`, which are one chunk."""
        c = self.c
        H, hd, T = c.n_heads, c.head_dim, len(tokens)
        if self.rows is not None and len(self.K[0][0]) + T > self.rows:
            for l in range(c.n_layers):
                for h in range(H):
                    stay = ref.evict(self.seen[l][h], len(self.seen[l][h]), self.budget, self.recent)
                    self.K[l][h], self.V[l][h], self.seen[l][h] = self.K[l][h][stay], self.V[l][h][stay], self.seen[l][h][stay]
        x = self.w("emb")[np.asarray(tokens)]
        cs, sn = self.cos[self.pos:self.pos + T], self.sin[self.pos:self.pos + T]
        for l in range(c.n_layers):
            n = self.norm(x, self.w("g1", l))
            q, k, v = (n @ self.w(name, l) for name in ("Wq", "Wk", "Wv"))
            att = np.empty_like(x)
            for h in range(H):
                s = slice(h * hd, (h + 1) * hd)
                K = np.concatenate((self.K[l][h], ref.stored(ref.rotate32(k[:, s].astype(np.float32), cs, sn))))
                V = np.concatenate((self.V[l][h], ref.stored(v[:, s].astype(np.float32))))
                old = len(K) - T
                sc = ref.rotate64(q[:, s], cs, sn) @ K.astype(np.float64).T / np.sqrt(hd)
                sc[np.arange(len(K))[None] > old + np.arange(T)[:, None]] = -np.inf
                p = np.exp(sc - sc.max(1, keepdims=True))
                p /= p.sum(1, keepdims=True)
                att[:, s] = p @ V
                self.K[l][h], self.V[l][h] = K, V
                self.seen[l][h] = np.concatenate((self.seen[l][h], np.zeros(T))) + p[-self.window:].sum(0)
            x = x + att @ self.w("Wo", l)
            n = self.norm(x, self.w("g2", l))
            gate = n @ self.w("Wg", l) + self.w("bg", l)
            x = x + (gate / (1.0 + np.exp(-gate)) * (n @ self.w("Wu", l) + self.w("bu", l))) @ self.w("Wd", l) + self.w("bd", l)
        self.pos += T
        return self.norm(x[-1], self.w("gF")) @ self.w("Wlm") + self.w("blm")


def pair(cfg, batch, seed=5, **kw):
    om = oracle.OracleModel(cfg.kind, cfg.vocab_size, cfg.max_seq_len, cfg.d_model, cfg.n_heads, cfg.n_layers, cfg.d_ff, seed=seed)
    dec = Q8Decoder(cfg, batch=batch, kv_dtype="q4", **kw)
    dec.load_weights(weight_getter(om, cfg))
    om.apply_q8()
    return om, dec


def close(got, want):
    """A key or value next to the border of two codes may fall on the other side (its inputs differ in the last bits): one code of some
    hundreds, which moves logits by a few thousandths of their range.  Without such a row the two agree to 1e-4."""
    return np.abs(got - want).max() <= 1e-2 * (want.max() - want.min())


@pytest.mark.parametrize("hd,d", [(32, 256), (64, 256), (128, 256)])
def test_steps_and_chunks_match_the_model_over_4_bit_rows(hd, d):
    cfg = DecoderConfig("llama", 256, 160, d, d // hd, 2, 352)
    om, dec = pair(cfg, 2)
    try:
        rng = np.random.default_rng(hd)
        toks = rng.integers(0, 256, (2, 70))
        models = [Model(om, cfg) for _ in range(2)]
        dec.prefill(toks[:, :50])                                    # a chunk
        for b in range(2):
            assert close(dec.logits()[b], models[b].run(toks[b, :50]))
        for t in range(50, 60):
            dec.step(toks[:, t])
            want = [models[b].run(toks[b, t:t + 1]) for b in range(2)]
            assert all(close(dec.logits()[b], want[b]) for b in range(2))
        dec.prefill(toks[:, 60:], chunked=True)                      # a short chunk behind them
        for b in range(2):
            assert close(dec.logits()[b], models[b].run(toks[b, 60:]))
        dec.set_position(50)                                         # back to the first chunk's end
        dec.step(toks[:, 50])
        again = dec.logits().copy()
        dec.reset()
        dec.prefill(toks[:, :50])
        dec.step(toks[:, 50])
        assert np.array_equal(dec.logits(), again)
        assert dec.stats()["device_error"] == 0
    finally:
        dec.close()


def test_prompts_of_different_lengths_run_packed():
    cfg = DecoderConfig("llama", 256, 300, 256, 4, 2, 352)
    om, dec = pair(cfg, 4)
    try:
        rng = np.random.default_rng(1)
        prompts = [rng.integers(0, 256, n) for n in (1, 130, 37, 64)]
        models = [Model(om, cfg) for _ in range(4)]
        nxt = dec.prefill_packed(prompts)
        got = dec.logits()
        for b in range(4):
            want = models[b].run(prompts[b])
            assert close(got[b], want)
            assert nxt[b] == got[b].argmax()
        for _ in range(3):                                           # steps from their own positions
            toks = rng.integers(0, 256, 4)
            dec.step(toks)
            got = dec.logits()
            assert all(close(got[b], models[b].run(toks[b:b + 1])) for b in range(4))
        more = [rng.integers(0, 256, n) for n in (90, 2, 33, 1)]     # the next turn
        dec.prefill_packed(more)
        got = dec.logits()
        assert all(close(got[b], models[b].run(more[b])) for b in range(4))
        dec.reset()
        dec.PREFILL_CHUNK = 48                                       # several passes, sequences ending in different ones
        dec.prefill_packed(prompts)
        for b in range(4):
            m = Model(om, cfg)
            for lo in range(0, len(prompts[b]), 48):
                want = m.run(prompts[b][lo:lo + 48])
            assert close(dec.logits()[b], want)
    finally:
        dec.close()


def test_generation_goes_on_past_the_end_of_the_rows():
    cfg = DecoderConfig("llama", 256, 300, 256, 4, 2, 352)
    om, dec = pair(cfg, 1, kv_rows=64, kv_budget=40, kv_recent=16)
    try:
        rng = np.random.default_rng(2)
        toks = rng.integers(0, 256, 140)
        m = Model(om, cfg, 64, 40, 16)
        dec.prefill(toks[None, :60], chunked=True)                   # chunks of 24: what fits behind an eviction
        for lo in range(0, 60, 24):
            want = m.run(toks[lo:min(60, lo + 24)])
        assert close(dec.logits()[0], want)
        agree = []
        for t in range(60, 140):
            dec.step(toks[t:t + 1])
            want = m.run(toks[t:t + 1])
            agree.append(close(dec.logits()[0], want))
        # weights next to each other may leave in another order: that changes what stays, so not every step has to agree
        assert np.mean(agree[:5]) == 1.0 and np.mean(agree) >= 0.5, agree
        assert dec.position == 140 and int(dec._rows[0]) <= 64
        assert np.array_equal(dec._download(dec.ids["len"], 1), dec._rows)
        with pytest.raises(ValueError):
            dec.set_position(30)
        dec.reset()
        out = dec.generate(toks[:20], 100, top_k=5, seed=3)
        assert out.size == 100 and dec.position == 119
        dec.reset()
        dec.prefill(toks[None, :20])
        dec.step_device(100)
        assert dec.position == 120
    finally:
        dec.close()


def test_gpt_packed_prompts_equal_each_one_alone():
    cfg = DecoderConfig("gpt", 384, 96, 256, 4, 2, 640)
    rng = np.random.default_rng(4)
    prompts = [rng.integers(0, 384, n) for n in (40, 7, 1)]
    tail = rng.integers(0, 384, (3, 33))
    dec, one = Q8Decoder(cfg, batch=3, kv_dtype="q4"), Q8Decoder(cfg, batch=1, id_base=1 << 25, kv_dtype="q4")
    try:
        for d in (dec, one):
            d.load_synthetic(9, 0.05)
        dec.prefill_packed(prompts)
        dec.step(tail[:, 0])
        dec.prefill(tail[:, 1:], chunked=True)                       # a chunk behind them: every sequence from its own position
        for b in range(3):
            one.reset()
            one.prefill(prompts[b][None])
            one.prefill(tail[b:b + 1])
            assert close(dec.logits()[b], one.logits()[0])
    finally:
        dec.close()
        one.close()


def test_what_a_decoder_refuses():
    cfg = DecoderConfig("llama", 256, 64, 256, 4, 1, 352)
    for kw in (dict(kv_rows=0), dict(kv_rows=65), dict(kv_recent=3), dict(kv_budget=64), dict(kv_rows=32, kv_budget=32), dict(kv_budget=0), dict(kv_budget=20, kv_recent=21),
               dict(fused_step=True)):
        with pytest.raises(ValueError):
            Q8Decoder(cfg, kv_dtype="q4", **kw)
    with pytest.raises(ValueError):
        Q8Decoder(cfg, kv_rows=32)
    with pytest.raises(ValueError):
        Q8Decoder(DecoderConfig("llama", 256, 64, 96, 2, 1, 352), kv_dtype="q4")
    om, dec = pair(cfg, 2, kv_rows=40)
    try:
        for bad in ([[1]], [[1], []], [[1], [256]], [[1], list(range(65))], [[1], [1] * 41]):
            with pytest.raises(ValueError):
                dec.prefill_packed(bad)
        dec.prefill_packed([[1] * 38, [2] * 3])
        dec.step([1, 2])
        dec.step([1, 2])
        with pytest.raises(ValueError):
            dec.step([1, 2])                                         # the first sequence's rows are full
        with pytest.raises(ValueError):
            dec.prefill([[1] * 35, [2] * 35], chunked=True)
        plain = Q8Decoder(cfg, batch=1, id_base=1 << 25)
        with pytest.raises(ValueError):
            plain.prefill_packed([[1]])
        plain.close()
    finally:
        dec.close()
