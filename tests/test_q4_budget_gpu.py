"""Decoders over a bounded 4-bit cache with several sequences: each is evicted from when it is full itself, and follows the model at every step."""
import numpy as np
import pytest

from deepj_b200 import _lib
from deepj_b200 import compute_graph as cg
from deepj_b200.decoder import DecoderConfig
from test_q4_decoder_gpu import Model, close, pair

pytestmark = pytest.mark.gpu
CFG = DecoderConfig("llama", 256, 400, 256, 4, 2, 352)
ROWS, BUDGET, RECENT = 64, 40, 16


class Pair:
    """A decoder and a model of every sequence.  The device's own sums of attention decide what leaves: the models take them over before they evict."""

    def __init__(self, batch):
        self.om, self.dec = pair(CFG, batch, kv_rows=ROWS, kv_budget=BUDGET, kv_recent=RECENT)
        self.models = [Model(self.om, CFG, ROWS, BUDGET, RECENT) for _ in range(batch)]
        self.evictions = np.zeros(batch, int)

    def seen(self, layer):
        d = self.dec
        return d._download(d.ids[f"seen.{layer}"], d.B * CFG.n_heads * ROWS).reshape(d.B, CFG.n_heads, ROWS)

    def rows(self, layer):
        """Values of all cached rows [2][B][H][ROWS][hd]."""
        d, n = self.dec, self.dec.B * CFG.n_heads * ROWS * CFG.head_dim
        ids = [d._f32("", n) for _ in range(2)]
        s = cg.stream([cg.OP_KV_LOAD_Q4, d.ids["kv"], layer, -1, -1, ROWS, *ids, d.B])
        _lib.check(d.lib.deepj_cuda_flush_ops(s.ctypes.data, s.size))
        got = np.stack([d._download(i, n) for i in ids]).reshape(2, d.B, CFG.n_heads, ROWS, CFG.head_dim)
        d._release(ids)
        return got

    def follow(self, parts):
        """The models' logits behind these tokens, where there are some; before the device runs them."""
        want = []
        for b, p in enumerate(parts):
            m = self.models[b]
            if len(p) and len(m.K[0][0]) + len(p) > ROWS:
                self.evictions[b] += 1
                for l in range(CFG.n_layers):
                    got = self.seen(l)[b]
                    for h in range(CFG.n_heads):
                        n = len(m.seen[l][h])
                        assert np.allclose(got[h, :n], m.seen[l][h], rtol=2e-2, atol=2e-3)
                        m.seen[l][h] = got[h, :n].astype(np.float64)
            want.append(m.run(p) if len(p) else None)
        return want

    def check(self, want):
        got = self.dec.logits()
        assert all(w is None or close(got[b], w) for b, w in enumerate(want))
        assert self.dec._rows.tolist() == [len(m.K[0][0]) for m in self.models]
        assert np.array_equal(self.dec._download(self.dec.ids["len"], self.dec.B), self.dec._rows)


def test_each_sequence_is_evicted_from_when_it_is_full():
    t = Pair(3)
    try:
        rng = np.random.default_rng(1)
        prompts = [rng.integers(0, 256, n) for n in (24, 9, 17)]
        want = t.follow(prompts)
        t.dec.prefill_packed(prompts)
        t.check(want)
        for i in range(70):
            toks = rng.integers(0, 256, 3)
            full = t.dec._rows + 1 > ROWS
            before = [(t.rows(l), t.seen(l)) for l in range(CFG.n_layers)] if full.any() else None
            n = t.dec._rows.copy()
            want = t.follow([toks[b:b + 1] for b in range(3)])
            t.dec.step(toks)
            t.check(want)
            if before is not None:
                assert full.sum() == 1                               # never two at once: their lengths differ
                for l, (kv, _) in enumerate(before):
                    after = t.rows(l)
                    for b in np.flatnonzero(~full):
                        assert np.array_equal(after[:, b, :, :n[b]], kv[:, b, :, :n[b]])
        assert t.evictions.min() >= 1 and t.dec.stats()["device_error"] == 0
    finally:
        t.dec.close()


def test_prompts_evict_where_they_would_not_fit():
    t = Pair(3)
    try:
        rng = np.random.default_rng(2)
        C = t.dec._chunk_tokens()
        assert C == ROWS - BUDGET
        room = t.dec._make_room
        for lengths in ((60, 10, 30), (20, 1, 24), (1, 50, 3), (70, 9, 41)):
            prompts, at, last = [rng.integers(0, 256, n) for n in lengths], [0], [None] * 3

            def follow_pass(tokens):
                """A pass of the prompts is about to run: the models go first.  A prompt that has ended leaves its sequence alone."""
                parts = [p[at[0]:at[0] + C] for p in prompts]
                assert [len(p) for p in parts] == list(tokens)
                for b, w in enumerate(t.follow(parts)):
                    last[b] = last[b] if w is None else w
                at[0] += C
                room(tokens)
            t.dec._make_room = follow_pass
            t.dec.prefill_packed(prompts)
            t.check(last)
        assert t.evictions.min() >= 1 and t.dec.stats()["device_error"] == 0
    finally:
        t.dec.close()
