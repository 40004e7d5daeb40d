"""The sharded decoder over the 4-bit cache on one GPU: both ranks' streams run in turn, piece by piece, and the host does the exchanges between the pieces, so that
no kernel waits for another rank's."""
import numpy as np
import pytest

from deepj_b200 import _lib
from deepj_b200 import compute_graph as cg
from deepj_b200.decoder import DecoderConfig, Q8Decoder
from test_decoder_gpu import weight_getter
from test_q4_decoder_gpu import Model, close
import oracle

pytestmark = pytest.mark.gpu
WORLD = 2


def pieces(words):
    """A stream as runs of other ops, each followed by one exchange or the end."""
    run, at = [], 0
    while at < len(words):
        n = cg.OP_METADATA[int(words[at])][0]
        op = words[at:at + n]
        at += n
        if op[0] in (cg.OP_TP_ALLREDUCE, cg.OP_TP_ALLGATHER):
            yield run, op
            run = []
        else:
            run.extend(op)
    yield run, None


class Ranks:
    def __init__(self, cfg, batch, **kw):
        self.om = oracle.OracleModel(cfg.kind, cfg.vocab_size, cfg.max_seq_len, cfg.d_model, cfg.n_heads, cfg.n_layers, cfg.d_ff, seed=5)
        self.decs = [Q8Decoder(cfg, batch=batch, kv_dtype="q4", id_base=(1 << 24) + (r << 20), tp_rank=r, tp_world=WORLD, tp_slot_floats=1 << 20, **kw) for r in range(WORLD)]
        for d in self.decs:
            d.load_weights(weight_getter(self.om, cfg))
        self.om.apply_q8()

    def run(self, streams):
        for parts in zip(*(pieces(s) for s in streams), strict=True):
            for d, (run, _) in zip(self.decs, parts):
                if run:
                    s = cg.stream(run)
                    _lib.check(d.lib.deepj_cuda_flush_ops(s.ctypes.data, s.size))
            ops = [op for _, op in parts]
            if ops[0] is None:
                return
            if ops[0][0] == cg.OP_TP_ALLREDUCE:
                M, N = int(ops[0][5]), int(ops[0][6])
                total = sum(d._download(int(op[1]), M * N) for d, op in zip(self.decs, ops))
                for d, op in zip(self.decs, ops):
                    out = total + (d._download(int(op[3]), M * N) if op[3] >= 0 else 0)
                    if op[2] >= 0:
                        out = out + np.tile(d._download(int(op[2]), N), M)
                    d._upload(int(op[4]), out)
            else:
                M, n = int(ops[0][3]), int(ops[0][4])
                rows = np.concatenate([d._download(int(op[1]), M * n).reshape(M, n) for d, op in zip(self.decs, ops)], 1)
                for d, op in zip(self.decs, ops):
                    d._upload(int(op[2]), rows)

    def step(self, tokens):
        for d in self.decs:
            d.set_tokens(tokens)
            d._make_room(1)
        self.run([d._streams()[0] for d in self.decs])
        for d in self.decs:
            d._advance(1)

    def chunk(self, tokens):
        for d in self.decs:
            d._check_tokens(tokens)
            d._ensure_prefill_buffers(tokens.shape[1])
            d._make_room(tokens.shape[1])
            d._upload_chunk(tokens)
        self.run([d._build_prefill(tokens.shape[1]) for d in self.decs])
        for d in self.decs:
            d._advance(tokens.shape[1])
        self.run([d._head_stream() for d in self.decs])

    def logits(self):
        a, b = (d.logits() for d in self.decs)
        assert np.array_equal(a, b)
        return a

    def close(self):
        for d in self.decs:
            d.close()


@pytest.mark.parametrize("bounds", [{}, dict(kv_rows=64, kv_budget=40, kv_recent=16)])
def test_sharded_steps_chunks_and_evictions(bounds):
    cfg = DecoderConfig("llama", 256, 200, 256, 4, 2, 384)
    t = Ranks(cfg, 2, **bounds)
    try:
        rng = np.random.default_rng(3)
        models = [Model(t.om, cfg, bounds.get("kv_rows"), bounds.get("kv_budget"), bounds.get("kv_recent")) for _ in range(2)]

        def follow(tokens):
            n = tokens.shape[1]
            for b, m in enumerate(models):
                if bounds and len(m.K[0][0]) + n > 64:               # the ranks' own sums decide, each for its heads
                    for l in range(cfg.n_layers):
                        seen = np.concatenate([d._download(d.ids[f"seen.{l}"], 2 * d.h_local * 64).reshape(2, d.h_local, 64) for d in t.decs], 1)
                        for h in range(cfg.n_heads):
                            m.seen[l][h] = seen[b, h, :len(m.seen[l][h])].astype(np.float64)
            return [m.run(tokens[b]) for b, m in enumerate(models)]

        for n in (24, 1, 20, 1, 1, 24, 1, 1, 9, 1, 24, 1):
            tokens = rng.integers(0, 256, (2, n))
            want = follow(tokens)
            if n == 1:
                t.step(tokens[:, 0])
            else:
                t.chunk(tokens)
            got = t.logits()
            assert all(close(got[b], want[b]) for b in range(2)), n
        assert all(d._rows.tolist() == [len(m.K[0][0]) for m in models] and d.stats()["device_error"] == 0 for d in t.decs)
    finally:
        t.close()
