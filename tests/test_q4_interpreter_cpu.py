"""What the interpreter does with the ops of the 4-bit cache, without a GPU."""
import pytest

from deepj_b200 import compute_graph as cg
from deepj_b200._lib import check
from q4_standin import box, standin  # noqa: F401


class Step:
    """A projection and a token step over one of two layers, and ops to put in front of them."""

    def __init__(self, box):  # noqa: F811
        self.box = box
        self.kv = box.cache(2, 2, 1, 64, 32)
        self.x, self.out, self.z, self.tab, self.acc = box.zeros(256), box.zeros(256), box.zeros(4), box.zeros(64 * 16), box.zeros(128)
        w = box.id()
        check(box.lib.deepj_cuda_q8_alloc(w, 32, 96))
        self.q8 = [cg.OP_Q8_LINEAR, self.out, 0, 32, -1, 0, w, -1, -1, 0, 0, self.x, 0, 96, 2]
        self.starts = box.buf([0, 1, 2])

    def step(self, layer=0):
        return [cg.OP_ATTN_DECODE_Q4, self.x, 0, 32, 64, 96, self.kv, layer, self.z, self.z, self.tab, self.tab, 64, self.out, 0, 32, 2, 1, -1, -1]

    def writers(self):
        lens = self.box.zeros(2)
        return {"store": [cg.OP_KV_STORE_Q4, self.x, 32, 64, 96, self.kv, 0, self.z, 2, 1],
                "packed": [cg.OP_ATTN_PACKED_Q4, self.x, 0, 32, 64, 96, self.kv, 0, self.starts, self.z, self.z, self.tab, self.tab, 64, self.out, 0, 32, 2, 1, 2, -1, -1, 0],
                "evict": [cg.OP_KV_EVICT_Q4, self.kv, self.kv, 0, self.z, self.acc, 8, 2, 2, self.acc, lens, -1],
                "step": self.step(0)}

    def idle(self):
        """Ops that launch nothing."""
        return {"copy": [cg.OP_COPY, self.x, 0, self.out, 0, 0], "add": [cg.OP_ADD, self.x, self.x, self.x, 0], "scalar": [cg.OP_ADD_SCALAR_INPLACE, self.z, 0, 0],
                "load": [cg.OP_KV_LOAD_Q4, self.kv, 1, -1, -1, 0, self.x, self.out, 2]}

    def early(self, *words):
        """Whether the last step of a stream may read cached rows before it has waited."""
        self.box.launched()
        self.box.flush(*words)
        return [n[1] for n in self.box.launched() if n[0] == cg.OP_ATTN_DECODE_Q4][-1]


def test_a_step_behind_projections_reads_its_pages_early(box):  # noqa: F811
    t = Step(box)
    copy = [cg.OP_COPY, t.x, 0, t.out, 0, 8]
    assert t.early(*copy, *t.q8, *t.step()) == 1
    assert t.early(*copy, *t.q8, *t.q8, *t.step()) == 1
    assert t.early(*t.step(1), *t.q8, *t.step(0)) == 1               # another layer's rows
    for w in t.writers().values():
        assert t.early(*w, *copy, *t.q8, *t.step()) == 1             # the copy has waited for the writer
    assert t.early(*copy, *t.step()) == 0                            # nothing to overlap with
    assert t.early(*t.q8, *t.step()) == 0                            # what ran before the stream is not known


@pytest.mark.parametrize("writer", ["store", "packed", "evict", "step"])
def test_a_step_waits_for_the_op_that_writes_its_rows(box, writer):  # noqa: F811
    t = Step(box)
    w = t.writers()[writer]
    assert t.early(*w, *t.q8, *t.step()) == 0
    for idle in t.idle().values():                                   # an op that launches nothing has not waited for anything
        assert t.early(*w, *idle, *t.q8, *t.step()) == 0
        assert t.early(*w, *idle, *idle, *t.q8, *t.q8, *t.step()) == 0
        assert t.early(*w, *t.q8, *idle, *t.step()) == 0
        t.box.flush(*w)
        assert t.early(*idle, *t.q8, *t.step()) == 0                 # nor when the writer ran in the stream before


# ───────────── outputs among the inputs ─────────────

def refused(box, words, at, value, match="another buffer"):  # noqa: F811
    words = list(words)
    words[at] = value
    box.launched()
    with pytest.raises(RuntimeError, match=match):
        box.flush(*words)
    assert box.launched() == []


@pytest.mark.parametrize("packed", [False, True])
def test_attention_writes_to_none_of_its_inputs(box, packed):  # noqa: F811
    t = Step(box)
    words, e = (t.writers()["packed"], 1) if packed else (t.step(), 0)
    old, new, pos = box.zeros(128), box.zeros(128), box.zeros(4)
    words[9 + e], words[11 + e] = pos, box.zeros(64 * 16)            # every input a buffer of its own
    words[-3:] = [old, new, 1] if packed else words[-3:-2] + [old, new]
    box.flush(*words)
    acc, acc_out = (20, 21) if packed else (18, 19)
    inputs = [1] + ([8] if packed else []) + [8 + e, 9 + e, 10 + e, 11 + e]
    big = {i: box.zeros(64 * 16) for i in inputs}                    # large enough for what is written
    for i in inputs:
        words[i] = big[i]
    box.flush(*words)
    for i in inputs:
        refused(box, words, 13 + e, big[i])
        refused(box, words, acc_out, big[i])
    refused(box, words, 13 + e, old)
    refused(box, words, 13 + e, new)
    refused(box, words, acc_out, words[13 + e])
    words[acc_out] = old                                             # added up in place
    box.flush(*words)
    assert acc == acc_out - 1 and words[acc] == old


def test_eviction_writes_to_none_of_its_inputs(box):  # noqa: F811
    kv, small = box.cache(1, 2, 1, 64, 32), box.cache(1, 2, 1, 16, 32)
    n, acc, new, n_out, kept = (box.zeros(512) for _ in range(5))
    words = [cg.OP_KV_EVICT_Q4, kv, small, 0, n, acc, 8, 2, 2, new, n_out, kept]
    box.flush(*words)
    for at, others in ((9, (n, n_out, kept)), (10, (n, acc, new, kept)), (11, (n, acc, new, n_out))):
        for other in others:
            refused(box, words, at, other)
    words[2], words[9] = kv, acc                                     # in place
    box.flush(*words)


def test_a_row_load_writes_to_none_of_its_inputs(box):  # noqa: F811
    kv = box.cache(1, 2, 1, 64, 32)
    at, end, k, v = (box.zeros(512) for _ in range(4))
    words = [cg.OP_KV_LOAD_Q4, kv, 0, at, end, 4, k, v, 2]
    box.flush(*words)
    for slot in (6, 7):
        refused(box, words, slot, at)
        refused(box, words, slot, end)
    words[3] = words[4] = -1
    box.flush(*words)
