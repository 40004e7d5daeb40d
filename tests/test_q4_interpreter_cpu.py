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
