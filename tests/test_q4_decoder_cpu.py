"""What a decoder over the 4-bit cache keeps about its sequences' rows, without a GPU: the interpreter over a stand-in for the kernels."""
import numpy as np
import pytest

from deepj_b200 import compute_graph as cg
from deepj_b200.decoder import DecoderConfig, Q8Decoder
from q4_standin import box, standin  # noqa: F401

CFG = DecoderConfig("gpt", 64, 200, 64, 2, 1, 96)


@pytest.fixture
def make(box):  # noqa: F811
    made = []

    def decoder(batch=1, **kw):
        d = Q8Decoder(CFG, batch=batch, kv_dtype="q4", id_base=(1 << 24) + (len(made) << 16), **kw)
        made.append(d)
        d.load_synthetic(1, 0.05)
        return d
    yield decoder
    for d in made:
        d.close()


def state(d):
    """Rows as the host counts them, lengths and positions as the device holds them."""
    return d._rows.tolist(), d._download(d.ids["len"], d.B).astype(int).tolist(), d._download(d.ids["pos"], d.B).astype(int).tolist()


def test_rows_and_positions_follow_what_is_fed(make):
    d = make(2)
    d.prefill_packed([[1] * 5, [2] * 40])
    assert state(d) == ([5, 40],) * 3
    d.step([1, 2])
    d.step_device(3)
    assert state(d) == ([9, 44],) * 3 and d.position == 44
    d.prefill([[1] * 33, [2] * 33])
    assert state(d) == ([42, 77],) * 3
    d.reset()
    assert state(d) == ([0, 0],) * 3


def test_no_sequence_is_set_to_rows_it_does_not_have(make):
    d = make(2)
    d.prefill_packed([[1] * 5, [2] * 40])
    for position in (6, 40, 41):
        with pytest.raises(ValueError, match="rows"):
            d.set_position(position)
    assert state(d) == ([5, 40],) * 3 and d.position == 40
    d.set_position(5)
    assert state(d) == ([5, 5],) * 3 and d.position == 5
    d.step([1, 2])
    d.set_position(6)
    assert state(d) == ([6, 6],) * 3
    d.set_position(0)
    with pytest.raises(ValueError, match="rows"):
        d.set_position(1)


def test_a_bounded_cache_is_not_set_back(make):
    """The attention that rows got from tokens behind the position cannot be taken away again, and it decides what is evicted."""
    d = make(2, kv_rows=64, kv_budget=40)
    d.prefill([[1] * 20, [2] * 20])
    for position in (1, 19):
        with pytest.raises(ValueError, match="attention"):
            d.set_position(position)
    d.set_position(20)                                               # where it is
    assert state(d) == ([20, 20],) * 3
    d.set_position(0)
    assert state(d) == ([0, 0],) * 3


def test_steps_that_do_not_fit_are_refused_before_the_first(make):
    d = make(2, kv_rows=48)
    d.prefill_packed([[1] * 40, [2] * 3])
    with pytest.raises(ValueError, match="48 rows"):
        d.step_device(9)
    assert state(d) == ([40, 3],) * 3 and d.position == 40
    d.step_device(8)
    assert state(d) == ([48, 11],) * 3 and d.position == 48
    with pytest.raises(ValueError, match="48 rows"):
        d.step([1, 2])
    assert state(d) == ([48, 11],) * 3


def test_what_did_not_run_is_not_counted(make, monkeypatch):
    """A flush that fails (no memory for the workspace, say) leaves rows and position as they were."""
    d = make(1, kv_rows=64, kv_budget=40)
    d.prefill([[1] * 33])

    def fails(*_):
        raise RuntimeError("out of memory")
    for call in (lambda: d.step([1]), lambda: d.step_device(2), lambda: d.prefill([[1] * 20], chunked=True), lambda: d.prefill_packed([[1] * 20])):
        d._streams()
        d._ensure_prefill_buffers(24)
        with monkeypatch.context() as m:
            m.setattr(d, "lib", Failing(d.lib, fails))
            with pytest.raises(RuntimeError, match="out of memory"):
                call()
        assert state(d) == ([33],) * 3 and d.position == 33


class Failing:
    """A library whose flushes fail."""

    def __init__(self, lib, fails):
        self._real, self.deepj_cuda_flush_ops, self.deepj_cuda_flush_ops_async = lib, fails, fails

    def __getattr__(self, name):
        return getattr(self._real, name)


def evictions(box):  # noqa: F811
    """(sequence, rows it had) of the sequences that the last launches evicted from; one layer."""
    return [(b, n) for kind, b, n, budget in box.launched() if kind == cg.OP_KV_EVICT_Q4 and n > budget]


def test_only_full_sequences_are_evicted_from(make, box):  # noqa: F811
    d = make(3, kv_rows=64, kv_budget=40)
    d.prefill_packed([[1] * 15, [2] * 1, [3] * 24])
    d.prefill_packed([[1] * 24, [2] * 24, [3] * 24])
    d.prefill_packed([[1] * 24, [2] * 20, [3] * 1])
    assert state(d)[0] == [63, 45, 49]
    box.launched()
    d.step([1, 2, 3])
    assert evictions(box) == [] and state(d)[:2] == ([64, 46, 50],) * 2
    d.step([1, 2, 3])
    assert evictions(box) == [(0, 64)] and state(d) == ([41, 47, 51], [41, 47, 51], [65, 47, 51])
    d.prefill_packed([[1] * 2, [2] * 20, [3] * 1])
    assert evictions(box) == [(1, 47)] and state(d)[:2] == ([43, 60, 52],) * 2
    d.prefill([[1] * 10] * 3, chunked=True)                          # fits the first; the others make room
    assert evictions(box) == [(1, 60)] and state(d)[:2] == ([53, 50, 62],) * 2
    d.prefill_packed([[1] * 1, [2] * 30, [3] * 25])                  # passes of 24: the first one's prompt has ended by the second
    assert evictions(box) == [(1, 50), (2, 62), (1, 64), (2, 64)] and state(d)[:2] == ([54, 46, 41],) * 2
    d.step_device(24)
    assert evictions(box) == [(0, 64), (1, 64), (2, 64)] and state(d)[0] == [54, 46, 41]
    with pytest.raises(ValueError, match="evicted"):
        d.set_position(20)


def test_a_refused_chunk_evicts_nothing(make, box):  # noqa: F811
    d = make(2, kv_rows=64, kv_budget=40)
    d.prefill_packed([[1] * 24, [2] * 24])
    d.prefill_packed([[1] * 24, [2] * 1])
    box.launched()
    with pytest.raises(ValueError, match="more tokens"):
        d._make_room(30)
    assert evictions(box) == [] and state(d)[:2] == ([48, 25],) * 2


def test_timing_leaves_what_decides_evictions(make):
    d = make(2, kv_rows=64, kv_budget=40)
    d.prefill_packed([[1] * 5, [2] * 3])
    d.step([1, 2])
    before = d._download(d.ids["seen.0"], 2 * 2 * 64)
    assert before[0] == 1.0 and d.time_ops({"attn"}, iters=4)[1] == 1
    assert np.array_equal(d._download(d.ids["seen.0"], 2 * 2 * 64), before) and state(d)[0] == [6, 4]
    d.step([1, 2])
    assert d._download(d.ids["seen.0"], 1)[0] == 2.0
