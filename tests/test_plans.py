"""Plans: positions given as an int, that of the first token, beside positions that only a dense block expresses; calls of several threads."""
import collections

import pytest
import torch

import ring_attention as ra
from ring_attention import ring as rr


@pytest.mark.parametrize("n", [1, 2])
@pytest.mark.parametrize("bias", [ra.causal_bias(), ra.sliding_window_bias(3), ra.alibi_bias([0.5, 0.25, 1.0]), ra.causal_bias() + ra.segment_bias()])
def test_int_on_one_side_and_arbitrary_positions_on_the_other(n, bias):
    q, k = torch.zeros(2, 4, 3, 64), torch.zeros(2, 8, 3, 64)
    padded = torch.tensor([[0, 0, 0, 1, 2, 3, 4, 5], [0, 0, 1, 2, 3, 4, 5, 6]])  # sequences behind padding
    ids = dict(q_segment_ids=torch.ones(2, 4), kv_segment_ids=torch.ones(2, 8)) if bias.segments else {}

    def blocks(q_positions, kv_positions):
        plan = rr._RingPlan(q, k, n, bias, {"q_positions": q_positions, **{a: x for a, x in ids.items() if a[0] == "q"}},
                            {"kv_positions": kv_positions, **{a: x for a, x in ids.items() if a[0] == "k"}})
        assert plan.callable is not None
        return [plan.block_bias(r, s).dense for r in range(n) for s in range(n)]

    at = (2 + torch.arange(4))[None].expand(2, 4)
    for got, want in zip(blocks(2, padded), blocks(at, padded)):
        assert torch.equal(got, want) and torch.isfinite(got).any()
    backward = at.flip(1)
    for got, want in zip(blocks(backward, 3), blocks(backward, (3 + torch.arange(8))[None].expand(2, 8))):
        assert torch.equal(got, want)


def test_int_out_of_range_beside_arbitrary_positions():
    q = torch.zeros(1, 4, 2, 64)
    with pytest.raises(ValueError, match="positions must lie"):
        rr._RingPlan(q, q, 1, ra.causal_bias(), {"q_positions": -1}, {"kv_positions": torch.tensor([[3, 1, 2, 0]])})


@pytest.mark.parametrize("kind", ["relative", "dropout"])
def test_arbitrary_positions_beside_an_int_stay_refused_where_one_launch_runs(kind):
    q, k = torch.zeros(1, 4, 2, 64), torch.zeros(1, 8, 2, 64)
    fn = ra.causal_bias() + ra.relative_bias(torch.zeros(32, 2)) if kind == "relative" else ra.causal_bias()
    with pytest.raises(ValueError, match="follow on"):
        rr._RingPlan(q, k, 1, fn, {"q_positions": 4}, {"kv_positions": torch.tensor([[0, 0, 1, 2, 3, 4, 5, 6]])}).single()


def test_a_plan_that_another_thread_puts_out_while_it_is_taken(monkeypatch):
    class Shared(collections.OrderedDict):
        def get(self, key, default=None):
            got = super().get(key, default)
            self.clear()  # what other threads' calls do between two statements of this one
            return got

    monkeypatch.setattr(rr, "_PLAN_CACHE", Shared())
    q = torch.zeros(1, 4, 2, 64)
    plan = rr._plan_for(q, q, 1, ra.causal_bias(), None, None)
    assert rr._plan_for(q, q, 1, ra.causal_bias(), None, None) is plan


def test_arrays_that_are_read_in_place_and_copies():
    q = torch.zeros(2, 8, 2, 64)
    ids = torch.zeros(2, 8, dtype=torch.int32)

    def made(q_ids, kv_ids):
        return rr._RingPlan(q, q, 2, ra.segment_bias(), {"q_segment_ids": q_ids}, {"kv_segment_ids": kv_ids}).made

    assert not made(ids, ids) and made(ids.long(), ids) and made(ids, ids.bool()) and made(ids, ids[:1].expand(2, 8))
    plan = rr._RingPlan(q, q, 2, ra.segment_bias(), {"q_segment_ids": ids.long()}, {"kv_segment_ids": ids})
    later = ids.long() + 3
    again = plan.laid_again({"q_segment_ids": later}, {"kv_segment_ids": ids})
    assert (again.q_seg == 3).all() and again.kv_seg is ids and (plan.q_seg == 0).all()
    assert again.joined().n == plan.joined().n and again.fn is plan.fn
