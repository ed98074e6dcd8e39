"""Captured calls whose id arrays have to be converted: a replay sees what the arrays hold then."""
import pytest
import torch

import ring_attention as ra

pytestmark = pytest.mark.gpu

KINDS = ["plain", "relative", "dropout"]


def _call(kind, x, table, ids, positions=None):
    fn = ra.segment_bias()
    kw = dict(q_segment_ids=ids), dict(kv_segment_ids=ids)
    if positions is not None:
        fn = ra.causal_bias() + fn
        kw[0]["q_positions"], kw[1]["kv_positions"] = positions, positions
    if kind == "relative":
        fn = fn + ra.relative_bias(table)
    return ra.ring_attention(x, x, x, 2, fn, *kw, dropout=ra.Dropout(0.2, 3) if kind == "dropout" else None)


@pytest.mark.parametrize("dtype", [torch.int64, torch.int32, torch.bool])
@pytest.mark.parametrize("warm,with_positions", [(True, False), (True, True), (False, False)])  # (positions are read on the host, before a capture)
@pytest.mark.parametrize("kind", KINDS)
def test_replays_see_new_ids(device, kind, warm, with_positions, dtype):
    ra.clear_plan_cache()
    x, table = torch.randn(2, 192, 2, 64, device=device).bfloat16(), torch.randn(32, 2, device=device)
    g = torch.Generator().manual_seed(1)
    drawn = [(torch.rand(2, 192, generator=g) < 0.03).to(torch.int64).cumsum(1).to(device) % 2 for _ in range(4)]
    at = torch.arange(192, device=device)[None].expand(2, 192) if with_positions else None
    ids = drawn[0].to(dtype)

    def eager(d):
        return _call(kind, x, table, d.to(dtype), at)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    if warm:
        with torch.cuda.stream(side):
            for _ in range(2):
                _call(kind, x, table, ids, at)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = _call(kind, x, table, ids, at)
    # an eager call beside the graph, before its first replay
    assert torch.equal(_call(kind, x, table, ids, at), eager(drawn[0]))
    for d in drawn:
        ids.copy_(d)
        graph.replay()
        got = held.clone()
        torch.cuda.synchronize()
        assert torch.equal(got, eager(d))
        assert torch.equal(_call(kind, x, table, ids, at), got)
    ra.clear_plan_cache()


def test_replays_see_new_positions_that_a_dense_block_expresses(device):
    """Positions of no order (a dense block per step), and ids, both converted; a callable's arrays are its own."""
    ra.clear_plan_cache()
    x = torch.randn(1, 128, 2, 64, device=device).bfloat16()
    at, ids = torch.arange(128, dtype=torch.int32, device=device)[None].flip(1), torch.zeros(1, 128, dtype=torch.int64, device=device)
    fn = ra.causal_bias() + ra.segment_bias()

    def call(at, ids):
        return ra.ring_attention(x, x, x, 1, fn, dict(q_positions=at, q_segment_ids=ids), dict(kv_positions=at, kv_segment_ids=ids))

    call(at, ids)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = call(at, ids)
    for step in (5, 9, 31):
        at.copy_((torch.arange(128, device=device) * step % 128)[None])
        ids.copy_((torch.arange(128, device=device) % 2)[None])
        graph.replay()
        got = held.clone()
        torch.cuda.synchronize()
        assert torch.equal(got, call(at.clone(), ids.clone()))
    ra.clear_plan_cache()


def test_ids_in_host_memory_stay_what_they_were_at_the_capture(device):
    ra.clear_plan_cache()
    x = torch.randn(1, 128, 2, 64, device=device).bfloat16()
    ids = (torch.arange(128) // 40)[None]
    kw = dict(q_segment_ids=ids), dict(kv_segment_ids=ids)
    want = ra.ring_attention(x, x, x, 1, ra.segment_bias(), *kw)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = ra.ring_attention(x, x, x, 1, ra.segment_bias(), *kw)
    for _ in range(2):
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(held, want)
    ra.clear_plan_cache()
