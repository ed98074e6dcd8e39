"""Calls on a paged cache that a program may make: arguments in other places and layouts, captures, the largest numbers."""
import math

import numpy as np
import pytest
import torch

import ring_attention as ra
from oracle import paged_oracle as R

pytestmark = pytest.mark.gpu
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


def _ints(x):
    return torch.tensor(np.asarray(x), dtype=torch.int32, device="cuda")


def _np(t):
    return t.detach().float().cpu().numpy() if t.is_floating_point() else t.cpu().numpy()


def _normal(*shape, seed=0, dtype=BF16):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    return torch.empty(shape, dtype=dtype, device="cuda").normal_(generator=gen)


@pytest.mark.parametrize("heads,group", [(2, 3), (350, 2), (1025, 1)])
@pytest.mark.parametrize("width", [2, 100])
def test_slopes_on_the_host_are_those_on_the_device(heads, group, width):
    """Up to more than two kernels' arguments of them."""
    k, v, q = _normal(4, 16, heads, 32), _normal(4, 16, heads, 32, seed=1), _normal(2, heads * group, 32, seed=2)
    table, n = torch.randint(0, 4, (2, width), dtype=torch.int32, device="cuda"), _ints([width * 16 - 3, 1])
    slopes = ra.alibi_slopes(heads * group)
    want = ra.paged_attention_with_lse(q, k, v, table, n, bias_fn=ra.alibi_bias(slopes.cuda()))
    plain = ra.paged_attention_with_lse(q, k, v, table, n)
    for host in (slopes, torch.stack((slopes, slopes), 1)[:, 0]):
        got = ra.paged_attention_with_lse(q, k, v, table, n, bias_fn=ra.alibi_bias(host))
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1]) and not torch.equal(got[1], plain[1])
    with pytest.raises(ValueError, match="one for each query head"):
        ra.paged_attention(q, k, v, table, n, bias_fn=ra.alibi_bias(slopes[:1]))


def test_slopes_on_the_host_are_not_waited_for():
    k, v, q = _normal(4, 16, 2, 64), _normal(4, 16, 2, 64, seed=1), _normal(1, 4, 64, seed=2)
    table, n, bias = _ints([[0, 1, 2, 3]]), _ints([60]), ra.alibi_bias(ra.alibi_slopes(4))
    x = _normal(8192, 8192)
    ra.paged_attention(q, k, v, table, n, bias_fn=bias), torch.mm(x, x)
    torch.cuda.synchronize()
    for _ in range(60):  # (some 50 ms of work)
        torch.mm(x, x)
    busy = torch.cuda.Event()
    busy.record()
    ra.paged_attention(q, k, v, table, n, bias_fn=bias)
    assert not busy.query()
    torch.cuda.synchronize()


def test_a_captured_step_with_slopes_on_the_host():
    """Made inside of the capture, as a model does it; the lengths move on between replays, and the program works and waits."""
    k, v, q = _normal(40, 16, 2, 64), _normal(40, 16, 2, 64, seed=1), _normal(2, 4, 64, seed=2)
    table, n = torch.randperm(40, device="cuda").to(torch.int32).view(2, 20), _ints([17, 250])

    def step(where="cpu"):
        return ra.paged_attention_with_lse(q, k, v, table, n, bias_fn=ra.sliding_window_bias(100) + ra.alibi_bias(ra.alibi_slopes(4).to(where)))

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for i in range(6):
        n.add_(3)
        want = step("cuda")
        graph.replay()
        if i % 2:
            torch.cuda.synchronize()
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1]), i


@pytest.mark.parametrize("B,nonsense", [(4, {1: 1 << 30, 2: 1 << 30, 3: 1 << 30}), (6, {1: 1 << 30, 2: (1 << 31) - 1, 3: 1 << 30, 4: 1 << 30}), (5, {0: -(1 << 31), 3: 1 << 30}),
                                        (1000, {500: 1 << 30, 501: 1 << 30, 502: (1 << 31) - 1, 700: -(1 << 31), 998: 1 << 30}),
                                        (4096, {i: (1 << 31) - 1 for i in range(2000, 4096)})])
def test_lengths_that_no_caller_should_ask_for_leave_the_rows_before_them_alone(B, nonsense):
    """Sums of the new tokens pass 31 and 32 bits.  The oracle is asked for lengths beyond what the table and the slots hold, but within reason: the same but for
    where the rows behind begin, which is at most 2^31 - 1."""
    size, width, tokens = 16, 4, 3 * B + 200
    rng = np.random.default_rng(B)
    P = 3 * B
    lengths = rng.integers(0, 30, B).astype(np.int32)
    table, at = np.full((B, width), -1, np.int32), 0
    order = rng.permutation(P).astype(np.int32)
    for b in range(B):
        held = R.n_pages(int(lengths[b]), size)
        table[b, :held] = order[at:at + held]
        at += held
    ring, state = np.roll(order, -at), np.array([0, P - at], np.int32)
    new = (lengths + rng.integers(0, 4, B)).astype(np.int64)
    for b, n in nonsense.items():
        new[b] = n
    t, r = _ints(table), _ints(ring)
    got = ra.page_slots(t, _ints(lengths), _ints(new), r, _ints(state), size, tokens)
    want = R.page_slots(table, lengths, np.clip(new, 0, tokens + 100), ring, state, size, tokens)
    starts = np.minimum(np.concatenate(([0], np.maximum(np.maximum(new, 0) - lengths, 0).cumsum())), (1 << 31) - 1)
    for x, y, name in zip((t, r, *got), want, ("table", "ring", "slots", "starts", "lengths", "state")):
        if name == "lengths":
            y = np.minimum(y, width * size)
        assert np.array_equal(_np(x), starts if name == "starts" else y), name


def test_the_most_slots():
    """2^31 - 1 of them, 17 GB: the last step of a thread's walk over them passes what an int holds."""
    table, ring = torch.full((2, 4), -1, dtype=torch.int32, device="cuda"), torch.arange(9, dtype=torch.int32, device="cuda")
    most = (1 << 31) - 1
    slots, starts, lengths, state = ra.page_slots(table, _ints([0, 0]), _ints([20, 40]), ring, _ints([0, 9]), 16, most)
    assert slots.shape == (most,) and starts.tolist() == [0, 20, 60] and lengths.tolist() == [20, 40] and state.tolist() == [5, 4]
    assert slots[:60].tolist() == [*range(20), *range(32, 72)] and table.tolist() == [[0, 1, -1, -1], [2, 3, 4, -1]]
    assert int(slots[60:].max()) == int(slots[60:].min()) == -1
    with pytest.raises(ValueError, match="num_tokens"):
        ra.page_slots(table, _ints([0, 0]), _ints([20, 40]), ring, _ints([0, 9]), 16, most + 1)


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("width", [40, 500, 1500, 9000])
def test_pages_that_are_not_in_the_pool_take_no_place_of_others(dtype, width):
    """Every score is negative, some are -inf; a third of the entries name no page, the first and the last of a sequence among them."""
    P, H, d = 30, 2, 64
    means = _normal(P, H, d, seed=3, dtype=dtype).abs()
    means[7, 0, 0] = math.inf
    q = -_normal(3, 2 * H, d, seed=4, dtype=dtype).abs() - 0.01
    gen = torch.Generator(device="cuda")
    gen.manual_seed(width)
    table = torch.randint(-P // 2, P, (3, width), generator=gen, device="cuda", dtype=torch.int32)
    table[:, 5], table[0, 0], table[1, width - 1] = P, -1, 1 << 30
    table[2] = -1
    table[2, 3:6] = torch.tensor([4, 2, 7], dtype=torch.int32)  # (fewer than are chosen)
    n = _ints([width * 16, width * 16 - 3, width * 16])
    inside = ((table >= 0) & (table < P)).sum(1)
    for count, first, last in ((2, 1, 1), (12, 0, 0), (int(inside[0]) - 1, 1, 1), (width - 2, 3, 4)):
        got = ra.select_pages(q, means, table, n, 16, count, first, last)
        assert np.array_equal(_np(got), R.select_pages(_np(q), _np(means), _np(table), _np(n), 16, count, first, last))
        there = torch.stack([table[b][got[b].long()] for b in range(3)])
        there = ((there >= 0) & (there < P)).sum(2)
        assert bool((there == inside.clamp(max=count)[:, None]).all())


def test_tangents_are_refused():
    """Operands of forward-mode differentiation ask for no gradient; without a refusal the output has no tangent."""
    fwd = torch.autograd.forward_ad
    k, v, q = _normal(4, 16, 2, 64), _normal(4, 16, 2, 64, seed=1), _normal(1, 4, 64, seed=2)
    table, n, means, slots = _ints([[0, 1, 2, 3]]), _ints([60]), k.mean(1), torch.zeros(1, dtype=torch.int64, device="cuda")
    before = [x.clone() for x in (k, v, means)]
    slopes = ra.alibi_slopes(4)
    with fwd.dual_level():
        def dual(x):
            return fwd.make_dual(x, torch.ones_like(x))

        for call in (lambda: ra.paged_attention(dual(q), k, v, table, n), lambda: ra.paged_attention(q, dual(k), v, table, n),
                     lambda: ra.paged_attention(q, k, dual(v), table, n), lambda: ra.paged_attention(q, k, v, table, n, bias_fn=ra.alibi_bias(dual(slopes))),
                     lambda: ra.paged_attention(q, k, v, table, n, bias_fn=ra.alibi_bias(dual(slopes.cuda()))),
                     lambda: ra.select_pages(dual(q), means, table, n, 16, 2), lambda: ra.select_pages(q, dual(means), table, n, 16, 2),
                     lambda: ra.write_pages(dual(q[:, :2]), q[:, 2:], k, v, slots), lambda: ra.write_pages(q[:, :2], dual(q[:, 2:]), k, v, slots),
                     lambda: ra.write_pages(q[:, :2], q[:, 2:], dual(k), v, slots), lambda: ra.page_means(dual(k), table, n - 1, n, means),
                     lambda: ra.page_means(k, table, n - 1, n, dual(means))):
            with pytest.raises(RuntimeError, match="tangent"):
                call()
            with torch.no_grad(), pytest.raises(RuntimeError, match="tangent"):  # (which leaves forward mode on)
                call()
        ra.paged_attention(q, k, v, table, n)
    assert all(torch.equal(x, y) for x, y in zip(before, (k, v, means)))


def test_tokens_that_lie_in_the_pool_in_another_order():
    """Heads and dimensions of the pool exchanged (as many of both): a copy that keeps the order of dense strides would not do."""
    k, v = _normal(3, 16, 32, 32), _normal(3, 16, 32, 32, seed=1)
    want = [x.flatten(0, 1).transpose(1, 2).contiguous().view_as(x) for x in (k, v)]
    ra.write_pages(k.flatten(0, 1).transpose(1, 2), v.flatten(0, 1).transpose(1, 2), k, v, torch.arange(48, device="cuda"))
    assert torch.equal(k, want[0]) and torch.equal(v, want[1])
    # every second token to the place behind it
    want = [x.clone() for x in (k, v)]
    for x in want:
        x.view(48, 32, 32)[1::2] = x.view(48, 32, 32)[::2]
    ra.write_pages(k.flatten(0, 1)[::2], v.flatten(0, 1)[::2], k, v, torch.arange(1, 48, 2, device="cuda"))
    assert torch.equal(k, want[0]) and torch.equal(v, want[1])


@pytest.mark.parametrize("by", [1, 4, 8])
def test_rows_that_begin_anywhere(by):
    """Contiguous, but not on 16 bytes, as a piece of a larger buffer lies; by 8 it is taken as it is."""
    k, v = _normal(4, 16, 2, 64), _normal(4, 16, 2, 64, seed=1)
    table, n, means = _ints([[0, 1, 2, 3]] * 3), _ints([60, 30, 5]), k.float().mean(1).to(BF16)

    def moved(x):
        at = torch.empty(x.numel() + by, dtype=x.dtype, device="cuda")[by:].view_as(x)
        assert at.copy_(x).is_contiguous()
        return at

    q, pools = _normal(3, 4, 64, seed=2), [(k.clone(), v.clone()) for _ in range(2)]
    slots = torch.tensor([3, 17, 40], device="cuda")
    for kind in (BF16, F32):
        new = [_normal(3, 2, 64, seed=s, dtype=kind) for s in (5, 6)]
        ra.write_pages(*new, *pools[0], slots)
        ra.write_pages(*(moved(x) for x in new), *pools[1], slots)
        assert torch.equal(pools[0][0], pools[1][0]) and torch.equal(pools[0][1], pools[1][1]) and not torch.equal(pools[0][0], k)
    for x, y in zip(ra.paged_attention_with_lse(q, k, v, table, n), ra.paged_attention_with_lse(moved(q), k, v, table, n)):
        assert torch.equal(x, y)
    assert torch.equal(ra.select_pages(q, means, table, n, 16, 2), ra.select_pages(moved(q), means, table, n, 16, 2))


def test_a_step_in_inference_mode():
    """The tensors of such a program have no versions; its results are of the same kind."""
    def step(s):
        slots, _, n, state = ra.page_slots(s["table"], s["n"], s["n"] + 3, s["ring"], s["state"], 16, 6)
        ra.write_pages(s["new"], s["new"] * 2, s["k"], s["v"], slots)
        ra.page_means(s["k"], s["table"], s["n"], n, s["means"])
        pages = ra.select_pages(s["q"], s["means"], s["table"], n, 16, 2)
        return (n, state, pages, *ra.paged_attention_with_lse(s["q"], s["k"], s["v"], s["table"], n, pages=pages, bias_fn=ra.alibi_bias(ra.alibi_slopes(4))))

    def made():
        k = _normal(9, 16, 2, 64)
        return dict(table=_ints([[0, 1, 2, -1], [3, 4, 5, -1]]), n=_ints([40, 47]), ring=_ints([6, 7, 8, 0, 0, 0, 0, 0, 0]), state=_ints([0, 3]), k=k, v=k * 3,
                    means=k.mean(1), new=_normal(6, 2, 64, seed=1), q=_normal(2, 4, 64, seed=2))

    want = made()
    out = step(want)
    with torch.inference_mode():
        got = step(made())
        assert all(x.is_inference() for x in got) and all(torch.equal(x, y) for x, y in zip(got, out))
    held = made()
    with torch.inference_mode():
        got = step(held)
    assert all(torch.equal(x, y) for x, y in zip(got, out)) and all(torch.equal(held[x], want[x]) for x in want)
