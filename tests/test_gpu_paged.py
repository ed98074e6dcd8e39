"""The paged cache on the GPU against the oracle in 64 bits: slots, writes, mean keys, chosen pages, attention; and as a program runs them together."""
import math
import threading

import numpy as np
import pytest
import torch

import ring_attention as ra
from oracle import paged_oracle as R
from oracle import ring_oracle

pytestmark = pytest.mark.gpu
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32
HALF_STEP = {BF16: 2.0 ** -8, F16: 2.0 ** -11}


def _ints(x, device="cuda"):
    return torch.tensor(np.asarray(x), dtype=torch.int32, device=device)


def _np(t):
    return t.detach().float().cpu().numpy() if t.is_floating_point() else t.cpu().numpy()


class Cache:
    """A pool whose unused places hold NaN, and a table whose unused entries hold nonsense."""

    def __init__(self, lengths, heads, d, size, dtype, seed=0, layout="tokens", spare=3, extra_width=2):
        rng = np.random.default_rng(seed)
        self.lengths = list(lengths)
        held = [R.n_pages(n, size) for n in lengths]
        P = sum(held) + spare
        shape = (P, size, heads, d)
        if layout == "heads":  # [pages, heads, page_size, d] in memory
            k, v = (torch.full((P, heads, size, d), math.nan, dtype=dtype, device="cuda").transpose(1, 2) for _ in range(2))
        elif layout == "both":  # keys and values side by side, rows padded
            kv = torch.full((P, size, 2, heads, d + 8), math.nan, dtype=dtype, device="cuda")
            k, v = kv[:, :, 0, :, :d], kv[:, :, 1, :, :d]
        else:
            k, v = (torch.full(shape, math.nan, dtype=dtype, device="cuda") for _ in range(2))
        self.k, self.v = k, v
        order = rng.permutation(P)
        width = max(max(held), 1) + extra_width
        table = np.where(np.arange(width)[None] % 2 == 0, -7, 1 << 30) * np.ones((len(lengths), 1), np.int64)
        at = 0
        gen = torch.Generator(device="cuda")
        gen.manual_seed(seed)
        for b, n in enumerate(held):
            table[b, :n] = order[at:at + n]
            for j in range(n):
                here = min(size, lengths[b] - j * size)
                for x in (k, v):
                    x[int(order[at + j]), :here] = torch.empty((here, heads, d), dtype=dtype, device="cuda").normal_(generator=gen)
            at += n
        self.table = _ints(table)
        self.n = _ints(self.lengths)
        self.gen = gen

    def queries(self, heads, scale=1.0):
        d = self.k.shape[3]
        return torch.empty((len(self.lengths), heads, d), dtype=self.k.dtype, device="cuda").normal_(0, scale, generator=self.gen)


def _check_attention(q, cache, got, scale, **kw):
    """Half a step for the output; the weights go in as two numbers of the type, off by half a step of half a step (and 2^-25, fp16's least, of a weight of
    2^15); scores are sums of d products in 32 bits, off by 2^-24 (d + 8) of the sum of their sizes
    (scale, exponential and their rounding counted in), which a weight and the sum of weights feel each, in base 2."""
    out, lse = got
    want, want_lse, weight, spread = R.attention(_np(q), _np(cache.k), _np(cache.v), _np(cache.table), _np(cache.n), scale, **kw)
    d, step = q.shape[2], HALF_STEP[q.dtype]
    longest = max(int(cache.n.max()), 1)
    score = 2.0 ** -24 * (2 * (d + 8) * spread + longest + 32)
    tol = (2 * step * step + 2 * score)[..., None] * weight + step * np.abs(want) + 2.0 ** -24
    err = np.abs(_np(out).astype(np.float64) - want)
    assert np.isfinite(_np(out)).all()
    assert (err <= tol).all(), (err - tol).max()
    empty = ~np.isfinite(want_lse)
    assert (_np(lse)[empty] == -np.inf).all() and (_np(out)[empty] == 0).all()
    err = np.abs(_np(lse)[~empty] - want_lse[~empty])
    assert (err <= score[~empty] + 2.0 ** -22 * np.abs(want_lse[~empty])).all(), err.max()


EDGES = [0, 1, 2, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 128, 129, 255, 257, 1000]


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("d", [32, 64, 96, 128])
@pytest.mark.parametrize("heads,group", [(1, 1), (2, 3), (4, 1), (1, 16), (2, 17), (1, 40)])
@pytest.mark.parametrize("columns", [0, 20])
def test_attention_at_every_edge(dtype, d, heads, group, columns):
    """Narrow tables, whose rows a workgroup takes whole, and wider ones, whose rows are shared."""
    size = {1: 16, 2: 64, 4: 128}[heads]
    c = Cache([n for n in EDGES if columns or n * d < 65000], heads, d, size, dtype, seed=d + group, extra_width=columns)
    q = c.queries(heads * group)
    scale = 1 / math.sqrt(d)
    _check_attention(q, c, ra.paged_attention_with_lse(q, c.k, c.v, c.table, c.n), scale)


def test_many_short_rows():
    """A table of 1024 tokens of D = 128 is taken whole where there are many rows."""
    rng = np.random.default_rng(18)
    c = Cache([int(n) for n in rng.integers(0, 1025, 70)], 2, 128, 16, BF16, seed=18, extra_width=0)
    q = c.queries(4)
    _check_attention(q, c, ra.paged_attention_with_lse(q, c.k, c.v, c.table, c.n), 128 ** -0.5)


@pytest.mark.parametrize("layout", ["tokens", "heads", "both"])
@pytest.mark.parametrize("size", [16, 32, 256, 1024])
def test_attention_over_layouts_and_page_sizes(layout, size):
    c = Cache([700, 1, 0, 2049], 3, 64, size, BF16, seed=size, layout=layout)
    wide = torch.empty((4, 6, 3, 64), dtype=BF16, device="cuda").normal_(generator=c.gen)
    for q in (wide[:, :, 1], wide[:, ::2, 0], wide.transpose(2, 3)[:, :, :, 2]):  # padded rows, every other head, no contiguous dimension
        got = ra.paged_attention_with_lse(q, c.k, c.v, c.table, c.n, sm_scale=0.3)
        _check_attention(q, c, got, 0.3)


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("window", [0, 1, 31, 32, 100, 1000, 1 << 40])
@pytest.mark.parametrize("alibi", [False, True])
def test_windows_and_alibi(dtype, window, alibi):
    c = Cache([0, 1, 30, 33, 130, 999, 1300], 2, 96, 32, dtype, seed=window % 97)
    q = c.queries(6)
    bias, slopes = ra.causal_bias(), None
    if window:
        bias = bias + ra.sliding_window_bias(window)
    if alibi:
        slopes = ra.alibi_slopes(6)
        bias = bias + ra.alibi_bias(slopes)
    got = ra.paged_attention_with_lse(q, c.k, c.v, c.table, c.n, bias_fn=bias)
    _check_attention(q, c, got, 96 ** -0.5, window=min(window, 1 << 20), slopes=slopes)


@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
def test_masked_places_may_hold_anything(bad):
    """Behind a sequence's end (Cache fills NaN), before its window, in pages that are not chosen."""
    c = Cache([400, 77], 2, 64, 32, BF16, seed=1)
    q = c.queries(4)
    clean = ra.paged_attention_with_lse(q, c.k, c.v, c.table, c.n, bias_fn=ra.sliding_window_bias(50))
    pages = _ints([[[0, 12, -1], [3, 5, 12]], [[1, 2, -1], [2, 99, -1]]])
    clean_pages = ra.paged_attention_with_lse(q, c.k, c.v, c.table, c.n, pages=pages)
    _check_attention(q, c, clean_pages, 0.125, pages=_np(pages))
    table = _np(c.table)
    dirty = Cache([400, 77], 2, 64, 32, BF16, seed=1)
    for x in (dirty.k, dirty.v):
        x[int(table[0, 10]), :30] = bad  # up to 350
        x[int(table[1, 0]), :27] = bad   # up to 27
    for a, b in zip(clean, ra.paged_attention_with_lse(q, dirty.k, dirty.v, c.table, c.n, bias_fn=ra.sliding_window_bias(50))):
        assert torch.equal(a, b)
    for a, b in zip(clean_pages, ra.paged_attention_with_lse(q, dirty.k, dirty.v, c.table, c.n, pages=pages)):
        assert torch.equal(a, b)


def test_scores_that_are_not_finite():
    """A query or a key that is not a number makes its own row one; a key whose score is -inf has no weight; a row of such keys has none."""
    c = Cache([200, 200, 200, 40], 1, 64, 16, BF16, seed=2)
    q = c.queries(2).abs() + 0.5
    q[0, 0, 5] = math.nan
    table = _np(c.table)
    c.k[int(table[1, 3]), 4, 0, 7] = math.nan
    c.k[int(table[2, 3]), 4, 0] = -math.inf
    for j in range(3):
        c.k[int(table[3, j])] = -math.inf
    out, lse = ra.paged_attention_with_lse(q, c.k, c.v, c.table, c.n)
    assert out[0, 0].isnan().all() and lse[0, 0].isnan() and out[1].isnan().all() and lse[1].isnan().all()
    assert out[0, 1].isfinite().all() and out[2].isfinite().all() and lse[2].isfinite().all()
    assert (out[3] == 0).all() and (lse[3] == -math.inf).all()


def test_pages_that_are_not_in_the_pool_take_no_part():
    c = Cache([300, 64], 2, 64, 16, F16, seed=3)
    c.table[0, 3], c.table[0, 4], c.table[1, 0] = -1, c.k.shape[0], 1 << 30
    q = c.queries(2)
    _check_attention(q, c, ra.paged_attention_with_lse(q, c.k, c.v, c.table, c.n), 0.125)
    c.table[1, :4] = -5
    _check_attention(q, c, ra.paged_attention_with_lse(q, c.k, c.v, c.table, c.n), 0.125)


def test_lengths_are_cut_to_the_table():
    c = Cache([64, 64], 2, 64, 16, BF16, seed=4, extra_width=0)
    q = c.queries(2)
    want = ra.paged_attention_with_lse(q, c.k, c.v, c.table, c.n)
    got = ra.paged_attention_with_lse(q, c.k, c.v, c.table, _ints([1 << 30, 64]))
    assert torch.equal(want[0], got[0]) and torch.equal(want[1], got[1])
    out, lse = ra.paged_attention_with_lse(q, c.k, c.v, c.table, _ints([-3, 64]))
    assert (out[0] == 0).all() and (lse[0] == -math.inf).all() and torch.equal(out[1], want[0][1])


@pytest.mark.parametrize("dtype,heads,group,d,lengths", [
    (BF16, 1, 1, 128, [70001]),              # one sequence over all workgroups
    (F16, 2, 4, 64, [33000, 5, 0, 12345]),
    (BF16, 1, 20, 32, [1, 20000, 1, 1]),
])
def test_long_sequences_are_shared_between_workgroups(dtype, heads, group, d, lengths):
    c = Cache(lengths, heads, d, 128, dtype, seed=5)
    q = c.queries(heads * group, 2.0)
    _check_attention(q, c, ra.paged_attention_with_lse(q, c.k, c.v, c.table, c.n), d ** -0.5)


def test_stretches_of_more_pages_than_shared_memory_holds():
    """2 x 2^20 tokens of 8 heads in pages of 16: a workgroup walks more than a thousand pages.  The pages of a few are named again and again."""
    P, width, H, d = 61, 1 << 16, 8, 32
    gen = torch.Generator(device="cuda")
    gen.manual_seed(6)
    k, v = (torch.empty((P, 16, H, d), dtype=BF16, device="cuda").normal_(generator=gen) for _ in range(2))
    q = torch.empty((2, H, d), dtype=BF16, device="cuda").normal_(generator=gen)
    table = torch.randint(0, P, (2, width), generator=gen, device="cuda", dtype=torch.int32)
    n = _ints([width * 16 - 5, width * 16 - 16 * 300])
    out, lse = ra.paged_attention_with_lse(q, k, v, table, n)
    for b in range(2):
        pages = table[b, :R.n_pages(int(n[b]), 16)].long()
        for h in range(H):
            s = torch.matmul(k[pages, :, h].double().reshape(-1, d)[:int(n[b])], q[b, h].double()) * d ** -0.5
            w = torch.softmax(s, 0)
            x = v[pages, :, h].double().reshape(-1, d)[:int(n[b])]
            want, size = (w[:, None] * x).sum(0), (w[:, None] * x.abs()).sum(0)
            # sums of 2^20 weights: in 32 bits over at most 2^11 at a time in a lane, then over lanes and parts
            tol = (2.0 ** -15 + 2.0 ** -24 * 2 ** 13) * size + 2.0 ** -8 * want.abs()
            assert ((out[b, h].double() - want).abs() <= tol).all()
            assert abs(float(lse[b, h]) - float(torch.logsumexp(s, 0))) <= 2.0 ** -24 * 2 ** 13


def test_the_longest_sequence():
    """2^30 tokens, pages named again and again, and one that is not in the pool: the pool's first page, which must not stand in for it, holds NaN."""
    k, v = torch.zeros((5, 64, 1, 32), dtype=BF16, device="cuda"), torch.ones((5, 64, 1, 32), dtype=BF16, device="cuda")
    k[0], v[0] = math.nan, math.nan
    table = torch.randint(1, 5, (1, 1 << 24), device="cuda", dtype=torch.int32)
    table[0, -3] = -1
    q = torch.ones((1, 1, 32), dtype=BF16, device="cuda")
    out, lse = ra.paged_attention_with_lse(q, k, v, table, _ints([1 << 30]))
    # equal weights: sums of whole numbers, of 2^30 in the end, in 32 bits
    assert bool((out == 1).all()) and abs(float(lse) - math.log(2.0 ** 30 - 64)) <= 2.0 ** -22 * 21


def test_small_weights_beside_a_large_one():
    """fp16: 60000 keys of 2^-20 of the largest weight each make up 5 percent of the output."""
    n, d = 60001, 64
    c = Cache([n], 1, d, 64, F16, seed=7)
    pages = c.table[0, :R.n_pages(n, 64)].long()
    c.k[pages] = 0
    c.k[pages[5], 3, 0, 0] = 20 * math.log(2) * math.sqrt(d) / 2
    c.v[pages] = 1.0
    c.v[pages[5], 3] = 0.0
    q = torch.zeros((1, 1, d), dtype=F16, device="cuda")
    q[0, 0, 0] = 2.0
    top = float(c.k[pages[5], 3, 0, 0].double()) * 2 / math.sqrt(d)
    share = (n - 1) / (n - 1 + math.exp(top))
    out = ra.paged_attention(q, c.k, c.v, c.table, c.n).double()
    assert share > 0.05 and ((out - share).abs() <= share * (2.0 ** -11 + 2.0 ** -21 + 2.0 ** -24 * 70000)).all()


def test_offsets_beyond_32_bits():
    """Pages 2^31 elements apart: 4 GB each way."""
    apart, H, d, size = 1 << 31, 2, 64, 16
    store = torch.empty(2 * apart + 2 * size * H * d, dtype=BF16, device="cuda")
    shape, strides = (3, size, H, d), (apart, H * d, d, 1)
    k, v = store.as_strided(shape, strides), store.as_strided(shape, strides, size * H * d)
    gen = torch.Generator(device="cuda")
    gen.manual_seed(8)
    new_k, new_v = (torch.empty((40, H, d), dtype=BF16, device="cuda").normal_(generator=gen) for _ in range(2))
    table, n = _ints([[2, 0, 1]]), _ints([40])
    token = torch.arange(40, device="cuda")
    slots = table[0].long()[token // size] * size + token % size
    ra.write_pages(new_k, new_v, k, v, slots)
    small_k, small_v = (torch.full(shape, math.nan, dtype=BF16, device="cuda") for _ in range(2))
    ra.write_pages(new_k, new_v, small_k, small_v, slots)
    means = [torch.zeros((3, H, d), dtype=BF16, device="cuda") for _ in range(2)]
    ra.page_means(k, table, _ints([0]), n, means[0])
    ra.page_means(small_k, table, _ints([0]), n, means[1])
    assert torch.equal(means[0], means[1]) and bool((means[0] != 0).any())
    q = torch.empty((1, H, d), dtype=BF16, device="cuda").normal_(generator=gen)
    got, want = (ra.paged_attention_with_lse(q, a, b, table, n) for a, b in ((k, v), (small_k, small_v)))
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1]) and bool(got[0].isfinite().all())


# ---------------------------------------------------------------------------------------
# slots
# ---------------------------------------------------------------------------------------
def _slots_agree(table, lengths, new, ring, state, size, tokens):
    t, r = _ints(table), _ints(ring)
    got = ra.page_slots(t, _ints(lengths), _ints(new), r, _ints(state), size, tokens)
    want = R.page_slots(table, lengths, new, ring, state, size, tokens)
    for x, y, name in zip((t, r, *got), want, ("table", "ring", "slots", "starts", "lengths", "state")):
        assert np.array_equal(_np(x), y), name
    return want


@pytest.mark.parametrize("B,P,width,size", [(1, 5, 4, 16), (7, 60, 16, 16), (64, 500, 33, 32), (300, 1000, 9, 16), (1000, 20000, 70, 16), (4096, 9000, 5, 64)])
def test_slots_over_a_server_s_life(B, P, width, size):
    """Step after step: sequences come, grow, wait, shrink and end, and now and then there are not enough pages."""
    rng = np.random.default_rng(B)
    table, ring, state = np.full((B, width), -1, np.int32), rng.permutation(P).astype(np.int32), np.array([P // 3, P], np.int32)
    lengths = np.zeros(B, np.int32)
    for step in range(8):
        kind = rng.random(B)
        new = lengths + (kind < 0.5)
        new = np.where((kind > 0.5) & (kind < 0.6), lengths + rng.integers(0, width * size, B), new)
        new = np.where((kind > 0.7) & (kind < 0.8), lengths // 2, new)
        new = np.where(kind > 0.9, 0, new)
        new = np.minimum(new, width * size + (3 if step == 5 else 0)).astype(np.int32)  # (and once beyond the table)
        tokens = int(np.maximum(new - lengths, 0).sum())
        tokens = (tokens, tokens + 77, max(tokens - 10, 0))[step % 3]
        table, ring, _, _, lengths, state = _slots_agree(table, lengths, new, ring, state, size, tokens)


def test_slots_refuse_and_survive_nonsense():
    table, ring = torch.full((2, 4), -1, dtype=torch.int32, device="cuda"), torch.arange(6, dtype=torch.int32, device="cuda")
    n, state = _ints([0, 0]), _ints([0, 6])
    # numbers that no caller should pass stay within the arrays
    got = ra.page_slots(table, _ints([-5, 1 << 30]), _ints([40, 1 << 30]), ring, _ints([-9, 1 << 30]), 16, 100)
    assert int(got[2].max()) <= 64 and int(got[0].max()) < 96
    for bad in (lambda: ra.page_slots(table.long(), n, n, ring, state, 16, 1), lambda: ra.page_slots(table, n.long(), n, ring, state, 16, 1),
                lambda: ra.page_slots(table, n[:1], n, ring, state, 16, 1), lambda: ra.page_slots(table, n, n, ring, _ints([0]), 16, 1),
                lambda: ra.page_slots(table, n, n, ring[::2], state, 16, 1), lambda: ra.page_slots(table.t(), n, n, ring, state, 16, 1),
                lambda: ra.page_slots(table, n, n, ring, state, 16, -1), lambda: ra.page_slots(table, n.cpu(), n, ring, state, 16, 1),
                lambda: ra.page_slots(table[:1].expand(2, 4), n, n, ring, state, 16, 1)):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(RuntimeError, match="power of two"):
        ra.page_slots(table, n, n, ring, state, 24, 1)


# ---------------------------------------------------------------------------------------
# writes and means
# ---------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("source", [BF16, F16, F32])
@pytest.mark.parametrize("heads,d,layout", [(1, 32, "tokens"), (3, 96, "heads"), (8, 128, "both"), (5, 64, "tokens")])
def test_writes_go_to_their_slots_and_nowhere_else(dtype, source, heads, d, layout):
    c = Cache([1], heads, d, 32, dtype, layout=layout, spare=6)
    P = c.k.shape[0]
    gen = torch.Generator(device="cuda")
    gen.manual_seed(9)
    for x in (c.k, c.v):
        x.copy_(torch.empty(x.shape, device="cuda").normal_(generator=gen))
    wide = torch.empty((70, 3, heads, d + 4), dtype=source, device="cuda").normal_(0, 3, generator=gen)
    new = [wide[:, 0, :, 4:], wide[:, 2, :, :d]]  # the first with rows that are not aligned
    slots = torch.randperm(P * 32, generator=gen, device="cuda")[:70]
    slots[3], slots[10], slots[11] = -1, P * 32, 1 << 40
    want = [x.clone() for x in (c.k, c.v)]
    for t in range(70):
        if 0 <= int(slots[t]) < P * 32:
            for x, y in zip(want, new):
                x[int(slots[t]) // 32, int(slots[t]) % 32] = y[t].to(dtype)
    version = c.k._version
    ra.write_pages(*new, c.k, c.v, slots)
    assert torch.equal(c.k, want[0]) and torch.equal(c.v, want[1]) and c.k._version > version
    ra.write_pages(new[0][:0], new[1][:0], c.k, c.v, slots[:0])
    assert torch.equal(c.k, want[0])


def test_tokens_that_lie_in_the_pool_are_read_first():
    """Tokens moved within the pool, each to the place of the next."""
    c = Cache([320], 2, 64, 16, BF16, seed=17, spare=0)
    k, v = (x.clone().flatten(0, 1) for x in (c.k, c.v))
    at = torch.arange(320, device="cuda")
    ra.write_pages(c.k.flatten(0, 1), c.v.flatten(0, 1), c.k, c.v, (at + 1) % 320)
    assert torch.equal(c.k.flatten(0, 1), k.roll(1, 0)) and torch.equal(c.v.flatten(0, 1), v.roll(1, 0))


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("heads,d,size", [(1, 32, 16), (3, 96, 32), (8, 128, 16), (2, 64, 128), (40, 128, 16)])
def test_means_of_the_pages_that_change(dtype, heads, d, size):
    before = [0, 0, 5, size, size - 1, 3 * size + 1, 4 * size, 2 * size + 3, 100, 7]
    after = [0, 2 * size + 1, 6, size + 1, size, 6 * size, 2 * size + 5, 0, 100, size + 7]
    c = Cache([max(x, y) for x, y in zip(before, after)], heads, d, size, dtype, seed=10)
    P = c.k.shape[0]
    means = torch.full((P, heads, d + 8), 7.0, dtype=dtype, device="cuda")[:, :, :d]
    ra.page_means(c.k, c.table, _ints(before), _ints(after), means)
    want = R.page_means(_np(c.k), _np(c.table), before, after, size)
    got = _np(means).astype(np.float64)
    for page in range(P):
        if page not in want:
            assert (got[page] == 7.0).all(), page
            continue
        # one rounding, and sums of up to `size` numbers of at most 6 in 32 bits
        assert (np.abs(got[page] - want[page]) <= HALF_STEP[dtype] * np.abs(want[page]) + 2.0 ** -24 * 6 * size + 2.0 ** -25).all(), page


# ---------------------------------------------------------------------------------------
# chosen pages
# ---------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("d,heads,group", [(32, 1, 1), (64, 2, 4), (96, 3, 5), (128, 2, 1)])
@pytest.mark.parametrize("count,first,last", [(2, 1, 1), (9, 1, 1), (64, 0, 0), (5, 2, 3), (200, 1, 1)])
def test_chosen_pages(dtype, d, heads, group, count, first, last):
    size = 16
    # (a table of up to 512 pages is one kernel's, one of up to 2048 and of 4096 others')
    longest = {2: 500 * 16, 9: 17 * 1024, 64: 3000 * 16, 5: 512 * 16 - 40, 200: 5000 * 16}[count]
    c = Cache([0, 1, 32, 33, 1000, 2500, longest], heads, d, size, dtype, seed=11)
    gen = c.gen
    means = torch.empty((c.k.shape[0], heads, d), dtype=dtype, device="cuda").normal_(generator=gen)
    q = c.queries(heads * group)
    got = ra.select_pages(q, means, c.table, c.n, size, count, first, last)
    want = R.select_pages(_np(q), _np(means), _np(c.table), c.lengths, size, count, first, last)
    assert np.array_equal(_np(got), want)


@pytest.mark.parametrize("width", [400, 5000, 20000])
def test_equal_scores_go_to_the_lowest_page(width):
    """Few different means over many pages (of 20000 the numbers do not stay in registers), means of zero of either sign, one that is not a number."""
    P, H, d = 12, 2, 64
    gen = torch.Generator(device="cuda")
    gen.manual_seed(12)
    means = torch.randint(-1, 2, (P, H, d), generator=gen, device="cuda").to(BF16)
    means[3], means[4] = 0.0, -0.0
    q = torch.randint(-2, 3, (2, H, d), generator=gen, device="cuda").to(BF16)
    table = torch.randint(0, P, (2, width), generator=gen, device="cuda", dtype=torch.int32)
    n = _ints([width * 16, 1111])
    for count in (3, 300, 1500, width - 1):
        got = ra.select_pages(q, means, table, n, 16, count)
        assert np.array_equal(_np(got), R.select_pages(_np(q), _np(means), _np(table), _np(n), 16, count))
    means[5, 0, 0] = math.nan
    got = ra.select_pages(q, means, table, n, 16, 300)
    assert np.array_equal(_np(got), R.select_pages(_np(q), _np(means), _np(table), _np(n), 16, 300))
    means[:] = 1.0  # all equal
    assert _np(ra.select_pages(q, means, table, n, 16, 9)).tolist() == [[[0, 1, 2, 3, 4, 5, 6, 7, width - 1]] * H, [[0, 1, 2, 3, 4, 5, 6, 7, 69]] * H]


def test_attention_over_chosen_pages():
    c = Cache([0, 1, 500, 3000, 20000], 2, 128, 32, BF16, seed=13)
    means = torch.zeros((c.k.shape[0], 2, 128), dtype=BF16, device="cuda")
    ra.page_means(c.k, c.table, _ints([0] * 5), c.n, means)
    q = c.queries(8)
    pages = ra.select_pages(q, means, c.table, c.n, 32, 40)
    got = ra.paged_attention_with_lse(q, c.k, c.v, c.table, c.n, pages=pages)
    _check_attention(q, c, got, 128 ** -0.5, pages=_np(pages))
    # all pages are all tokens
    every = ra.select_pages(q, means, c.table, c.n, 32, 700)
    whole, chosen = (ra.paged_attention_with_lse(q, c.k, c.v, c.table, c.n, pages=x) for x in (None, every))
    _check_attention(q, c, chosen, 128 ** -0.5)
    assert float((whole[1] - chosen[1])[1:].abs().max()) <= 2.0 ** -24 * 40000
    # with a window and ALiBi the places are those of the sequence
    slopes = ra.alibi_slopes(8)
    got = ra.paged_attention_with_lse(q, c.k, c.v, c.table, c.n, bias_fn=ra.sliding_window_bias(900) + ra.alibi_bias(slopes), pages=pages)
    _check_attention(q, c, got, 128 ** -0.5, pages=_np(pages), window=900, slopes=slopes)


# ---------------------------------------------------------------------------------------
# refusals, streams, graphs, threads, and all of it together
# ---------------------------------------------------------------------------------------
def test_refusals():
    c = Cache([100, 50], 2, 64, 16, BF16)
    q = c.queries(4)
    means = c.k[:, 0].contiguous()
    ok = dict(q=q, k=c.k, v=c.v, table=c.table, n=c.n)

    def attend(pages=None, bias=None, **kw):
        a = {**ok, **kw}
        return ra.paged_attention(a["q"], a["k"], a["v"], a["table"], a["n"], bias_fn=bias, pages=pages)

    attend()
    for kw in (dict(q=q.half()), dict(q=q[:, :3]), dict(q=q[:1]), dict(q=q[..., :32]), dict(q=q[None]), dict(k=c.k.half()), dict(v=c.v[:, :, :1]),
               dict(k=c.k.float(), v=c.v.float()), dict(k=c.k[0], v=c.v[0]), dict(k=c.k[..., 1:], v=c.v[..., 1:]), dict(table=c.table.long()),
               dict(table=c.table[0]), dict(table=c.table.t()), dict(n=c.n.long()), dict(n=c.n[:1]), dict(n=c.n.cpu()), dict(table=c.table.cpu()),
               dict(v=c.v.cpu()), dict(pages=_ints([[[0]]])), dict(pages=torch.zeros((2, 2, 1), device="cuda")),
               dict(pages=torch.zeros((2, 2, 0), dtype=torch.int32, device="cuda")), dict(bias=ra.alibi_bias(ra.alibi_slopes(3))),
               dict(bias=ra.segment_bias()), dict(bias=ra.prefix_lm_bias()), dict(bias=lambda **kw: None),
               dict(bias=ra.relative_bias(torch.zeros((8, 4), device="cuda")))):
        with pytest.raises(ValueError):
            attend(**kw)
    for kw in (dict(k=c.k[:, :8], v=c.v[:, :8]), dict(k=c.k[..., :16], v=c.v[..., :16], q=q[..., :16])):
        with pytest.raises(RuntimeError):
            attend(**kw)
    with pytest.raises(RuntimeError, match="gradient"):
        attend(q=q.clone().requires_grad_())
    for device in ("cuda", "cpu"):
        with pytest.raises(RuntimeError, match="slopes requires a gradient"):
            attend(bias=ra.alibi_bias(ra.alibi_slopes(4).to(device).requires_grad_()))
    with torch.no_grad():
        attend(q=q.clone().requires_grad_())
        with pytest.raises(RuntimeError, match="traced"), pytest.warns(DeprecationWarning):
            torch.jit.trace(lambda x: ra.paged_attention(x, c.k, c.v, c.table, c.n, sm_scale=0.1), (q,))
    for call in (lambda: ra.write_pages(q[:, :2], q[:, 2:], c.k, c.v.float(), c.n.long()), lambda: ra.write_pages(q[:, :2], q[:1, 2:], c.k, c.v, c.n.long()),
                 lambda: ra.write_pages(q[:, :2], q[:, 2:].float(), c.k, c.v, c.n.long()), lambda: ra.write_pages(q[:, :2], q[:, 2:], c.k, c.v, c.n),
                 lambda: ra.write_pages(q[:, :2], q[:, 2:], c.k[:1].expand(3, -1, -1, -1), c.v[:1].expand(3, -1, -1, -1), c.n.long()),
                 lambda: ra.page_means(c.k, c.table, c.n, c.n, means[:2]), lambda: ra.page_means(c.k, c.table, c.n, c.n, means.float()),
                 lambda: ra.page_means(c.k, c.table, c.n, c.n[:1], means), lambda: ra.select_pages(q, means, c.table, c.n, 16, 0),
                 lambda: ra.select_pages(q, means, c.table, c.n, 16, 3, 2, 2), lambda: ra.select_pages(q, means, c.table, c.n, 16, 3, -1, 2),
                 lambda: ra.select_pages(q.half(), means, c.table, c.n, 16, 3), lambda: ra.select_pages(q[:1], means, c.table, c.n, 16, 3)):
        with pytest.raises(ValueError):
            call()


def _step(s, q, k, v, count=None):
    """One step of one layer over the state s, in place."""
    slots, _, lengths, state = ra.page_slots(s["table"], s["n"], s["n"] + 1, s["ring"], s["state"], 16, q.shape[0])
    ra.write_pages(k, v, s["k"], s["v"], slots)
    ra.page_means(s["k"], s["table"], s["n"], lengths, s["means"])
    pages = None if count is None else ra.select_pages(q, s["means"], s["table"], lengths, 16, count)
    out = ra.paged_attention(q, s["k"], s["v"], s["table"], lengths, pages=pages)
    s["n"].copy_(lengths)
    s["state"].copy_(state)
    return out


def _serving(B=3, H=2, d=64, P=400, width=100):
    return dict(table=torch.full((B, width), -1, dtype=torch.int32, device="cuda"), n=_ints([0] * B), ring=torch.arange(P, dtype=torch.int32, device="cuda"),
                state=_ints([0, P]), k=torch.full((P, 16, H, d), math.nan, dtype=BF16, device="cuda"),
                v=torch.full((P, 16, H, d), math.nan, dtype=BF16, device="cuda"), means=torch.full((P, H, d), math.nan, dtype=BF16, device="cuda"))


def test_a_prompt_and_steps_behind_it_are_a_causal_sequence():
    """Prompts through ring_attention, their keys and values into pages, then a token at a time: what causal attention over the whole sequences gives."""
    B, H, G, d, steps = 3, 2, 2, 64, 40
    prompts = [200, 33, 1]
    s = _serving()
    rng = np.random.default_rng(14)
    L = [n + steps for n in prompts]
    q, k, v = ([torch.from_numpy(rng.standard_normal((n, h, d)).astype(np.float32)).to(BF16).cuda() for n in L] for h in (H * G, H, H))
    want = []
    for b in range(B):
        kk, vv = (_np(x[b]).repeat(G, 1)[None] for x in (k, v))
        pos = np.arange(L[b])[None]
        want.append(ring_oracle.mha_dense(_np(q[b])[None], kk, vv, ring_oracle.make_bias_fn(causal=True)(q_positions=pos, kv_positions=pos))[0][0])
    slots, starts, s["n"], s["state"] = ra.page_slots(s["table"], s["n"], _ints(prompts), s["ring"], s["state"], 16, sum(prompts))
    ra.write_pages(torch.cat([x[:n] for x, n in zip(k, prompts)]), torch.cat([x[:n] for x, n in zip(v, prompts)]), s["k"], s["v"], slots)
    ra.page_means(s["k"], s["table"], _ints([0] * B), s["n"], s["means"])
    for b, n in enumerate(prompts):
        out = ra.ring_attention(q[b][None, :n], k[b][None, :n].repeat_interleave(G, 2), v[b][None, :n].repeat_interleave(G, 2), 1, ra.causal_bias())
        assert np.abs(_np(out)[0] - want[b][:n]).max() <= 1e-2
    for t in range(steps):
        now = [torch.stack([x[b][prompts[b] + t] for b in range(B)]) for x in (q, k, v)]
        out = _step(s, *now, count=None if t % 2 else 200)  # (all pages are chosen: the same)
        for b in range(B):
            # the output is rounded once, values are below 6; scores of sums of 64 products below 6 * 6
            assert np.abs(_np(out)[b] - want[b][prompts[b] + t]).max() <= 2.0 ** -8 * 6 + 2.0 ** -24 * 2 * 72 * 64 * 36 / 8
    assert s["n"].tolist() == L


def test_a_captured_step_is_the_eager_one():
    """The state moves on in the graph itself; between replays the program works and waits."""
    eager, held = _serving(), _serving()
    gen = torch.Generator(device="cuda")
    gen.manual_seed(15)
    tokens = [[torch.empty((3, h, 64), dtype=BF16, device="cuda").normal_(generator=gen) for h in (4, 2, 2)] for _ in range(40)]
    now = [x.clone() for x in tokens[0]]
    start = {k: x.clone() for k, x in held.items()}
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        _step(held, *now, count=2)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = _step(held, *now, count=2)
    for k, x in held.items():
        x.copy_(start[k])
    for t, token in enumerate(tokens):
        want = _step(eager, *token, count=2)
        for x, y in zip(now, token):
            x.copy_(y)
        graph.replay()
        if t % 3 == 0:
            torch.cuda.synchronize()
        assert torch.equal(out, want), t
        for k in ("table", "n", "ring", "state"):
            assert torch.equal(held[k], eager[k]), (t, k)
        used = held["table"][:, :1].long().flatten()
        assert torch.equal(held["means"][used], eager["means"][used])


def test_two_graphs_two_streams_and_two_threads_share_nothing():
    c = Cache([9000, 300, 4097], 2, 64, 16, BF16, seed=16)
    qs = [c.queries(4) for _ in range(2)]
    means = torch.zeros((c.k.shape[0], 2, 64), dtype=BF16, device="cuda")
    ra.page_means(c.k, c.table, _ints([0, 0, 0]), c.n, means)

    def work(q):
        pages = ra.select_pages(q, means, c.table, c.n, 16, 30)
        return (*ra.paged_attention_with_lse(q, c.k, c.v, c.table, c.n), pages, *ra.paged_attention_with_lse(q, c.k, c.v, c.table, c.n, pages=pages))

    want = [work(q) for q in qs]
    torch.cuda.synchronize()
    graphs = []
    for q in qs:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            got = work(q)
        graphs.append((g, got))
    streams = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(5):
        for (g, _), st in zip(graphs, streams):
            with torch.cuda.stream(st):
                g.replay()
        torch.cuda.synchronize()
        for (_, got), w in zip(graphs, want):
            assert all(torch.equal(a, b) for a, b in zip(got, w))
    found = [None, None]

    def run(i):
        with torch.cuda.stream(streams[i]):
            for _ in range(20):
                got = work(qs[i])
            streams[i].synchronize()
            found[i] = got

    threads = [threading.Thread(target=run, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    for got, w in zip(found, want):
        assert all(torch.equal(a, b) for a, b in zip(got, w))
