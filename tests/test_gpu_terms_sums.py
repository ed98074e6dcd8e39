"""Gradients of a relative bias's table bucket by bucket: what a bucket gets is the sum over its own pairs, whatever the others hold."""
import struct

import pytest
import torch

import ring_attention as ra
from oracle import terms_oracle as T
from ring_attention import _lib, ring as rr
from test_gpu_terms import MASKS, Case

pytestmark = pytest.mark.gpu


class Call:
    """A call with a bias whose table is `table` [buckets, H]; ids: (q side, kv side) of a segment term, window: of a window term."""

    def __init__(self, device, table, *, Sq, Sk=None, B=1, D=64, q_off=0, causal=False, window=None, ids=None, two=True, distance=128, p=0.0,
                 dtype=torch.bfloat16, seed=0):
        Sk = Sq if Sk is None else Sk
        g = torch.Generator().manual_seed(seed)
        H = table.shape[1]
        self.q, self.k, self.v, self.do = (torch.randn(B, S, H, D, generator=g).to(device, dtype) for S in (Sq, Sk, Sk, Sq))
        self.table = table.to(device)
        at = torch.arange(Sk, device=device)[None] - q_off - torch.arange(Sq, device=device)[:, None]
        self.buckets, self.bucket = table.shape[0], T.bucket_of(at, table.shape[0], distance, two)
        self.fn = ra.causal_bias() if causal else None
        add = lambda t: t if self.fn is None else self.fn + t  # noqa: E731
        if window is not None:
            self.fn = add(ra.sliding_window_bias(window, causal=causal))
        self.q_kw, self.kv_kw = ({"q_positions": q_off} if q_off else {}), {}
        if ids is not None:
            self.fn = add(ra.segment_bias())
            self.q_kw["q_segment_ids"], self.kv_kw["kv_segment_ids"] = (x.to(device) for x in ids)
        self.term = dict(max_distance=distance, bidirectional=two)
        self.live = T.scores_mask(Sq, Sk, q_off=q_off, causal=causal, window=window, segments=ids, device=device).expand(B, 1, Sq, Sk)
        self.dropout = ra.Dropout(p, 99) if p else None
        self.threshold = round(p * 65536)
        self.keep = T.keep_mask(99, self.threshold, B, H, Sq, Sk, device) if p else None
        self.eps = 2.0 ** -7 if dtype == torch.bfloat16 else 2.0 ** -10

    def gradient(self):
        leaf = self.table.clone().requires_grad_(True)
        term = ra.relative_bias(leaf, **self.term)
        out = ra.ring_attention(self.q, self.k, self.v, 1, term if self.fn is None else self.fn + term, self.q_kw, self.kv_kw, dropout=self.dropout)
        return torch.autograd.grad(out, leaf, self.do)[0]

    def reached(self):
        """Which buckets a live pair lies in."""
        got = torch.zeros(self.buckets, dtype=torch.bool, device=self.table.device)
        got[self.bucket.expand(self.live.shape)[self.live].unique()] = True
        return got

    def want(self):
        """[buckets, H] in 64 bits, and how far off a sum over a bucket's own pairs in 32 bits may be."""
        bias = self.table.double()[self.bucket].permute(2, 0, 1)
        w = T.Attention(self.q, self.k, self.v, do=self.do, live=self.live, bias=bias, keep=self.keep, threshold=self.threshold, eps=self.eps)
        return w.table_gradient(self.bucket, self.buckets, 2.0 ** -23, own=True)


def _documents(B, S, n):
    ids = (torch.arange(S) // n).to(torch.int32)[None].expand(B, S).contiguous()
    return ids, ids


def _table(buckets, H, seed=3):
    return torch.randn(buckets, H, generator=torch.Generator().manual_seed(seed))


ENDS = [dict(Sq=300, causal=True, window=100, two=False), dict(Sq=701, causal=True, window=113, two=False, D=128, p=0.2),
        dict(Sq=600, ids=_documents(2, 600, 50), B=2), dict(Sq=600, causal=True, ids=_documents(1, 600, 90), two=False, dtype=torch.float16),
        dict(Sq=1000, window=90, p=0.1)]


@pytest.mark.parametrize("kw", ENDS)
def test_an_end_that_other_terms_mask_gets_zero(device, kw):
    """Keys far away are there by their positions, but a window or documents leave none of them: the last bucket's gradient is zero, not a remainder of
    the others'."""
    c = Call(device, _table(32, 3), **kw)
    empty = ~c.reached()
    assert empty.any()
    grad = c.gradient()
    assert (grad[~empty] != 0).any() and (grad[empty] == 0).all(), grad[empty]


@pytest.mark.parametrize("kw", [dict(Sq=500, two=True), dict(Sq=500, causal=True, two=False, D=128), dict(Sq=400, two=True, p=0.2, dtype=torch.float16)])
def test_buckets_of_little_weight_are_their_own_sums(device, kw):
    """The last buckets of either side hold most pairs, others a diagonal or a few between others, and all of these next to no weight (a learned bias of
    -40): their gradients are that small."""
    table, small = _table(32, 2), [0, 3, 10, 15, 18, 22, 31]
    table[small] = -40.0
    c = Call(device, table, **kw)
    grad, (want, off) = c.gradient().double(), c.want()
    for u in small:
        assert ((grad[u] - want[u]).abs() <= off[u]).all(), (u, grad[u], want[u], off[u])


@pytest.mark.parametrize("mask", MASKS)
@pytest.mark.parametrize("kw", [dict(relative="both", Sq=333, distance=100), dict(relative="one", Sq=290, p=0.25, D=128, dtype=torch.float16),
                                dict(relative="both", Sq=200, Sk=450, buckets=128, distance=300)])
def test_every_bucket_by_its_own_pairs(device, mask, kw):
    """Many of a call's buckets hold a few pairs beside one that holds most."""
    c = Case(device, B=2, H=2, mask=mask, table_dtype=torch.float32, **kw)
    want, off = c.want().table_gradient(c.bucket, c.buckets, 2.0 ** -23, own=True)
    assert ((c.grads()[2][3].double() - want).abs() <= off).all()


def test_two_layers_with_a_table_each_and_with_one(device):
    """The table's gradient of either of two layers, and of a table that both take (whose gradient goes through the first layer's output too)."""
    g = torch.Generator().manual_seed(6)
    B, S, H = 2, 256, 4
    table = torch.randn(32, H, generator=g).to(device)
    x, do = (torch.randn(B, S, H, 64, generator=g).to(device, torch.bfloat16) for _ in range(2))
    bucket = T.bucket_of(torch.arange(S, device=device)[None] - torch.arange(S, device=device)[:, None], 32, 128, False)
    bias, live = table.double()[bucket].permute(2, 0, 1), T.scores_mask(S, S, causal=True, device=device)

    def layer(x, table):
        return ra.ring_attention(x, x, x, 1, ra.causal_bias() + ra.relative_bias(table, bidirectional=False))

    leaves = [table.clone().requires_grad_(True) for _ in range(2)]
    y = layer(x, leaves[0])
    z = layer(y, leaves[1])
    gy, g1, g2 = torch.autograd.grad(z, (y, *leaves), do)
    for got, at, grad in ((g2, y.detach(), do), (g1, x, gy)):
        w = T.Attention(at, at, at, do=grad, live=live, bias=bias)
        want, off = w.table_gradient(bucket, 32, 2.0 ** -23, own=True)
        assert ((got.double() - want).abs() <= off).all()
    one = table.clone().requires_grad_(True)
    both, = torch.autograd.grad(layer(layer(x, one), one), one, do)
    assert ((both - (g1 + g2)).abs() <= 2.0 ** -23 * (g1.abs() + g2.abs())).all()


@pytest.mark.parametrize("two", [False, True])
@pytest.mark.parametrize("starts", [(0, 0, 0, 3), (0, 0, 7, 40), (0, 1, 1, 1)])
def test_buckets_that_start_where_the_next_one_does(device, starts, two):
    """Starts as the C interface takes them: a bucket that begins with the next one is empty, but for bucket 0 of a one-sided bias, which holds the keys ahead."""
    B, Sq, Sk, H, q_off = 1, 150, 200, 2, 1
    g = torch.Generator().manual_seed(5)
    q, k, v, do = (torch.randn(B, S, H, 64, generator=g).to(device, torch.bfloat16) for S in (Sq, Sk, Sk, Sq))
    table = _table(8 if two else 4, H).to(device).requires_grad_(True)
    at = torch.arange(Sk, device=device)[None] - q_off - torch.arange(Sq, device=device)[:, None]
    n = at.abs() if two else -at
    bucket = (n[..., None] >= torch.tensor(starts, device=device)).sum(-1).clamp(min=1) - 1
    bucket = bucket + (4 * (at > 0) if two else 0)
    w = T.Attention(q, k, v, do=do, bias=table.detach().double()[bucket].permute(2, 0, 1))
    plan = rr._RingPlan(q, k, 1, ra.relative_bias(table, bidirectional=two), {"q_positions": q_off}, None).single()
    out, _ = _lib.host().attend_terms(q, k, v, plan.native(q), 0.125, torch.bfloat16, torch.bfloat16, q_off, 0, table, two,
                                      struct.pack("4i", *starts), 0, None)
    assert ((out.detach().double() - w.out).abs() <= w.out_off).all()
    grad, = torch.autograd.grad(out, table, do)
    want, off = w.table_gradient(bucket, table.shape[0], 2.0 ** -23, own=True)
    assert ((grad.double() - want).abs() <= off).all()
    empty = torch.ones(table.shape[0], dtype=torch.bool, device=device)
    empty[bucket.unique()] = False
    assert (grad[empty] == 0).all()
