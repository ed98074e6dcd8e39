"""The relative position bias and dropout on the GPU against their plain forms in 64 bits (oracle/terms_oracle.py), whose bounds count the
roundings that the kernels make: every element is held to its own."""
import math

import pytest
import torch

import ring_attention as ra
from oracle import terms_oracle as T
from ring_attention import _lib, ring as rr

pytestmark = pytest.mark.gpu

EPS = {torch.bfloat16: 2.0 ** -7, torch.float16: 2.0 ** -10}
TABLE_EPS = {torch.bfloat16: 2.0 ** -7, torch.float16: 2.0 ** -10, torch.float32: 2.0 ** -23}


def _ids(B, S, kind, gen):
    if kind == "documents":
        starts = torch.rand(B, S, generator=gen) < 4.0 / S
        starts[:, 0] = False
        return starts.to(torch.int32).cumsum(1, dtype=torch.int32)
    return torch.randint(0, 3, (B, S), generator=gen, dtype=torch.int32)  # "ids": in no order, rows without a key among them


class Case:
    """Inputs of a call, the call, and its plain form."""

    def __init__(self, device, *, B=1, H=2, Sq=64, Sk=None, D=64, mask="none", relative=None, buckets=16, distance=24, p=0.0, dtype=torch.bfloat16,
                 table_dtype=torch.bfloat16, ring=1, q_off=0, seed=1234567890123, scale=None, std=1.0, gen_seed=0):
        Sk = Sq if Sk is None else Sk
        gen = torch.Generator().manual_seed(gen_seed)
        self.B, self.H, self.Sq, self.Sk, self.D, self.device, self.dtype = B, H, Sq, Sk, D, device, dtype
        self.q, self.k, self.v, self.do = (
            (torch.randn(B, S, H, D, generator=gen) * std).to(device=device, dtype=dtype) for S in (Sq, Sk, Sk, Sq))
        self.table = None
        bias, self.q_kw, self.kv_kw, parts = None, {}, {}, dict(q_off=q_off)
        terms = []
        if "causal" in mask:
            terms.append(ra.causal_bias())
            parts["causal"] = True
        if "window" in mask:
            w = max(1, Sk // 3)
            terms.append(ra.sliding_window_bias(w, causal="causal" in mask))
            parts["window"] = w
        if "documents" in mask or "ids" in mask:
            kind = "documents" if "documents" in mask else "ids"
            ids = _ids(B, Sk, kind, gen)
            q_ids = ids if Sq == Sk and kind == "documents" else _ids(B, Sq, kind, gen) + (1 if kind == "ids" else 0)
            terms.append(ra.segment_bias())
            parts["segments"] = q_ids, ids
            self.q_kw["q_segment_ids"], self.kv_kw["kv_segment_ids"] = q_ids.to(device), ids.to(device)
        if "prefix" in mask:
            pre = [(torch.arange(S)[None] < torch.randint(1, S + 1, (B, 1), generator=gen)).to(torch.int32) for S in (Sq, Sk)]
            terms.append(ra.prefix_lm_bias())
            parts["prefix"] = pre
            self.q_kw["q_prefix_mask"], self.kv_kw["kv_prefix_mask"] = (x.to(device) for x in pre)
        distance_of = torch.arange(Sk, device=device)[None] - q_off - torch.arange(Sq, device=device)[:, None]
        self.bias = None
        if "alibi" in mask:
            slopes = torch.linspace(0.05, 0.5, H)
            terms.append(ra.alibi_bias(slopes.to(device)))
            self.bias = -slopes.to(device).double()[:, None, None] * distance_of.abs()
        self.buckets, self.bucket = buckets, None
        if relative is not None:
            two = relative == "both"
            self.table = torch.randn(buckets, H, generator=gen).to(device=device, dtype=table_dtype)
            self.term = dict(max_distance=distance, bidirectional=two)
            self.bucket = T.bucket_of(distance_of, buckets, distance, two)
            b = self.table.double()[self.bucket].permute(2, 0, 1)
            self.bias = b if self.bias is None else self.bias + b
        self.fn = None
        for t in terms:
            self.fn = t if self.fn is None else self.fn + t
        if q_off:
            self.q_kw["q_positions"] = q_off
        self.live = None if not terms else T.scores_mask(Sq, Sk, device=device, **parts)
        self.threshold = round(p * 65536)
        self.dropout = ra.Dropout(p, seed) if p else None
        self.keep = T.keep_mask(seed, self.threshold, B, H, Sq, Sk, device) if p else None
        self.ring, self.scale = ring, scale

    def want(self, do=True):
        return T.Attention(self.q, self.k, self.v, do=self.do if do else None, scale=self.scale, live=self.live, bias=self.bias, keep=self.keep,
                           threshold=self.threshold, eps=EPS[self.dtype])

    def call(self, q=None, k=None, v=None, table=None, **kw):
        fn = self.fn
        if self.table is not None:
            term = ra.relative_bias(self.table if table is None else table, **self.term)
            fn = term if fn is None else fn + term
        kw = {"dropout": self.dropout, "sm_scale": self.scale, **kw}
        q, k, v = (x if y is None else y for x, y in ((self.q, q), (self.k, k), (self.v, v)))
        return ra.ring_attention_with_lse(q, k, v, self.ring, fn, self.q_kw, self.kv_kw, **kw)

    def grads(self, **kw):
        leaves = [x.detach().requires_grad_(True) for x in (self.q, self.k, self.v)]
        if self.table is not None:
            leaves.append(self.table.detach().requires_grad_(True))
        out, lse = self.call(*leaves, **kw)
        return out.detach(), lse, torch.autograd.grad(out, leaves, self.do)


def _close(name, got, want, off):
    got = got.double()
    bad = ~((got - want).abs() <= off)
    bad &= ~(torch.isnan(got) & torch.isnan(want)) & (got != want)
    assert not bad.any(), f"{name}: {int(bad.sum())} of {bad.numel()} off, at {bad.nonzero()[0].tolist()}: {float(got[bad][0])} for {float(want[bad][0])}, " \
                          f"at most {float(off[bad][0])}"


def _check(c, norm=True, **kw):
    w = c.want()
    out, lse, grads = c.grads(**kw)
    dead = w.dead.permute(0, 2, 1)
    assert torch.isnan(out[dead]).all() and (lse[w.dead] == -math.inf).all()
    _close("out", out[~dead], w.out[~dead], w.out_off[~dead])
    _close("lse", lse[~w.dead], w.lse[~w.dead], w.lse_off[~w.dead])
    pairs = [("dq", grads[0], w.dq, w.dq_off), ("dk", grads[1], w.dk, w.dk_off), ("dv", grads[2], w.dv, w.dv_off)]
    if c.table is not None:
        pairs.append(("table", grads[3], *w.table_gradient(c.bucket, c.buckets, TABLE_EPS[c.table.dtype])))
    for name, got, want, off in pairs:
        _close(name, got, want, off)
    if norm:
        # of all elements together: fewer than twelve roundings to half a step each, independent, in rms at most eps / 2 / sqrt(3) apiece
        for name, got, want, _ in [("out", out[~dead], w.out[~dead], None)] + pairs:
            if want.numel() >= 256:
                assert float((got.double() - want).norm()) <= EPS[c.dtype] * float(want.norm()), name
    return out, lse, grads


SIZES = [(1, 1), (1, 65), (2, 1), (33, 130), (127, 64), (128, 129), (130, 300), (257, 257)]


@pytest.mark.parametrize("Sq,Sk", SIZES)
@pytest.mark.parametrize("relative", ["both", "one"])
def test_relative_bias_sizes(device, Sq, Sk, relative):
    _check(Case(device, B=2, Sq=Sq, Sk=Sk, relative=relative), norm=min(Sq, Sk) > 32)


@pytest.mark.parametrize("Sq,Sk", SIZES)
def test_dropout_sizes(device, Sq, Sk):
    _check(Case(device, B=2, H=3, Sq=Sq, Sk=Sk, p=0.3), norm=min(Sq, Sk) > 32)


MASKS = ["causal", "window", "causal+window", "documents", "causal+documents", "ids", "prefix", "prefix+documents", "alibi", "causal+alibi", "ids+alibi"]


@pytest.mark.parametrize("mask", MASKS)
@pytest.mark.parametrize("relative,p", [("both", 0.0), (None, 0.25), ("one", 0.25)])
def test_masks(device, mask, relative, p):
    _check(Case(device, B=2, H=2, Sq=333, mask=mask, relative=relative, p=p, distance=100), norm="ids" not in mask)


@pytest.mark.parametrize("D", [8, 32, 40, 64, 80, 96, 104, 128])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_head_dims_and_types(device, D, dtype):
    _check(Case(device, B=2, H=3, Sq=200, Sk=290, D=D, dtype=dtype, relative="both", p=0.2))


@pytest.mark.parametrize("buckets,distance,relative,table_dtype", [
    (4, 3, "both", torch.float32), (2, 2, "one", torch.float16), (128, 200, "both", torch.bfloat16), (64, 1000, "one", torch.float32),
    (32, 128, "both", torch.float16), (33, 70, "one", torch.bfloat16), (6, 100000, "both", torch.float32), (64, 40, "both", torch.float32)])
@pytest.mark.parametrize("mask", ["none", "causal"])
def test_buckets(device, buckets, distance, relative, table_dtype, mask):
    _check(Case(device, B=2, H=2, Sq=400, mask=mask, buckets=buckets, distance=distance, relative=relative, table_dtype=table_dtype))


def test_a_bucket_that_no_pair_has_gets_zero(device):
    c = Case(device, Sq=100, mask="causal", relative="both", buckets=32, distance=500)
    grad = _check(c)[2][3]
    empty = torch.ones(32, dtype=torch.bool, device=device)
    empty[c.bucket[c.live[0, 0]].unique()] = False
    assert empty.any() and (grad[empty] == 0).all() and (grad[~empty] != 0).any()
    # ... the far ends too, of which one is derived from the others
    c = Case(device, Sq=700, mask="causal+window", relative="both", buckets=32, distance=500)
    assert not c.bucket[c.live[0, 0]].eq(15).any()
    assert (_check(c)[2][3][15] == 0).all()


@pytest.mark.parametrize("Sq,Sk,q_off,mask,relative", [(1, 1500, 1499, "causal", "one"), (7, 4000, 3993, "causal", "both"), (129, 2000, 0, "none", "both"),
                                                        (100, 130, 1 << 29, "none", "both"), (64, 3000, 900, "window", "both"), (16, 5000, 0, "none", "both")])
def test_positions_and_shared_rows(device, Sq, Sk, q_off, mask, relative):
    """Rows whose keys several workgroups share, and positions that are far from each other (the window of 1000 and the bias's constant ends)."""
    for p in (0.0, 0.1):
        _check(Case(device, B=1, H=3, Sq=Sq, Sk=Sk, q_off=q_off, mask=mask, relative=relative, buckets=32, distance=128, p=p))


def test_longer_than_the_tile_lists(device):
    """Segment ids of more tokens than the kernels list tiles for, on a few rows of the sequence, which the plain form takes alone."""
    S, H, D = 66000, 1, 32
    c = Case(device, H=H, Sq=128, Sk=S, D=D, mask="documents", relative="both", buckets=32, distance=128, p=0.1)
    g = torch.Generator().manual_seed(4)
    ids = (torch.rand(1, S, generator=g) < 0.001).to(torch.int32).cumsum(1, dtype=torch.int32)
    q = torch.randn(1, S, H, D, generator=g).to(device, torch.bfloat16)
    kw = {"q_segment_ids": ids.to(device)}, {"kv_segment_ids": ids.to(device)}
    fn = ra.segment_bias() + ra.relative_bias(c.table, **c.term)
    out, lse = ra.ring_attention_with_lse(q, c.k, c.v, 2, fn, *kw, dropout=c.dropout)
    for first in (0, 30000, S - 128):
        rows = slice(first, first + 128)
        at = torch.arange(S, device=device)[None] - torch.arange(first, first + 128, device=device)[:, None]
        bias = c.table.double()[T.bucket_of(at, 32, 128, True)].permute(2, 0, 1)
        keep = T.keep_mask(c.dropout.seed, c.threshold, 1, H, first + 128, S, "cpu")[:, :, rows].to(device) if first < 1000 else _keep_rows(c, first, S, device)
        w = T.Attention(q[:, rows], c.k, c.v, live=T.scores_mask(128, S, segments=(ids[:, rows], ids), device=device), bias=bias, keep=keep,
                        threshold=c.threshold)
        _close("out", out[:, rows], w.out, w.out_off)
        _close("lse", lse[:, :, rows], w.lse, w.lse_off)


def _keep_rows(c, first, S, device):
    i = first + torch.arange(128, device=device)[:, None]
    j = torch.arange(S, device=device)[None]
    zero = torch.zeros_like(i * j)
    w = torch.stack(T.philox((zero + j // 2, zero + i // 4, zero, zero), (c.dropout.seed & 0xFFFFFFFF, c.dropout.seed >> 32), 7))
    word = w.gather(0, (zero + i % 4)[None])[0]
    return (((word >> 16 * (zero + j % 2)) & 0xFFFF) >= c.threshold)[None, None]


def test_backward_longer_than_the_tile_lists(device):
    """dV of a sequence of more tiles than are listed: documents of 64 tokens, each of which the plain form takes alone."""
    S, D = 66048, 32
    g = torch.Generator().manual_seed(4)
    q, k, v, do = (torch.randn(1, S, 1, D, generator=g).to(device, torch.bfloat16) for _ in range(4))
    ids = (torch.arange(S, device=device) // 64).to(torch.int32)[None]
    table = torch.randn(32, 1, generator=g).to(device)
    leaves = [x.requires_grad_(True) for x in (q, k, v, table)]
    out = ra.ring_attention(*leaves[:3], 1, ra.segment_bias() + ra.relative_bias(table), {"q_segment_ids": ids}, {"kv_segment_ids": ids})
    grads = torch.autograd.grad(out, leaves, do)
    at = torch.arange(64, device=device)
    bucket = T.bucket_of(at[None] - at[:, None], 32, 128, True)
    w = T.Attention(*(x.detach().reshape(-1, 64, 1, D) for x in (q, k, v)), do=do.reshape(-1, 64, 1, D), bias=table.detach().double()[bucket].permute(2, 0, 1))
    for name, got in (("out", out.detach()), ("dq", grads[0]), ("dk", grads[1]), ("dv", grads[2])):
        _close(name, got.reshape(-1, 64, 1, D), getattr(w, name), getattr(w, name + "_off"))
    _close("table", grads[3], *w.table_gradient(bucket, 32, 2.0 ** -23))


def test_dropout_leaves_out_what_the_generator_says(device):
    """With values of the unit matrix the output is the weights themselves."""
    c = Case(device, B=2, H=3, Sq=75, Sk=128, D=128, p=0.4)
    v = torch.eye(128, device=device).to(torch.bfloat16)[None, :, None].expand(2, 128, 3, 128)
    out = c.call(v=v)[0]
    assert torch.equal(out.permute(0, 2, 1, 3) != 0, c.keep)
    # the same in the gradient of the values
    vv = v.contiguous().requires_grad_(True)
    do = torch.zeros_like(out)
    do[:, 11, :, 0] = 1
    g, = torch.autograd.grad(c.call(v=vv)[0], vv, do)
    assert torch.equal(g[..., 0].permute(0, 2, 1) != 0, c.keep[:, :, 11])


@pytest.mark.parametrize("relative,p,mask", [("both", 0.0, "none"), ("one", 0.2, "causal+documents")])
def test_results_do_not_change_with_the_ring_or_from_call_to_call(device, relative, p, mask):
    c = Case(device, B=2, H=3, Sq=768, mask=mask, relative=relative, p=p)
    first = c.grads()
    for ring in (1, 2, 8):
        for impl in ("pallas", "hip", "hip_fused"):
            c.ring = ring
            got = c.grads(block_impl=impl)
            assert all(torch.equal(x, y) for x, y in zip((*first[:2], *first[2]), (*got[:2], *got[2])))


@pytest.mark.parametrize("kw", [dict(mask="", relative="both", B=2, Sq=672, D=128, buckets=16), dict(mask="causal", relative="past", Sq=700, p=0.1),
                                dict(mask="causal", relative="past", Sq=300, dtype=torch.float16),
                                dict(mask="", relative="both", Sq=500, D=96, p=0.3, buckets=16, dtype=torch.float16)])
def test_table_gradient_is_free_of_the_weights_roundings(device, kw):
    """A bucket's sum cancels to a small part of its terms, so the roundings of the forward's weights (half a step of 16 bits) must not reach it through
    delta.  What they would do is computed here; what remains are roundings of twice 16 bits, 2^-9 of that (fp16: 2^-12, and weights below 2^-14 lose up
    to 2^-25), and scores in 32 bits, some 2^-20 of a weight and so 2^-11 (fp16: 2^-8) of it: an eighth leaves room for both."""
    c = Case(device, H=4, **{"B": 1, "table_dtype": torch.float32, "dtype": torch.bfloat16, **kw})
    w = c.want()
    got = c.grads()[2][3].double()
    want, _ = w.table_gradient(c.bucket, c.buckets, 0.0)
    v, do = (x.double().permute(0, 2, 1, 3) for x in (c.v, c.do))
    weights = w.P / w.P.amax(3, keepdim=True)
    rounded = weights.to(c.dtype).double()
    lost = (rounded / rounded.sum(3, keepdim=True) - w.P) * (1.0 if c.keep is None else c.keep.double() / (1 - c.threshold / 65536))
    through_delta = w.P * ((lost @ v) * do).sum(3, keepdim=True)
    lossy = torch.stack([(through_delta * (c.bucket == u)).sum((0, 2, 3)) for u in range(c.buckets)])
    assert float((got - want).norm()) <= float(lossy.norm()) / 8


def test_seed_on_the_device(device):
    c = Case(device, B=1, H=2, Sq=130, p=0.5, relative="both")
    for seed in (c.dropout.seed, (1 << 64) - 3, -3):
        c.dropout = ra.Dropout(0.5, seed)
        want = c.grads()
        c.dropout = ra.Dropout(0.5, torch.tensor([seed if seed < 1 << 63 else seed - (1 << 64)], device=device))
        got = c.grads()
        assert all(torch.equal(x, y) for x, y in zip((*want[:2], *want[2]), (*got[:2], *got[2])))
    # changed between forward and backward: autograd refuses
    leaf = c.q.detach().requires_grad_(True)
    out = c.call(leaf)[0]
    c.dropout.seed.add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        out.backward(c.do)


def test_operand_and_table_layouts(device):
    """Transposed and padded operands, an expanded and a transposed table, k and v of more batch rows, heads and tokens than q."""
    c = Case(device, B=2, H=4, Sq=150, Sk=170, relative="both", p=0.1)
    want = c.grads()
    t = [x.transpose(1, 2).contiguous().transpose(1, 2) for x in (c.q, c.k, c.v)]
    wide = [torch.nn.functional.pad(x, (0, 24)) for x in t]
    odd = [torch.nn.functional.pad(x, (0, 3))[..., :64] for x in t]
    for q, k, v in (t, [x[..., :64] for x in wide], odd):
        got = c.call(q, k, v)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    table = c.table.t().contiguous().t().detach().requires_grad_(True)
    grad, = torch.autograd.grad(c.call(table=table)[0], table, c.do)
    assert torch.equal(grad, want[2][3])
    # one column for all heads: the sum of the heads' gradients, which autograd takes in the table's type
    col = c.table[:, :1].float().detach().requires_grad_(True)
    out = c.call(table=col.expand(-1, 4))[0]
    grad, = torch.autograd.grad(out, col, c.do)
    full = c.table[:, :1].float().expand(-1, 4).contiguous().requires_grad_(True)
    each, = torch.autograd.grad(c.call(table=full)[0], full, c.do)
    assert torch.allclose(grad, each.sum(1, keepdim=True), rtol=4 * 2.0 ** -23, atol=float(each.abs().sum(1).max()) * 4 * 2.0 ** -23)
    more_k = torch.nn.functional.pad(c.k, (0, 0, 0, 1, 0, 0, 0, 1)).requires_grad_(True)
    more_v = torch.nn.functional.pad(c.v, (0, 0, 0, 1, 0, 5, 0, 1)).requires_grad_(True)
    out = c.call(k=more_k, v=more_v)[0]
    gk, gv = torch.autograd.grad(out, (more_k, more_v), c.do)
    assert torch.equal(gk[:2, :, :4], want[2][1]) and torch.equal(gv[:2, :170, :4], want[2][2])
    assert not gk[2:].any() and not gk[:, :, 4:].any() and not gv[:, 170:].any()


def test_one_head_of_keys_for_all(device):
    """Keys and values that are expanded over the heads: their gradients are the heads' sum, which autograd takes in bf16."""
    c = Case(device, B=2, H=4, Sq=140, relative="both", p=0.1)
    k, v = (x[:, :, :1].contiguous().requires_grad_(True) for x in (c.k, c.v))
    out = c.call(k=k.expand(-1, -1, 4, -1), v=v.expand(-1, -1, 4, -1))[0]
    gk, gv = torch.autograd.grad(out, (k, v), c.do)
    c.k, c.v = (x.detach().expand(-1, -1, 4, -1).contiguous() for x in (k, v))
    w = c.want()
    _close("out", out.detach(), w.out, w.out_off)
    for name, got in (("dk", gk), ("dv", gv)):
        want, off = getattr(w, name), getattr(w, name + "_off")
        # (a sum in bf16 of four: at most three more roundings of partial sums, and the result's)
        _close(name, got, want.sum(2, keepdim=True), off.sum(2, keepdim=True) + 4 * 2.0 ** -8 * want.abs().sum(2, keepdim=True))


def test_cache_of_more_than_two_to_the_31_elements(device):
    S, H, D = 262400, 64, 128
    k, v = (torch.empty(1, S, H, D, device=device, dtype=torch.bfloat16).normal_() for _ in range(2))
    assert k.numel() > 1 << 31
    q = torch.randn(1, 1, H, D, device=device).to(torch.bfloat16)
    table = torch.randn(32, H, device=device)
    fn = ra.causal_bias() + ra.relative_bias(table, bidirectional=False)
    out, lse = ra.ring_attention_with_lse(q, k, v, 1, fn, {"q_positions": S - 1}, dropout=ra.Dropout(0.1, 5))
    bucket = T.bucket_of(torch.arange(S, device=device)[None] - (S - 1), 32, 128, False)
    for h in (0, H - 1):
        j = torch.arange(S, device=device)[None]
        zero = torch.zeros_like(j)
        w0 = T.philox((j // 2, zero, zero + h, zero), (5, 0), 7)[0]
        keep = (((w0 >> 16 * (j % 2)) & 0xFFFF) >= 6554)[None, None]
        w = T.Attention(q[:, :, h:h + 1], k[:, :, h:h + 1], v[:, :, h:h + 1], bias=table[:, h].double()[bucket][None], keep=keep, threshold=6554)
        _close("out", out[:, :, h:h + 1], w.out, w.out_off)
        _close("lse", lse[:, h:h + 1], w.lse, w.lse_off)


def test_capture_beside_a_live_graph_of_leaves_further_up(device):
    """The same through what the arguments are computed from; without gradients such a capture is an ordinary one."""
    c = Case(device, Sq=40, relative="both", p=0.1)
    leaf = c.q.detach().clone().requires_grad_(True)
    alive = c.call(leaf * 1)[0]
    graph = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match="live autograd graph"):
        with torch.cuda.graph(graph):
            c.call(leaf * 1)
    graph = torch.cuda.CUDAGraph()
    with torch.no_grad(), torch.cuda.graph(graph):
        held = c.call(leaf)[0]
    for _ in range(2):
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(held, alive.detach())


def test_capture_beside_a_live_graph_of_the_same_leaves(device):
    c = Case(device, Sq=40, relative="both", p=0.1)
    leaf = c.q.detach().clone().requires_grad_(True)
    alive = c.call(leaf)[0]
    graph = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match="live autograd graph"):
        with torch.cuda.graph(graph):
            c.call(leaf)
    del alive
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = torch.autograd.grad(c.call(leaf)[0], leaf, c.do)[0]
    want = c.grads()[2][0]
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(held, want)


def test_empty_arrays_are_refused(device):
    c = Case(device, Sq=16, relative="both", p=0.1)
    for q, k in ((c.q[:, :0], c.k), (c.q, c.k[:, :0]), (c.q[:0], c.k[:0]), (c.q[:, :, :0], c.k[:, :, :0])):
        with pytest.raises((RuntimeError, ValueError)):
            c.call(q=q, k=k, v=k)


def test_other_dtypes_are_rounded_to_bf16(device):
    c = Case(device, B=1, H=2, Sq=190, D=80, relative="one", mask="causal", p=0.2)
    leaves = [x.float().requires_grad_(True) for x in (c.q, c.k, c.v)]
    out, lse = c.call(*leaves)
    assert out.dtype == torch.float32
    w = c.want()
    _close("out", out.detach(), w.out, w.out_off)
    for name, g in zip(("dq", "dk", "dv"), torch.autograd.grad(out, leaves, c.do.float())):
        assert g.dtype == torch.float32
        _close(name, g, getattr(w, name), getattr(w, name + "_off"))
    # mixed: bf16 operands, the results in q's type
    out = c.call(c.q.half(), c.k.float(), c.v)[0]
    assert out.dtype == torch.float16


def test_only_the_gradients_that_are_wanted(device):
    c = Case(device, B=1, H=2, Sq=300, relative="both", p=0.1)
    full = c.grads()[2]
    leaves = [c.q, c.k, c.v, c.table]
    for i in range(4):
        x = leaves[i].detach().requires_grad_(True)
        args = [x if n == i else y for n, y in enumerate(leaves)]
        out = c.call(*args)[0]
        g, = torch.autograd.grad(out, x, c.do)
        assert torch.equal(g, full[i])
    with_gradients = c.grads()[0]
    with torch.no_grad():
        assert torch.equal(c.call()[0], with_gradients)
    lse_only = c.call(*(x.detach().requires_grad_(True) for x in leaves))[1]
    assert not lse_only.requires_grad


def test_large_and_infinite_table_values(device):
    """A bucket of -inf masks its pairs; large values are numbers like any other."""
    c = Case(device, B=1, H=2, Sq=200, relative="both", buckets=8, distance=20, table_dtype=torch.float32)
    c.table[3] = -math.inf   # the past from the last start on: the far end
    c.table[6] = -math.inf   # some way ahead
    c.table[0] = 30.0
    c.bias = c.table.double()[c.bucket].permute(2, 0, 1)
    g = _check(c, norm=False)[2][3]
    assert (g[3] == 0).all() and (g[6] == 0).all()
    # only masked buckets left for a row: no key at all
    c.table[:] = -math.inf
    out, lse = c.call()
    assert torch.isnan(out).all() and (lse == -math.inf).all()


def test_what_lies_in_masked_places_does_not_matter(device):
    """NaN and infinities in the keys, values and queries of padding."""
    for p, relative in ((0.0, "both"), (0.2, None), (0.2, "both")):
        c = Case(device, B=2, H=2, Sq=200, relative=relative, p=p, mask="documents")
        ids = torch.ones(2, 200, dtype=torch.int32, device=device)
        ids[0, 150:] = 0
        c.q_kw["q_segment_ids"], c.kv_kw["kv_segment_ids"] = ids, ids
        want = c.grads()
        k, v = c.k.clone(), c.v.clone()
        k[0, 192:] = math.inf   # a whole tile of the padding, which no row of the sequence meets
        v[0, 192:] = math.nan
        out = c.call(k=k, v=v)[0]
        assert torch.equal(out[0, :128], want[0][0, :128]) and torch.equal(out[1], want[0][1])


def test_graph_replays_with_a_new_seed(device):
    """A training step captured once: each replay has the mask of the seed that it finds, with eager work in between."""
    c = Case(device, B=2, H=2, Sq=260, mask="causal", relative="one", p=0.3)
    seed = torch.tensor([7], device=device)
    c.dropout = ra.Dropout(0.3, seed)
    leaves = [x.detach().clone().requires_grad_(True) for x in (c.q, c.k, c.v, c.table)]

    def step():
        out, lse = c.call(*leaves)
        return (out.detach(), lse, *torch.autograd.grad(out, leaves, c.do))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for n in (7, 8, 7, -5, 1 << 62):
        seed.fill_(n)
        graph.replay()
        got = [x.clone() for x in held]
        torch.cuda.synchronize()
        want = step()
        assert all(torch.equal(x, y) for x, y in zip(got, want)), n
    # two graphs at once, each with its own workspaces
    other = Case(device, B=1, H=3, Sq=1, Sk=3000, q_off=2999, mask="causal", relative="one", gen_seed=5)
    graph2 = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph2):
        held2 = other.call()
    want2 = other.call()
    want = step()
    for _ in range(3):
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            graph2.replay()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(held2, want2)) and all(torch.equal(x, y) for x, y in zip(held, want))


def test_on_another_stream(device):
    c = Case(device, B=1, H=2, Sq=500, relative="both", p=0.1)
    want = c.grads()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = c.grads()
    s.synchronize()
    assert all(torch.equal(x, y) for x, y in zip((*want[:2], *want[2]), (*got[:2], *got[2])))


def test_refusals(device):
    c = Case(device, B=1, H=2, Sq=64, relative="both", p=0.1)
    with pytest.raises(ValueError, match="column per head"):
        c.call(table=torch.zeros(16, 3, device=device))
    with pytest.raises(TypeError, match="Dropout"):
        c.call(dropout=0.1)
    with pytest.raises(ValueError, match="one int64"):
        c.call(dropout=ra.Dropout(0.1, torch.zeros(1, dtype=torch.int32, device=device)))
    with pytest.raises(ValueError, match="one int64"):
        c.call(dropout=ra.Dropout(0.1, torch.zeros(2, dtype=torch.int64, device=device)))
    with pytest.raises(ValueError, match="one int64"):
        c.call(dropout=ra.Dropout(0.1, torch.zeros(1, dtype=torch.int64)))
    with pytest.raises(TypeError):
        c.call(dropout=ra.Dropout(0.1, 0.5))
    dense = lambda **kw: torch.zeros(1, 1, 64, 64, device=device)  # noqa: E731
    with pytest.raises(ValueError, match="callable"):
        ra.ring_attention(c.q, c.k, c.v, 1, dense, dropout=ra.Dropout(0.1, 1))
    at = torch.arange(64, device=device)[None]
    with pytest.raises(ValueError, match="follow on"):
        ra.ring_attention(c.q, c.k, c.v, 1, ra.relative_bias(c.table), {"q_positions": at.flip(1)})
    with pytest.raises(ValueError, match="whole sequences"):
        x = c.q.permute(0, 2, 1, 3)
        ra.fwd_block(x, x, x, ra.BlockBias(ra.relative_bias(c.table)), *rr.init_carry(1, 2, 64, 64, device), 0.1)
    with pytest.raises(ValueError, match="divisible"):
        ra.ring_attention(c.q, c.k, c.v, 3, ra.relative_bias(c.table))
    # dropout of nothing is the call without it
    assert torch.equal(ra.ring_attention(c.q, c.k, c.v, 1, dropout=ra.Dropout(0.0, 1)), ra.ring_attention(c.q, c.k, c.v, 1))


def test_table_gradient_against_differences(device):
    """The kernels' own output along a direction of the table: a difference of two outputs in fp32 has twice the output's bound, over the step, and
    the third derivative's part of the step squared, which the plain form gives."""
    c = Case(device, B=2, H=2, Sq=150, relative="both", table_dtype=torch.float32)
    way = torch.randn(c.table.shape, generator=torch.Generator().manual_seed(2)).to(device)
    leaf = c.table.clone().requires_grad_(True)
    grad, = torch.autograd.grad(c.call(table=leaf, out_dtype=torch.float32)[0], leaf, c.do.float())
    step, base, f, exact, room = 0.25, c.table.clone(), [], [], 0.0
    for s in (1, -1):
        c.table = base + s * step * way
        c.bias = c.table.double()[c.bucket].permute(2, 0, 1)
        w = c.want(do=False)
        f.append(float((c.call(out_dtype=torch.float32)[0].double() * c.do.double()).sum()))
        exact.append(float((w.out * c.do.double()).sum()))
        room += float((w.out_off * c.do.double().abs()).sum()) / (2 * step)
    got, plain = (f[0] - f[1]) / (2 * step), (exact[0] - exact[1]) / (2 * step)
    c.table, c.bias = base, base.double()[c.bucket].permute(2, 0, 1)
    want, off = c.want().table_gradient(c.bucket, c.buckets, 2.0 ** -23)
    truncation = abs(plain - float((want * way).sum()))
    assert abs(got - float((grad.double() * way).sum())) <= room + truncation + float((off * way.abs()).sum())


def test_used_together(device):
    """What a decoder with a learned bias does: two layers of attention with the bias and dropout in training, their step's gradients against
    the same in 64 bits of one layer each; then a prompt and tokens one by one, which give what the whole sequence gives."""
    g = torch.Generator().manual_seed(6)
    B, S, H, D = 2, 256, 4, 64
    table = torch.randn(32, H, generator=g).to(device).requires_grad_(True)
    x = torch.randn(B, S, H, D, generator=g).to(device, torch.bfloat16).requires_grad_(True)
    do = torch.randn(B, S, H, D, generator=g).to(device, torch.bfloat16)
    fn = ra.relative_bias(table, bidirectional=False)
    at = torch.arange(S, device=device)[None].expand(B, S)
    y = ra.ring_self_attention(x, x, x, ra.RingAxis("sp", 4), causal=True, positions=at, relative=fn, dropout=ra.Dropout(0.1, 11))
    z = ra.ring_self_attention(y, y, y, ra.RingAxis("sp", 4), causal=True, positions=at, relative=fn, dropout=ra.Dropout(0.1, 12))
    gy, g2 = torch.autograd.grad(z, (y, table), do, retain_graph=True)
    gx, gt = torch.autograd.grad(z, (x, table), do)
    bucket = T.bucket_of(torch.arange(S, device=device)[None] - torch.arange(S, device=device)[:, None], 32, 128, False)
    bias, live = table.detach().double()[bucket].permute(2, 0, 1), T.scores_mask(S, S, causal=True, device=device)
    threshold = round(0.1 * 65536)

    def layer(x, do, seed):
        return T.Attention(x.detach(), x.detach(), x.detach(), do=do, live=live, bias=bias, keep=T.keep_mask(seed, threshold, B, H, S, S, device),
                           threshold=threshold)

    w2 = layer(y, do, 12)
    two = w2.dq + w2.dk + w2.dv
    # (autograd adds the three up in bf16: two more roundings of their partial sums)
    off = w2.dq_off + w2.dk_off + w2.dv_off + 2.0 ** -8 * 2 * (w2.dq.abs() + w2.dk.abs() + w2.dv.abs())
    _close("second layer", gy, two, off)
    w1 = layer(x, gy, 11)
    _close("first layer", gx, w1.dq + w1.dk + w1.dv, w1.dq_off + w1.dk_off + w1.dv_off + 2.0 ** -8 * 2 * (w1.dq.abs() + w1.dk.abs() + w1.dv.abs()))
    t2, o2 = w2.table_gradient(bucket, 32, 2.0 ** -23)
    t1, o1 = w1.table_gradient(bucket, 32, 2.0 ** -23)
    _close("table, second layer", g2, t2, o2)
    _close("table, both", gt, t1 + t2, o1 + o2 + 2.0 ** -22 * (t1.abs() + t2.abs()))
    # generation
    with torch.no_grad():
        k, v = (torch.randn(B, S, H, D, generator=g).to(device, torch.bfloat16) for _ in range(2))
        q = x.detach()
        w = T.Attention(q, k, v, live=live, bias=bias)
        causal = ra.causal_bias() + fn
        whole, lse = ra.ring_attention_with_lse(q, k, v, 1, causal)
        _close("whole", whole, w.out, w.out_off)
        prompt = ra.ring_attention(q[:, :200], k[:, :200], v[:, :200], 1, causal)
        _close("prompt", prompt, w.out[:, :200], w.out_off[:, :200])
        for n in (200, 201, 254, 255):
            token, l = ra.ring_attention_with_lse(q[:, n:n + 1], k[:, :n + 1], v[:, :n + 1], 1, causal, {"q_positions": n})
            _close("token", token, w.out[:, n:n + 1], w.out_off[:, n:n + 1])
            _close("token lse", l, w.lse[:, :, n:n + 1], w.lse_off[:, :, n:n + 1])
        chunk = ra.ring_attention(q[:, 200:], k, v, 1, causal, {"q_positions": 200})
        _close("chunk", chunk, w.out[:, 200:], w.out_off[:, 200:])


def test_plans_hold_no_tables(device):
    """Every step of a training or decoding loop has a table, a seed and positions of its own: a plan serves them all."""
    ra.clear_plan_cache()
    c = Case(device, Sq=16, Sk=64, relative="both", p=0.1)
    for n in range(5):
        c.dropout = ra.Dropout(0.1, n)
        c.q_kw = {"q_positions": 10 + n}
        c.call(table=torch.randn(16, 2, device=device))
    assert len(rr._PLAN_CACHE) == 1
    plan = next(iter(rr._PLAN_CACHE.values()))
    assert plan[1].relative.table is None and not plan[2] and plan[0].fn.relative is None
    ra.clear_plan_cache()
