"""The relative position bias and dropout on the CPU: buckets, the generator, refusals, plans, and the oracle's gradients
against differences."""
import ctypes as C
import math
import struct

import pytest
import torch

import ring_attention as ra
from oracle import terms_oracle as T
from ring_attention import _lib, bias as bias_module, ring as rr


@pytest.mark.parametrize("side,distance", [(2, 2), (2, 5000), (3, 7), (8, 128), (16, 128), (16, 9), (32, 128), (32, 17), (33, 800), (64, 33), (64, 100000)])
def test_bucket_starts(side, distance):
    got = struct.unpack(f"{side}i", bias_module._bucket_starts(side, distance))
    if distance <= 5000:
        assert list(got) == T.bucket_starts(side, distance)
    exact = side // 2
    assert list(got[:exact + 1]) == list(range(exact + 1)) and list(got) == sorted(got) and got[-1] <= distance
    for b in range(exact + 1, side):
        # the logarithm's floor, clear of the rounding of a border
        for n, below in ((got[b], 0), (got[b] - 1, 1)):
            x = exact + (side - exact) * math.log(n / exact) / math.log(distance / exact)
            assert (x > b - 1e-9) if not below else (x < b + 1e-9)


def test_buckets_of_known_distances():
    # 32 buckets, 128: the layout that models with such a bias are trained with
    at = torch.tensor([0, -1, -7, -8, -11, -12, -90, -91, -127, -128, -10 ** 6, 1, 7, 8, 127, 10 ** 6])
    assert T.bucket_of(at, 32, 128, True).tolist() == [0, 1, 7, 8, 8, 9, 14, 15, 15, 15, 15, 17, 23, 24, 31, 31]
    assert T.bucket_of(torch.tensor([5, 0, -15, -16, -18, -19, -127, -128]), 32, 128, False).tolist() == [0, 0, 15, 16, 16, 17, 31, 31]


def test_generator_known_answers():
    # the published known answers for a key and counter of zeros
    assert T.philox((0, 0, 0, 0), (0, 0), 7) == [0x5F6FB709, 0x0D893F64, 0x4F121F81, 0x4F730A48]
    assert T.philox((0, 0, 0, 0), (0, 0), 10) == [0x6627E8D5, 0xE169C58D, 0xBC57AC4C, 0x9B00DBD8]
    mask = T.keep_mask(12345, 16384, 2, 3, 200, 300)
    assert abs(float(mask.double().mean()) - 0.75) < 5 * math.sqrt(0.75 * 0.25 / mask.numel())
    assert not torch.equal(mask[0, 0], mask[0, 1]) and not torch.equal(mask, T.keep_mask(12346, 16384, 2, 3, 200, 300))
    part = T.keep_mask(12345, 16384, 2, 3, 77, 31)  # by places alone: another length changes nothing
    assert torch.equal(part, mask[:, :, :77, :31])


@pytest.mark.parametrize("table,kw", [
    (torch.zeros(32), {}), (torch.zeros(2, 32, 4), {}), (torch.zeros(32, 4, dtype=torch.float64), {}), (torch.zeros(32, 4, dtype=torch.int32), {}),
    (torch.zeros(31, 4), {}), (torch.zeros(2, 4), {}), (torch.zeros(130, 4), {}), (torch.zeros(65, 4), dict(bidirectional=False)),
    (torch.zeros(1, 4), dict(bidirectional=False)), (torch.zeros(32, 4), dict(max_distance=8)), (torch.zeros(32, 4), dict(max_distance=0)),
    (torch.zeros(32, 4), dict(max_distance=1 << 24)), (torch.zeros(32, 4), dict(max_distance=16, bidirectional=False))])
def test_relative_bias_refusals(table, kw):
    with pytest.raises(ValueError):
        ra.relative_bias(table, **kw)


def test_relative_bias_adds_up():
    table = torch.zeros(32, 4)
    fn = ra.causal_bias() + ra.relative_bias(table, bidirectional=False) + ra.alibi_bias([1.0] * 4)
    assert fn.causal and fn.relative.table is table and fn.alibi_slopes is not None and fn.needs_positions
    assert fn.flags == ra.causal_bias().flags | ra.alibi_bias([1.0]).flags
    with pytest.raises(ValueError, match="one relative term"):
        fn + ra.relative_bias(table)
    with pytest.raises(ValueError, match="whole sequences"):
        ra.BlockBias(fn).to_struct(torch.device("cpu"))


@pytest.mark.parametrize("p", [-0.1, 1.0, 1.5, float("nan"), float("inf"), 1 - 2.0 ** -18])
def test_dropout_refusals(p):
    with pytest.raises(ValueError):
        ra.Dropout(p).threshold


def test_dropout_steps():
    assert [ra.Dropout(p).threshold for p in (0, 0.1, 0.5, 1 - 2.0 ** -16, 2.0 ** -18)] == [0, 6554, 32768, 65535, 0]


def test_cpu_tensors_are_refused():
    q = torch.zeros(1, 4, 2, 64)
    with pytest.raises(RuntimeError, match="GPU only"):
        ra.ring_attention(q, q, q, 1, ra.relative_bias(torch.zeros(32, 2)))
    with pytest.raises(RuntimeError, match="GPU only"):
        ra.ring_attention(q, q, q, 1, dropout=ra.Dropout(0.1, 1))


def _plan(n, Sq, Sk, fn, q_kw=None, kv_kw=None, D=64):
    q, k = torch.zeros(2, Sq, 3, D), torch.zeros(2, Sk, 3, D)
    return rr._RingPlan(q, k, n, fn, q_kw, kv_kw)


def test_single_plan():
    fn = ra.causal_bias() + ra.relative_bias(torch.zeros(32, 3))
    p = _plan(4, 64, 128, fn, D=80).single()
    assert (p.n, p.Lq, p.Lk, p.q_off, p.kv_off, p.D) == (1, 64, 128, [0], [0], 96) and p.fn.relative is None
    # positions as an int: of the first token
    assert _plan(4, 64, 128, fn, {"q_positions": 64}).single().q_off == [64]
    assert _plan(4, 64, 128, ra.causal_bias(), {"q_positions": 64}).q_off == [64, 80, 96, 112]
    at = torch.arange(64)[None].expand(2, 64)
    assert _plan(2, 64, 128, fn, {"q_positions": at + 7}).single().q_off == [7]
    swapped = torch.cat([at[:, 32:], at[:, :32]], 1)
    for bad in (swapped, at.flip(1), at * 2):
        with pytest.raises(ValueError, match="follow on"):
            _plan(2, 64, 128, fn, {"q_positions": bad}).single()
    with pytest.raises(ValueError, match="callable"):
        _plan(2, 64, 128, lambda **kw: None).single()
    for bad in (-1, _lib.RA_MAX_POSITION - 63):
        with pytest.raises(ValueError, match="positions must lie"):
            _plan(1, 64, 128, fn, {"q_positions": bad})


# ---- the C ABI -----------------------------------------------------------------------------------
def _terms(**kw):
    t = _lib.RaTerms()
    t.table, t.table_dtype, t.n_buckets, t.two_sided = 0x1000, 1, 8, 1
    t.table_stride_bucket, t.table_stride_head = 2, 1
    t._starts = (C.c_int32 * 4)(0, 1, 2, 11)
    t.starts = C.cast(t._starts, C.POINTER(C.c_int32))
    t.drop, t.seed = 100, 5
    for name, x in kw.items():
        if name == "starts" and x is not None:
            t._starts = (C.c_int32 * 4)(*x)
            x = C.cast(t._starts, C.POINTER(C.c_int32))
        setattr(t, name, x)
    return t


def _fwd():
    p = _lib.RaFwdStepParams()
    p.B, p.H, p.Lq, p.Lk, p.D, p.sm_scale = 1, 2, 64, 64, 64, 0.1
    for t in (p.q, p.k, p.v):
        t.ptr, t.stride_b, t.stride_h, t.stride_l = 0x1000, 64 * 128, 64, 128
    return p


def _bwd():
    p = _lib.RaBwdStepParams()
    p.B, p.H, p.Lq, p.Lk, p.D, p.sm_scale = 1, 2, 64, 64, 64, 0.1
    for t in (p.q, p.k, p.v, p.dout):
        t.ptr, t.stride_b, t.stride_h, t.stride_l = 0x1000, 64 * 128, 64, 128
    p.lse = 0x2000
    return p


def _call_fwd(lib, p, t, dtype=0):
    return lib.ra_fwd_terms(None, 0, C.byref(p), C.byref(t) if t is not None else None, 0x3000, dtype, 64 * 128, 64, 128, 0x4000, None, 0, None)


def _call_bwd(lib, p, t, d_table=0x5000, dtype=0, ws=0x6000, ws_bytes=1 << 40):
    return lib.ra_bwd_terms(None, 0, C.byref(p), C.byref(t), 0x3000, dtype, 64 * 128, 64, 128, 0, 0x7000, 64 * 128, 64, 128, 0x8000, 0x9000, 64 * 128,
                            64, 128, d_table, ws, ws_bytes, None)


@pytest.mark.parametrize("change,code", [
    (dict(table=None, drop=0), -1), (dict(drop=65536), -5), (dict(table_dtype=3), -7), (dict(table_dtype=-1), -7), (dict(table=0x1002), -4),
    (dict(table=0x1001, table_dtype=0), -4), (dict(n_buckets=7), -5), (dict(n_buckets=2), -5), (dict(n_buckets=130), -5), (dict(n_buckets=0), -5),
    (dict(n_buckets=65, two_sided=0), -5), (dict(starts=None), -1), (dict(starts=(1, 2, 3, 4)), -5), (dict(starts=(0, 2, 1, 4)), -5),
    (dict(starts=(0, 1, 2, 1 << 30)), -5), (dict(starts=(0, 0, 0, 0)), -5), (dict(seed_at=0x1004), -4), (dict(operands=1), -7), (dict(operands=5), -7),
    (dict(operands=2), -7), (dict(rest=0x1008), -4)])
def test_terms_are_checked_before_anything_runs(lib, change, code):
    assert _call_fwd(lib, _fwd(), _terms(**change)) == code, lib.ra_last_error()
    assert _call_bwd(lib, _bwd(), _terms(**change)) == code, lib.ra_last_error()


def test_calls_with_terms_are_checked_before_anything_runs(lib):
    assert _call_fwd(lib, _fwd(), None) == -1
    assert _call_fwd(lib, _fwd(), _terms(rest=0x1000), dtype=1) == -4      # nothing is lacking in fp32
    assert _call_fwd(lib, _fwd(), _terms(), dtype=3) == -7
    p = _fwd()
    p.bias.flags, p.bias.dense_bias, p.bias.dense_stride_q = _lib.RA_BIAS_DENSE, 0x1000, 64
    assert _call_fwd(lib, p, _terms()) == -5
    p = _fwd()
    p.D = 48
    assert _call_fwd(lib, p, _terms()) == -3
    p = _fwd()
    p.sm_scale = 0.0
    assert _call_fwd(lib, p, _terms()) == -2
    assert _call_bwd(lib, _bwd(), _terms(table=None)) == -1                # a gradient of no table
    assert _call_bwd(lib, _bwd(), _terms(), d_table=0x5002) == -4
    assert _call_bwd(lib, _bwd(), _terms(), ws=0x6008) == -4
    assert _call_bwd(lib, _bwd(), _terms(), ws_bytes=100) == -2
    p = _bwd()
    p.B, p.H, p.Lq = 128, 128, 1 << 16                                     # B * H * Lq = 2^30
    assert _call_bwd(lib, p, _terms()) == -8


def test_workspaces(lib):
    p, t = _bwd(), _terms()
    with_table, without = lib.ra_bwd_terms_workspace(C.byref(p), C.byref(t)), lib.ra_bwd_terms_workspace(C.byref(p), C.byref(_terms(table=None)))
    assert with_table > without >= 12 * 2 * 64 and lib.ra_bwd_terms_workspace(C.byref(p), None) == 0
    f = _fwd()
    assert lib.ra_fwd_terms_workspace(C.byref(f), C.byref(t)) == 0 and lib.ra_fwd_terms_workspace(C.byref(f), None) == 0
    f.Lq, f.Lk = 1, 1 << 20
    assert lib.ra_fwd_terms_workspace(C.byref(f), C.byref(t)) > 0          # a row's keys are shared


# ---- the oracle ----------------------------------------------------------------------------------
@pytest.mark.parametrize("p,causal,bidirectional", [(0.0, True, False), (0.25, True, True), (0.25, False, True), (0.5, False, False)])
def test_oracle_gradients_against_differences(p, causal, bidirectional):
    g = torch.Generator().manual_seed(3)
    B, H, Sq, Sk, D, nb = 2, 2, 9, 13, 8, 8
    q, k, v, do = (torch.randn(B, S, H, D, generator=g, dtype=torch.float64) for S in (Sq, Sk, Sk, Sq))
    table = torch.randn(nb, H, generator=g, dtype=torch.float64)
    at = torch.arange(Sk)[None] - torch.arange(Sq)[:, None] - 3
    bucket = T.bucket_of(at, nb, 9, bidirectional)
    threshold = round(p * 65536)
    keep = T.keep_mask(77, threshold, B, H, Sq, Sk) if p else None
    live = T.scores_mask(Sq, Sk, q_off=3, causal=causal)

    def run(q, k, v, table):
        return T.Attention(q, k, v, do=do, live=live, bias=table[bucket].permute(2, 0, 1), keep=keep, threshold=threshold)

    a = run(q, k, v, table)
    grads = [a.dq, a.dk, a.dv, a.table_gradient(bucket, nb, 2.0 ** -7)[0]]
    args = [q, k, v, table]
    for i, want in enumerate(grads):
        way = torch.randn(args[i].shape, generator=g, dtype=torch.float64)
        step = 1e-5
        f = [(run(*[x + s * step * way if n == i else x for n, x in enumerate(args)]).out * do).sum() for s in (1, -1)]
        # central differences: an error of step^2 times a third derivative of order 1e2, and of 1e-15 / step
        assert abs(float((f[0] - f[1]) / (2 * step) - (want * way).sum())) < 1e-7


def test_oracle_rows_without_keys():
    g = torch.Generator().manual_seed(1)
    q, k, v, do = (torch.randn(1, 6, 2, 8, generator=g, dtype=torch.float64) for _ in range(4))
    live = T.scores_mask(6, 6, segments=(torch.tensor([[0, 0, 1, 1, 9, 9]]), torch.tensor([[0, 0, 1, 1, 2, 2]])))
    a = T.Attention(q, k, v, do=do, live=live)
    assert a.dead[0, :, 4:].all() and not a.dead[0, :, :4].any()
    assert (a.dq[0, 4:] == 0).all() and (a.dk[0, 4:] == 0).all() and torch.isfinite(a.dv).all()
