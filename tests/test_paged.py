"""The paged cache without a GPU: the C ABI's argument checks, the layout of its structs, and the oracle's own consistency."""
import ctypes as C

import numpy as np
import pytest
import torch

from oracle import paged_oracle as R
from ring_attention import _lib

TABLE, LENGTHS, WORK = 0x10000, 0x20000, 0x30000


def _table():
    return _lib.RaPageTable(TABLE, 64, 64, 1000, 16)


def _params():
    p = _lib.RaPagedParams()
    p.B, p.H, p.group, p.D, p.dtype, p.sm_scale = 2, 4, 2, 128, _lib.RA_DTYPE_BF16, 0.1
    p.q, p.q_stride_b, p.q_stride_h = 0x1000, 8 * 128, 128
    for pool in (p.k, p.v):
        pool.ptr, pool.stride_page, pool.stride_token, pool.stride_head = 0x4000, 16 * 512, 512, 128
    p.table, p.lengths = _table(), LENGTHS
    return p


def test_struct_layout():
    assert C.sizeof(_lib.RaPool) == 32
    assert C.sizeof(_lib.RaPageTable) == 32
    assert C.sizeof(_lib.RaPagedParams) == 32 + 24 + 64 + 32 + 24


@pytest.mark.parametrize("change,code", [
    (lambda p: setattr(p, "B", 0), -2),
    (lambda p: setattr(p, "B", _lib.RA_MAX_PAGED_ROWS + 1), -2),
    (lambda p: setattr(p, "H", 0), -2),
    (lambda p: setattr(p, "group", 0), -2),
    (lambda p: setattr(p, "group", 65536), -2),
    (lambda p: setattr(p, "D", 80), -3),
    (lambda p: setattr(p, "D", 256), -3),
    (lambda p: setattr(p, "dtype", _lib.RA_DTYPE_F32), -7),
    (lambda p: setattr(p, "window", -1), -5),
    (lambda p: setattr(p, "sm_scale", float("inf")), -2),
    (lambda p: setattr(p, "sm_scale", 3e38), -2),
    (lambda p: setattr(p, "q", None), -1),
    (lambda p: setattr(p, "q", 0x1008), -4),
    (lambda p: setattr(p, "q_stride_h", 129), -4),
    (lambda p: setattr(p, "q_stride_b", -8), -2),
    (lambda p: setattr(p.k, "ptr", None), -1),
    (lambda p: setattr(p.v, "ptr", 0x4002), -4),
    (lambda p: setattr(p.v, "stride_token", 516), -4),
    (lambda p: setattr(p.k, "stride_token", 1 << 28), -2),  # the last token of a page beyond 2^31 elements
    (lambda p: setattr(p.k, "stride_head", -128), -2),
    (lambda p: setattr(p.table, "ptr", None), -1),
    (lambda p: setattr(p.table, "ptr", TABLE + 2), -4),
    (lambda p: setattr(p.table, "page_size", 8), -2),
    (lambda p: setattr(p.table, "page_size", 48), -2),
    (lambda p: setattr(p.table, "page_size", 1 << 17), -2),
    (lambda p: setattr(p.table, "width", 0), -2),
    (lambda p: setattr(p.table, "n_pages", 0), -2),
    (lambda p: setattr(p.table, "stride_b", 63), -2),
    (lambda p: (setattr(p.table, "width", 1 << 27), setattr(p.table, "stride_b", 1 << 27)), -2),  # more than 2^30 tokens
    (lambda p: setattr(p, "lengths", None), -1),
    (lambda p: setattr(p, "lengths", LENGTHS + 1), -4),
    (lambda p: setattr(p, "pages", 0x50000), -2),  # none of them
    (lambda p: (setattr(p, "pages", 0x50000), setattr(p, "n_pages_read", 1 << 27)), -2),
    (lambda p: (setattr(p, "B", 4096), setattr(p, "H", 1024), setattr(p.table, "width", 1 << 18), setattr(p.table, "stride_b", 1 << 18),
                setattr(p, "group", 1)), -8),
])
def test_attention_rejects_bad_parameters(lib, change, code):
    p = _params()
    change(p)
    assert lib.ra_paged_attention(C.byref(p), 0x6000, 0x7000, WORK, 1 << 40, None) == code
    assert lib.ra_last_error() != b""


def test_attention_rejects_bad_results_and_workspaces(lib):
    p = _params()
    p.table.width = p.table.stride_b = 65  # 1040 tokens: shared between workgroups
    need = lib.ra_paged_attention_workspace(C.byref(p))
    assert need > 0
    for args, code in (((None, 0x7000, WORK, need), -1), ((0x6000, None, WORK, need), -1), ((0x6002, 0x7000, WORK, need), -4),
                       ((0x6000, 0x7002, WORK, need), -4), ((0x6000, 0x7000, None, need), -1), ((0x6000, 0x7000, WORK, need - 1), -1),
                       ((0x6000, 0x7000, WORK + 4, need), -4)):
        assert lib.ra_paged_attention(C.byref(p), *args, None) == code
    p.table.width = p.table.stride_b = 32  # 512 tokens are not, and nothing is joined
    assert lib.ra_paged_attention_workspace(C.byref(p)) == 0
    assert lib.ra_paged_attention(None, 0x6000, 0x7000, None, 0, None) == -1


def test_slots_writes_means_and_selection_reject_bad_arguments(lib):
    t = _table()

    def slots(table=t, B=2, lengths=LENGTHS, ring=0x1000, out=0x2000, n=8, starts=0x3000):
        return lib.ra_page_slots(C.byref(table), lengths, LENGTHS, B, ring, 0x5000, out, n, starts, 0x7000, 0x8000, None)

    assert slots(B=0) == -2 and slots(B=4097) == -2 and slots(lengths=None) == -1 and slots(ring=None) == -1 and slots(out=None) == -1
    assert slots(out=0x2004) == -4 and slots(n=-1) == -2 and slots(starts=None) == -1 and slots(ring=0x1002) == -4
    assert slots(table=_lib.RaPageTable(TABLE, 64, 64, 1000, 24)) == -2
    pool = _lib.RaPool(0x4000, 16 * 512, 512, 128)

    def write(src=_lib.RA_DTYPE_F32, T=4, H=4, D=128, k=0x1000, ks=512, kp=pool, dtype=0, pages=10, size=16, slots=0x2000):
        return lib.ra_write_pages(k, ks, 128, 0x9000, 512, 128, src, T, H, D, C.byref(kp), C.byref(pool), dtype, pages, size, slots, None)

    assert write(T=0) == 0  # nothing to do, nothing launched
    assert write(src=5) == -7 and write(dtype=1) == -7 and write(D=100) == -3 and write(T=-1) == -2 and write(k=None) == -1 and write(k=0x1004) == -4
    assert write(ks=4) == -4 and write(kp=_lib.RaPool(None, 0, 0, 0)) == -1 and write(pages=0) == -2 and write(size=17) == -2 and write(slots=None) == -1
    assert write(slots=0x2004) == -4 and write(T=1 << 26, H=4) == -8

    def means(kp=pool, dtype=0, B=2, out=0x1000, sp=512):
        return lib.ra_page_means(C.byref(kp), dtype, C.byref(t), LENGTHS, LENGTHS, B, 4, 128, out, sp, 128, None)

    assert means(dtype=1) == -7 and means(B=0) == -2 and means(out=None) == -1 and means(sp=12) == -4 and means(kp=_lib.RaPool(0x4001, 0, 0, 0)) == -4

    def select(q=0x1000, count=4, first=1, last=1, group=2, work=WORK, size=1 << 30, out=0x2000, table=t):
        return lib.ra_select_pages(q, 1024, 128, 0x8000, 512, 128, 0, C.byref(table), LENGTHS, 2, 4, group, 128, count, first, last, out, work, size, None)

    assert select(q=None) == -1 and select(count=0) == -2 and select(first=-1) == -2 and select(first=3, last=2) == -2 and select(group=0) == -2
    assert select(out=None) == -1 and lib.ra_select_pages_workspace(C.byref(t), 2, 4) == 0  # (few pages)
    wide = _lib.RaPageTable(TABLE, 600, 600, 1000, 16)
    assert lib.ra_select_pages_workspace(C.byref(wide), 2, 4) == 2 * 4 * 600 * 8
    assert select(work=None, table=wide) == -1 and select(size=2 * 4 * 600 * 8 - 1, table=wide) == -1 and select(work=WORK + 8, table=wide) == -4


def test_tensors_on_the_host_are_refused():
    import ring_attention as ra

    z = torch.zeros
    table, n = z((1, 4), dtype=torch.int32), z(1, dtype=torch.int32)
    pool = z((4, 16, 2, 64), dtype=torch.bfloat16)
    for call in (lambda: ra.page_slots(table, n, n, z(4, dtype=torch.int32), z(2, dtype=torch.int32), 16, 1),
                 lambda: ra.write_pages(z(1, 2, 64), z(1, 2, 64), pool, pool, z(1, dtype=torch.int64)),
                 lambda: ra.page_means(pool, table, n, n, pool[:, 0]),
                 lambda: ra.select_pages(pool[0, :1], pool[:, 0], table, n, 16, 2),
                 lambda: ra.paged_attention(pool[0, :1], pool, pool, table, n)):
        with pytest.raises(RuntimeError, match="on the GPU only"):
            call()
    with pytest.raises(ValueError, match="causal, sliding-window and ALiBi"):
        ra.paged_attention(pool[0, :1], pool, pool, table, n, bias_fn=ra.segment_bias())
    with pytest.raises(TypeError):
        ra.page_slots(table, n, n, n, n, None, 1)


def test_oracle_keeps_every_page_once():
    rng = np.random.default_rng(0)
    P, width, size, B = 40, 8, 16, 6
    table, ring, state = np.full((B, width), -1, np.int32), rng.permutation(P).astype(np.int32), np.array([0, P], np.int32)
    lengths = np.zeros(B, np.int32)
    for _ in range(50):
        new = np.where(rng.random(B) < 0.3, 0, np.minimum(lengths + rng.integers(0, 40, B), width * size)).astype(np.int32)
        table, ring, slots, starts, lengths, state = R.page_slots(table, lengths, new, ring, state, size, 400)
        held = [int(p) for b in range(B) for p in table[b, :R.n_pages(int(lengths[b]), size)]]
        free = [int(ring[(state[0] + i) % P]) for i in range(state[1])]
        assert sorted(held + free) == list(range(P))
        live = slots[slots >= 0]
        assert len(set(live.tolist())) == len(live)


def test_numbers_from_the_host_reject_bad_arguments(lib):
    assert lib.ra_put_floats(0x1000, 0, 0x2000, None) == 0 and lib.ra_put_floats(None, 0, None, None) == 0  # nothing to do, nothing launched
    assert lib.ra_put_floats(0x1000, -1, 0x2000, None) == -2 and lib.ra_put_floats(None, 1, 0x2000, None) == -1
    assert lib.ra_put_floats(0x1000, 1, None, None) == -1 and lib.ra_put_floats(0x1002, 1, 0x2000, None) == -4 and lib.ra_put_floats(0x1000, 1, 0x2001, None) == -4


def test_numbers_from_the_host_are_as_many_as_there_are_heads(lib):
    """More would pass 31 bits in the loop over them."""
    assert lib.ra_put_floats(None, (1 << 31) - 1, None, None) == -2 and lib.ra_put_floats(None, 65536, None, None) == -2
    assert lib.ra_put_floats(None, 65535, None, None) == -1
