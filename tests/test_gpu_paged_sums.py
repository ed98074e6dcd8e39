"""Sums of the paged cache's kernels, seen one weight at a time: data for which a weight, a step of keys or a part that is off by little or missing changes what comes out."""
import math

import numpy as np
import pytest
import torch

import ring_attention as ra
from oracle import paged_oracle as R

pytestmark = pytest.mark.gpu
BF16, F16 = torch.bfloat16, torch.float16
HALF_STEP = {BF16: 2.0 ** -8, F16: 2.0 ** -11}


def _ints(x):
    return torch.tensor(np.asarray(x), dtype=torch.int32, device="cuda")


def _np(t):
    return t.detach().float().cpu().numpy() if t.is_floating_point() else t.cpu().numpy()


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("d", [32, 64, 96, 128])
@pytest.mark.parametrize("width", [1, 80])
def test_weights_keep_their_32_bits(dtype, d, width):
    """Three keys a sequence: one of the largest score and no value, and two of nearly the same score with values 1 and -1, whose weights all but cancel.

    Scores are sums of two exact products that fit 24 bits: s = a c + e 2^-10 with a = 1 or 1/2, in base 2 (sm_scale = ln 2), at most 4.  A weight 2^(s - top) is off by ln 2 times the
    exponent's error, 4 (2^-23 of the scale's two roundings, 2^-24 of the product, 2^-24 of the difference), and by 2^-23 of the exponential; sums and the division by 2^-22 in all."""
    B, H, G = 64, 2, 16
    rng = np.random.default_rng(d + width)
    P = B
    k, v = (torch.full((P, 16, H, d), math.nan, dtype=dtype, device="cuda") for _ in range(2))
    k[:, :3], v[:, :3] = 0, 0
    c = torch.tensor(rng.integers(32, 120, (P, 1, H)) / 32.0, device="cuda").to(dtype)  # (1 to 3.75, seven bits)
    k[:, 1:3, :, 0] = c
    k[:, 2, :, 1] = torch.tensor(rng.integers(1, 4, (P, H)), device="cuda").to(dtype)
    k[:, 0, :, 0] = 4.0
    v[:, 1], v[:, 2] = 1.0, -1.0
    q = torch.zeros((B, H * G, d), dtype=dtype, device="cuda")
    q[:, ::2, 0], q[:, 1::2, 0], q[:, :, 1] = 1.0, 0.5, 2.0 ** -10
    table = torch.arange(P, dtype=torch.int32, device="cuda")[:, None].repeat(1, width)
    n = _ints([3] * B)
    out = ra.paged_attention(q, k, v, table, n, sm_scale=math.log(2))
    want, _, weight, _ = R.attention(_np(q), _np(k), _np(v), _np(table), _np(n), math.log(2))
    each = math.log(2) * 4 * (2.0 ** -23 + 2 * 2.0 ** -24) + 2.0 ** -23 + 2.0 ** -22
    assert (np.abs(want) < 2.0 ** -9 * weight).all() and (want != 0).all()
    assert (np.abs(_np(out) - want) <= each * weight + HALF_STEP[dtype] * np.abs(want)).all()


class Switches:
    """Keys whose score is 0 (on) or so low that their weight is 0 (off), by two independent bits of which even and odd query heads of a group see one each, and values of
    1 and -1.  Weights and all sums of them are whole numbers, exact in any order below 2^24, so that a key that is left out, read twice or taken from elsewhere changes the output,
    sum of signs / number of keys that are on, by more than its rounding.  The first token of a page is on for both.  Rows may name the same pages."""

    def __init__(self, P, size, H, d, dtype, share, seed):
        gen = torch.Generator(device="cuda")
        gen.manual_seed(seed)
        self.gen, self.size = gen, size
        bits = torch.rand((2, P, size, H), generator=gen, device="cuda") < share
        bits[:, :, 0] = True
        signs = torch.randint(0, 2, (P, size, H, d), generator=gen, device="cuda", dtype=torch.int8) * 2 - 1
        self.k, self.v = torch.zeros((P, size, H, d), dtype=dtype, device="cuda"), signs.to(dtype)
        at = torch.arange(H, device="cuda")
        self.dims = torch.stack(((7 * at + 3) % d, (7 * at + 3 + d // 2) % d))
        for bit, dim in zip(bits, self.dims):
            self.k.scatter_(3, dim.view(1, 1, H, 1).expand(P, size, H, 1), torch.where(bit, 0.0, -64.0).to(dtype)[..., None])
        self.bits, self.signs = bits, signs

    def queries(self, B, group):
        H, d = self.k.shape[2:]
        q = torch.zeros((B, H, group, d), dtype=self.k.dtype, device="cuda")
        for i in range(2):
            q[:, torch.arange(H, device="cuda"), i::2, self.dims[i]] = 64.0
        return q.reshape(B, H * group, d)

    def check(self, got, table, lengths, group):
        """One rounding of the output; its quotient's two (a reciprocal and a product) are counted with 2^-22.  The logsumexp is a logarithm of an exact number, in base 2 off by a step of
        its own, times ln 2: 2^-22 of it in all; fp16's weights are 2^15 as large, the logarithm lies in [15, 32), with steps of 2^-19, and 15 is taken off again."""
        size, (P, _, H, d) = self.size, self.k.shape
        whole = torch.stack([bit.double().sum(1) for bit in self.bits])                               # [2, P, H]
        signed = torch.stack([(bit[..., None] * self.signs).double().sum(1) for bit in self.bits])    # [2, P, H, d]
        out, lse = got[0].double().view(len(lengths), H, group, d), got[1].double().view(len(lengths), H, group)
        for b, n in enumerate(lengths):
            if n == 0:
                assert (out[b] == 0).all() and (lse[b] == -math.inf).all(), b
                continue
            full, rest = divmod(n, size)
            pages = table[b, :full].long()
            for i in range(min(2, group)):
                count, total = whole[i][pages].sum(0), signed[i][pages].sum(0)
                if rest:
                    last = int(table[b, full])
                    count = count + self.bits[i, last, :rest].double().sum(0)
                    total = total + (self.bits[i, last, :rest, :, None] * self.signs[last, :rest]).double().sum(0)
                want = (total / count[:, None])[:, None]
                step = HALF_STEP[got[0].dtype] + 2.0 ** -22
                assert ((out[b, :, i::2] - want).abs() <= step * want.abs()).all(), (b, n, i)
                off = 2.0 ** -22 * (1 + count.log()[:, None]) + (2.0 ** -19 if got[0].dtype == F16 else 0.0)
                assert ((lse[b, :, i::2] - count.log()[:, None]).abs() <= off).all(), (b, n, i)


@pytest.mark.parametrize("dtype,heads,group,d,size,lengths", [
    (BF16, 1, 1, 128, 128, [70001]),
    (BF16, 1, 3, 96, 16, [50007, 1, 0]),
    (F16, 2, 4, 64, 32, [33000, 5, 0, 12345]),
    (BF16, 1, 20, 32, 64, [1, 20000, 1, 1]),
    (F16, 16, 1, 128, 16, [8191, 100, 3001, 0, 128]),
    (BF16, 8, 2, 64, 1024, [1023, 1024, 1025, 4097]),
])
def test_every_key_of_rows_that_are_shared_counts_once(dtype, heads, group, d, size, lengths):
    """Steps at the begin and the end of a stretch, the four waves' keys, parts that are joined: each holds keys that are on, and their own signs."""
    c = Switches(max(64, 4096 // size), size, heads, d, dtype, 0.5, seed=d + size)
    width = R.n_pages(max(lengths), size) + 3
    table = torch.randint(0, c.k.shape[0], (len(lengths), width), generator=c.gen, device="cuda", dtype=torch.int32)
    q = c.queries(len(lengths), group)
    c.check(ra.paged_attention_with_lse(q, c.k, c.v, table, _ints(lengths)), table, lengths, group)


def test_stretches_that_list_their_pages_again():
    """8 x 2^20 tokens of 8 heads in pages of 16 are 524288 steps: 256 for each of 2048 workgroups, 2048 pages, and a workgroup lists 1024 at a time.  One key in 64 (and the
    first of a page of every 16 tokens) is on: some 2^16 in a row."""
    width, H, d = 1 << 16, 8, 32
    c = Switches(4096, 16, H, d, BF16, 1 / 64, seed=6)
    table = torch.randint(0, 4096, (8, width), generator=c.gen, device="cuda", dtype=torch.int32)
    lengths = [width * 16 - 5 - 16 * 300 * b for b in range(8)]
    q = c.queries(8, 2)
    c.check(ra.paged_attention_with_lse(q, c.k, c.v, table, _ints(lengths)), table, lengths, 2)


@pytest.mark.parametrize("B", [257, 1500, 4096])
@pytest.mark.parametrize("d,width", [(32, 6), (32, 700), (128, 40)])
def test_attention_of_many_rows(B, d, width):
    """More rows than a workgroup has threads, and than lengths fit its shared memory; rows taken whole, shared ones, and a table far wider than its rows."""
    c = Switches(300, 16, 2, d, BF16, 0.5, seed=B + d)
    rng = np.random.default_rng(B)
    lengths = [int(n) for n in np.where(rng.random(B) < 0.1, 0, rng.integers(1, 97, B))]
    if width > 100:
        lengths[B - 2], lengths[7] = 9001, 4444
    table = torch.randint(0, 300, (B, width), generator=c.gen, device="cuda", dtype=torch.int32)
    q = c.queries(B, 2)
    c.check(ra.paged_attention_with_lse(q, c.k, c.v, table, _ints(lengths)), table, lengths, 2)


@pytest.mark.parametrize("B", [257, 1500, 4096])
def test_means_and_choice_of_many_rows(B):
    rng = np.random.default_rng(B)
    size, width, H, d = 16, 6, 2, 32
    before = rng.integers(0, 60, B)
    after = np.where(rng.random(B) < 0.2, rng.integers(0, 96, B), before + (rng.random(B) < 0.7))
    held = [R.n_pages(int(max(x, y)), size) for x, y in zip(before, after)]
    P = sum(held) + 5
    order, at = rng.permutation(P), 0
    host = np.full((B, width), -1)
    for b, n in enumerate(held):
        host[b, :n] = order[at:at + n]
        at += n
    gen = torch.Generator(device="cuda")
    gen.manual_seed(B)
    k = torch.empty((P, size, H, d), dtype=BF16, device="cuda").normal_(generator=gen)
    means, table = torch.full((P, H, d), 7.0, dtype=BF16, device="cuda"), _ints(host)
    ra.page_means(k, table, _ints(before), _ints(after), means)
    want, got = R.page_means(_np(k), host, before, after, size), _np(means).astype(np.float64)
    changed = sorted(want)
    assert (np.delete(got, changed, 0) == 7.0).all()
    expected = np.stack([want[p] for p in changed])
    # one rounding, and sums of 16 numbers of at most 6 in 32 bits
    assert (np.abs(got[changed] - expected) <= HALF_STEP[BF16] * np.abs(expected) + 2.0 ** -24 * 6 * size).all()
    means.normal_(generator=gen)
    q = torch.empty((B, 2 * H, d), dtype=BF16, device="cuda").normal_(generator=gen)
    choice = R.select_pages(_np(q), _np(means), host, after, size, 3)
    for wide in (width, 520):
        t = torch.nn.functional.pad(table, (0, wide - width), value=-1)
        assert np.array_equal(_np(ra.select_pages(q, means, t, _ints(after), size, 3)), choice)


@pytest.mark.parametrize("heads,group", [(65535, 1), (1, 65535), (3, 21845)])
def test_the_most_heads(heads, group):
    for width in (2, 150):
        c = Switches(3, 16, heads, 32, BF16, 0.5, seed=heads)
        lengths = [20, width * 16 - 1]
        table = torch.randint(0, 3, (2, width), generator=c.gen, device="cuda", dtype=torch.int32)
        q = c.queries(2, group)
        c.check(ra.paged_attention_with_lse(q, c.k, c.v, table, _ints(lengths)), table, lengths, group)


def test_means_of_the_most_heads():
    """65531 heads of 96 are 786372 chunks: 98297 workgroups of eight of them."""
    k = torch.randint(-4, 5, (2, 16, 65531, 96), device="cuda").to(BF16)
    means = torch.zeros((2, 65531, 96), dtype=BF16, device="cuda")
    ra.page_means(k, _ints([[1, 0]]), _ints([0]), _ints([20]), means)
    for page, n in ((1, 16), (0, 4)):
        assert torch.equal(means[page], (k[page, :n].float().sum(0) / n).to(BF16))


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("d", [32, 64, 96, 128])
@pytest.mark.parametrize("width", [13, 90])
def test_values_that_are_not_finite(dtype, d, width):
    """An infinite value that counts makes its own element of the output infinite, two of different signs or one that is no number make it none, and all other elements are
    as they are without."""
    c = Switches(20, 16, 2, d, dtype, 0.5, seed=d)
    table = torch.arange(13, dtype=torch.int32, device="cuda").repeat(2, 1)
    table = torch.nn.functional.pad(table, (0, width - 13), value=-1)
    lengths, q = [200, 77], c.queries(2, 3)
    want, want_lse = ra.paged_attention_with_lse(q, c.k, c.v, table, _ints(lengths))
    v = c.v.clone()
    v[1, 0, 0, 3], v[2, 0, 1, 5], v[4, 0, 1, d - 1], v[3, 0, 0, 8], v[4, 0, 0, 8], v[2, 0, 0, 0] = math.inf, -math.inf, math.inf, math.inf, -math.inf, math.nan
    v[4, 13, 0, 4] = v[12, 8, 1, 4] = math.inf  # behind the second row's end and the first one's
    want = want.view(2, 2, 3, d)
    want[:, 0, :, 3], want[:, 1, :, 5], want[:, 1, :, d - 1], want[:, 0, :, 8], want[:, 0, :, 0] = math.inf, -math.inf, math.inf, math.nan, math.nan
    seen = c.bits[:, 4, 13, 0]  # (within the first row, by the query heads for which it is on)
    for g in range(3):
        if seen[g % 2]:
            want[0, 0, g, 4] = math.inf
        else:
            want[0, 0, g, 4] = math.nan  # (a weight of 0 times infinity)
    got, lse = ra.paged_attention_with_lse(q, c.k, v, table, _ints(lengths))
    assert torch.equal(lse, want_lse) and torch.allclose(got.view_as(want), want, rtol=0, atol=0, equal_nan=True)
