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
