"""fp16 calls with a relative bias or dropout where dS or the weights lie outside fp16's range, and the gradients inside it."""
import math

import pytest
import torch

import ring_attention as ra
from oracle import terms_oracle as T
from test_gpu_terms import EPS, Case

pytestmark = pytest.mark.gpu

HALF = EPS[torch.float16]
FORMS = [dict(relative="both"), dict(relative=None, p=0.2), dict(relative="both", p=0.2)]


def _case(device, q=1.0, k=1.0, v=1.0, do=1.0, **kw):
    """A case whose arrays are scaled by powers of two (no rounding of their own, where that leaves normal numbers)."""
    c = Case(device, dtype=torch.float16, **kw)
    c.q, c.k, c.v, c.do = c.q * q, c.k * k, c.v * v, c.do * do
    return c


def _near(name, got, want, dim=None):
    """In norm, of all elements or along `dim`: fewer than twelve roundings to half a step each, independent, in rms at most eps / 2 / sqrt(3) apiece; a
    result below 2^-14 is off by up to 2^-25 of its own."""
    assert torch.isfinite(got).all(), name
    got = got.double()
    dims = tuple(range(got.dim())) if dim is None else dim
    n = got.numel() / want.sum(dims).numel()
    off = torch.linalg.vector_norm(got - want, dim=dims)
    room = HALF * torch.linalg.vector_norm(want, dim=dims) + 2.0 ** -25 * n ** 0.5
    assert (off <= room).all(), (name, float((off / torch.linalg.vector_norm(want, dim=dims)).max()))


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("D,mask", [(64, "none"), (128, "causal"), (96, "none")])
@pytest.mark.parametrize("do", [2.0 ** -10, 2.0 ** -13, 2.0 ** -17])
def test_small_output_gradients(device, form, D, mask, do):
    """Without loss scaling: dO of 1e-3, 1e-4 and 1e-5, so that dS is next to or below fp16's smallest number, and keys or queries that bring the gradient back
    into the range."""
    for q, k, name in ((2.0 ** -6, 64.0, "dq"), (64.0, 2.0 ** -6, "dk")):
        c = _case(device, H=2, Sq=1500, D=D, mask=mask, q=q, k=k, do=do, **form)
        w, grads = c.want(), c.grads()[2]
        _near(name, grads["dq dk".split().index(name)], getattr(w, name))


@pytest.mark.parametrize("form", FORMS)
def test_large_output_gradients(device, form):
    """dS above fp16's largest number (1e5: first rows of a causal call, weights of a half), the gradients below it."""
    c = _case(device, H=2, Sq=70, D=64, mask="causal", q=0.125, k=0.125, v=256.0, do=256.0, **form)
    w = c.want()
    assert float(w.dS.abs().max()) > 65504
    _, _, grads = c.grads()
    for name, got in zip(("dq", "dk", "dv"), grads):
        assert float(getattr(w, name).abs().max()) < 60000
        _near(name, got, getattr(w, name))


@pytest.mark.parametrize("form", FORMS)
def test_small_weights(device, form):
    """Weights of one key in 131072 (8e-6), below fp16's normal numbers: dV."""
    c = _case(device, H=1, Sq=96, Sk=131072, D=32, do=256.0, **form)
    _near("dv", c.grads()[2][2], c.want().dv)


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("way", [1, -1])
def test_output_gradients_of_many_sizes(device, form, D, way):
    """dO that grows or shrinks by 2^20 along the rows: each row of dQ to its own size, dK with the largest's, however late it comes."""
    Sq = 1300
    sizes = torch.exp2(-torch.linspace(0, 20, Sq, device=device).round() + 6)
    sizes = sizes.flip(0) if way > 0 else sizes
    c = _case(device, H=2, Sq=Sq, Sk=900, D=D, q=2.0 ** -8, k=256.0, **form)
    c.do = (c.do.float() * sizes[None, :, None, None]).half()
    _near("dq", c.grads()[2][0], c.want().dq, dim=3)
    c = _case(device, H=2, Sq=Sq, Sk=900, D=D, q=16.0, k=0.0625, **form)
    c.do = (c.do.float() * sizes[None, :, None, None]).half()
    w, grads = c.want(), c.grads()[2]
    _near("dk", grads[1], w.dk)
    _near("dv", grads[2], w.dv)


@pytest.mark.parametrize("form", FORMS)
def test_keys_and_values_of_many_sizes(device, form):
    """Values that grow by 2^16 along the keys, so that dS does inside every row."""
    c = _case(device, H=2, Sq=200, Sk=1100, D=64, **form)
    sizes = torch.exp2(torch.linspace(-8, 8, 1100, device=device).round())
    c.v = (c.v.float() * sizes[None, :, None, None]).half()
    c.k = c.k * 4
    c.q = c.q / 4
    w, grads = c.want(), c.grads()[2]
    for name, got in zip(("dq", "dk", "dv"), grads):
        _near(name, got, getattr(w, name))


@pytest.mark.parametrize("form", FORMS)
def test_no_output_gradient_and_an_infinite_one(device, form):
    """Zeros give zeros; a row of infinities reaches that row of dQ, and no other."""
    c = _case(device, H=2, Sq=150, Sk=300, **form)
    c.do = torch.zeros_like(c.do)
    assert all(not g.any() for g in c.grads()[2])
    c.do = torch.randn(c.do.shape, generator=torch.Generator().manual_seed(1)).to(device, torch.float16)
    w = c.want()
    c.do[0, 77] = torch.inf
    dq = c.grads()[2][0]
    assert not torch.isfinite(dq[0, 77]).any()
    others = torch.arange(150, device=device) != 77
    _near("dq", dq[:, others], w.dq[:, others])


@pytest.mark.parametrize("sink", [0, 70000, 131071])
@pytest.mark.parametrize("relative,p", [(True, 0.0), (False, 0.2), (True, 0.2)])
def test_many_small_weights_beside_a_large_one(device, sink, relative, p):
    """131072 keys of 2^-26 of one key's weight are 2e-3 of a row, of so many rows that each stays with one workgroup.  A weight is off by 2^-31 of the largest
    at most (half of 2^-24, the largest being 2^6 or more), divided by what dropout leaves."""
    n, H, Sq = 131072, 8, 16384
    q, k, v = (torch.zeros(1, S, H, 64, device=device, dtype=torch.float16) for S in (Sq, n, n))
    q[..., 0] = 1
    k[:, sink, :, 0] = 18.015625
    v[:] = 1
    v[:, sink] = 0
    fn = ra.relative_bias(torch.zeros(32, H, device=device)) if relative else None
    out, lse = ra.ring_attention_with_lse(q, k, v, 1, fn, sm_scale=1.0, dropout=ra.Dropout(p, 5) if p else None)
    small = math.exp(-18.015625)
    total = 1 + (n - 1) * small
    # (a logsumexp of 18: steps of 2^-19, and of the sums and exponentials some 2^-18)
    assert ((lse.double() - (18.015625 + math.log(total))).abs() <= 2.0 ** -16).all()
    i, j = torch.tensor([0, 77, 9000, Sq - 1], device=device)[:, None], torch.arange(n, device=device)[None]
    zero = torch.zeros_like(i * j)
    for h in (0, H - 1):
        kept = torch.ones_like(zero)
        if p:
            word = torch.stack(T.philox((zero + j // 2, zero + i // 4, zero + h, zero), (5, 0), 7)).gather(0, (zero + i % 4)[None])[0]
            kept = ((word >> 16 * (zero + j % 2)) & 0xFFFF) >= round(p * 65536)
        kept[:, sink] = 0
        want = kept.sum(1).double() * small / total / (1 - round(p * 65536) / 65536)
        got = out[0, i[:, 0], h].double()
        assert ((got - want[:, None]).abs() <= HALF * want[:, None] + 2.0 ** -25 + n * 2.0 ** -31 / (1 - p)).all(), (got[:, 0], want)
