"""Plain forms in 64 bits of the terms that take arguments of their own: the relative position bias by buckets and dropout of the
attention weights, with the gradients and with how far results in 16 bits may be off.

All arrays are torch tensors, on any device; q, k, v, do are [b, l, h, d], what the kernels see of them (rounded to 16 bits already).
"""
import math

import torch


def bucket_starts(side, max_distance):
    """Least distance of each bucket of a side, by brute force over the whole numbers."""
    exact, starts, n = side // 2, [], 0
    k = side - exact
    for b in range(side):
        if b <= exact:
            n = b
        else:
            i = b - exact
            while n ** k * exact ** i < max_distance ** i * exact ** k:
                n += 1
        starts.append(n)
    return starts


def bucket_of(distance, num_buckets, max_distance, bidirectional):
    """Bucket of key position - query position, elementwise."""
    side = num_buckets // 2 if bidirectional else num_buckets
    starts = torch.tensor(bucket_starts(side, max_distance), device=distance.device)
    n = distance.abs() if bidirectional else (-distance).clamp(min=0)
    b = torch.searchsorted(starts, n.contiguous(), right=True) - 1
    return b + side * (distance > 0) if bidirectional else b


def philox(counter, key, rounds):
    """Philox 4x32 on int64 tensors (or ints) of 32-bit words."""
    c, k = list(counter), list(key)
    low = 0xFFFFFFFF
    for _ in range(rounds):
        a, b = c[0] * 0xD2511F53, c[2] * 0xCD9E8D57  # (int64 products wrap: the shift and the mask take the right bits all the same)
        c = [((b >> 32) & low) ^ c[1] ^ k[0], b & low, ((a >> 32) & low) ^ c[3] ^ k[1], a & low]
        k = [(k[0] + 0x9E3779B9) & low, (k[1] + 0xBB67AE85) & low]
    return c


def keep_mask(seed, threshold, B, H, Sq, Sk, device="cpu"):
    """Which weights dropout leaves, [b, h, sq, sk]."""
    i = torch.arange(Sq, device=device)[None, :, None]
    j = torch.arange(Sk, device=device)[None, None, :]
    hh = torch.arange(B * H, device=device)[:, None, None]
    zero = torch.zeros((B * H, Sq, Sk), dtype=torch.int64, device=device)
    w = philox((zero + j // 2, zero + i // 4, zero + hh, zero), (seed & 0xFFFFFFFF, (seed >> 32) & 0xFFFFFFFF), 7)
    word = torch.stack(w).gather(0, (zero + i % 4)[None])[0]
    return (((word >> 16 * (zero + j % 2)) & 0xFFFF) >= threshold).reshape(B, H, Sq, Sk)


def scores_mask(Sq, Sk, q_off=0, kv_off=0, causal=False, window=None, prefix=None, segments=None, device="cpu"):
    """Which pairs take part, [b | 1, 1, sq, sk].  prefix, segments: (q side [b, sq], kv side [b, sk])."""
    qp = q_off + torch.arange(Sq, device=device)[:, None]
    kp = kv_off + torch.arange(Sk, device=device)[None]
    live = torch.ones((1, 1, Sq, Sk), dtype=torch.bool, device=device)
    if causal:
        live = live & (kp <= qp)
    if window is not None:
        live = live & ((qp - kp < window) if causal else ((qp - kp).abs() < window))
    if prefix is not None:
        q, k = (x.to(device) != 0 for x in prefix)
        live = live & ((q[:, :, None] & k[:, None])[:, None] | (kp <= qp))
    if segments is not None:
        q, k = (x.to(device) for x in segments)
        live = live & (q[:, :, None] == k[:, None])[:, None]
    return live


class Attention:
    """Forward, gradients, and bounds on how far kernels may be off that round each weight, each dS and each result to 16 bits (`eps`: of that
    type) and do everything else in 32 bits."""

    def __init__(self, q, k, v, *, do=None, scale=None, live=None, bias=None, keep=None, threshold=0, eps=2.0 ** -7):
        u = eps / 2
        q, k, v = (x.double().permute(0, 2, 1, 3) for x in (q, k, v))
        D = q.shape[3]
        scale = D ** -0.5 if scale is None else scale
        raw = q @ k.transpose(2, 3) * scale
        s = raw if bias is None else raw + bias
        if live is not None:
            s = s.masked_fill(~live, -math.inf)
        self.dead = (s == -math.inf).all(3)
        self.lse = torch.logsumexp(s, 3)
        P = torch.exp(s - self.lse.masked_fill(self.dead, 0.0)[..., None])
        f = 1.0 if keep is None else 1 - threshold / 65536
        Z = 1.0 if keep is None else keep.double() / f
        W = P * Z
        self.P, self.keep = P, keep
        # 32-bit sums of products: what they may add to a score, and so (relatively) to a weight
        size = (q.abs() @ k.abs().transpose(2, 3)).amax() * scale + (0 if bias is None else bias.masked_fill(torch.isinf(bias), 0.0).abs().amax())
        e32 = 2.0 ** -23
        self.e_w = float((D + 32) * e32 * size + 64 * e32)
        e = u + self.e_w
        n32 = k.shape[2] * e32
        absout = W @ v.abs()
        o = W @ v
        d_o = (2 * e + n32) * absout
        self.out, self.out_off = o.permute(0, 2, 1, 3), (u * o.abs() + d_o).permute(0, 2, 1, 3) + 1e-30
        self.lse_off = self.e_w * 2 + 4 * e32 * self.lse.abs().masked_fill(self.dead, 0.0) + n32
        if do is None:
            return
        do = do.double().permute(0, 2, 1, 3).masked_fill(self.dead[..., None], 0.0)
        dW = do @ v.transpose(2, 3)
        absdW = do.abs() @ v.abs().transpose(2, 3)
        delta = (do * o).sum(3, keepdim=True)
        # the output enters delta in 16 bits twice over: what it lacks is kept as well
        d_delta = (do.abs() * (d_o + eps * u * o.abs())).sum(3, keepdim=True) + D * e32 * (do.abs() * o.abs()).sum(3, keepdim=True)
        dS = P * (Z * dW - delta)
        off = P * (d_delta + (self.e_w + D * e32) * (Z * absdW + delta.abs()))  # of dS in 32 bits
        dS_off = off + u * dS.abs()
        n32q = q.shape[2] * e32

        def grad(x, xoff):
            return x.permute(0, 2, 1, 3), (u * x.abs() + xoff).permute(0, 2, 1, 3) + 1e-30

        self.dq, self.dq_off = grad(dS @ k * scale, (dS_off + n32 * dS.abs()) @ k.abs() * scale)
        self.dk, self.dk_off = grad(dS.transpose(2, 3) @ q * scale, (dS_off + n32q * dS.abs()).transpose(2, 3) @ q.abs() * scale)
        self.dv, self.dv_off = grad(W.transpose(2, 3) @ do, (e + n32q) * (W.transpose(2, 3) @ do.abs()))
        self.dS, self.dS_off32 = dS, off

    def table_gradient(self, bucket, num_buckets, eps, own=False):
        """[num_buckets, h] sums of dS, and their bounds: of all pairs together, or of a bucket's own."""
        n = self.dS.shape[2] * self.dS.shape[3] * self.dS.shape[0]
        e_sum = 2.0 ** -24 * (math.log2(n) + 64)  # sums of sums, at most so deep each
        got, off = [], []
        for u in range(num_buckets):
            at = bucket == u
            got.append(self.dS[:, :, at].sum((0, 2)))
            off.append((self.dS_off32 + 64 * e_sum * self.dS.abs())[:, :, at].sum((0, 2)))
        got, off = torch.stack(got), torch.stack(off)
        return got, (off if own else off.sum(0, keepdim=True)) + eps / 2 * got.abs() + (1e-36 if own else 1e-30)
