"""The learned relative position bias and attention dropout: what a program that uses them has this package compute.

A case is one call of ``ring_attention`` as such a program makes it, with a learned bias by buckets of the distance
between query and key (``relative``), with dropout of the attention weights (``p``), or with both:

* ``forward``  inference: output and logsumexp, of a whole sequence, of a chunk behind a context that is already there,
               or of a single token (``q_len`` = 1);
* ``train``    a training step's attention: the output and the gradients of q, k, v and, under a bias, of its table.

``mask`` is the rest of the bias.  Under ``causal`` the queries are the last ``q_len`` of ``kv_len`` positions; under
``padded`` too, and the sequences of the batch start behind padding of various lengths, as in batched generation.

Where ``own`` is false the operators are computed from elementary operations in 32 bits, the scores held whole.
"""
import math
import os
import sys

import torch

own = False

_DTYPES = {"bfloat16": torch.bfloat16, "float16": torch.float16}


def _case(path, mask, dtype, batch, heads, dim, q_len, kv_len, ring, *, relative="none", buckets=0, distance=0, p=0.0, mean_document=0,
          name=None):
    c = dict(path=path, mask=mask, dtype=dtype, batch=batch, heads=heads, dim=dim, q_len=q_len, kv_len=kv_len, ring=ring,
             relative=relative, buckets=buckets, distance=distance, p=p, mean_document=mean_document)
    return c if name is None else dict(c, name=name)


def listed():
    one = dict(relative="one-sided", buckets=32, distance=128)
    both = dict(relative="bidirectional", buckets=32, distance=128)
    return [
        # the smallest call: the next token of a small decoder with a bias, behind a short prompt, where latency counts
        _case("forward", "causal", "bfloat16", 1, 8, 64, 1, 1000, 1, **one, name="bias_token_1k"),
        # batched generation: a token each behind caches of different lengths
        _case("forward", "padded", "bfloat16", 4, 16, 128, 1, 32768, 1, **one, name="bias_token_32k_padded"),
        # an encoder's output over two sequences of different lengths that fit no tile, a head dim that needs padding, wide buckets
        _case("forward", "none", "float16", 2, 8, 80, 1047, 4791, 3, relative="bidirectional", buckets=64, distance=800,
              name="bias_forward_cross_ragged"),
        # fine-tuning a small encoder on sequences of an odd length
        _case("train", "none", "float16", 4, 12, 64, 771, 771, 1, **both, name="bias_train_771"),
        # training a small decoder
        _case("train", "causal", "bfloat16", 2, 16, 64, 4096, 4096, 4, **one, name="bias_train_4k"),
        # training an encoder of wide heads on packed documents
        _case("train", "documents", "bfloat16", 1, 16, 128, 8192, 8192, 4, **both, mean_document=1024, name="bias_train_8k_packed"),
        # the smallest training call with dropout: a short sequence on a small model
        _case("train", "causal", "bfloat16", 1, 4, 64, 512, 512, 1, p=0.1, name="dropout_train_512"),
        # cross attention of sequences that fit no tile, more dropout, fp16
        _case("train", "none", "float16", 2, 8, 96, 1047, 4791, 3, p=0.25, name="dropout_train_cross_ragged"),
        # training on packed documents, head dim 64
        _case("train", "causal+documents", "bfloat16", 2, 16, 64, 4096, 4096, 2, p=0.1, mean_document=1024, name="dropout_train_4k_packed"),
        # the largest: training at 8192 tokens, 8 shards of 1024
        _case("train", "causal", "bfloat16", 1, 16, 128, 8192, 8192, 8, p=0.1, name="dropout_train_8k"),
        # both, as encoders and decoders with a learned bias train: short sequences in a large batch, then long ones
        _case("train", "none", "bfloat16", 16, 12, 64, 512, 512, 1, **both, p=0.1, name="both_train_512"),
        _case("train", "causal", "bfloat16", 1, 16, 128, 4096, 4096, 4, **one, p=0.1, name="both_train_4k"),
    ]


def draw(rng):
    """One more case of the ranges above: lengths spread over their logarithm, most of them odd."""
    def spread(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    every = listed()
    most = max(work(c)["flops"] for c in every)
    most_bytes = max(work(c)["bytes"] for c in every)
    most_scores = max(c["batch"] * c["heads"] * c["q_len"] * c["kv_len"] for c in every)
    while True:
        what = rng.choice(["bias", "bias", "dropout", "both"])
        path = "train" if what != "bias" else rng.choice(["train", "forward"])
        ring = rng.choice([1, 1, 2, 3, 4, 8])
        heads, batch = rng.choice([4, 5, 8, 12, 16]), rng.choice([1, 1, 2, 3, 4, 16])
        dim = rng.choice([64, 64, 64, 128, 128, 96, 80, 32])
        length = ring * spread(max(8, 128 // ring), 8192 // ring)
        q_len, extra = length, {}
        mask = rng.choice(["causal", "causal", "none", "documents", "causal+documents"])
        if path == "forward" and rng.random() < 0.7:
            # a chunk or a token behind a context
            mask, ring = rng.choice(["causal", "padded"]), 1
            length = spread(300, 32768)
            q_len = rng.choice([1, 1, spread(2, 256)])
        elif mask == "none" and rng.random() < 0.5:
            q_len = ring * spread(16, length // ring)
        if "documents" in mask:
            extra["mean_document"] = spread(64, 2048)
        if what != "dropout":
            extra["relative"] = rng.choice(["one-sided", "bidirectional"]) if mask in ("causal", "causal+documents", "padded") else "bidirectional"
            extra["buckets"] = rng.choice([32, 32, 16, 64])
            extra["distance"] = rng.choice([128, 128, spread(40, 2000)])
        if what != "bias":
            extra["p"] = rng.choice([0.1, 0.1, round(rng.uniform(0.01, 0.5), 3)])
        c = _case(path, mask, rng.choice(["bfloat16", "bfloat16", "float16"]), batch, heads, dim, q_len, length, ring, **extra)
        w = work(c)
        if w["flops"] <= most and w["bytes"] <= most_bytes and batch * heads * q_len * length <= most_scores:
            return c


def prepare(case, seed):
    B, H, D, Sq, Sk = (case[x] for x in ("batch", "heads", "dim", "q_len", "kv_len"))
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    dtype = _DTYPES[case["dtype"]]

    def normal(*shape, std=1.0):
        return torch.empty(shape, device="cuda", dtype=dtype).normal_(0.0, std, generator=gen)

    s = dict(case=case, q=normal(B, Sq, H, D), k=normal(B, Sk, H, D), v=normal(B, Sk, H, D), table=None, q_ids=None, kv_ids=None)
    if case["relative"] != "none":
        s["table"] = normal(case["buckets"], H)
    if case["path"] == "train":
        s["do"] = normal(B, Sq, H, D)
        for x in ("q", "k", "v", "table"):
            if s[x] is not None:
                s[x].requires_grad_(True)
    if "documents" in case["mask"]:
        starts = torch.rand((B, Sk), generator=gen, device="cuda") < 1.0 / case["mean_document"]
        starts[:, 0] = False
        s["q_ids"] = s["kv_ids"] = starts.to(torch.int32).cumsum(1, dtype=torch.int32)
    elif case["mask"] == "padded":
        # padding of up to three quarters of the cache
        pad = torch.randint(0, max(1, 3 * (Sk - Sq) // 4), (B, 1), generator=gen, device="cuda")
        s["kv_ids"] = (torch.arange(Sk, device="cuda")[None] >= pad).to(torch.int32)
        s["q_ids"] = torch.ones((B, Sq), dtype=torch.int32, device="cuda")
    # a step's seed
    s["seed"] = (seed * 0x9E3779B97F4A7C15 + 0x1234567) % (1 << 63)
    return s


def _offset(case):
    """The position of the first query (the first key's is 0)."""
    return case["kv_len"] - case["q_len"] if "causal" in case["mask"] or case["mask"] == "padded" else 0


def _bucket_starts(case):
    """The least distance of each bucket of one side, in whole numbers: half of the buckets hold one distance each, the rest
    grow by a constant factor up to the largest distance."""
    side = case["buckets"] // (2 if case["relative"] == "bidirectional" else 1)
    exact_ones = side // 2
    steps = side - exact_ones
    starts = list(range(exact_ones + 1))
    n = exact_ones
    for i in range(1, steps):
        while n ** steps * exact_ones ** i < case["distance"] ** i * exact_ones ** steps:
            n += 1
        starts.append(n)
    return starts


def _buckets(case, relative):
    """Bucket of each of the (key - query) distances in a tensor."""
    side = case["buckets"] // (2 if case["relative"] == "bidirectional" else 1)
    starts = torch.tensor(_bucket_starts(case), device=relative.device)
    if case["relative"] == "bidirectional":
        n, base = relative.abs(), torch.where(relative > 0, side, 0)
    else:
        n, base = (-relative).clamp(min=0), 0
    return (n[:, None] >= starts).sum(1) - 1 + base


def _live(s):
    """Which (query, key) pairs take part, [b | 1, 1, q, k]; None for all."""
    case = s["case"]
    Sq, Sk = case["q_len"], case["kv_len"]
    live = None
    if "causal" in case["mask"] or case["mask"] == "padded":
        at = torch.arange(Sk, device="cuda")
        live = (at[None] <= at[:Sq, None] + _offset(case))[None, None]
    if s["kv_ids"] is not None:
        same = (s["q_ids"][:, :, None] == s["kv_ids"][:, None, :])[:, None]
        live = same if live is None else live & same
    return live


_MASK32 = 0xFFFFFFFF


def _keep(s):
    """Which weights dropout leaves, [b, h, q, k], and the fraction of them: 16 random bits each, Philox-4x32 of 7 rounds, a call for four
    queries of two keys."""
    case = s["case"]
    B, H, Sq, Sk = (case[x] for x in ("batch", "heads", "q_len", "kv_len"))
    threshold = int(round(case["p"] * 65536))
    n_q, n_k = (Sq + 3) // 4, (Sk + 1) // 2
    c0 = torch.arange(n_k, device="cuda")[None, None, :]
    c1 = torch.arange(n_q, device="cuda")[None, :, None]
    c2 = torch.arange(B * H, device="cuda")[:, None, None]
    c3 = torch.zeros((1, 1, 1), dtype=torch.int64, device="cuda")
    k0, k1 = s["seed"] & _MASK32, s["seed"] >> 32
    for _ in range(7):
        a, b = c0 * 0xD2511F53, c2 * 0xCD9E8D57
        c0, c1, c2, c3 = ((b >> 32) & _MASK32) ^ c1 ^ k0, b & _MASK32, ((a >> 32) & _MASK32) ^ c3 ^ k1, a & _MASK32
        k0, k1 = (k0 + 0x9E3779B9) & _MASK32, (k1 + 0xBB67AE85) & _MASK32
    halves = [torch.stack(((w & 0xFFFF) >= threshold, (w >> 16) >= threshold), dim=-1) for w in torch.broadcast_tensors(c0, c1, c2, c3)]
    keep = torch.stack(halves, dim=2).reshape(B, H, 4 * n_q, 2 * n_k)
    return keep[:, :, :Sq, :Sk], 1.0 - threshold / 65536


def _heads_first(x):
    return x.detach().float().permute(0, 2, 1, 3).contiguous()


def _run_plain(s):
    case = s["case"]
    Sq, Sk = case["q_len"], case["kv_len"]
    scale = 1.0 / math.sqrt(case["dim"])
    q, k, v = _heads_first(s["q"]), _heads_first(s["k"]), _heads_first(s["v"])
    scores = torch.matmul(q, k.transpose(2, 3)).mul_(scale)
    bucket = None
    if s["table"] is not None:
        # by distance first: it is the same along a diagonal
        bucket = _buckets(case, torch.arange(1 - Sq, Sk, device="cuda") - _offset(case))
        at = torch.arange(Sk, device="cuda")[None] - torch.arange(Sq, device="cuda")[:, None] + (Sq - 1)
        scores += s["table"].detach().float()[bucket].t().contiguous()[:, at]
    live = _live(s)
    if live is not None:
        scores.masked_fill_(~live, -math.inf)
    top = scores.amax(3, keepdim=True)
    weights = (scores - top).exp_()
    total = weights.sum(3, keepdim=True)
    weights /= total
    lse = (top + total.log()).squeeze(3)
    kept = weights
    if case["p"]:
        keep, fraction = _keep(s)
        kept = weights * keep / fraction
    out = torch.matmul(kept, v)

    def as_given(x):
        return x.permute(0, 2, 1, 3).to(s["q"].dtype)

    if case["path"] == "forward":
        return as_given(out), lse
    do = _heads_first(s["do"])
    dv = torch.matmul(kept.transpose(2, 3), do)
    ds = torch.matmul(do, v.transpose(2, 3))
    if case["p"]:
        ds = ds * keep / fraction
    ds = (ds - (do * out).sum(3, keepdim=True)).mul_(weights)
    grads = [as_given(torch.matmul(ds, k).mul_(scale)), as_given(torch.matmul(ds.transpose(2, 3), q).mul_(scale)), as_given(dv)]
    if bucket is not None:
        # sums over the diagonals, each a column once every row is shifted by one against the next
        rows = torch.nn.functional.pad(ds.sum(0).flip(1), (0, Sq)).reshape(case["heads"], -1)
        diagonals = rows[:, :Sq * (Sq + Sk - 1)].reshape(-1, Sq, Sq + Sk - 1).sum(1, dtype=torch.float64)
        of_bucket = bucket[:, None] == torch.arange(case["buckets"], device="cuda")
        grads.append(torch.matmul(diagonals, of_bucket.double()).t().to(s["table"].dtype))
    return as_given(out), grads


def _package():
    at = os.path.abspath("ring-attention-jax-pallas_amd")
    if at not in sys.path:
        sys.path.insert(1, at)
    import ring_attention
    return ring_attention


def _run_own(s):
    ra = _package()
    case = s["case"]
    bias, q_kw, kv_kw = None, {}, {}
    if "causal" in case["mask"] or case["mask"] == "padded":
        bias = ra.causal_bias()
        if _offset(case):
            q_kw["q_positions"] = _offset(case)  # of the first query, the others follow
    if s["kv_ids"] is not None:
        bias = ra.segment_bias() if bias is None else bias + ra.segment_bias()
        q_kw["q_segment_ids"], kv_kw["kv_segment_ids"] = s["q_ids"], s["kv_ids"]
    if s["table"] is not None:
        term = ra.relative_bias(s["table"], max_distance=case["distance"], bidirectional=case["relative"] == "bidirectional")
        bias = term if bias is None else bias + term
    dropout = ra.Dropout(case["p"], s["seed"]) if case["p"] else None
    axis = ra.RingAxis("sp", case["ring"])
    if case["path"] == "forward":
        return ra.ring_attention_with_lse(s["q"], s["k"], s["v"], axis, bias, q_kw, kv_kw, dropout=dropout)
    out = ra.ring_attention(s["q"], s["k"], s["v"], axis, bias, q_kw, kv_kw, dropout=dropout)
    wrt = [s[x] for x in ("q", "k", "v", "table") if s[x] is not None]
    return out, list(torch.autograd.grad(out, wrt, s["do"]))


def run(state):
    return _run_own(state) if own else _run_plain(state)


def _exact_keep(case, seed, head):
    """Dropout's mask of one (batch, head), 16 bits of a Philox word for each (query, key), word by word; products by 16-bit parts."""
    i = torch.arange(case["q_len"], device="cuda")[:, None]
    j = torch.arange(case["kv_len"], device="cuda")[None, :]
    x = [(j // 2).expand(len(i), -1), (i // 4).expand(-1, j.shape[1]), torch.full_like(i * j, head), torch.zeros_like(i * j)]
    key = [seed % 2 ** 32, seed // 2 ** 32]

    def product(m, y):  # high and low word
        low, high = m % 65536 * y, m // 65536 * y
        t = low // 65536 + high % 65536
        return high // 65536 + t // 65536, low % 65536 + t % 65536 * 65536

    for r in range(7):
        h0, l0 = product(0xD2511F53, x[0])
        h1, l1 = product(0xCD9E8D57, x[2])
        x = [h1 ^ x[1] ^ (key[0] + r * 0x9E3779B9) % 2 ** 32, l1, h0 ^ x[3] ^ (key[1] + r * 0xBB67AE85) % 2 ** 32, l0]
    word = torch.where(i % 4 < 2, torch.where(i % 2 == 0, x[0], x[1]), torch.where(i % 2 == 0, x[2], x[3]))
    bits = torch.where(j % 2 == 0, word % 65536, word // 65536)
    t = round(case["p"] * 65536)
    return (bits >= t).double() * (65536 / (65536 - t))


def exact(case, seed):
    """One (batch, head) after the other, in 64 bits."""
    s = prepare(case, seed)
    B, H, D, Sq, Sk = (case[x] for x in ("batch", "heads", "dim", "q_len", "kv_len"))
    position = torch.arange(Sq, device="cuda")[:, None] + _offset(case)
    key_position = torch.arange(Sk, device="cuda")[None, :]
    far = key_position - position
    bucket = None
    if case["relative"] != "none":
        two = case["relative"] == "bidirectional"
        side = case["buckets"] // 2 if two else case["buckets"]
        small = side // 2
        n = far.abs() if two else (-far).clamp(min=0)
        # logarithmic beyond the first half; a distance next to a border goes by whole numbers
        grown = torch.log(n.double().clamp(min=1) / small) / math.log(case["distance"] / small) * (side - small)
        up = torch.floor(grown + 1e-9)
        bucket = torch.where(n < small, n, (small + up.long()).clamp(max=side - 1))
        if two:
            bucket = bucket + side * (far > 0)
    out, lse = torch.empty_like(s["q"], dtype=torch.float64), torch.empty((B, H, Sq), dtype=torch.float64, device="cuda")
    train = case["path"] == "train"
    if train:
        dq, dk, dv = (torch.empty_like(s[x], dtype=torch.float64) for x in "qkv")
        dt = torch.zeros((max(case["buckets"], 1), H), dtype=torch.float64, device="cuda")
    with torch.no_grad():
        for b in range(B):
            for h in range(H):
                q, k, v = (s[x][b, :, h].double() for x in "qkv")
                t = q @ k.t() / math.sqrt(D)
                if bucket is not None:
                    t += s["table"][:, h].double()[bucket]
                hidden = far > 0 if ("causal" in case["mask"] or case["mask"] == "padded") else torch.zeros_like(far, dtype=torch.bool)
                if s["kv_ids"] is not None:
                    hidden = hidden | (s["q_ids"][b][:, None] != s["kv_ids"][b][None, :])
                t[hidden] = -math.inf
                lse[b, h] = torch.logsumexp(t, 1)
                w = torch.exp(t - lse[b, h][:, None])
                keep = _exact_keep(case, s["seed"], b * H + h) if case["p"] else None
                used = w * keep if keep is not None else w
                out[b, :, h] = used @ v
                if not train:
                    continue
                do = s["do"][b, :, h].double()
                dv[b, :, h] = used.t() @ do
                dw = do @ v.t()
                if keep is not None:
                    dw *= keep
                dt_h = w * (dw - (dw * w).sum(1, keepdim=True))
                dq[b, :, h] = dt_h @ k / math.sqrt(D)
                dk[b, :, h] = dt_h.t() @ q / math.sqrt(D)
                if bucket is not None:
                    for u in range(case["buckets"]):
                        dt[u, h] += dt_h[bucket == u].sum()
    if not train:
        return out, lse
    return out, [dq, dk, dv] + ([dt] if bucket is not None else [])


def _pairs(case):
    """(query, key) pairs that take part, of one batch row and head; where the seed draws the mask, their mean."""
    Sq, Sk, mask = case["q_len"], case["kv_len"], case["mask"]
    if mask == "none":
        return Sq * Sk
    if mask in ("causal", "padded"):
        pad = max(0, 3 * (Sk - Sq) // 4 - 1) / 2 if mask == "padded" else 0.0
        return Sq * (Sk - Sq - pad) + Sq * (Sq + 1) / 2
    # documents: two tokens d apart share one with probability r^d; sum over d = 1 .. S - 1 of (S - d) r^d
    r = 1.0 - 1.0 / case["mean_document"]
    apart = r * (Sq * (1 - r) - 1 + r ** Sq) / (1 - r) ** 2
    return Sq + apart * (1 if mask.startswith("causal") else 2)


def work(case):
    B, H, D, Sq, Sk = (case[x] for x in ("batch", "heads", "dim", "q_len", "kv_len"))
    train = case["path"] == "train"
    keys = _pairs(case) if Sq == 1 else Sk  # a token reads the keys that it sees
    # q and out, k and v; behind them dO and dq, dk and dv; the table and its gradient
    data = 2 * (4 if train else 2) * B * H * D * (Sq + keys) + (0 if train else 4 * B * H * Sq) + (4 if train else 2) * case["buckets"] * H
    return {"bytes": float(data), "flops": float((12 if train else 4) * D * B * H * _pairs(case))}
