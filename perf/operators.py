"""The attention layer of a sequence encoder, as timed cases: per-head norms of queries
and keys with the position rotation, attention with its gradients, the learned relative
position bias and the dropout inside it.  The embeddings that such an encoder makes are
what a user multiplies into the score matrices of the alignment functions.

``run`` computes a case in its plain form (elementary torch operations in 32 bits) where
``own`` is false, and through the package's public functions where it is true.
"""
from __future__ import annotations

import math
import random

import torch

own = False

DTYPES = {"float32": torch.float32, "float16": torch.float16, "bfloat16": torch.bfloat16}


def _rope(name, B, L, Hq, Hkv, D, **kw):
    case = dict(op="rope", B=B, L=L, Hq=Hq, Hkv=Hkv, D=D, R=D, dtype="bfloat16", train=False,
                interleaved=False, packed=False, positions=False)
    case.update(kw)
    if name:
        case["name"] = name
    return case


def _attention(name, B, Lq, Lk, Hq, Hkv, D, **kw):
    case = dict(op="attention", B=B, Lq=Lq, Lk=Lk, Hq=Hq, Hkv=Hkv, D=D, dtype="bfloat16",
                train=False, causal=False, ragged=False, buckets=0, distance=0, dropout=0.0)
    case.update(kw)
    if name:
        case["name"] = name
    return case


def listed():
    return [
        # the smallest call: one new token of a few sequences, where the launch is everything
        _rope("rope_token", 8, 1, 16, 4, 64, positions=True),
        # a training batch of protein-length sequences, queries and keys as views of one
        # projection of queries, keys and values
        _rope("rope_batch", 32, 512, 8, 8, 64, train=True, packed=True),
        # long odd sequences in 32 bits, part of each head rotated, neighbours as pairs
        _rope("rope_long_odd", 3, 4097, 12, 2, 96, R=64, dtype="float32", train=True,
              interleaved=True),
        # one pair of short sequences attending to each other (unit tests, notebooks)
        _attention("attn_pair", 2, 100, 120, 4, 4, 32, dtype="float32", train=True),
        # the encoder's training step: ragged protein-length sequences, with everything on
        _attention("attn_batch", 32, 512, 512, 8, 8, 64, train=True, ragged=True, buckets=32,
                   distance=128, dropout=0.1),
        # causal training on genome-scale rows with wide heads
        _attention("attn_long", 2, 4096, 4096, 16, 16, 128, train=True, causal=True),
        # shared heads, an odd length and a head size between the usual ones
        _attention("attn_groups_odd", 4, 1023, 1023, 12, 3, 80, dtype="float16", train=True,
                   causal=True, ragged=True, dropout=0.2),
        # training without mixed precision, as the alignment sweeps themselves run
        _attention("attn_float", 4, 1024, 1024, 8, 8, 64, dtype="float32", train=True,
                   buckets=64, distance=256),
        # embedding long sequences: the forward alone, the largest call
        _attention("attn_embed_long", 2, 8192, 8192, 16, 16, 128),
        # one new token for each of a batch of sequences, heads shared by four
        _attention("attn_token", 16, 1, 4096, 32, 8, 128, causal=True, ragged=True),
        # a few tokens at the end of one very long sequence
        _attention("attn_tokens_long", 1, 4, 100003, 16, 2, 64, dtype="float16", causal=True,
                   buckets=32, distance=128),
        # causal training with bias and dropout over longer rows
        _attention("attn_bias_dropout", 4, 2048, 2048, 8, 8, 64, train=True, causal=True,
                   buckets=32, distance=128, dropout=0.1),
    ]


def _log_uniform(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    dtype = rng.choice(["bfloat16", "bfloat16", "float16", "float32"])
    Hkv = rng.choice([1, 2, 3, 4, 8])
    Hq = Hkv * rng.choice([1, 1, 2, 4])
    D = rng.choice([32, 64, 64, 128, 128, 8 * rng.randint(1, 16)])
    if rng.random() < 0.2:
        L = _log_uniform(rng, 1, 8192)
        B = _log_uniform(rng, 1, max(1, min(64, (1 << 25) // (L * Hq * D))))
        return _rope(None, B, L, Hq, Hkv, D, R=D if rng.random() < 0.6 else 2 * rng.randint(1, D // 2),
                     dtype=dtype, train=rng.random() < 0.7, interleaved=rng.random() < 0.4,
                     packed=rng.random() < 0.5, positions=rng.random() < 0.4)
    kind = rng.choice(["self", "self", "self", "cross", "tokens"])
    if kind == "tokens":
        Lq, Lk = rng.choice([1, 1, 1, 2, 3, 4, 8]), _log_uniform(rng, 8, 131072)
    else:
        Lq = _log_uniform(rng, 2, 4096)
        Lk = Lq if kind == "self" else _log_uniform(rng, 2, 4096)
    room = 1 << (25 if dtype == "float32" else 27)
    while Hq * Lq * Lk > room:
        Lq, Lk = (Lq + 1) // 2, (Lk + 1) // 2
    most = max(1, min(64, room // (Hq * Lq * Lk), (1 << 28) // (Hkv * Lk * D)))
    case = _attention(None, _log_uniform(rng, 1, most), Lq, Lk, Hq, Hkv, D, dtype=dtype,
                      train=kind != "tokens" and rng.random() < 0.75,
                      causal=kind == "tokens" or (kind == "self" and rng.random() < 0.5),
                      ragged=rng.random() < 0.4)
    if rng.random() < 0.4:
        case["buckets"], case["distance"] = rng.choice([(16, 32), (32, 128), (64, 256), (33, 100)])
    if case["train"] and rng.random() < 0.4:
        case["dropout"] = rng.choice([0.05, 0.1, 0.1, 0.25, 0.5])
    return case


def _lengths(case):
    """[(query length, key length)] of a ragged batch: from half to all of each length."""
    B, Lq, Lk = case["B"], case["Lq"], case["Lk"]
    if not case["ragged"]:
        return [(Lq, Lk)] * B
    rng = random.Random(B * 1000003 + Lq * 1009 + Lk)
    out = []
    for _ in range(B):
        lk = rng.randint((Lk + 1) // 2, Lk)
        lq = lk if Lq == Lk else Lq if Lq <= 8 else rng.randint((Lq + 1) // 2, Lq)
        out.append((lq, lk))
    return out


def _bucket_of(distance, buckets, most):
    """Signed distances to buckets: half of them for keys ahead, half for keys behind; the
    near distances one by one, the far ones by their logarithm."""
    half = buckets // 2
    exact = max(1, half // 2)
    n = min(abs(distance), most)
    if n < exact or exact == half:
        b = min(n, half - 1)
    else:
        b = min(half - 1, exact + int(math.log(n / exact + 1e-9) / math.log(most / exact) * (half - exact)))
    return b + (half if distance > 0 else 0)


def _tables(L, R):
    t = torch.arange(L, dtype=torch.float64)[:, None]
    f = 10000.0 ** (-torch.arange(0, R, 2, dtype=torch.float64) / R)
    return (t * f).cos().float().cuda(), (t * f).sin().float().cuda()


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt = DTYPES[case["dtype"]]
    B, Hq, Hkv, D = case["B"], case["Hq"], case["Hkv"], case["D"]

    def randn(*shape, dtype=dt, scale=1.0):
        return (torch.randn(shape, generator=g, device="cuda") * scale).to(dtype)

    s = dict(case=case)
    if case["op"] == "rope":
        L = case["L"]
        if case["packed"]:
            qkv = randn(B, L, Hq + 2 * Hkv, D)
            q, k = qkv[:, :, :Hq], qkv[:, :, Hq:Hq + Hkv]
        else:
            q, k = randn(B, L, Hq, D), randn(B, L, Hkv, D)
        wq = 1.0 + randn(D, dtype=torch.float32, scale=0.1)
        wk = 1.0 + randn(D, dtype=torch.float32, scale=0.1)
        table = max(2 * L, 64) if case["positions"] else L
        s["cos"], s["sin"] = _tables(table, case["R"])
        s["positions"] = torch.randint(0, table, (B, L), generator=g, device="cuda",
                                       dtype=torch.int32) if case["positions"] else None
        if case["train"]:
            s["grads"] = (randn(B, L, Hq, D), randn(B, L, Hkv, D))
        s["q"], s["k"], s["wq"], s["wk"] = (t.detach().requires_grad_(case["train"])
                                            for t in (q, k, wq, wk))
        return s

    Lq, Lk = case["Lq"], case["Lk"]
    q, k, v = randn(B, Lq, Hq, D), randn(B, Lk, Hkv, D), randn(B, Lk, Hkv, D)
    s["lengths"] = None
    if case["ragged"]:
        lens = _lengths(case)
        lens = lens[seed % B:] + lens[:seed % B]
        s["lengths"] = torch.tensor(lens, dtype=torch.int32, device="cuda")
    s["bias"] = s["map"] = None
    leaves = [q, k, v]
    if case["buckets"]:
        n, most = case["buckets"], case["distance"]
        leaves.append(randn(n, Hq))
        s["map"] = torch.tensor([_bucket_of(d, n, most) for d in range(-most, most + 1)],
                                dtype=torch.int32, device="cuda")
    leaves = [t.detach().requires_grad_(case["train"]) for t in leaves]
    s["q"], s["k"], s["v"] = leaves[:3]
    s["bias"] = leaves[3] if case["buckets"] else None
    s["leaves"] = leaves
    s["seed"] = torch.randint(0, 1 << 62, (1,), generator=g, device="cuda", dtype=torch.int64) \
        if case["dropout"] else None
    if case["train"]:
        s["grad"] = randn(B, Lq, Hq, D)
    return s


# ---------------------------------------------------------------- the package's functions

def _run_own(s):
    import d2p_amd
    c = s["case"]
    if c["op"] == "rope":
        q, k = d2p_amd.qk_norm_rope(s["q"], s["k"], s["wq"], s["wk"], s["cos"], s["sin"],
                                    s["positions"], interleaved=c["interleaved"])
        if not c["train"]:
            return [q, k]
        return [q.detach(), k.detach(),
                *torch.autograd.grad((q, k), (s["q"], s["k"], s["wq"], s["wk"]), s["grads"])]
    out = d2p_amd.attention(s["q"], s["k"], s["v"], s["lengths"], causal=c["causal"],
                            bias=s["bias"], buckets=s["map"], dropout=c["dropout"], seed=s["seed"])
    if not c["train"]:
        return [out]
    return [out.detach(), *torch.autograd.grad(out, s["leaves"], s["grad"])]


# ---------------------------------------------------------------- plain forms, in 32 bits

def _turn(x, cos, sin, R, interleaved):
    """The first R features of x rotated by the angles of cos and sin (broadcast [.., R/2])."""
    r, rest = x[..., :R], x[..., R:]
    a, b = (r[..., 0::2], r[..., 1::2]) if interleaved else (r[..., :R // 2], r[..., R // 2:])
    u, v = a * cos - b * sin, b * cos + a * sin
    r = torch.stack((u, v), -1).flatten(-2) if interleaved else torch.cat((u, v), -1)
    return torch.cat((r, rest), -1)


def _rope_plain(s):
    c = s["case"]
    R, il = c["R"], c["interleaved"]
    at = s["positions"].long() if s["positions"] is not None else torch.arange(c["L"], device="cuda")[None]
    cos, sin = s["cos"][at][:, :, None], s["sin"][at][:, :, None]
    dt = s["q"].dtype
    outs, dxs, dws = [], [], []
    for x, w, g in zip((s["q"], s["k"]), (s["wq"], s["wk"]),
                       s["grads"] if c["train"] else (None, None)):
        x, w = x.detach().float(), w.detach()
        r = torch.rsqrt((x * x).mean(-1, keepdim=True) + 1e-6)
        h = x * r
        outs.append(_turn(h * w, cos, sin, R, il).to(dt))
        if g is not None:
            b = _turn(g.float(), cos, -sin, R, il)
            dws.append((b * h).sum((0, 1, 2)))
            b = b * w
            dxs.append((r * (b - h * (b * h).mean(-1, keepdim=True))).to(dt))
    return outs + dxs + dws


def _philox(c0, c1, c2, seed):
    """Philox4x32 with 7 rounds on the counters (c0, c1, c2, 0): four int64 tensors of words."""
    m = 0xffffffff
    x = [c0, c1, c2, torch.zeros_like(c0)]
    k0, k1 = seed & m, (seed >> 32) & m
    for _ in range(7):
        a, b = x[0] * 0xD2511F53, x[2] * 0xCD9E8D57     # the low 64 bits; >> then & drops the sign
        x = [((b >> 32) & m) ^ x[1] ^ k0, b & m, ((a >> 32) & m) ^ x[3] ^ k1, a & m]
        k0, k1 = (k0 + 0x9E3779B9) & m, (k1 + 0xBB67AE85) & m
    return x


def _keep(B, H, Lq, Lk, p, seed):
    """[B, H, Lq, Lk] truth values: byte j % 4 of word i % 4 of the 4 x 4 block's draw is at
    least the drop probability in 256ths."""
    dev = seed.device
    nq, nk = (Lq + 3) // 4, (Lk + 3) // 4
    c2, c1, c0 = torch.meshgrid(torch.arange(B * H, device=dev), torch.arange(nq, device=dev),
                                torch.arange(nk, device=dev), indexing="ij")
    words = torch.stack(_philox(c0, c1, c2, seed), 2)           # [BH, nq, 4 rows, nk]
    shift = torch.arange(0, 32, 8, device=dev)
    bits = (words[..., None] >> shift) & 255                    # [BH, nq, 4, nk, 4 columns]
    return (bits >= round(p * 256)).reshape(B, H, 4 * nq, 4 * nk)[:, :, :Lq, :Lk]


def _attention_plain(s):
    c = s["case"]
    B, Lq, Lk, Hq, Hkv, D = (c[n] for n in ("B", "Lq", "Lk", "Hq", "Hkv", "D"))
    G, dev, dt, scale = Hq // Hkv, s["q"].device, s["q"].dtype, c["D"] ** -0.5

    def heads(x, groups):                                       # [B, L, H, D] -> [B, Hq, L, D]
        return x.detach().float().transpose(1, 2).repeat_interleave(groups, 1)

    q, k, v = heads(s["q"], 1), heads(s["k"], G), heads(s["v"], G)
    lq = s["lengths"][:, 0].long() if s["lengths"] is not None else torch.full((B,), Lq, device=dev)
    lk = s["lengths"][:, 1].long() if s["lengths"] is not None else torch.full((B,), Lk, device=dev)
    i = torch.arange(Lq, device=dev)[None, :, None]
    j = torch.arange(Lk, device=dev)[None, None, :]
    at = i + (lk - lq)[:, None, None] if c["causal"] else i     # a query's place among the keys
    seen = (i < lq[:, None, None]) & (j < lk[:, None, None])
    if c["causal"]:
        seen = seen & (j <= at)
    seen = seen[:, None]                                        # [B, 1, Lq, Lk]
    a = scale * (q @ k.transpose(-1, -2))
    if c["buckets"]:
        where = s["map"].long()[(j - at).clamp(-c["distance"], c["distance"]) + c["distance"]]
        a += s["bias"].detach().float()[where].permute(0, 3, 1, 2)
    a = torch.where(seen, a, float("-inf"))
    top = a.amax(-1, keepdim=True)
    a = torch.exp(a - torch.where(top.isinf(), 0.0, top))
    total = a.sum(-1, keepdim=True)
    a = a / torch.where(total > 0, total, 1.0)                  # a row that sees nothing: zeros
    keep = 1.0
    if c["dropout"]:
        keep = _keep(B, Hq, Lq, Lk, c["dropout"], s["seed"]) / (1 - round(c["dropout"] * 256) / 256)
    ad = a * keep
    out = ad @ v
    back = lambda x: x.transpose(1, 2).contiguous().to(dt)      # noqa: E731
    if not c["train"]:
        return [back(out)]
    do = torch.where((i < lq[:, None, None])[:, None], heads(s["grad"], 1), 0.0)
    join = lambda x: x.reshape(B, Hkv, G, Lk, D).sum(2)         # noqa: E731
    dv = join(ad.transpose(-1, -2) @ do)
    da = (do @ v.transpose(-1, -2)) * keep
    ds = a * (da - (a * da).sum(-1, keepdim=True))
    grads = [back(out), back(scale * (ds @ k)), back(join(scale * (ds.transpose(-1, -2) @ q))), back(dv)]
    if c["buckets"]:
        # row by row, so that no sum in 32 bits takes more than a row at a time
        sums = torch.zeros(B, Hq, Lq, c["buckets"], device=dev)
        sums.scatter_add_(3, where[:, None].expand(B, Hq, Lq, Lk), ds)
        grads.append(sums.sum((0, 2)).t().contiguous().to(dt))
    return grads


def run(state):
    if own:
        return _run_own(state)
    return _rope_plain(state) if state["case"]["op"] == "rope" else _attention_plain(state)


# ---------------------------------------------------------------- the definitions, in 64 bits

def _rope_exact(s):
    c = s["case"]
    B, L, D, R = c["B"], c["L"], c["D"], c["R"]
    at = s["positions"].long() if s["positions"] is not None else \
        torch.arange(L, device="cuda").expand(B, L)
    # a pair of features as one complex number, turned by a product
    first = torch.arange(R // 2, device="cuda") * (2 if c["interleaved"] else 1)
    second = first + (1 if c["interleaved"] else R // 2)
    unit = torch.complex(s["cos"].double(), s["sin"].double())[at][:, :, None]

    def turn(x, by):
        z, y = torch.complex(x[..., first], x[..., second]) * by, x.clone()
        y[..., first], y[..., second] = z.real, z.imag
        return y

    outs, dx, dw = [], [], []
    for name, g in (("q", 0), ("k", 1)):
        x, w = s[name].detach().double(), s["w" + name].detach().double()
        norm = torch.sqrt((x ** 2).sum(-1, keepdim=True) / D + 1e-6)
        outs.append(turn(x / norm * w, unit))
        if c["train"]:
            gn = turn(s["grads"][g].double(), unit.conj())
            dw.append((gn * x / norm).sum((0, 1, 2)))
            gh = gn * w
            dx.append(gh / norm - x * (gh * x).sum(-1, keepdim=True) / (D * norm ** 3))
    return outs + dx + dw


def _kept_exact(H, b, h, Lq, Lk, p, seed):
    """The same draw, the products put together from 16-bit halves so that none overflows."""
    m = 0xffffffff

    def product(x, k):
        lo, hi = (x & 0xffff) * k, (x >> 16) * k
        mid = (lo >> 16) + (hi & 0xffffffff)
        return (hi >> 32 << 16) + (mid >> 16) & m, ((mid & 0xffff) << 16 | lo & 0xffff) & m

    i, j = torch.arange(Lq, device="cuda"), torch.arange(Lk, device="cuda")
    w0 = (j // 4).expand((Lq + 3) // 4, Lk)[:, ::4]
    w1 = (i[::4] // 4)[:, None].expand_as(w0)
    w2, w3 = torch.full_like(w0, b * H + h), torch.zeros_like(w0)
    k0, k1 = seed % (1 << 32), seed // (1 << 32)
    for r in range(7):
        h0, l0 = product(w0, 0xD2511F53)
        h1, l1 = product(w2, 0xCD9E8D57)
        w0, w1, w2, w3 = h1 ^ w1 ^ ((k0 + r * 0x9E3779B9) & m), l1, \
            h0 ^ w3 ^ ((k1 + r * 0xBB67AE85) & m), l0
    words = torch.stack((w0, w1, w2, w3))[(i % 4)[:, None], (i // 4)[:, None], (j // 4)[None]]
    return words // (1 << 8 * (j % 4)) % 256 >= round(256 * p)


def _attention_exact(s):
    c = s["case"]
    B, Lq, Lk, Hq, Hkv, D = (c[n] for n in ("B", "Lq", "Lk", "Hq", "Hkv", "D"))
    q, k, v = (s[n].detach().double() for n in "qkv")
    z = lambda t: torch.zeros_like(t)                           # noqa: E731
    out, dq, dk, dv = z(q), z(q), z(k), z(v)
    n = c["buckets"]
    db = torch.zeros(n, Hq, dtype=torch.float64, device="cuda")
    lens = s["lengths"].tolist() if s["lengths"] is not None else [(Lq, Lk)] * B
    seed = int(s["seed"]) if s["seed"] is not None else 0
    for b, (nq, nk) in enumerate(lens):
        rel = torch.arange(nk, device="cuda") - torch.arange(nq, device="cuda")[:, None]
        if c["causal"]:
            rel = rel - (nk - nq)
        if n:
            where = s["map"].long()[rel.clamp(-c["distance"], c["distance"]) + c["distance"]]
        for h in range(Hq):
            f = h * Hkv // Hq
            Q, K, V = q[b, :nq, h], k[b, :nk, f], v[b, :nk, f]
            a = Q @ K.T / math.sqrt(D)
            if n:
                a += s["bias"].detach().double()[:, h][where]
            if c["causal"]:
                a.masked_fill_(rel > 0, float("-inf"))
            a = torch.softmax(a, -1).nan_to_num(0.0)            # rows with no keys: zeros
            w = 1.0
            if c["dropout"]:
                w = _kept_exact(Hq, b, h, Lq, Lk, c["dropout"], seed)[:nq, :nk] * \
                    (256 / (256 - round(256 * c["dropout"])))
            out[b, :nq, h] = (a * w) @ V
            if c["train"]:
                do = s["grad"][b, :nq, h].double()
                dv[b, :nk, f] += (a * w).T @ do
                da = do @ V.T * w
                ds = a * da - a * (a * da).sum(-1, keepdim=True)
                dq[b, :nq, h] = ds @ K / math.sqrt(D)
                dk[b, :nk, f] += ds.T @ Q / math.sqrt(D)
                if n:
                    rows = torch.zeros(nq, n, dtype=torch.float64, device="cuda")
                    db[:, h] += rows.scatter_add_(1, where, ds).sum(0)
    return [out] + ([dq, dk, dv] + ([db] if n else []) if c["train"] else [])


def exact(case, seed):
    s = prepare(case, seed)
    return _rope_exact(s) if case["op"] == "rope" else _attention_exact(s)


def work(case):
    size = 4 if case["dtype"] == "float32" else 2
    B, Hq, Hkv, D = case["B"], case["Hq"], case["Hkv"], case["D"]
    if case["op"] == "rope":
        n = B * case["L"] * (Hq + Hkv) * D
        rows = B * case["L"] if case["positions"] else case["L"]    # of the angles' tables
        # forward: read and write; training reads the gradients and writes theirs too
        return {"bytes": n * size * (4 if case["train"] else 2) + rows * case["R"] * 4,
                "flops": n * (24 if case["train"] else 8)}
    lens = _lengths(case)
    if case["causal"]:                      # query i of nq sees nk - nq + i + 1 keys, at least none
        pairs = sum(sum(range(max(0, nk - nq) + 1, nk + 1)) if nk > nq else nk * (nk + 1) // 2
                    for nq, nk in lens)
    else:
        pairs = sum(nq * nk for nq, nk in lens)
    rows, keys = sum(nq for nq, _ in lens) * Hq * D, sum(nk for _, nk in lens) * Hkv * D
    # forward: q, k, v read, the result written (2 products); training: the result's gradient
    # read, three gradients written (5 products more)
    extra = case["buckets"] * Hq * size * (2 if case["train"] else 1)
    if case["train"]:
        return {"bytes": (4 * rows + 4 * keys) * size + extra, "flops": 14 * pairs * Hq * D}
    return {"bytes": (2 * rows + 2 * keys) * size + extra, "flops": 4 * pairs * Hq * D}
