"""What stands around the attention layer in a sequence encoder's training step, as timed
cases: the token embedding with its gradient, the norms before and after a block with its
gate and the residual stream, and the norm and clipping of all gradients.

``run`` computes a case in its plain form (elementary torch operations in 32 bits) where
``own`` is false, and through the package's public functions where it is true.
"""
from __future__ import annotations

import math
import random

import torch

own = False

DTYPES = {"float32": torch.float32, "float16": torch.float16, "bfloat16": torch.bfloat16}
EPS = 1e-6


def _embed(name, V, B, L, D, **kw):
    # dtype: of the weight; out: of the embeddings; wide: tokens in 64 bits
    case = dict(op="embed", V=V, B=B, L=L, D=D, dtype="bfloat16", out="bfloat16", train=False,
                ragged=False, padding=False, wide=True, scale=1.0)
    case.update(kw)
    if name:
        case["name"] = name
    return case


def _residual(name, B, L, D, **kw):
    # dtype: of the residual stream; block: of the block's output and of the next one's input;
    # gate: none, or one for each feature, sequence or token; first: the norm before any block
    case = dict(op="residual", B=B, L=L, D=D, dtype="bfloat16", block="bfloat16", norm="rms",
                post="none", gate="none", first=False, train=False, scale=1.0, residual_scale=1.0)
    case.update(kw)
    if name:
        case["name"] = name
    return case


def _clip(name, tensors, total, **kw):
    # ratio: the largest norm allowed over the expected one; flat: the gradients are views of
    # one buffer for each type, with gaps, and so are the results; norm_only: no clipping
    case = dict(op="clip", tensors=tensors, total=total, dtype="float32", ratio=0.4, flat=False,
                norm_only=False)
    case.update(kw)
    if name:
        case["name"] = name
    return case


def listed():
    return [
        # one new token of a few sequences, where the launch is everything
        _embed("embed_token", 32, 8, 1, 256),
        # the encoder's training step on padded batches of protein-length sequences: 32-bit
        # weights, 16-bit activations, each letter thousands of times
        _embed("embed_letters", 21, 32, 512, 512, dtype="float32", train=True, ragged=True,
               padding=True, scale=512 ** 0.5),
        # words of six nucleotides and one for padding, odd lengths
        _embed("embed_words_odd", 4097, 3, 4099, 200, dtype="float16", out="float16", train=True,
               padding=True, wide=False),
        # words of eight, wide features, a whole training batch: the largest table
        _embed("embed_large", 65536, 16, 8192, 1024, train=True, scale=32.0),
        # between two layers while single tokens go through
        _residual("residual_token", 8, 1, 512, post="rms"),
        # the norm before the first layer, 32 bits throughout, long odd sequences
        _residual("residual_first", 3, 4097, 96, dtype="float32", block="float32", norm="layer",
                  first=True, train=True),
        # the encoder's training step: the residual stream in 32 bits, the block in 16, norms
        # on both sides and a learned scale for each feature
        _residual("residual_batch", 32, 512, 512, dtype="float32", post="rms", gate="feature",
                  train=True),
        # odd sizes, mean and variance on both sides, a gate that the model computes for each token
        _residual("residual_gated_odd", 5, 1023, 333, dtype="float16", block="float16",
                  norm="layer", post="layer", gate="token", train=True, scale=0.5,
                  residual_scale=1.25),
        # long sequences of wide features, conditioned on something said once for each: the largest
        _residual("residual_long", 4, 8192, 2048, gate="sequence", train=True, scale=0.25),
        # the gradients of a small encoder, as its own tensors
        _clip("clip_encoder", 18, 280_000),
        # hundreds of tensors of mixed types in one buffer a type, many small or odd
        _clip("clip_buckets", 301, 24_000_001, dtype="mixed", flat=True),
        # the gradients of a large encoder, which no cache holds
        _clip("clip_large", 40, 320_000_000, dtype="bfloat16"),
    ]


def _log_uniform(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["embed", "residual", "residual", "clip"])
    dtype = rng.choice(["bfloat16", "float16", "float32"])
    if op == "clip":
        flat = rng.random() < 0.5
        tensors = _log_uniform(rng, 1, 500 if flat else 60)
        return _clip(None, tensors, max(tensors, _log_uniform(rng, 100, 100_000_000)),
                     dtype=rng.choice([dtype, "mixed"]), flat=flat,
                     ratio=rng.choice([0.1, 0.5, 0.9, 2.0]), norm_only=rng.random() < 0.2)
    D = rng.choice([64, 128, 256, 512, 768, 1024, 8 * rng.randint(2, 256), rng.randint(16, 2048)])
    short = rng.choice([dtype, rng.choice(["bfloat16", "float16"])]) if dtype == "float32" else dtype
    rows = min(_log_uniform(rng, 1, 1 << 18), (1 << 26) // D)
    B = min(rows, _log_uniform(rng, 1, 64))
    L = max(1, rows // B)
    train = rng.random() < 0.75
    if op == "embed":
        V = min(_log_uniform(rng, 4, 1 << 17), (1 << 26) // D)
        return _embed(None, V, B, L, D, dtype=dtype, out=short, train=train,
                      ragged=rng.random() < 0.5, padding=rng.random() < 0.5,
                      wide=rng.random() < 0.6, scale=rng.choice([1.0, D ** 0.5]))
    if rng.random() < 0.15:
        return _residual(None, B, L, D, dtype=dtype, block=short, norm=rng.choice(["rms", "layer"]),
                         first=True, train=train)
    return _residual(None, B, L, D, dtype=dtype, block=short,
                     norm=rng.choice(["rms", "rms", "layer", "none"]),
                     post=rng.choice(["none", "rms", "layer"]),
                     gate=rng.choice(["none", "feature", "sequence", "token"]), train=train,
                     scale=rng.choice([1.0, 1.0, 0.5]), residual_scale=rng.choice([1.0, 1.0, 1.5]))


def _tensor_sizes(case):
    """[(size, type)] of the gradients: matrices of a network and vectors beside them."""
    n, total = case["tensors"], case["total"]
    rng = random.Random(n * 1000003 + total)
    share = [rng.choice([1.0, 1.0, 3.0, 4.0]) if rng.random() < 0.6 else 0.002 * rng.random()
             for _ in range(n)]
    left = total - n
    sizes = [1 + int(left * s / sum(share)) for s in share]
    sizes[-1] += total - sum(sizes)
    types = ["float32", "bfloat16", "float32", "float16"] if case["dtype"] == "mixed" else [case["dtype"]]
    return [(m, types[i % len(types)]) for i, m in enumerate(sizes)]


def _prepare_clip(case, g):
    sizes = _tensor_sizes(case)
    # each tensor's gradients are of a size of their own
    scales = [10.0 ** random.Random(i).uniform(-4, -1) for i in range(len(sizes))]
    expected = math.sqrt(sum(m * s * s for (m, _), s in zip(sizes, scales)))
    state = dict(case=case, max_norm=expected * case["ratio"])

    def fill(t, s):
        return t.copy_(torch.randn(t.shape, generator=g, device="cuda", dtype=torch.float32) * s)

    if not case["flat"]:
        state["grads"] = [fill(torch.empty(m, dtype=DTYPES[t], device="cuda"), s)
                          for (m, t), s in zip(sizes, scales)]
        return state
    # one buffer a type; every other tensor begins wherever the one before it ended
    ends, places = {}, []
    for i, (m, t) in enumerate(sizes):
        at = ends.get(t, 0)
        at += -at % 8 if i % 2 else 0
        places.append((t, at, at + m))
        ends[t] = at + m
    for name in ("grads", "out"):
        flat = {t: torch.zeros(n, dtype=DTYPES[t], device="cuda") for t, n in sorted(ends.items())}
        state[name + "_flat"] = list(flat.values())
        state[name] = [flat[t][a:b] for t, a, b in places]
    for t, s in zip(state["grads"], scales):
        fill(t, s)
    return state


def _token_counts(case):
    """How many tokens of each sequence of a padded batch are there: from half to all."""
    B, L = case["B"], case["L"]
    rng = random.Random(B * 1000003 + L)
    return [rng.randint((L + 1) // 2, L) if case["ragged"] else L for _ in range(B)]


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def randn(*shape, dtype, scale=1.0):
        return (torch.randn(shape, generator=g, device="cuda") * scale).to(DTYPES[dtype])

    if case["op"] == "clip":
        return _prepare_clip(case, g)
    s = dict(case=case)
    B, L, D = case["B"], case["L"], case["D"]
    if case["op"] == "embed":
        V = case["V"]
        # some tokens are far more frequent than others, the more so the more there are
        u = torch.rand((B, L), generator=g, device="cuda", dtype=torch.float64)
        rank = (u ** (1.3 if V < 64 else 3.0) * V).long().clamp(max=V - 1)
        names = torch.randperm(V, generator=g, device="cuda")
        s["tokens"] = names[rank].to(torch.int64 if case["wide"] else torch.int32)
        s["padding"] = int(V - 1) if case["padding"] else None
        s["lengths"] = None
        if case["ragged"]:
            counts = _token_counts(case)
            counts = counts[seed % B:] + counts[:seed % B]
            s["lengths"] = torch.tensor(counts, dtype=torch.int32, device="cuda")
        w = randn(V, D, dtype=case["dtype"], scale=1.0 / case["scale"])
        s["weight"] = w.requires_grad_(case["train"])
        if case["train"]:
            s["grad"] = randn(B, L, D, dtype=case["out"])
        return s
    s["x"] = randn(B, L, D, dtype=case["dtype"], scale=2.0)
    s["y"] = s["gate"] = None
    if not case["first"]:
        s["y"] = randn(B, L, D, dtype=case["block"])
    if case["gate"] == "feature":
        s["gate"] = 0.5 + randn(D, dtype="float32", scale=0.1)
    elif case["gate"] != "none":
        s["gate"] = randn(B, 1 if case["gate"] == "sequence" else L, D, dtype=case["block"])
    for name, kind in (("", case["norm"]), ("post_", case["post"])):
        s[name + "weight"] = 1.0 + randn(D, dtype="float32", scale=0.1) if kind != "none" else None
        s[name + "bias"] = randn(D, dtype="float32", scale=0.1) if kind == "layer" else None
    names = ("x", "y", "gate", "weight", "bias", "post_weight", "post_bias")
    if case["train"]:
        for name in names:
            if s[name] is not None:
                s[name] = s[name].detach().requires_grad_()
        s["grad_h"] = randn(B, L, D, dtype=case["dtype"])
        s["grad_n"] = randn(B, L, D, dtype=case["block"])
    s["leaves"] = [s[name] for name in names if s[name] is not None]
    return s


# ---------------------------------------------------------------- the package's functions

def _run_own(s):
    import d2p_amd
    c = s["case"]
    if c["op"] == "clip":
        if c["norm_only"]:
            return [d2p_amd.global_norm(s["grads"])]
        if c["flat"]:
            _, norm = d2p_amd.clip_gradients(s["grads"], s["max_norm"], out=s["out"])
            return [*s["out_flat"], norm]
        out, norm = d2p_amd.clip_gradients(s["grads"], s["max_norm"])
        return [*out, norm]
    if c["op"] == "embed":
        out = d2p_amd.token_embedding(s["tokens"], s["weight"], s["lengths"], scale=c["scale"],
                                      padding=s["padding"], dtype=DTYPES[c["out"]])
        if not c["train"]:
            return [out]
        return [out.detach(), *torch.autograd.grad(out, s["weight"], s["grad"])]
    name = {"none": None, "rms": "rms", "layer": "layer"}
    h, n = d2p_amd.residual_norm(
        s["x"], s["y"], s["weight"], s["bias"], norm=name[c["norm"]], post_norm=name[c["post"]],
        post_weight=s["post_weight"], post_bias=s["post_bias"], gate=s["gate"], scale=c["scale"],
        residual_scale=c["residual_scale"], eps=EPS, dtype=DTYPES[c["block"]])
    outs, grads = [], []
    if not c["first"]:
        outs, grads = [h], [s["grad_h"]] if c["train"] else []
    if c["norm"] != "none":
        outs = outs + [n]
        grads = grads + [s["grad_n"]] if c["train"] else []
    if not c["train"]:
        return outs
    return [t.detach() for t in outs] + list(torch.autograd.grad(outs, s["leaves"], grads))


# ---------------------------------------------------------------- plain forms, in 32 bits

def _embed_plain(s):
    c = s["case"]
    tokens, V, D = s["tokens"].long(), c["V"], c["D"]
    used = torch.ones_like(tokens, dtype=torch.bool)
    if s["lengths"] is not None:
        used = torch.arange(c["L"], device=tokens.device) < s["lengths"][:, None]
    if s["padding"] is not None:
        used = used & (tokens != s["padding"])
    used = used[..., None]
    w = s["weight"].detach()
    out = torch.where(used, w[tokens].float() * c["scale"], 0.0).to(DTYPES[c["out"]])
    if not c["train"]:
        return [out]
    g = torch.where(used, s["grad"].float(), 0.0).view(-1, D)
    dw = torch.zeros(V, D, device=g.device).index_add_(0, tokens.view(-1), g)
    return [out, (dw * c["scale"]).to(w.dtype)]


def _normed(x, kind):
    """x without its scale (and mean), and one over what it was divided by."""
    if kind == "layer":
        x = x - x.mean(-1, keepdim=True)
    r = torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS)
    return x * r, r


def _unnormed(g, normed, r, kind):
    """The gradient of what _normed took, g being that of what it gave."""
    if kind == "layer":
        g = g - g.mean(-1, keepdim=True)
    return r * (g - normed * (g * normed).mean(-1, keepdim=True))


def _affine(x, w, b):
    x = x * w
    return x if b is None else x + b


def _residual_plain(s):
    c = s["case"]
    f = {k: s[k].detach().float() if s[k] is not None else None
         for k in ("x", "y", "gate", "weight", "bias", "post_weight", "post_bias")}
    dt, bt = s["x"].dtype, DTYPES[c["block"]]
    h, gate = f["x"], 1.0 if f["gate"] is None else f["gate"]
    outs = []
    if not c["first"]:
        z = f["y"]
        if c["post"] != "none":
            yn, yr = _normed(z, c["post"])
            z = _affine(yn, f["post_weight"], f["post_bias"])
        h = c["residual_scale"] * h + c["scale"] * gate * z
        outs.append(h.to(dt))
    if c["norm"] != "none":
        hn, hr = _normed(h, c["norm"])
        outs.append(_affine(hn, f["weight"], f["bias"]).to(bt))
    if not c["train"]:
        return outs
    dh, sums = 0.0 if c["first"] else s["grad_h"].float(), []
    if c["norm"] != "none":
        dn = s["grad_n"].float()
        dh = dh + _unnormed(dn * f["weight"], hn, hr, c["norm"])
        sums.append((dn * hn).sum((0, 1)))
        if f["bias"] is not None:
            sums.append(dn.sum((0, 1)))
    if c["first"]:
        return outs + [dh.to(dt)] + sums
    grads = [(c["residual_scale"] * dh).to(dt)]
    dz, dgate = c["scale"] * gate * dh, []
    if f["gate"] is not None:
        t = c["scale"] * dh * z
        t = t.sum((0, 1)) if c["gate"] == "feature" else t.sum(1, keepdim=True) if c["gate"] == "sequence" else t
        dgate.append(t.to(s["gate"].dtype))
    if c["post"] != "none":
        sums.append((dz * yn).sum((0, 1)))
        if f["post_bias"] is not None:
            sums.append(dz.sum((0, 1)))
        dz = _unnormed(dz * f["post_weight"], yn, yr, c["post"])
    return outs + grads + [dz.to(bt)] + dgate + sums


def _clip_plain(s):
    c = s["case"]
    squares = torch.stack([g.float().square().sum() for g in s["grads"]])
    norm = squares.double().sum().sqrt()
    if c["norm_only"]:
        return [norm.float()]
    by = torch.where(norm <= s["max_norm"], 1.0, s["max_norm"] / norm).float()
    if c["flat"]:
        for g, o in zip(s["grads"], s["out"]):
            o.copy_(g.float() * by)
        return [*s["out_flat"], norm.float()]
    return [*((g.float() * by).to(g.dtype) for g in s["grads"]), norm.float()]


def run(state):
    if own:
        return _run_own(state)
    return {"embed": _embed_plain, "residual": _residual_plain, "clip": _clip_plain}[state["case"]["op"]](state)


# ---------------------------------------------------------------- the definitions, in 64 bits

def _embed_exact(s):
    c = s["case"]
    V, B, L, D = c["V"], c["B"], c["L"], c["D"]
    counts = s["lengths"].tolist() if s["lengths"] is not None else [L] * B
    t = s["tokens"].long().clone()
    for b, n in enumerate(counts):
        t[b, n:] = V                    # a row of zeros behind the table
    if s["padding"] is not None:
        t[t == s["padding"]] = V
    w = torch.cat((s["weight"].detach().double() * c["scale"],
                   torch.zeros(1, D, dtype=torch.float64, device="cuda")))
    out = [w[t]]
    if not c["train"]:
        return out
    # tokens in order: a row's gradient is the difference of two sums from the start
    order = torch.argsort(t.view(-1), stable=True)
    ends = torch.searchsorted(t.view(-1)[order], torch.arange(V + 1, device="cuda"))
    dw = torch.empty(V, D, dtype=torch.float64, device="cuda")
    g = s["grad"].view(-1, D)
    for a in range(0, D, 64):
        sums = torch.zeros(B * L + 1, min(64, D - a), dtype=torch.float64, device="cuda")
        torch.cumsum(g[order, a:a + 64].double(), 0, out=sums[1:])
        dw[:, a:a + 64] = c["scale"] * (sums[ends[1:]] - sums[ends[:-1]])
    return out + [dw]


def _residual_exact(s):
    c = s["case"]
    D = c["D"]

    def get(name, other=None):
        return s[name].detach().double() if s[name] is not None else other

    def spread(v, kind):
        m = v.sum(-1, keepdim=True) / D if kind == "layer" else 0.0
        return m, ((v - m).pow(2).sum(-1, keepdim=True) / D + EPS) ** 0.5

    def back(v, kind, g):
        """Of (v - m) / d: g / d, less what goes through d and through m."""
        m, d = spread(v, kind)
        t = g / d - (v - m) * (g * (v - m)).sum(-1, keepdim=True) / (D * d ** 3)
        return t - t.sum(-1, keepdim=True) / D if kind == "layer" else t

    h, gate, outs = get("x"), get("gate", 1.0), []
    if not c["first"]:
        y = z = get("y")
        if c["post"] != "none":
            m, d = spread(y, c["post"])
            z = (y - m) / d * get("post_weight") + get("post_bias", 0.0)
        h = h * c["residual_scale"] + gate * z * c["scale"]
        outs.append(h)
    if c["norm"] != "none":
        m, d = spread(h, c["norm"])
        hn = (h - m) / d
        outs.append(hn * get("weight") + get("bias", 0.0))
    if not c["train"]:
        return outs
    total, last = torch.zeros_like(h) if c["first"] else get("grad_h"), []
    if c["norm"] != "none":
        dn = get("grad_n")
        total = total + back(h, c["norm"], dn * get("weight"))
        last.append((dn * hn).flatten(0, 1).sum(0))
        if s["bias"] is not None:
            last.append(dn.flatten(0, 1).sum(0))
    if c["first"]:
        return outs + [total] + last
    grads = [total * c["residual_scale"]]
    total = total * c["scale"]
    dz = total * gate
    if c["post"] != "none":
        m, d = spread(y, c["post"])
        grads.append(back(y, c["post"], dz * get("post_weight")))
        last.append((dz * (y - m) / d).flatten(0, 1).sum(0))
        if s["post_bias"] is not None:
            last.append(dz.flatten(0, 1).sum(0))
    else:
        grads.append(dz)
    if s["gate"] is not None:
        grads.append((total * z).sum_to_size(s["gate"].shape))
    return outs + grads + last


def _clip_exact(s):
    c = s["case"]
    norm = torch.zeros((), dtype=torch.float64, device="cuda")
    for g in s["grads"]:
        norm += (g.double() ** 2).sum()
    norm = norm.sqrt()
    if c["norm_only"]:
        return [norm]
    by = min(1.0, s["max_norm"] / float(norm))
    if c["flat"]:
        return [*(g.double() * by for g in s["grads_flat"]), norm]   # the gaps are zeros
    return [*(g.double() * by for g in s["grads"]), norm]


def exact(case, seed):
    s = prepare(case, seed)
    return {"embed": _embed_exact, "residual": _residual_exact, "clip": _clip_exact}[case["op"]](s)


def work(case):
    size = {"float32": 4, "float16": 2, "bfloat16": 2}
    if case["op"] == "clip":
        n = sum(m * size[t] for m, t in _tensor_sizes(case))
        return {"bytes": n if case["norm_only"] else 2 * n,
                "flops": case["total"] * (2 if case["norm_only"] else 3)}
    B, L, D = case["B"], case["L"], case["D"]
    if case["op"] == "embed":
        used, V = sum(_token_counts(case)), case["V"]
        w, o, t = size[case["dtype"]], size[case["out"]], 8 if case["wide"] else 4
        n = {"bytes": B * L * D * o + min(V, used) * D * w + used * t, "flops": used * D}
        if case["train"]:       # the gradient read and the table's written
            n["bytes"] += used * D * o + V * D * w
            n["flops"] += used * D
        return n
    x, y, N = size[case["dtype"]], size[case["block"]], B * L * D
    block, norm = not case["first"], case["norm"] != "none"
    gate = {"none": 0, "feature": 4 * D, "sequence": B * D * y, "token": N * y}[case["gate"]]
    moved = N * (x * (2 if block else 1) + y * (block + norm)) + gate
    flops = N * (4 * norm + 4 * (case["post"] != "none") + 4 * block)
    if case["train"]:
        # the gradients of the results read; those of the stream, the block and the gate written
        moved += N * (x * (2 if block else 1) + y * (block + norm)) + gate
        flops *= 4
    return {"bytes": moved, "flops": flops}
