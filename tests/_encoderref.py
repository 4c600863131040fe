"""Plain 64-bit forms of the sequence-encoder operators and rounding bounds for them.

Unit roundoff u: 2^-24, 2^-11, 2^-8 for float32, float16, bfloat16.  The kernels hold
scores, statistics and sums in 32 bits and round P and dS (once each) and the results to the
inputs' type, so with eta a bound of the relative error of a probability from its score,
  |out - out*|  <= u |out| + (u + 4 eta) sum_j p d |v|
  |dv - dv*|    <= u |dv| + (u + 4 eta) sum_i p d |g|
  |ds - ds*|    <= p (4 eta (|dp| + |delta|) + (D + 8) 2^-24 sum |g v| + 2 u sum_j p d |g| |v|)
delta coming from the rounded result (its rounding, and P's in it), and dq, dk the sums of
(|ds error| + u |ds|) |k|, |q| plus u |dq|, |dk|; every result may also be off by half the
smallest number of its type.  eta = 2^-24 ((D + 8) max |s|_1 + Lk + 64),
|s|_1 the score with all its terms positive.
"""
import numpy as np
import torch

# a result below its type's normal numbers is rounded to a multiple of TINY * 2
TINY = {torch.float32: 2.0 ** -150, torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -134}
U = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}


def philox(c0, c1, c2, c3, k0, k1, rounds=7):
    """Philox4x32 (Salmon et al., SC 2011) on numpy arrays of 32-bit numbers."""
    x = [np.asarray(c, dtype=np.uint64) for c in (c0, c1, c2, c3)]
    m, s = np.uint64(0xffffffff), np.uint64(32)
    for r in range(rounds):
        ka, kb = np.uint64((k0 + r * 0x9E3779B9) & 0xffffffff), np.uint64((k1 + r * 0xBB67AE85) & 0xffffffff)
        a, b = x[0] * np.uint64(0xD2511F53), x[2] * np.uint64(0xCD9E8D57)
        x = [(b >> s) ^ x[1] ^ ka, b & m, (a >> s) ^ x[3] ^ kb, a & m]
    return x


def keep_mask(B, H, Lq, Lk, drop, seed):
    """[B, H, Lq, Lk]: byte j % 4 of word i % 4 of the 4 x 4 block's draw is at least drop."""
    seed &= 2 ** 64 - 1
    c2, c1, c0 = np.meshgrid(np.arange(B * H), np.arange((Lq + 3) // 4), np.arange((Lk + 3) // 4),
                             indexing="ij")
    w = philox(c0, c1, c2, np.zeros_like(c0), seed & 0xffffffff, seed >> 32)
    out = np.zeros((B * H, 4 * c0.shape[1], 4 * c0.shape[2]), dtype=bool)
    for i in range(4):
        for j in range(4):
            out[:, i::4, j::4] = ((w[i] >> np.uint64(8 * j)) & np.uint64(255)) >= drop
    return torch.from_numpy(out[:, :Lq, :Lk].reshape(B, H, Lq, Lk))


def attention(q, k, v, grad=None, lengths=None, causal=False, scale=None, bias=None,
              buckets=None, drop=0, seed=0):
    """(results, bounds): dicts of out, dq, dk, dv, dbias in float64 on the CPU."""
    u, tiny = U[q.dtype], TINY[q.dtype]
    ub, tinyb = (U[bias.dtype], TINY[bias.dtype]) if bias is not None else (0.0, 0.0)
    q, k, v = (t.detach().cpu().double() for t in (q, k, v))
    B, Lq, Hq, D = q.shape
    Lk, Hkv = k.shape[1], k.shape[2]
    scale = D ** -0.5 if scale is None else scale
    lens = lengths.tolist() if lengths is not None else [(Lq, Lk)] * B
    keep = keep_mask(B, Hq, Lq, Lk, drop, seed) if drop else None
    res = {"out": torch.zeros_like(q), "dq": torch.zeros_like(q), "dk": torch.zeros_like(k),
           "dv": torch.zeros_like(v)}
    err = {n: torch.zeros_like(t) for n, t in res.items()}
    if bias is not None:
        table, where = bias.detach().cpu().double(), buckets.cpu().long()
        R = where.numel() // 2
        for d in (res, err):
            d["dbias"] = torch.zeros_like(table)
    for b, (nq, nk) in enumerate(lens):
        at = torch.arange(nq)[:, None] + (nk - nq if causal else 0)
        rel = torch.arange(nk)[None] - at
        for h in range(Hq):
            f = h // (Hq // Hkv)
            Q, K, V = q[b, :nq, h], k[b, :nk, f], v[b, :nk, f]
            s = scale * Q @ K.T
            top = scale * Q.abs() @ K.abs().T
            if bias is not None:
                n = where[rel.clamp(-R, R) + R]
                s = s + table[n, h]
                top = top + table[n, h].abs().nan_to_num(0, posinf=0).clamp(max=1e4)
            if causal:
                s = s.masked_fill(rel > 0, -np.inf)
            p = torch.softmax(s, -1).nan_to_num(0.0) if nk else s
            if nk:
                p = torch.where((s == -np.inf).all(-1, keepdim=True), 0.0, p)
            eta = 2.0 ** -24 * ((D + 8) * (float(top.max()) if top.numel() else 0.0) + Lk + 64)
            w = torch.ones_like(p)
            if drop:
                w = keep[b, h, :nq, :nk] * (256.0 / (256 - drop))
            pd = p * w
            o = pd @ V
            res["out"][b, :nq, h] = o
            err["out"][b, :nq, h] = u * o.abs() + (u + 4 * eta) * pd @ V.abs()
            if grad is None:
                continue
            G = grad[b, :nq, h].detach().cpu().double()
            res["dv"][b, :nk, f] += pd.T @ G
            err["dv"][b, :nk, f] += (u + 4 * eta) * pd.T @ G.abs()
            dp = G @ V.T * w
            delta = (p * dp).sum(-1, keepdim=True)
            ds = p * (dp - delta)
            e = p * (4 * eta * (dp.abs() + delta.abs()) + (D + 8) * 2.0 ** -24 * (G.abs() @ V.abs().T) * w
                     + 2 * u * (pd * (G.abs() @ V.abs().T)).sum(-1, keepdim=True))
            res["dq"][b, :nq, h] = scale * ds @ K
            err["dq"][b, :nq, h] = scale * (e + u * ds.abs()) @ K.abs()
            res["dk"][b, :nk, f] += scale * ds.T @ Q
            err["dk"][b, :nk, f] += scale * (e + u * ds.abs()).T @ Q.abs()
            if bias is not None:
                res["dbias"][:, h].index_add_(0, n.flatten(), ds.flatten())
                # the sum itself in 32 bits, over a tree of sums of 32, tiles and blocks
                err["dbias"][:, h].index_add_(0, n.flatten(),
                                              (e + 2.0 ** -24 * 256 * ds.abs()).flatten())
    for n in ("dq", "dk", "dv"):
        err[n] += u * res[n].abs() + tiny
    err["out"] += tiny
    if bias is not None:
        err["dbias"] += ub * res["dbias"].abs() + tinyb
    return res, err


def norm_rope(x, w, cos, sin, positions, eps, interleaved, g=None):
    """(y, dx, dw) of one of q, k in float64 on the CPU, by matrices: y = M(position) (w xhat)."""
    x = x.detach().cpu().double()
    B, L, H, D = x.shape
    w = torch.ones(D, dtype=torch.float64) if w is None else w.detach().cpu().double()
    at = torch.arange(L).expand(B, L) if positions is None else positions.cpu().long()
    half = cos.shape[1]
    M = torch.eye(D, dtype=torch.float64).repeat(B, L, 1, 1)
    for m in range(half):
        a, c = (2 * m, 2 * m + 1) if interleaved else (m, m + half)
        co, si = cos.cpu().double()[at, m], sin.cpu().double()[at, m]
        M[:, :, a, a], M[:, :, a, c], M[:, :, c, c], M[:, :, c, a] = co, -si, co, si
    r = 1 / torch.sqrt((x * x).mean(-1, keepdim=True) + eps)
    n = x * r
    y = torch.einsum("blij,blhj->blhi", M, n * w)
    if g is None:
        return y, None, None
    t = torch.einsum("blji,blhj->blhi", M, g.detach().cpu().double())
    dw = (t * n).sum((0, 1, 2))
    t = t * w
    return y, r * (t - n * (t * n).mean(-1, keepdim=True)), dw
