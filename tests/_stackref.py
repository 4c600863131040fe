"""Plain 64-bit forms of the operators around a sequence encoder's attention layers, and
rounding bounds for them.

e = 2^-24 is the roundoff of the 32 bits that everything is held in, u that of a tensor's type
(2^-24, 2^-11, 2^-8), which each result is rounded to once.  A sum of n terms in any order is
off by at most n e times the sum of their sizes.  The bounds follow the formulas term by term;
products of two roundoffs are covered by a factor of 1.01.
"""
import torch

E = 2.0 ** -24
U = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8,
     torch.float64: 0.0}
# a result below its type's normal numbers is rounded to a multiple of twice this
TINY = {torch.float32: 2.0 ** -150, torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -134,
        torch.float64: 0.0}


def rounded(bound, value, dtype):
    return 1.01 * bound + U[dtype] * value.abs() + TINY[dtype]


def double(t):
    return None if t is None else t.detach().cpu().double()


def embedding(tokens, weight, lengths=None, scale=1.0, padding=None, dtype=None, grad=None):
    """(out, its bound, dweight, its bound); rows of NaN where tokens or lengths are wrong."""
    dtype = dtype or weight.dtype
    w, t = double(weight), tokens.detach().cpu().long()
    V, D = w.shape
    used = torch.ones(t.shape, dtype=torch.bool)
    wrong = (t < 0) | (t >= V)
    if lengths is not None:
        n = lengths.cpu().long()
        used = torch.arange(t.shape[1]) < n[:, None]
        bad = ((n < 0) | (n > t.shape[1]))[:, None].expand(t.shape)
        wrong = (wrong & used) | bad
    if padding is not None:
        pads = t == padding
        if lengths is not None:
            pads = pads & ~bad
        used, wrong = used & ~pads, wrong & ~pads
    out = torch.zeros(*t.shape, D, dtype=torch.float64)
    rows = used & ~wrong
    out[rows] = scale * w[t[rows]]
    bound = rounded(2 * E * out.abs(), out, dtype)      # scale in 32 bits, and its product
    out[wrong] = float("nan")
    if grad is None:
        return out, bound, None, None
    g = double(grad)[rows]
    dw = torch.zeros(V, D, dtype=torch.float64).index_add_(0, t[rows], g)
    size = torch.zeros(V, D, dtype=torch.float64).index_add_(0, t[rows], g.abs())
    count = torch.zeros(V, dtype=torch.float64).index_add_(0, t[rows], torch.ones(int(rows.sum()),
                                                                                  dtype=torch.float64))
    dw = scale * dw
    return out, bound, dw, rounded(abs(scale) * (count[:, None] + 2) * E * size, dw, weight.dtype)


class _Norm:
    """One norm of v (whose numbers are off by dv): v's normed values, what they are off by."""

    def __init__(self, v, dv, kind, w, b, eps):
        D = v.shape[-1]
        self.kind, self.D = kind, D
        self.w = torch.ones(D, dtype=torch.float64) if w is None else w
        self.b = torch.zeros(D, dtype=torch.float64) if b is None else b
        self.m = v.mean(-1, keepdim=True) if kind == "layer" else torch.zeros_like(v[..., :1])
        c = v - self.m
        q = (c * c).mean(-1, keepdim=True) + eps
        self.r = 1 / torch.sqrt(q)
        # the mean's error, and the relative one of r: squares and their sum, the mean's
        # error (whose first order cancels), v's own
        self.dm = 0.0
        if kind == "layer":
            self.dm = (D + 4) * E * v.abs().mean(-1, keepdim=True) + dv.mean(-1, keepdim=True)
        off = dv + self.dm + 2 * E * (v.abs() + self.m.abs())
        self.dr = (D + 16) * E + ((c.abs() * (dv + 2 * E * (v.abs() + self.m.abs()))).mean(-1, keepdim=True)
                                  + (off * off).mean(-1, keepdim=True)) / q
        self.hat = c * self.r
        self.dhat = self.r * off + self.hat.abs() * (self.dr + 2 * E)
        self.out = self.hat * self.w + self.b
        self.dout = self.w.abs() * self.dhat + 2 * E * ((self.hat * self.w).abs() + self.b.abs())

    def back(self, g, dg, more):
        """(gradient of v, bound, gradient of w before its sum, bound), g off by dg; more: what
        v as the backward pass reads it is off by, relatively to r."""
        dhat = self.dhat + self.r * more
        a, da = g * self.w, dg * self.w.abs() + E * (g * self.w).abs()
        D = self.D
        m1 = a.mean(-1, keepdim=True) if self.kind == "layer" else torch.zeros_like(a[..., :1])
        dm1 = 0.0
        if self.kind == "layer":
            dm1 = (D + 4) * E * a.abs().mean(-1, keepdim=True) + da.mean(-1, keepdim=True)
        p = a * self.hat
        m2 = p.mean(-1, keepdim=True)
        dp = a.abs() * dhat + da * self.hat.abs()
        dm2 = (D + 4) * E * p.abs().mean(-1, keepdim=True) + dp.mean(-1, keepdim=True)
        t = a - m1 - self.hat * m2
        size = a.abs() + m1.abs() + (self.hat * m2).abs()
        dt = da + dm1 + dhat * m2.abs() + self.hat.abs() * dm2 + 4 * E * size
        return (self.r * t, self.r * (dt + t.abs() * (self.dr + 2 * E)), g * self.hat,
                g.abs() * dhat + dg * self.hat.abs() + E * (g * self.hat).abs())


def residual(x, y=None, weight=None, bias=None, norm="rms", post_norm=None, post_weight=None,
             post_bias=None, gate=None, scale=1.0, residual_scale=1.0, eps=1e-6, dtype=None,
             dh=None, dn=None):
    """(results, bounds): dicts of h, n, dx, dy, dgate, dweight, dbias, dpost_weight, dpost_bias."""
    kind = y.dtype if y is not None else dtype or x.dtype
    X, Y, G = double(x), double(y), double(gate)
    N = X.shape[0] * X.shape[1]
    res, off = {}, {}

    def put(name, value, bound, dtype):
        res[name], off[name] = value, rounded(bound, value, dtype)

    h, h_off, post = X, torch.zeros_like(X), None
    if Y is not None:
        z, dz_off = Y, torch.zeros_like(Y)
        if post_norm:
            post = _Norm(Y, torch.zeros_like(Y), post_norm, double(post_weight), double(post_bias), eps)
            z, dz_off = post.out, post.dout
        g = torch.ones_like(z) if G is None else G.expand_as(z)
        h = residual_scale * X + scale * g * z
        h_off = abs(scale) * g.abs() * dz_off + 5 * E * ((residual_scale * X).abs() + (scale * g * z).abs())
        put("h", h, h_off, x.dtype)
    n = None
    if norm:
        n = _Norm(h, h_off, norm, double(weight), double(bias), eps)
        put("n", n.out, n.dout, kind)
    if dh is None and dn is None:
        return res, off
    # the backward pass reads a float32 h as it was written, and forms others again
    read = E * h.abs()
    H, dH = (torch.zeros_like(X),) * 2
    if dh is not None:
        H = double(dh)

    def summed(name, v, dv, dims, dtype):
        count = v.numel() // max(1, v.sum(dims).numel())
        put(name, v.sum(dims), (count * E * v.abs()).sum(dims) + dv.sum(dims), dtype)

    if dn is not None and n is not None:
        d = double(dn)
        t, dt, w, dw = n.back(d, torch.zeros_like(d), read)
        H, dH = H + t, dt + E * (H.abs() + t.abs())
        if weight is not None:
            summed("dweight", w, dw, (0, 1), weight.dtype)
        if bias is not None:
            summed("dbias", d, torch.zeros_like(d), (0, 1), bias.dtype)
    if Y is None:
        put("dx", H, dH, x.dtype)
        return res, off
    put("dx", residual_scale * H, abs(residual_scale) * dH + 2 * E * (residual_scale * H).abs(), x.dtype)
    sH, dsH = scale * H, abs(scale) * dH + 2 * E * (scale * H).abs()
    if G is not None:
        t, dt = sH * z, dsH * z.abs() + sH.abs() * dz_off + E * (sH * z).abs()
        if G.dim() == 1:
            summed("dgate", t, dt, (0, 1), gate.dtype)
        elif G.shape[1] != X.shape[1]:
            summed("dgate", t, dt, (1,), gate.dtype)
            res["dgate"], off["dgate"] = res["dgate"][:, None], off["dgate"][:, None]
        else:
            put("dgate", t, dt, gate.dtype)
    dz, ddz = sH * g, dsH * g.abs() + E * (sH * g).abs()
    if post:
        t, dt, w, dw = post.back(dz, ddz, 0.0)
        if post_weight is not None:
            summed("dpost_weight", w, dw, (0, 1), post_weight.dtype)
        if post_bias is not None:
            summed("dpost_bias", dz, ddz, (0, 1), post_bias.dtype)
        dz, ddz = t, dt
    put("dy", dz, ddz, y.dtype)
    return res, off


def clipped(tensors, max_norm):
    """(results, bounds, norm): squares are summed in 64 bits, the factor is rounded once and
    its product once more."""
    ts = [double(t) for t in tensors]
    norm = sum(float((t * t).sum()) for t in ts) ** 0.5
    c = 1.0 if norm <= max_norm else max_norm / norm
    out = [c * t for t in ts]
    return out, [rounded(2 * E * o.abs(), o, t.dtype) for o, t in zip(out, tensors)], norm
