"""The attention layer of a sequence encoder, whose embeddings a caller multiplies into the
score matrices of the alignment functions: ``qk_norm_rope``, ``attention`` and the module
``SequenceAttention`` that runs them together.

No counterpart in the reference, whose callers bring finished scores.  All of it runs in
hand-written kernels on the HIP device, takes float32, float16 and bfloat16, and
differentiates once.  Tensors are laid out [batch, length, heads, features], so that the
heads of a projection are views of it; lengths are prefix lengths, as everywhere here.
"""
from __future__ import annotations

from typing import NamedTuple, Optional, Tuple, Union

import torch
import torch.nn as nn

from . import _ops  # noqa: F401  (loads the operator library)


def rope_tables(length: int, features: int, base: float = 10000.0,
                device=None) -> Tuple[torch.Tensor, torch.Tensor]:
    """Cosines and sines [length, features / 2] (float32) of the angles
    position * base^(-2 m / features)."""
    if features % 2 or features < 0:
        raise ValueError(f"rotated features must be even in number, got {features}")
    rate = base ** (-torch.arange(0, features, 2, dtype=torch.float64) / max(features, 1))
    angle = torch.arange(length, dtype=torch.float64)[:, None] * rate
    return angle.cos().float().to(device), angle.sin().float().to(device)


def relative_buckets(num_buckets: int, max_distance: int, bidirectional: bool = True,
                     device=None) -> torch.Tensor:
    """The bucket of each distance key - query from -max_distance to max_distance (int32
    [2 max_distance + 1]; further ones count as those ends), for ``attention``'s bias.

    The scheme of C. Raffel et al., "Exploring the limits of transfer learning with a unified
    text-to-text transformer" (JMLR 2020): near distances have a bucket each, the others
    share buckets of logarithmic width, keys ahead of the query have the upper half of the
    buckets (``bidirectional``) or bucket 0.
    """
    ways = 2 if bidirectional else 1
    n = num_buckets // ways
    if n < 1 or max_distance < 1 or max_distance > 1024:
        raise ValueError("need at least one bucket a direction and a max_distance from 1 to "
                         f"1024, got {num_buckets} and {max_distance}")
    exact = n // 2
    out = []
    for d in range(-max_distance, max_distance + 1):
        a = abs(d) if bidirectional else max(-d, 0)
        if a < exact or a == 0:
            b = min(a, n - 1)
        elif max_distance <= exact or exact == 0:
            b = n - 1
        else:
            # exact + floor((n - exact) log(a / exact) / log(max_distance / exact)), compared in
            # whole numbers: it reaches exact + t where (a / exact)^(n - exact) >=
            # (max_distance / exact)^t
            m, t = n - exact, 0
            while t + 1 < m and a ** m * exact ** (t + 1) >= max_distance ** (t + 1) * exact ** m:
                t += 1
            b = exact + t
        out.append(b + (n if bidirectional and d > 0 else 0))
    return torch.tensor(out, dtype=torch.int32, device=device)


def qk_norm_rope(q: torch.Tensor, k: torch.Tensor, q_weight: Optional[torch.Tensor] = None,
                 k_weight: Optional[torch.Tensor] = None, cos: Optional[torch.Tensor] = None,
                 sin: Optional[torch.Tensor] = None, positions: Optional[torch.Tensor] = None, *,
                 eps: float = 1e-6,
                 interleaved: bool = False) -> Tuple[torch.Tensor, torch.Tensor]:
    """Root-mean-square norm of each head of queries q [B, L, Hq, D] and keys k [B, L, Hkv, D]
    (D a multiple of 8 up to 128) and the rotation of their first features by position, in
    one pass.

    ``q_weight``, ``k_weight`` [D] scale the normed features (ones by default).  ``cos``,
    ``sin`` [rows, R / 2] (float32, see ``rope_tables``) rotate the first R features, row
    ``positions[b, l]`` for token l (int32 or int64 [B, L] or [L]; by default l); a token whose
    position the tables do not have comes back NaN.  Pairs are features m and m + R / 2, or
    2 m and 2 m + 1 with ``interleaved``.  Gradients flow to q, k and the weights.
    """
    if (cos is None) != (sin is None):
        raise ValueError("cos and sin go together")
    if cos is None:
        cos = sin = torch.empty((0, 0), dtype=torch.float32, device=q.device)
    if positions is not None:
        if positions.dtype == torch.int64:
            positions = positions.clamp(-1, 2 ** 31 - 1).to(torch.int32)
        if positions.dim() == 1:
            positions = positions.expand(q.shape[0], -1)
        positions = positions.contiguous()
    return torch.ops.d2p_amd.qk_norm_rope(q, k, q_weight, k_weight, cos, sin, positions,
                                          float(eps), interleaved)


def attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor,
              lengths: Optional[torch.Tensor] = None, *, causal: bool = False,
              scale: Optional[float] = None, bias: Optional[torch.Tensor] = None,
              buckets: Optional[torch.Tensor] = None, dropout: float = 0.0,
              seed: Union[int, torch.Tensor, None] = None) -> torch.Tensor:
    """Softmax attention of queries q [B, Lq, Hq, D] over keys and values k, v
    [B, Lk, Hkv, D]; Hq a multiple of Hkv, whose heads are shared in order; D a multiple of 8
    up to 128.  Returns [B, Lq, Hq, D].

    ``lengths`` (int32 [B, 2]): queries and keys of each element; rows past the queries are
    zeros, as are rows that see no key, and nothing past the lengths is used.  They are read
    on the device, so a call never waits; an element whose lengths do not lie within the
    tensors comes back NaN.  ``causal``: the last query sits on the last key, and a query sees
    no key ahead of it (so one query sees its whole cache).  ``scale``: D^-0.5 by default.

    ``bias`` [num_buckets, Hq] (float32 or q's type) with ``buckets`` (see
    ``relative_buckets``) adds a learned number to each score by the clipped distance from
    query to key.  ``dropout`` drops pairs after the softmax, with a probability held in
    256ths, and scales the others up by what that leaves; the mask comes from a counter-based
    generator keyed by ``seed`` (a number, or an int64 tensor of one on the device, which a
    graph can read anew on each replay) and is never stored.

    Gradients flow to q, k, v and bias.  Under torch.autocast the products run in its type.
    A tensor whose rows are not 16-byte aligned and at least a row apart is copied first.
    """
    if dropout and seed is None:
        raise ValueError("dropout needs a seed")
    key, key_tensor = 0, None
    if isinstance(seed, torch.Tensor):
        key_tensor = seed
    elif seed is not None:
        key = seed & (2 ** 64 - 1)
        key -= (key >> 63) << 64            # as a signed 64-bit number
    if scale is None:
        scale = max(q.shape[-1], 1) ** -0.5
    return torch.ops.d2p_amd.attention(q, k, v, lengths, causal, float(scale), bias, buckets,
                                       float(dropout), key, key_tensor)


def _lengths32(lengths: torch.Tensor) -> torch.Tensor:
    """Lengths in 32 bits; those of 64 that do not fit stay wrong ones."""
    if lengths.dtype == torch.int64:
        lengths = lengths.clamp(-1, 2 ** 31 - 1)
    return lengths.to(torch.int32)


class KeyValueCache(NamedTuple):
    """Keys and values [B, max length, Hkv, D] of the tokens seen so far, and how many there
    are of each sequence (int32 [B])."""
    keys: torch.Tensor
    values: torch.Tensor
    lengths: torch.Tensor


class SequenceAttention(nn.Module):
    """Self-attention layer of a sequence encoder: one projection to queries, keys and values,
    their norm and rotation, attention with a learned relative position bias
    (``num_buckets`` > 0) and dropout, and the output projection.

    ``forward(x, lengths)`` takes whole sequences x [B, L, dim]; ``step(x, cache)`` appends
    tokens to a cache and attends to it (causal layers).
    """

    def __init__(self, dim: int, heads: int, kv_heads: Optional[int] = None,
                 head_dim: Optional[int] = None, *, causal: bool = False, dropout: float = 0.0,
                 num_buckets: int = 0, max_distance: int = 128, max_length: int = 4096,
                 rope_base: float = 10000.0, eps: float = 1e-6):
        super().__init__()
        if heads < 1 or (kv_heads is not None and (kv_heads < 1 or heads % kv_heads)):
            raise ValueError(f"heads must be a positive multiple of kv_heads, got {heads} and "
                             f"{kv_heads}")
        if head_dim is None and dim % heads:
            raise ValueError(f"dim {dim} does not divide into {heads} heads; give head_dim")
        self.heads, self.kv_heads = heads, heads if kv_heads is None else kv_heads
        self.head_dim = dim // heads if head_dim is None else head_dim
        if self.head_dim % 8 or not 8 <= self.head_dim <= 128:
            raise ValueError(f"head_dim must be a multiple of 8 from 8 to 128, got {self.head_dim}")
        self.causal, self.dropout, self.eps = causal, dropout, eps
        self.qkv = nn.Linear(dim, (heads + 2 * self.kv_heads) * self.head_dim, bias=False)
        self.out = nn.Linear(heads * self.head_dim, dim, bias=False)
        self.q_norm = nn.Parameter(torch.ones(self.head_dim))
        self.k_norm = nn.Parameter(torch.ones(self.head_dim))
        cos, sin = rope_tables(max_length, self.head_dim, rope_base)
        self.register_buffer("cos", cos, persistent=False)
        self.register_buffer("sin", sin, persistent=False)
        self.bias = None
        self.register_buffer("buckets", None, persistent=False)
        if num_buckets:
            self.bias = nn.Parameter(torch.zeros(num_buckets, heads))
            self.buckets = relative_buckets(num_buckets, max_distance, not causal)

    def _apply(self, fn, recurse=True):
        # a layer moved to another type: the angles, which the kernels read in 32 bits, keep theirs
        tables = self.cos, self.sin
        super()._apply(fn, recurse)
        if self.cos.dtype != torch.float32:
            self.cos, self.sin = (t.to(self.cos.device) for t in tables)
        return self

    def _project(self, x, positions):
        B, L, _ = x.shape
        qkv = self.qkv(x).view(B, L, self.heads + 2 * self.kv_heads, self.head_dim)
        q, k, v = qkv.split((self.heads, self.kv_heads, self.kv_heads), dim=2)
        q, k = qk_norm_rope(q, k, self.q_norm, self.k_norm, self.cos, self.sin, positions,
                            eps=self.eps)
        return q, k, v

    def _attend(self, q, k, v, lengths, dropout=0.0, seed=None):
        bias = self.bias
        if bias is not None and bias.dtype not in (torch.float32, q.dtype):
            bias = bias.float()     # (a 16-bit layer and a cache of another type)
        return attention(q, k, v, lengths, causal=self.causal, bias=bias,
                         buckets=self.buckets, dropout=dropout, seed=seed).flatten(2)

    def forward(self, x: torch.Tensor, lengths: Optional[torch.Tensor] = None,
                seed: Union[int, torch.Tensor, None] = None) -> torch.Tensor:
        """x [B, L, dim], lengths int32 or int64 [B]; a dropping layer in training draws its seed from
        torch's generator unless it is given one."""
        q, k, v = self._project(x, None)
        if lengths is not None:
            lengths = _lengths32(lengths)[:, None].expand(-1, 2).contiguous()
        p = self.dropout if self.training else 0.0
        if p and seed is None:
            seed = torch.randint(-2 ** 63, 2 ** 63 - 1, (1,), device=x.device)
        return self.out(self._attend(q, k, v, lengths, p, seed))

    def _check_room(self, room):
        # past the tables a key would be NaN, and all that attend to it
        if room > self.cos.shape[0]:
            raise ValueError(f"a cache of {room} tokens exceeds the layer's max_length "
                             f"{self.cos.shape[0]}")

    def _check_step(self, batch, n, cache):
        if not self.causal:
            raise ValueError("step() needs a causal layer")
        there, room = cache.keys.shape[:2]
        if batch != there:
            raise ValueError(f"{batch} sequences beside a cache of {there}")
        if n > room:
            raise ValueError(f"{n} tokens do not fit a cache of {room}")
        self._check_room(room)

    def new_cache(self, batch: int, max_length: int, dtype=None) -> KeyValueCache:
        self._check_room(max_length)
        like = self.qkv.weight
        shape = (batch, max_length, self.kv_heads, self.head_dim)
        return KeyValueCache(torch.zeros(shape, dtype=dtype or like.dtype, device=like.device),
                             torch.zeros(shape, dtype=dtype or like.dtype, device=like.device),
                             torch.zeros(batch, dtype=torch.int32, device=like.device))

    @torch.no_grad()
    def step(self, x: torch.Tensor, cache: KeyValueCache) -> torch.Tensor:
        """New tokens x [B, n, dim] of each sequence: their keys and values go into the cache,
        whose lengths grow by n, and each attends to all before it.  The host does not know
        the lengths, so nothing waits: a sequence that outgrows its cache comes back NaN, in
        that call and all later ones, and so does one whose length is below zero."""
        self._check_step(x.shape[0], x.shape[1], cache)
        n, room = x.shape[1], cache.keys.shape[1]
        at = cache.lengths[:, None] + torch.arange(n, dtype=torch.int32, device=x.device)
        q, k, v = self._project(x, at)
        where = at.long().clamp(0, room - 1)[:, :, None, None].expand_as(k)
        cache.keys.scatter_(1, where, k.to(cache.keys.dtype))
        cache.values.scatter_(1, where, v.to(cache.values.dtype))
        # n queries; -1, which attention answers with NaN, where the length is below zero
        queries = cache.lengths >> 31 | n
        cache.lengths.add_(n)
        lengths = torch.stack((queries, cache.lengths), 1)
        o = self._attend(q.to(cache.keys.dtype), cache.keys, cache.values, lengths)
        return self.out(o.to(q.dtype))
