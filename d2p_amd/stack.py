"""A sequence encoder around its attention layers: the token embedding, the norms before and
after each block with the residual stream, the module ``SequenceEncoder`` that runs them, and
the norm and clipping of a training step's gradients.

No counterpart in the reference, whose callers bring finished scores.  All of it runs in
hand-written kernels on the HIP device, takes float32, float16 and bfloat16, and
differentiates once.
"""
from __future__ import annotations

from typing import Iterable, List, Optional, Sequence, Tuple, Union

import torch
import torch.nn as nn

from . import _ops  # noqa: F401  (loads the operator library)
from .encoder import KeyValueCache, SequenceAttention, _lengths32

_NORMS = {None: 0, "rms": 1, "layer": 2}


def _norm_code(name, norm):
    if norm not in _NORMS:
        raise ValueError(f"{name} must be 'rms', 'layer' or None, got {norm!r}")
    return _NORMS[norm]


def token_embedding(tokens: torch.Tensor, weight: torch.Tensor,
                    lengths: Optional[torch.Tensor] = None, *, scale: float = 1.0,
                    padding: Optional[int] = None,
                    dtype: Optional[torch.dtype] = None) -> torch.Tensor:
    """``scale`` times the rows of weight [V, D] that tokens (int32 or int64, of any shape) name:
    [*tokens.shape, D], in ``dtype`` (weight's by default; 16 bits beside a float32 weight).  D
    is 8 at least.

    ``padding``: a token whose embeddings are zeros.  ``lengths`` (int32 [B], tokens [B, L]):
    positions past them are zeros too, whatever they hold.  Neither has a part in weight's
    gradient, which is summed in float32, in a fixed order.  Tokens and lengths are read on the
    device, so a call never waits: a token outside the table comes back NaN, as does a sequence
    whose length does not lie within 0 and L, and adds nothing to the gradient.
    """
    if padding is not None and not 0 <= padding < weight.shape[0]:
        raise ValueError(f"padding must be a token of {weight.shape[0]}, got {padding}")
    return torch.ops.d2p_amd.token_embedding(tokens, weight, lengths, float(scale),
                                             -1 if padding is None else padding,
                                             dtype or weight.dtype)


def residual_norm(x: torch.Tensor, y: Optional[torch.Tensor] = None,
                  weight: Optional[torch.Tensor] = None, bias: Optional[torch.Tensor] = None, *,
                  norm: Optional[str] = "rms", post_norm: Optional[str] = None,
                  post_weight: Optional[torch.Tensor] = None,
                  post_bias: Optional[torch.Tensor] = None, gate: Optional[torch.Tensor] = None,
                  scale: float = 1.0, residual_scale: float = 1.0, eps: float = 1e-6,
                  dtype: Optional[torch.dtype] = None
                  ) -> Tuple[torch.Tensor, Optional[torch.Tensor]]:
    """What stands between two blocks of a residual network, in one pass: y [B, L, D], the first
    block's output, joins the stream x [B, L, D] that went round it, and the next block's input
    is made of the two.  Returns (h, n):

        z = post_norm(y) * post_weight + post_bias
        h = residual_scale * x + scale * gate * z
        n = norm(h) * weight + bias

    Norms are "rms" (v / sqrt(mean(v^2) + eps)), "layer" (mean taken off first) or None (z is y;
    no n).  Vectors [D] of any type are ones and zeros by default.  ``gate``: [D], [B, 1, D]
    or [B, L, D], in float32 or y's type.  D is from 8 to 8192.

    h has x's type and n has y's: the same, or 16 bits beside a float32 stream.  Without y (the
    norm before the first block) h is x, and n has ``dtype`` (x's by default).  n is formed from
    h before h is rounded.  A row whose squares (a layer norm's: around its mean) pass float32 is
    normed to zeros.  Gradients flow to all tensors.
    """
    if y is None:
        if post_norm is not None or gate is not None or residual_scale != 1.0:
            raise ValueError("post_norm, gate and residual_scale need y")
        if norm is None:
            raise ValueError("nothing to do without y and norm")
    elif dtype is not None and dtype != y.dtype:
        raise ValueError(f"dtype is y's, got {dtype} and {y.dtype}")
    if norm is None and (weight is not None or bias is not None):
        raise ValueError("weight and bias need norm")
    if post_norm is None and (post_weight is not None or post_bias is not None):
        raise ValueError("post_weight and post_bias need post_norm")
    kind = y.dtype if y is not None else dtype or x.dtype
    h, n = torch.ops.d2p_amd.residual_norm(
        x, y, weight, bias, post_weight, post_bias, gate, _norm_code("norm", norm),
        _norm_code("post_norm", post_norm), float(scale), float(residual_scale), float(eps), kind)
    return (x if y is None else h), (None if norm is None else n)


def _some(tensors):
    tensors = list(tensors)
    if not tensors:
        raise ValueError("need at least one tensor")
    return tensors


def global_norm(tensors: Sequence[torch.Tensor]) -> torch.Tensor:
    """The 2-norm of all numbers of all tensors (of any of the three types, on one device), as a
    float32 scalar on the device; squares are summed in float64."""
    return torch.ops.d2p_amd.global_norm(_some(tensors))


def clip_gradients(tensors: Sequence[torch.Tensor], max_norm: float,
                   out: Optional[Sequence[torch.Tensor]] = None
                   ) -> Tuple[List[torch.Tensor], torch.Tensor]:
    """(results, norm): the tensors scaled by max_norm / norm if their ``global_norm`` is above
    ``max_norm``, as they are otherwise.  Nothing waits for the device.

    Results go to ``out`` if it is given: tensors of the same shapes and types, which may be
    the sources themselves but may not share memory otherwise.  New ones share one buffer.  An
    infinite norm scales by zero, a NaN makes all results NaN.
    """
    tensors = _some(tensors)
    if out is None:
        results, norm = torch.ops.d2p_amd.clip_gradients(tensors, float(max_norm))
        return results, norm
    out = list(out)
    if len(out) != len(tensors):
        raise ValueError(f"out must have {len(tensors)} tensors, got {len(out)}")
    return out, torch.ops.d2p_amd.clip_gradients_into(tensors, float(max_norm), out)


@torch.no_grad()
def clip_grad_norm_(parameters: Union[torch.Tensor, Iterable[torch.Tensor]],
                    max_norm: float) -> torch.Tensor:
    """Clips the gradients of ``parameters`` in place to a common 2-norm of ``max_norm`` at most,
    and returns the norm that they had (float32, on the device).  Parameters without a gradient
    are left out, one that is listed twice counts once.  The factor is max_norm / norm; torch's
    function of this name divides by norm + 1e-6."""
    parameters = [parameters] if isinstance(parameters, torch.Tensor) else list(parameters)
    grads = {id(p.grad): p.grad for p in parameters if p.grad is not None}
    if not grads:
        return torch.zeros((), device=parameters[0].device if parameters else None)
    grads = list(grads.values())
    return torch.ops.d2p_amd.clip_gradients_into(grads, float(max_norm), grads)


class SequenceEncoder(nn.Module):
    """Tokens to embeddings: a token embedding, ``layers`` of ``SequenceAttention`` around a
    residual stream with a norm before each (and, with ``post_norm``, after each), and a last
    norm.  ``gated``: a learned number for each feature of each layer's output, at first
    ``gated``.  Further options are the attention layers'.

    ``forward(tokens, lengths)`` gives [B, L, dim]; ``step(tokens, caches)`` appends tokens to
    the layers' caches (causal encoders).
    """

    def __init__(self, vocabulary: int, dim: int, heads: int, layers: int,
                 kv_heads: Optional[int] = None, *, norm: str = "rms",
                 post_norm: Optional[str] = None, gated: Optional[float] = None,
                 scale: float = 1.0, padding: Optional[int] = None, eps: float = 1e-6, **attention):
        super().__init__()
        if norm is None or _norm_code("norm", norm) == 0:
            raise ValueError("norm must be 'rms' or 'layer'")
        _norm_code("post_norm", post_norm)
        if padding is not None and not 0 <= padding < vocabulary:
            raise ValueError(f"padding must be a token of {vocabulary}, got {padding}")
        self.norm, self.post_norm, self.eps = norm, post_norm, eps
        self.scale, self.padding = scale, padding
        self.embedding = nn.Parameter(torch.randn(vocabulary, dim) / scale)
        self.layers = nn.ModuleList(SequenceAttention(dim, heads, kv_heads, eps=eps, **attention)
                                    for _ in range(layers))

        def vectors(n, value):
            return nn.ParameterList(nn.Parameter(torch.full((dim,), float(value)))
                                    for _ in range(n))

        self.weights = vectors(layers + 1, 1)
        self.biases = vectors(layers + 1 if norm == "layer" else 0, 0)
        self.post_weights = vectors(layers if post_norm else 0, 1)
        self.post_biases = vectors(layers if post_norm == "layer" else 0, 0)
        self.gates = vectors(layers if gated is not None else 0, gated or 0)

    def _run(self, tokens, lengths, attend):
        def at(vectors, i):
            return vectors[i] if len(vectors) else None

        x = token_embedding(tokens, self.embedding, lengths, scale=self.scale, padding=self.padding)
        kind = torch.get_autocast_dtype("cuda") if torch.is_autocast_enabled("cuda") else x.dtype
        x, n = residual_norm(x, None, self.weights[0], at(self.biases, 0), norm=self.norm,
                             eps=self.eps, dtype=kind if x.dtype == torch.float32 else None)
        for i, layer in enumerate(self.layers):
            y = attend(i, layer, n)
            if x.dtype != torch.float32:
                y = y.to(x.dtype)       # (a 16-bit stream under autocast to the other 16 bits)
            x, n = residual_norm(
                x, y, self.weights[i + 1], at(self.biases, i + 1), norm=self.norm,
                post_norm=self.post_norm, post_weight=at(self.post_weights, i),
                post_bias=at(self.post_biases, i), gate=at(self.gates, i), eps=self.eps)
        return n

    def forward(self, tokens: torch.Tensor, lengths: Optional[torch.Tensor] = None) -> torch.Tensor:
        """tokens [B, L], lengths int32 or int64 [B]; a dropping encoder in training draws its seeds
        from torch's generator."""
        if lengths is not None:
            lengths = _lengths32(lengths)
        return self._run(tokens, lengths, lambda i, layer, n: layer(n, lengths))

    def new_caches(self, batch: int, max_length: int, dtype=None) -> List[KeyValueCache]:
        return [layer.new_cache(batch, max_length, dtype) for layer in self.layers]

    @torch.no_grad()
    def step(self, tokens: torch.Tensor, caches: Sequence[KeyValueCache]) -> torch.Tensor:
        """New tokens [B, n] of each sequence, caches from ``new_caches``; see
        ``SequenceAttention.step``.  A call that is refused leaves all caches as they are."""
        if len(caches) < len(self.layers):
            raise ValueError(f"need a cache for each of {len(self.layers)} layers, got {len(caches)}")
        if tokens.dim() != 2:
            raise ValueError(f"tokens must be [B, n], got {tuple(tokens.shape)}")
        for layer, cache in zip(self.layers, caches):
            layer._check_step(*tokens.shape, cache)
        return self._run(tokens, None, lambda i, layer, n: layer.step(n, caches[i]))
