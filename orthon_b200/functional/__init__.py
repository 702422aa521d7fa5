"""Functional forms of composite operators.
(reference project: python/orthon/functional/math.py:39-96, functional/shape.py)"""
import builtins as _builtins
import math as _math
from functools import lru_cache as _lru_cache

import numpy as _np

from .. import _C
from .._random import randbits as _randbits


def layer_norm(tensor, normalized_shape, weight=None, bias=None, eps=1e-5):
    """Normalises the last dimension with one fused kernel (mean / rstd kept for backward)."""
    if isinstance(normalized_shape, int):
        normalized_shape = (normalized_shape,)
    normalized_shape = tuple(int(v) for v in normalized_shape)
    if len(normalized_shape) != 1:
        raise ValueError("layer_norm normalises the last dimension only")
    if tensor.shape[-1] != normalized_shape[0]:
        raise ValueError(
            f"layer_norm: normalized_shape {normalized_shape} does not match input shape {tuple(tensor.shape)}")
    return _C._layer_norm(tensor, weight, bias, float(eps))


def causal_mask(length, dtype="float32", device="cpu", fill=-1e9):
    """Additive [T, T] mask with `fill` above the diagonal."""
    import numpy as np
    m = np.triu(np.full((length, length), fill, dtype=np.float32), k=1)
    t = _C.from_numpy(m, dtype)
    return t if str(device) == "cpu" else t.to(device)


def scaled_dot_product_attention(q, k, v, mask=None, dropout_p=0.0, training=True, is_causal=False, seed=None):
    """softmax(q kᵀ / sqrt(d) + mask) v for [N, T, D] or [B, H, T, D] operands.

    The score scaling, additive mask, optional in-kernel causal mask and softmax are one
    kernel; scores stay in the operand dtype instead of a float32 [B·H, T, T] tensor."""
    if not 0.0 <= dropout_p < 1.0:
        raise ValueError("dropout_p must be in [0, 1)")
    scale = 1.0 / _math.sqrt(q.shape[-1])
    p = float(dropout_p) if training else 0.0
    if p > 0.0 and seed is None:
        seed = _randbits(64)
    return _C._attention(q, k, v, mask, bool(is_causal), scale, p, int(seed or 0))


def _rotary_scaling(scaling):
    """Checked (type, factor, original_length, beta_fast, beta_slow, attention_factor) of a scaling description."""
    if scaling is None:
        return None
    if not isinstance(scaling, dict) or scaling.get("type") not in ("linear", "ntk", "yarn"):
        raise ValueError("rotary scaling must be None or a dict whose 'type' is 'linear', 'ntk' or 'yarn'")
    kind, rest = scaling["type"], {k: v for k, v in scaling.items() if k != "type"}
    allowed = {"factor"} | ({"original_length", "beta_fast", "beta_slow", "attention_factor"} if kind == "yarn" else set())
    if set(rest) - allowed:
        raise ValueError(f"rotary scaling '{kind}' does not take {sorted(set(rest) - allowed)}")
    if rest.get("factor") is None or (kind == "yarn" and rest.get("original_length") is None):
        raise ValueError(f"rotary scaling '{kind}' needs " + ("'factor' and 'original_length'" if kind == "yarn" else "'factor'"))
    values = {"original_length": 1.0, "beta_fast": 32.0, "beta_slow": 1.0, **{k: v for k, v in rest.items() if v is not None}}
    for name, value in values.items():
        if not (float(value) > 0.0 and _math.isfinite(float(value))):
            raise ValueError(f"rotary scaling: {name} must be positive and finite")
    if values["beta_fast"] <= values["beta_slow"]:
        raise ValueError("rotary scaling: beta_fast must be larger than beta_slow")
    attention = values.get("attention_factor")
    return (kind, float(values["factor"]), float(values["original_length"]), float(values["beta_fast"]), float(values["beta_slow"]),
            None if attention is None else float(attention))


def _rotary_frequencies(rotary_dim, base, scaling):
    """(radians per position of each pair, factor on the turned values), in float64.

    f_i = base^(-2i/R).  'linear' divides every frequency by the factor; 'ntk' enlarges the base so that the slowest pair is
    stretched by the factor and the fastest not at all; 'yarn' (Peng et al., 2023) stretches pairs that turn less than
    beta_slow times over the original length, leaves those that turn more than beta_fast times, ramps in between, and
    enlarges queries and keys by 0.1 ln(factor) + 1 (not at all for a factor below 1)."""
    kind, factor, original, fast, slow, attention = scaling or (None, 1.0, 1.0, 32.0, 1.0, None)
    if kind == "ntk":
        if rotary_dim <= 2:
            raise ValueError("rotary scaling 'ntk' needs a rotary_dim of at least 4")
        base = base * factor ** (rotary_dim / (rotary_dim - 2))
    plain = [base ** (-2.0 * i / rotary_dim) for i in range(rotary_dim // 2)]
    if kind == "linear":
        return [f / factor for f in plain], 1.0
    if kind != "yarn":
        return plain, 1.0

    def pair_that_turns(times):
        return rotary_dim * _math.log(original / (times * 2.0 * _math.pi)) / (2.0 * _math.log(base))

    low, high = _builtins.max(_math.floor(pair_that_turns(fast)), 0), min(_math.ceil(pair_that_turns(slow)), rotary_dim - 1)
    span = high - low if high > low else 0.001
    ramp = [min(1.0, _builtins.max(0.0, (i - low) / span)) for i in range(rotary_dim // 2)]
    mixed = [f * (1.0 - r) + f / factor * r for f, r in zip(plain, ramp)]
    return mixed, 0.1 * _math.log(_builtins.max(factor, 1.0)) + 1.0 if attention is None else attention


@_lru_cache(maxsize=256)
def _rotary_plan(rotary_dim, base, scaling):
    """Turns per position (a float64 host tensor, as the kernels take it) and the magnitude of one configuration."""
    radians, magnitude = _rotary_frequencies(rotary_dim, base, scaling)
    return _C.from_numpy(_np.asarray(radians, dtype=_np.float64) / (2.0 * _np.pi)), magnitude


def _checked_rotary_plan(rotary_dim, base, scaling):
    if not (float(base) > 1.0 and _math.isfinite(float(base))):
        raise ValueError("rotary base must be finite and larger than 1")
    return _rotary_plan(rotary_dim, float(base), _rotary_scaling(scaling))


def _rotary_call(native, x, positions, rotary_dim, rotary_heads, base, interleaved, scaling, transposed):
    if x.ndim != 4:
        raise ValueError("rotary_embedding expects input with shape [B, T, H, D]")
    rotary_dim = int(x.shape[3] if rotary_dim is None else rotary_dim)
    if rotary_dim < 2 or rotary_dim % 2 or rotary_dim > x.shape[3]:
        raise ValueError(f"rotary_dim must be even and in [2, {x.shape[3]}], got {rotary_dim}")
    turns, magnitude = _checked_rotary_plan(rotary_dim, base, scaling)
    return native(x, positions, turns, magnitude, int(x.shape[2] if rotary_heads is None else rotary_heads), bool(interleaved), bool(transposed))


def rotary_embedding(x, positions=None, rotary_dim=None, rotary_heads=None, base=10000.0, interleaved=False, scaling=None, transposed=False):
    """Rotary positions for x [B, T, H, D]: pair i of a head at position p is turned by p * base^(-2i/rotary_dim).

    ``positions``: integer tensor [T] or [B, T] (default 0..T-1).  Pairs are (i, i + rotary_dim/2), or (2i, 2i+1) with
    ``interleaved``.  Only the first ``rotary_dim`` values of the first ``rotary_heads`` heads are turned, the rest is copied:
    a packed projection viewed as [B, T, 3H, D] turns its queries and keys with ``rotary_heads=2 * H``.  ``scaling`` stretches
    the angles for long contexts: ``{"type": "linear" | "ntk", "factor": f}`` or ``{"type": "yarn", "factor": f,
    "original_length": n}``.  ``transposed`` applies the transposed map (the opposite turn), which carries gradients back."""
    return _rotary_call(_C._rotary_embedding, x, positions, rotary_dim, rotary_heads, base, interleaved, scaling, transposed)


def rotary_embedding_(x, positions=None, rotary_dim=None, rotary_heads=None, base=10000.0, interleaved=False, scaling=None, transposed=False):
    """`rotary_embedding` in place: only the turned values are read and written."""
    return _rotary_call(_C._rotary_embedding_, x, positions, rotary_dim, rotary_heads, base, interleaved, scaling, transposed)


def paged_append_(k_pages, v_pages, k, v, page_table, starts, counts=None):
    """Writes new keys and values into the pages of a cache, in place.

    ``k_pages`` / ``v_pages`` [N, H, P, D] hold P tokens of every head per page; row b of ``page_table`` (int32 [B, M]) lists
    the pages of sequence b in order.  Token t of ``k`` / ``v`` [B, T, H, D] goes to place ``starts[b] + t`` (int32 [B]); only
    the first ``counts[b]`` tokens are written when ``counts`` (int32 [B]) is given, as for a padded batch.  Two sequences
    must not write to the same place.  On the CPU a place without a page raises; on CUDA it is left out and counted."""
    _C._paged_append_(k_pages, v_pages, k, v, page_table, starts, counts)
    return k_pages, v_pages


def copy_pages_(pages, sources, destinations, dim=0):
    """Copies pages of a contiguous tensor onto other pages along ``dim``, in place: the page ``destinations[i]`` becomes a copy
    of the page ``sources[i]``.  A page may be a source several times; destinations are distinct and no page is both."""
    return _C._copy_pages_(pages, sources, destinations, int(dim))


def paged_attention(q, k_pages, v_pages, page_table, lengths, scale=None):
    """Attention of one new token per sequence over a paged cache: softmax(scale q kᵀ) v for q [B, H, D] -> [B, H, D].

    Pages and ``page_table`` as in `paged_append_`; sequence b sees its first ``lengths[b]`` tokens (int32 [B]), whatever lies
    behind them in its pages.  The H query heads may be a multiple of the cached heads: neighbouring query heads share one.
    ``scale`` defaults to 1 / sqrt(D).  A sequence of length 0 gives zeros.  Has no gradient."""
    return _C._paged_attention(q, k_pages, v_pages, page_table, lengths, 1.0 / _math.sqrt(q.shape[-1]) if scale is None else float(scale))


def beam_search_step(logits, scores, finished=None, eos_token=None):
    """One selection of beam search: (scores, parents, tokens, finished), all [B, W], best first.

    ``logits`` [B, W, V] of the next token, ``scores`` (float32 [B, W]) the log-probabilities of the beams so far.  A beam w
    offers its V continuations at scores[w] + log_softmax(logits[w])[v]; a beam marked in ``finished`` (bool [B, W]) offers
    only itself, as ``eos_token`` at its score.  The W best of all are taken, ties to the lowest beam and then the lowest
    token.  ``parents`` and ``tokens`` (int64) tell the beam and the token of each; a beam is finished with its parent or with
    ``eos_token``.  A beam whose score is not finite, or whose logits have a NaN or +inf or are all -inf, offers nothing:
    its continuations count as -inf."""
    if eos_token is not None and int(eos_token) < 0:
        raise IndexError("beam_search_step: the end token is out of range")
    return _C._beam_search_step(logits, scores, finished, -1 if eos_token is None else int(eos_token))


def flatten(tensor, start_dim=0, end_dim=-1):
    return tensor.flatten(start_dim, end_dim)


from .._C import (  # noqa: E402,F401
    relu, sigmoid, tanh, leaky_relu, gelu, softmax, log_softmax, cross_entropy, nll_loss,
    dropout, embedding, conv2d, maxpool2d, linear, fused_linear_relu, matmul,
)


def exp(x):
    return x.exp()


def sum(x, dim=None, keepdim=False):  # noqa: A001 - mirrors the tensor method
    return x.sum(dim, keepdim)


def mean(x, dim=None, keepdim=False):
    return x.mean(dim, keepdim)


def max(x, dim=None, keepdim=False):  # noqa: A001
    return x.max(dim, keepdim)


def argmax(x, dim=None, keepdim=False):
    return x.argmax(dim, keepdim)
