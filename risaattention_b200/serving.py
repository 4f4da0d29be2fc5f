"""Serving: rotary positions, a paged key/value cache, attention of new tokens over it, and eviction from it
by the attention that its keys have received.  (The reference attends whole sequences and keeps nothing
between calls, so nothing here has a counterpart there.)

A step of a batch is described by three int32 tensors on the device: ``page_table`` [batch, pages of a
sequence], ``lengths`` [batch] (tokens of each sequence, this step's included) and ``query_offsets``
[batch + 1] (whose tokens are where in the packed tensors [tokens, heads, head_dim]; None: one token for
every sequence).  They are read by the kernels, never by the host: nothing here synchronises, and a captured
CUDA graph replays with whatever they hold by then.  Tokens behind ``query_offsets[-1]`` belong to nobody, so
a padded batch replays too.

All calls run on the current stream of the tensors' device and, rotation apart, are for inference: their
outputs carry no gradient."""
from __future__ import annotations

import math
from dataclasses import dataclass
from typing import NamedTuple

import torch

from . import _backend
from ._validation import UNAVAILABLE, is_available

PAGE_SIZES = (16, 32, 64, 128)
CACHE_HEAD_DIMS = (64, 128, 256)
ROTARY_SCALINGS = (None, "linear", "base", "parts")


def _native(device):
    if _backend._C is None:
        _backend.require_extension()
    if device.type == "cuda" and not is_available(device):
        raise RuntimeError(UNAVAILABLE)
    return _backend._C


def _stream(device):
    return _backend.current_stream_ptr(device) if device.type == "cuda" else 0


# ---- rotary positions ---------------------------------------------------------------------------------
@dataclass(frozen=True)
class RotaryTable:
    """Angle per position of every rotated pair of channels, ``turns`` int64 [rotary_dim / 2] in units of
    2^-64 turns (an angle matters modulo one turn, and positions are whole numbers, so the product with a
    position wraps exactly where the angle does and far positions lose nothing), and the factor that
    multiplies cosines and sines."""

    turns: torch.Tensor
    magnitude: float = 1.0

    @property
    def rotary_dim(self) -> int:
        return 2 * self.turns.shape[0]


def rotary_frequencies(rotary_dim, *, base=10000.0, scaling=None, factor=1.0, original_length=None,
                       slow_turns=1.0, fast_turns=32.0) -> list[float]:
    """Radians per position of each pair: ``base ** (-2 i / rotary_dim)``, scaled for contexts ``factor``
    times as long as the model was trained on:

    ``"linear"``  every pair turns ``factor`` times slower
    ``"base"``    the base is raised so that the slowest pair does, and the fastest stays
    ``"parts"``   pairs that make more than ``fast_turns`` turns over ``original_length`` stay, those of fewer
                  than ``slow_turns`` turn ``factor`` times slower, those between are blended linearly"""
    if not isinstance(rotary_dim, int) or rotary_dim <= 0 or rotary_dim % 2:
        raise ValueError(f"rotary_dim must be a positive even number, got {rotary_dim!r}")
    if scaling not in ROTARY_SCALINGS:
        raise ValueError(f"scaling must be one of {ROTARY_SCALINGS}, got {scaling!r}")
    if not (base > 1 and math.isfinite(base)):
        raise ValueError(f"base must be finite and larger than 1, got {base}")
    if not (factor > 0 and math.isfinite(factor)):
        raise ValueError(f"factor must be finite and positive, got {factor}")
    pairs = rotary_dim // 2
    if scaling == "base" and rotary_dim > 2:
        base = base * factor ** (rotary_dim / (rotary_dim - 2))
    plain = [base ** (-i / pairs) for i in range(pairs)]
    if scaling == "linear":
        return [f / factor for f in plain]
    if scaling == "parts":
        if original_length is None or original_length <= 0:
            raise ValueError("scaling by parts needs the positive original_length")
        if not fast_turns > slow_turns:
            raise ValueError("fast_turns must be larger than slow_turns")
        out = []
        for f in plain:
            turns = original_length * f / (2 * math.pi)
            keep = min(1.0, max(0.0, (turns - slow_turns) / (fast_turns - slow_turns)))
            out.append(f / factor * (1 - keep) + f * keep)
        return out
    return plain


def rotary_table(rotary_dim, *, base=10000.0, scaling=None, factor=1.0, original_length=None,
                 slow_turns=1.0, fast_turns=32.0, magnitude=1.0, device="cuda") -> RotaryTable:
    """The table of ``rotary_frequencies`` on a device.  ``magnitude`` multiplies cosines and sines (some
    long-context scalings raise it above 1)."""
    if not math.isfinite(magnitude):
        raise ValueError(f"magnitude must be finite, got {magnitude}")
    frequencies = rotary_frequencies(rotary_dim, base=base, scaling=scaling, factor=factor,
                                     original_length=original_length, slow_turns=slow_turns,
                                     fast_turns=fast_turns)
    units = [round(f / (2 * math.pi) * 2.0 ** 64) % 2 ** 64 for f in frequencies]
    signed = [u - 2 ** 64 if u >= 2 ** 63 else u for u in units]
    return RotaryTable(torch.tensor(signed, dtype=torch.int64, device=device), float(magnitude))


def _check_table(rotary):
    if not isinstance(rotary, RotaryTable):
        raise TypeError(f"rotary must be a RotaryTable, got {type(rotary).__name__}")


def rotate_positions(x, positions, rotary, *, interleaved=False, transposed=False, out=None):
    """Rotates the first ``rotary.rotary_dim`` channels of every row of ``x`` by its position; the others
    are copied.

    ``x``: packed tokens [tokens, heads, head_dim] with ``positions`` [tokens], or [batch, heads, tokens,
    head_dim] with ``positions`` [tokens] or [batch, tokens]; float32, float16 or bfloat16, any strides with
    contiguous rows.  ``positions``: int32 or int64 (negative ones turn backwards).  Pair i is channels
    (i, i + rotary_dim / 2), or (2 i, 2 i + 1) where ``interleaved``.  ``transposed`` applies the transposed
    rotation (the inverse where the table's magnitude is 1).  ``out``: where to write, ``x`` itself included, no other
    view of its memory.

    Arithmetic is FP32 on angles reduced exactly; the gradient of ``x`` is the transposed rotation, from the
    same kernel.  Tensors with a forward-mode tangent are refused (its rotation is the same call)."""
    _check_table(rotary)
    if torch.is_grad_enabled() and x.requires_grad:
        if out is not None:
            raise ValueError("out cannot be given where x requires a gradient")
        return _native(x.device).rotate_with_gradient(x, positions, rotary.turns, rotary.magnitude,
                                                      bool(interleaved), bool(transposed))
    return _native(x.device).rotate(x, positions, rotary.turns, rotary.magnitude, bool(interleaved),
                                    bool(transposed), out, _stream(x.device))


# ---- the cache --------------------------------------------------------------------------------------------
@dataclass(frozen=True)
class KeyValueCache:
    """Pages of keys and values, [pages, kv_heads, page_size, head_dim] contiguous: float16 or bfloat16, or
    int8 codes with one FP32 scale per token and head, [pages, kv_heads, page_size].  Pages hold 16, 32, 64
    or 128 tokens of 64, 128 or 256 channels.  Which sequence owns which page is the caller's page table."""

    keys: torch.Tensor
    values: torch.Tensor
    key_scales: torch.Tensor | None = None
    value_scales: torch.Tensor | None = None

    def __post_init__(self):
        _backend.require_extension()
        _backend._C.check_cache(*self.tensors)

    @property
    def tensors(self):
        return self.keys, self.values, self.key_scales, self.value_scales

    @property
    def page_size(self) -> int:
        return self.keys.shape[2]

    @property
    def quantized(self) -> bool:
        return self.keys.dtype == torch.int8


def allocate_key_value_cache(pages, kv_heads, page_size, head_dim, *, dtype=torch.bfloat16, device="cuda") -> KeyValueCache:
    """An empty cache; ``dtype`` torch.int8 allocates scales beside the codes."""
    shape = (pages, kv_heads, page_size, head_dim)
    keys, values = torch.zeros(shape, dtype=dtype, device=device), torch.zeros(shape, dtype=dtype, device=device)
    if dtype != torch.int8:
        return KeyValueCache(keys, values)
    return KeyValueCache(keys, values, torch.zeros(shape[:3], device=device), torch.zeros(shape[:3], device=device))


def _check_cache(cache):
    if not isinstance(cache, KeyValueCache):
        raise TypeError(f"cache must be a KeyValueCache, got {type(cache).__name__}")


def append_to_cache(cache, k, v, page_table, lengths, *, query_offsets=None, q=None, rotary=None,
                    positions=None, interleaved=False):
    """Writes a step's keys and values [tokens, kv_heads, head_dim] to their places: token i of the n new
    ones of sequence s is token ``lengths[s] - n + i`` of it.

    With ``rotary`` the keys are rotated first, by ``positions`` [tokens] or, without them, by those places;
    ``q`` [tokens, q_heads, head_dim] is rotated in the same launch and returned (None without it; rows
    behind the last sequence give 0).  An int8 cache stores absmax / 127 as a token's scale and the codes
    rounded to nearest even.  Tokens that their sequence is too short for are not written; a page outside
    the pool is not written either, and ``device_status()`` of the native module reports it.  Two sequences of
    a step must not share the pages they write to."""
    _check_cache(cache)
    if rotary is not None:
        _check_table(rotary)
    device = cache.keys.device
    return _native(device).cache_append(
        *cache.tensors, k, v, page_table, lengths, query_offsets, q, None if rotary is None else rotary.turns,
        1.0 if rotary is None else rotary.magnitude, bool(interleaved), positions, _stream(device))


def paged_attention(q, cache, page_table, lengths, *, query_offsets=None, scale=None, is_causal=True,
                    window=None, return_lse=False, out=None):
    """Attention of a step's new tokens ``q`` [tokens, q_heads, head_dim] over the cached keys of their
    sequences, the tokens' own included (append them first).  One token of each sequence, chunks of a
    prompt, or both in one call.

    With ``is_causal`` (aligned to the end: the last new token sees all ``lengths[s]`` keys) and ``window``
    a token sees the last ``window`` keys up to its own place; without ``is_causal`` every token sees all.
    ``q_heads`` is a multiple of the cache's heads.  ``scale``: head_dim ** -0.5 unless given.  A token that
    sees nothing gives 0 and an LSE of -inf.  Rows of no sequence (behind the last, in front of the first) give
    the same; where ``out`` is given (``q`` itself included, no other view of its memory) its rows stay as they
    were.  Returns the output, with ``return_lse`` also the natural logarithm of the denominators, FP32
    [tokens, q_heads].

    Unlike ``int8_attention`` nothing is quantised on the way: scores, softmax and sums are FP32 over the
    cache's 16-bit values or codes as they are; probabilities are rounded to the type of ``q`` for the product
    with V.  Over a cache of codes it is probability times the key's scale that is rounded, to float16, in units
    of the largest such product that the token sees: of two scales that differ by more than 2^24 the smaller one's
    values may be lost in that token.  A value that is not finite may also reach tokens of the same call
    that do not see its key: it is multiplied by their probability, 0."""
    _check_cache(cache)
    if scale is None:
        scale = q.shape[-1] ** -0.5
    output, lse = _native(q.device).paged_attention(
        q, *cache.tensors, page_table, lengths, query_offsets, float(scale), bool(is_causal), window,
        bool(return_lse), out, _stream(q.device))
    return (output, lse) if return_lse else output


def cached_key_weights(q, lse, cache, page_table, lengths, *, query_offsets=None, scale=None, is_causal=True,
                       window=None, previous=None):
    """The attention that each cached key received from a step's tokens: FP32 [batch, kv_heads, pages of a
    sequence * page_size], the sum of the probabilities over the sequence's new tokens and the query heads
    of the key's head.  ``q``, ``lse`` and the options as in ``paged_attention(..., return_lse=True)``;
    ``previous`` (weights of earlier steps) is added.  Keys that no token sees hold 0 or what ``previous``
    gave."""
    _check_cache(cache)
    if scale is None:
        scale = q.shape[-1] ** -0.5
    return _native(q.device).key_weights(
        q, lse, *cache.tensors, page_table, lengths, query_offsets, float(scale), bool(is_causal), window,
        previous, _stream(q.device))


class Eviction(NamedTuple):
    """``kept`` int32 [batch, kv_heads, budget]: the places that stayed, ascending, -1 behind the last;
    ``lengths`` int32 [batch]; ``weights`` FP32 [batch, kv_heads, pages of target_table * page_size]: theirs,
    in their new places, 0 behind the last."""

    kept: torch.Tensor
    lengths: torch.Tensor
    weights: torch.Tensor


def evict_from_cache(cache, page_table, lengths, weights, target_table, *, budget, recent=0) -> Eviction:
    """Shortens every sequence to ``budget`` tokens: each key head keeps the ``recent`` last ones and, of the
    others, those of the largest ``weights`` (as ``cached_key_weights`` gives them; of equal ones the
    earliest), and copies them in their order to the pages of ``target_table`` int32 [batch, pages], which
    takes the place of ``page_table`` from then on.  Sequences that are no longer than the budget are copied
    whole.  NaN counts as the largest weight.

    The target pages must belong to the sequence alone and be none that the call reads; the old pages are
    the caller's again afterwards (they are not written, so they may be shared).  Keys were rotated when
    they were appended and heads keep different tokens, so new tokens need explicit ``positions`` from
    here on."""
    _check_cache(cache)
    device = cache.keys.device
    return Eviction(*_native(device).cache_evict(*cache.tensors, page_table, lengths, weights, target_table,
                                                 int(budget), int(recent), _stream(device)))
