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
MOST_AXES = 8
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
    multiplies cosines and sines.  Where positions have several axes, ``axes`` uint8 [rotary_dim / 2] says
    which of the ``axis_count`` each pair follows."""

    turns: torch.Tensor
    magnitude: float = 1.0
    axes: torch.Tensor | None = None
    axis_count: int = 1

    @property
    def rotary_dim(self) -> int:
        return 2 * self.turns.shape[0]

    @property
    def _arguments(self):
        return self.turns, self.axes, self.axis_count, self.magnitude


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
                 slow_turns=1.0, fast_turns=32.0, magnitude=1.0, sections=None, dealt=False, restart=False,
                 device="cuda") -> RotaryTable:
    """The table of ``rotary_frequencies`` on a device.  ``magnitude`` multiplies cosines and sines (some
    long-context scalings raise it above 1).

    ``sections``, for positions of several axes (time, height and width of a video, say): how many pairs
    follow each axis, ``rotary_dim / 2`` together.  The sections lie one behind the other or, ``dealt``, the
    pairs go to the axes in turn while their sections last.  The frequencies run on through all pairs or,
    with ``restart``, each axis has those of a ``rotary_dim`` of its own."""
    if not math.isfinite(magnitude):
        raise ValueError(f"magnitude must be finite, got {magnitude}")
    options = dict(base=base, scaling=scaling, factor=factor, original_length=original_length,
                   slow_turns=slow_turns, fast_turns=fast_turns)
    frequencies, axes = rotary_frequencies(rotary_dim, **options), None
    if sections is None:
        if dealt or restart:
            raise ValueError("dealt and restart need sections")
    else:
        sections = list(sections)
        axes = _axes_of_pairs(rotary_dim, sections, dealt)
        if restart:
            own = [iter(rotary_frequencies(2 * n, **options)) for n in sections]
            frequencies = [next(own[axis]) for axis in axes]
    units = [round(f / (2 * math.pi) * 2.0 ** 64) % 2 ** 64 for f in frequencies]
    signed = [u - 2 ** 64 if u >= 2 ** 63 else u for u in units]
    turns = torch.tensor(signed, dtype=torch.int64, device=device)
    if axes is None:
        return RotaryTable(turns, float(magnitude))
    return RotaryTable(turns, float(magnitude), torch.tensor(axes, dtype=torch.uint8, device=device), len(sections))


def _axes_of_pairs(rotary_dim, sections, dealt):
    if not 1 <= len(sections) <= MOST_AXES or any(not isinstance(n, int) or n <= 0 for n in sections):
        raise ValueError(f"sections must be 1 to {MOST_AXES} positive numbers of pairs, got {sections}")
    if 2 * sum(sections) != rotary_dim:
        raise ValueError(f"sections must add up to rotary_dim / 2 = {rotary_dim // 2}, got {sum(sections)}")
    if not dealt:
        return [axis for axis, n in enumerate(sections) for _ in range(n)]
    return [axis for turn in range(max(sections)) for axis, n in enumerate(sections) if turn < n]


def _check_table(rotary):
    if not isinstance(rotary, RotaryTable):
        raise TypeError(f"rotary must be a RotaryTable, got {type(rotary).__name__}")


def rotate_positions(x, positions, rotary, *, interleaved=False, transposed=False, out=None):
    """Rotates the first ``rotary.rotary_dim`` channels of every row of ``x`` by its position; the others
    are copied.

    ``x``: packed tokens [tokens, heads, head_dim] with ``positions`` [tokens], or [batch, heads, tokens,
    head_dim] with ``positions`` [tokens] or [batch, tokens]; float32, float16 or bfloat16, any strides with
    contiguous rows.  ``positions``: int32 or int64 (negative ones turn backwards); of a table with sections
    [axes, tokens] or [axes, batch, tokens], or [tokens] where all axes have the same.  Pair i is channels
    (i, i + rotary_dim / 2), or (2 i, 2 i + 1) where ``interleaved``.  ``transposed`` applies the transposed
    rotation (the inverse where the table's magnitude is 1).  ``out``: where to write, ``x`` itself included, no other
    view of its memory.

    Arithmetic is FP32 on angles reduced exactly; the gradient of ``x`` is the transposed rotation, from the
    same kernel.  Tensors with a forward-mode tangent are refused (its rotation is the same call)."""
    _check_table(rotary)
    if torch.is_grad_enabled() and x.requires_grad:
        if out is not None:
            raise ValueError("out cannot be given where x requires a gradient")
        return _native(x.device).rotate_with_gradient(x, positions, *rotary._arguments, bool(interleaved),
                                                      bool(transposed))
    return _native(x.device).rotate(x, positions, *rotary._arguments, bool(interleaved), bool(transposed), out,
                                    _stream(x.device))


# ---- the cache --------------------------------------------------------------------------------------------
@dataclass(frozen=True)
class KeyValueCache:
    """Pages of keys and values, [pages, kv_heads, page_size, head_dim] contiguous: float16 or bfloat16, or
    int8 codes with one FP32 scale per token and head, [pages, kv_heads, page_size].  Pages hold 16, 32, 64
    or 128 tokens of 64, 128 or 256 channels.  Which sequence owns which page is the caller's page table.

    Or 4-bit codes -7..7, two in a byte: uint8 [pages, kv_heads, page_size, head_dim / 2] with scales uint8
    [pages, kv_heads, page_size * (1 + head_dim / 16)].  A value is code * group scale * token scale.  Of each
    page and head the scales are first those of the tokens, powers of two as the exponent field of a float32
    (0: a scale of zero; 255: infinity, which makes the row NaN), then for each token those of its groups of
    16 channels: float8_e4m3fn numbers from 0 to 448, so neither a sign bit nor the NaN of that type (whoever
    fills a cache without ``append_to_cache`` sees to that; they are read by their bits and not checked).
    Channel 8 w + 2 i + j of a row is ``code + 8`` in bits 16 j + 4 i of its 32-bit word w."""

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
    def head_dim(self) -> int:
        return self.keys.shape[3] * (2 if self.keys.dtype == torch.uint8 else 1)

    @property
    def quantized(self) -> bool:
        return self.key_scales is not None


def allocate_key_value_cache(pages, kv_heads, page_size, head_dim, *, dtype=torch.bfloat16, device="cuda") -> KeyValueCache:
    """An empty cache; ``dtype`` torch.int8 allocates scales beside the codes, torch.uint8 is a cache in 4 bits."""
    shape = (pages, kv_heads, page_size, head_dim)
    if dtype == torch.uint8:
        shapes = ((*shape[:3], head_dim // 2),) * 2 + ((*shape[:2], page_size * (1 + head_dim // 16)),) * 2
        return KeyValueCache(*(torch.zeros(s, dtype=dtype, device=device) for s in shapes))
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

    With ``rotary`` the keys are rotated first, by ``positions`` [tokens] (of a table with sections also
    [axes, tokens]) or, without them, by those places; ``q`` [tokens, q_heads, head_dim] is rotated in the
    same launch and returned (None without it; rows behind the last sequence give 0).

    An int8 cache stores absmax / 127 as a token's scale and the codes rounded to nearest even.  A cache in 4
    bits stores the codes of the exactly rotated keys:

    token scale t  the smallest power of two, 2^-126 at least, with absmax <= 7 * 448 * t
    group scale g  the group's absmax / (7 t), rounded to e4m3
    code           x / (g t), rounded to nearest even, -7..7

    (a row that is not finite, or whose absmax needs a token scale above 2^119, becomes NaN)

    Tokens that their sequence is too short for are not written; a page outside the pool is not written
    either, and ``device_status()`` of the native module reports it.  Two sequences of a step must not share
    the pages they write to."""
    _check_cache(cache)
    if rotary is not None:
        _check_table(rotary)
    device = cache.keys.device
    return _native(device).cache_append(
        *cache.tensors, k, v, page_table, lengths, query_offsets, q,
        *((None, None, 1, 1.0) if rotary is None else rotary._arguments), bool(interleaved), positions, _stream(device))


def read_from_cache(cache, page_table, lengths, *, query_offsets=None, tokens=None, dtype=None):
    """Keys and values of a step's tokens as they lie in the cache, each [tokens, kv_heads, head_dim] (the step
    may be whole sequences).  Codes are read as the values they stand for, in ``dtype`` float16 or bfloat16.
    ``tokens``: rows of the result where ``query_offsets`` are given; those of no sequence, or that their sequence
    is too short for, give 0."""
    _check_cache(cache)
    if tokens is None:
        if query_offsets is not None:
            raise ValueError("with query_offsets the number of tokens must be given")
        tokens = page_table.shape[0]
    device = cache.keys.device
    return _native(device).cache_read(*cache.tensors, page_table, lengths, query_offsets, int(tokens), dtype, _stream(device))


def paged_attention(q, cache, page_table, lengths, *, query_offsets=None, scale=None, is_causal=True,
                    window=None, sinks=0, return_lse=False, out=None):
    """Attention of a step's new tokens ``q`` [tokens, q_heads, head_dim] over the cached keys of their
    sequences, the tokens' own included (append them first).  One token of each sequence, chunks of a
    prompt, or both in one call.

    With ``is_causal`` (aligned to the end: the last new token sees all ``lengths[s]`` keys) and ``window``
    a token sees the last ``window`` keys up to its own place and, of those in front of them, the first ``sinks``
    of the sequence; keys between them are not read, nor are their entries of the page table.  (Keys keep the
    rotation that they were appended with: in an endless conversation the distance to the first ones grows past
    what a model was trained on, unless the ``positions`` given to ``append_to_cache`` stay within it.)
    Without ``is_causal`` every token sees all.
    ``q_heads`` is a multiple of the cache's heads.  ``scale``: head_dim ** -0.5 unless given.  A token that
    sees nothing gives 0 and an LSE of -inf.  Rows of no sequence (behind the last, in front of the first) give
    the same; where ``out`` is given (``q`` itself included, no other view of its memory) its rows stay as they
    were.  Returns the output, with ``return_lse`` also the natural logarithm of the denominators, FP32
    [tokens, q_heads].

    Unlike ``int8_attention`` nothing is quantised on the way: scores, softmax and sums are FP32 over the
    cache's 16-bit values or codes as they are.  What is rounded for the product with V:

    * over 16-bit values the probability, to the type of ``q``;
    * over codes the probability times the key's scale, to float16, in units of the largest such product that
      the token sees: of two scales that differ by more than 2^24 the smaller one's values may be lost in that
      token (codes of 4 bits enter times their group's scale, which is exact);
    * over codes of 4 bits with bfloat16 queries, where a key head has 33 query rows or more of a sequence, the
      probability, to bfloat16 (the codes enter times all their scales, which is exact).

    A value that is not finite may also reach tokens of the same call that do not see its key: it is multiplied
    by their probability, 0."""
    _check_cache(cache)
    if scale is None:
        scale = q.shape[-1] ** -0.5
    output, lse = _native(q.device).paged_attention(
        q, *cache.tensors, page_table, lengths, query_offsets, float(scale), bool(is_causal), window,
        int(sinks), bool(return_lse), out, _stream(q.device))
    return (output, lse) if return_lse else output


def cached_key_weights(q, lse, cache, page_table, lengths, *, query_offsets=None, scale=None, is_causal=True,
                       window=None, sinks=0, previous=None):
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
        int(sinks), previous, _stream(q.device))


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


# ---- pages --------------------------------------------------------------------------------------------------
# ``references`` int32 [pages] counts for each page how many entries of page tables lead to it; a page with
# none is free.  (zeros for a new cache; every table whose pages are counted goes through these calls.)
def fork_sequences(cache, references, page_table, lengths, parents):
    """Sequences that begin as copies of others and share their pages (several answers to a prompt, beams):
    ``parents`` int32 [children] names a row of ``page_table`` for each (or none, -1: an empty sequence).
    Returns their page table [children, pages of a sequence], -1 behind their lengths, and their lengths;
    ``references`` counts the new entries.  Nothing is copied until one of them grows (``resize_sequences``)."""
    _check_cache(cache)
    device = cache.keys.device
    return _native(device).fork_sequences(*cache.tensors, references, page_table, lengths, parents, _stream(device))


def resize_sequences(cache, references, page_table, lengths, new_lengths):
    """Brings sequences to ``new_lengths`` int32 [batch] (at most what a row of ``page_table`` holds) and
    returns the lengths that were granted; ``page_table`` and ``references`` are changed in place.

    Before tokens are appended: a longer sequence gets the lowest free pages, in the order of the sequences;
    where its last page is not full and shared, a page of its own in place of that, with a copy of its
    tokens (each of those that share it, also where all of them grow in one call).  If pages run out it is
    granted the length that its pages hold (the old one, where a shared page could not be replaced).  A
    shorter one, or length 0, gives its pages back; they may be handed out from the next call on, by when
    nobody else may lead to them uncounted."""
    _check_cache(cache)
    device = cache.keys.device
    return _native(device).resize_sequences(*cache.tensors, references, page_table, lengths, new_lengths, _stream(device))


class Compaction(NamedTuple):
    """``page_table`` for the target's pages, -1 behind the lengths; ``references`` int32 [pages of the target];
    ``used`` int32 [1]: how many pages were in use."""

    page_table: torch.Tensor
    references: torch.Tensor
    used: torch.Tensor


def compact_cache(cache, references, page_table, lengths, target) -> Compaction:
    """Copies the pages in use, shared ones once and all in their order, to the front of ``target``, another
    cache with pages of the same kind (a smaller one, say, when most requests have left).  Where the target
    has fewer pages than ``used`` tells, the last ones are not copied and entries that led to them are -1."""
    _check_cache(cache)
    _check_cache(target)
    device = cache.keys.device
    return Compaction(*_native(device).cache_compact(*cache.tensors, references, page_table, lengths, *target.tensors, _stream(device)))
